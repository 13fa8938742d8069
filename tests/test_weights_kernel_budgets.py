"""The kernels of 4-bit rows, of the sums of attention weights and of eviction as
the Makefile builds them (CPU only): their names, registers, LDS, no spills."""
import os
import re
import shlex
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "qwen3.8_27b_in_rust_amd", "csrc")
HIPCC = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "hipcc")
TYPES = ("f16", "bf16", "q8k", "mxfp4")

#: kernels of each file, and the registers that its workgroups launch with: 8 waves 256, the rows' four workgroups a CU 64,
#: 16 waves 128, the others what they have
KERNELS = {
    "attn_decode_mxfp4": ([f"q38_attn_decode_mxfp4{p}" for p in ("", "_pre", "_one", "_pre_one")], 256),
    "kv_rows_mxfp4": ([f"q38_kv_{c}_mxfp4{s}" for c in ("append", "gather") for s in ("", "_few")], 64),
    "attn_weigh": ([f"q38_attn_weigh_{t}{p}" for t in TYPES for p in ("", "_pre")] + ["q38_attn_weigh_merge"], 256),
    "attn_observe": ([f"q38_observe_{c}_{t}" for c in ("stats", "sums") for t in TYPES + ("bf16_few", "mxfp4_few")] +
                     [f"q38_observe_stats_{t}" for t in [t + "_short" for t in TYPES] + ["bf16_short_few", "mxfp4_short_few"]] +
                     ["q38_observe_add"], 256),
    "kv_weights": (["q38_kv_weights_copy", "q38_kv_evict_select"] + [f"q38_kv_evict_move_{t}" for t in TYPES], 128),
}


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_budgets(tmp_path, name):
    if not os.path.exists(HIPCC) or shutil.which("make") is None:
        pytest.skip("needs hipcc and make")
    plan = subprocess.run(["make", "-n", "-B", "-C", CSRC], check=True, capture_output=True, text=True).stdout
    words = shlex.split(next(ln for ln in plan.splitlines() if f"/{name}.hsaco" in ln and "--genco" in ln))
    words[words.index("-o") + 1] = str(tmp_path / "a.s")
    words[words.index("--genco"):words.index("--genco") + 1] = ["--cuda-device-only", "-S"]
    subprocess.run(words, check=True, capture_output=True, cwd=CSRC)
    want, limit = KERNELS[name]
    got = {}
    for m in re.finditer(r"\.amdhsa_kernel (\S+)\n(.*?)\.end_amdhsa_kernel", (tmp_path / "a.s").read_text(), re.S):
        got[m.group(1)] = [int(re.search(rf"\.amdhsa_{k} (\d+)", m.group(2)).group(1))
                           for k in ("next_free_vgpr", "private_segment_fixed_size", "group_segment_fixed_size")]
    assert sorted(got) == sorted(want)
    for kernel, (vgpr, spilled, lds) in got.items():
        assert spilled == 0 and vgpr <= limit and lds <= 160 * 1024, (kernel, vgpr, spilled, lds)
