"""Register budgets of the typed cache's and the norm's kernels, from their
device assembly (CPU only: hipcc compiles for gfx950 without a GPU).  None
spills; the decode workgroups of 8 waves launch only at 256 registers or fewer,
two row workgroups of 16 waves share a CU at 64, and a decode wave waits for
one page's loads at a time (its page loop holds no wait for all of them)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "qwen3.8_27b_in_rust_amd", "csrc")
HIPCC = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "hipcc")
TYPES = ("f16", "bf16", "q8k")


def _assembly(tmp_path_factory, name):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm") / (name + ".s")
    flags = ["--offload-arch=gfx950", "--cuda-device-only", "-S", "-O3", "-std=c++17", "-ffp-contract=off",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-I" + os.path.join(CSRC, "kernels"), "-I" + CSRC]
    subprocess.run([HIPCC, *flags, "-o", str(out), os.path.join(CSRC, "kernels", name + ".hip")], check=True, capture_output=True)
    return out.read_text()


def _budgets(text):
    res = {}
    for m in re.finditer(r"\.amdhsa_kernel (\S+)\n(.*?)\.end_amdhsa_kernel", text, re.S):
        body = m.group(2)
        res[m.group(1)] = (int(re.search(r"\.amdhsa_next_free_vgpr (\d+)", body).group(1)),
                           int(re.search(r"\.amdhsa_private_segment_fixed_size (\d+)", body).group(1)))
    return res


@pytest.fixture(scope="module")
def decode(tmp_path_factory):
    return _assembly(tmp_path_factory, "attn_decode_typed")


def test_decode(decode):
    got = _budgets(decode)
    assert sorted(got) == sorted(f"q38_attn_decode_{t}{p}" for t in TYPES for p in ("", "_pre", "_one", "_pre_one"))
    for name, (vgpr, scratch) in got.items():
        assert scratch == 0 and vgpr <= 256, (name, vgpr, scratch)


def test_decode_waits_for_a_page_at_a_time(decode):
    """8-bit rows, two pages a wave: the first score of a page waits with the
    other page's ten loads, and this page's later ones, still in flight."""
    body = re.search(r"^q38_attn_decode_q8k:(.*?)s_endpgm", decode, re.S | re.M).group(1)
    first = body[:body.index("v_mfma_f32_16x16x32_f16")]
    waits = [int(n) for n in re.findall(r"s_waitcnt vmcnt\((\d+)\)", first)]
    assert waits and waits[-1] >= 10


def test_rows(tmp_path_factory):
    got = _budgets(_assembly(tmp_path_factory, "kv_rows"))
    names = [f"q38_kv_{c}_{t}" for c in ("append", "gather") for t in ("f32",) + TYPES] + ["q38_kv_gather_16"]
    assert sorted(got) == sorted(n + s for n in names for s in ("", "_few"))
    for name, (vgpr, scratch) in got.items():
        assert scratch == 0 and vgpr <= 64, (name, vgpr, scratch)


def test_norm(tmp_path_factory):
    got = _budgets(_assembly(tmp_path_factory, "norm"))
    assert len(got) == 12
    for name, (vgpr, scratch) in got.items():
        assert scratch == 0 and vgpr <= (64 if "_1024_" in name or name.endswith(("_1", "_2", "_3")) else 84), (name, vgpr, scratch)
