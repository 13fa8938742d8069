"""The typed cache's and the norm's kernels as the Makefile builds them, from the
device assembly that its own command gives (CPU only): registers, spills, the
arguments that are in registers when a wave starts, and, in every decode kernel,
what the page loop waits for."""
import os
import re
import shlex
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "qwen3.8_27b_in_rust_amd", "csrc")
HIPCC = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "hipcc")
TYPES = ("f16", "bf16", "q8k")
DECODE = [f"q38_attn_decode_{t}{p}" for t in TYPES for p in ("", "_pre", "_one", "_pre_one")]


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    """name of a .hip file -> the assembly of its Makefile command"""
    if not os.path.exists(HIPCC) or shutil.which("make") is None:
        pytest.skip("needs hipcc and make")
    plan = subprocess.run(["make", "-n", "-B", "-C", CSRC], check=True, capture_output=True, text=True).stdout
    out, done = tmp_path_factory.mktemp("asm"), {}

    def get(name):
        if name not in done:
            line = next(ln for ln in plan.splitlines() if f"{name}.hsaco" in ln and "--genco" in ln)
            words = shlex.split(line)
            at = words.index("-o")
            words[at + 1] = str(out / (name + ".s"))
            words[words.index("--genco"):words.index("--genco") + 1] = ["--cuda-device-only", "-S"]
            subprocess.run(words, check=True, capture_output=True, cwd=CSRC)
            done[name] = (out / (name + ".s")).read_text()
        return done[name]

    return get


def _kernels(text):
    """kernel -> (registers, spilled bytes, argument words in registers)"""
    res = {}
    for m in re.finditer(r"\.amdhsa_kernel (\S+)\n(.*?)\.end_amdhsa_kernel", text, re.S):
        word = lambda key: int(re.search(rf"\.amdhsa_{key} (\d+)", m.group(2)).group(1))  # noqa: B023, E731
        res[m.group(1)] = (word("next_free_vgpr"), word("private_segment_fixed_size"), word("user_sgpr_kernarg_preload_length"))
    return res


def test_decode(built):
    """Eight waves launch at 256 registers or fewer."""
    got = _kernels(built("attn_decode_typed"))
    assert sorted(got) == sorted(DECODE)
    for name, (vgpr, spilled, words) in got.items():
        assert spilled == 0 and vgpr <= 256, (name, vgpr, spilled)
        assert (words > 0) == name.endswith("_one"), (name, words)


def test_rows(built):
    """Four workgroups of eight waves a CU: 64 registers."""
    got = _kernels(built("kv_rows"))
    names = [f"q38_kv_{c}_{t}" for c in ("append", "gather") for t in ("f32",) + TYPES] + ["q38_kv_gather_16"]
    assert sorted(got) == sorted(n + s for n in names for s in ("", "_few"))
    for name, (vgpr, spilled, words) in got.items():
        assert spilled == 0 and vgpr <= 64, (name, vgpr, spilled)
        assert (words > 0) == ("gather" in name and name.endswith("_few")), (name, words)


def test_norm_and_merge(built):
    for name, (vgpr, spilled, words) in _kernels(built("norm")).items():
        small = "_1024_" in name or name.endswith(("_1", "_2", "_3"))
        assert spilled == 0 and vgpr <= (64 if small else 84) and words > 0, (name, vgpr, spilled, words)
    assert _kernels(built("attn_decode"))["q38_attn_decode_merge_one"][2] > 0


@pytest.mark.parametrize("name", DECODE)
def test_a_page_is_waited_for_alone(built, name):
    """Loads come back in order.  Before a page's first score eight younger loads (a
    16-bit page's values) or ten (8-bit rows: the wave's other page) are still on their way; in the loop
    over 8-bit pages no wait leaves fewer than ten."""
    body = re.search(rf"^{name}:(.*?)s_endpgm", built("attn_decode_typed"), re.S | re.M).group(1)
    lines = body.split("\n")
    products = [i for i, ln in enumerate(lines) if "v_mfma" in ln]
    waits = lambda part: [int(n) for ln in part for n in re.findall(r"s_waitcnt.*vmcnt\((\d+)\)", ln)]  # noqa: E731
    least = 10 if "q8k" in name else 8
    assert waits(lines[:products[0]])[-1] >= least
    if "q8k" in name:
        labels = {ln.split(":")[0]: i for i, ln in enumerate(lines) if re.match(r"\.LBB\w+:", ln)}
        jumps = [(labels[m.group(1)], i) for i, ln in enumerate(lines)
                 for m in [re.search(r"s_c?branch\w*\s+(\.LBB\w+)", ln)] if m and labels.get(m.group(1), i) < i]
        # the loop over pages: it holds every product of both pages in flight
        loops = [lines[a:b] for a, b in jumps if sum("v_mfma" in ln for ln in lines[a:b]) == len(products)]
        assert loops
        for loop in loops:
            assert waits(loop) and min(waits(loop)) >= 10
