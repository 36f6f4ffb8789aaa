"""How attention over a cache in 8 bits shares a step out, without a GPU: its host
code with launches that only write down what they were given
(tests/cpp/cache8_plan_check.cpp)."""
import itertools
import json
import math
import os
import subprocess

import numpy as np
import pytest

import kernelh as kh
from test_cache8_cpu import attention
from test_cache_cpu import refused

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


def run(cmd, timeout):
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=timeout)
    assert r.returncode == 0, r.stdout[-4000:]
    return r.stdout


@pytest.fixture(scope="module")
def plan_check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plans") / "cache8_plan_check")
    src = os.path.join(REPO, "kernel.h_amd", "csrc")
    run(["g++", "-O1", "-g", "-std=c++20", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-D__HIP_PLATFORM_AMD__",
         "-I", os.path.join(REPO, "include"), "-I", os.path.join(src, "include"), "-I", os.path.join(src, "kernels"),
         "-I", os.path.join(ROCM, "include"), os.path.join(REPO, "tests", "cpp", "cache8_plan_check.cpp"), "-o", exe], 300)
    return exe


@pytest.fixture
def plan(plan_check):
    """What a step's first launch is told."""
    return lambda **kw: json.loads(run([plan_check, *(f"{k}={v}" for k, v in kw.items())], 60))


def test_every_entry_is_somebodys(plan_check):
    """Over a grid of steps: parts of shared entries reach as far as the sequences' own
    begin, and what the kernels write lies in the workspace."""
    assert run([plan_check], 300).strip().endswith("cache8_plan_check ok")


def test_shared_entries_past_the_expected_length(plan):
    """max_len below shared: the entries past it are each sequence's own."""
    p = plan(tokens=64, seqs=64, hq=32, hk=8, d=128, shared=8192, max_len=4096)
    assert p["shared_blocks"] > 0 and p["shared"] <= p["shared_splits"] * p["shared_each"]


def test_the_steps_that_are_run_share_entries(plan):
    """Those of tests/test_gpu_cache8_plans.py."""
    for max_len in (600, 1499):
        assert plan(tokens=194, seqs=65, hq=4, hk=4, d=128, width=200, shared=1500, max_len=max_len, max_new=130)["shared"] == max_len
    for max_len in (600, 1101):
        assert plan(tokens=64, seqs=64, hq=4, hk=4, d=128, width=200, shared=1500, max_len=max_len)["shared"] == max_len
    assert plan(tokens=41, seqs=41, hq=4, hk=4, d=128, width=120, shared=1500, cap=200)["shared"] == 1500
    assert plan(tokens=67, seqs=64, hq=4, hk=4, d=128, width=122, shared=1500)["shared"] == 1500
    assert plan(tokens=285, seqs=150, hq=8, hk=4, d=64, width=69, shared=688, max_new=0)["shared"] == 688
    for page_size, dtype, (tokens, max_new) in itertools.product((16, 24), (0, 2), ((120, 1), (159, 40))):
        assert plan(tokens=tokens, seqs=120, hq=4, hk=2, d=128, width=36, page_size=page_size, dtype=dtype, shared=500,
                    max_new=max_new)["shared"] == 500


def test_a_large_step_asks_no_memory_for_parts_it_does_not_make(plan):
    """Sequences of more than 33 rows a kv head on the whole do not share entries, nor do
    steps of more than 2^22 rows: a step asks for two parts of so many rows at the most, or
    for one and a unit of 128 to a CU, beside what parts of other kinds take."""
    def sizes(**kw):
        p, without = (plan(hq=32, hk=8, d=128, max_new=0, shared=n, **kw) for n in (8192, 0))
        return p["shared"] > 0, p["bytes"] - without["bytes"]

    row = (128 + 2) * 4
    for tokens in (64, 512, 528, 1000, 8192, 200000, 1 << 20):
        shares, more = sizes(tokens=tokens, seqs=64)
        assert shares == (tokens * 4 // 33 < 62) and more <= (64 * 33 * 8 + max(64 * 33 * 8, 256 * 128)) * row
    for tokens in (1 << 17, (1 << 17) + 1, 1 << 20):
        shares, more = sizes(tokens=tokens, seqs=1 << 17)
        assert shares == (tokens == 1 << 17) and more <= 2 * (1 << 22) * row


@pytest.mark.parametrize("scale", [0.125, 1.0, -3e-20, 1e-30, 100.0, 1e25])
@pytest.mark.parametrize("cap", [1e-40, 1e-3, 30.0, 1e30, 1e37, 3e37, 2.3e38, 2.4e38, 3e38, 3.4028e38])
def test_factors_of_caps_hold_their_bits(plan, scale, cap):
    """cap tanh(x / cap) as two factors in 32 bits, each the formula's but for a few
    roundings; or no cap, where one of them is not a normal number: then no q . k and no
    score below 2^114 is off by more than half a step for it. Small caps have their first factor cut to
    the largest number, where all but a score of 0 is the cap itself."""
    p = plan(tokens=2, seqs=2, hq=4, hk=2, d=64, scale=scale, cap=cap)
    scale, cap = float(np.float32(scale)), float(np.float32(cap))
    top = float(np.finfo(np.float32).max)
    want_in, want_out = 2 * abs(scale) / math.log(2) / cap, cap / math.log(2)
    if p["cap_in"] == 0:
        assert want_in < 2.0 ** -125 or want_out > top * (1 - 2.0 ** -22)
        # tanh(y) = y - y^3 / 3 + ..
        assert want_in * 2.0 ** 114 / 2 < 2.0 ** -11 or want_out > top * (1 - 2.0 ** -22)
        return
    assert abs(p["cap_in"] / min(want_in, top) - 1) < 2.0 ** -21
    assert 2.0 ** -126 <= p["cap_in"] and want_out < top * (1 + 2.0 ** -22)
    assert abs(p["cap_out"] - want_out) <= 2.0 ** -22 * want_out + 2.0 ** -149


@pytest.mark.parametrize("written", ["out", "lse", "workspace"])
def test_attention_does_not_write_what_it_reads(written):
    """Equal pointers show that it would."""
    read = dict(q=16, k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, pages=1 << 12, lens=2 << 12, q_starts=1 << 14)
    others = {"out": dict(lse=64), "lse": dict(out=64), "workspace": dict(out=64, lse=128)}[written]
    for at in [*read.values(), *others.values()]:
        kw = dict(q_starts=1 << 14, out=32, lse=48) | others
        workspace = 1 << 15
        if written == "workspace":
            workspace = at
        else:
            kw[written] = at
        refused(lambda: kh.paged_attention8(attention(**kw), workspace, 1 << 20), "paged_attention8")
