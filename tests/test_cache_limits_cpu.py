"""The sequence-cache operators at their limits, without a GPU: that no address
leaves its array whatever device memory holds."""
import itertools
import os
import subprocess

import pytest

import kernelh as kh
from test_cache_cpu import attention, cache, evict, refused, rope, table, weights

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_addresses_stay_inside(tmp_path):
    exe = tmp_path / "paged_bounds_check"
    r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined",
                        "-fno-sanitize-recover=all", "-I", os.path.join(REPO, "kernel.h_amd", "csrc", "kernels"),
                        os.path.join(REPO, "tests", "cpp", "paged_bounds_check.cpp"), "-o", str(exe)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("paged_bounds_check ok"), r.stdout


@pytest.mark.parametrize("dtype", [kh.F32, kh.BF16])
@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (16, 16, 64), (8, 1, 256), (7, 1, 80)])
def test_a_workspace_suffices_for_every_smaller_step(dtype, hq, hk, d):
    """What the largest step reports, no smaller one asks more than: of fewer
    tokens, fewer sequences, shorter ones, under a window."""
    st = dict(k_page_stride=16 * hk * d, k_slot_stride=hk * d, k_head_stride=d, v_page_stride=16 * hk * d, v_slot_stride=hk * d,
              v_head_stride=d)
    tokens, seqs, lens, windows = (1, 4, 33, 127, 512, 2048, 8192), (1, 4, 64), (300, 1024, 8192, 131072), (0, 4096, 100)

    def size(t, s, n, w):
        return kh.paged_attention_workspace(attention(
            cache=cache(kv_heads=hk, head_dim=d, dtype=dtype, **st), table=table(seqs=s, width=8192, row_stride=8192, max_len=n),
            q_heads=hq, q_stride=hq * d, out_stride=hq * d, tokens=t, window=w))

    all_of = {x: size(*x) for x in itertools.product(tokens, seqs, lens, windows)}
    for t, s, n, w in all_of:
        for x, need in all_of.items():
            if x[0] <= t and x[1] <= s and x[2] <= n and (w == 0 or 0 < x[3] <= w):
                assert need <= all_of[t, s, n, w], (x, (t, s, n, w))
    # A single token of a long sequence is split, whatever else the step may have had.
    assert all_of[1, 1, 131072, 0] >= 100 * (d + 2) * 4
    # Two workgroups to a CU, of two parts of 16 rows or one of 128.
    assert max(all_of.values()) <= 512 * (32 + 128) * (d + 2) * 4


def test_attention_refuses_a_negative_max_new():
    refused(lambda: kh.paged_attention(attention(max_new=-1)), "paged_attention")


# ---------------------------------------------------------------- rows that are written lie apart

def test_rows_of_weights_lie_apart():
    """Three sequences of two heads. The page table and the pointers are not
    touched: what is accepted here would go on to the device."""
    for kw in (dict(seq_stride=48, head_stride=48), dict(seq_stride=60, head_stride=40), dict(seq_stride=100, head_stride=200),
               dict(seq_stride=50, head_stride=139)):
        refused(lambda: kh.paged_evict_workspace(evict(**kw)), "paged_evict_workspace")
    for kw in (dict(seq_stride=80, head_stride=40), dict(seq_stride=40, head_stride=120), dict(seq_stride=100, head_stride=50),
               dict(seq_stride=100, head_stride=140), dict(seq_stride=50, head_stride=140)):
        assert kh.paged_evict_workspace(evict(**kw)) > 0, kw
    for kw in (dict(weights_seq_stride=64, weights_head_stride=64), dict(weights_seq_stride=64, weights_head_stride=128)):
        refused(lambda: kh.paged_weights(weights(**kw)), "paged_weights")


def test_rows_of_a_cache_that_is_written_lie_apart():
    """Ten pages of sixteen slots of two heads of 64."""
    page, slot, head = 16 * 2 * 64, 2 * 64, 64
    for x in "kv":
        def strides(p, t, h):
            return cache(**{f"{x}_page_stride": p, f"{x}_slot_stride": t, f"{x}_head_stride": h})

        for bad in ((page, head, head), (page, slot, slot), (page - 64, slot, head), (page, slot - 64, head), (head, slot, head),
                    (page, 64, 15 * 64)):
            refused(lambda: kh.paged_evict_workspace(evict(cache=strides(*bad))), "paged_evict_workspace")
            refused(lambda: kh.qk_norm_rope(rope(cache=strides(*bad))), "qk_norm_rope")
        for good in ((page, slot, head), (page, 64, 16 * 64), (2 * page, 2 * slot, head), (slot, 10 * slot, head), (64, 10 * 64, 160 * 64)):
            assert kh.paged_evict_workspace(evict(cache=strides(*good))) > 0, good
    refused(lambda: kh.qk_norm_rope(rope(cache=cache(v=1 << 20))), "qk_norm_rope")
    assert kh.paged_evict_workspace(evict(cache=cache(v=1 << 20))) > 0  # one row that is both: copied twice, the same
