"""The sequence-cache operators on the GPU at the ends of their ranges:
sequences without new tokens, long caches, scores of any size, rows that add
nothing."""
import math

import numpy as np
import pytest

import kernelh as kh
from cachetest import DTYPES, Step, ints_on_gpu, same_bits, values_from_gpu, values_on_gpu
from khtest import say
from test_gpu_cache import check_attention, check_weights, close

pytestmark = pytest.mark.gpu


def run_weights_without(s, lse, cap):
    """paged_weights with no weights_in; rows behind the sequences' lengths hold a pattern."""
    cache, keep1 = s.cache_on_gpu()
    table, keep2 = s.table_on_gpu()
    q, starts, dlse = values_on_gpu(s.q, s.dtype), ints_on_gpu(s.starts), values_on_gpu(lse, "f32")
    shape = (len(s.lens), s.hk, cap)
    out = values_on_gpu(np.full(shape, 7.0), "f32")
    kh.paged_weights(kh.PagedWeights(
        cache=cache, table=table, q=q.ptr, lse=dlse.ptr, q_starts=starts.ptr, q_stride=s.q_pitch, weights_in=None,
        weights=out.ptr, weights_seq_stride=s.hk * cap, weights_head_stride=cap, tokens=s.tokens, q_heads=s.hq,
        window=s.window, scale=s.scale))
    got = values_from_gpu(out, shape, "f32")
    del keep1, keep2
    return got


# ---------------------------------------------------------------- sequences without new tokens

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("page_size", [16, 24])
@pytest.mark.parametrize("in_place", [False, True])
def test_weights_of_idle_sequences_behind_the_last_token(dev, dtype, page_size, in_place):
    """The last sequences have entries and no new tokens, and start where the
    tokens end: their weights are what they were."""
    for q_lens in ([1, 0, 0], [40, 1, 0], [3, 0, 2, 0, 0]):
        lens = [300, 77, 130, 16, 513][:len(q_lens)]
        s = Step(dtype, q_lens, lens, 4, 2, 64, page_size=page_size, seed=page_size)
        got = check_weights(s, in_place)
        idle = len(q_lens) - 1
        y = np.zeros((s.tokens, s.hq), np.float32)
        without = run_weights_without(s, y, got.shape[2])
        assert (without[idle, :, :lens[idle]] == 0).all() and (without[idle, :, lens[idle]:] == 7.0).all()


@pytest.mark.parametrize("page_size", [16, 24])
def test_weights_where_starts_lie_past_the_tokens(dev, page_size):
    s = Step("bf16", [2, 0, 0], [300, 77, 130], 4, 2, 64, page_size=page_size, seed=3)
    lse = s.attention()[2].astype(np.float32)
    before = s.g.random((3, 2, 305), np.float32)
    want = s.run_weights(lse, before)
    s.starts = [0, 2, 1 << 30, (1 << 31) - 1]
    got = s.run_weights(lse, before)
    assert same_bits(got, want)
    assert same_bits(got[1, :, :77], before[1, :, :77]) and same_bits(got[2, :, :130], before[2, :, :130])


# ---------------------------------------------------------------- long caches

def test_weights_of_a_sequence_past_2_30_entries(dev):
    """A table that repeats one page of 2^20 entries (heads of 8, 16 MB): what
    entries had received before stays, at both ends, where a row of weights
    passes 4 GB."""
    ps, d = 1 << 20, 8
    n = (1 << 30) + 100
    g = np.random.default_rng(0)
    k = values_on_gpu(np.zeros((ps, d)), "bf16")
    table, lens = ints_on_gpu(np.zeros(1025)), ints_on_gpu([n])
    cache = kh.PagedCache(k=k.ptr, v=k.ptr, k_page_stride=ps * d, k_slot_stride=d, k_head_stride=d, v_page_stride=ps * d,
                          v_slot_stride=d, v_head_stride=d, pages=1, page_size=ps, kv_heads=1, head_dim=d, dtype=kh.BF16)
    # Keys of zeros: every entry receives exp(0 - lse), a power of two as a float.
    q, starts = values_on_gpu(g.standard_normal((1, d)), "bf16"), ints_on_gpu([0, 1])
    lse = values_on_gpu([math.log(4.0)], "f32")
    w, out = kh.Buffer(n * 4), kh.Buffer(n * 4)
    parts = [(0, 4096), ((1 << 29) - 5, 4096), (n - 4096, 4096)]
    old = [g.random(m, np.float32) for _, m in parts]
    for (at, m), x in zip(parts, old):
        kh.check(kh.lib.khrt_memcpy_h2d(w.ptr + at * 4, x.ctypes.data, x.nbytes))
    say("weights of 2^30 + 100 entries")
    kh.paged_weights(kh.PagedWeights(
        cache=cache, table=kh.PageTable(pages=table.ptr, lens=lens.ptr, row_stride=1025, seqs=1, width=1025, max_len=n),
        q=q.ptr, lse=lse.ptr, q_starts=starts.ptr, q_stride=d, weights_in=w.ptr, weights=out.ptr, weights_seq_stride=n,
        weights_head_stride=n, tokens=1, q_heads=1, window=0, scale=1.0))
    kh.synchronize()
    for (at, m), x in zip(parts, old):
        got = np.empty(m, np.float32)
        kh.check(kh.lib.khrt_memcpy_d2h(got.ctypes.data, out.ptr + at * 4, got.nbytes))
        want = x.astype(np.float64) + 0.25
        if at + m == n:
            want[-1] = 0.25  # the new token's own
        # lse and its exponent round once each, 2^x and the sum once more.
        close(got, want, np.abs(want) * 8 * 2.0 ** -24, f"entries from {at}")
