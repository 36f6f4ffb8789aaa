"""Attention over a cache in 8 bits where its launch is shaped by what the caller
expects and the lengths turn out otherwise, and in steps large enough that shared
entries are worked on apart (tests/test_cache8_plans_cpu.py checks that they are)."""
import numpy as np
import pytest

import kernelh as kh
from cache8test import Step8, codes_of, held
from cachetest import DTYPES, ints_on_gpu, rounded, values_on_gpu
from khtest import say
from test_gpu_cache import check_attention, close
from test_gpu_cache_steps import Graph

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("page_size,window", [(16, 0), (24, 0), (16, 1200)])
def test_shared_entries_past_the_expected_length(dev, dtype, page_size, window):
    """As captured calls whose sequences have grown: the expected length ends inside the
    shared entries, and so do some sequences; a chunk among the single tokens."""
    lens = [1620] + [1501 + 7 * i for i in range(60)] + [1100, 640, 500, 1900]
    s = Step8(dtype, [1] * 64 + [130], lens, 4, 4, 128, seed=page_size, page_size=page_size, shared=1500, window=window)
    for max_len in (600, 1499, 1):
        check_attention(s, max_len=max_len, max_new=130)
    s = Step8(dtype, [1] * 64, lens[:64], 4, 4, 128, seed=page_size + 1, page_size=page_size, shared=1500, window=window)
    for max_len in (600, 1101):
        check_attention(s, max_len=max_len, max_new=1)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_more_sequences_than_lanes_behind_shared_entries(dev, dtype):
    """A hundred and fifty sequences: single tokens, drafts, chunks, some without new tokens."""
    g = np.random.default_rng(5)
    q_lens = [int(x) for x in g.choice([0, 1, 1, 1, 2, 40], 150, p=[0.1, 0.3, 0.2, 0.2, 0.18, 0.02])]
    lens = [int(x) for x in g.integers(700, 1100, 150)]
    check_attention(Step8(dtype, q_lens, lens, 8, 4, 64, seed=6, shared=688, before=1, after=2))


@pytest.mark.parametrize("starts", ["claimed twice", "descending", "past the last token"])
def test_starts_that_do_not_ascend_behind_shared_entries(dev, starts):
    """Whatever the sequences get, the call ends, and tokens of none are left alone."""
    s = Step8("bf16", [1] * 64, [1501 + 7 * i for i in range(64)], 4, 4, 128, seed=3, before=1, after=2, shared=1500)
    say(f"starts {starts}")
    s.starts = {"claimed twice": [1, 60] * 32 + [1], "descending": [60 - i for i in range(65)],
                "past the last token": [1] * 60 + [65, 1 << 30, 70, 1 << 30, 65]}[starts]
    for workspace in (None, 0):
        out, lse = s.run_attention(max_new=1, workspace=workspace)
        none = {"claimed twice": [0, 60, 65, 66], "descending": list(range(67)), "past the last token": [0]}[starts]
        assert (out[none] == 7.0).all() and (lse[none] == 7.0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page_size,scales_far", [(16, True), (16, False), (24, True)])
def test_shared_entries_past_4_gb(dev, dtype, page_size, scales_far):
    """Pages 128 MB apart, their scales behind the rows or elsewhere."""
    far, pages, hq, hk, d = 1 << 27, 36, 4, 2, 128
    say(f"far pages of {page_size}, scales far: {scales_far}")
    g = np.random.default_rng(page_size)
    bufs = [kh.Buffer(pages * far) for _ in "kv"]
    near = [kh.Buffer.from_array(np.zeros((pages, hk, page_size), np.uint8)) for _ in "kv"]
    at = page_size * hk * d
    cache = kh.PagedCache8(k=bufs[0].ptr, v=bufs[1].ptr, k_scale=bufs[0].ptr + at if scales_far else near[0].ptr,
                           v_scale=bufs[1].ptr + at if scales_far else near[1].ptr, k_page_stride=far, k_slot_stride=hk * d,
                           k_head_stride=d, v_page_stride=far, v_slot_stride=hk * d, v_head_stride=d,
                           scale_page_stride=far if scales_far else hk * page_size, scale_head_stride=page_size, pages=pages,
                           page_size=page_size, kv_heads=hk, head_dim=d)
    order, n = g.permutation(pages).astype(np.int32), pages * page_size
    slots = order[np.arange(n) // page_size].astype(np.int64) * page_size + np.arange(n) % page_size
    q, k, v = (rounded(g.standard_normal((n, h, d), np.float32), "bf16") for h in (1, hk, hk))
    dq, dk, dv, dslots = (*(values_on_gpu(x, "bf16") for x in (q, k, v)), ints_on_gpu(slots, np.int64))
    dqo = values_on_gpu(np.zeros((n, 1, d)), "bf16")
    kh.synchronize()
    kh.qk_norm_rope8(kh.QkNormRope8(q=dq.ptr, k=dk.ptr, v=dv.ptr, q_out=dqo.ptr, slots=dslots.ptr, q_stride=d, k_stride=hk * d,
                                    v_stride=hk * d, q_out_stride=d, cache=cache, tokens=n, q_heads=1, dtype=kh.BF16, eps=0.0))
    kh.synchronize()
    lens = [n - i % 60 for i in range(120)]
    for q_lens in ([1] * 120, [1] * 119 + [40]):
        s = Step8(dtype, q_lens, [1] * 120, hq, hk, d, page_size=page_size, seed=len(q_lens), shared=0)
        s.pages, s.table, s.lens, s.shared = pages, np.repeat(order[None], 120, 0), lens, 500
        for name, x in (("k", k), ("v", v)):
            codes, scales = np.zeros((n, hk, d), np.uint8), np.zeros((n, hk), np.uint8)
            codes[slots], scales[slots] = held(x)
            s.put(name, codes.reshape(pages, page_size, hk, d), scales.reshape(pages, page_size, hk))
        s.cache8_on_gpu = lambda: (cache, None)
        check_attention(s, max_new=max(q_lens))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("cap,scale", [(3e38, 0.125), (2.4e38, 30.0), (3e37, 0.125), (1e37, 1e-3), (1e30, 1e-30)])
def test_caps_past_every_score(dev, dtype, cap, scale):
    s = Step8(dtype, [1, 3, 40], [70, 300, 90], 4, 2, 64, seed=9, cap=cap)
    s.scale = scale
    check_attention(s)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("cap", [20.0, 200.0])
@pytest.mark.parametrize("beside,max_len", [(2000, 0), (2000, 40), (600, 600)])
def test_small_scores_under_a_cap_beside_long_sequences(dev, dtype, cap, beside, max_len):
    """A chunk's first row, which sees one entry, has its score for lse, as exact as where
    the step holds nothing longer: exact before the cap (small whole numbers), and off by
    some 8 roundings of the series behind it, or where the other form takes over, at a
    quarter of the cap, by 2^-23 of the cap: 2^-20 of it."""
    s = Step8(dtype, [40] * 31, [40] * 30 + [beside], 4, 2, 64, cap=cap, seed=beside)
    whole = s.g.integers(-2, 3, s.k_codes.shape).astype(float)
    s.put("k", codes_of(whole), np.full(s.k_scales.shape, 127, np.uint8))
    s.q = s.g.integers(-2, 3, s.q.shape).astype(np.float32)
    s.scale = 0.125
    _, lse = s.run_attention(max_len=max_len)
    first = np.arange(30) * 40  # these tokens see one entry
    k = whole[s.table[:30, 0], 0]
    x = s.scale * (s.q.reshape(-1, 4, 64)[first] * np.repeat(k, 2, 1)).sum(-1)
    y = cap * np.tanh(x / cap)
    close(lse[first], y, np.abs(y) * 2.0 ** -20, "lse")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_small_scores_under_a_cap_beside_shared_entries(dev, dtype):
    """A sequence that ends inside the shared entries, its first token after its first entry."""
    cap = 200.0
    s = Step8(dtype, [1] * 40 + [1], [1501 + 7 * i for i in range(40)] + [1], 4, 4, 128, cap=cap, seed=41, shared=1500)
    whole = s.g.integers(-1, 2, s.k_codes.shape).astype(float)
    s.put("k", codes_of(whole), np.full(s.k_scales.shape, 127, np.uint8))
    s.q = s.g.integers(-1, 2, s.q.shape).astype(np.float32)
    s.scale = 0.125
    _, lse = s.run_attention(max_new=1)
    x = s.scale * (s.q[-1].reshape(4, 128) * whole[s.table[-1, 0], 0]).sum(-1)
    y = cap * np.tanh(x / cap)
    close(lse[-1], y, np.abs(y) * 2.0 ** -20, "lse")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_small_scores_under_a_cap_and_a_window_of_one(dev, dtype):
    """Every row sees its own entry alone, far from the first."""
    cap, n = 200.0, 700
    s = Step8(dtype, [n], [n], 4, 2, 64, cap=cap, seed=42, window=1)
    whole = s.g.integers(-2, 3, s.k_codes.shape).astype(float)
    s.put("k", codes_of(whole), np.full(s.k_scales.shape, 127, np.uint8))
    s.q = s.g.integers(-2, 3, s.q.shape).astype(np.float32)
    s.scale = 0.125
    _, lse = s.run_attention()
    j = np.arange(n)
    x = s.scale * (s.q.reshape(n, 4, 64) * np.repeat(whole[s.table[0][j // 16], j % 16], 2, 1)).sum(-1)
    y = cap * np.tanh(x / cap)
    close(lse, y, np.abs(y) * 2.0 ** -20, "lse")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_captured_call_whose_sequences_grow_past_what_it_expected(dev, dtype):
    """Captured with an expected length inside the shared entries, and replayed as the
    lengths go from below it to past the shared entries and back."""
    full = [1501 + 7 * i for i in range(64)]
    s = Step8(dtype, [1] * 64, full, 4, 4, 128, seed=50, shared=1500)
    a, bufs = s.args8(max_len=600, max_new=1)
    lens = bufs["keep"][1][1]
    size = kh.paged_attention8_workspace(a)
    ws, stream = kh.Buffer(size), kh.Stream()
    kh.synchronize()
    graph = Graph(stream, lambda: kh.paged_attention8(a, ws, size, stream))
    for most in (550, 1400, 2000, 601, 3000, 1):
        s.lens = [min(n, most) for n in full]
        say(f"captured, lengths up to {most}")
        lens.copy_from_host(np.array(s.lens, np.int32))
        for b in (ws, bufs["out"], bufs["lse"]):
            b.fill(7.0, stream)
        stream.synchronize()
        graph.replay()
        stream.synchronize()
        out, lse = s.results(bufs)
        want, bound, y, y_bound = s.attention()
        close(out, want, bound, "out")
        close(lse, y, y_bound, "lse")
    graph.destroy()
    stream.destroy()
