"""The operators over a cache in 8 bits on the GPU against their definitions in
64 bits (tests/cache8test.py, tests/cachetest.py): the write, the reading back,
attention. What the cache holds is compared bit for bit, but where 32 bits may
round across a border."""
import math

import numpy as np
import pytest

import kernelh as kh
from cachetest import DTYPES, ints_on_gpu, rope_reference, rounded, same_bits, values_from_gpu, values_on_gpu
from cache8test import Step8, codes_of, held, numbers, stand_for
from khtest import say
from test_gpu_cache import check_attention, close

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d", [(1, 1, 64), (4, 4, 64), (8, 2, 128), (32, 8, 128), (7, 1, 80), (6, 2, 16), (5, 5, 256),
                                     (24, 1, 96), (4, 2, 144), (3, 1, 208)])
def test_single_tokens(dev, dtype, hq, hk, d):
    check_attention(Step8(dtype, [1, 1, 1, 1, 1], [1, 2, 33, 500, 129], hq, hk, d, seed=d + hq))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("page_size,scale_pad", [(1, 0), (3, 0), (16, 0), (16, 3), (24, 0), (64, 4), (1000, 1)])
def test_pages_that_end_inside_a_tile(dev, dtype, page_size, scale_pad):
    check_attention(Step8(dtype, [1, 2, 1], [1, 257, 700], 4, 2, 64, page_size=page_size, scale_pad=scale_pad, seed=page_size))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d", [(4, 4, 64), (8, 2, 128), (3, 1, 80), (2, 2, 256), (6, 2, 48)])
@pytest.mark.parametrize("window,cap", [(0, 0.0), (1, 0.0), (50, 3.0)])
def test_chunks(dev, dtype, hq, hk, d, window, cap):
    check_attention(Step8(dtype, [17, 1, 64, 5, 130], [17, 40, 200, 5, 333], hq, hk, d, page_size=24, window=window,
                          cap=cap, seed=d + window))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q_lens,lens,hq,hk,d", [([50], [4000], 4, 2, 64), ([70], [2100], 2, 1, 128), ([20], [1500], 4, 1, 256),
                                                 ([40, 1, 0, 130, 9], [3000, 2000, 50, 700, 1300], 8, 2, 128),
                                                 ([33, 32, 8], [900, 901, 902], 1, 1, 80)])
@pytest.mark.parametrize("window", [0, 700])
def test_chunks_over_long_caches(dev, dtype, q_lens, lens, hq, hk, d, window):
    """Sequences of many rows whose entries are split over workgroups, alone
    and beside sequences of few rows; with and without a workspace."""
    s = Step8(dtype, q_lens, lens, hq, hk, d, seed=d, window=window, page_size=24, before=1, after=2)
    for workspace in (None, 0, 300000):
        check_attention(s, workspace=workspace)


def test_more_sequences_than_lanes(dev):
    """A hundred and fifty sequences of all kinds."""
    g = np.random.default_rng(0)
    q_lens = [int(x) for x in g.choice([0, 1, 1, 1, 2, 30], 150)]
    lens = [int(x) for x in g.integers(0, 300, 150)]
    check_attention(Step8("bf16", q_lens, lens, 4, 2, 64, seed=1))
    check_attention(Step8("f16", [1] * 150, lens, 4, 2, 64, seed=2, shared=64))


@pytest.mark.parametrize("shared", [0, 60])
def test_starts_that_do_not_ascend(dev, shared):
    """Sequences that claim the same tokens: whatever they get, the call ends,
    and tokens of no sequence are left alone."""
    s = Step8("bf16", [40] * 6, [100] * 6, 4, 2, 64, seed=3, before=1, after=2, shared=shared)
    s.starts = [1, 200, 1, 200, 1, 200, 150]
    out, lse = s.run_attention()
    assert (out[[0, -1, -2]] == 7.0).all() and (lse[[0, -1, -2]] == 7.0).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("workspace", [0, None, 20000])
@pytest.mark.parametrize("q", [1, 5])
def test_long_sequences_split_and_not(dev, dtype, workspace, q):
    """One long sequence and short ones, with all splits, few and none; the
    expected length said, not said, and said too short."""
    s = Step8(dtype, [q, q, q], [5000, 7, 130], 4, 1, 64, seed=11, page_size=16)
    for max_len in (0, 5000, 300):
        check_attention(s, workspace=workspace, max_len=max_len)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("window", [0, 3])
def test_rows_that_see_nothing(dev, dtype, window):
    """No entries, fewer entries than new tokens, a sequence without new
    tokens, and a length below zero."""
    s = Step8(dtype, [2, 9, 0, 3, 1], [0, 4, 50, 3, -5], 4, 2, 64, seed=5, window=window, before=2, after=3, cap=2.0)
    out, lse = check_attention(s)
    assert (out[2:4] == 0).all() and (lse[2:4] == -math.inf).all()
    assert (out[4:9] == 0).all() and (lse[4:9] == -math.inf).all()
    assert (out[-4] == 0).all() and (lse[-4] == -math.inf).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [-1, 1 << 30, "pages"])
def test_pages_that_do_not_exist(dev, dtype, bad):
    s = Step8(dtype, [1, 40, 1], [100, 90, 64], 4, 2, 64, seed=6)
    s.table[0, 2] = s.table[1, 0] = s.pages if bad == "pages" else bad
    s.table[2, :] = s.pages if bad == "pages" else bad
    out, lse = check_attention(s)
    assert (out[-1] == 0).all() and (lse[-1] == -math.inf).all()


@pytest.mark.parametrize("heads_first", [False, True])
def test_other_layouts_and_strides(dev, heads_first):
    check_attention(Step8("bf16", [3, 1, 50], [90, 40, 200], 6, 2, 96, seed=8, heads_first=heads_first, pad=64, scale_pad=16))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("scale", [0.0, -0.2, 40.0, 1e4])
@pytest.mark.parametrize("cap", [0.0, 1.5, 30.0])
def test_scales_and_caps(dev, dtype, scale, cap):
    """A scale of 0 and below, scores far past the cap, weights of one entry."""
    s = Step8(dtype, [1, 3, 40], [70, 300, 90], 4, 2, 64, seed=9, cap=cap)
    s.scale = scale
    check_attention(s)


@pytest.mark.parametrize("cap", [1e-3, 1e5, 1e30])
def test_caps_that_scores_are_far_from(dev, cap):
    check_attention(Step8("f32", [1, 40], [300, 90], 4, 2, 64, seed=10, cap=cap))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q", [1, 40])
def test_nan_that_a_token_does_not_see(dev, dtype, q):
    """NaN in v, and in k, of entries that later tokens of the sequence see."""
    s = Step8(dtype, [q, q], [100, 64 + q], 4, 2, 128, seed=12, window=40 if q > 1 else 0)
    for at, where in ((s.v_codes, 100 - q + 3), (s.v_codes, 70), (s.k_codes, 95)):
        page, slot = s.table[0, where // 16], where % 16
        at[page, slot, 0, 17] = 0x7F
        at[page, slot, 1, 5] = 0xFF
    s.put("k", s.k_codes, s.k_scales)
    s.put("v", s.v_codes, s.v_scales)
    s2 = s
    out, lse = s.run_attention()
    want, bound, y, y_bound = s2.attention()
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(out), ~fine)
    close(np.where(fine, out, 0), np.where(fine, want, 0), bound, "out")


def test_scales_out_of_range_count_as_the_nearest(dev):
    s = Step8("f32", [1, 2], [40, 50], 2, 1, 64, seed=13)
    for x in (s.k_scales, s.v_scales):
        x[s.table[0, 0], 3:5, 0] = 0, 9
    s.v_scales[s.table[1, 0], 7:9, 0] = 247, 255
    s.put("k", s.k_codes, s.k_scales)
    s.put("v", s.v_codes, s.v_scales)
    check_attention(s)


# ---------------------------------------------------------------- entries that sequences share

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d,page_size", [(4, 4, 128, 16), (16, 4, 64, 7), (2, 2, 256, 24)])
@pytest.mark.parametrize("window,cap", [(0, 0.0), (0, 20.0), (900, 0.0)])
def test_shared_entries(dev, dtype, hq, hk, d, page_size, window, cap):
    """Many single tokens and short drafts behind a long shared beginning, which
    ends inside a page; sequences that end inside it, one without new tokens, tokens
    of no sequence, and with no workspace."""
    q_lens = [1, 2, 0, 1, 5, 1] + [1] * 44
    lens = [2500, 1904, 1950, 1000, 1903, 0] + [1901 + 3 * i for i in range(44)]
    s = Step8(dtype, q_lens, lens, hq, hk, d, seed=d, page_size=page_size, shared=1900, window=window, cap=cap, before=1, after=2)
    check_attention(s)
    check_attention(s, max_len=2500, max_new=5)
    check_attention(s, workspace=0)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_shared_entries_that_sequence_0_ends_inside(dev, dtype):
    for first in (0, 7, 1000):
        check_attention(Step8(dtype, [1] * 50, [first] + [1600 + i for i in range(49)], 4, 4, 64, seed=first, shared=1590))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_shared_entries_before_long_ones(dev, dtype):
    """The sequences' own entries in parts, and a chunk among them."""
    s = Step8(dtype, [1] * 30 + [70], [2500 + 61 * i for i in range(30)] + [2400], 4, 2, 128, seed=14, shared=2300)
    check_attention(s)
    check_attention(s, max_len=300)
    check_attention(Step8(dtype, [1] * 60 + [300, 2], [1700 + 5 * i for i in range(60)] + [2100, 1999], 4, 2, 128, seed=15, shared=1650))


# ---------------------------------------------------------------- the write

def positions_of(axes, tokens, g, far):
    return g.integers(0, far, (axes, tokens))


def run_write(dtype, q, k, v, gammas, freq, pos, pair_axis, slots, pages, page_size, rotary, interleaved=False, norm=True, eps=1e-6,
              k_out=False, in_place=False, axis_stride=None, stream=None):
    """q_out, k_out, and the cache's codes and scales, pattern 0x55 where not written."""
    t, hq, d = q.shape
    hk = k.shape[1]
    dq, dk, dv = (values_on_gpu(x, dtype) for x in (q, k, v))
    dqo = dq if in_place else values_on_gpu(np.full(q.shape, 7.0), dtype)
    dko = values_on_gpu(np.full(k.shape, 7.0), dtype) if k_out else None
    codes = [kh.Buffer.from_array(np.full((pages, page_size, hk, d), 0x55, np.uint8)) for _ in "kv"]
    scales = [kh.Buffer.from_array(np.full((pages, hk, page_size), 0x55, np.uint8)) for _ in "kv"]
    gq, gk = (values_on_gpu(x, dtype) if x is not None else None for x in gammas)
    df, dp = values_on_gpu(freq, "f32"), ints_on_gpu(pos, np.int64)
    da = ints_on_gpu(pair_axis) if pair_axis is not None else None
    ds = ints_on_gpu(slots, np.int64)
    cache = kh.PagedCache8(k=codes[0].ptr, v=codes[1].ptr, k_scale=scales[0].ptr, v_scale=scales[1].ptr,
                           k_page_stride=page_size * hk * d, k_slot_stride=hk * d, k_head_stride=d,
                           v_page_stride=page_size * hk * d, v_slot_stride=hk * d, v_head_stride=d,
                           scale_page_stride=hk * page_size, scale_head_stride=page_size, pages=pages, page_size=page_size,
                           kv_heads=hk, head_dim=d)
    kh.synchronize()
    kh.qk_norm_rope8(kh.QkNormRope8(
        q=dq.ptr, k=dk.ptr, v=dv.ptr, q_out=dqo.ptr, k_out=dko.ptr if dko else None, q_gamma=gq.ptr if gq else None,
        k_gamma=gk.ptr if gk else None, inv_freq=df.ptr, positions=dp.ptr, pair_axis=da.ptr if da else None, slots=ds.ptr,
        q_stride=hq * d, k_stride=hk * d, v_stride=hk * d, q_out_stride=hq * d, k_out_stride=hk * d,
        axis_stride=pos.shape[1] if axis_stride is None else axis_stride, cache=cache, tokens=t, q_heads=hq, rotary_dim=rotary,
        axes=pos.shape[0], interleaved=interleaved, norm=norm, dtype=DTYPES[dtype], eps=eps), stream)
    if stream is not None:
        stream.synchronize()
    kh.synchronize()
    got = [b.to_host(np.uint8, pages * page_size * hk * d).reshape(pages, page_size, hk, d) for b in codes]
    got += [b.to_host(np.uint8, pages * page_size * hk).reshape(pages, hk, page_size) for b in scales]
    return (values_from_gpu(dqo, q.shape, dtype), values_from_gpu(dko, k.shape, dtype) if k_out else None, *got)


def rotated(x, gamma, pos, freq, pair_axis, rotary, interleaved, eps, norm, dtype):
    """rope_reference with an axis for each pair: one pass to an axis, its pairs kept."""
    axis = np.zeros(rotary // 2, int) if pair_axis is None else np.clip(pair_axis, 0, len(pos) - 1)
    y, bound = rope_reference(x, gamma, pos[0], freq, rotary, interleaved, eps, norm, dtype)
    for a in range(1, len(pos)):
        ya, ba = rope_reference(x, gamma, pos[a], freq, rotary, interleaved, eps, norm, dtype)
        pairs = np.flatnonzero(axis == a)
        cols = np.concatenate((2 * pairs, 2 * pairs + 1) if interleaved else (pairs, pairs + rotary // 2)).astype(int)
        y[..., cols], bound[..., cols] = ya[..., cols], ba[..., cols]
    return y, bound


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d,rotary,axes,interleaved", [(4, 2, 64, 64, 1, False), (8, 1, 128, 128, 3, False), (3, 3, 80, 40, 2, True),
                                                              (2, 2, 256, 256, 3, True), (5, 5, 16, 8, 2, False), (2, 1, 96, 0, 1, False)])
@pytest.mark.parametrize("tokens", [1, 37])
def test_write(dev, dtype, hq, hk, d, rotary, axes, interleaved, tokens):
    say(f"write {dtype} {hq}/{hk} d={d} rotary={rotary} axes={axes} interleaved={interleaved} tokens={tokens}")
    g = np.random.default_rng(d + tokens)
    q, k, v = (rounded(3 * g.standard_normal((tokens, h, d), np.float32), dtype) for h in (hq, hk, hk))
    v = rounded(v * np.exp2(g.integers(-6, 6, v.shape[:2] + (1,))).astype(np.float32), dtype)
    gammas = [rounded(1 + 0.2 * g.standard_normal(d).astype(np.float32), dtype) for _ in "qk"]
    freq = (10000.0 ** (-np.arange(0, max(rotary, 1), 2) / max(rotary, 1))).astype(np.float32)[:max(rotary // 2, 1)]
    pos = positions_of(axes, tokens, g, 1000000)
    pair_axis = g.integers(-1, axes + 1, max(rotary // 2, 1)) if axes > 1 else None
    page_size, pages = 8, tokens // 8 + 3
    slots = g.permutation(pages * page_size)[:tokens]
    if tokens > 5:
        slots[[2, 5]] = -1, pages * page_size  # padding
    out = run_write(dtype, q, k, v, gammas, freq, pos, pair_axis, slots, pages, page_size, rotary, interleaved, k_out=True)
    args = (pos, freq, pair_axis, rotary, interleaved, 1e-6, True)
    want_q, q_bound = rotated(q, gammas[0], *args, dtype)
    close(out[0], want_q, q_bound, "q")
    want_k, k_bound = rotated(k, gammas[1], *args, dtype)
    close(out[1], want_k, k_bound, "k_out")
    # The cache: v is exact; k may round to the next number where 32 bits cross a border.
    want_k, k_off = rotated(k, gammas[1], *args, "f32")
    written = np.zeros((pages, page_size), bool)
    for t, slot in enumerate(slots):
        if not 0 <= slot < pages * page_size:
            continue
        page, at = slot // page_size, slot % page_size
        written[page, at] = True
        codes, scales = held(v[t])
        assert np.array_equal(out[3][page, at], codes) and np.array_equal(out[5][page, :, at], scales)
        got = stand_for(out[2][page, at], out[4][page, :, at])
        top = np.abs(want_k[t]).max(-1)
        power = np.exp2(out[4][page, :, at].astype(float) - 127)
        assert (448 * power >= top * (1 - 1e-5)).all() and (224 * power < top * (1 + 1e-5)).all()
        # Half a step: 2^-4 of the value, 2^-10 of the power below its 2^-6.
        close(got, want_k[t], np.abs(want_k[t]) * 2.0 ** -4 + power[:, None] * 2.0 ** -10 + 2 * k_off[t], "k")
    for x in out[2:4]:
        assert (x[~written] == 0x55).all()
    for x in out[4:6]:
        assert (x.transpose(0, 2, 1)[~written] == 0x55).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rounding_and_powers(dev, dtype):
    """Rows as they are (no norm, no rotation): ties, the smallest numbers, zeros,
    rows whose largest is 448 times a power, a step past it, denormal, the largest
    there is; infinities and NaN. Bit for bit, and k as v."""
    d, g = 64, np.random.default_rng(1)
    rows = [g.standard_normal(d) * s for s in (1, 1e-3, 1e3, 1e-7, 6e4, 1e-30, 1e30, 1e-37, 1e-44, 3e38)]
    rows += [np.full(d, x) for x in (0.0, -0.0, 448.0, 449.0, 450.0, 1.75, 1.76, 7 / 4 + 2.0 ** -7, 65504.0, 3.38e38, 1.2e-38)]
    ties = np.concatenate((np.arange(8, 16) + 0.5, -np.arange(8, 16) - 0.5, (np.arange(0, 8) + 0.5) * 2.0 ** -9, [448], np.zeros(39)))
    rows.append(ties)
    for odd in (math.inf, -math.inf, math.nan):
        x = g.standard_normal(d)
        x[::9] = odd
        rows.append(x)
    rows.append(np.full(d, math.nan))
    with np.errstate(over="ignore"):
        x = rounded(np.array(rows).astype(np.float32), dtype)[:, None]
    t = len(x)
    zero = np.zeros((t, 1, d), np.float32)
    _, _, kc, vc, ks, vs = run_write(dtype, zero, x, x, (None, None), np.ones(1, np.float32), np.zeros((1, t), int), None,
                                     np.arange(t), 4, 8, 0, norm=False)
    codes, scales = held(x)
    for c, s in ((kc, ks), (vc, vs)):
        c, s = c.reshape(32, 1, d)[:t], s.transpose(0, 2, 1).reshape(32, 1)[:t]
        assert np.array_equal(s, scales), (s.ravel(), scales.ravel())
        nan = np.isnan(x)
        assert np.array_equal(numbers(c), numbers(codes), equal_nan=True)
        # Zeros keep their sign where they had one.
        assert np.array_equal(np.signbit(numbers(c))[~nan & np.isfinite(x)], np.signbit(x)[~nan & np.isfinite(x)])


def test_write_in_place_and_many_tokens(dev):
    """q in place; more tokens than a workgroup has waves for each."""
    g = np.random.default_rng(2)
    t, d = 3001, 128
    q, k, v = (rounded(g.standard_normal((t, h, d), np.float32), "bf16") for h in (4, 2, 2))
    freq = (10000.0 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
    pos = np.arange(t)[None]
    slots = g.permutation(3200)[:t]
    a = run_write("bf16", q, k, v, (None, None), freq, pos, None, slots, 200, 16, d)
    b = run_write("bf16", q, k, v, (None, None), freq, pos, None, slots, 200, 16, d, in_place=True)
    for x, y in zip(a, b):
        assert x is None or np.array_equal(x, y)
    want, bound = rope_reference(q, None, pos[0], freq, d, False, 1e-6, True, "bf16")
    close(a[0], want, bound, "q")


# ---------------------------------------------------------------- reading back

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hk,d,page_size", [(1, 16, 1), (2, 64, 16), (5, 80, 7), (8, 128, 16), (3, 256, 24), (40, 208, 5)])
@pytest.mark.parametrize("tokens", [1, 50, 1500])
def test_read(dev, dtype, hk, d, page_size, tokens):
    say(f"read {dtype} heads={hk} d={d} page={page_size} tokens={tokens}")
    g = np.random.default_rng(d + tokens)
    s = Step8("f32", [1], [min(tokens, 300)], hk, hk, d, page_size=page_size, seed=d)
    s.put("k", g.integers(0, 256, s.k_codes.shape).astype(np.uint8), g.integers(0, 256, s.k_scales.shape).astype(np.uint8))
    cache, bufs = s.cache8_on_gpu()
    slots = g.integers(-3, s.pages * page_size + 3, tokens)
    pitch = hk * d + 8
    ds = ints_on_gpu(slots, np.int64)
    outs = [values_on_gpu(np.full((tokens, pitch), 7.0), dtype) for _ in "kv"]
    kh.synchronize()
    kh.paged_read8(kh.PagedRead8(cache=cache, slots=ds.ptr, k_out=outs[0].ptr, v_out=outs[1].ptr, k_out_stride=pitch,
                                 v_out_stride=pitch, tokens=tokens, dtype=DTYPES[dtype]))
    there = (slots >= 0) & (slots < s.pages * page_size)
    page, at = np.clip(slots, 0, s.pages * page_size - 1) // page_size, np.clip(slots, 0, s.pages * page_size - 1) % page_size
    for o, x in zip(outs, (s.k, s.v)):
        got = values_from_gpu(o, (tokens, pitch), dtype)
        with np.errstate(over="ignore"):
            want = rounded(x[page, at].reshape(tokens, hk * d).astype(np.float32), dtype)
        assert (got[:, hk * d:] == 7.0).all() and (got[~there] == 7.0).all()
        got, want = got[there, :hk * d], want[there]
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got), nan) and same_bits(got[~nan], want[~nan])


def test_read_one_of_both(dev):
    s = Step8("bf16", [1], [100], 2, 2, 64, seed=3)
    cache, bufs = s.cache8_on_gpu()
    ds, out = ints_on_gpu(np.arange(32), np.int64), values_on_gpu(np.zeros((32, 2, 64)), "bf16")
    for name, x in (("k_out", s.k), ("v_out", s.v)):
        kh.paged_read8(kh.PagedRead8(cache=cache, slots=ds.ptr, tokens=32, dtype=kh.BF16, k_out_stride=128, v_out_stride=128,
                                     **{name: out.ptr}))
        got, want = values_from_gpu(out, (32, 2, 64), "bf16"), x[:2].reshape(32, 2, 64)
        assert np.array_equal(got, want.astype(np.float32), equal_nan=True)


# ---------------------------------------------------------------- the three together

@pytest.mark.parametrize("dtype", list(DTYPES))
def test_written_rows_are_read_and_attended(dev, dtype):
    """Rows written, read back, written again (the same values), and attended over."""
    g = np.random.default_rng(4)
    t, hq, hk, d, ps = 70, 4, 2, 64, 16
    q, k, v = (rounded(g.standard_normal((t, h, d), np.float32), dtype) for h in (hq, hk, hk))
    freq = (10000.0 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
    pos = np.stack((np.arange(t), np.arange(t) // 8, np.arange(t) % 8))
    pair_axis = np.arange(d // 2) % 3
    order = g.permutation(5)
    slots = order[np.arange(t) // ps] * ps + np.arange(t) % ps
    qo, _, kc, vc, ks, vs = run_write(dtype, q, k, v, (None, None), freq, pos, pair_axis, slots, 5, ps, d)
    s = Step8(dtype, [t], [t], hq, hk, d, seed=4)
    s.pages, s.table, s.q = 5, order[None].astype(np.int32), qo.reshape(t, hq * d)
    s.put("k", kc, ks.transpose(0, 2, 1))
    s.put("v", vc, vs.transpose(0, 2, 1))
    check_attention(s)
    cache, bufs = s.cache8_on_gpu()
    ds = ints_on_gpu(slots, np.int64)
    outs = [values_on_gpu(np.zeros((t, hk, d)), dtype) for _ in "kv"]
    kh.synchronize()
    kh.paged_read8(kh.PagedRead8(cache=cache, slots=ds.ptr, k_out=outs[0].ptr, v_out=outs[1].ptr, k_out_stride=hk * d,
                                 v_out_stride=hk * d, tokens=t, dtype=DTYPES[dtype]))
    k2, v2 = (values_from_gpu(o, (t, hk, d), dtype) for o in outs)
    again = run_write(dtype, q, k2, v2, (None, None), freq, pos, None, slots, 5, ps, 0, norm=False)
    for codes, scales, codes2, scales2 in ((kc, ks, again[2], again[4]), (vc, vs, again[3], again[5])):
        assert np.array_equal(stand_for(codes2, scales2.transpose(0, 2, 1)), stand_for(codes, scales.transpose(0, 2, 1)))
