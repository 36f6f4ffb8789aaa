"""The sequence-cache operators on the GPU against their definitions in 64
bits: norms and rotation with the write to the cache, attention over ragged
sequences, the entries' weights, eviction. Bounds are of the arithmetic the
kernels are written in (tests/cachetest.py derives them); copies are exact."""
import math

import numpy as np
import pytest

import kernelh as kh
from cachetest import (DTYPES, Step, encode, evict_reference, ints_on_gpu, rope_reference, rounded, same_bits,
                       values_from_gpu, values_on_gpu)
from khtest import say

pytestmark = pytest.mark.gpu


def close(got, want, bound, what):
    got = got.astype(np.float64)
    with np.errstate(invalid="ignore"):
        off = np.where((got == want) | (np.isnan(got) & np.isnan(want)), 0.0, np.abs(got - want) / bound)
    off = np.where(np.isnan(off), math.inf, off)
    if off.size and off.max() > 1:
        at = np.unravel_index(off.argmax(), off.shape)
        pytest.fail(f"{what}: {off.max():.3g} of its bound at {tuple(map(int, at))}: {got[at]!r} for {want[at]!r}; "
                    f"{int((off > 1).sum())} of {off.size} are past it", pytrace=False)


def check_attention(s, what="attention", **kw):
    say(f"{what} {s.dtype} q={s.q_lens} n={s.lens} heads={s.hq}/{s.hk} d={s.d} page={s.page_size} window={s.window} {kw}")
    out, lse = s.run_attention(**kw)
    want, bound, y, y_bound = s.attention()
    inside = np.zeros(s.tokens, bool)
    inside[s.starts[0]:s.starts[-1]] = True
    close(out[inside], want[inside], bound[inside], "out")
    if kw.get("with_lse", True):
        close(lse[inside], y[inside], y_bound[inside], "lse")
    assert (out[~inside] == 7.0).all() and (lse[~inside] == 7.0).all()  # tokens of no sequence
    return out, lse


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d", [(1, 1, 64), (4, 4, 64), (8, 2, 128), (32, 8, 128), (7, 1, 80), (6, 2, 8), (5, 5, 256),
                                     (24, 1, 96), (4, 2, 136), (2, 1, 72), (3, 1, 200)])
def test_single_tokens(dev, dtype, hq, hk, d):
    check_attention(Step(dtype, [1, 1, 1, 1, 1], [1, 2, 33, 500, 129], hq, hk, d, seed=d + hq))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("page_size", [1, 3, 16, 24, 64, 1000])
def test_pages_that_end_inside_a_tile(dev, dtype, page_size):
    check_attention(Step(dtype, [1, 2, 1], [1, 257, 700], 4, 2, 64, page_size=page_size, seed=page_size))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d", [(4, 4, 64), (8, 2, 128), (3, 1, 80), (2, 2, 256), (6, 2, 40)])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_chunks(dev, dtype, hq, hk, d, window):
    check_attention(Step(dtype, [17, 1, 64, 5, 130], [17, 40, 200, 5, 333], hq, hk, d, page_size=24, window=window,
                         seed=d + window))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_long_chunk(dev, dtype):
    check_attention(Step(dtype, [300, 515], [300, 1100], 4, 2, 128, seed=3))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q_lens,lens,hq,hk,d", [([50], [4000], 4, 2, 64), ([70], [2100], 2, 1, 128), ([20], [1500], 4, 1, 256),
                                                 ([40, 1, 0, 130, 9], [3000, 2000, 50, 700, 1300], 8, 2, 128),
                                                 ([33, 32, 8], [900, 901, 902], 1, 1, 80)])
@pytest.mark.parametrize("window", [0, 700])
def test_chunks_over_long_caches(dev, dtype, q_lens, lens, hq, hk, d, window):
    """Sequences of many rows whose entries are split over workgroups, alone
    and beside sequences of few rows; with and without a workspace."""
    s = Step(dtype, q_lens, lens, hq, hk, d, seed=d, window=window, page_size=24, before=1, after=2)
    for workspace in (None, 0, 300000):
        check_attention(s, workspace=workspace)


def test_more_sequences_than_lanes(dev):
    """A hundred and fifty sequences of all kinds."""
    g = np.random.default_rng(0)
    q_lens = [int(x) for x in g.choice([0, 1, 1, 1, 2, 30], 150)]
    lens = [int(x) for x in g.integers(0, 300, 150)]
    check_attention(Step("bf16", q_lens, lens, 4, 2, 64, seed=1))
    check_attention(Step("f16", [1] * 150, lens, 4, 2, 64, seed=2))


def test_starts_that_do_not_ascend(dev):
    """Sequences that claim the same tokens: whatever they get, the call ends,
    and tokens of no sequence are left alone."""
    s = Step("bf16", [40] * 6, [100] * 6, 4, 2, 64, seed=3, before=1, after=2)
    s.starts = [1, 200, 1, 200, 1, 200, 150]
    out, lse = s.run_attention()
    assert (out[[0, -1, -2]] == 7.0).all() and (lse[[0, -1, -2]] == 7.0).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("workspace", [0, None, 20000])
@pytest.mark.parametrize("q", [1, 5])
def test_long_sequences_split_and_not(dev, dtype, workspace, q):
    """One long sequence and short ones, with all splits, few and none; the
    expected length said, not said, and said too short."""
    s = Step(dtype, [q, q, q], [5000, 7, 130], 4, 1, 64, seed=11, page_size=16)
    for max_len in (0, 5000, 300):
        check_attention(s, workspace=workspace, max_len=max_len)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("window", [0, 3])
def test_rows_that_see_nothing(dev, dtype, window):
    """No entries, fewer entries than new tokens, a sequence without new
    tokens, and a length below zero."""
    s = Step(dtype, [2, 9, 0, 3, 1], [0, 4, 50, 3, -5], 4, 2, 64, seed=5, window=window, before=2, after=3)
    out, lse = check_attention(s)
    assert (out[2:4] == 0).all() and (lse[2:4] == -math.inf).all()
    assert (out[4:9] == 0).all() and (lse[4:9] == -math.inf).all()
    assert (out[-4] == 0).all() and (lse[-4] == -math.inf).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [-1, 1 << 30, "pages"])
def test_pages_that_do_not_exist(dev, dtype, bad):
    s = Step(dtype, [1, 40, 1], [100, 90, 64], 4, 2, 64, seed=6)
    s.table[0, 2] = s.table[1, 0] = s.pages if bad == "pages" else bad
    s.table[2, :] = s.pages if bad == "pages" else bad
    out, lse = check_attention(s)
    assert (out[-1] == 0).all() and (lse[-1] == -math.inf).all()


def test_a_length_past_the_table_and_starts_out_of_range(dev):
    """Lengths past what the row can hold are cut to it; starts past the
    tokens are cut to them."""
    s = Step("bf16", [1, 1], [40, 64], 4, 2, 64, seed=7)
    s.lens = [40, 1 << 30]
    check_attention(s)
    out, _ = check_attention(s)
    s.starts = [0, 1, 1 << 30]
    again, _ = s.run_attention()
    assert same_bits(again, out)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["keys", "values"])
def test_later_entries_do_not_reach_earlier_tokens(dev, dtype, value, where):
    """An infinity or NaN in the key or value of a token of the chunk, and,
    with a window, of one that has left it, stays out of the rows that do not
    see it."""
    for window, at in ((0, 70), (20, 3), (0, 79)):
        s = Step(dtype, [50], [80], 4, 2, 64, seed=8, window=window)
        x = s.k if where == "keys" else s.v
        x[s.table[0, at // 16], at % 16, 1, 5] = value
        say(f"poison {dtype} {value} {where} {window} {at}")
        out, lse = s.run_attention()
        want, bound, y, y_bound = s.attention()
        sees = s.seen(0)[:, at]
        clean = ~sees
        close(out[clean], want[clean], bound[clean], "rows that do not see it")
        close(lse[clean], y[clean], y_bound[clean], "their lse")
        close(out[:, :2], want[:, :2], bound[:, :2], "the other kv head")
        if where == "values":
            rest = [e for e in range(64) if e != 5]
            close(out[..., rest], want[..., rest], bound[..., rest], "the other columns")
            hit = out[sees, 2:, 5]
            assert np.isnan(hit).all() if math.isnan(value) else (hit == value).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_layouts_and_strides(dev, dtype):
    """Heads before slots in a page; tokens of q further apart than their
    heads; padding rows on both sides left alone."""
    check_attention(Step(dtype, [1, 30, 1], [90, 64, 33], 8, 4, 64, seed=9, heads_first=True, pad=128, before=3, after=5))
    check_attention(Step(dtype, [1, 1, 1], [3000, 64, 33], 8, 4, 64, seed=9, heads_first=True, pad=64, before=1, after=2))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_large_scores(dev, dtype):
    """Scores of a few hundred: only the largest of a row counts."""
    check_attention(Step(dtype, [3, 20], [400, 20], 4, 2, 64, seed=10, spread=6.0))


def test_without_lse_and_on_another_stream(dev):
    s = Step("bf16", [1, 1], [2000, 40], 4, 2, 64, seed=12)
    st = kh.Stream()
    a, _ = check_attention(s, stream=st, with_lse=False)
    b, _ = check_attention(s)
    st.destroy()
    assert same_bits(a, b)


def test_repeated_calls_give_the_same_bits(dev):
    for s in (Step("bf16", [1, 1], [3000, 40], 8, 2, 128, seed=13), Step("f32", [200], [900], 4, 2, 64, seed=13)):
        a, b = s.run_attention(), s.run_attention()
        assert all(same_bits(x, y) for x, y in zip(a, b))


def test_a_cache_past_32_bit_offsets(dev):
    """Entries whose offsets (in elements, and in bytes) pass 2^31 and 2^32: a
    view with a stride of 2^28 elements a page, of which only the rows that
    are used are written."""
    d, hk, pages, stride = 64, 1, 18, 1 << 28
    g = np.random.default_rng(1)
    buf = kh.Buffer(pages * stride * 2)
    rows = rounded(g.standard_normal((2, pages, d), np.float32), "bf16")
    for p in range(pages):
        for x in range(2):
            a = encode(rows[x, p], "bf16")
            kh.check(kh.lib.khrt_memcpy_h2d(buf.ptr + p * stride * 2 + x * 256, a.ctypes.data, a.nbytes))
    s = Step("bf16", [1], [pages], 2, hk, d, page_size=1, seed=2)
    s.pages, s.table = pages, g.permutation(pages).astype(np.int32).reshape(1, -1)
    s.k, s.v = rows.reshape(2, pages, 1, 1, d)
    cache = kh.PagedCache(k=buf.ptr, v=buf.ptr + 256, k_page_stride=stride, k_slot_stride=0, k_head_stride=0,
                          v_page_stride=stride, v_slot_stride=0, v_head_stride=0, pages=pages, page_size=1, kv_heads=hk,
                          head_dim=d, dtype=kh.BF16)
    s.cache_on_gpu = lambda: (cache, buf)
    check_attention(s, "far offsets")


# ---------------------------------------------------------------- norms and rotation

def run_rope(dtype, tokens, hq, hk, d, rotary, interleaved, norm=1, far=5000, page_size=16, gamma=True, in_place=False,
             with_cache=True, with_k=True, heads_first=False, seed=0, eps=1e-6):
    g = np.random.default_rng(seed)
    pitch = (hq + 2 * hk) * d + 16
    qkv = rounded(2 * g.standard_normal((tokens, pitch), np.float32), dtype)
    ends = ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk))
    parts = [qkv[:, a * d:b * d].reshape(tokens, b - a, d) for a, b in ends]
    gam = [rounded(1 + 0.3 * g.standard_normal(d, np.float32), dtype) if gamma else None for _ in "qk"]
    freq = (10000.0 ** (-np.arange(0, max(rotary, 2), 2) / max(rotary, 2))).astype(np.float32)
    pos = g.integers(-far // 10, far, tokens)
    pages = -(-tokens // page_size) + 2
    slots = g.permutation(pages * page_size)[:tokens]
    if tokens > 3:
        slots[1], slots[2], slots[3] = -1, pages * page_size, 1 << 40  # padding, and slots that do not exist
    shape = (pages, hk, page_size, d) if heads_first else (pages, page_size, hk, d)
    e = 4 if dtype == "f32" else 2
    dqkv = values_on_gpu(qkv, dtype)
    dq, dk = (values_on_gpu(np.full((tokens, h, d), 7.0), dtype) for h in (hq, hk))
    dc = [values_on_gpu(np.full(shape, 7.0), dtype) for _ in "kv"]
    dg = [values_on_gpu(x, dtype) if gamma else None for x in gam]
    df, dp, ds = values_on_gpu(freq, "f32"), ints_on_gpu(pos, np.int64), ints_on_gpu(slots, np.int64)
    cache = kh.PagedCache(kv_heads=hk, head_dim=d, dtype=DTYPES[dtype])
    if with_cache:
        st = (hk * page_size * d,) + ((d, page_size * d) if heads_first else (hk * d, d))
        cache = kh.PagedCache(k=dc[0].ptr, v=dc[1].ptr, k_page_stride=st[0], k_slot_stride=st[1], k_head_stride=st[2],
                              v_page_stride=st[0], v_slot_stride=st[1], v_head_stride=st[2], pages=pages,
                              page_size=page_size, kv_heads=hk, head_dim=d, dtype=DTYPES[dtype])
    qp, kp, vp = (dqkv.ptr + x * d * e for x in (0, hq, hq + hk))
    say(f"rope {dtype} t={tokens} {hq}/{hk} d={d} r={rotary} inter={interleaved} norm={norm} place={in_place} cache={with_cache}")
    kh.qk_norm_rope(kh.QkNormRope(
        q=qp, k=kp, v=vp, q_out=qp if in_place else dq.ptr, k_out=(kp if in_place else dk.ptr) if with_k else None,
        q_gamma=dg[0].ptr if gamma else None, k_gamma=dg[1].ptr if gamma else None, inv_freq=df.ptr, positions=dp.ptr,
        slots=ds.ptr, q_stride=pitch, k_stride=pitch, v_stride=pitch, q_out_stride=pitch if in_place else hq * d,
        k_out_stride=pitch if in_place else hk * d, cache=cache, tokens=tokens, q_heads=hq, rotary_dim=rotary,
        interleaved=interleaved, norm=norm, eps=eps))
    after = values_from_gpu(dqkv, qkv.shape, dtype)
    if in_place:
        got = [after[:, a * d:b * d].reshape(tokens, b - a, d) for a, b in ends[:2]]
        assert same_bits(after[:, (hq + hk) * d:], qkv[:, (hq + hk) * d:])
    else:
        got = [values_from_gpu(x, (tokens, h, d), dtype) for x, h in ((dq, hq), (dk, hk))]
        assert same_bits(after, qkv)
    want = []
    for i, name in enumerate("qk"):
        want.append(rope_reference(parts[i], gam[i], pos, freq, rotary, interleaved, eps, norm, dtype))
        if name == "k" and not with_k:
            assert (got[1] == 7.0).all()
        else:
            close(got[i], *want[i], name)
    cg = [values_from_gpu(x, shape, dtype) for x in dc]
    cg = [(x.transpose(0, 2, 1, 3) if heads_first else x).reshape(pages * page_size, hk, d) for x in cg]
    written = np.zeros(pages * page_size, bool)
    if with_cache:
        real = (slots >= 0) & (slots < pages * page_size)
        written[slots[real]] = True
        close(cg[0][slots[real]], want[1][0][real], want[1][1][real], "k in the cache")
        assert same_bits(cg[1][slots[real]], parts[2][real])
    assert all((x[~written] == 7.0).all() for x in cg)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d,rotary", [(16, 16, 64, 64), (32, 8, 128, 128), (3, 1, 80, 32), (5, 5, 96, 48), (2, 1, 256, 256),
                                            (7, 7, 8, 8), (4, 2, 72, 72), (9, 3, 136, 0), (6, 2, 248, 8)])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_norm_and_rotation(dev, dtype, hq, hk, d, rotary, interleaved):
    run_rope(dtype, 37, hq, hk, d, rotary, interleaved, seed=d + rotary)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens", [1, 2, 63, 1500, 5000])
def test_token_counts(dev, dtype, tokens):
    run_rope(dtype, tokens, 6, 2, 64, 64, 0, seed=tokens, page_size=24)


@pytest.mark.parametrize("kw", [dict(norm=0), dict(gamma=False), dict(in_place=True), dict(with_cache=False),
                                dict(with_k=False), dict(heads_first=True), dict(in_place=True, with_cache=False),
                                dict(far=2 ** 31), dict(far=2000000, interleaved=1), dict(norm=0, with_k=False)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_forms(dev, dtype, kw):
    run_rope(dtype, 50, 8, 2, 128, 128, **{"interleaved": 0, **kw})


def test_rotation_keeps_an_infinity_to_its_row_and_pair(dev):
    """Elements past the rotated ones are not multiplied by sines."""
    q = np.random.default_rng(1).standard_normal((4, 1, 64), np.float32)
    q[1, 0, 50] = math.inf
    dq, dk, out, kout = (values_on_gpu(x, "f32") for x in (q, q, 0 * q, 0 * q))
    pos, freq = ints_on_gpu(np.arange(4), np.int64), values_on_gpu(np.ones(8), "f32")
    kh.qk_norm_rope(kh.QkNormRope(q=dq.ptr, k=dk.ptr, q_out=out.ptr, k_out=kout.ptr, inv_freq=freq.ptr, positions=pos.ptr,
                                  q_stride=64, k_stride=64, q_out_stride=64, k_out_stride=64,
                                  cache=kh.PagedCache(kv_heads=1, head_dim=64, dtype=kh.F32), tokens=4, q_heads=1,
                                  rotary_dim=16, interleaved=0, norm=0, eps=0.0))
    got = values_from_gpu(out, q.shape, "f32")
    assert np.array_equal(got[..., 16:], q[..., 16:]) and np.isfinite(got[[0, 2, 3]]).all()


# ---------------------------------------------------------------- weights

def check_weights(s, in_place=False, lse=None):
    y = s.attention()[2] if lse is None else lse
    y = np.where(np.isnan(y), 0.0, y).astype(np.float32)
    cap = max(1, max(s.lens)) + 5
    before = s.g.random((len(s.lens), s.hk, cap), np.float32)
    say(f"weights {s.dtype} q={s.q_lens} n={s.lens} heads={s.hq}/{s.hk} d={s.d} page={s.page_size} window={s.window}")
    got = s.run_weights(y, before, in_place)
    want, bound = s.weights(y, before)
    for i in range(len(s.lens)):
        n = s.length(i)
        close(got[i, :, :n], want[i, :, :n], bound[i, :, :n], f"sequence {i}")
        assert (got[i, :, n:] == (before[i, :, n:] if in_place else 7.0)).all()
    return got


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d", [(4, 4, 64), (32, 8, 128), (7, 1, 80), (5, 5, 256), (24, 1, 96), (6, 2, 8)])
def test_weights_of_single_tokens(dev, dtype, hq, hk, d):
    check_weights(Step(dtype, [1, 1, 1, 1], [1, 33, 500, 129], hq, hk, d, seed=d))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (8, 2, 128), (3, 1, 80), (2, 2, 256)])
@pytest.mark.parametrize("window", [0, 1, 50])
@pytest.mark.parametrize("in_place", [False, True])
def test_weights_of_chunks(dev, dtype, hq, hk, d, window, in_place):
    check_weights(Step(dtype, [17, 1, 64, 0, 130], [17, 40, 200, 60, 333], hq, hk, d, page_size=24, window=window,
                       seed=d + window, before=2, after=1), in_place)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_weights_where_rows_see_nothing(dev, dtype):
    s = Step(dtype, [2, 9, 0, 3, 1, 1], [0, 4, 50, 3, -5, 64], 4, 2, 64, seed=5)
    s.table[5, 1] = -1
    check_weights(s)


def test_weights_repeat_bit_for_bit_and_skip_minus_infinity(dev):
    s = Step("bf16", [40, 1], [200, 100], 8, 2, 64, seed=4)
    y = s.attention()[2]
    y[3, :4] = -math.inf
    check_weights(s, lse=y)
    before = s.g.random((2, 2, 205), np.float32)
    a, b = s.run_weights(y, before), s.run_weights(y, before)
    assert same_bits(a, b)


# ---------------------------------------------------------------- eviction

def run_evict(dtype, lens, hk, d, budget, recent, page_size=16, seed=0, weights=None, heads_first=False):
    s = Step(dtype, [0] * len(lens), lens, 1 * hk, hk, d, page_size=page_size, seed=seed, stale=3.0, heads_first=heads_first)
    seqs, width = len(lens), -(-budget // page_size)
    first, extra = s.pages, seqs * width
    s.k, s.v = (np.concatenate((x, np.full((extra,) + x.shape[1:], 7.0, np.float32))) for x in (s.k, s.v))
    kept_table = (first + s.g.permutation(extra)).astype(np.int32).reshape(seqs, width)
    s.pages += extra
    cap = max(lens) + 3
    w = np.exp(2 * s.g.standard_normal((seqs, hk, cap), np.float32)) if weights is None else weights(seqs, hk, cap)
    cache, bufs = s.cache_on_gpu()
    table, keep = s.table_on_gpu()
    dkt, dw = ints_on_gpu(kept_table), values_on_gpu(w, "f32")
    want_w = np.full((seqs, hk, budget + 2), 7.0, np.float32)
    dout, dlens = values_on_gpu(want_w, "f32"), ints_on_gpu(np.full(seqs, -7))
    a = kh.PagedEvict(cache=cache, table=table, kept_pages=dkt.ptr, kept_row_stride=width, kept_width=width,
                      kept_lens=dlens.ptr, weights_in=dw.ptr, in_seq_stride=hk * cap, in_head_stride=cap,
                      weights=dout.ptr, seq_stride=hk * (budget + 2), head_stride=budget + 2, budget=budget, recent=recent)
    size = kh.paged_evict_workspace(a)
    ws = kh.Buffer(size)
    say(f"evict {dtype} n={lens} heads={hk} d={d} budget={budget} recent={recent} page={page_size}")
    kh.paged_evict(a, ws, size)
    kh.synchronize()
    got_lens, got_w = dlens.to_host(np.int32), values_from_gpu(dout, want_w.shape, "f32")
    want = [x.copy() for x in (s.k, s.v)]
    for i, n in enumerate(lens):
        n = max(n, 0)
        assert got_lens[i] == min(n, budget)
        for h in range(hk):
            ids = np.array(evict_reference(w[i, h], n, budget, recent), int)
            to = np.arange(len(ids))
            src, dst = s.table[i][ids // page_size], kept_table[i][to // page_size]
            for x in want:
                x[dst, to % page_size, h] = x[src, ids % page_size, h]
            want_w[i, h, :len(ids)] = w[i, h, ids]
    assert same_bits(got_w, want_w)
    for buf, x, was in zip(bufs, want, (s.k, s.v)):
        got = s.cache_from_gpu(buf)
        assert same_bits(got, x) and same_bits(got[:first], was[:first])  # the source as it was
    del keep


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hk,d,page_size", [(1, 64, 16), (8, 128, 16), (3, 80, 24), (2, 256, 1), (2, 8, 7)])
@pytest.mark.parametrize("budget,recent", [(100, 20), (64, 64), (1, 0), (130, 0)])
def test_eviction(dev, dtype, hk, d, page_size, budget, recent):
    run_evict(dtype, [300, 100, 101, 0, 1, 64, -3, 257], hk, d, budget, recent, page_size, seed=budget + d)


@pytest.mark.parametrize("n,budget,recent", [(5000, 4096, 256), (1025, 1024, 1), (1024, 1023, 0), (3000, 17, 5), (2049, 2048, 2048),
                                             (16384, 9000, 7), (16386, 16000, 100), (40000, 3333, 1111)])
def test_eviction_of_longer_sequences(dev, n, budget, recent):
    run_evict("bf16", [n, n - 1], 2, 64, budget, recent, seed=n)


@pytest.mark.parametrize("kind", ["equal", "zeros", "few values", "specials"])
def test_eviction_with_ties(dev, kind):
    """Of equal weights the lowest index is kept; -0 equals 0, NaN is above
    infinity."""
    def weights(seqs, hk, cap):
        g, shape = np.random.default_rng(3), (seqs, hk, cap)
        if kind == "equal":
            return np.full(shape, 0.25, np.float32)
        if kind == "zeros":
            return np.where(g.random(shape) < 0.5, 0.0, -0.0).astype(np.float32)
        if kind == "few values":
            return g.integers(0, 3, shape).astype(np.float32)
        w = g.standard_normal(shape, np.float32)
        w[..., 7::31], w[..., 9::31], w[..., 11::97] = math.inf, -math.inf, math.nan
        return w

    run_evict("f32", [1500, 700], 2, 64, 600, 50, weights=weights, heads_first=True)
