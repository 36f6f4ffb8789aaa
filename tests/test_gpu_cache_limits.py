"""The sequence-cache operators on the GPU at the ends of their ranges:
sequences without new tokens, long caches, scores of any size, rows that add
nothing."""
import math

import numpy as np
import pytest

import kernelh as kh
from cachetest import (DTYPES, Step, decode, encode, evict_reference, half_step, ints_on_gpu, rope_reference, rounded, same_bits,
                       values_from_gpu, values_on_gpu)
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


# ---------------------------------------------------------------- scores of any size

def row_of_scores(dtype, m, n, spread, window=0, hq=2, hk=1, d=64):
    """A step of m tokens of n entries whose scores are a * c_j in every row, a
    product of one column: c_j from `spread` in turn. Values of V are small whole
    numbers. The Step, and c."""
    s = Step(dtype, [m], [n], hq, hk, d, seed=n, window=window)
    c = np.array([spread[j % len(spread)] for j in range(n)], np.float64)
    page, slot = s.table[0][np.arange(n) // 16], np.arange(n) % 16
    s.k[page, slot] = 0.0
    s.q[:] = 0.0
    s.v[page, slot] = s.g.integers(-8, 9, (n, hk, d)).astype(np.float32)
    return s, c, page, slot


@pytest.mark.parametrize("dtype,q,k", [("f32", 2.0 ** 60, -2.0 ** 55), ("bf16", 2.0 ** 60, -2.0 ** 55), ("f32", 2.0 ** 60, 2.0 ** 55),
                                       ("f32", 1.1e18, -1.3e17), ("bf16", -1.3125e19, 1.0625e17), ("f16", 60000.0, -20000.0),
                                       ("f16", 60000.0, 21024.0), ("bf16", 23040.0, -52480.0), ("f32", 60001.0, -20011.0)])
@pytest.mark.parametrize("m,n", [(1, 50), (1, 3000), (9, 700), (100, 1500)])
def test_scores_far_from_zero(dev, dtype, q, k, m, n):
    """Scores of 10^8 to 10^35 of either sign, few values apart by more than
    the exponential can tell: a row's largest, each counted once, and nothing
    else. Single tokens, chunks, whole and in parts."""
    spread = [3.0, 2.0, 1.0, 1.0, 2.0]
    s, c, page, slot = row_of_scores(dtype, m, n, spread)
    s.q.reshape(s.tokens, s.hq, s.d)[:, :, 7] = q = rounded(np.full(1, q), dtype)[0]
    s.k[page, slot, 0, 7] = k = rounded(c * k, dtype)
    for workspace in (None, 0):
        say(f"far scores {dtype} {q} {k} m={m} n={n} ws={workspace}")
        out, lse = s.run_attention(workspace=workspace)
        x = k.astype(np.float64) * float(q) * s.scale
        for i in range(m):
            here = x[:n - m + i + 1]
            top = here == here.max()
            want = s.v[page, slot, 0][:n - m + i + 1][top].astype(np.float64).mean(0)
            # Weights of ones: their sums are exact, the quotient rounds twice
            # (reciprocal and product), the result once.
            bound = np.abs(want) * (2.0 ** -21 + half_step(dtype)) + (2.0 ** -25 if dtype == "f16" else 1e-30)
            for h in range(s.hq):
                close(out[i, h], want, bound, f"token {i}")
                # The product and the factor round, and what the sum adds is less than a step of it.
                close(lse[i, h], here.max(), abs(here.max()) * 2.0 ** -21, "lse")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,n", [(1, 4000), (1, 60000), (5, 4000), (100, 4000)])
def test_many_small_weights_beside_a_large_one(dev, dtype, m, n):
    """An entry whose value is 0 takes all but e^-18 of the others' weight, each
    a little below 2^-25 of its own: what the others add is the result."""
    s, _, page, slot = row_of_scores(dtype, m, n, [0.0])
    s.q.reshape(s.tokens, s.hq, s.d)[:, :, 7] = 1.0
    s.k[page[0], slot[0], 0, 7] = 18.0 / s.scale
    s.v[page, slot] = 64.0
    s.v[page[0], slot[0]] = 0.0
    for workspace in (None, 0):
        say(f"small weights {dtype} m={m} n={n} ws={workspace}")
        out, lse = s.run_attention(workspace=workspace)
        rest = (n - m + np.arange(m)) * math.exp(-18.0)
        want = (64.0 * rest / (1.0 + rest))[:, None, None]
        # A small weight rounds once to the type, all of them alike, and so does
        # the result; the exponent is off by a few steps of 26 in 32 bits, and n
        # terms are added in that many.
        u = half_step(dtype)
        rel = 8 * 26 * 2.0 ** -24 + 2 * (n + 64) * 2.0 ** -24
        bound = want * ((2 * u if dtype != "f32" else u) + rel) + (2.0 ** -25 if dtype == "f16" else 0.0)
        close(out, np.broadcast_to(want, out.shape), np.broadcast_to(bound, out.shape), "out")
        y = (18.0 + np.log1p(rest))[:, None]
        close(lse, np.broadcast_to(y, lse.shape), np.broadcast_to(rel + 2.0 ** -22 * y, lse.shape), "lse")


@pytest.mark.parametrize("dtype,size", [("f32", 2.0 ** 62), ("bf16", 2.0 ** 62), ("f16", 2.0 ** 14)])
@pytest.mark.parametrize("scale", [0.0, -0.0, 2.0 ** -149, -2.0 ** -140, 2.0 ** -120, 3.4e38])
@pytest.mark.parametrize("m,n", [(1, 300), (100, 300)])
def test_scales_at_their_ends(dev, dtype, size, scale, m, n):
    """Scores of q . k = 0 or +-size^2 under scales of 0, of denormal numbers and
    of the largest: the softmax of the scaled ones."""
    s, _, page, slot = row_of_scores(dtype, m, n, [0.0])
    s.scale = scale
    signs = s.g.integers(-1, 2, n)
    signs[0] = 1
    if scale > 1:
        signs[:] = 0  # the largest scale has only scores of 0 left that are numbers
    s.q.reshape(s.tokens, s.hq, s.d)[:, :, 7] = size
    s.k[page, slot, 0, 7] = signs * size
    say(f"scale {scale} {dtype} m={m}")
    out, lse = s.run_attention()
    # The scale as it is taken: a float of the call.
    x = signs.astype(np.float64) * size * size * float(np.float32(scale))
    for i in range(m):
        here = x[:n - m + i + 1]
        top = here.max()
        p = np.exp(here - top)
        v = s.v[page, slot, 0][:len(here)].astype(np.float64)
        want, room = p @ v / p.sum(), p @ np.abs(v) / p.sum()
        # The factor of a denormal scale is one too, off by half the smallest of
        # them (2^-150) or less: of 2^124 at the most. The exponent rounds, and n terms.
        off = 2.0 ** -150 * size * size + 2.0 ** -22 * np.abs(here).max() + 2 * (n + 64) * 2.0 ** -24
        u = half_step(dtype)
        bound = room * (off + u) + np.abs(want) * u + (2.0 ** -25 if dtype == "f16" else 1e-30)
        for h in range(s.hq):
            close(out[i, h], want, bound, f"token {i}")
            y = top + math.log(p.sum())
            close(lse[i, h], y, off + 2.0 ** -22 * (abs(y) + 1), "lse")


@pytest.mark.parametrize("scale", [3.4e38, -3.4e38, 0.0])
@pytest.mark.parametrize("m", [1, 100])
def test_weights_of_scores_of_zero(dev, scale, m):
    """Keys of zeros under the largest scales: every entry receives exp(-lse)."""
    s, _, page, slot = row_of_scores("bf16", m, 200, [0.0])
    s.scale = scale
    s.q[:] = 1.0
    y = np.full((s.tokens, s.hq), math.log(4.0), np.float32)
    before = s.g.random((1, 1, 205), np.float32)
    say(f"weights, scale {scale} m={m}")
    got = s.run_weights(y, before)
    want, bound = s.weights(y, before)
    close(got[0, :, :200], want[0, :, :200], bound[0, :, :200], "weights")


# ---------------------------------------------------------------- rows that add nothing

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("page_size", [16, 24])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("m", [3, 70])
def test_weights_skip_rows_of_minus_infinity_whatever_they_hold(dev, dtype, page_size, value, m):
    """lse = -inf says that a row saw nothing: what stands in its queries, or in
    a key that only such rows see, reaches no weight."""
    s = Step(dtype, [m, 1], [m + 130, 40], 4, 2, 64, page_size=page_size, seed=m)
    y = s.attention()[2].astype(np.float32)
    rows = [1, 2] if m == 3 else [1, 30, 31, 47, 69]
    y[rows] = -math.inf
    want_from = Step(dtype, [m, 1], [m + 130, 40], 4, 2, 64, page_size=page_size, seed=m)
    s.q[rows] = value
    # The last token's own entry, which no other token sees.
    at = m + 129
    s.k[s.table[0, at // page_size], at % page_size, 0, 5] = value
    cap = m + 135
    before = want_from.g.random((2, 2, cap), np.float32)
    say(f"weights {dtype} page={page_size} m={m} value={value} in rows of lse -inf")
    got = s.run_weights(y, before)
    want, bound = want_from.weights(y, before)
    for i, n in enumerate((m + 130, 40)):
        close(got[i, :, :n], want[i, :, :n], bound[i, :, :n], f"sequence {i}")


# ---------------------------------------------------------------- many tokens

def test_rotation_of_more_tokens_than_a_launch_has_threads_for(dev):
    """2^26 and some tokens of one short head, one row shared by all as a stride
    of 0 says: each turned by its own position."""
    t, d = (1 << 26) + 1003, 8
    g = np.random.default_rng(2)
    x = [rounded(g.standard_normal((1, 1, d), np.float32), "bf16") for _ in "qk"]
    dx = [values_on_gpu(v, "bf16") for v in x]
    freq = np.array([1.0, 0.37, 0.01, 1e-4], np.float32)
    df, pos = values_on_gpu(freq, "f32"), np.arange(t, dtype=np.int64)
    dp = ints_on_gpu(pos, np.int64)
    out = [kh.Buffer(t * d * 2) for _ in "qk"]
    say(f"rope of {t} tokens")
    kh.qk_norm_rope(kh.QkNormRope(q=dx[0].ptr, k=dx[1].ptr, q_out=out[0].ptr, k_out=out[1].ptr, inv_freq=df.ptr, positions=dp.ptr,
                                  q_stride=0, k_stride=0, q_out_stride=d, k_out_stride=d,
                                  cache=kh.PagedCache(kv_heads=1, head_dim=d, dtype=kh.BF16), tokens=t, q_heads=1, rotary_dim=d,
                                  interleaved=0, norm=1, eps=1e-6))
    kh.synchronize()
    for at in (0, (1 << 25) - 500, (1 << 26) - 500, t - 1000):
        mine = pos[at:at + 1000]
        for i, name in enumerate("qk"):
            bits = np.empty((1000, 1, d), np.int16)
            kh.check(kh.lib.khrt_memcpy_d2h(bits.ctypes.data, out[i].ptr + at * d * 2, bits.nbytes))
            want, bound = rope_reference(np.broadcast_to(x[i], (1000, 1, d)), None, mine, freq, d, 0, 1e-6, 1, "bf16")
            close(decode(bits, "bf16"), want, bound, f"{name} from token {at}")


# ---------------------------------------------------------------- workspaces

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_the_largest_steps_workspace_splits_smaller_ones_as_far_as_pays(dev, dtype):
    """With what the largest step reports, every smaller one comes out bit for
    bit as with any amount."""
    hq, hk, d = 8, 2, 64
    most = Step(dtype, [2048, 1, 1, 1], [4000, 3000, 2000, 100], hq, hk, d)
    cache, keep1 = most.cache_on_gpu()
    table, keep2 = most.table_on_gpu(4000)
    size = kh.paged_attention_workspace(kh.PagedAttention(
        cache=cache, table=table, q=cache.k, out=cache.v, lse=None, q_starts=table.lens, q_stride=hq * d, out_stride=hq * d,
        tokens=most.tokens, q_heads=hq, window=0, scale=0.125))
    del keep1, keep2
    for q_lens, lens in (([1], [4000]), ([1, 1, 1, 1], [4000, 3000, 2000, 100]), ([40], [4000]), ([300], [3999]),
                         ([128, 1], [2000, 4000]), ([700, 5, 9], [1000, 4000, 3000]), ([2048], [4000])):
        s = Step(dtype, q_lens, lens, hq, hk, d, seed=len(lens))
        a = check_attention(s, workspace=size, max_len=max(lens))
        b = s.run_attention(workspace=1 << 28, max_len=max(lens))
        assert all(same_bits(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------------- a chunk among single tokens

class Hinted(Step):
    """A step whose attention says max_new."""
    max_new = 0

    def run_attention(self, *args, **kw):
        made = kh.PagedAttention
        kh.PagedAttention = lambda **f: made(max_new=self.max_new, **f)
        try:
            return super().run_attention(*args, **kw)
        finally:
            kh.PagedAttention = made


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("chunk", [60, 150, 400])
def test_a_chunk_among_single_tokens(dev, dtype, chunk):
    """Forty single tokens with a chunk first, between and last; the longest
    said, not said, said too short and too long; with and without a workspace."""
    g = np.random.default_rng(chunk)
    lens = [int(x) for x in g.integers(1, 900, 41)]
    for at in (0, 17, 40):
        q_lens = [1] * 41
        q_lens[at], lens[at] = chunk, chunk + int(g.integers(0, 500))
        s = Hinted(dtype, q_lens, lens, 4, 1, 64, seed=chunk + at)
        for s.max_new in (0, chunk, 1, 1 << 40):
            for workspace in (None, 0):
                say(f"max_new={s.max_new} workspace={workspace}")
                check_attention(s, workspace=workspace)


# ---------------------------------------------------------------- caches past 4 GB

class Far:
    """A cache whose pages lie 2^28 elements of 16 bits apart, past 2^31 elements
    and 2^32 bytes: of each page only the slots are ever written or read."""

    def __init__(self, page_size, d=64, pages=20, seed=1):
        self.ps, self.d, self.pages, self.stride = page_size, d, pages, 1 << 28
        self.buf = kh.Buffer(pages * self.stride * 2)
        self.v_at = page_size * d * 2  # V behind K in each page
        self.g = np.random.default_rng(seed)
        self.k, self.v = (rounded(self.g.standard_normal((pages, page_size, 1, d), np.float32), "bf16") for _ in "kv")
        for p in range(pages):
            for at, x in ((0, self.k), (self.v_at, self.v)):
                a = encode(x[p], "bf16")
                kh.check(kh.lib.khrt_memcpy_h2d(self.buf.ptr + p * self.stride * 2 + at, a.ctypes.data, a.nbytes))
        self.cache = kh.PagedCache(k=self.buf.ptr, v=self.buf.ptr + self.v_at, k_page_stride=self.stride, k_slot_stride=d,
                                   k_head_stride=0, v_page_stride=self.stride, v_slot_stride=d, v_head_stride=0, pages=pages,
                                   page_size=page_size, kv_heads=1, head_dim=d, dtype=kh.BF16)

    def read(self):
        kh.synchronize()
        out = []
        for at in (0, self.v_at):
            x = np.empty((self.pages, self.ps, 1, self.d), np.int16)
            for p in range(self.pages):
                page = np.empty((self.ps, 1, self.d), np.int16)
                kh.check(kh.lib.khrt_memcpy_d2h(page.ctypes.data, self.buf.ptr + p * self.stride * 2 + at, page.nbytes))
                x[p] = page
            out.append(decode(x, "bf16"))
        return out

    def step(self, m, n):
        s = Step("bf16", [m], [n], 4, 1, self.d, page_size=self.ps, seed=m)
        s.pages, s.k, s.v = self.pages, self.k, self.v
        s.table = self.g.permutation(self.pages)[:-(-n // self.ps)].astype(np.int32).reshape(1, -1)
        s.cache_on_gpu = lambda: (self.cache, self.buf)
        return s


@pytest.mark.parametrize("page_size", [16, 24])
def test_attention_and_weights_past_4_gb(dev, page_size):
    far = Far(page_size)
    for m in (1, 5, 100):
        s = far.step(m, 20 * page_size - 3)
        say(f"far pages of {page_size}, {m} tokens")
        check_attention(s)
        check_weights(s)


@pytest.mark.parametrize("page_size", [16, 24])
def test_rotation_and_eviction_past_4_gb(dev, page_size):
    """New keys and values into every page, then eviction from the last pages
    to the first and the other way."""
    far = Far(page_size)
    d, t, pages = far.d, 20 * page_size, far.pages
    x = rounded(far.g.standard_normal((t, 6, d), np.float32), "bf16")
    slots = far.g.permutation(t).astype(np.int64)
    dx, ds, dq = values_on_gpu(x, "bf16"), ints_on_gpu(slots, np.int64), values_on_gpu(np.zeros((t, 4, d)), "bf16")
    say(f"far pages of {page_size}, rope")
    kh.qk_norm_rope(kh.QkNormRope(q=dx.ptr, k=dx.ptr + 4 * d * 2, v=dx.ptr + 5 * d * 2, q_out=dq.ptr, k_out=None, slots=ds.ptr,
                                  q_stride=6 * d, k_stride=6 * d, v_stride=6 * d, q_out_stride=4 * d, k_out_stride=d, cache=far.cache,
                                  tokens=t, q_heads=4, rotary_dim=0, interleaved=0, norm=0, eps=0.0))
    for got, want, i in zip(far.read(), (far.k, far.v), (4, 5)):
        want.reshape(t, d)[slots] = x[:, i]
        assert same_bits(got, want)
    for source, kept in ((np.arange(pages - 10, pages), np.arange(5)), (np.arange(8), np.arange(pages - 5, pages))):
        n, budget, recent = len(source) * page_size, 5 * page_size - 1, 7
        w = far.g.random((1, 1, n), np.float32)
        table, lens, dw, kt = ints_on_gpu(source), ints_on_gpu([n]), values_on_gpu(w, "f32"), ints_on_gpu(kept)
        out, klens = values_on_gpu(np.full((1, 1, budget), 7.0), "f32"), ints_on_gpu([-7])
        a = kh.PagedEvict(cache=far.cache, table=kh.PageTable(pages=table.ptr, lens=lens.ptr, row_stride=len(source), seqs=1,
                                                              width=len(source), max_len=0),
                          kept_pages=kt.ptr, kept_row_stride=5, kept_width=5, kept_lens=klens.ptr, weights_in=dw.ptr, in_seq_stride=n,
                          in_head_stride=n, weights=out.ptr, seq_stride=budget, head_stride=budget, budget=budget, recent=recent)
        size = kh.paged_evict_workspace(a)
        ws = kh.Buffer(size)
        say(f"far pages of {page_size}, eviction")
        kh.paged_evict(a, ws, size)
        ids = np.array(evict_reference(w[0, 0], n, budget, recent))
        to = np.arange(len(ids))
        for y in (far.k, far.v):
            y[kept[to // page_size], to % page_size] = y[source[ids // page_size], ids % page_size]
        for got, want in zip(far.read(), (far.k, far.v)):
            assert same_bits(got, want)
        assert same_bits(values_from_gpu(out, (budget,), "f32"), w[0, 0, ids]) and klens.to_host(np.int32)[0] == budget
