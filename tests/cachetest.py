"""Batches over a paged cache and the operators' definitions in 64 bits
(imported by tests/test_gpu_cache*.py). Values are held as float32 arrays that
the element type represents exactly, and encoded on their way to the GPU."""
import math

import numpy as np

import kernelh as kh

DTYPES = {"f32": kh.F32, "f16": kh.F16, "bf16": kh.BF16}
_HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # a rounding's largest relative error


def half_step(dtype):
    return _HALF_STEP[dtype]


def encode(x, dtype):
    """float32 values in the element type's bits, rounded to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x.view(np.int32)
    if dtype == "f16":
        return x.astype(np.float16).view(np.int16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + (b >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r).view(np.int16)


def decode(b, dtype):
    if dtype == "f32":
        return b.view(np.float32)
    if dtype == "f16":
        return b.view(np.float16).astype(np.float32)
    return (b.view(np.uint16).astype(np.uint32) << 16).view(np.float32)


def rounded(x, dtype):
    return decode(encode(x, dtype), dtype)


def values_on_gpu(x, dtype):
    return kh.Buffer.from_array(encode(x, dtype))


def values_from_gpu(b, shape, dtype):
    kh.synchronize()
    n = int(np.prod(shape))
    return decode(b.to_host(np.int32 if dtype == "f32" else np.int16, n), dtype).reshape(shape)


def ints_on_gpu(x, dtype=np.int32):
    return kh.Buffer.from_array(np.asarray(x, dtype))


def same_bits(x, y):
    return np.array_equal(np.ascontiguousarray(x, np.float32).view(np.int32), np.ascontiguousarray(y, np.float32).view(np.int32))


def finite(x):
    """x with zeros for infinities and NaN."""
    return np.where(np.isfinite(x), x, 0.0)


class Step:
    """A step's inputs on the host: a cache whose unused slots hold `stale`,
    a table in random page order whose unused entries hold `spare_page`, and
    queries whose tokens lie `pad` elements apart more than they need."""

    def __init__(self, dtype, q_lens, lens, hq, hk, d, page_size=16, window=0, seed=0, stale=math.nan, spread=1.0,
                 heads_first=False, pad=0, before=0, after=0, spare_page=-1, width=None):
        self.g = g = np.random.default_rng(seed)
        self.dtype, self.heads_first = dtype, heads_first
        self.q_lens, self.lens, self.hq, self.hk, self.d = list(q_lens), list(lens), hq, hk, d
        self.page_size, self.window, self.scale = page_size, window, d ** -0.5
        need = [-(-max(n, 0) // page_size) for n in lens]
        width = width or max(1, max(need))
        self.pages = sum(need) + 2
        order = g.permutation(self.pages)
        self.table = np.full((len(lens), width), spare_page, np.int32)
        shape = (self.pages, page_size, hk, d)
        self.k, self.v = (np.full(shape, stale, np.float32) for _ in "kv")
        at = 0
        for s, n in enumerate(lens):
            mine = order[at:at + need[s]]
            at += need[s]
            self.table[s, :need[s]] = mine[:width]
            for x in (self.k, self.v):
                rows = self.normal((need[s] * page_size, hk, d), spread)
                rows[max(n, 0):] = stale
                x[mine] = rows.reshape(need[s], page_size, hk, d)
        self.starts = [before]
        for q in q_lens:
            self.starts.append(self.starts[-1] + q)
        self.tokens = self.starts[-1] + after
        self.q_pitch = hq * d + pad
        self.q = self.normal((self.tokens, self.q_pitch), spread)

    def normal(self, shape, spread=1.0):
        return rounded(spread * self.g.standard_normal(shape, np.float32), self.dtype)

    def rows(self, x, s, n):
        """Entries 0..n-1 of sequence s, [n, hk, d]; NaN where there is no page."""
        j = np.arange(n)
        page = self.table[s][j // self.page_size]
        out = x[np.clip(page, 0, self.pages - 1), j % self.page_size].astype(np.float64)
        out[(page < 0) | (page >= self.pages)] = math.nan
        return out

    def there(self, s, n):
        page = self.table[s][np.arange(n) // self.page_size]
        return (page >= 0) & (page < self.pages)

    def length(self, s):
        return min(max(self.lens[s], 0), self.table.shape[1] * self.page_size)

    def seen(self, s):
        """[new tokens, entries]: which see which."""
        n, m = self.length(s), self.q_lens[s]
        at, j = np.arange(n - m, n)[:, None], np.arange(n)
        on = (j <= at) & self.there(s, n)
        return on & (j > at - self.window) if self.window else on

    def queries(self, s, h):
        a = self.starts[s]
        return self.q[a:a + self.q_lens[s], h * self.d:(h + 1) * self.d].astype(np.float64)

    def scores(self, s, h, k, on):
        """Scores of head h of sequence s, -inf where not seen, and a bound of their error in 32 bits."""
        k = np.where(on.any(0)[:, None], k[:, h // (self.hq // self.hk)], 0.0)
        q = self.queries(s, h)
        with np.errstate(invalid="ignore"):
            x = q @ k.T * self.scale
            # A dot product of d terms in any order is off by d half steps of the
            # sum of magnitudes; the factor, the subtraction and 2^x add one each of
            # the values they take.
            off = (self.d + 4) * 2.0 ** -24 * abs(self.scale) * (np.abs(q) @ np.abs(k).T)
        return np.where(on, x, -math.inf), np.where(on, off, 0.0)

    # -- the operators' definitions

    def attention(self):
        """out, lse and bounds of their errors, [tokens, hq, ..]; NaN where no sequence has the token."""
        t, hq, d = self.tokens, self.hq, self.d
        out, bound = np.full((t, hq, d), math.nan), np.zeros((t, hq, d))
        lse, lse_bound = np.full((t, hq), math.nan), np.zeros((t, hq))
        u = half_step(self.dtype)
        for s, m in enumerate(self.q_lens):
            if m == 0:
                continue
            n, a = self.length(s), self.starts[s]
            on = self.seen(s)
            some = on.any(1)
            ks, vs = self.rows(self.k, s, n), self.rows(self.v, s, n)
            for h in range(hq):
                x, off = self.scores(s, h, ks, on)
                v = vs[:, h // (hq // self.hk)]
                with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
                    top = np.where(some, x.max(1, initial=-math.inf), 0.0)
                    y = np.where(some, top + np.log(np.exp(x - top[:, None]).sum(1)), -math.inf)
                    p = np.where(on, np.exp(x - np.where(some, y, 0.0)[:, None]), 0.0)
                    # Values that a row does not see do not count, whatever they are.
                    if np.isfinite(v).all():
                        o = p @ v
                    else:
                        o = np.stack([(p[i][on[i], None] * v[on[i]]).sum(0) for i in range(m)])
                size = finite(p) @ np.abs(finite(v))
                # p is off by the score's error and the maximum's, by the rounding of
                # the exponent (two values of that size) and of 2^x, and p and its
                # sum accumulate over n terms; 16 bits round p, and the result.
                largest = np.abs(finite(np.where(on, x, 0.0))).max(1, initial=0.0)
                rel = 2 * finite(off).max(1, initial=0.0) + 8 * 2.0 ** -24 * (largest + 1) + 2 * (n + 64) * 2.0 ** -24
                out[a:a + m, h] = o
                bound[a:a + m, h] = size * (rel[:, None] + (u if self.dtype != "f32" else 0.0)) + np.abs(finite(o)) * u + 1e-30
                if self.dtype == "f16":
                    # Below 2^-14 a step of fp16 no longer shrinks: p and out are off
                    # by up to 2^-25 on their own.
                    bound[a:a + m, h] += 2.0 ** -25 * (1 + np.abs(finite(v)).sum(0))
                lse[a:a + m, h] = y
                lse_bound[a:a + m, h] = rel + 2.0 ** -22 * np.abs(finite(y)) + 1e-30
        return out, bound, lse, lse_bound

    def weights(self, lse, before):
        """weights [seqs, hk, entries] after this step, and a bound of their error."""
        out, bound = before.astype(np.float64), np.zeros(before.shape)
        for s, m in enumerate(self.q_lens):
            n = self.length(s)
            out[s, :, max(0, n - m):n] = 0.0
            ks, seen = self.rows(self.k, s, n), self.seen(s)
            for h in range(self.hq if m else 0):
                y = lse[self.starts[s]:self.starts[s] + m, h].astype(np.float64)[:, None]
                x, off = self.scores(s, h, ks, seen)
                on = seen & (y > -math.inf)
                w = np.where(on, np.exp(x - np.where(y > -math.inf, y, 0.0)), 0.0)
                rel = off + 4 * 2.0 ** -24 * (np.abs(np.where(on, x, 0.0)) + np.abs(finite(y)) + 1)
                out[s, h // (self.hq // self.hk), :n] += w.sum(0)
                bound[s, h // (self.hq // self.hk), :n] += (w * rel).sum(0)
            bound[s, :, :n] += np.abs(out[s, :, :n]) * (m * self.hq // self.hk + 8) * 2.0 ** -24 + 1e-30
        return out, bound

    # -- the same on the GPU

    def cache_on_gpu(self):
        """The cache's structure and its two buffers."""
        bufs = tuple(values_on_gpu(x.transpose(0, 2, 1, 3) if self.heads_first else x, self.dtype) for x in (self.k, self.v))
        ps, hk, d = self.page_size, self.hk, self.d
        page, slot, head = (hk * ps * d, d, ps * d) if self.heads_first else (hk * ps * d, hk * d, d)
        return kh.PagedCache(k=bufs[0].ptr, v=bufs[1].ptr, k_page_stride=page, k_slot_stride=slot, k_head_stride=head,
                             v_page_stride=page, v_slot_stride=slot, v_head_stride=head, pages=self.pages, page_size=ps,
                             kv_heads=hk, head_dim=d, dtype=DTYPES[self.dtype]), bufs

    def cache_from_gpu(self, buf):
        shape = (self.pages, self.hk, self.page_size, self.d) if self.heads_first else (self.pages, self.page_size, self.hk, self.d)
        x = values_from_gpu(buf, shape, self.dtype)
        return x.transpose(0, 2, 1, 3) if self.heads_first else x

    def table_on_gpu(self, max_len=0):
        bufs = ints_on_gpu(self.table), ints_on_gpu(self.lens)
        return kh.PageTable(pages=bufs[0].ptr, lens=bufs[1].ptr, row_stride=self.table.shape[1], seqs=len(self.lens),
                            width=self.table.shape[1], max_len=max_len), bufs

    def run_attention(self, workspace=None, max_len=0, stream=None, with_lse=True):
        """out and lse; the buffers are filled with a pattern first."""
        cache, keep1 = self.cache_on_gpu()
        table, keep2 = self.table_on_gpu(max_len)
        q, starts = values_on_gpu(self.q, self.dtype), ints_on_gpu(self.starts)
        shape = (self.tokens, self.hq, self.d)
        dout = values_on_gpu(np.full(shape, 7.0), self.dtype)
        dlse = values_on_gpu(np.full(shape[:2], 7.0), "f32")
        a = kh.PagedAttention(cache=cache, table=table, q=q.ptr, out=dout.ptr, lse=dlse.ptr if with_lse else None,
                              q_starts=starts.ptr, q_stride=self.q_pitch, out_stride=self.hq * self.d,
                              tokens=self.tokens, q_heads=self.hq, window=self.window, scale=self.scale)
        size = kh.paged_attention_workspace(a) if workspace is None else workspace
        ws = kh.Buffer(max(16, size))
        ws.fill(math.nan)
        kh.synchronize()
        kh.paged_attention(a, ws if size else None, size, stream)
        if stream is not None:
            stream.synchronize()
        r = values_from_gpu(dout, shape, self.dtype), values_from_gpu(dlse, shape[:2], "f32")
        del keep1, keep2
        return r

    def run_weights(self, lse, before, in_place=False, stream=None, max_len=0):
        cache, keep1 = self.cache_on_gpu()
        table, keep2 = self.table_on_gpu(max_len)
        q, starts = values_on_gpu(self.q, self.dtype), ints_on_gpu(self.starts)
        dlse, din = values_on_gpu(lse, "f32"), values_on_gpu(before, "f32")
        dout = din if in_place else values_on_gpu(np.full(before.shape, 7.0), "f32")
        kh.paged_weights(kh.PagedWeights(
            cache=cache, table=table, q=q.ptr, lse=dlse.ptr, q_starts=starts.ptr, q_stride=self.q_pitch,
            weights_in=din.ptr, weights=dout.ptr, weights_seq_stride=before.shape[1] * before.shape[2],
            weights_head_stride=before.shape[2], tokens=self.tokens, q_heads=self.hq, window=self.window,
            scale=self.scale), stream)
        if stream is not None:
            stream.synchronize()
        r = values_from_gpu(dout, before.shape, "f32")
        del keep1, keep2
        return r


def rope_reference(x, gamma, pos, freq, rotary, interleaved, eps, norm, dtype):
    """x [tokens, heads, d] normalised and rotated in 64 bits, and a bound of the error of the 32-bit form."""
    d = x.shape[-1]
    x = x.astype(np.float64)
    if norm:
        x = x / np.sqrt(np.square(x).mean(-1, keepdims=True) + eps)
        if gamma is not None:
            x = x * gamma
    half = rotary // 2
    y, size = x.copy(), np.abs(x)
    if rotary:
        w = pos.astype(np.float64)[:, None] * freq.astype(np.float64)
        c, s = np.cos(w)[:, None], np.sin(w)[:, None]
        ia = np.arange(0, rotary, 2) if interleaved else np.arange(half)
        ib = ia + 1 if interleaved else ia + half
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        size[..., ia] = size[..., ib] = np.abs(a) + np.abs(b)
    # The sum of d squares, its root, the division and two products: (d + 8) half
    # steps; sine and cosine (their series in 32 bits, the last term left out) 8.
    bound = size * (d + 16) * 2.0 ** -24 + np.abs(y) * half_step(dtype) + 1e-30
    return y, bound + 2.0 ** -25 if dtype == "f16" else bound


def evict_reference(weights, n, budget, recent):
    """The kept entries of one head, in order; NaN ranks above infinity."""
    if n <= budget:
        return list(range(n))
    old = n - recent
    rank = [(0, 0.0) if math.isnan(w) else (1, -w) for w in weights[:old].tolist()]
    best = sorted(range(old), key=lambda j: (rank[j], j))[:budget - recent]
    return sorted(best) + list(range(old, n))
