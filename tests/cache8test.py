"""Batches over a paged cache in 8 bits and what the cache holds (imported by
tests/test_gpu_cache8*.py); the operators' definitions in 64 bits are
cachetest.Step's, over the values that the bytes stand for."""
import math

import numpy as np

import kernelh as kh
from cachetest import DTYPES, Step, ints_on_gpu, values_from_gpu, values_on_gpu

LEAST, MOST = -117, 119  # of a row's exponent


def numbers(codes):
    """What e4m3 codes stand for."""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    e, f = c >> 3 & 15, c & 7
    size = np.where(e == 0, f * 2.0 ** -9, (8 + f) * np.exp2(e - 10.0))
    size = np.where(c & 0x7F == 0x7F, math.nan, size)
    return np.where(c & 0x80 != 0, -size, size)


def codes_of(x):
    """e4m3 codes of numbers of magnitude up to 448, rounded to nearest even."""
    x = np.asarray(x, np.float64)
    size = np.abs(np.nan_to_num(x, nan=0.0))
    e = np.maximum(np.frexp(np.where(size > 0, size, 1.0))[1] - 1, -6)
    e = np.where(size > 0, e, -6)
    steps = np.rint(np.ldexp(size, 3 - e)).astype(np.int64)  # 8..16 of them above 2^-6, 0..8 below
    up = steps == 16
    e, steps = np.where(up, e + 1, e), np.where(up, 8, steps)
    code = np.where(steps < 8, steps, (e + 7 << 3) + steps - 8)
    assert (code <= 0x7E).all()
    code = np.where(np.isnan(x), 0x7F, code)
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def held(x):
    """Codes and exponents, 127 added, that rows of x (float64, exact) are held as."""
    x = np.asarray(x, np.float64)
    ok = np.isfinite(x)
    top = np.where(ok, np.abs(x), 0.0).max(-1)
    part, e = np.frexp(top)
    e = np.where(top > 0, e - 9 + (part > 0.875), LEAST)
    e = np.clip(e, LEAST, MOST)
    with np.errstate(invalid="ignore"):
        y = np.where(ok, np.clip(np.ldexp(np.where(ok, x, 0.0), -e[..., None]), -448, 448), math.nan)
    return codes_of(y), (e + 127).astype(np.uint8)


_NUMBERS = numbers(np.arange(256)).astype(np.float32)


def stand_for(codes, scales):
    """Exact in 32 bits."""
    power = np.ldexp(np.float32(1), np.clip(np.asarray(scales, np.int32), 10, 246) - 127)
    return _NUMBERS[codes] * power[..., None]


class Step8(Step):
    """A step over a cache in 8 bits; k and v are what its bytes stand for, rows
    of v of many sizes. cap: of the scores. shared: the first entries of all
    sequences are the same, in the same pages or (an end of a page) copies."""

    def __init__(self, dtype, q_lens, lens, hq, hk, d, cap=0.0, shared=0, scale_pad=0, **kw):
        # Whole pages of shared entries are there once, the longest sequence's.
        ps = kw.get("page_size", 16)
        common, first = shared // ps * ps, max(range(len(lens)), key=lambda s: lens[s])
        own = [n if s == first else max(n - common, 0) if n > 0 else n for s, n in enumerate(lens)]
        super().__init__(dtype, q_lens, own, hq, hk, d, **kw)
        if shared:
            short, self.lens = self.table, list(lens)
            self.table = np.full((len(lens), max(1, max(-(-n // ps) for n in lens))), -1, np.int32)
            for s, n in enumerate(lens):
                have = min(common, max(n, 0))
                self.table[s, :-(-have // ps)] = short[first, :-(-have // ps)]
                rest = -(-max(n, 0) // ps) - common // ps
                if rest > 0:
                    at = common // ps if s == first else 0
                    self.table[s, common // ps:common // ps + rest] = short[s, at:at + rest]
        self.cap, self.shared, self.scale_pad = cap, shared, scale_pad
        # Rows of a pool, each with a size of its own.
        pool, pool_scales = held(kw.get("spread", 1.0) * self.g.standard_normal((257, d)))
        for name in "kv":
            stale = np.isnan(getattr(self, name)[..., 0])
            at = self.g.integers(0, 257, stale.shape)
            size = self.g.integers(-1, 2, stale.shape) * (1 if name == "k" else 8)
            codes, scales = pool[at], pool_scales[at] + size
            codes[stale], scales[stale] = 0x7F, 255
            self.put(name, codes, scales.astype(np.uint8))
        rest = shared - common
        for s in range(len(lens)) if rest else ():
            here = min(rest, lens[s] - common)
            if s != first and here > 0:
                a, b = self.table[s, common // ps], self.table[first, common // ps]
                for x in (self.k, self.v, self.k_codes, self.v_codes, self.k_scales, self.v_scales):
                    x[a, :here] = x[b, :here]

    def put(self, name, codes, scales):
        setattr(self, name + "_codes", codes)
        setattr(self, name + "_scales", scales)
        setattr(self, name, stand_for(codes, scales))

    def scores(self, s, h, k, on):
        x, off = super().scores(s, h, k, on)
        if self.cap:
            with np.errstate(invalid="ignore"):
                y = self.cap * np.tanh(np.where(on, x, 0.0) / self.cap)
            # The cap's slope is at most 1. Its own error: some 8 roundings of the
            # series; 2^-22 of the cap past a quarter of it, which is 2^-20 of the score.
            off = off + np.where(on, 2.0 ** -20 * np.abs(y), 0.0)
            x = np.where(on, y, -math.inf)
        return x, off

    def cache8_on_gpu(self):
        ps, hk, d = self.page_size, self.hk, self.d
        data = [np.ascontiguousarray(x.transpose(0, 2, 1, 3) if self.heads_first else x) for x in (self.k_codes, self.v_codes)]
        row = ps + self.scale_pad
        scales = np.full((2, self.pages, hk, row), 77, np.uint8)
        for x, y in zip(scales, (self.k_scales, self.v_scales)):
            x[:, :, :ps] = y.transpose(0, 2, 1)
        bufs = [kh.Buffer.from_array(x) for x in (*data, *scales)]
        page, slot, head = (hk * ps * d, d, ps * d) if self.heads_first else (hk * ps * d, hk * d, d)
        return kh.PagedCache8(k=bufs[0].ptr, v=bufs[1].ptr, k_scale=bufs[2].ptr, v_scale=bufs[3].ptr, k_page_stride=page,
                              k_slot_stride=slot, k_head_stride=head, v_page_stride=page, v_slot_stride=slot, v_head_stride=head,
                              scale_page_stride=hk * row, scale_head_stride=row, pages=self.pages, page_size=ps, kv_heads=hk,
                              head_dim=d), bufs

    def args8(self, max_len=0, max_new=0, with_lse=True, shared=None):
        """The call's structure, and its buffers."""
        cache, keep1 = self.cache8_on_gpu()
        table, keep2 = self.table_on_gpu(max_len)
        q, starts = values_on_gpu(self.q, self.dtype), ints_on_gpu(self.starts)
        shape = (self.tokens, self.hq, self.d)
        out = values_on_gpu(np.full(shape, 7.0), self.dtype)
        lse = values_on_gpu(np.full(shape[:2], 7.0), "f32")
        a = kh.PagedAttention8(cache=cache, table=table, q=q.ptr, out=out.ptr, lse=lse.ptr if with_lse else None,
                               q_starts=starts.ptr, q_stride=self.q_pitch, out_stride=self.hq * self.d, tokens=self.tokens,
                               q_heads=self.hq, window=self.window, max_new=max_new,
                               shared=self.shared if shared is None else shared, scale=self.scale, cap=self.cap,
                               dtype=DTYPES[self.dtype])
        return a, {"out": out, "lse": lse, "keep": (keep1, keep2, q, starts)}

    def results(self, bufs):
        shape = (self.tokens, self.hq, self.d)
        return values_from_gpu(bufs["out"], shape, self.dtype), values_from_gpu(bufs["lse"], shape[:2], "f32")

    def run_attention(self, workspace=None, stream=None, **kw):
        a, bufs = self.args8(**kw)
        size = kh.paged_attention8_workspace(a) if workspace is None else workspace
        ws = kh.Buffer(max(16, size))
        ws.fill(math.nan)
        kh.synchronize()
        kh.paged_attention8(a, ws if size else None, size, stream)
        if stream is not None:
            stream.synchronize()
        return self.results(bufs)
