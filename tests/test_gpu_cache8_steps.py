"""The operators over a cache in 8 bits as a program uses them: steps of a
decoder one after the other, on two streams, captured and replayed, repeated;
and over caches past 4 GB."""
import math

import numpy as np
import pytest

import kernelh as kh
from cachetest import DTYPES, half_step, ints_on_gpu, rounded, same_bits, values_from_gpu, values_on_gpu
from cache8test import Step8, codes_of, held, stand_for
from khtest import say
from test_gpu_cache import check_attention, close
from test_gpu_cache8 import rotated, run_write
from test_gpu_cache_steps import Graph

pytestmark = pytest.mark.gpu


class Decoder:
    """Sequences that share a beginning, in a cache of their own, grown step by
    step: the host keeps the tables, the GPU the cache."""

    def __init__(self, dtype, hq, hk, d, page_size, shared, seqs, window=0, cap=0.0, stream=None, seed=0):
        self.g = np.random.default_rng(seed)
        self.dtype, self.hq, self.hk, self.d, self.ps = dtype, hq, hk, d, page_size
        self.shared, self.window, self.cap, self.stream = shared, window, cap, stream
        self.pages = shared // page_size + seqs * 6 + 2
        self.order = list(self.g.permutation(self.pages))
        first = [self.order.pop() for _ in range(-(-shared // page_size))]
        assert shared % page_size == 0
        self.rows = [list(first) for _ in range(seqs)]
        self.lens = [shared] * seqs
        self.codes = [kh.Buffer.from_array(np.full((self.pages, page_size, hk, d), 0x7F, np.uint8)) for _ in "kv"]
        self.scales = [kh.Buffer.from_array(np.full((self.pages, hk, page_size), 255, np.uint8)) for _ in "kv"]
        self.cache = kh.PagedCache8(k=self.codes[0].ptr, v=self.codes[1].ptr, k_scale=self.scales[0].ptr, v_scale=self.scales[1].ptr,
                                    k_page_stride=page_size * hk * d, k_slot_stride=hk * d, k_head_stride=d,
                                    v_page_stride=page_size * hk * d, v_slot_stride=hk * d, v_head_stride=d,
                                    scale_page_stride=hk * page_size, scale_head_stride=page_size, pages=self.pages,
                                    page_size=page_size, kv_heads=hk, head_dim=d)
        self.freq = (10000.0 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
        self.axis = (np.arange(d // 2) % 3).astype(np.int32)
        self.dfreq, self.daxis = values_on_gpu(self.freq, "f32"), ints_on_gpu(self.axis)
        self.write([shared], [0], first_only=True)

    def write(self, new, seqs, first_only=False):
        """New tokens of these sequences: their rows written, q rotated. The step's inputs."""
        t = sum(new)
        slots, pos = [], []
        for m, s in zip(new, seqs):
            if first_only:
                at = range(m)
            else:
                at = range(self.lens[s], self.lens[s] + m)
                self.lens[s] += m
                while len(self.rows[s]) * self.ps < self.lens[s]:
                    self.rows[s].append(self.order.pop())
            slots += [self.rows[s][j // self.ps] * self.ps + j % self.ps for j in at]
            pos += [(j, j // 7, j % 7) for j in at]
        pos = np.array(pos).T.copy()
        qkv = rounded(self.g.standard_normal((t, self.hq + 2 * self.hk, self.d), np.float32), self.dtype)
        dqkv = values_on_gpu(qkv, self.dtype)
        e = 4 if self.dtype == "f32" else 2
        pitch = (self.hq + 2 * self.hk) * self.d
        dq = values_on_gpu(np.zeros((t, self.hq, self.d)), self.dtype)
        dpos, dslots = ints_on_gpu(pos, np.int64), ints_on_gpu(slots, np.int64)
        kh.synchronize()
        args = kh.QkNormRope8(q=dqkv.ptr, k=dqkv.ptr + self.hq * self.d * e, v=dqkv.ptr + (self.hq + self.hk) * self.d * e, q_out=dq.ptr,
                              inv_freq=self.dfreq.ptr, positions=dpos.ptr, pair_axis=self.daxis.ptr, slots=dslots.ptr, q_stride=pitch,
                              k_stride=pitch, v_stride=pitch, q_out_stride=self.hq * self.d, axis_stride=t, cache=self.cache, tokens=t,
                              q_heads=self.hq, rotary_dim=self.d, axes=3, norm=1, dtype=DTYPES[self.dtype], eps=1e-6)
        kh.qk_norm_rope8(args, self.stream)
        return {"qkv": qkv, "pos": pos, "slots": slots, "dq": dq, "t": t, "new": new, "seqs": seqs, "args": args,
                "keep": (dqkv, dpos, dslots)}

    def attend(self, step):
        """Attention of a step over the cache as it is, queued behind the write."""
        seqs, new = step["seqs"], step["new"]
        width = max(len(self.rows[s]) for s in seqs)
        table = np.full((len(seqs), width), -1, np.int32)
        for i, s in enumerate(seqs):
            table[i, :len(self.rows[s])] = self.rows[s]
        lens, starts = [self.lens[s] for s in seqs], np.concatenate(([0], np.cumsum(new)))
        keep = ints_on_gpu(table), ints_on_gpu(lens), ints_on_gpu(starts)
        out = values_on_gpu(np.full((step["t"], self.hq, self.d), 7.0), self.dtype)
        lse = values_on_gpu(np.full((step["t"], self.hq), 7.0), "f32")
        a = kh.PagedAttention8(cache=self.cache, table=kh.PageTable(pages=keep[0].ptr, lens=keep[1].ptr, row_stride=width, seqs=len(seqs),
                                                                   width=width, max_len=max(lens)),
                               q=step["dq"].ptr, out=out.ptr, lse=lse.ptr, q_starts=keep[2].ptr, q_stride=self.hq * self.d,
                               out_stride=self.hq * self.d, tokens=step["t"], q_heads=self.hq, window=self.window, max_new=max(new),
                               shared=self.shared, scale=self.d ** -0.5, cap=self.cap, dtype=DTYPES[self.dtype])
        size = kh.paged_attention8_workspace(a)
        ws = kh.Buffer(max(16, size))
        ws.fill(math.nan)
        kh.synchronize()
        kh.paged_attention8(a, ws, size, self.stream)
        step |= {"table": table, "lens": lens, "starts": starts, "out": out, "lse": lse, "ws": ws, "attention": a, "size": size, "keep2": keep}
        return step

    def check(self, step):
        """Against the definitions over what the cache holds now."""
        if self.stream is not None:
            self.stream.synchronize()
        kh.synchronize()
        shape = (self.pages, self.ps, self.hk, self.d)
        codes = [b.to_host(np.uint8, math.prod(shape)).reshape(shape) for b in self.codes]
        scales = [b.to_host(np.uint8, math.prod(shape[:3])).reshape(self.pages, self.hk, self.ps) for b in self.scales]
        want_q, bound = rotated(step["qkv"][:, :self.hq], None, step["pos"], self.freq, self.axis, self.d, False, 1e-6, True, self.dtype)
        q = values_from_gpu(step["dq"], (step["t"], self.hq, self.d), self.dtype)
        close(q, want_q, bound, "q")
        slots = np.array(step["slots"])
        v, vs = held(step["qkv"][:, self.hq + self.hk:])
        assert np.array_equal(codes[1][slots // self.ps, slots % self.ps], v)
        assert np.array_equal(scales[1][slots // self.ps, :, slots % self.ps], vs)
        s = Step8(self.dtype, step["new"], [1] * len(step["new"]), self.hq, self.hk, self.d, page_size=self.ps, window=self.window, cap=self.cap)
        s.pages, s.table, s.lens, s.tokens = self.pages, step["table"], step["lens"], step["t"]
        s.starts, s.q = list(step["starts"]), q.reshape(step["t"], -1)
        s.put("k", codes[0], scales[0].transpose(0, 2, 1))
        s.put("v", codes[1], scales[1].transpose(0, 2, 1))
        want, bound, y, y_bound = s.attention()
        close(values_from_gpu(step["out"], want.shape, self.dtype), want, bound, "out")
        close(values_from_gpu(step["lse"], y.shape, "f32"), y, y_bound, "lse")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d,page_size,window,cap", [(4, 4, 128, 16, 0, 0.0), (8, 2, 64, 24, 300, 5.0)])
def test_a_prompt_and_its_answers(dev, dtype, hq, hk, d, page_size, window, cap):
    """A common beginning is written; each sequence adds a chunk of its own, then
    single tokens and drafts, some sequences sitting out."""
    say(f"decoder {dtype} {hq}/{hk} d={d} page={page_size}")
    n = 30
    dec = Decoder(dtype, hq, hk, d, page_size, 1440, n, window, cap)
    for new, seqs in (([5 + 3 * i % 37 for i in range(n)], list(range(n))), ([1] * n, list(range(n))),
                      ([1 + i % 3 for i in range(n - 4)], list(range(2, n - 2))), ([1] * n, list(range(n)))):
        dec.check(dec.attend(dec.write(new, seqs)))


def programs(seed0, stream, dtype):
    """Steps whose attention shares out long sequences, joins parts, and works on
    shared entries apart; and a read."""
    steps = [Step8(dtype, [1, 2, 1], [3000, 40, 700], 8, 4, 128, seed=seed0),
             Step8(dtype, [1] * 40, [1500 + i for i in range(40)], 8, 8, 64, seed=seed0 + 1, shared=1400),
             Step8(dtype, [60, 1, 130], [900, 300, 200], 4, 2, 128, page_size=24, cap=4.0, seed=seed0 + 2)]
    calls = []
    for s in steps:
        a, bufs = s.args8()
        size = kh.paged_attention8_workspace(a)
        calls.append((s, a, bufs, kh.Buffer(max(16, size)), size))
    s = steps[0]
    cache, keep = s.cache8_on_gpu()
    slots = ints_on_gpu(np.arange(200), np.int64)
    out = [values_on_gpu(np.zeros((200, s.hk, s.d)), dtype) for _ in "kv"]
    read = kh.PagedRead8(cache=cache, slots=slots.ptr, k_out=out[0].ptr, v_out=out[1].ptr, k_out_stride=s.hk * s.d,
                         v_out_stride=s.hk * s.d, tokens=200, dtype=DTYPES[dtype])
    g = np.random.default_rng(seed0)
    t = 33
    rows = [values_on_gpu(rounded(g.standard_normal((t, h, s.d), np.float32), dtype), dtype) for h in (s.hq, s.hk, s.hk)]
    dq = values_on_gpu(np.zeros((t, s.hq, s.d)), dtype)
    freq, pos = values_on_gpu((10000.0 ** (-np.arange(0, s.d, 2) / s.d)).astype(np.float32), "f32"), ints_on_gpu(np.arange(t), np.int64)
    into = ints_on_gpu(np.arange(t) * 3, np.int64)
    codes = [kh.Buffer.from_array(np.zeros((8, 16, s.hk, s.d), np.uint8)) for _ in "kv"]
    scales = [kh.Buffer.from_array(np.zeros((8, s.hk, 16), np.uint8)) for _ in "kv"]
    own = kh.PagedCache8(k=codes[0].ptr, v=codes[1].ptr, k_scale=scales[0].ptr, v_scale=scales[1].ptr, k_page_stride=16 * s.hk * s.d,
                         k_slot_stride=s.hk * s.d, k_head_stride=s.d, v_page_stride=16 * s.hk * s.d, v_slot_stride=s.hk * s.d,
                         v_head_stride=s.d, scale_page_stride=16 * s.hk, scale_head_stride=16, pages=8, page_size=16, kv_heads=s.hk,
                         head_dim=s.d)
    write = kh.QkNormRope8(q=rows[0].ptr, k=rows[1].ptr, v=rows[2].ptr, q_out=dq.ptr, inv_freq=freq.ptr, positions=pos.ptr,
                           slots=into.ptr, q_stride=s.hq * s.d, k_stride=s.hk * s.d, v_stride=s.hk * s.d, q_out_stride=s.hq * s.d,
                           axis_stride=t, axes=1, cache=own, tokens=t, q_heads=s.hq, rotary_dim=s.d, norm=1, dtype=DTYPES[dtype], eps=1e-6)

    def launch():
        kh.qk_norm_rope8(write, stream)
        for _, a, _, ws, size in calls:
            kh.paged_attention8(a, ws, size, stream)
        kh.paged_read8(read, stream)

    written = [dq, *codes, *scales, *out] + [b for c in calls for b in (c[2]["out"], c[2]["lse"])]

    def clear():
        for b in written + [c[3] for c in calls]:
            b.fill(7.0, stream)
        (stream.synchronize if stream is not None else kh.synchronize)()

    def results():
        (stream.synchronize if stream is not None else kh.synchronize)()
        return [b.to_host(np.int32, b.nbytes // 4) for b in written]

    def check():
        for s, _, bufs, _, _ in calls:
            out, lse = s.results(bufs)
            want, bound, y, y_bound = s.attention()
            close(out, want, bound, "out")
            close(lse, y, y_bound, "lse")

    kh.synchronize()
    return launch, clear, results, check, (keep, slots, rows, freq, pos, into)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_two_streams_at_once(dev, dtype):
    streams = [kh.Stream(), kh.Stream()]
    ps = [programs(10 * i, st, dtype) for i, st in enumerate(streams)]
    for p in ps:
        p[1]()
    for _ in range(3):
        for p in ps:
            p[0]()
    got = [p[2]() for p in ps]
    for p, g in zip(ps, got):
        p[3]()
        p[1]()
        p[0]()
        assert all(np.array_equal(a, b) for a, b in zip(p[2](), g))  # alone: the same bits
    for st in streams:
        st.destroy()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_captured_calls_replay_as_they_ran(dev, dtype):
    """Every replay, from buffers and workspaces that were overwritten before it,
    with eager calls between, gives the bits of the eager run."""
    stream = kh.Stream()
    launch, clear, results, check, keep = programs(30, stream, dtype)
    clear()
    launch()
    want = results()
    check()
    graph = Graph(stream, launch)
    for turn in range(4):
        clear()
        graph.replay()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want)), f"replay {turn}"
        check_attention(Step8("f32", [1, 40], [90 + turn, 40], 4, 2, 64, seed=turn), "between replays", stream=stream)
        launch()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want)), f"eager after replay {turn}"
    graph.destroy()
    stream.destroy()


# ---------------------------------------------------------------- other forms of a call

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq", [8, 6])
def test_tokens_that_share_their_queries(dev, dtype, hq):
    """q_stride 0: one row of q is every token's."""
    s = Step8(dtype, [70, 1], [200, 90], hq, 2, 64, seed=32)
    s.q, s.q_pitch = np.repeat(s.q[:1], s.tokens, 0), 0
    check_attention(s)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,q_lens", [(20, [1, 1]), (64, [1, 2]), (40, [3, 1]), (17, [1, 30])])
@pytest.mark.parametrize("page_size", [16, 24, 512])
def test_many_heads_to_a_kv_head(dev, dtype, hq, q_lens, page_size):
    check_attention(Step8(dtype, q_lens, [200, 700], hq, 1, 64, page_size=page_size, seed=hq))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hk,d", [(3, 128), (5, 64), (6, 64), (7, 128), (9, 64), (2, 256)])
def test_heads_that_do_not_fill_their_group(dev, dtype, hk, d):
    """Long enough for heads of an entry to be read together; the last group has fewer."""
    check_attention(Step8(dtype, [1] * 40, [300 + 40 * i for i in range(40)], 2 * hk, hk, d, seed=hk))


@pytest.mark.parametrize("n", [4095, 4096, 4097, 8192 + 65, 20000])
def test_page_numbers_are_found_again_and_again(dev, n):
    """Sequences past the blocks whose pages a wave finds at a time, in one workgroup and in several."""
    check_attention(Step8("bf16", [1, 1], [n, 100], 2, 1, 128, page_size=32, seed=n))
    check_attention(Step8("f32", [2], [n], 1, 1, 256, page_size=16, seed=n), workspace=0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n,hq,d", [(40000, 1, 64), (70001, 16, 128), (140000, 3, 64), (36000, 2, 256)])
def test_more_parts_than_a_join_takes_at_a_time(dev, dtype, n, hq, d):
    """One kv head, so that every workgroup has a part of the one unit: up to 512 of them."""
    check_attention(Step8(dtype, [1], [n], hq, 1, d, seed=hq))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_parts_with_and_without_scores(dev, dtype):
    """Windows that end inside parts: some of a unit's rows have nothing in its first ones."""
    check_attention(Step8(dtype, [5, 3], [30000, 9000], 6, 2, 64, window=4000, seed=44))
    check_attention(Step8(dtype, [4], [60000], 8, 1, 128, window=50001, seed=45))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q", [1, 40])
def test_infinite_scores_and_queries(dev, dtype, q):
    """Scores that overflow, and a cap that takes them back."""
    s = Step8(dtype, [q], [100], 2, 1, 64, seed=33, cap=0.0)
    s.scale = 3e38
    out, lse = s.run_attention()
    assert out.shape == (q, 2, 64)  # whatever they are, the call ends
    s.cap = 10.0
    out, lse = s.run_attention()
    assert np.isfinite(out).all() and np.isfinite(lse).all()


def laid_out(s, k_strides, v_strides, offsets):
    """The step's cache with rows at these (page, slot, head) strides, K's and V's in
    one buffer from these offsets on, and NaN between them."""
    size = max(o + (s.pages - 1) * st[0] + (s.page_size - 1) * st[1] + (s.hk - 1) * st[2] + s.d
               for o, st in zip(offsets, (k_strides, v_strides)))
    both = np.full(-(-size // 16) * 16, 0x7F, np.uint8)
    for o, st, codes in zip(offsets, (k_strides, v_strides), (s.k_codes, s.v_codes)):
        at = np.add.outer(np.add.outer(np.arange(s.pages) * st[0], np.arange(s.page_size) * st[1]), np.arange(s.hk) * st[2])
        both[o + at[..., None] + np.arange(s.d)] = codes
    data = kh.Buffer.from_array(both)
    scales = [kh.Buffer.from_array(np.ascontiguousarray(x.transpose(0, 2, 1))) for x in (s.k_scales, s.v_scales)]
    s.cache8_on_gpu = lambda: (kh.PagedCache8(
        k=data.ptr + offsets[0], v=data.ptr + offsets[1], k_scale=scales[0].ptr, v_scale=scales[1].ptr, k_page_stride=k_strides[0],
        k_slot_stride=k_strides[1], k_head_stride=k_strides[2], v_page_stride=v_strides[0], v_slot_stride=v_strides[1],
        v_head_stride=v_strides[2], scale_page_stride=s.hk * s.page_size, scale_head_stride=s.page_size, pages=s.pages,
        page_size=s.page_size, kv_heads=s.hk, head_dim=s.d), (data, scales))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["k and v in turn", "short heads first", "padded heads", "one head for all", "k by heads, v by slots"])
@pytest.mark.parametrize("q", [1, 40])
def test_heads_at_other_distances(dev, dtype, layout, q):
    """Heads of an entry that lie near each other, but not end to end."""
    hk, d = {"k and v in turn": (4, 64), "short heads first": (4, 16), "padded heads": (3, 64), "one head for all": (4, 64),
             "k by heads, v by slots": (2, 16)}[layout]
    s = Step8(dtype, [q] * 40, [500 + 11 * i for i in range(40)], 2 * hk, hk, d, page_size=16, seed=d + hk)
    ps = 16
    slots = (hk * ps * d, hk * d, d)
    k, v, offsets = slots, slots, (0, -(-s.pages * hk * ps * d // 16) * 16)
    if layout == "k and v in turn":
        k = v = (2 * hk * ps * d, 2 * hk * d, 2 * d)
        offsets = (0, d)
    elif layout == "short heads first":
        k = v = (hk * ps * d, d, ps * d)
    elif layout == "padded heads":
        k = v = (hk * ps * (d + 16), hk * (d + 16), d + 16)
        offsets = (0, s.pages * k[0])
    elif layout == "one head for all":
        k = v = (ps * d, d, 0)
        for name in "kv":
            codes, scales = getattr(s, name + "_codes"), getattr(s, name + "_scales")
            codes[:] = codes[:, :, :1]
            s.put(name, codes, scales)
        offsets = (0, s.pages * ps * d)
    else:
        k = (hk * ps * d, d, ps * d)
    laid_out(s, k, v, offsets)
    check_attention(s)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q,page_size", [(1, 16), (1, 7), (40, 16)])
def test_rows_of_v_of_any_size(dev, dtype, q, page_size):
    """Sequences whose rows of V are near the largest or the smallest that a row can be,
    each within a factor of 2^6."""
    lens = [900, 300, 70, 33]
    s = Step8(dtype, [q if q == 1 else min(q, n) for n in lens], lens, 4, 2, 64, page_size=page_size, seed=q + page_size)
    codes, scales = s.v_codes, s.v_scales
    codes[(codes & 0x7F) == 0x7F] = 0
    for i, byte in enumerate((230, 127, 40, 24)):
        pages = s.table[i][:-(-lens[i] // page_size)]
        scales[pages] = byte + s.g.integers(0, 6, scales[pages].shape)
    s.put("v", codes, scales)
    check_attention(s)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hk,d,rotary,interleaved", [(8, 128, 128, False), (8, 96, 48, True), (4, 256, 256, False), (8, 64, 64, True)])
def test_keys_are_rounded_once(dev, dtype, hk, d, rotary, interleaved):
    """Worked out in 64 bits: of more than a million numbers none goes to the other side of
    a tie, as some do in 32 bits."""
    say(f"keys {dtype} {hk} d={d} rotary={rotary}")
    g = np.random.default_rng(d)
    t, page_size = 1 << 20 >> int(math.log2(hk * d)), 16
    pages = t // page_size + 1
    q, k = (rounded(3 * g.standard_normal((t, h, d), np.float32), dtype) for h in (1, hk))
    gamma = rounded(1 + 0.2 * g.standard_normal(d).astype(np.float32), dtype)
    freq = (10000.0 ** (-np.arange(0, rotary, 2) / rotary)).astype(np.float32)
    pos, pair_axis = g.integers(0, 1000000, (3, t)), g.integers(0, 3, rotary // 2)
    slots = g.permutation(pages * page_size)[:t]
    out = run_write(dtype, np.repeat(q, hk, 1), k, k, (gamma, gamma), freq, pos, pair_axis, slots, pages, page_size, rotary, interleaved,
                    eps=0.0, k_out=True)
    want, _ = rotated(k, gamma, pos, freq, pair_axis, rotary, interleaved, 0.0, True, dtype)
    codes, scales = held(want)
    at = slots // page_size, slots % page_size
    assert np.array_equal(out[4][at[0], :, at[1]], scales)
    assert np.array_equal(out[2][at], codes)
    # k_out: half a step of its type, and what is left of 64 bits. An angle of up to 2^20
    # is 2^20 quarters, rounded to 2^-53 of them: 2^-32 rad; the series' rest is less.
    size = 2 * np.abs(want).max(-1, keepdims=True)
    close(out[1], want, np.abs(want) * half_step(dtype) + size * 2.0 ** -31 + (2.0 ** -25 if dtype == "f16" else 0.0), "k_out")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q", [1, 40])
@pytest.mark.parametrize("cap", [20.0, 200.0])
def test_small_scores_under_a_cap(dev, dtype, q, cap):
    """A row that sees one entry has its score for lse: exact before the cap (small whole
    numbers), and off by some 8 roundings of the series behind it, or where the
    other form takes over, at a quarter of the cap, by 2^-23 of the cap: 2^-20 of it."""
    s = Step8(dtype, [q] * 30, [q] * 30, 4, 2, 64, cap=cap, seed=q)
    whole = s.g.integers(-2, 3, s.k_codes.shape).astype(float)
    s.put("k", codes_of(whole), np.full(s.k_scales.shape, 127, np.uint8))
    s.q = s.g.integers(-2, 3, s.q.shape).astype(np.float32)
    s.scale = 0.125
    _, lse = s.run_attention()
    first = np.arange(30) * q  # these tokens see one entry
    k = whole[s.table[:, 0], 0]
    x = s.scale * (s.q.reshape(-1, 4, 64)[first] * np.repeat(k, 2, 1)).sum(-1)
    y = cap * np.tanh(x / cap)
    close(lse[first], y, np.abs(y) * 2.0 ** -20, "lse")


# ---------------------------------------------------------------- caches past 4 GB

FAR = 1 << 27  # from page to page


@pytest.mark.parametrize("page_size", [16, 24])
@pytest.mark.parametrize("pages,scales_far", [(36, False), (36, True), (20, True)])
def test_a_cache_past_4_gb(dev, page_size, pages, scales_far):
    """Pages 128 MB apart, their scales behind the rows or elsewhere: written, read
    and attended over, by every form."""
    say(f"far pages: {pages} of {page_size}, scales far: {scales_far}")
    hq, hk, d, t = 4, 2, 128, 40
    g = np.random.default_rng(pages)
    bufs = [kh.Buffer(pages * FAR) for _ in "kv"]
    near = [kh.Buffer.from_array(np.zeros((pages, hk, page_size), np.uint8)) for _ in "kv"]
    at = page_size * hk * d
    cache = kh.PagedCache8(k=bufs[0].ptr, v=bufs[1].ptr, k_scale=bufs[0].ptr + at if scales_far else near[0].ptr,
                           v_scale=bufs[1].ptr + at if scales_far else near[1].ptr, k_page_stride=FAR, k_slot_stride=hk * d,
                           k_head_stride=d, v_page_stride=FAR, v_slot_stride=hk * d, v_head_stride=d,
                           scale_page_stride=FAR if scales_far else hk * page_size, scale_head_stride=page_size, pages=pages,
                           page_size=page_size, kv_heads=hk, head_dim=d)
    table = np.stack((np.arange(pages)[::-1], np.roll(np.arange(pages), 3))).astype(np.int32)
    n = pages * page_size - 3
    # All the entries are written, those of sequence 0, as k and v of a few calls.
    slots = table[0][np.arange(n) // page_size].astype(np.int64) * page_size + np.arange(n) % page_size
    q, k, v = (rounded(g.standard_normal((n, h, d), np.float32), "bf16") for h in (hq, hk, hk))
    dq, dk, dv, dslots = (*(values_on_gpu(x, "bf16") for x in (q, k, v)), ints_on_gpu(slots, np.int64))
    dqo = values_on_gpu(np.zeros((n, hq, d)), "bf16")
    kh.synchronize()
    kh.qk_norm_rope8(kh.QkNormRope8(q=dq.ptr, k=dk.ptr, v=dv.ptr, q_out=dqo.ptr, slots=dslots.ptr, q_stride=hq * d, k_stride=hk * d,
                                    v_stride=hk * d, q_out_stride=hq * d, cache=cache, tokens=n, q_heads=hq, dtype=kh.BF16, eps=0.0))
    back = [values_on_gpu(np.zeros((n, hk, d)), "f32") for _ in "kv"]
    kh.paged_read8(kh.PagedRead8(cache=cache, slots=dslots.ptr, k_out=back[0].ptr, v_out=back[1].ptr, k_out_stride=hk * d,
                                 v_out_stride=hk * d, tokens=n, dtype=kh.F32))
    for b, x in zip(back, (k, v)):
        assert same_bits(values_from_gpu(b, (n, hk, d), "f32"), stand_for(*held(x)))
    for q_lens, shared in (([1, 1], 0), ([t, 1], 0), ([1, 100], 0)):
        s = Step8("bf16", q_lens, [1, 1], hq, hk, d, page_size=page_size, seed=t)
        s.pages, s.table, s.lens = pages, table, [n, n - 70]
        for name, x in (("k", k), ("v", v)):
            codes, scales = np.full((pages * page_size, hk, d), 0x7F, np.uint8), np.full((pages * page_size, hk), 127, np.uint8)
            codes[slots], scales[slots] = held(x)
            s.put(name, codes.reshape(pages, page_size, hk, d), scales.reshape(pages, page_size, hk))
        # Slots that nobody wrote hold what was there: no sequence has them.
        s.table[1][s.table[1] == table[0][-1]] = table[0][0]
        real = s.cache8_on_gpu
        s.cache8_on_gpu = lambda: (cache, None)
        check_attention(s)
        s.cache8_on_gpu = real
