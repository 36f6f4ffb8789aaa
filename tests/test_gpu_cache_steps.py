"""The sequence-cache operators one after another, as a server runs them: a
prompt and further tokens through norm, rotation and the write to the cache,
attention over it and the entries' weights, then eviction to another table and
further steps on that; eagerly, on streams of their own, and as captured graphs
that are replayed. Every stage is held to its definition in 64 bits with what
the stage before it left on the GPU."""
import ctypes
import math

import numpy as np
import pytest

import kernelh as kh
from cachetest import (DTYPES, Step, evict_reference, ints_on_gpu, rope_reference, rounded, same_bits, values_from_gpu,
                       values_on_gpu)
from khtest import say
from test_gpu_cache import check_attention, check_weights, close

pytestmark = pytest.mark.gpu

EPS = 1e-6


class Server:
    """Sequences over one cache; every launch goes to `stream`, none waits."""

    def __init__(self, dtype, seqs, hq, hk, d, page_size, window, width, seed=0, stream=None):
        self.g = np.random.default_rng(seed)
        self.dtype, self.seqs, self.hq, self.hk, self.d = dtype, seqs, hq, hk, d
        self.page_size, self.window, self.width, self.stream = page_size, window, width, stream
        self.pages = 2 * seqs * width + 1
        order = self.g.permutation(self.pages).astype(np.int32)
        self.table, self.kept_table = order[:2 * seqs * width].reshape(2, seqs, width)
        shape = (self.pages, page_size, hk, d)
        self.k, self.v = (values_on_gpu(np.full(shape, math.nan), dtype) for _ in "kv")
        st = (page_size * hk * d, hk * d, d)
        self.cache = kh.PagedCache(k=self.k.ptr, v=self.v.ptr, k_page_stride=st[0], k_slot_stride=st[1], k_head_stride=st[2],
                                   v_page_stride=st[0], v_slot_stride=st[1], v_head_stride=st[2], pages=self.pages,
                                   page_size=page_size, kv_heads=hk, head_dim=d, dtype=DTYPES[dtype])
        self.gamma = [rounded(1 + 0.3 * self.g.standard_normal(d, np.float32), dtype) for _ in "qk"]
        self.freq = (1e4 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
        self.dgamma, self.dfreq = [values_on_gpu(x, dtype) for x in self.gamma], values_on_gpu(self.freq, "f32")
        self.cap = width * page_size
        self.keep = []  # device memory of launches that may still run

    def new_weights(self):
        w = values_on_gpu(np.full((self.seqs, self.hk, self.cap), 7.0), "f32")
        self.keep.append(w)
        return w

    def page_table(self, table, lens):
        b = ints_on_gpu(table), ints_on_gpu(lens)
        self.keep.append(b)
        return kh.PageTable(pages=b[0].ptr, lens=b[1].ptr, row_stride=self.width, seqs=self.seqs, width=self.width, max_len=0)

    def prepare(self, table, lens, q_lens, positions, weights_in):
        """A step of q_lens new tokens that end at lens: what its launches take."""
        s = type("Prepared", (), {})()
        s.lens, s.q_lens, s.positions, s.hosttable = list(lens), list(q_lens), np.concatenate(positions), table
        tokens = s.tokens = sum(q_lens)
        s.starts = np.concatenate(([0], np.cumsum(q_lens)))
        hq, hk, d = self.hq, self.hk, self.d
        s.qkv = rounded(self.g.standard_normal((tokens, (hq + 2 * hk) * d), np.float32), self.dtype)
        entries = [np.arange(n - m, n) for n, m in zip(lens, q_lens)]
        s.slots = np.concatenate([table[i][e // self.page_size].astype(np.int64) * self.page_size + e % self.page_size
                                  for i, e in enumerate(entries)])
        s.dqkv, s.dpos, s.dslots = values_on_gpu(s.qkv, self.dtype), ints_on_gpu(s.positions, np.int64), ints_on_gpu(s.slots, np.int64)
        s.dstarts = ints_on_gpu(s.starts)
        s.dq, s.dout = (values_on_gpu(np.full((tokens, hq, d), 7.0), self.dtype) for _ in range(2))
        s.dlse = values_on_gpu(np.full((tokens, hq), 7.0), "f32")
        s.weights_in, s.dw = weights_in, self.new_weights()
        e = 4 if self.dtype == "f32" else 2
        at, pitch = [s.dqkv.ptr + x * d * e for x in (0, hq, hq + hk)], (hq + 2 * hk) * d
        pages = self.page_table(table, lens)
        s.rope = kh.QkNormRope(q=at[0], k=at[1], v=at[2], q_out=s.dq.ptr, k_out=None, q_gamma=self.dgamma[0].ptr,
                               k_gamma=self.dgamma[1].ptr, inv_freq=self.dfreq.ptr, positions=s.dpos.ptr, slots=s.dslots.ptr,
                               q_stride=pitch, k_stride=pitch, v_stride=pitch, q_out_stride=hq * d, k_out_stride=hk * d,
                               cache=self.cache, tokens=tokens, q_heads=hq, rotary_dim=d, interleaved=0, norm=1, eps=EPS)
        s.attention = kh.PagedAttention(cache=self.cache, table=pages, q=s.dq.ptr, out=s.dout.ptr, lse=s.dlse.ptr,
                                        q_starts=s.dstarts.ptr, q_stride=hq * d, out_stride=hq * d, tokens=tokens, q_heads=hq,
                                        window=self.window, scale=d ** -0.5)
        s.size = kh.paged_attention_workspace(s.attention)
        s.ws = kh.Buffer(max(16, s.size))
        s.weigh = kh.PagedWeights(cache=self.cache, table=pages, q=s.dq.ptr, lse=s.dlse.ptr, q_starts=s.dstarts.ptr,
                                  q_stride=hq * d, weights_in=weights_in.ptr if weights_in else None, weights=s.dw.ptr,
                                  weights_seq_stride=hk * self.cap, weights_head_stride=self.cap, tokens=tokens, q_heads=hq,
                                  window=self.window, scale=d ** -0.5)
        return s

    def run(self, s):
        kh.qk_norm_rope(s.rope, self.stream)
        kh.paged_attention(s.attention, s.ws if s.size else None, s.size, self.stream)
        kh.paged_weights(s.weigh, self.stream)

    def prepare_eviction(self, lens, weights, budget, recent):
        e = type("Eviction", (), {})()
        e.lens, e.weights_in, e.budget, e.recent = list(lens), weights, budget, recent
        e.dw, e.dlens, e.dkt = self.new_weights(), ints_on_gpu(np.full(self.seqs, -7)), ints_on_gpu(self.kept_table)
        st = self.hk * self.cap
        e.args = kh.PagedEvict(cache=self.cache, table=self.page_table(self.table, lens), kept_pages=e.dkt.ptr,
                               kept_row_stride=self.width, kept_width=self.width, kept_lens=e.dlens.ptr, weights_in=weights.ptr,
                               in_seq_stride=st, in_head_stride=self.cap, weights=e.dw.ptr, seq_stride=st, head_stride=self.cap,
                               budget=budget, recent=recent)
        e.size = kh.paged_evict_workspace(e.args)
        e.ws = kh.Buffer(e.size)
        return e

    def evict(self, e):
        kh.paged_evict(e.args, e.ws, e.size, self.stream)

    # -- what lies on the GPU after the launches, held to the definitions

    def check(self, s, what):
        """Entries are only ever added, so the cache as it is now holds what this step saw."""
        hq, hk, d = self.hq, self.hk, self.d
        shape = (self.pages, self.page_size, hk, d)
        k, v = (values_from_gpu(x, shape, self.dtype) for x in (self.k, self.v))
        q = values_from_gpu(s.dq, (s.tokens, hq, d), self.dtype)
        parts = [s.qkv[:, a * d:b * d].reshape(s.tokens, b - a, d) for a, b in ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk))]
        rope = [rope_reference(x, g, s.positions, self.freq, d, 0, EPS, 1, self.dtype) for x, g in zip(parts, self.gamma)]
        close(q, *rope[0], f"{what}: q")
        close(k.reshape(-1, hk, d)[s.slots], *rope[1], f"{what}: k in the cache")
        assert same_bits(v.reshape(-1, hk, d)[s.slots], parts[2])
        r = Step(self.dtype, s.q_lens, s.lens, hq, hk, d, page_size=self.page_size, window=self.window)
        r.pages, r.table, r.k, r.v, r.q, r.q_pitch = self.pages, s.hosttable, k, v, q.reshape(s.tokens, hq * d), hq * d
        want, bound, y, y_bound = r.attention()
        out, lse = values_from_gpu(s.dout, (s.tokens, hq, d), self.dtype), values_from_gpu(s.dlse, (s.tokens, hq), "f32")
        close(out, want, bound, f"{what}: out")
        close(lse, y, y_bound, f"{what}: lse")
        wshape = (self.seqs, hk, self.cap)
        before = values_from_gpu(s.weights_in, wshape, "f32") if s.weights_in else np.zeros(wshape, np.float32)
        w, w_bound = r.weights(lse, before)
        got = values_from_gpu(s.dw, wshape, "f32")
        for i, n in enumerate(s.lens):
            close(got[i, :, :n], w[i, :, :n], w_bound[i, :, :n], f"{what}: weights")

    def check_eviction(self, e):
        shape, wshape = (self.pages, self.page_size, self.hk, self.d), (self.seqs, self.hk, self.cap)
        cache = [values_from_gpu(x, shape, self.dtype) for x in (self.k, self.v)]
        w, got = values_from_gpu(e.weights_in, wshape, "f32"), values_from_gpu(e.dw, wshape, "f32")
        assert e.dlens.to_host(np.int32).tolist() == [min(n, e.budget) for n in e.lens]
        for i, n in enumerate(e.lens):
            for h in range(self.hk):
                ids = np.array(evict_reference(w[i, h], n, e.budget, e.recent))
                to = np.arange(len(ids))
                assert same_bits(got[i, h, :len(ids)], w[i, h, ids])
                for x in cache:
                    assert same_bits(x[self.kept_table[i][to // self.page_size], to % self.page_size, h],
                                     x[self.table[i][ids // self.page_size], ids % self.page_size, h])


def program(dtype, hq, hk, d, page_size, window, stream=None, seed=0):
    """A prompt, two steps, an eviction and two steps after it, prepared."""
    lens = np.array([70, 9, 131])
    sv = Server(dtype, 3, hq, hk, d, page_size, window, -(-160 // page_size), seed, stream)
    steps = [sv.prepare(sv.table, lens, lens, [np.arange(n) for n in lens], None)]
    for _ in range(2):
        lens = lens + 1
        steps.append(sv.prepare(sv.table, lens, [1, 1, 1], [[n - 1] for n in lens], steps[-1].dw))
    ev = sv.prepare_eviction(lens, steps[-1].dw, 48, 16)
    kept, w = np.minimum(lens, 48), ev.dw
    after = []
    for i in range(2):
        kept = kept + 1
        after.append(sv.prepare(sv.kept_table, kept, [1, 1, 1], [[n + i] for n in lens], w))
        w = after[-1].dw
    return sv, steps, ev, after


def launch(sv, steps, ev, after):
    for s in steps:
        sv.run(s)
    sv.evict(ev)
    for s in after:
        sv.run(s)


def check(sv, steps, ev, after):
    for i, s in enumerate(steps):
        sv.check(s, f"step {i}")
    sv.check_eviction(ev)
    for i, s in enumerate(after):
        sv.check(s, f"step {i} after eviction")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hk,d,page_size,window", [(8, 2, 64, 16, 0), (4, 4, 128, 24, 0), (6, 1, 80, 16, 40)])
def test_steps_of_a_server(dev, dtype, hq, hk, d, page_size, window):
    say(f"server {dtype} {hq}/{hk} d={d} page={page_size} window={window}")
    p = program(dtype, hq, hk, d, page_size, window)
    launch(*p)
    check(*p)


def test_two_servers_on_two_streams(dev):
    """Launches of two programs alternate over two streams and share nothing."""
    say("two servers")
    streams = kh.Stream(), kh.Stream()
    programs = [program(t, 8, 2, 64, 16, 0, st, seed) for seed, (t, st) in enumerate(zip(("bf16", "f32"), streams))]
    kh.synchronize()
    for i in range(3):
        for p in programs:
            p[0].run(p[1][i])
    for p in programs:
        p[0].evict(p[2])
    for i in range(2):
        for p in programs:
            p[0].run(p[3][i])
    for st in streams:
        st.synchronize()
    for p in programs:
        check(*p)
    for st in streams:
        st.destroy()


class Graph:
    """Launches on a stream, captured, by the HIP runtime that this process has loaded."""

    def __init__(self, stream, launches):
        with open("/proc/self/maps", encoding="ascii") as f:
            path = next(line.split()[-1] for line in f if "libamdhip64" in line)
        self.hip, self.stream = ctypes.CDLL(path), stream
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        self.check(self.hip.hipStreamBeginCapture(ctypes.c_void_p(stream.ptr), 0))
        try:
            launches()
        finally:
            rc = self.hip.hipStreamEndCapture(ctypes.c_void_p(stream.ptr), ctypes.byref(graph))
        self.check(rc)
        self.check(self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)))
        self.check(self.hip.hipGraphDestroy(graph))

    def check(self, rc):
        assert rc == 0, f"HIP error {rc}"

    def replay(self):
        self.check(self.hip.hipGraphLaunch(self.exec, ctypes.c_void_p(self.stream.ptr)))

    def destroy(self):
        self.check(self.hip.hipGraphExecDestroy(self.exec))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_captured_steps_replay_as_they_ran(dev, dtype):
    """Two programs captured, each with its workspaces, and replayed in turn
    with eager launches and copies between them: every replay gives the bits of
    the eager run, from buffers that were cleared before it."""
    say(f"captured {dtype}")
    stream = kh.Stream()
    programs = [program(dtype, 8, 2, 64, 16, 0, stream, seed) for seed in (5, 6)]
    sv, steps, ev, after = programs[0]

    def results(p):
        sv, steps, ev, after = p
        stream.synchronize()
        t = np.int32
        return [b.to_host(t) for s in steps + after for b in (s.dq, s.dout, s.dlse, s.dw)] + [
            b.to_host(t) for b in (ev.dw, ev.dlens, sv.k, sv.v)]

    def clear(p):
        sv, steps, ev, after = p
        for b in [x for s in steps + after for x in (s.dq, s.dout, s.dlse, s.dw, s.ws)] + [ev.dw, ev.ws, sv.k, sv.v]:
            b.fill(7.0, stream)
        stream.synchronize()

    want = []
    for p in programs:
        clear(p)
        launch(*p)
        want.append(results(p))
    graphs = []
    for p in programs:
        graphs.append(Graph(stream, lambda: launch(*p)))
    for turn in range(4):
        for p, g, w in zip(programs, graphs, want):
            clear(p)
            g.replay()
            got = results(p)
            assert all(np.array_equal(a, b) for a, b in zip(got, w)), f"replay {turn}"
            eager = Step("f16", [1, 40], [90 + turn, 40], 4, 2, 64, seed=turn)
            check_attention(eager, "between replays", stream=stream)
            launch(*p)
            assert all(np.array_equal(a, b) for a, b in zip(results(p), w)), f"eager after replay {turn}"
    for g in graphs:
        g.destroy()
    stream.destroy()


# ---------------------------------------------------------------- further forms

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
@pytest.mark.parametrize("q", [1, 40])
def test_scales(dev, dtype, scale, q):
    s = Step(dtype, [q, 1], [100, 60], 4, 2, 64, seed=21)
    s.scale = scale
    check_attention(s)
    check_weights(s)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,q_lens", [(20, [1, 1]), (64, [1, 2]), (40, [3, 1]), (17, [1, 30])])
@pytest.mark.parametrize("page_size", [16, 24, 512])
def test_many_heads_to_a_kv_head(dev, dtype, hq, q_lens, page_size):
    s = Step(dtype, q_lens, [200, 700], hq, 1, 64, page_size=page_size, seed=hq)
    check_attention(s)
    check_weights(s)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [1, 9, 50]])
def test_weights_over_pages_of_heads(dev, dtype, q_lens):
    """[pages, heads, slots, head_dim], padded queries, another stream."""
    for d in (64, 128, 96):
        s = Step(dtype, q_lens, [300, 9, 77], 8, 2, d, heads_first=True, pad=24, seed=d)
        y = s.attention()[2].astype(np.float32)
        before = s.g.random((3, 2, 320), np.float32)
        st = kh.Stream()
        kh.synchronize()
        got = s.run_weights(y, before, stream=st)
        st.destroy()
        want, bound = s.weights(y, before)
        for i, n in enumerate(s.lens):
            close(got[i, :, :n], want[i, :, :n], bound[i, :, :n], f"sequence {i}")


def test_a_length_past_the_hint(dev):
    """max_len sizes the launch; sequences longer than it are done all the same."""
    for q in (1, 40):
        s = Step("bf16", [q, 1], [1500, 900], 4, 2, 64, seed=31)
        _, lse = check_attention(s, max_len=20)
        before = s.g.random((2, 2, 1500), np.float32)
        want, bound = s.weights(lse, before)
        got = s.run_weights(lse, before, max_len=20)
        for i, n in enumerate(s.lens):
            close(got[i, :, :n], want[i, :, :n], bound[i, :, :n], f"sequence {i}")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq", [8, 6])
def test_tokens_that_share_their_queries(dev, dtype, hq):
    """q_stride 0: one row of q is every token's."""
    s = Step(dtype, [70, 1], [200, 90], hq, 2, 64, seed=32)
    s.q, s.q_pitch = np.repeat(s.q[:1], s.tokens, 0), 0
    check_attention(s)
    check_weights(s)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [128, 511, 512, 513, 641, 3500])
def test_few_units_of_many_blocks(dev, dtype, n):
    """One or two heads' rows over several workgroups, or whole in one."""
    check_attention(Step(dtype, [1], [n], 1, 1, 80, page_size=24, seed=n))
    check_attention(Step(dtype, [11, 3], [n, 600], 1, 1, 64, seed=n))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("window", [0, 90])
def test_row_counts_on_both_sides_of_the_forms(dev, dtype, window):
    """Sequences of 16 to 132 rows in one batch, and one alone."""
    check_attention(Step(dtype, [4, 8, 9, 16, 17, 33], [300, 40, 700, 1500, 64, 128], 8, 2, 64, window=window, seed=41))
    for q in (15, 16, 17, 33):
        check_attention(Step(dtype, [q], [900], 4, 1, 128, page_size=24, window=window, seed=q))
