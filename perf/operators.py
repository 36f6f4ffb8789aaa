"""The calls the sequence-cache operators are timed at, and their plain forms.

A serving step of a decoder writes the keys and values of its new tokens to a
paged cache (qk_norm_rope), attends over that cache (paged_attention), sums the
attention that each cached entry received (paged_weights) and, now and then,
keeps only the entries that received most (paged_evict).

The plain forms are elementary torch operations on the whole padded batch, in
32 bits (rotation angles in 64), rounded once at the end. Lengths are part of a
case; values, page orders and positions come from the seed.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _kh():
    path = os.path.join(os.getcwd(), "kernel.h_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kernelh

    return kernelh


def listed():
    return [
        # A decoding step of a small batch, heads as the attention benchmark
        # has them: one launch of a few workgroups, where latency counts.
        {"name": "rope_f32_5x16", "op": "qk_norm_rope", "dtype": "f32", "tokens": 5, "q_heads": 16, "kv_heads": 16,
         "head_dim": 64, "rotary": 64, "interleaved": False, "page_size": 16, "far": 4096},
        # A prompt's chunk of a grouped-query model: bound by memory.
        {"name": "rope_bf16_8192", "op": "qk_norm_rope", "dtype": "bf16", "tokens": 8192, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "rotary": 128, "interleaved": False, "page_size": 16, "far": 131072},
        # Half of each head rotated in neighbouring pairs, a ragged token
        # count, positions past a million.
        {"name": "rope_f16_1999", "op": "qk_norm_rope", "dtype": "f16", "tokens": 1999, "q_heads": 24, "kv_heads": 24,
         "head_dim": 96, "rotary": 48, "interleaved": True, "page_size": 32, "far": 2000000},
        # One new token for each of four sequences (the attention benchmark's
        # batch, heads and shorter length).
        {"name": "decode_f32_b4_1024", "op": "paged_attention", "dtype": "f32", "seqs": 4, "q_min": 1, "q_max": 1,
         "len_min": 1024, "len_max": 1024, "q_heads": 16, "kv_heads": 16, "head_dim": 64, "window": 0,
         "page_size": 16},
        # A serving batch in the middle of its answers: lengths all over.
        {"name": "decode_bf16_64_ragged", "op": "paged_attention", "dtype": "bf16", "seqs": 64, "q_min": 1, "q_max": 1,
         "len_min": 513, "len_max": 8192, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0,
         "page_size": 16},
        # One very long sequence: few rows, so its length is what fills the chip.
        {"name": "decode_bf16_131071", "op": "paged_attention", "dtype": "bf16", "seqs": 1, "q_min": 1, "q_max": 1,
         "len_min": 131071, "len_max": 131071, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0,
         "page_size": 64},
        # A chunk of a long prompt over what is cached of it: bound by the
        # matrix units.
        {"name": "chunk_bf16_2048of8192", "op": "paged_attention", "dtype": "bf16", "seqs": 1, "q_min": 2048,
         "q_max": 2048, "len_min": 8192, "len_max": 8192, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0,
         "page_size": 16},
        # Chunks and single tokens in one batch, a sliding window, heads of no
        # power of two, pages that end inside every tile.
        {"name": "mixed_f16_window", "op": "paged_attention", "dtype": "f16", "seqs": 16, "q_min": 1, "q_max": 301,
         "len_min": 400, "len_max": 4001, "q_heads": 12, "kv_heads": 4, "head_dim": 80, "window": 1000,
         "page_size": 24},
        # What one decoding step adds to the entries' weights.
        {"name": "weights_bf16_decode", "op": "paged_weights", "dtype": "bf16", "seqs": 32, "q_min": 1, "q_max": 1,
         "len_min": 1025, "len_max": 8192, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0,
         "page_size": 16},
        # What a prompt's chunk adds.
        {"name": "weights_bf16_chunk", "op": "paged_weights", "dtype": "bf16", "seqs": 2, "q_min": 777, "q_max": 1024,
         "len_min": 4097, "len_max": 6000, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0,
         "page_size": 16},
        # A small cache back to its budget.
        {"name": "evict_f32_3x1031", "op": "paged_evict", "dtype": "f32", "seqs": 3, "len_min": 777, "len_max": 1031,
         "kv_heads": 16, "head_dim": 64, "budget": 777, "recent": 64, "page_size": 16},
        # A batch whose caches have grown a few pages past their budget.
        {"name": "evict_bf16_16x4352", "op": "paged_evict", "dtype": "bf16", "seqs": 16, "len_min": 4200,
         "len_max": 4352, "kv_heads": 8, "head_dim": 128, "budget": 4096, "recent": 256, "page_size": 16},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "paged_attention", "paged_attention", "paged_weights", "paged_evict"])
    d = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    case = {"op": op, "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "head_dim": d}
    kv, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 7, 8])
    case |= {"kv_heads": kv, "page_size": rng.choice([1, 7, 16, 16, 24, 32, 64, 100, 256])}
    if op == "qk_norm_rope":
        return case | {"tokens": _spread(rng, 1, 8192), "q_heads": kv * group, "rotary": rng.choice([d, d, d // 16 * 8]),
                       "interleaved": rng.random() < 0.4, "far": _spread(rng, 1000, 2000000)}
    if op == "paged_evict":
        top = _spread(rng, 2, 16384)
        low = rng.randint(1, top)
        budget = rng.randint(1, top)
        seqs = _spread(rng, 1, max(1, min(64, (1 << 28) // (top * kv * d))))
        return case | {"seqs": seqs, "len_min": low, "len_max": top, "budget": budget, "recent": rng.randint(0, budget)}
    case |= {"q_heads": kv * group, "window": rng.choice([0, 0, 0, _spread(rng, 1, 4096)])}
    if rng.random() < 0.5:  # decoding, a token or a few proposed ones
        q_max = rng.choice([1, 1, 1, 2, 5])
        top = _spread(rng, q_max, 65536)
        seqs = _spread(rng, 1, max(1, min(128, (1 << 28) // (top * kv * d))))
    else:  # chunks
        q_max = _spread(rng, 2, 2048)
        top = _spread(rng, q_max, 16384)
        while q_max * top * kv * group > 1 << 28:
            q_max, top = max(2, q_max // 2), max(2, q_max // 2, top // 2)
        seqs = _spread(rng, 1, max(1, min(16, (1 << 28) // (q_max * top * kv * group), (1 << 28) // (top * kv * d))))
    return case | {"seqs": seqs, "q_min": 1 if rng.random() < 0.5 else q_max, "q_max": q_max,
                   "len_min": rng.randint(q_max, top), "len_max": top}


def _between(lo, hi, n, step):
    """n whole numbers spread evenly, in no order, from lo to hi; the first is hi."""
    return [hi - int((i * step) % 1.0 * (hi - lo + 1)) for i in range(n)]


def _lengths(case):
    """(new tokens, entries in the cache with them) of each sequence."""
    lens = _between(case["len_min"], case["len_max"], case["seqs"], 0.6180339887498949)
    if "q_max" not in case:
        return [0] * len(lens), lens
    return _between(case["q_min"], case["q_max"], case["seqs"], 0.7548776662466927), lens


def _visible(case, q, n):
    """Entries that the q new tokens of a sequence of n see, summed over them."""
    w = case["window"] or n
    return sum(min(n - q + i + 1, w) for i in range(q))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _cache_pages(g, case, widths, spare):
    """A cache in some order of its pages, and a table of `widths` pages each."""
    need = sum(widths)
    pages = need + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(widths), max(widths)), dtype=torch.int32, device="cuda")
    at = 0
    for s, w in enumerate(widths):
        table[s, :w] = order[at:at + w]
        at += w
    shape = (pages, case["page_size"], case["kv_heads"], case["head_dim"])
    dtype = _DTYPES[case["dtype"]]
    return table, order[at:], _normal(g, shape, dtype), _normal(g, shape, dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    dtype, d, ps = _DTYPES[case["dtype"]], case["head_dim"], case["page_size"]
    if case["op"] == "qk_norm_rope":
        t, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
        # q, k and v are parts of one projection's output.
        qkv = _normal(g, (t, hq + 2 * hk, d), dtype) * 2
        pages = -(-t // ps) + 3
        shape = (pages, ps, hk, d)
        r = case["rotary"]
        return {"case": case, "q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "v": qkv[:, hq + hk:],
                "q_gamma": (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype),
                "k_gamma": (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype),
                "inv_freq": (10000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)).float(),
                "positions": torch.randint(0, case["far"], (t,), generator=g, device="cuda"),
                "slots": torch.randperm(pages * ps, generator=g, device="cuda")[:t],
                "q_out": torch.zeros((t, hq, d), dtype=dtype, device="cuda"),
                "k_cache": torch.zeros(shape, dtype=dtype, device="cuda"),
                "v_cache": torch.zeros(shape, dtype=dtype, device="cuda")}
    q_lens, lens = _lengths(case)
    s = {"case": case, "lens": _ints(lens)}
    widths = [-(-n // ps) for n in lens]
    if case["op"] == "paged_evict":
        kept = -(-case["budget"] // ps)
        s["table"], rest, s["k"], s["v"] = _cache_pages(g, case, widths, kept * len(lens))
        s["kept_table"] = rest.view(len(lens), kept).contiguous()
        # Sums of attention: a few large, most small, some none at all.
        w = torch.exp(2 * torch.randn((len(lens), case["kv_heads"], max(lens)), generator=g, device="cuda"))
        s["weights_in"] = w * (torch.rand(w.shape, generator=g, device="cuda") > 0.1)
        cap = kept * ps
        s["weights"] = torch.zeros((len(lens), case["kv_heads"], cap), device="cuda")
        s["kept_lens"] = torch.zeros_like(s["lens"])
        # Which entries are kept is worked out on the way: room for their numbers.
        s["workspace"] = torch.empty(len(lens) * case["kv_heads"] * (case["budget"] + 64) * 4, dtype=torch.uint8,
                                     device="cuda")
        return s
    s["table"], _, s["k"], s["v"] = _cache_pages(g, case, widths, 1)
    starts = [sum(q_lens[:i]) for i in range(len(q_lens) + 1)]
    t, hq = starts[-1], case["q_heads"]
    s["q"] = _normal(g, (t, hq, d), dtype)
    s["q_starts"] = _ints(starts)
    s["token_seq"] = _ints([i for i, q in enumerate(q_lens) for _ in range(q)], torch.int64)
    s["token_at"] = _ints([j for q in q_lens for j in range(q)], torch.int64)
    s["q_most"], s["len_most"] = max(q_lens), max(lens)
    if case["op"] == "paged_attention":
        s["out"] = torch.zeros((t, hq, d), dtype=dtype, device="cuda")
        s["lse"] = torch.zeros((t, hq), device="cuda")
        s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
        return s
    # About what scores of unit spread come to.
    seen = _ints([n - q + j + 1 for q, n in zip(q_lens, lens) for j in range(q)], torch.float32)
    seen = torch.clamp(seen, max=float(case["window"] or max(lens)))
    s["lse"] = seen.log()[:, None] + 0.5 + 0.1 * torch.randn((t, hq), generator=g, device="cuda")
    s["weights_in"] = torch.rand((len(lens), case["kv_heads"], max(lens)), generator=g, device="cuda")
    s["weights"] = torch.zeros_like(s["weights_in"])
    return s


# ---------------------------------------------------------------- the framework's calls


def _struct_cache(kh, case, k, v):
    return kh.PagedCache(k=k.data_ptr(), v=v.data_ptr(), k_page_stride=k.stride(0), k_slot_stride=k.stride(1),
                         k_head_stride=k.stride(2), v_page_stride=v.stride(0), v_slot_stride=v.stride(1),
                         v_head_stride=v.stride(2), pages=k.shape[0], page_size=case["page_size"],
                         kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                         dtype=getattr(kh, case["dtype"].upper()))


def _struct_table(kh, s):
    t = s["table"]
    return kh.PageTable(pages=t.data_ptr(), lens=s["lens"].data_ptr(), row_stride=t.stride(0), seqs=t.shape[0],
                        width=t.shape[1], max_len=s.get("len_most", 0))


def _own_rope(s):
    kh, c = _kh(), s["case"]
    kh.qk_norm_rope(kh.QkNormRope(
        q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), q_stride=s["q"].stride(0),
        k_stride=s["k"].stride(0), v_stride=s["v"].stride(0), q_out=s["q_out"].data_ptr(),
        q_out_stride=s["q_out"].stride(0), q_gamma=s["q_gamma"].data_ptr(), k_gamma=s["k_gamma"].data_ptr(),
        inv_freq=s["inv_freq"].data_ptr(), positions=s["positions"].data_ptr(), slots=s["slots"].data_ptr(),
        cache=_struct_cache(kh, c, s["k_cache"], s["v_cache"]), tokens=c["tokens"], q_heads=c["q_heads"],
        rotary_dim=c["rotary"], interleaved=c["interleaved"], norm=1, eps=1e-6))
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attention(s):
    kh, c = _kh(), s["case"]
    kh.paged_attention(kh.PagedAttention(
        cache=_struct_cache(kh, c, s["k"], s["v"]), table=_struct_table(kh, s), q=s["q"].data_ptr(),
        q_stride=s["q"].stride(0), out=s["out"].data_ptr(), out_stride=s["out"].stride(0), lse=s["lse"].data_ptr(),
        q_starts=s["q_starts"].data_ptr(), tokens=s["q"].shape[0], q_heads=c["q_heads"], window=c["window"],
        scale=c["head_dim"] ** -0.5), s["workspace"].data_ptr(), s["workspace"].numel())
    return {"out": s["out"], "lse": s["lse"]}


def _own_weights(s):
    kh, c, w = _kh(), s["case"], s["weights"]
    kh.paged_weights(kh.PagedWeights(
        cache=_struct_cache(kh, c, s["k"], s["v"]), table=_struct_table(kh, s), q=s["q"].data_ptr(),
        q_stride=s["q"].stride(0), lse=s["lse"].data_ptr(), q_starts=s["q_starts"].data_ptr(),
        tokens=s["q"].shape[0], q_heads=c["q_heads"], window=c["window"], scale=c["head_dim"] ** -0.5,
        weights_in=s["weights_in"].data_ptr(), weights=w.data_ptr(), weights_seq_stride=w.stride(0),
        weights_head_stride=w.stride(1)))
    return {"weights": w}


def _own_evict(s):
    kh, c, a, b = _kh(), s["case"], s["weights_in"], s["weights"]
    kh.paged_evict(kh.PagedEvict(
        cache=_struct_cache(kh, c, s["k"], s["v"]), table=_struct_table(kh, s), kept_pages=s["kept_table"].data_ptr(),
        kept_row_stride=s["kept_table"].stride(0), kept_width=s["kept_table"].shape[1],
        kept_lens=s["kept_lens"].data_ptr(), weights_in=a.data_ptr(), in_seq_stride=a.stride(0),
        in_head_stride=a.stride(1), weights=b.data_ptr(), seq_stride=b.stride(0), head_stride=b.stride(1),
        budget=c["budget"], recent=c["recent"]), s["workspace"].data_ptr(), s["workspace"].numel())
    return {"k": s["k"], "v": s["v"], "weights": b, "lens": s["kept_lens"]}


# ---------------------------------------------------------------- the plain forms


def _plain_normed(x, gamma):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gamma.float()


def _plain_rotated(x, cos, sin, rotary, interleaved):
    half, rest = rotary // 2, x[..., rotary:]
    a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :half], x[..., half:rotary])
    y, z = a * cos - b * sin, b * cos + a * sin
    both = torch.stack((y, z), -1).flatten(-2) if interleaved else torch.cat((y, z), -1)
    return torch.cat((both, rest), -1)


def _plain_rope(s):
    c, dtype = s["case"], s["q"].dtype
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    q, k = (_plain_rotated(_plain_normed(s[n], s[n + "_gamma"]), cos, sin, c["rotary"], c["interleaved"])
            for n in ("q", "k"))
    s["k_cache"].view(-1, c["kv_heads"], c["head_dim"])[s["slots"]] = k.to(dtype)
    s["v_cache"].view(-1, c["kv_heads"], c["head_dim"])[s["slots"]] = s["v"]
    return {"q": q.to(dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _rows_of(table, ps, n):
    """The cache row that holds entry j of each sequence: [sequences, n]."""
    j = torch.arange(n, device="cuda")
    return table.long()[:, j // ps] * ps + j % ps


def _plain_scores(s):
    """Scores of every head's new tokens, padded, [sequences, kv heads, heads of a group, new tokens, entries]; -inf where not seen."""
    c = s["case"]
    hk, d, n, m = c["kv_heads"], c["head_dim"], s["len_most"], s["q_most"]
    group, seqs = c["q_heads"] // hk, c["seqs"]
    rows = _rows_of(s["table"], c["page_size"], n)
    k = s["k"].view(-1, hk, d)[rows].float().permute(0, 2, 3, 1).contiguous()
    i, j = torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
    q_lens = (s["q_starts"][1:] - s["q_starts"][:-1]).long()
    token = torch.clamp(s["q_starts"][:-1].long()[:, None] + i, max=s["q"].shape[0] - 1)
    q = s["q"][token].float().view(seqs, m, hk, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hk, group * m, d)
    x = (torch.matmul(q, k) * d ** -0.5).view(seqs, hk, group, m, n)
    at = s["lens"].long()[:, None] - q_lens[:, None] + i
    seen = (j <= at[..., None]) & (i < q_lens[:, None])[..., None]
    if c["window"]:
        seen = seen & (j > at[..., None] - c["window"])
    return x.masked_fill(~seen[:, None, None], -math.inf), rows, token


def _plain_attention(s):
    c = s["case"]
    hk, d, n, m = c["kv_heads"], c["head_dim"], s["len_most"], s["q_most"]
    x, rows, _ = _plain_scores(s)
    top = torch.clamp(x.amax(-1, keepdim=True), min=-1e30)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    v = s["v"].view(-1, hk, d)[rows].float().permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p.view(c["seqs"], hk, -1, n), v).view(c["seqs"], hk, -1, m, d) / torch.clamp(total, min=1e-30)
    lse = (top + torch.log(total))[..., 0]
    o, lse = (t[s["token_seq"], :, :, s["token_at"]] for t in (o, lse))
    return {"out": o.reshape(-1, c["q_heads"], d).to(s["q"].dtype), "lse": lse.reshape(-1, c["q_heads"])}


def _plain_weights(s):
    c = s["case"]
    x, _, token = _plain_scores(s)
    lse = s["lse"][token].view(c["seqs"], s["q_most"], c["kv_heads"], -1).permute(0, 2, 3, 1)
    total = torch.exp(x - lse[..., None]).sum((2, 3))
    q_lens = (s["q_starts"][1:] - s["q_starts"][:-1]).long()
    j = torch.arange(s["len_most"], device="cuda")
    old = j < (s["lens"].long() - q_lens)[:, None]
    inside = (j < s["lens"].long()[:, None])[:, None]
    s["weights"].copy_(torch.where(inside, torch.where(old[:, None], s["weights_in"], 0) + total, 0))
    return {"weights": s["weights"]}


def _plain_evict(s):
    c = s["case"]
    hk, d, ps, budget, recent = c["kv_heads"], c["head_dim"], c["page_size"], c["budget"], c["recent"]
    n = s["weights_in"].shape[2]
    j = torch.arange(n, device="cuda")
    lens = s["lens"].long()[:, None, None]
    # The newest rank before all else, what lies past the end after it.
    rank = torch.where(j >= lens - recent, math.inf, s["weights_in"])
    rank = torch.where(j < lens, rank, -1.0)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept_lens = torch.clamp(s["lens"].long(), max=budget)
    at = torch.arange(kept.shape[-1], device="cuda")
    kept = torch.where(at < kept_lens[:, None, None], kept, n)
    kept = torch.sort(kept, dim=-1).values
    real = (kept < n).nonzero(as_tuple=True)
    seq, head, to = real
    entry = kept[real]
    table, kept_table = s["table"].long(), s["kept_table"].long()
    src = table[seq, entry // ps] * ps + entry % ps
    dst = kept_table[seq, to // ps] * ps + to % ps
    for name in ("k", "v"):
        rows = s[name].view(-1, hk, d)
        rows[dst, head] = rows[src, head]
    s["weights"][seq, head, to] = s["weights_in"][seq, head, entry]
    s["kept_lens"].copy_(kept_lens)
    return {"k": s["k"], "v": s["v"], "weights": s["weights"], "lens": s["kept_lens"]}


_PLAIN = {"qk_norm_rope": _plain_rope, "paged_attention": _plain_attention, "paged_weights": _plain_weights,
          "paged_evict": _plain_evict}
_OWN = {"qk_norm_rope": _own_rope, "paged_attention": _own_attention, "paged_weights": _own_weights,
        "paged_evict": _own_evict}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def work(case):
    e, d, hk = _BYTES[case["dtype"]], case["head_dim"], case["kv_heads"]
    if case["op"] == "qk_norm_rope":
        t, heads = case["tokens"], case["q_heads"] + hk
        # q and k read and written, v copied; angles, positions and slots once.
        return {"bytes": t * (2 * (heads + hk) * d * e + 16) + 2 * d * e + 2 * case["rotary"],
                "flops": t * heads * (4 * d + 3 * case["rotary"])}
    q_lens, lens = _lengths(case)
    if case["op"] == "paged_evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": hk * (4 * kept * d * e + 4 * sum(lens) + 4 * kept), "flops": hk * sum(lens)}
    hq, t = case["q_heads"], sum(q_lens)
    seen = sum(_visible(case, q, n) for q, n in zip(q_lens, lens))
    # Entries that some new token sees; with a window the oldest are not read.
    read = sum(min(n, (case["window"] or n) + q - 1) for q, n in zip(q_lens, lens))
    if case["op"] == "paged_weights":
        return {"bytes": hk * read * d * e + t * hq * (d * e + 4) + 8 * hk * sum(lens), "flops": hq * seen * (2 * d + 3)}
    return {"bytes": 2 * hk * read * d * e + t * hq * (2 * d * e + 4), "flops": hq * seen * (4 * d + 4)}


# ---------------------------------------------------------------- from the definitions, in 64 bits


def _exact_rope(s):
    c = s["case"]
    r, half = c["rotary"], c["rotary"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double().outer(s["inv_freq"].double()))[:, None]
    out = {}
    for n in ("q", "k"):
        x = s[n].double()
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * s[n + "_gamma"].double()
        re, im = (x[..., :r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :half], x[..., half:r])
        z = torch.complex(re, im) * turn
        y = x.clone()
        if c["interleaved"]:
            y[..., :r:2], y[..., 1:r:2] = z.real, z.imag
        else:
            y[..., :half], y[..., half:r] = z.real, z.imag
        out[n] = y
    rows = {n: torch.zeros(s[n + "_cache"].shape, dtype=torch.float64, device="cuda") for n in ("k", "v")}
    rows["k"].view(-1, c["kv_heads"], c["head_dim"])[s["slots"]] = out["k"]
    rows["v"].view(-1, c["kv_heads"], c["head_dim"])[s["slots"]] = s["v"].double()
    return {"q": out["q"], "k_cache": rows["k"], "v_cache": rows["v"]}


def _exact_pass(s):
    """Attention and weights, a sequence and a head at a time."""
    c = s["case"]
    hk, d, ps = c["kv_heads"], c["head_dim"], c["page_size"]
    group = c["q_heads"] // hk
    q_lens, lens = _lengths(c)
    want_out = c["op"] == "paged_attention"
    if want_out:
        out, lse = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("out", "lse"))
    else:
        weights = torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for b, (m, n) in enumerate(zip(q_lens, lens)):
        pages = s["table"][b, : -(-n // ps)].long()
        k, v = (s[x][pages].flatten(0, 1)[:n] for x in ("k", "v"))
        j = torch.arange(n, device="cuda")
        at = torch.arange(n - m, n, device="cuda")[:, None]
        hidden = j > at
        if c["window"]:
            hidden |= j <= at - c["window"]
        for h in range(c["q_heads"]):
            x = (s["q"][start:start + m, h].double() @ k[:, h // group].double().T) / math.sqrt(d)
            x[hidden] = -math.inf
            if want_out:
                lse[start:start + m, h] = torch.logsumexp(x, 1)
                out[start:start + m, h] = torch.softmax(x, 1) @ v[:, h // group].double()
            else:
                weights[b, h // group, :n] += torch.exp(x - s["lse"][start:start + m, h, None].double()).sum(0)
        if not want_out:
            weights[b, :, : n - m] += s["weights_in"][b, :, : n - m].double()
        start += m
    return {"out": out, "lse": lse} if want_out else {"weights": weights}


def _exact_evict(s):
    c = s["case"]
    ps, budget, recent = c["page_size"], c["budget"], c["recent"]
    k, v = s["k"].double(), s["v"].double()
    weights = torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(c)[1]):
        keep = min(n, budget)
        for h in range(c["kv_heads"]):
            w = s["weights_in"][b, h, :n].double()
            old = max(0, n - recent)
            best = torch.argsort(-w[:old], stable=True)[: keep - (n - old)]
            ids = torch.cat((best.sort().values, torch.arange(old, n, device="cuda"))) if n > budget else torch.arange(n, device="cuda")
            to = torch.arange(keep, device="cuda")
            src, dst = s["table"][b].long()[ids // ps], s["kept_table"][b].long()[to // ps]
            for x in (k, v):
                x[dst, to % ps, h] = x[src, ids % ps, h]
            weights[b, h, :keep] = w[ids]
    return {"k": k, "v": v, "weights": weights, "lens": None}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "qk_norm_rope":
        return _exact_rope(s)
    return _exact_evict(s) if case["op"] == "paged_evict" else _exact_pass(s)
