"""The calls the operators over a cache in 8 bits are timed at, and their plain
forms.

A serving step of a decoder whose cache holds keys and values as e4m3 numbers,
each row with a power of two of its own: the new tokens' rows are normalised,
rotated by one or several positions (text; time, height and width of images and
video), rounded and written (qk_norm_rope8); rows are read back where a cache
is moved or inspected (paged_read8); and the step attends over the cache
(paged_attention8), with scores capped by a tanh where a model has that, and
with the entries that all sequences of a batch share read once for all.

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
        {"name": "write_f32_5x16", "op": "qk_norm_rope8", "dtype": "f32", "tokens": 5, "q_heads": 16, "kv_heads": 16,
         "head_dim": 64, "rotary": 64, "interleaved": False, "axes": 1, "turns": False, "page_size": 16, "far": 4096},
        # A prompt's chunk of a grouped-query model that sees images: a section
        # of each head for time, height and width. Bound by memory.
        {"name": "write_bf16_8192_3axes", "op": "qk_norm_rope8", "dtype": "bf16", "tokens": 8192, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "rotary": 128, "interleaved": False, "axes": 3, "turns": False,
         "page_size": 16, "far": 131072},
        # Half of each head rotated in neighbouring pairs, the axes taking
        # turns, a ragged token count, positions past a million.
        {"name": "write_f16_1999_2axes", "op": "qk_norm_rope8", "dtype": "f16", "tokens": 1999, "q_heads": 24,
         "kv_heads": 24, "head_dim": 96, "rotary": 48, "interleaved": True, "axes": 2, "turns": True, "page_size": 32,
         "far": 2000000},
        # The pages of a short conversation read back to be sent elsewhere.
        {"name": "read_f16_777", "op": "paged_read8", "dtype": "f16", "tokens": 777, "kv_heads": 5, "head_dim": 80,
         "page_size": 24},
        # A long one's, as bf16 rows for a cache of that type.
        {"name": "read_bf16_65536", "op": "paged_read8", "dtype": "bf16", "tokens": 65536, "kv_heads": 8,
         "head_dim": 128, "page_size": 16},
        # One new token for each of four sequences (the attention benchmark's
        # batch, heads and shorter length).
        {"name": "decode_f32_b4_1024", "op": "paged_attention8", "dtype": "f32", "seqs": 4, "q_min": 1, "q_max": 1,
         "len_min": 1024, "len_max": 1024, "shared": 0, "q_heads": 16, "kv_heads": 16, "head_dim": 64, "window": 0,
         "cap": 0.0, "page_size": 16},
        # A serving batch in the middle of its answers: lengths all over.
        {"name": "decode_bf16_64_ragged", "op": "paged_attention8", "dtype": "bf16", "seqs": 64, "q_min": 1,
         "q_max": 1, "len_min": 513, "len_max": 8192, "shared": 0, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "window": 0, "cap": 0.0, "page_size": 16},
        # One very long sequence: few rows, so its length is what fills the chip.
        {"name": "decode_bf16_131071", "op": "paged_attention8", "dtype": "bf16", "seqs": 1, "q_min": 1, "q_max": 1,
         "len_min": 131071, "len_max": 131071, "shared": 0, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "window": 0, "cap": 0.0, "page_size": 64},
        # A chunk of a long prompt over what is cached of it: bound by the
        # matrix units.
        {"name": "chunk_bf16_2048of8192", "op": "paged_attention8", "dtype": "bf16", "seqs": 1, "q_min": 2048,
         "q_max": 2048, "len_min": 8192, "len_max": 8192, "shared": 0, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "window": 0, "cap": 0.0, "page_size": 16},
        # Chunks and single tokens in one batch, a sliding window and capped
        # scores, heads of no power of two, pages that end inside every tile.
        {"name": "mixed_f16_window_cap", "op": "paged_attention8", "dtype": "f16", "seqs": 16, "q_min": 1,
         "q_max": 301, "len_min": 400, "len_max": 4001, "shared": 0, "q_heads": 12, "kv_heads": 4, "head_dim": 80,
         "window": 1000, "cap": 30.0, "page_size": 24},
        # A batch of answers to questions about one long document.
        {"name": "shared_bf16_64x8192", "op": "paged_attention8", "dtype": "bf16", "seqs": 64, "q_min": 1, "q_max": 1,
         "len_min": 8200, "len_max": 8900, "shared": 8192, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0,
         "cap": 0.0, "page_size": 16},
        # Drafts of a few tokens each behind a common prompt of odd length.
        {"name": "shared_f32_7x1001_drafts", "op": "paged_attention8", "dtype": "f32", "seqs": 7, "q_min": 1,
         "q_max": 5, "len_min": 1010, "len_max": 1321, "shared": 1001, "q_heads": 16, "kv_heads": 4, "head_dim": 64,
         "window": 0, "cap": 50.0, "page_size": 7},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk_norm_rope8", "paged_read8", "paged_attention8", "paged_attention8", "paged_attention8"])
    d = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    case = {"op": op, "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "head_dim": d}
    kv, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 7, 8])
    ps = rng.choice([1, 7, 16, 16, 24, 32, 64, 100, 256])
    case |= {"kv_heads": kv, "page_size": ps}
    if op == "qk_norm_rope8":
        return case | {"tokens": _spread(rng, 1, 8192), "q_heads": kv * group, "rotary": rng.choice([d, d, d // 16 * 8]),
                       "interleaved": rng.random() < 0.4, "axes": rng.choice([1, 2, 3, 3]), "turns": rng.random() < 0.5,
                       "far": _spread(rng, 1000, 2000000)}
    if op == "paged_read8":
        return case | {"tokens": _spread(rng, 1, 65536)}
    case |= {"q_heads": kv * group, "window": rng.choice([0, 0, 0, _spread(rng, 1, 4096)]),
             "cap": rng.choice([0.0, 0.0, 20.0, 50.0])}
    if rng.random() < 0.6:  # decoding, a token or a few proposed ones
        q_max = rng.choice([1, 1, 1, 2, 5])
        top = _spread(rng, q_max, 65536)
        seqs = _spread(rng, 1, max(1, min(128, (1 << 28) // (top * kv * d))))
    else:  # chunks
        q_max = _spread(rng, 2, 2048)
        top = _spread(rng, q_max, 16384)
        while q_max * top * kv * group > 1 << 28:
            q_max, top = max(2, q_max // 2), max(2, q_max // 2, top // 2)
        seqs = _spread(rng, 1, max(1, min(16, (1 << 28) // (q_max * top * kv * group), (1 << 28) // (top * kv * d))))
    low = rng.randint(q_max, top)
    shared = 0
    if seqs > 1 and low - q_max >= ps and rng.random() < 0.5:
        shared = rng.randint(ps, low - q_max) // ps * ps
    return case | {"seqs": seqs, "q_min": 1 if rng.random() < 0.5 else q_max, "q_max": q_max, "len_min": low,
                   "len_max": top, "shared": shared}


def _between(lo, hi, n, step):
    """n whole numbers spread evenly, in no order, from lo to hi; the first is hi."""
    return [hi - int((i * step) % 1.0 * (hi - lo + 1)) for i in range(n)]


def _lengths(case):
    """(new tokens, entries in the cache with them) of each sequence."""
    lens = _between(case["len_min"], case["len_max"], case["seqs"], 0.6180339887498949)
    return _between(case["q_min"], case["q_max"], case["seqs"], 0.7548776662466927), lens


def _visible(case, q, n):
    """Entries that the q new tokens of a sequence of n see, summed over them."""
    w = case["window"] or n
    return sum(min(n - q + i + 1, w) for i in range(q))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _power(e):
    """2^e, exactly, for e from -126 to 127."""
    return (e.to(torch.int32) + 127 << 23).view(torch.float32)


def _held(x):
    """Rows of x in 32 bits as the cache holds them: e4m3 numbers in bytes, and
    the exponent e of the power of two that each row is a multiple of, plus 127:
    the smallest from -117 to 119 with 448 2^e no less than the row's largest."""
    top = x.abs().amax(-1)
    part, e = torch.frexp(top)  # top = part 2^e, part in [1/2, 1); 448 = 7/8 2^9
    e = torch.clamp(e - 9 + (part > 0.875).int(), -117, 119)
    y = torch.clamp(x * _power(-e)[..., None], -448.0, 448.0)
    return y.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _value(codes, scales):
    """What the cache's bytes stand for."""
    return codes.view(torch.float8_e4m3fn).float() * _power(scales.to(torch.int32) - 127)[..., None]


def prepare(case, seed):
    g = _gen(seed)
    dtype, d, ps, hk = _DTYPES[case["dtype"]], case["head_dim"], case["page_size"], case["kv_heads"]
    if case["op"] == "qk_norm_rope8":
        t, hq = case["tokens"], case["q_heads"]
        # q, k and v are parts of one projection's output.
        qkv = _normal(g, (t, hq + 2 * hk, d), dtype) * 2
        pages, r, axes = -(-t // ps) + 3, case["rotary"], case["axes"]
        pair = torch.arange(r // 2, device="cuda")
        # Sections of about a quarter, three eighths and the rest, or the axes in turn.
        axis = pair % axes if case["turns"] else (pair >= r // 8).int() + (pair >= r // 8 + r * 3 // 16).int()
        return {"case": case, "q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "v": qkv[:, hq + hk:],
                "q_gamma": (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype),
                "k_gamma": (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype),
                "inv_freq": (10000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)).float(),
                "axis": torch.clamp(axis, max=axes - 1).to(torch.int32),
                "positions": torch.randint(0, case["far"], (axes, t), generator=g, device="cuda"),
                "slots": torch.randperm(pages * ps, generator=g, device="cuda")[:t],
                "q_out": torch.zeros((t, hq, d), dtype=dtype, device="cuda"),
                "k_cache": torch.zeros((pages, ps, hk, d), dtype=torch.uint8, device="cuda"),
                "v_cache": torch.zeros((pages, ps, hk, d), dtype=torch.uint8, device="cuda"),
                "k_scale": torch.zeros((pages, hk, ps), dtype=torch.uint8, device="cuda"),
                "v_scale": torch.zeros((pages, hk, ps), dtype=torch.uint8, device="cuda")}
    s = {"case": case}
    if case["op"] == "paged_read8":
        t = case["tokens"]
        pages = -(-t // ps) + 3
        s["slots"] = torch.randperm(pages * ps, generator=g, device="cuda")[:t]
        s["k_out"], s["v_out"] = (torch.zeros((t, hk, d), dtype=dtype, device="cuda") for _ in "kv")
    else:
        q_lens, lens = _lengths(case)
        s["lens"] = _ints(lens)
        # Each sequence's pages, the shared ones first; a page that the shared
        # entries end inside is each sequence's own.
        common = case["shared"] // ps
        widths = [-(-n // ps) for n in lens]
        pages = common + sum(w - common for w in widths) + 1
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        s["table"] = torch.zeros((len(lens), max(widths)), dtype=torch.int32, device="cuda")
        at = common
        for i, w in enumerate(widths):
            s["table"][i, :common] = order[:common]
            s["table"][i, common:w] = order[at:at + w - common]
            at += w - common
    for name in ("k", "v"):
        codes, scales = _held(torch.randn((pages, ps, hk, d), generator=g, device="cuda"))
        s[name + "_cache"], s[name + "_scale"] = codes, scales.transpose(1, 2).contiguous()
    if case["op"] == "paged_read8":
        return s
    rest = case["shared"] % ps
    if rest:
        own_pages = s["table"][:, common].long()
        for name in ("k", "v"):
            s[name + "_cache"][own_pages, :rest] = s[name + "_cache"][own_pages[0], :rest].clone()
            s[name + "_scale"][own_pages, :, :rest] = s[name + "_scale"][own_pages[0], :, :rest].clone()
    starts = [sum(q_lens[:i]) for i in range(len(q_lens) + 1)]
    t, hq = starts[-1], case["q_heads"]
    s["q"] = _normal(g, (t, hq, d), dtype)
    s["q_starts"] = _ints(starts)
    s["token_seq"] = _ints([i for i, q in enumerate(q_lens) for _ in range(q)], torch.int64)
    s["token_at"] = _ints([j for q in q_lens for j in range(q)], torch.int64)
    s["q_most"], s["len_most"] = max(q_lens), max(lens)
    s["out"] = torch.zeros((t, hq, d), dtype=dtype, device="cuda")
    s["lse"] = torch.zeros((t, hq), device="cuda")
    s["workspace"] = torch.empty(128 << 20, dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------- the framework's calls
# A program that repeats a call keeps its structure of arguments.


def _struct_cache(kh, case, s):
    k, v, ks, vs = s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    return kh.PagedCache8(k=k.data_ptr(), v=v.data_ptr(), k_scale=ks.data_ptr(), v_scale=vs.data_ptr(),
                          k_page_stride=k.stride(0), k_slot_stride=k.stride(1), k_head_stride=k.stride(2),
                          v_page_stride=v.stride(0), v_slot_stride=v.stride(1), v_head_stride=v.stride(2),
                          scale_page_stride=ks.stride(0), scale_head_stride=ks.stride(1), pages=k.shape[0],
                          page_size=case["page_size"], kv_heads=case["kv_heads"], head_dim=case["head_dim"])


def _own_write(s):
    kh, c = _kh(), s["case"]
    if "args" not in s:
        s["args"] = kh.QkNormRope8(
            q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), q_out=s["q_out"].data_ptr(),
            q_gamma=s["q_gamma"].data_ptr(), k_gamma=s["k_gamma"].data_ptr(), inv_freq=s["inv_freq"].data_ptr(),
            positions=s["positions"].data_ptr(), pair_axis=s["axis"].data_ptr(), slots=s["slots"].data_ptr(),
            q_stride=s["q"].stride(0), k_stride=s["k"].stride(0), v_stride=s["v"].stride(0),
            q_out_stride=s["q_out"].stride(0), axis_stride=s["positions"].stride(0), axes=c["axes"],
            cache=_struct_cache(kh, c, s), tokens=c["tokens"], q_heads=c["q_heads"], rotary_dim=c["rotary"],
            interleaved=c["interleaved"], norm=1, dtype=getattr(kh, c["dtype"].upper()), eps=1e-6)
    kh.qk_norm_rope8(s["args"])
    return s["q_out"]


def _own_read(s):
    kh, c = _kh(), s["case"]
    if "args" not in s:
        s["args"] = kh.PagedRead8(
            cache=_struct_cache(kh, c, s), slots=s["slots"].data_ptr(), k_out=s["k_out"].data_ptr(),
            v_out=s["v_out"].data_ptr(), k_out_stride=s["k_out"].stride(0), v_out_stride=s["v_out"].stride(0),
            tokens=c["tokens"], dtype=getattr(kh, c["dtype"].upper()))
    kh.paged_read8(s["args"])


def _own_attention(s):
    kh, c = _kh(), s["case"]
    if "args" not in s:
        t = s["table"]
        s["args"] = kh.PagedAttention8(
            cache=_struct_cache(kh, c, s),
            table=kh.PageTable(pages=t.data_ptr(), lens=s["lens"].data_ptr(), row_stride=t.stride(0), seqs=t.shape[0],
                               width=t.shape[1], max_len=s["len_most"]),
            q=s["q"].data_ptr(), out=s["out"].data_ptr(), lse=s["lse"].data_ptr(), q_starts=s["q_starts"].data_ptr(),
            q_stride=s["q"].stride(0), out_stride=s["out"].stride(0), tokens=s["q"].shape[0], q_heads=c["q_heads"],
            window=c["window"], max_new=s["q_most"], shared=c["shared"], scale=c["head_dim"] ** -0.5, cap=c["cap"],
            dtype=getattr(kh, c["dtype"].upper()))
    kh.paged_attention8(s["args"], s["workspace"].data_ptr(), s["workspace"].numel())


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


def _plain_write(s):
    c, dtype, ps = s["case"], s["q"].dtype, s["case"]["page_size"]
    angle = s["positions"].double()[s["axis"].long()].T * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    q, k = (_plain_rotated(_plain_normed(s[n], s[n + "_gamma"]), cos, sin, c["rotary"], c["interleaved"])
            for n in ("q", "k"))
    for name, x in (("k", k), ("v", s["v"].float())):
        codes, scales = _held(x)
        s[name + "_cache"].view(-1, c["kv_heads"], c["head_dim"])[s["slots"]] = codes
        s[name + "_scale"][s["slots"] // ps, :, s["slots"] % ps] = scales
    return q.to(dtype)


def _plain_read(s):
    c, ps = s["case"], s["case"]["page_size"]
    for name in ("k", "v"):
        codes = s[name + "_cache"].view(-1, c["kv_heads"], c["head_dim"])[s["slots"]]
        s[name + "_out"].copy_(_value(codes, s[name + "_scale"][s["slots"] // ps, :, s["slots"] % ps]))


def _rows_of(s, name, n):
    """Entries 0 .. n - 1 of each sequence, [sequences, n, kv heads, head_dim]."""
    ps = s["case"]["page_size"]
    j = torch.arange(n, device="cuda")
    page = s["table"].long()[:, j // ps]
    return _value(s[name + "_cache"][page, j % ps], s[name + "_scale"][page, :, j % ps])


def _plain_attention(s):
    c = s["case"]
    hk, d, n, m = c["kv_heads"], c["head_dim"], s["len_most"], s["q_most"]
    group, seqs = c["q_heads"] // hk, c["seqs"]
    k = _rows_of(s, "k", n).permute(0, 2, 3, 1).contiguous()
    i, j = torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
    q_lens = (s["q_starts"][1:] - s["q_starts"][:-1]).long()
    token = torch.clamp(s["q_starts"][:-1].long()[:, None] + i, max=s["q"].shape[0] - 1)
    q = s["q"][token].float().view(seqs, m, hk, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hk, group * m, d)
    x = torch.matmul(q, k).view(seqs, hk, group, m, n)
    x = c["cap"] * torch.tanh(x * (d ** -0.5 / c["cap"])) if c["cap"] else x * d ** -0.5
    at = s["lens"].long()[:, None] - q_lens[:, None] + i
    seen = (j <= at[..., None]) & (i < q_lens[:, None])[..., None]
    if c["window"]:
        seen = seen & (j > at[..., None] - c["window"])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = torch.clamp(x.amax(-1, keepdim=True), min=-1e30)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    v = _rows_of(s, "v", n).permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p.view(seqs, hk, -1, n), v).view(seqs, hk, -1, m, d) / torch.clamp(total, min=1e-30)
    lse = (top + torch.log(total))[..., 0]
    o, lse = (t[s["token_seq"], :, :, s["token_at"]] for t in (o, lse))
    s["out"].copy_(o.reshape(-1, c["q_heads"], d))
    s["lse"].copy_(lse.reshape(-1, c["q_heads"]))


_PLAIN = {"qk_norm_rope8": _plain_write, "paged_read8": _plain_read, "paged_attention8": _plain_attention}
_OWN = {"qk_norm_rope8": _own_write, "paged_read8": _own_read, "paged_attention8": _own_attention}


def run(state):
    got = (_OWN if own else _PLAIN)[state["case"]["op"]](state)
    if state["case"]["op"] == "paged_read8":
        return {"k": state["k_out"], "v": state["v_out"]}
    if state["case"]["op"] == "paged_attention8":
        return {"out": state["out"], "lse": state["lse"]}
    # The cache as it is held: e4m3 numbers, and the powers of two they are multiples of.
    held = {n: state[n + "_cache"].view(torch.float8_e4m3fn) for n in "kv"}
    return {"q": got, **held, **{n + "_scale": state[n + "_scale"].view(torch.float8_e8m0fnu) for n in "kv"}}


def work(case):
    e, d, hk = _BYTES[case["dtype"]], case["head_dim"], case["kv_heads"]
    if case["op"] == "qk_norm_rope8":
        t, heads = case["tokens"], case["q_heads"] + hk
        # Rows read in their type, q written in it, k and v in 8 bits with a
        # scale each; positions and slots once.
        return {"bytes": t * ((2 * case["q_heads"] + 2 * hk) * d * e + 2 * hk * (d + 1) + 8 * case["axes"] + 8)
                + 2 * d * e + 4 * case["rotary"],
                "flops": t * heads * (4 * d + 3 * case["rotary"]) + t * hk * 4 * d}
    if case["op"] == "paged_read8":
        return {"bytes": case["tokens"] * (2 * hk * (d + 1 + d * e) + 8), "flops": case["tokens"] * 2 * hk * d}
    q_lens, lens = _lengths(case)
    hq, t = case["q_heads"], sum(q_lens)
    seen = sum(_visible(case, q, n) for q, n in zip(q_lens, lens))
    # Entries that some new token sees, the shared ones counted once.
    first = [max(0, n - (case["window"] or n) - q + 1) for q, n in zip(q_lens, lens)]
    read = sum(n - max(f, case["shared"]) for n, f in zip(lens, first)) + max(0, case["shared"] - min(first))
    return {"bytes": 2 * hk * read * (d + 1) + t * hq * (2 * d * e + 4),
            "flops": hq * seen * (4 * d + (7 if case["cap"] else 4))}


# ---------------------------------------------------------------- from the definitions, in 64 bits


def _numbers():
    """The value of each of the 256 codes."""
    codes = range(256)
    size = [(c & 7) * 2.0 ** -9 if c & 0x78 == 0 else (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10) for c in codes]
    values = [math.nan if c & 0x7F == 0x7F else -v if c & 0x80 else v for c, v in zip(codes, size)]
    return torch.tensor(values, dtype=torch.float64, device="cuda")


def _exact_power(e):
    return (e.to(torch.int64) + 1023 << 52).view(torch.float64)


def _exact_held(x):
    """The numbers and powers of two that rows of x are held as."""
    top = x.abs().amax(-1, keepdim=True)
    power = torch.full_like(top, 2.0 ** -117)
    rough = torch.floor(torch.log2(torch.clamp(top, min=1e-300))) - 9
    for more in range(3):  # the logarithm is off by less than one
        e = torch.clamp(rough + more, -117, 119)
        p = _exact_power(e)
        power = torch.where((448 * p >= top) & ((448 * power < top) | (more == 0)), p, power)
    y = torch.clamp(x / power, -448, 448)
    # Eight steps to each power of two from 2^-6 on, steps of 2^-9 below.
    _, e = torch.frexp(torch.clamp(y.abs(), min=2.0 ** -6))
    step = _exact_power(e - 4)
    return torch.round(y / step) * step, power[..., 0]


def _exact_write(s):
    c = s["case"]
    ps, r, half = c["page_size"], c["rotary"], c["rotary"] // 2
    angles = torch.stack([s["positions"][a].double() * f.double() for a, f in zip(s["axis"].tolist(), s["inv_freq"])], 1)
    turn = torch.polar(torch.ones_like(angles), angles)[:, None]
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
    got = {"q": out["q"]}
    for n, x in (("k", out["k"]), ("v", s["v"].double())):
        numbers, powers = _exact_held(x)
        got[n] = torch.zeros(s[n + "_cache"].shape, dtype=torch.float64, device="cuda")
        got[n + "_scale"] = torch.full(s[n + "_scale"].shape, 2.0 ** -127, dtype=torch.float64, device="cuda")
        got[n][s["slots"] // ps, s["slots"] % ps] = numbers
        got[n + "_scale"][s["slots"] // ps, :, s["slots"] % ps] = powers
    return got


def _exact_rows(s, name, pages, slots):
    """Rows of the entries in these slots of these pages, [entries, kv heads, head_dim]."""
    power = _exact_power(s[name + "_scale"][pages, :, slots].long() - 127)
    return _numbers()[s[name + "_cache"][pages, slots].long()] * power[..., None]


def _exact_attention(s):
    """A sequence and a head at a time."""
    c = s["case"]
    ps, group = c["page_size"], c["q_heads"] // c["kv_heads"]
    out, lse = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("out", "lse"))
    start = 0
    for b, (m, n) in enumerate(zip(*_lengths(c))):
        j = torch.arange(n, device="cuda")
        k, v = (_exact_rows(s, x, s["table"][b].long()[j // ps], j % ps) for x in "kv")
        at = torch.arange(n - m, n, device="cuda")[:, None]
        hidden = j > at
        if c["window"]:
            hidden |= j <= at - c["window"]
        for h in range(c["q_heads"]):
            x = (s["q"][start:start + m, h].double() @ k[:, h // group].T) / math.sqrt(c["head_dim"])
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            x[hidden] = -math.inf
            lse[start:start + m, h] = torch.logsumexp(x, 1)
            out[start:start + m, h] = torch.softmax(x, 1) @ v[:, h // group]
        start += m
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "qk_norm_rope8":
        return _exact_write(s)
    if case["op"] == "paged_read8":
        return {n: _exact_rows(s, n, s["slots"] // case["page_size"], s["slots"] % case["page_size"]) for n in "kv"}
    return _exact_attention(s)
