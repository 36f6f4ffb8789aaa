"""The operators over a cache in 8 bits without a GPU: what the host refuses
before any device work, workspaces, structures, what the kernels spill, and the
search for a token's sequence."""
import ctypes
import glob
import itertools
import json
import math
import os
import subprocess

import numpy as np
import pytest

import kernelh as kh
from cache8test import codes_of, held, numbers, stand_for
from test_cache_cpu import BAD_QUERIES, BAD_TABLE, refused, table

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CO = os.path.join(REPO, "kernel.h_amd", "build", "co")


def cache(**kw):
    f = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, k_page_stride=16 * 2 * 64, k_slot_stride=2 * 64,
             k_head_stride=64, v_page_stride=16 * 2 * 64, v_slot_stride=2 * 64, v_head_stride=64, scale_page_stride=32,
             scale_head_stride=16, pages=10, page_size=16, kv_heads=2, head_dim=64)
    return kh.PagedCache8(**{**f, **kw})


def rope(**kw):
    f = dict(q=16, k=32, v=48, q_out=64, k_out=80, inv_freq=8, positions=8, slots=8, q_stride=256, k_stride=128,
             v_stride=128, q_out_stride=256, k_out_stride=128, axis_stride=5, axes=3, cache=cache(), tokens=5, q_heads=4,
             rotary_dim=64, norm=1, dtype=kh.BF16, eps=1e-6)
    return kh.QkNormRope8(**{**f, **kw})


def read(**kw):
    f = dict(cache=cache(), slots=8, k_out=16, v_out=32, k_out_stride=128, v_out_stride=128, tokens=5, dtype=kh.BF16)
    return kh.PagedRead8(**{**f, **kw})


def attention(**kw):
    f = dict(cache=cache(), table=table(), q=16, out=32, lse=4, q_starts=4, q_stride=256, out_stride=256, tokens=5,
             q_heads=4, window=0, scale=0.125, cap=0.0, dtype=kh.BF16)
    return kh.PagedAttention8(**{**f, **kw})


BAD_CACHE = [
    dict(head_dim=0), dict(head_dim=72), dict(head_dim=8), dict(head_dim=272), dict(kv_heads=0), dict(kv_heads=65536), dict(k=None),
    dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(pages=0), dict(pages=1 << 31), dict(page_size=0),
    dict(page_size=(1 << 20) + 1), dict(k=(1 << 20) + 8), dict(v=(1 << 20) + 2), dict(k_page_stride=-64), dict(v_slot_stride=-16),
    dict(k_head_stride=72), dict(v_page_stride=2049), dict(k_slot_stride=1 << 60), dict(k_page_stride=1 << 56),
    dict(v_page_stride=1 << 32), dict(scale_page_stride=-1), dict(scale_head_stride=-1), dict(scale_page_stride=1 << 32)]
BAD_WRITTEN = [dict(k_page_stride=0), dict(v_slot_stride=48), dict(k_head_stride=16), dict(k_slot_stride=64), dict(scale_page_stride=0),
               dict(scale_head_stride=15), dict(scale_page_stride=31), dict(v=1 << 20), dict(v_scale=3 << 20), dict(k_scale=1 << 20)]


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_caches_are_refused(kw):
    refused(lambda: kh.qk_norm_rope8(rope(cache=cache(**kw))), "qk_norm_rope8")
    refused(lambda: kh.paged_read8(read(cache=cache(**kw))), "paged_read8")
    refused(lambda: kh.paged_attention8(attention(cache=cache(**kw))), "paged_attention8")
    refused(lambda: kh.paged_attention8_workspace(attention(cache=cache(**kw))), "paged_attention8_workspace")


@pytest.mark.parametrize("kw", BAD_WRITTEN, ids=str)
def test_caches_whose_rows_overlap_are_not_written(kw):
    refused(lambda: kh.qk_norm_rope8(rope(cache=cache(**kw))), "qk_norm_rope8")
    assert kh.paged_attention8_workspace(attention(cache=cache(**kw))) >= 0


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(slots=None), dict(positions=None), dict(inv_freq=None),
    dict(rotary_dim=-8), dict(rotary_dim=72), dict(rotary_dim=12), dict(eps=-1.0), dict(eps=float("nan")), dict(q=8),
    dict(k_out=8), dict(q_gamma=8), dict(v=50), dict(q_stride=-8), dict(k_stride=100), dict(v_stride=9), dict(q_out_stride=128),
    dict(k_out_stride=64), dict(tokens=0), dict(q_heads=0), dict(q_heads=65536), dict(tokens=1 << 40), dict(dtype=3), dict(dtype=-1),
    dict(axes=0), dict(axes=129), dict(axis_stride=-1), dict(axis_stride=1 << 41), dict(q_out=16, q_out_stride=512),
    dict(k_out=32, k_out_stride=256), dict(q_out=32), dict(q_out=48), dict(q_out=80), dict(k_out=16), dict(k_out=48),
    dict(q_out=1 << 20), dict(k_out=2 << 20), dict(v=3 << 20)], ids=str)
def test_writes_are_refused(kw):
    refused(lambda: kh.qk_norm_rope8(rope(**kw)), "qk_norm_rope8")


@pytest.mark.parametrize("kw", [
    dict(slots=None), dict(k_out=None, v_out=None), dict(k_out=8), dict(v_out=40), dict(k_out_stride=127), dict(v_out_stride=64),
    dict(k_out_stride=-128), dict(tokens=0), dict(tokens=1 << 40), dict(dtype=3), dict(k_out=32), dict(k_out=1 << 20),
    dict(v_out=4 << 20), dict(slots=16)], ids=str)
def test_reads_are_refused(kw):
    refused(lambda: kh.paged_read8(read(**kw)), "paged_read8")


@pytest.mark.parametrize("call,op", [(kh.paged_attention8, "paged_attention8"), (kh.paged_attention8_workspace, "paged_attention8_workspace")])
def test_attention_is_refused(call, op):
    for kw in BAD_TABLE:
        refused(lambda: call(attention(table=table(**kw))), op)
    for kw in BAD_QUERIES + [
            dict(out=None), dict(out=8), dict(out_stride=248), dict(out_stride=-1), dict(out=16), dict(max_new=-1), dict(shared=-1),
            dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(dtype=3), dict(dtype=-1)]:
        refused(lambda: call(attention(**kw)), op)


def test_attention_refuses_a_misaligned_workspace():
    refused(lambda: kh.paged_attention8(attention(), 24, 1 << 20), "paged_attention8")


def test_null_arguments():
    for fn, args in ((kh.lib.kh_qk_norm_rope8, (None, None)), (kh.lib.kh_paged_read8, (None, None)),
                     (kh.lib.kh_paged_attention8, (None, None, 0, None)), (kh.lib.kh_paged_attention8_workspace, (None, None))):
        assert fn(*args) == kh.KHRT_E_INVALID and kh.last_error()


@pytest.mark.parametrize("dtype", [kh.F32, kh.BF16])
@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (16, 16, 64), (8, 1, 256), (7, 1, 80), (6, 3, 64)])
def test_a_workspace_suffices_for_every_smaller_step(dtype, hq, hk, d):
    """What the largest step reports, no smaller one asks more than: of fewer
    tokens, fewer sequences, shorter ones, under a window, with fewer shared
    entries."""
    st = dict(k_page_stride=16 * hk * d, k_slot_stride=hk * d, k_head_stride=d, v_page_stride=16 * hk * d, v_slot_stride=hk * d,
              v_head_stride=d, scale_page_stride=16 * hk)
    grid = (1, 4, 33, 512, 8192), (1, 4, 64), (300, 1024, 8192, 131072), (0, 4096, 100), (0, 256, 8000)

    def size(t, s, n, w, c):
        return kh.paged_attention8_workspace(attention(
            cache=cache(kv_heads=hk, head_dim=d, **st), table=table(seqs=s, width=8192, row_stride=8192, max_len=n), dtype=dtype,
            q_heads=hq, q_stride=hq * d, out_stride=hq * d, tokens=t, window=w, shared=c))

    all_of = {x: size(*x) for x in itertools.product(*grid)}
    for t, s, n, w, c in all_of:
        for x, need in all_of.items():
            if x[0] <= t and x[1] <= s and x[2] <= n and (w == 0 or 0 < x[3] <= w) and x[4] <= c:
                assert need <= all_of[t, s, n, w, c], (x, (t, s, n, w, c))
    assert all_of[1, 1, 131072, 0, 0] >= 100 * (d + 2) * 4


def test_structures_match_the_header(tmp_path):
    """The binding's structures have the C compiler's sizes and offsets."""
    structs = {"kh_paged_cache8": kh.PagedCache8, "kh_qk_norm_rope8_args": kh.QkNormRope8, "kh_paged_read8_args": kh.PagedRead8,
               "kh_paged_attention8_args": kh.PagedAttention8}
    lines = [f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in s._fields_)
             for c, s in structs.items()]
    src = tmp_path / "sizes.c"
    src.write_text('#include "khrt.h"\n#include <stdio.h>\nint main(void) {' + "\n".join(lines) + "return 0;}")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True, timeout=60)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True, timeout=60).stdout.split()]
    want = [x for s in structs.values() for x in [ctypes.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]]
    assert got == want


def test_index_arithmetic(tmp_path):
    """kh_sequence_of and what is each sequence's own, against their definitions."""
    src = tmp_path / "check.cpp"
    src.write_text(r'''
#include "kh_paged.h"
#include <cstdio>
#include <cstdlib>
static void expect(bool ok, const char *what) { if (!ok) { std::printf("FAIL: %s\n", what); std::exit(1); } }
int main() {
  unsigned seed = 1;
  auto random = [&](int below) { seed = seed * 1664525u + 1013904223u; return static_cast<int>((static_cast<uint64_t>(seed) * below) >> 32); };
  for (int run = 0; run < 2000; ++run) {
    int32_t starts[65];
    const int seqs = 1 + random(64);
    starts[0] = random(3);
    for (int s = 0; s < seqs; ++s) starts[s + 1] = starts[s] + (random(3) ? random(9) : 0);
    for (int t = 0; t < starts[seqs]; ++t) {
      const int s = kh_sequence_of(starts, seqs, t);
      expect(s >= 0 && s < seqs, "a sequence");
      if (t >= starts[0]) expect(starts[s] <= t && t < starts[s + 1], "the token's");
    }
    for (int s = 0; s <= seqs; ++s) starts[s] = random(100) - 20;  // whatever: it ends, in range
    for (int t = 0; t < 100; ++t) {
      const int s = kh_sequence_of(starts, seqs, t);
      expect(s >= 0 && s < seqs, "in range");
    }
    KhAttention8Params p{};
    p.group = 1 + random(8), p.window = random(2) ? random(50) : 0, p.shared = random(300), p.whole = random(2);
    const KhSeq q{random(400), 1 + random(20), 0};
    const KhUnits u = kh_units_of(p, q);
    expect(u.first % 16 == 0 && u.blocks >= 1, "units");
    for (int i = 0; i < q.m; ++i) {
      const KhSpan seen = kh_seen(q, i, p.window), own = kh_span_of(p, q, i);
      expect(own.first >= p.shared && own.end == seen.end && own.first >= seen.first, "behind the shared entries");
      expect(own.first == seen.first || own.first == p.shared, "as far as they go");
      if (own.first < own.end) expect(u.first <= own.first && (p.whole || u.first + u.blocks * KH_STRETCH >= own.end), "inside the unit");
    }
  }
  std::puts("ok");
}
''')
    exe = tmp_path / "check"
    r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined",
                        "-fno-sanitize-recover=all", "-I", os.path.join(REPO, "kernel.h_amd", "csrc", "kernels"), str(src), "-o", str(exe)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


# Symbols that spill, and how much at the most: registers and bytes of scratch of a lane.
SPILLS = {"attention8_odd_128_f32": (24, 100), "attention8_odd_128_f16": (6, 28), "attention8_wide_256_f32": (106, 416),
          "attention8_wide_128_f16": (20, 48), "attention8_wide_256_f16": (42, 160),
          "rope8_8_f16": (2, 12), "rope8_16_f16": (2, 12), "rope8_32_f16": (4, 20), "rope8_32_bf16": (1, 8)}


def test_what_the_kernels_spill():
    found = 0
    for path in glob.glob(os.path.join(CO, "*.notes.json")):
        if not os.path.basename(path).startswith(("attention8_", "read8_", "rope8_")):
            continue
        with open(path) as f:
            for k in json.load(f):
                registers, scratch = SPILLS.get(k["name"], (0, 0))
                assert k["vgpr_spill_count"] <= registers and k["private_segment_bytes"] <= scratch, k
                found += 1
    assert found == 9 + 3 + 3 * 15 or not os.path.isdir(CO)


# ---------------------------------------------------------------- the oracle

def test_the_oracle_rounds_to_nearest_even():
    """Every number is its own code; what lies between two goes to the nearer,
    a tie to the even code."""
    c = np.arange(127)
    x = numbers(c)
    assert np.array_equal(codes_of(x), c) and np.array_equal(codes_of(-x), c | 0x80)
    middle = (x[1:] + x[:-1]) / 2
    even = np.where(c[:-1] % 2 == 0, c[:-1], c[1:])
    assert np.array_equal(codes_of(middle), even)
    assert np.array_equal(codes_of(np.nextafter(middle, 1e9)), c[1:]) and np.array_equal(codes_of(np.nextafter(middle, 0)), c[:-1])
    assert codes_of(math.nan) == 0x7F


def test_the_oracle_takes_the_least_power():
    g = np.random.default_rng(0)
    x = g.standard_normal((500, 16)) * np.exp2(g.integers(-100, 100, (500, 1)))
    x[0], x[1, 0], x[2, 0] = 0.0, 448 * 2.0 ** 150, 1e-40
    codes, scales = held(x)
    e = scales.astype(int) - 127
    top = np.abs(x).max(1)
    assert ((448 * np.exp2(e) >= top) | (e == 119)).all() and ((448 * np.exp2(e - 1.0) < top) | (e == -117)).all()
    y = stand_for(codes, scales).astype(np.float64)
    keep = e < 119
    assert (np.abs(y - x)[keep] <= (np.abs(x) * 2.0 ** -4 + np.exp2(e - 10.0)[:, None])[keep]).all()


# ---------------------------------------------------------------- the kernels' assembly

@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CO, "attention8_*.isa"))), ids=os.path.basename)
def test_loads_to_lds_bring_their_wait_states_and_keep_m0(path):
    """A run of loads straight to LDS begins with M0 saved, set and five wait
    states, moves M0 and waits one between its loads, and ends with M0 restored."""
    from test_device_code_cpu import instructions

    code, runs = instructions(path), 0
    to_lds = [op.startswith("buffer_load") and "lds" in args[-1].split() for op, args in code]
    for i in range(len(code)):
        if not to_lds[i] or (to_lds[i - 3] and code[i - 2][0] == "s_add_u32"):
            continue
        save, set_m0, nop = code[i - 3], code[i - 2], code[i - 1]
        assert save[0] == set_m0[0] == "s_mov_b32" and save[1][1] == "m0" and set_m0[1][0] == "m0", code[i - 3:i + 1]
        assert nop[0] == "s_nop" and int(nop[1][0]) + 3 >= 5, code[i - 3:i + 1]
        j = i
        while code[j + 1][0] == "s_add_u32":
            assert code[j + 1][1][:2] == ["m0", "m0"] and code[j + 2][0] == "s_nop" and to_lds[j + 3], code[i:j + 4]
            j += 3
        assert code[j + 1] == ("s_mov_b32", ["m0", save[1][0]]), code[i:j + 2]
        runs += 1
    assert runs > 0
