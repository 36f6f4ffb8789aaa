"""The sequence-cache operators without a GPU: the index arithmetic that their
kernels share with the launcher, and everything the host refuses before any
device work."""
import ctypes
import os
import subprocess

import pytest

import kernelh as kh

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_index_arithmetic(tmp_path):
    exe = tmp_path / "paged_check"
    r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined",
                        "-fno-sanitize-recover=all", "-I", os.path.join(REPO, "kernel.h_amd", "csrc", "kernels"),
                        os.path.join(REPO, "tests", "cpp", "paged_check.cpp"), "-o", str(exe)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("paged_check ok"), r.stdout


def cache(**kw):
    f = dict(k=1 << 20, v=2 << 20, k_page_stride=16 * 2 * 64, k_slot_stride=2 * 64, k_head_stride=64,
             v_page_stride=16 * 2 * 64, v_slot_stride=2 * 64, v_head_stride=64, pages=10, page_size=16, kv_heads=2,
             head_dim=64, dtype=kh.BF16)
    return kh.PagedCache(**{**f, **kw})


def table(**kw):
    return kh.PageTable(**{**dict(pages=1 << 12, lens=2 << 12, row_stride=4, seqs=3, width=4, max_len=0), **kw})


def rope(**kw):
    f = dict(q=16, k=32, v=48, q_out=64, k_out=80, inv_freq=8, positions=8, slots=8, q_stride=256, k_stride=128,
             v_stride=128, q_out_stride=256, k_out_stride=128, cache=cache(), tokens=5, q_heads=4, rotary_dim=64, norm=1,
             eps=1e-6)
    return kh.QkNormRope(**{**f, **kw})


def attention(**kw):
    f = dict(cache=cache(), table=table(), q=16, out=32, lse=4, q_starts=4, q_stride=256, out_stride=256, tokens=5,
             q_heads=4, window=0, scale=0.125)
    return kh.PagedAttention(**{**f, **kw})


def weights(**kw):
    f = dict(cache=cache(), table=table(), q=16, lse=4, q_starts=4, q_stride=256, weights_in=4, weights=8,
             weights_seq_stride=128, weights_head_stride=64, tokens=5, q_heads=4, window=0, scale=0.125)
    return kh.PagedWeights(**{**f, **kw})


def evict(**kw):
    f = dict(cache=cache(), table=table(), kept_pages=4, kept_row_stride=3, kept_width=3, kept_lens=8, weights_in=16,
             in_seq_stride=128, in_head_stride=64, weights=32, seq_stride=96, head_stride=48, budget=40, recent=8)
    return kh.PagedEvict(**{**f, **kw})


BAD_ROWS = [dict(dtype=3), dict(dtype=-1), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(kv_heads=0),
            dict(kv_heads=65536)]
BAD_CACHE = BAD_ROWS + [
    dict(k=None), dict(v=None), dict(pages=0), dict(pages=1 << 31), dict(page_size=0), dict(page_size=(1 << 20) + 1),
    dict(k=(1 << 20) + 8), dict(v=(1 << 20) + 2), dict(k_page_stride=-64), dict(v_slot_stride=-8),
    dict(k_head_stride=60), dict(v_page_stride=2049), dict(k_slot_stride=1 << 60), dict(k_page_stride=1 << 56),
    dict(v_page_stride=1 << 31)]
BAD_WRITTEN = [dict(k_page_stride=0), dict(v_slot_stride=56), dict(k_head_stride=8)]
BAD_TABLE = [dict(pages=None), dict(lens=None), dict(seqs=0), dict(seqs=-1), dict(width=0), dict(width=1 << 31),
             dict(row_stride=-1), dict(seqs=1 << 20), dict(max_len=-1)]
BAD_QUERIES = [dict(q=None), dict(q_starts=None), dict(tokens=0), dict(q_heads=0), dict(q_heads=5), dict(q_heads=65538),
               dict(q=8), dict(q_stride=-256), dict(q_stride=255), dict(window=-1), dict(window=1 << 31),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(tokens=1 << 30), dict(tokens=1 << 40)]


def refused(call, op):
    with pytest.raises(kh.KhrtError) as e:
        call()
    assert e.value.code == kh.KHRT_E_INVALID and e.value.message.startswith(op + ": "), e.value.message


@pytest.mark.parametrize("kw", BAD_CACHE + BAD_WRITTEN, ids=str)
def test_rope_refuses_caches(kw):
    refused(lambda: kh.qk_norm_rope(rope(cache=cache(**kw)) if kw != dict(k=None) else
                                    rope(cache=cache(**kw), k_out=None)), "qk_norm_rope")


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(slots=None), dict(positions=None), dict(inv_freq=None),
    dict(rotary_dim=-8), dict(rotary_dim=72), dict(rotary_dim=12), dict(eps=-1.0), dict(eps=float("nan")), dict(q=8),
    dict(k_out=8), dict(q_gamma=8), dict(v=50), dict(q_stride=-8), dict(k_stride=100), dict(v_stride=9),
    dict(q_out_stride=128), dict(k_out_stride=64), dict(tokens=0), dict(q_heads=0), dict(q_heads=65536), dict(tokens=1 << 40),
    dict(q_out=16, q_out_stride=512), dict(k_out=32, k_out_stride=256)], ids=str)
def test_rope_refuses(kw):
    refused(lambda: kh.qk_norm_rope(rope(**kw)), "qk_norm_rope")


@pytest.mark.parametrize("kw", BAD_ROWS, ids=str)
def test_rope_without_a_cache_refuses(kw):
    refused(lambda: kh.qk_norm_rope(rope(cache=kh.PagedCache(**{**dict(kv_heads=2, head_dim=64, dtype=1), **kw}))),
            "qk_norm_rope")


@pytest.mark.parametrize("make,call,op", [
    (attention, kh.paged_attention, "paged_attention"), (attention, kh.paged_attention_workspace, "paged_attention_workspace"),
    (weights, kh.paged_weights, "paged_weights")], ids=["attention", "workspace", "weights"])
def test_attention_and_weights_refuse(make, call, op):
    for kw in BAD_CACHE:
        refused(lambda: call(make(cache=cache(**kw))), op)
    for kw in BAD_TABLE:
        refused(lambda: call(make(table=table(**kw))), op)
    for kw in BAD_QUERIES:
        refused(lambda: call(make(**kw)), op)


@pytest.mark.parametrize("kw", [dict(out=None), dict(out=8), dict(out_stride=248), dict(out_stride=-1), dict(out_stride=257),
                                dict(out=16)], ids=str)
def test_attention_refuses(kw):
    refused(lambda: kh.paged_attention(attention(**kw)), "paged_attention")


def test_attention_refuses_a_misaligned_workspace():
    refused(lambda: kh.paged_attention(attention(), 24, 1 << 20), "paged_attention")


@pytest.mark.parametrize("kw", [dict(lse=None), dict(weights=None), dict(weights_seq_stride=-1), dict(weights_head_stride=0),
                                dict(weights_seq_stride=0), dict(weights_head_stride=1 << 41), dict(q_stride=1 << 23)], ids=str)
def test_weights_refuse(kw):
    refused(lambda: kh.paged_weights(weights(**kw)), "paged_weights")


@pytest.mark.parametrize("kw", [
    dict(kept_pages=None), dict(kept_lens=None), dict(weights_in=None), dict(weights=None), dict(budget=0), dict(budget=-1),
    dict(budget=1 << 30, kept_width=1 << 28, seq_stride=1 << 32, head_stride=1 << 31),
    dict(recent=-1), dict(recent=41), dict(kept_width=0), dict(kept_row_stride=2), dict(kept_row_stride=-1), dict(budget=49),
    dict(kept_pages=1 << 12), dict(kept_lens=2 << 12), dict(weights=16), dict(seq_stride=39), dict(head_stride=39),
    dict(in_seq_stride=-1), dict(in_head_stride=-1)], ids=str)
def test_evict_refuses(kw):
    for call, op in ((lambda a: kh.paged_evict(a, 16, 1 << 20), "paged_evict"),
                     (kh.paged_evict_workspace, "paged_evict_workspace")):
        refused(lambda: call(evict(**kw)), op)


def test_evict_refuses_caches_tables_and_workspaces():
    for kw in BAD_CACHE + BAD_WRITTEN:
        refused(lambda: kh.paged_evict(evict(cache=cache(**kw)), 16, 1 << 20), "paged_evict")
    for kw in BAD_TABLE:
        refused(lambda: kh.paged_evict(evict(table=table(**kw)), 16, 1 << 20), "paged_evict")
    need = kh.paged_evict_workspace(evict())
    assert need == 3 * 2 * 40 * 4
    refused(lambda: kh.paged_evict(evict(), None, need), "paged_evict")
    refused(lambda: kh.paged_evict(evict(), 16, need - 1), "paged_evict")
    refused(lambda: kh.paged_evict(evict(), 24, need), "paged_evict")


def test_null_arguments():
    for fn, args in ((kh.lib.kh_qk_norm_rope, (None, None)), (kh.lib.kh_paged_attention, (None, None, 0, None)),
                     (kh.lib.kh_paged_weights, (None, None)), (kh.lib.kh_paged_evict, (None, None, 0, None)),
                     (kh.lib.kh_paged_attention_workspace, (None, None)), (kh.lib.kh_paged_evict_workspace, (None, None))):
        assert fn(*args) == kh.KHRT_E_INVALID and kh.last_error()


def test_workspace_of_attention():
    """Nothing where no sequence is long enough to be shared out; otherwise two
    parts of 16 fp32 rows and their statistics for each workgroup."""
    assert kh.paged_attention_workspace(attention(table=table(seqs=4096, width=4), tokens=4096)) == 0
    n = kh.paged_attention_workspace(attention(table=table(seqs=1, width=8192), tokens=1))
    assert n > 0 and n % (2 * 16 * (64 + 2) * 4) == 0
    assert kh.paged_attention_workspace(attention(table=table(seqs=1, width=8192), tokens=1, window=100)) == 0


def test_structures_match_the_header(tmp_path):
    """The binding's structures have the C compiler's sizes and offsets."""
    structs = {"kh_paged_cache": kh.PagedCache, "kh_page_table": kh.PageTable, "kh_qk_norm_rope_args": kh.QkNormRope,
               "kh_paged_attention_args": kh.PagedAttention, "kh_paged_weights_args": kh.PagedWeights,
               "kh_paged_evict_args": kh.PagedEvict}
    lines = [f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in s._fields_)
             for c, s in structs.items()]
    src = tmp_path / "sizes.c"
    src.write_text('#include "khrt.h"\n#include <stdio.h>\nint main(void) {' + "\n".join(lines) + "return 0;}")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True, timeout=60)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True, timeout=60).stdout.split()]
    want = [x for s in structs.values() for x in [ctypes.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]]
    assert got == want
