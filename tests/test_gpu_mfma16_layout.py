"""In-bounds check of the 16-bit matrix instructions' lane layouts and of the
transposing LDS read, as the sequence-cache kernels are written against them
(one wavefront, one instruction each):

v_mfma_f32_16x16x32_f16  A: lane l holds A[l % 16][8 (l / 16) + i], B alike
                         D: lane l, register r holds D[4 (l / 16) + r][l % 16]
v_mfma_f32_32x32x16_f16  A: lane l holds A[l % 32][8 (l / 32) + i], B alike
                         D: D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32]
ds_read_b64_tr_b16       of the 4 x 16 values that lanes 16 g .. 16 g + 15 point
                         at (lane 4 r + c: row r, columns 4 c ..), lane i of
                         them receives column i, its rows in order
"""
import os

import numpy as np
import pytest

import kernelh as kh
from khtest import say

pytestmark = pytest.mark.gpu


def _run(fn, a, b, out_dtype, count):
    with open(os.path.join(kh.CO_DIR, "mfma16_probe.hsaco"), "rb") as f:
        m = kh.GpuModule(f.read())
    da, db, out = kh.Buffer.from_array(a), kh.Buffer.from_array(b), kh.Buffer(count * np.dtype(out_dtype).itemsize)
    args = kh.LaunchArgs()
    for buf in (da, db, out):
        args.slots.append(buf.ptr)
    say(f"probe {fn}")
    kh.launch_raw(m.get_function(fn), (1, 1, 1), (64, 1, 1), args)
    kh.synchronize()
    return out.to_host(out_dtype, count)


@pytest.mark.parametrize("n,k", [(16, 32), (32, 16)])
def test_mfma_f16(dev, n, k):
    rng = np.random.default_rng(n)
    A, B = (rng.integers(-8, 9, (n, k)).astype(np.float16) for _ in "ab")  # exact in any order
    lane = np.arange(64)
    idx = 8 * (lane // n)[:, None] + np.arange(8)
    a, b = A[(lane % n)[:, None], idx], B[(lane % n)[:, None], idx]
    regs = n * n // 64
    got = _run(f"probe_mfma_{n}x{n}x{k}_f16", a, b, np.float32, 64 * regs).reshape(64, regs)
    D = A.astype(np.float64) @ B.astype(np.float64).T
    r = np.arange(regs)
    row = 4 * (lane // 16)[:, None] + r if n == 16 else 8 * (r // 4) + 4 * (lane // 32)[:, None] + r % 4
    assert np.array_equal(got, D[row, (lane % n)[:, None]])


def test_read_tr16(dev):
    a = np.arange(256, dtype=np.int16)
    got = _run("probe_read_tr16", a, a, np.int16, 256).reshape(4, 16, 4)
    want = a.reshape(4, 4, 16).transpose(0, 2, 1)  # [group][column][row]
    assert np.array_equal(got, want), got[0]
