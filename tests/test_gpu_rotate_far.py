"""Rotation at far positions with frequencies of many turns a position, against angles reduced in whole numbers.

Bound: the angle is within 2^-31 of a turn (frequencies up to 2^40 radians a position), its float 2^-26 of one, sine and cosine
2^-22 each: 2^-20 of the pair's magnitudes in all, and one rounding of the result."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from test_gpu_decode import TYPES, f64, half_ulp, ok, stream

pytestmark = pytest.mark.gpu
BITS = 320


def inverse_of_two_pi():
    """2^BITS / (2 pi), by Machin's formula."""
    one = 1 << BITS + 64

    def atan_inverse(x):
        total = term = one // x
        n, sign = 3, -1
        while term:
            term //= x * x
            total += sign * (term // n)
            n, sign = n + 2, -sign
        return total

    pi = 4 * (4 * atan_inverse(5) - atan_inverse(239))
    return (one << BITS) // (2 * pi)


def angles(pos, freqs):
    """[rows, pairs]: pos * freq less whole turns, in radians."""
    inverse, out = inverse_of_two_pi(), np.empty((len(pos), len(freqs)))
    for j, f in enumerate(freqs):
        num, den = float(f).as_integer_ratio()
        for i, p in enumerate(pos):
            turn = int(p) * num * inverse // den % (1 << BITS)
            out[i, j] = turn / (1 << BITS)
    return (out - np.rint(out)) * 2 * math.pi


def test_reduction_itself():
    """On small angles doubles know the answer."""
    pos, freqs = np.arange(4), np.float32([0.5, 1.0, 0.001])
    want = pos[:, None] * freqs.astype(np.float64)
    assert np.abs(np.exp(1j * angles(pos, freqs)) - np.exp(1j * want)).max() < 2.0 ** -50


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("inter", [0, 1])
@pytest.mark.parametrize("size", [1.0, 100.0, 12345.678, 2.0 ** 24 + 2, 1e9, 2.0 ** 40, -3000.7])
def test_rotate_far_and_fast(lib, cuda, size, inter, t):
    from yolo11_cu_b200 import runtime as rt
    dt, code = TYPES[t]
    rows, dim = 200, 64
    g = torch.Generator().manual_seed(7)
    x = torch.randn(rows, dim, generator=g).to(dt).cuda()
    pos = (2 ** 31 - 1 - torch.randint(0, 10 ** 8, (rows,), generator=g)).int()
    pos[:3] = torch.tensor([2 ** 31 - 1, 0, 1])
    freqs = (size * (1 - torch.rand(dim // 2, generator=g) / 2)).float()
    freqs[0] = size
    out, at, by = torch.empty_like(x), pos.cuda(), freqs.cuda()
    a = rt.YkQkRotate(q=x.data_ptr(), q_out=out.data_ptr(), pos=at.data_ptr(), freqs=by.data_ptr(), q_row=dim, q_out_row=dim,
                      rows=rows, heads=1, dim=dim, rot=dim, axes=1, interleaved=inter, dtype=code)
    ok(lib, lib.yk_qk_rotate(C.byref(a), stream()))
    turn = np.exp(1j * angles(pos.tolist(), freqs.tolist()))
    v = f64(x)
    lo, hi = (slice(0, dim, 2), slice(1, dim, 2)) if inter else (slice(0, dim // 2), slice(dim // 2, dim))
    want, big = np.empty_like(v), np.empty_like(v)
    z = (v[:, lo] + 1j * v[:, hi]) * turn
    want[:, lo], want[:, hi] = z.real, z.imag
    big[:, lo] = big[:, hi] = np.abs(v[:, lo]) + np.abs(v[:, hi])
    err = 2.0 ** -20 * big
    fine = np.abs(f64(out) - want) <= half_ulp(dt, np.abs(want) + err) + err
    assert fine.all(), (np.argwhere(~fine)[:5], f64(out)[~fine][:5], want[~fine][:5])
