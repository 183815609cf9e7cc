"""Sampling at the ends of its parameters' and scores' ranges, both kernels and every split, against the 64-bit definition.
Tokens and counts are exact (the inputs keep sums 10^-9 of the total away from borders, which run_sample checks); log
probabilities have run_sample's bound."""
import math

import numpy as np
import pytest
import torch

from test_gpu_decode import TYPES, ok, run_sample

pytestmark = pytest.mark.gpu
INF = math.inf
KERNELS = {"f16": (1, 2), "bf16": (1, 2), "f32": (1,)}


def everywhere(lib, x, t, splits=(1, 2, 4, 8), **kw):
    """run_sample against the definition, by each kernel and split."""
    from yolo11_cu_b200 import runtime as rt
    for kernel in KERNELS[t]:
        for split in splits:
            ok(lib, lib.yk_test_sample_kernel(kernel))
            ok(lib, lib.yk_test_sample(split))
            run_sample(lib, rt, x, **kw)


def u_of(m, seed):
    return torch.rand(m, generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("temperature", [INF, 3e38, 2e37, 1.2e37, 9e36])
@pytest.mark.parametrize("n", [5, 200, 1000, 1300])
def test_flat_temperatures_with_top_p(lib, cuda, n, temperature, t):
    """Scores that a temperature makes equal: what is masked (-infinity, NaN) or behind the row weighs nothing still."""
    g = torch.Generator().manual_seed(n)
    m = 8
    x = torch.randn(m, n, generator=g)
    x[1, 1::2] = -INF                       # masked rows
    x[2, : n - n // 3] = -INF
    x[3, ::3] = math.nan
    x[4, n // 2:] = math.nan
    x[5, 1:] = -INF
    x = x.to(TYPES[t][0])
    wide = torch.zeros(m, n + 9, dtype=x.dtype)
    wide[:, 3:n + 3] = x
    for rows in (x.cuda(), wide.cuda()[:, 3:n + 3]):
        for top_p in (0.9, 0.31, 0.0567):
            everywhere(lib, rows, t, temperature=[temperature] * m, u=u_of(m, n), top_p=[top_p] * m)
        everywhere(lib, rows, t, splits=(1, 8), temperature=[temperature] * m, u=u_of(m, n), top_p=[0.62] * m, top_k=[0, 3, n // 2, n - 1] * 2)
        everywhere(lib, rows, t, splits=(1, 8), temperature=[temperature] * m, u=u_of(m, n), top_p=[0.62] * m, min_p=[0.0, 0.4] * 4)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("temperature", [INF, 3e38, 1e37])
def test_flat_temperatures_of_the_largest_scores(lib, cuda, temperature, t):
    """The type's lowest value beside its largest: their difference is none of the type's, and has a weight still."""
    top = float(torch.finfo(TYPES[t][0]).max)
    x = torch.tensor([[top, -top, 0.0, 1.0] * 5 + [-top] * 7, [1.0, -top, 0.0, -top] * 6 + [top] * 3, [-top] * 20 + [-INF] * 7]).to(TYPES[t][0]).cuda()
    for kw in (dict(top_p=[0.55] * 3), dict(top_k=[13] * 3), dict(top_k=[22, 9, 4], top_p=[0.83] * 3), {}):
        everywhere(lib, x, t, temperature=[temperature] * 3, u=[0.93, 0.4, 0.07], **kw)
    x = torch.full((3, 256), -top).to(TYPES[t][0])
    x[:, 100:120] = top
    for kw in (dict(top_k=[100] * 3), dict(top_k=[256, 37, 20], top_p=[0.83, 0.61, 0.567]), dict(top_p=[0.0567, 0.31, 0.9])):
        everywhere(lib, x.cuda(), t, temperature=[temperature] * 3, u=[0.93, 0.4, 0.0731], **kw)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("temperature", [INF, 5e36, 2e36, 1e36, 1e30, 1.0])
def test_lowest_scores_lead(lib, cuda, temperature, t):
    """Rows of which nothing is above the type's lowest values; those of -infinity and what is behind the row weigh nothing."""
    low = -float(torch.finfo(TYPES[t][0]).max)
    x = torch.full((4, 200), low)
    x[1, 90:] = -INF
    x[2, ::2] = math.nan
    x[3] *= 0.5
    x[3, 7::3] = -INF
    x = x.to(TYPES[t][0]).cuda()
    for kw in (dict(top_p=[0.9] * 4), dict(top_p=[0.31] * 4, top_k=[0, 70, 0, 55]), dict(top_k=[90, 89, 1, 60])):
        everywhere(lib, x, t, temperature=[temperature] * 4, u=[0.93, 0.41, 0.0731, 0.62], **kw)


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_infinite_scores_beside_every_nan(lib, cuda, t):
    """The NaN next to infinity in the order of codes (and all others) are scores of no weight, also where infinity leads."""
    inf = {"f16": 0x7c00, "bf16": 0x7f80}[t]
    nans = np.concatenate([inf + np.arange(1, 12), 0x8000 + inf + np.arange(1, 12), [0x7fff, 0xffff, inf + 0x40]]).astype(np.uint16)
    rows = []
    for lead in ([inf] * 3, [inf], [0x3c00, 0x3c00, 0x2000], [0x8000 + inf - 1] * 2):
        row = np.zeros(100, np.uint16)
        row[:nans.size] = nans
        row[nans.size:] = 0x8000 + inf                      # -infinity
        row[60:60 + len(lead)] = lead
        row[2:5], row[80:83] = row[80:83].copy(), row[2:5].copy()
        rows.append(row)
    x = torch.from_numpy(np.stack(rows).view(np.int16)).view(TYPES[t][0]).cuda()
    m = len(rows)
    for u in (0.0, 0.4, 0.9):
        for k in (1, 2, 3, 5, 99):
            everywhere(lib, x, t, u=[u] * m, top_k=[k] * m)
            everywhere(lib, x, t, splits=(1, 8), u=[u] * m, top_k=[k] * m, top_p=[0.55] * m)
        everywhere(lib, x, t, splits=(1, 8), u=[u] * m, top_p=[0.3] * m)
        everywhere(lib, x, t, splits=(1, 8), u=[u] * m, min_p=[0.5] * m)
