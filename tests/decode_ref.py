"""64-bit definitions of the decoder's rotation, 4-bit float and sampling operators, for the GPU parity tests
(numpy, CPU)."""
import math

import numpy as np

from text_ref import e4m3_round, e4m3_values

NV, MX = 0, 1
GROUP = {NV: 16, MX: 32}
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def rotate(x, weight, pos, freqs, sections, rot, interleaved, eps):
    """x [rows, heads, dim] float64, pos [axes, rows], freqs float32 -> rotated, and the values before the turn."""
    y = x.copy()
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight
    axis = np.repeat(np.arange(len(sections)), sections)
    angle = pos[axis].T.astype(np.float64) * freqs.astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    p = rot // 2
    a, b = (np.arange(p) * 2, np.arange(p) * 2 + 1) if interleaved else (np.arange(p), np.arange(p) + p)
    out = y.copy()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    big = np.abs(y)
    big[..., a] = big[..., b] = np.abs(y[..., a]) + np.abs(y[..., b])
    return out, big


def scale_at(rows, groups):
    """Places of the scales [rows, groups] in their bytes."""
    r, g = np.arange(rows)[:, None], np.arange(groups)[None]
    return (r // 128 * -(-groups // 4) + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4


def scale_size(rows, groups):
    return -(-rows // 128) * -(-groups // 4) * 512


def quant(x, fmt, scale):
    """x [rows, cols] float32 -> (codes, one a column, padded to whole groups; scale bytes [rows, groups]; values)."""
    m, n = x.shape
    g = GROUP[fmt]
    k = -(-n // g)
    full = np.zeros((m, k * g), np.float32)
    full[:, :n] = x
    full = full.reshape(m, k, g)
    nan = np.isnan(full).any(-1)
    amax = np.where(np.isfinite(full), np.abs(full), 0).max(-1).astype(np.float32)
    with np.errstate(over="ignore"):
        t = (amax / np.float32(np.float32(6) * np.float32(scale))).astype(np.float32)
    if fmt == NV:
        s = e4m3_round(np.clip(t.astype(np.float64), 2.0 ** -9, 448))
        table = e4m3_values(np.arange(127))
        byte = np.searchsorted(table, s).astype(np.uint8)
        byte[nan] = 127
    else:
        f, e = np.frexp(t.astype(np.float64))
        e = np.where(t > 0, np.where(f == 0.5, e - 1, e), -96)
        e = np.clip(np.where(np.isinf(t), 96, e), -96, 96)
        s = np.exp2(e.astype(np.float64))
        byte = (e + 127).astype(np.uint8)
        byte[nan] = 255
    S = (s.astype(np.float32) * np.float32(scale)).astype(np.float64)[..., None]
    v = np.clip(np.where(nan[..., None], 0, full.astype(np.float64)) / S, -6, 6)
    a = np.abs(v)
    code = np.zeros(a.shape, np.uint8)
    for i, edge in enumerate((E2M1[1:] + E2M1[:-1]) / 2):       # a tie goes to the even code
        code += (a >= edge) if i % 2 else (a > edge)
    val = E2M1[code] * np.where(nan[..., None], np.nan, S)
    val = np.where(np.signbit(v), -val, val)
    code = code + 8 * (np.signbit(v) & ~nan[..., None]).astype(np.uint8)
    return code.reshape(m, k * g), byte, val.reshape(m, k * g)[:, :n]


def values(codes, scales, cols, fmt):
    """float64 [rows, cols] of codes (one a column) and scale bytes [rows, groups]."""
    s = e4m3_values(scales) if fmt == NV else np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    return v[:, :cols] * np.repeat(s, GROUP[fmt], 1)[:, :cols]


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1 + np.exp(-v))


def sample(x, temperature, top_k, top_p, min_p, u):
    """One row of float64 scores -> token, log probability, how many stay, and how near the choice was to another one:
    the least distance of a border from a sum, over the total."""
    ok = ~np.isnan(x) & (x != -np.inf)
    if not ok.any():
        return -1, -math.inf, 0, math.inf
    top = x[ok].max()
    if u is None or not temperature > 0:
        return int(np.flatnonzero(ok & (x == top))[0]), 0.0, 1, math.inf
    d = np.full(x.shape, -np.inf)
    with np.errstate(invalid="ignore"):
        d[ok] = np.where(x[ok] == top, 0.0, (x[ok] - top) / temperature)
    w = np.exp(d)
    order = np.lexsort((np.arange(x.size), np.where(ok, -x, np.inf)))
    order = order[:ok.sum()]
    near = math.inf
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        sums = np.cumsum(w[order])
        want = max(float(np.float32(top_p)), 0) * sums[-1]
        m = max(int((sums < want).sum()), 0)
        near = min(near, np.abs(sums - want).min() / sums[-1]) if want > 0 else near
        order = order[:m + 1]
    if min_p > 0:
        least = min(float(np.float32(min_p)), 1.0)
        gap = np.abs(w[order] - least)
        near = min(near, gap[gap > 0].min() if (gap > 0).any() else math.inf)
        order = order[w[order] >= least]
    order = order[w[order] > 2.0 ** -45]
    by_index = np.sort(order)
    sums = np.cumsum(w[by_index])
    want = min(max(u if u == u else 0.0, 0.0), 1.0) * sums[-1]
    i = min(int((sums <= want).sum()), sums.size - 1)
    if want > 0:
        near = min(near, np.abs(sums - want)[:-1].min() / sums[-1] if sums.size > 1 else math.inf)
    token = int(by_index[i])
    return token, float(d[token] - math.log(sums[-1])), int(order.size), near
