"""64-bit definitions of the text-decoder operators, for the GPU parity tests (numpy, CPU)."""
import math

import numpy as np
import torch

F8 = torch.float8_e4m3fn


def e4m3_values(codes):
    """e4m3 codes (uint8 array) as float64."""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * np.exp2(e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


def e4m3_round(v):
    """float64 to the nearest e4m3 value (ties to even), saturating; NaN stays."""
    v = np.asarray(v, np.float64)
    a = np.minimum(np.abs(v), 448.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6)
    step = np.exp2(e - 3)
    return np.copysign(np.where(np.isnan(v), np.nan, np.rint(a / step) * step), v)


def pow2_scale(amax):
    """The smallest power of two s >= 2^-126 with 448 s >= amax."""
    s = 2.0 ** -126
    if amax > 0:
        s = max(s, 2.0 ** (math.frexp(amax)[1] - 10))
        while 448 * s < amax:
            s *= 2
    return s


def plan(past, fresh, free, head, table, T, rows, max_blocks, blocks):
    R = len(past)
    table = [list(t) for t in table]
    cu, slots, pos, kv = [0], [-1] * rows, [-1] * rows, []
    taken = placed = refused = off = total = 0
    for r in range(R):
        p, f = past[r], fresh[r]
        g = max(f, 0)
        end = p + f
        fits = p >= 0 and f >= 0 and not (f and total + f > rows) and end <= max_blocks * T
        need = -(-end // T) - -(-p // T) if fits else 0
        ok = fits and (need == 0 or off + need <= len(free) - head)
        held = -(-p // T) if p >= 0 else 0
        if ok:
            for i in range(need):
                table[r][held + i] = free[head + off + i]
            taken = max(taken, off + need) if need else taken
            placed += f
        else:
            refused += 1
        off += need
        for j in range(g):
            n = total + j
            if n >= rows:
                break
            if p >= 0:
                pos[n] = p + j
            if ok:
                b = table[r][(p + j) // T]
                slots[n] = b * T + (p + j) % T if 0 <= b < blocks else -1
        kv.append(p + f if ok else p)
        total += g
        cu.append(min(total, rows))
    return table, kv, cu, slots, pos, [taken, placed, refused, total], head + taken


def append(x, slots, codes, scales, T):
    """x [rows, heads, dim] float64; codes [blocks, heads, T, dim] uint8 -> values of the codes
    (float64, in units of the scale) and scales, both updated."""
    val, sc = e4m3_values(codes), scales.astype(np.float64).copy()
    pool = codes.shape[0] * T
    i = 0
    while i < len(slots):
        s = slots[i]
        if not 0 <= s < pool:
            i += 1
            continue
        n = 1
        while i + n < len(slots) and slots[i + n] == s + n and (s + n) // T == s // T:
            n += 1
        b, off = divmod(s, T)
        for h in range(codes.shape[1]):
            t = x[i:i + n, h]
            a = np.abs(t[np.isfinite(t)])
            scale = pow2_scale(a.max() if a.size else 0.0)
            if off:
                scale = max(scale, sc[b, h])
                if scale > sc[b, h]:
                    val[b, h, :off] = e4m3_round(val[b, h, :off] * (sc[b, h] / scale))
            val[b, h, off:off + n] = e4m3_round(t / scale)
            sc[b, h] = scale
        i += n
    return val, sc


def attention(q, codes_k, ks, codes_v, vs, table, lens, cu, T, causal, window, scale):
    """-> out, lse and the bounds' ingredients: mean |v| under the weights, largest sum |q||k|."""
    n, hq, d = q.shape
    hk = ks.shape[1]
    out, lse = np.zeros((n, hq, d)), np.full((n, hq), -np.inf)
    mag, big = np.zeros((n, hq, d)), np.zeros((n, hq))
    for r in range(len(lens)):
        kv, nq = lens[r], cu[r + 1] - cu[r]
        if not nq or not kv:
            continue
        ids = [table[r][j // T] for j in range(kv)]
        good = np.array([0 <= b < ks.shape[0] for b in ids])
        ids = np.where(good, ids, 0)
        off = np.arange(kv) % T
        for h in range(hq):
            g = h // (hq // hk)
            k = e4m3_values(codes_k[ids, g, off]) * ks[ids, g][:, None]
            v = e4m3_values(codes_v[ids, g, off]) * vs[ids, g][:, None]
            for i in range(nq):
                p = kv - nq + i
                see = good.copy()
                if causal:
                    see &= np.arange(kv) <= p
                    if window:
                        see &= np.arange(kv) > p - window
                if not see.any():
                    continue
                qi, row = q[cu[r] + i, h], cu[r] + i
                s = scale * (k[see] @ qi)
                m = s.max()
                w = np.exp(s - m)
                out[row, h] = w @ v[see] / w.sum()
                mag[row, h] = w @ np.abs(v[see]) / w.sum()
                big[row, h] = scale * (np.abs(k[see]) @ np.abs(qi)).max()
                lse[row, h] = m + np.log(w.sum())
    return out, lse, mag, big
