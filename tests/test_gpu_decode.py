"""GPU parity of the decoder's rotation, 4-bit float and sampling operators against their 64-bit definitions
(decode_ref.py).

Bounds.  One rounding of a result is at most eps / 2 of it (2^-11 fp16, 2^-8 bf16; below the smallest normal fp16
2^-25).  Rotation: norm, cosine, sine and products in 32 bits, 2^-20 of the magnitudes that meet in a channel
(a sum of squares: 8 roundings, rsqrt and the angle 2^-22 each).  Quantisation is exact.  Products: a sum
of K exact products in 32 bits, whose steps of 64 lose at most 2^-22 of the magnitudes so far: (K / 64 + 8) 2^-22 of the sum of
magnitudes.  Sampling: tokens are exact unless a sum comes within 10^-9 of the total of a border, which the inputs
are checked to avoid; log probabilities are rounded once to 32 bits, and 2^-44 n off before."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import decode_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"f16": (torch.float16, 0), "bf16": (torch.bfloat16, 1), "f32": (torch.float32, 3)}


@pytest.fixture(autouse=True)
def the_librarys_rules(lib):
    yield
    lib.yk_test_gemm_fp4(0, 0)
    lib.yk_test_sample(0)


def half_ulp(dt, v):
    return torch.finfo(dt).eps / 2 * np.abs(v) + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -134)


def ok(lib, code):
    assert code == 0, (code, lib.yk_last_cuda_error())


def stream():
    return torch.cuda.current_stream().cuda_stream


def f64(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------------- rotate

def run_rotate(lib, rt, *, rows, heads, kv, dim, rot, axes=1, inter=False, norm=True, t="f16", place="apart", gap=0, seed=0,
               far=300000, hidden=()):
    dt, code = TYPES[t]
    g = torch.Generator(device="cuda").manual_seed(seed)
    row = (heads + 2 * kv) * dim + gap
    x = (torch.randn(rows + 1, row, generator=g, device="cuda") * 3).to(dt)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g, device="cuda")).to(dt) for _ in range(2))
    pos = torch.randint(0, far, (axes, rows + 2), generator=g, device="cuda", dtype=torch.int32)
    pos[0, list(hidden)] = -1
    freqs = (10000.0 ** (-2 * torch.arange(rot // 2, dtype=torch.float64) / rot)).float().cuda()
    sections = [rot // 2, 0, 0, 0] if axes == 1 else [rot // 2 - (axes - 1) * 3] + [3] * (axes - 1) + [0] * (4 - axes)
    q, k = x[:rows, :heads * dim], x[:rows, heads * dim:(heads + kv) * dim]
    q0, k0 = (f64(v).reshape(rows, -1, dim) for v in (q, k))
    if place == "apart":
        out = torch.full((rows + 1, row + 8), 7.0, dtype=dt, device="cuda")
        qo, ko, orow = out[:, :heads * dim], out[:, heads * dim:], row + 8
        kept_q, kept_k = np.full_like(q0, 7), np.full_like(k0, 7)
    else:
        qo, ko, orow = q, k, row
        kept_q, kept_k = q0, k0
    rest = x[:, (heads + kv) * dim:].clone(), x[rows].clone()
    a = rt.YkQkRotate(q=q.data_ptr(), k=k.data_ptr() if kv else None, q_out=qo.data_ptr(), k_out=ko.data_ptr() if kv else None,
                      q_weight=wq.data_ptr() if norm else None, k_weight=wk.data_ptr() if norm else None, pos=pos.data_ptr(),
                      freqs=freqs.data_ptr(), q_row=row, k_row=row, q_out_row=orow, k_out_row=orow, pos_axis=rows + 2,
                      rows=rows, heads=heads, kv_heads=kv, dim=dim, rot=rot, axes=axes, sections=(C.c_int * 4)(*sections),
                      interleaved=inter, dtype=code, eps=1e-6)
    ok(lib, lib.yk_qk_rotate(C.byref(a), stream()))
    assert torch.equal(x[:, (heads + kv) * dim:], rest[0]) and torch.equal(x[rows], rest[1])
    for x0, got, w, kept in ((q0, qo, wq, kept_q), (k0, ko, wk, kept_k)):
        n = x0.shape[1]
        if not n:
            continue
        want, big = ref.rotate(x0, f64(w) if norm else None, pos[:, :rows].cpu().numpy(), freqs.cpu().numpy(),
                               sections[:axes], rot, inter, 1e-6)
        have = f64(got[:rows, :n * dim]).reshape(rows, n, dim)
        bound = half_ulp(dt, np.abs(want) + 2.0 ** -20 * big) + 2.0 ** -20 * big
        fine = np.abs(have - want) <= bound
        fine[list(hidden)] = have[list(hidden)] == kept[list(hidden)]
        assert fine.all(), (np.argwhere(~fine)[:5], have[~fine][:5], want[~fine][:5])
    if place == "apart":
        assert (out[:, (heads + kv) * dim:] == 7).all() and (out[rows] == 7).all()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("dim,rot", [(32, 16), (64, 64), (64, 48), (128, 128), (128, 64), (256, 256), (256, 16)])
@pytest.mark.parametrize("inter", [False, True])
def test_rotate(lib, cuda, dim, rot, inter, t):
    from yolo11_cu_b200 import runtime as rt
    run_rotate(lib, rt, rows=37, heads=6, kv=2, dim=dim, rot=rot, inter=inter, t=t)
    run_rotate(lib, rt, rows=5, heads=3, kv=1, dim=dim, rot=rot, inter=inter, t=t, norm=False, place="same", gap=8)


@pytest.mark.parametrize("axes", [2, 3, 4])
@pytest.mark.parametrize("place", ["apart", "same"])
def test_rotate_axes(lib, cuda, axes, place):
    from yolo11_cu_b200 import runtime as rt
    run_rotate(lib, rt, rows=50, heads=4, kv=4, dim=64, rot=64, axes=axes, place=place, hidden=[0, 7, 49], t="bf16")


@pytest.mark.parametrize("rows,heads,kv", [(1, 1, 0), (1, 1, 1), (3000, 1, 1), (2, 700, 324), (1201, 7, 1), (4097, 32, 8)])
def test_rotate_sizes(lib, cuda, rows, heads, kv):
    from yolo11_cu_b200 import runtime as rt
    run_rotate(lib, rt, rows=rows, heads=heads, kv=kv, dim=64 if heads > 8 else 128, rot=32, seed=rows, place="same")


def test_rotate_far_positions(lib, cuda):
    """Angles of up to 2^31 radians: their turns are taken off in 64 bits."""
    from yolo11_cu_b200 import runtime as rt
    run_rotate(lib, rt, rows=64, heads=2, kv=1, dim=64, rot=64, far=2 ** 31 - 1)


def test_rotate_keeps_infinities_to_their_pair(lib, cuda):
    from yolo11_cu_b200 import runtime as rt
    x = torch.ones(2, 1, 64, device="cuda", dtype=torch.float16)
    x[0, 0, 3] = float("nan")
    x[1, 0, 40] = float("inf")
    pos, freqs = torch.ones(2, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")
    a = rt.YkQkRotate(q=x.data_ptr(), q_out=x.data_ptr(), pos=pos.data_ptr(), freqs=freqs.data_ptr(), q_row=64, q_out_row=64,
                      rows=2, heads=1, dim=64, rot=64, axes=1)
    ok(lib, lib.yk_qk_rotate(C.byref(a), stream()))
    bad = ~torch.isfinite(x[:, 0])
    assert bad[0].nonzero().flatten().tolist() == [3, 35] and bad[1].nonzero().flatten().tolist() == [8, 40]


# ---------------------------------------------------------------- 4-bit floats

def pitch(cols):
    return -(-(-(-cols // 2)) // 16) * 16


def run_quant(lib, rt, x, fmt, scale, code, dt, want_values=True, x_row=None):
    m, n = x.shape
    g = -(-n // ref.GROUP[fmt])
    size = lib.yk_fp4_scale_bytes(m, n, fmt)
    assert size == ref.scale_size(m, g)
    codes = torch.full((m + 1, pitch(n) + 16), 0x99, dtype=torch.uint8, device="cuda")
    scales = torch.full((size + 16,), 0x77, dtype=torch.uint8, device="cuda")
    vals = torch.full((m + 1, n + 3), 5.0, dtype=dt, device="cuda")
    a = rt.YkQuantFp4(x=x.data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr(),
                      values=vals.data_ptr() if want_values else None, x_row=x.stride(0), values_row=n + 3,
                      codes_row=pitch(n) + 16, rows=m, cols=n, format=fmt, dtype=code, scale=scale)
    ok(lib, lib.yk_quant_fp4(C.byref(a), stream()))
    q, sb, v = ref.quant(x.float().cpu().numpy(), fmt, scale or 1.0)
    eight = -(-n // 8) * 4
    c = codes.cpu().numpy()
    full = np.zeros((m, 2 * eight), np.uint8)
    full[:, :n] = q[:, :n]
    assert np.array_equal(c[:m, :eight], full[:, 0::2] | full[:, 1::2] << 4)
    assert (c[:m, eight:] == 0x99).all() and (c[m] == 0x99).all()
    want = np.zeros(size, np.uint8)
    want[ref.scale_at(m, g)] = sb
    s = scales.cpu().numpy()
    assert np.array_equal(s[:size], want) and (s[size:] == 0x77).all()
    if want_values:
        got = vals.cpu()
        assert (got[:, n:] == 5).all() and (got[m] == 5).all()
        assert np.array_equal(got[:m, :n].double().numpy(), torch.from_numpy(v).float().to(dt).double().numpy(), equal_nan=True)
    return codes, scales


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 17), (5, 255), (130, 64), (129, 257), (33, 1000), (300, 776)])
def test_quant(lib, cuda, rows, cols, t, fmt):
    from yolo11_cu_b200 import runtime as rt
    dt, code = TYPES[t]
    g = torch.Generator(device="cuda").manual_seed(rows * cols)
    x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(2 * torch.randn(rows, cols, generator=g, device="cuda"))
    run_quant(lib, rt, x.to(dt), fmt, 0.0, code, dt)
    run_quant(lib, rt, (x * 1e-3).to(dt), fmt, 0.003, code, dt)
    wide = torch.zeros(rows, cols + 5, dtype=dt, device="cuda")      # rows off any 16-byte boundary
    wide[:, 1:cols + 1] = x.to(dt)
    run_quant(lib, rt, wide[:, 1:cols + 1], fmt, 0.5, code, dt, want_values=rows % 2 == 1)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_quant_borders(lib, cuda, fmt, t):
    """Values halfway between codes, of every scale; zeros, subnormals, the largest, infinities and NaN."""
    from yolo11_cu_b200 import runtime as rt
    dt, code = TYPES[t]
    mid = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0]
    rows = []
    for s in [1, 1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875, 2 ** -9, 448, 2.0 ** -14, 3 * 2.0 ** -20]:
        base = torch.tensor((mid + [6.0, 0.0]) * 2, dtype=torch.float64) * s
        rows += [base, torch.nextafter(base.float(), torch.tensor(9e9)).double() * (1 + 2.0 ** -8), base * (1 - 2.0 ** -8)]
    top = float(torch.finfo(dt).max)
    inf, nan = math.inf, math.nan
    special = [[0.0] * 32, [top] * 32, [-top] + [1.0] * 31, [inf] * 32, [inf, -inf, 1.0, 3.0] * 8, [nan] * 32,
               [nan] + [2.0] * 31, [2.0] * 20 + [nan] + [inf] * 11, [float(torch.finfo(dt).tiny) / 4] * 32, [-0.0] * 32]
    rows += [torch.tensor(r, dtype=torch.float64) for r in special]
    x = torch.stack(rows).to(dt).cuda()
    for scale in (0.0, 2.0 ** -6, 0.3, 2.0 ** 30, 2.0 ** -30):
        run_quant(lib, rt, x, fmt, scale, code, dt)


def random_matrix(rows, cols, fmt, gen, dt, size=1.0):
    """Codes and scales of a random matrix as the library takes them, and their 64-bit values."""
    x = torch.randn(rows, cols, generator=gen) * torch.exp(0.7 * torch.randn(rows, cols, generator=gen)) * size
    q, sb, _ = ref.quant(x.numpy(), fmt, 1.0)
    full = np.zeros((rows, 2 * pitch(cols)), np.uint8)
    full[:, :cols] = q[:, :cols]
    packed = full[:, 0::2] | full[:, 1::2] << 4
    g = sb.shape[1]
    scales = np.zeros(ref.scale_size(rows, g), np.uint8)
    scales[ref.scale_at(rows, g)] = sb
    return torch.from_numpy(packed).cuda(), torch.from_numpy(scales).cuda(), ref.values(q, sb, cols, fmt)


def run_gemm(lib, rt, m, n, k, fmt, t="f16", gated=False, bias=False, alpha=0.0, seed=0, matrices=None):
    dt, code = TYPES[t]
    gen = torch.Generator().manual_seed(seed)
    mats = matrices or [random_matrix(r, k, fmt, gen, dt, s) for r, s in ((m, 1.0), (n, 0.1)) + (((n, 0.1),) if gated else ())]
    b = torch.randn(n, generator=gen).cuda() if bias else None
    yrow = n + 5 if seed % 2 else -(-n // 8) * 8
    y = torch.full((m + 1, yrow), 9.0, dtype=dt, device="cuda")
    p = lambda i, j: mats[i][j].data_ptr() if i < len(mats) else None  # noqa: E731
    a = rt.YkGemmFp4(x=p(0, 0), xscale=p(0, 1), w=p(1, 0), wscale=p(1, 1), w2=p(2, 0), w2scale=p(2, 1),
                     bias=b.data_ptr() if bias else None, y=y.data_ptr(), x_row=mats[0][0].stride(0), w_row=mats[1][0].stride(0),
                     y_row=yrow, rows=m, n=n, k=k, format=fmt, dtype=code, alpha=alpha, alpha2=2 * alpha)
    ok(lib, lib.yk_gemm_fp4(C.byref(a), stream()))
    assert lib.yk_fetch_device_error() == 0
    al, al2 = (float(np.float32(alpha)), float(np.float32(2 * alpha))) if alpha else (1.0, 1.0)
    x, w = mats[0][2], mats[1][2]
    slack = (k / 64 + 8) * 2.0 ** -22
    want = x @ w.T * al
    err = slack * (np.abs(x) @ np.abs(w).T) * abs(al) + 2.0 ** -23 * np.abs(want)
    if bias:
        want = want + f64(b)
        err += 2.0 ** -23 * np.abs(want)
    if gated:
        u = x @ mats[2][2].T * al2
        eu = slack * (np.abs(x) @ np.abs(mats[2][2]).T) * abs(al2) + 2.0 ** -23 * np.abs(u)
        g, eg = want, err
        # silu's slope is below 1.1; its exponential is within 2^-21 + |g| 2^-23
        es = 1.1 * eg + np.abs(ref.silu(g)) * (2.0 ** -20 + np.abs(g) * 2.0 ** -22)
        want = ref.silu(g) * u
        err = es * np.abs(u) + np.abs(ref.silu(g)) * eu + es * eu + 2.0 ** -23 * np.abs(want)
    got = f64(y[:m, :n])
    fine = np.abs(got - want) <= half_ulp(dt, np.abs(want) + err) + err
    fine |= np.isnan(want) & np.isnan(got)
    assert fine.all(), (np.argwhere(~fine)[:5], got[~fine][:5], want[~fine][:5], err[~fine][:5])
    assert (y[:m, n:] == 9).all() and (y[m] == 9).all()
    return y[:m, :n]


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("kernel,split", [(1, 0), (2, 1), (2, 2), (2, 4), (2, 8), (0, 0)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 130, 2048), (17, 129, 300), (33, 384, 257), (128, 128, 256), (130, 300, 2113),
                                   (257, 65, 64), (300, 520, 96)])
def test_gemm(lib, cuda, m, n, k, kernel, split, fmt):
    from yolo11_cu_b200 import runtime as rt
    ok(lib, lib.yk_test_gemm_fp4(kernel, split))
    run_gemm(lib, rt, m, n, k, fmt, seed=m + k, bias=n % 2 == 0, alpha=0.25 if n > 200 else 0.0, t="bf16" if k % 2 else "f16")


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("kernel,split", [(1, 0), (2, 1), (2, 4), (0, 0)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 33), (9, 200, 1100), (40, 128, 512), (129, 260, 770), (300, 129, 2049)])
def test_gemm_gated(lib, cuda, m, n, k, kernel, split, fmt):
    from yolo11_cu_b200 import runtime as rt
    ok(lib, lib.yk_test_gemm_fp4(kernel, split))
    run_gemm(lib, rt, m, n, k, fmt, seed=m + k, gated=True, alpha=0.5 if n > 200 else 0.0, t="bf16" if n % 2 else "f16")


def test_gemm_many_tiles(lib, cuda):
    """More tiles than SMs, so that a CTA takes several: accumulators by turns, bands of rows."""
    from yolo11_cu_b200 import runtime as rt
    ok(lib, lib.yk_test_gemm_fp4(1, 0))
    run_gemm(lib, rt, 2500, 3900, 200, 0, seed=1)
    run_gemm(lib, rt, 1500, 3900, 130, 1, seed=2, gated=True)
    run_gemm(lib, rt, 2300, 5000, 600, 0, seed=4, t="bf16")


def test_gemm_nan_groups_stay_in_their_row(lib, cuda):
    from yolo11_cu_b200 import runtime as rt
    for fmt in (0, 1):
        for kernel in (1, 2):
            ok(lib, lib.yk_test_gemm_fp4(kernel, 0))
            gen = torch.Generator().manual_seed(3)
            mats = [list(random_matrix(r, 500, fmt, gen, torch.float16)) for r in (140, 150)]
            g = -(-500 // ref.GROUP[fmt])
            at = ref.scale_at(140, g)[131, 3]
            mats[0][1][int(at)] = 127 if fmt == 0 else 255
            lo, hi = 3 * ref.GROUP[fmt], 4 * ref.GROUP[fmt]
            mats[0][2][131, lo:hi] = np.nan
            y = run_gemm(lib, rt, 140, 150, 500, fmt, seed=0, matrices=mats)
            bad = torch.isnan(y)
            assert bad[131].all() and not bad[:131].any() and not bad[132:].any()


def test_gemm_other_rows_scales_do_not_matter(lib, cuda):
    """Scales past the last row and garbage in codes past the last column are not used."""
    from yolo11_cu_b200 import runtime as rt
    for kernel in (1, 2):
        ok(lib, lib.yk_test_gemm_fp4(kernel, 0))
        for fmt in (0, 1):
            gen = torch.Generator().manual_seed(5)
            mats = [list(random_matrix(r, 130, fmt, gen, torch.float16)) for r in (20, 140)]
            g = -(-130 // ref.GROUP[fmt])
            for mat, rows in zip(mats, (20, 140)):
                used = torch.zeros_like(mat[1], dtype=torch.bool)
                whole = -(-g // 4) * 4
                used[torch.from_numpy(ref.scale_at(rows, whole).ravel()).cuda()] = True
                mat[1][~used] = 0xff
                mat[0][:, 65:] = 0x77
            run_gemm(lib, rt, 20, 140, 130, fmt, seed=0, matrices=mats)


def test_linear_of_sixteen_bit_rows(lib, cuda):
    """Rows to 4 bits, then the product, then its rows to 4 bits again: as a feed-forward block runs them."""
    from yolo11_cu_b200 import runtime as rt
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(70, 320, generator=gen).half().cuda()
    codes, scales = run_quant(lib, rt, x, 0, 0.01, 0, torch.float16)
    q, sb, _ = ref.quant(x.float().cpu().numpy(), 0, 0.01)
    mats = [(codes[:70], scales, ref.values(q, sb, 320, 0))] + [random_matrix(96, 320, 0, gen, torch.float16, 0.1) for _ in range(2)]
    y = run_gemm(lib, rt, 70, 96, 320, 0, gated=True, alpha=0.01, matrices=mats)
    run_quant(lib, rt, y, 0, 0.0, 0, torch.float16)


# ---------------------------------------------------------------- sample

def run_sample(lib, rt, x, temperature=None, top_k=None, top_p=None, min_p=None, u=None, check=True, row=None):
    m, n = x.shape
    code = {v[0]: v[1] for v in TYPES.values()}[x.dtype]
    dev = lambda v, d: None if v is None else torch.tensor(v, dtype=d, device="cuda")  # noqa: E731
    t, k, p, mp, uu = dev(temperature, torch.float32), dev(top_k, torch.int32), dev(top_p, torch.float32), dev(min_p, torch.float32), \
        dev(u, torch.float32)
    token, kept = (torch.full((m + 1,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    logprob = torch.full((m + 1,), 3.0, device="cuda")
    ptr = lambda v: None if v is None else v.data_ptr()  # noqa: E731
    a = rt.YkSample(logits=x.data_ptr(), temperature=ptr(t), top_k=ptr(k), top_p=ptr(p), min_p=ptr(mp), u=ptr(uu),
                    token=token.data_ptr(), logprob=logprob.data_ptr(), kept=kept.data_ptr(), row=x.stride(0), rows=m, n=n, dtype=code)
    ok(lib, lib.yk_sample(C.byref(a), stream()))
    out = token.tolist(), logprob.tolist(), kept.tolist()
    assert out[0][m] == -9 and out[1][m] == 3.0 and out[2][m] == -9
    if check:
        scores = f64(x)
        one = lambda v, i, d: d if v is None else v[i].item()  # noqa: E731
        for r in range(m):
            want = ref.sample(scores[r], one(t, r, 1.0), one(k, r, 0), one(p, r, 1.0), one(mp, r, 0.0), one(uu, r, None))
            assert want[3] > 1e-9 * 1.0 or want[3] == 0, "an input whose choice is too near a border"
            if want[3] == 0:
                continue
            assert (out[0][r], out[2][r]) == (want[0], want[2]), (r, out[0][r], want, out[2][r])
            assert math.isclose(out[1][r], want[1], rel_tol=2.0 ** -23, abs_tol=2.0 ** -44 * n) or out[1][r] == want[1]
    return out[0][:m], out[1][:m], out[2][:m]


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("split", [1, 2, 8])
@pytest.mark.parametrize("n", [1, 7, 1000, 5003, 32768])
def test_sample(lib, cuda, n, split, t):
    from yolo11_cu_b200 import runtime as rt
    ok(lib, lib.yk_test_sample(split))
    g = torch.Generator().manual_seed(n)
    m = 24
    x = (torch.randn(m, n, generator=g) * 3).to(TYPES[t][0]).cuda()
    u = torch.rand(m, generator=g).tolist()
    run_sample(lib, rt, x, u=u)
    run_sample(lib, rt, x, temperature=[0.5 + 0.05 * i for i in range(m)], u=u, top_k=[i * 3 for i in range(m)])
    run_sample(lib, rt, x, u=u, top_p=[0.04 * i + 0.05 for i in range(m)])
    run_sample(lib, rt, x, u=u, min_p=[0.01 * i for i in range(m)])
    run_sample(lib, rt, x, temperature=[0.3 * (i % 5) for i in range(m)], top_k=[[0, 40, -3, n + 5][i % 4] for i in range(m)],
               top_p=[[1.0, 0.9, 0.5][i % 3] for i in range(m)], min_p=[[0.0, 0.05][i % 2] for i in range(m)], u=u)


def test_sample_splits_agree(lib, cuda):
    """The same rows alone, in a batch and under every split: the same bits; row strides off any 16 bytes too."""
    from yolo11_cu_b200 import runtime as rt
    g = torch.Generator().manual_seed(4)
    for dt in (torch.float16, torch.bfloat16, torch.float32):
        x = (torch.randn(12, 30001, generator=g) * 2).to(dt).cuda()
        odd = torch.zeros(12, 30010, dtype=dt, device="cuda")
        odd[:, 3:30004] = x
        kw = dict(temperature=[0.9] * 12, top_k=[0, 500, 3000] * 4, top_p=[0.97] * 12, u=torch.rand(12, generator=g).tolist())
        runs = []
        for split in (0, 1, 2, 4, 8):
            ok(lib, lib.yk_test_sample(split))
            runs.append(run_sample(lib, rt, x, **kw, check=split == 0))
            runs.append(run_sample(lib, rt, odd[:, 3:30004], **kw, check=False))
        ok(lib, lib.yk_test_sample(0))
        runs.append(tuple(sum(v, []) for v in zip(*(run_sample(lib, rt, x[i:i + 1], **{k: [w[i]] for k, w in kw.items()}, check=False)
                                                    for i in range(12)))))
        assert all(r == runs[0] for r in runs)


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
def test_sample_ties(lib, cuda, t):
    """Few distinct scores: borders fall among equal ones, of which the lowest indexes stay."""
    from yolo11_cu_b200 import runtime as rt
    g = torch.Generator().manual_seed(6)
    x = torch.randint(0, 4, (16, 3001), generator=g).to(TYPES[t][0]).cuda()
    u = torch.rand(16, generator=g).tolist()
    for split in (1, 4):
        ok(lib, lib.yk_test_sample(split))
        run_sample(lib, rt, x, u=u, top_k=[1, 2, 5, 100, 700, 760, 800, 1500, 2250, 2999, 3000, 3001, 9999, 0, 751, 1503])
        run_sample(lib, rt, x, u=u, top_p=[0.01 + 0.061 * i for i in range(16)])
        run_sample(lib, rt, x, u=u, top_k=[900] * 16, top_p=[0.01 + 0.061 * i for i in range(16)], min_p=[0.0, 0.2] * 8)
    run_sample(lib, rt, torch.zeros(3, 5000, dtype=TYPES[t][0], device="cuda"), u=[0.1234, 0.5, 0.99], top_k=[0, 17, 0], top_p=[1, 1, 0.0101])
    zeros = torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0]] * 4, dtype=TYPES[t][0], device="cuda")
    assert run_sample(lib, rt, zeros, u=[0.1, 0.3, 0.6, 0.9], top_k=[4] * 4)[0] == [0, 1, 2, 3]
    assert run_sample(lib, rt, -zeros[:, :4], temperature=[0.0] * 4)[0] == [0] * 4


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
def test_sample_special_scores(lib, cuda, t):
    from yolo11_cu_b200 import runtime as rt
    dt, inf, nan = TYPES[t][0], math.inf, math.nan
    rows = [[nan, 1, 2, nan], [-inf] * 4, [nan] * 4, [inf, 1, inf, -inf], [nan, inf, inf, inf], [-inf, -inf, 3, -inf],
            [float(torch.finfo(dt).max), float(torch.finfo(dt).min), 0, 0], [-5, -5, nan, -5]]
    x = torch.tensor(rows, dtype=dt, device="cuda")
    for u in (0.0, 0.3, 0.7, 0.999):
        got = run_sample(lib, rt, x, u=[u] * 8)
        assert got[0][1] == got[0][2] == -1 and got[0][5] == 2 and got[0][0] in (1, 2)
        run_sample(lib, rt, x, u=[u] * 8, top_k=[2] * 8)
        run_sample(lib, rt, x, u=[u] * 8, top_p=[0.6] * 8, min_p=[0.1] * 8)
        run_sample(lib, rt, x, u=[u] * 8, temperature=[inf] * 8)
    assert run_sample(lib, rt, x)[0] == [2, -1, -1, 0, 1, 2, 0, 0]
    assert run_sample(lib, rt, x, u=[0.5] * 8, temperature=[nan, 0, -1, 0, 0, 0, 0, 0])[0] == [2, -1, -1, 0, 1, 2, 0, 0]


def test_sample_special_parameters(lib, cuda):
    """Random numbers outside [0, 1), borders at their ends, temperatures near 0."""
    from yolo11_cu_b200 import runtime as rt
    x = torch.randn(6, 2000, generator=torch.Generator().manual_seed(1)).half().cuda()
    top, last = x.argmax(1).tolist(), 1999
    got = run_sample(lib, rt, x, u=[-1.0, math.nan, 0.0, 1.0, math.inf, 7.0], check=False)
    assert got[0] == [0, 0, 0, last, last, last] and got[2] == [2000] * 6
    assert run_sample(lib, rt, x, u=[0.99] * 6, top_p=[0.0, -1.0, 1e-30, 1e-9, 1e-6, -math.inf], check=False)[0] == top
    assert run_sample(lib, rt, x, u=[0.99] * 6, min_p=[1.0, 2.0, math.inf, 1.0, 5.0, 1.0], check=False)[0] == top
    assert run_sample(lib, rt, x, u=[0.99] * 6, temperature=[1e-6, 1e-30, 1e-45, 1e-38, 1e-10, 1e-5], check=False)[0] == top
    got = run_sample(lib, rt, x, u=[0.5] * 6, top_p=[math.nan, 1.0, 2.0, math.inf, 1.0, 1.0], min_p=[math.nan, 0, -1, -math.inf, 0, 0],
                     top_k=[0, -1, -2 ** 31, 2000, 2001, 2 ** 31 - 1], check=False)
    assert got[2] == [2000] * 6


@pytest.fixture
def by_place(lib, cuda):
    """16-bit scores counted by place whatever their number, which only long rows are by themselves."""
    ok(lib, lib.yk_test_sample_kernel(2))
    yield
    ok(lib, lib.yk_test_sample_kernel(0))


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("split", [1, 2, 8])
@pytest.mark.parametrize("n", [1, 7, 1000, 5003, 40001])
def test_sample_by_place(lib, cuda, by_place, n, split, t):
    test_sample(lib, cuda, n, split, t)


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_sample_by_place_ties(lib, cuda, by_place, t):
    test_sample_ties(lib, cuda, t)


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_sample_by_place_special_scores(lib, cuda, by_place, t):
    test_sample_special_scores(lib, cuda, t)


def test_sample_by_place_special_parameters(lib, cuda, by_place):
    test_sample_special_parameters(lib, cuda)


@pytest.mark.parametrize("scale", [0.01, 3.0, 300.0])
def test_sample_kernels_agree(lib, cuda, scale):
    """Bins and places give the same bits: scores around zero (both zeros among them), far from it, in strided rows."""
    from yolo11_cu_b200 import runtime as rt
    g = torch.Generator().manual_seed(8)
    for dt in (torch.float16, torch.bfloat16):
        x = torch.randn(9, 20011, generator=g) * scale
        x[:, ::5] = 0
        x[:, 1::10] = -0.0
        x[3, 7:20000] = -math.inf
        x[4, :19000] = torch.finfo(dt).min
        x[5, 100:] = math.nan
        x = x.to(dt).cuda()
        kw = dict(temperature=[1.0, 0.2, 5.0] * 3, u=torch.rand(9, generator=g).tolist())
        for more in ({}, dict(top_p=[0.9] * 9), dict(top_k=[0, 3, 4000] * 3), dict(top_k=[6000] * 9, top_p=[0.4, 0.99, 1.0] * 3, min_p=[0.0, 0.1, 0.01] * 3)):
            runs = []
            for kernel, split in ((1, 0), (2, 0), (2, 1), (2, 4), (2, 8)):
                ok(lib, lib.yk_test_sample_kernel(kernel))
                ok(lib, lib.yk_test_sample(split))
                runs.append(run_sample(lib, rt, x[:, 2:], **kw, **more, check=False))
            ok(lib, lib.yk_test_sample_kernel(0))
            ok(lib, lib.yk_test_sample(0))
            assert all(r == runs[0] for r in runs), more


def test_sample_counts_of_one_place(lib, cuda):
    """As many equal scores as a CTA can have: a 16-bit count by place stays in its half of a word."""
    from yolo11_cu_b200 import runtime as rt
    for n in (64000, 128000, 262144):
        x = torch.zeros(2, n, dtype=torch.bfloat16, device="cuda")
        x[1] = 1.0078125                          # (an odd place: the upper half)
        for kw in (dict(top_k=[n - 1] * 2), dict(top_p=[0.75] * 2)):
            got = run_sample(lib, rt, x, u=[0.5] * 2, check=False, **kw)
            stay = n - 1 if "top_k" in kw else math.ceil(0.75 * n)
            assert got[2] == [stay] * 2 and got[0] == [stay // 2] * 2


def test_sample_long_rows(lib, cuda):
    from yolo11_cu_b200 import runtime as rt
    g = torch.Generator().manual_seed(9)
    for dt, n in ((torch.float16, 262144), (torch.float32, 262143), (torch.bfloat16, 131073)):
        x = (torch.randn(3, n, generator=g) * 2).to(dt).cuda()
        run_sample(lib, rt, x, u=[0.2, 0.6, 0.9], top_p=[0.9, 1.0, 0.5], top_k=[0, 1000, 0])


# ---------------------------------------------------------------- as a program uses them

def test_captured_and_on_another_stream(lib, cuda):
    """All four in one captured graph on a side stream, replayed with new inputs: what the eager calls give."""
    from yolo11_cu_b200 import runtime as rt
    m, d, n = 24, 64, 500
    gen = torch.Generator().manual_seed(2)
    new = lambda *s, dtype=torch.half: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    qkv, x, u = new(m, 3 * d), new(m, 2 * d), new(m, dtype=torch.float32)
    pos, freqs = torch.arange(m, dtype=torch.int32, device="cuda"), torch.rand(d // 2, generator=gen).cuda()
    codes, scales = new(m, d, dtype=torch.uint8), new(lib.yk_fp4_scale_bytes(m, 2 * d, 0), dtype=torch.uint8)
    w = random_matrix(n, 2 * d, 0, gen, torch.half, 0.1)
    y, token, lp = new(m, n), new(m, dtype=torch.int32), new(m, dtype=torch.float32)
    rot = rt.YkQkRotate(q=qkv.data_ptr(), k=qkv.data_ptr() + 2 * d, q_out=qkv.data_ptr(), k_out=qkv.data_ptr() + 2 * d, pos=pos.data_ptr(),
                        freqs=freqs.data_ptr(), q_row=3 * d, k_row=3 * d, q_out_row=3 * d, k_out_row=3 * d, rows=m, heads=1, kv_heads=1,
                        dim=d, rot=d, axes=1)
    qu = rt.YkQuantFp4(x=x.data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr(), x_row=2 * d, codes_row=d, rows=m, cols=2 * d)
    ge = rt.YkGemmFp4(x=codes.data_ptr(), xscale=scales.data_ptr(), w=w[0].data_ptr(), wscale=w[1].data_ptr(), y=y.data_ptr(), x_row=d,
                      w_row=w[0].stride(0), y_row=n, rows=m, n=n, k=2 * d)
    sa = rt.YkSample(logits=y.data_ptr(), u=u.data_ptr(), token=token.data_ptr(), logprob=lp.data_ptr(), row=n, rows=m, n=n)

    def step():
        ok(lib, lib.yk_qk_rotate(C.byref(rot), stream()))
        x.copy_(qkv[:, :2 * d])
        ok(lib, lib.yk_quant_fp4(C.byref(qu), stream()))
        ok(lib, lib.yk_gemm_fp4(C.byref(ge), stream()))
        ok(lib, lib.yk_sample(C.byref(sa), stream()))

    inputs = [(torch.randn(m, 3 * d, generator=gen).half().cuda(), torch.rand(m, generator=gen).cuda()) for _ in range(3)]
    want = []
    for a, b in inputs:
        qkv.copy_(a)
        u.copy_(b)
        step()
        want.append((qkv.clone(), y.clone(), token.clone(), lp.clone()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in (0, 2, 1, 1):
        qkv.copy_(inputs[i][0])
        u.copy_(inputs[i][1])
        graph.replay()
        for a, b in zip((qkv, y, token, lp), want[i]):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qkv.copy_(inputs[2][0])
        u.copy_(inputs[2][1])
        step()
    side.synchronize()
    for a, b in zip((qkv, y, token, lp), want[2]):
        assert torch.equal(a, b)


def test_two_graphs_at_once(lib, cuda):
    """Two captured graphs of the large forms (whole tiles by pairs, split columns, scores by place and by bin, rows in
    several turns) replayed side by side on two streams: what each gives alone."""
    from yolo11_cu_b200 import runtime as rt
    gen = torch.Generator().manual_seed(12)
    new = lambda *s, dtype=torch.half: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731

    def program(m, n, k):
        qkv = torch.randn(4000, 24, 64, generator=gen).half().cuda()
        out, pos, freqs = torch.zeros_like(qkv), torch.arange(4000, dtype=torch.int32, device="cuda"), torch.rand(32, generator=gen).cuda()
        x, codes, scales = torch.randn(m, k, generator=gen).half().cuda(), new(m, k // 2, dtype=torch.uint8), \
            new(lib.yk_fp4_scale_bytes(m, k, 0), dtype=torch.uint8)
        w, y, small = random_matrix(n, k, 0, gen, torch.half, 0.1), new(m, n), new(8, n)
        logits, u = torch.randn(9, 40000, generator=gen).half().cuda(), torch.rand(9, generator=gen).cuda()
        top_p = torch.full((9,), 0.9, device="cuda")
        token, other = new(9, dtype=torch.int32), new(9, dtype=torch.int32)
        rot = rt.YkQkRotate(q=qkv.data_ptr(), k=qkv.data_ptr() + 2 * 64 * 16, q_out=out.data_ptr(), k_out=out.data_ptr() + 2 * 64 * 16,
                            pos=pos.data_ptr(), freqs=freqs.data_ptr(), q_row=24 * 64, k_row=24 * 64, q_out_row=24 * 64, k_out_row=24 * 64,
                            rows=4000, heads=16, kv_heads=8, dim=64, rot=64, axes=1)
        qu = rt.YkQuantFp4(x=x.data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr(), x_row=k, codes_row=k // 2, rows=m, cols=k)
        ge = [rt.YkGemmFp4(x=codes.data_ptr(), xscale=scales.data_ptr(), w=w[0].data_ptr(), wscale=w[1].data_ptr(), y=o.data_ptr(),
                           x_row=k // 2, w_row=w[0].stride(0), y_row=n, rows=len(o), n=n, k=k) for o in (y, small)]
        sa = [rt.YkSample(logits=logits.data_ptr(), u=u.data_ptr(), top_p=top_p.data_ptr(), token=o.data_ptr(), row=40000, rows=9, n=c)
              for o, c in ((token, 40000), (other, 20000))]

        def step():
            ok(lib, lib.yk_qk_rotate(C.byref(rot), stream()))
            ok(lib, lib.yk_quant_fp4(C.byref(qu), stream()))
            for a in ge:
                ok(lib, lib.yk_gemm_fp4(C.byref(a), stream()))
            for a, kernel in zip(sa, (2, 1)):
                ok(lib, lib.yk_test_sample_kernel(kernel))
                ok(lib, lib.yk_sample(C.byref(a), stream()))
            ok(lib, lib.yk_test_sample_kernel(0))

        return step, (out, codes, scales, y, small, token, other), (qkv, x, w, logits, u, top_p, pos, freqs, rot, qu, ge, sa)

    graphs, wants, outs, keep = [], [], [], []
    for size in ((600, 5000, 1024), (1300, 2100, 2016)):
        step, out, held = program(*size)
        step()
        torch.cuda.synchronize()
        wants.append([o.clone() for o in out])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append(graph)
        outs.append(out)
        keep.append((step, held))
    for o in outs[0] + outs[1]:
        o.zero_()
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out, want in zip(outs, wants):
        for a, b in zip(out, want):
            assert torch.equal(a, b)
