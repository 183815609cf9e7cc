"""GPU parity of the text-decoder operators against their 64-bit definitions (text_ref.py).

Bounds, with u = 2^-11 (fp16) or 2^-8 (bf16, a full ulp) for the one rounding of a result:
plan and append are exact (append: power-of-two scales, one rounding to e4m3 from fp32 values
that are exact); norm, attention and GEMV allow their fp32 sums n * 2^-24 of the sum of
magnitudes; attention's weights enter the products in 16 bits (2^-11 of the weighted |v|, twice
that allowed)."""
import ctypes as C
import math
import random

import numpy as np
import pytest
import torch

import text_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"f16": (torch.float16, 0, 2.0 ** -11), "bf16": (torch.bfloat16, 1, 2.0 ** -8)}


@pytest.fixture(autouse=True)
def the_librarys_rule(lib):
    yield
    lib.yk_test_attn_kv8(0)


def within(got, want, bound, dt):
    """|got - want| <= bound, where a result that the type does not hold is an infinity."""
    top = 65520.0 if dt == torch.float16 else 3.3961775e38     # rounds up to infinity from here on
    with np.errstate(invalid="ignore"):
        fine = np.abs(got - want) <= bound
    inf = got == np.copysign(np.inf, want)
    over, under = np.abs(want) - bound >= top, np.abs(want) + bound < top
    good = np.where(over, inf, np.where(under, fine, fine | inf))
    return np.where(np.isnan(want), np.isnan(got), good)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def ok(lib, code):
    assert code == 0, (code, lib.yk_last_cuda_error())


def stream():
    return torch.cuda.current_stream().cuda_stream


def f64(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------------- plan

def run_plan(lib, rt, past, fresh, free, T, rows, max_blocks, blocks, head=None, inplace=False,
             table=None, stride=None, pos=True, counts=True):
    R, stride = len(past), stride or max_blocks
    full = np.full((R, stride), -7, np.int32)
    table = [[-1] * max_blocks for _ in past] if table is None else table
    for r in range(R):
        full[r, :max_blocks] = table[r]
    t = i32(full)
    p, f, fr = i32(past), i32(fresh), i32(free or [0])
    kv = p if inplace else torch.full((R,), -9, dtype=torch.int32, device="cuda")
    cu, hd = i32([-9] * (R + 1)), i32([head or 0])
    slots, ps, cnt = i32([-9] * (rows + 1)), i32([-9] * (rows + 1)), i32([-9] * 4)
    a = rt.YkKvPlan(past=p.data_ptr(), fresh=f.data_ptr(), free_blocks=fr.data_ptr(),
                    free_head=hd.data_ptr() if head is not None else None, table=t.data_ptr(),
                    kv_lens=kv.data_ptr(), cu=cu.data_ptr(), slots=slots.data_ptr(),
                    pos=ps.data_ptr() if pos else None, counts=cnt.data_ptr() if counts else None,
                    table_stride=stride, requests=R, rows=rows, free_count=len(free),
                    blocks=blocks, max_blocks=max_blocks, tokens=T)
    ok(lib, lib.yk_kv_plan(C.byref(a), stream()))
    want = ref.plan(past, fresh, free, head or 0, table, T, rows, max_blocks, blocks)
    got = t.cpu().numpy()
    assert got[:, :max_blocks].tolist() == want[0]
    assert (got[:, max_blocks:] == -7).all()
    assert kv.tolist() == want[1]
    assert cu.tolist() == want[2]
    assert slots.tolist() == want[3] + [-9]
    assert ps.tolist() == (want[4] if pos else [-9] * rows) + [-9]
    assert cnt.tolist() == (want[5] if counts else [-9] * 4)
    assert hd.tolist() == [want[6] if head is not None else 0]
    return want


PLANS = {
    "one": ([0], [1], 1), "nothing": ([0, 5, 0], [0, 0, 0], 1), "edges": ([15, 16, 17, 0, 31], [1, 1, 1, 16, 2], 1),
    "refused": ([0, 16, 3, 40, 0], [33, 1, 4, 90, 0], 0.4), "negative": ([5, -1, 7, 2], [3, 2, -4, 1], 1),
    "long": ([3, 900, 100], [500, 60, 1000], 1),
}


@pytest.mark.parametrize("T", [16, 64])
@pytest.mark.parametrize("name", sorted(PLANS))
@pytest.mark.parametrize("inplace", [False, True])
def test_plan(lib, cuda, name, T, inplace):
    from yolo11_cu_b200 import runtime as rt
    past, fresh, share = PLANS[name]
    rng = random.Random(3)
    blocks = 400
    ids = rng.sample(range(blocks), blocks)
    table = [[-1] * 90 for _ in past]
    for r, p in enumerate(past):
        for i in range(-(-max(p, 0) // T)):
            table[r][i] = ids.pop()
    need = sum(-(-(p + f) // T) - -(-p // T) for p, f in zip(past, fresh) if p >= 0 and f >= 0)
    free = ids[:int(need * share) + 2]
    rows = sum(max(f, 0) for f in fresh)
    for head in (None, 0, 2):
        run_plan(lib, rt, past, fresh, free, T, rows, 90, blocks, head=head, inplace=inplace,
                 table=table, stride=95)
    run_plan(lib, rt, past, fresh, free, T, rows + 5, 90, blocks, pos=False, counts=False, table=table)
    run_plan(lib, rt, past, fresh, free, T, max(rows - 2, 0), 90, blocks, table=table)   # rows do not fit
    run_plan(lib, rt, past, fresh, free, T, rows, 2, blocks, table=[t[:2] for t in table]
             if all(p <= 2 * T for p in past) else None)                                # table too narrow
    run_plan(lib, rt, past, fresh, [], T, rows, 90, blocks, table=table)                 # nothing free


@pytest.mark.parametrize("R,top,head", [(1, 30000, 3), (1000, 70, None), (3001, 9, 1), (16384, 2, 0)])
@pytest.mark.parametrize("inplace", [False, True])
def test_plan_many(lib, cuda, R, top, head, inplace):
    from yolo11_cu_b200 import runtime as rt
    rng = random.Random(R)
    T, cols = 32, -(-(100 + top) // 32)
    past = [rng.randrange(100) for _ in range(R)]
    fresh = [rng.randrange(top) if R > 1 else top for _ in range(R)]
    held = sum(-(-p // T) for p in past)
    need = sum(-(-(p + f) // T) - -(-p // T) for p, f in zip(past, fresh))
    ids = rng.sample(range(held + need + 9), held + need + 9)
    table = []
    for p in past:
        n = -(-p // T)
        table.append(ids[:n] + [-1] * (cols - n))
        ids = ids[n:]
    run_plan(lib, rt, past, fresh, ids[:need - need // 10 + (head or 0)], T, sum(fresh), cols,
             held + need + 9, head=head, inplace=inplace, table=table)


def test_plan_table_entry_outside_pool(lib, cuda):
    from yolo11_cu_b200 import runtime as rt
    run_plan(lib, rt, [5, 20], [3, 20], [1, 99, 2], 16, 23, 4, 8, table=[[8, -1, -1, -1], [0, -3, -1, -1]])


@pytest.mark.parametrize("past,fresh,free,want", [
    # one free block: the first request needs three, so the second, which needs one, waits behind it
    ([0, 0], [33, 1], [7], dict(kv=[0, 0], counts=[0, 0, 2, 34], head=0, slots=[-1] * 34, tables=[[-1] * 4, [-1] * 4])),
    # a request that needs none goes on; whoever needs one after the shortage does not
    ([16, 3, 16], [40, 2, 1], [7, 9], dict(kv=[16, 5, 16], counts=[0, 2, 2, 43], head=0,
                                           slots=[-1] * 40 + [4 * 16 + 3, 4 * 16 + 4, -1],
                                           tables=[[4, -1, -1, -1], [4, -1, -1, -1], [4, -1, -1, -1]])),
    # the shortage comes second: what the first took stays its own
    ([0, 0, 0], [5, 20, 1], [7, 9], dict(kv=[5, 0, 0], counts=[1, 5, 2, 26], head=1,
                                         slots=[7 * 16 + i for i in range(5)] + [-1] * 21,
                                         tables=[[7, -1, -1, -1], [-1] * 4, [-1] * 4])),
    # past the table's end or negative: refused for itself, the ones after it find the blocks untouched
    ([0, -1, 0], [65, 4, 1], [7], dict(kv=[0, -1, 1], counts=[1, 1, 2, 70], head=1,
                                       slots=[-1] * 69 + [7 * 16], tables=[[-1] * 4, [-1] * 4, [7, -1, -1, -1]]))])
def test_plan_does_not_overtake(lib, cuda, past, fresh, free, want):
    """Results written out by hand: no request goes past one before it that waits for blocks."""
    from yolo11_cu_b200 import runtime as rt
    table = [[4 if p > 0 else -1, -1, -1, -1] for p in past]
    got = run_plan(lib, rt, past, fresh, free, 16, sum(max(f, 0) for f in fresh), 4, 20, head=0, table=table)
    assert (got[0], got[1], got[3], got[5], got[6]) == (want["tables"], want["kv"], want["slots"], want["counts"],
                                                         want["head"])


# ---------------------------------------------------------------- cache

def make_cache(rt, blocks, heads, T, D, seed=0, joint=False, spread=0.5, vspread=0.5):
    """A random cache; joint: keys and values of a block side by side in one buffer."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = heads * T * D
    buf = torch.randn(blocks, 2, n, generator=g, device="cuda").mul(120).clamp(-448, 448)
    buf = buf.to(ref.F8).view(torch.uint8)
    if not joint:
        buf = buf.transpose(0, 1).contiguous().transpose(0, 1)
    sc = torch.randn(2, blocks, heads + 1, generator=g, device="cuda")
    sc[0] = torch.exp2((sc[0] * spread - 7).round())
    sc[1] = torch.exp2((sc[1] * vspread - 7).round())
    c = rt.YkKvCache(k=buf[:, 0].data_ptr(), v=buf[:, 1].data_ptr(), kscale=sc[0].data_ptr(),
                     vscale=sc[1].data_ptr(), block_stride=buf.stride(0), scale_stride=heads + 1,
                     blocks=blocks, heads=heads, tokens=T, dim=D)
    return c, buf, sc


def view4(buf, part, heads, T, D):
    return buf[:, part].reshape(-1, heads, T, D).cpu().numpy()


def same_values(codes, want):
    got = ref.e4m3_values(codes)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    bad = np.argwhere(~((got == want) | np.isnan(want)))
    assert len(bad) == 0, (len(bad), bad[:3], got[tuple(bad[0])], want[tuple(bad[0])])


def slots_of(lens, T, seed, spare=2):
    """Slots of (past, fresh) requests in a shuffled pool, and the pool's blocks."""
    rng = random.Random(seed)
    need = [-(-(p + f) // T) for p, f in lens]
    ids = rng.sample(range(sum(need) + spare), sum(need))
    out = []
    for (p, f), n in zip(lens, need):
        mine, ids = ids[:n], ids[n:]
        out += [mine[i // T] * T + i % T for i in range(p, p + f)]
    return out, sum(need) + spare


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,T,D", [(1, 16, 64), (8, 32, 128), (3, 128, 256), (5, 64, 128), (17, 16, 128)])
@pytest.mark.parametrize("lens", [[(0, 1)], [(5, 1), (31, 1), (16, 1), (0, 1), (63, 1)], [(7, 300), (0, 1), (3, 129)]])
@pytest.mark.parametrize("joint", [False, True])
def test_append(lib, cuda, kind, heads, T, D, lens, joint):
    from yolo11_cu_b200 import runtime as rt
    dt, code, _ = TYPES[kind]
    slots, blocks = slots_of(lens, T, heads + T)
    c, buf, sc = make_cache(rt, blocks, heads, T, D, seed=T, joint=joint)
    g = torch.Generator(device="cuda").manual_seed(D)
    n = len(slots)
    # rows of a fused projection: [q | k | v], heads side by side; the rows' loudness varies
    x = torch.randn(n, 3, heads, D, generator=g, device="cuda") * torch.exp2(
        torch.randn(n, 1, heads, 1, generator=g, device="cuda") * 4)
    x = x.to(dt)
    a = rt.YkKvRows(k=x[:, 1].data_ptr(), v=x[:, 2].data_ptr(), slots=i32(slots).data_ptr(),
                    k_row=3 * heads * D, v_row=3 * heads * D, k_head=D, v_head=D, rows=n, dtype=code)
    s = i32(slots)
    a.slots = s.data_ptr()
    before, scales = [view4(buf, i, heads, T, D).copy() for i in (0, 1)], f64(sc)
    ok(lib, lib.yk_kv_append(C.byref(c), C.byref(a), stream()))
    torch.cuda.synchronize()
    for i in (0, 1):
        val, want = ref.append(f64(x[:, 1 + i]), slots, before[i], scales[i, :, :heads], T)
        assert np.array_equal(f64(sc)[i, :, :heads], want)
        assert np.array_equal(f64(sc)[i, :, heads], scales[i, :, heads])
        same_values(view4(buf, i, heads, T, D), val)
    # again with the same rows: nothing moves
    again = buf.clone()
    ok(lib, lib.yk_kv_append(C.byref(c), C.byref(a), stream()))
    if max(f for _, f in lens) == 1:
        assert torch.equal(again, buf)


def test_append_head_major_rows_and_many(lib, cuda):
    """[heads][rows][dim] inputs, and a batch long enough that a CTA takes several rows."""
    from yolo11_cu_b200 import runtime as rt
    heads, T, D = 2, 32, 64
    rng = random.Random(1)
    lens = [(rng.randrange(40), rng.choice([1, 1, 1, 1, 2, 50])) for _ in range(1500)]
    slots, blocks = slots_of(lens, T, 4)
    n = len(slots)
    assert n > 2 * 148 * 8
    slots[7] = -1
    slots[-3] = blocks * T          # both outside the pool: left out
    c, buf, sc = make_cache(rt, blocks, heads, T, D)
    x = torch.randn(2, heads, n, D, device="cuda").half()
    s = i32(slots)
    a = rt.YkKvRows(k=x[0].data_ptr(), v=x[1].data_ptr(), slots=s.data_ptr(), k_row=D, v_row=D,
                    k_head=n * D, v_head=n * D, rows=n, dtype=0)
    before, scales = [view4(buf, i, heads, T, D).copy() for i in (0, 1)], f64(sc)
    ok(lib, lib.yk_kv_append(C.byref(c), C.byref(a), stream()))
    torch.cuda.synchronize()
    for i in (0, 1):
        val, want = ref.append(f64(x[i].transpose(0, 1)), slots, before[i], scales[i, :, :heads], T)
        assert np.array_equal(f64(sc)[i, :, :heads], want)
        same_values(view4(buf, i, heads, T, D), val)


def test_append_special_values(lib, cuda):
    """Zero rows, infinities, NaN, the smallest and largest numbers; a stale loud block is
    started anew; a scale that grows rounds the earlier tokens."""
    from yolo11_cu_b200 import runtime as rt
    heads, T, D = 1, 16, 64
    c, buf, sc = make_cache(rt, 6, heads, T, D)
    x = torch.zeros(7, 2, 1, D, device="cuda")
    x[1, :, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan], device="cuda")
    x[1, :, 0, 3] = 448.0
    x[2, :, 0, 5] = 448.1
    x[3, :, 0, :] = 3.0e38
    x[4, :, 0, :] = 1.0e-38
    x[5, :, 0, :] = 1.0
    x[6, :, 0, :] = 4000.0
    x = x.bfloat16()
    slots = [0, 16, 32, 48, 64, 80 + 4, 80 + 5]
    s = i32(slots)
    a = rt.YkKvRows(k=x[:, 0].data_ptr(), v=x[:, 1].data_ptr(), slots=s.data_ptr(), k_row=2 * D,
                    v_row=2 * D, k_head=D, v_head=D, rows=7, dtype=1)
    before, scales = [view4(buf, i, heads, T, D).copy() for i in (0, 1)], f64(sc)
    ok(lib, lib.yk_kv_append(C.byref(c), C.byref(a), stream()))
    torch.cuda.synchronize()
    for i in (0, 1):
        val, want = ref.append(f64(x[:, i]), slots, before[i], scales[i, :, :heads], T)
        assert np.array_equal(f64(sc)[i, :, :heads], want)
        same_values(view4(buf, i, heads, T, D), val)
    assert f64(sc)[0, 0, 0] == 2.0 ** -126 and f64(sc)[0, 1, 0] == 1.0


# ---------------------------------------------------------------- attention

def run_attention(lib, rt, kind, heads, kv_heads, D, T, lens, causal=1, window=0, scale=0.0,
                  qscale=1.0, pad=0, joint=False, lse=True, spoil=True, vspread=0.5, bad_block=None,
                  repeat=2, seed=0, nan=()):
    """lens: (kv, q) of each request; pad: rows of no request at the end."""
    dt, code, u = TYPES[kind]
    rng = random.Random(seed)
    need = [-(-kv // T) for kv, _ in lens]
    blocks, cols = sum(need) + 2, max(need + [1]) + 1
    ids = rng.sample(range(blocks), blocks)
    table = []
    for n in need:
        table.append(ids[:n] + [blocks + 5] * (cols - n))
        ids = ids[n:]
    if bad_block is not None:
        table[bad_block[0]][bad_block[1]] = bad_block[2]
    c, buf, sc = make_cache(rt, blocks, kv_heads, T, D, seed=seed, joint=joint, vspread=vspread)
    view = buf.view(blocks, 2, kv_heads, T, D)
    if spoil:                      # whatever lies past a request's end is NaN
        view[ids] = 127
        for (kv, _), row in zip(lens, table):
            if kv % T and 0 <= row[kv // T] < blocks:
                view[row[kv // T], :, :, kv % T:] = 127
    for r, j, part, ch in nan:     # NaN in the middle: seen by the rows from token j on
        view[table[r][j // T], part, :, j % T, ch] = 255
    cu = np.cumsum([0] + [q for _, q in lens]).tolist()
    n = cu[-1] + pad
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    qkv = (torch.randn(n, heads + 3, D, generator=g, device="cuda") * qscale).to(dt)
    q = qkv[:, 1:1 + heads]
    out = torch.full((n, heads + 1, D), 9.0, dtype=dt, device="cuda")
    ls = torch.full((n, heads), 9.0, device="cuda")
    size = lib.yk_attn_kv8_workspace_bytes(len(lens), n, heads, kv_heads, D)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    t, cud, kvd = i32(table), i32(cu), i32([kv for kv, _ in lens])
    a = rt.YkAttnKv8(q=q.data_ptr(), out=out.data_ptr(), lse=ls.data_ptr() if lse else None,
                     q_row=(heads + 3) * D, out_row=(heads + 1) * D, cu=cud.data_ptr(),
                     kv_lens=kvd.data_ptr(), table=t.data_ptr(), table_stride=cols, max_blocks=cols,
                     requests=len(lens), rows=n, heads=heads, dtype=code, causal=causal,
                     window=window, scale=scale, ws=ws.data_ptr(), ws_bytes=size)
    results = []
    for kernel in (1, 2, 0):           # both kernels, and the one that the rule takes
        assert lib.yk_test_attn_kv8(kernel) == 0
        first = None
        for _ in range(repeat):        # the workspace is left as it was found: the same bits again
            out.fill_(9.0)
            ls.fill_(9.0)
            ok(lib, lib.yk_attn_kv8(C.byref(c), C.byref(a), stream()))
            torch.cuda.synchronize()
            if first is None:
                first = out.clone()
            assert torch.equal(first.view(torch.int16), out.view(torch.int16))
        assert lib.yk_fetch_device_error() == 0
        results.append((out.clone(), ls.clone()))
    o, l, mag, big = ref.attention(f64(q), view[:, 0].cpu().numpy(), f64(sc[0])[:, :kv_heads],
                                   view[:, 1].cpu().numpy(), f64(sc[1])[:, :kv_heads], table,
                                   [kv for kv, _ in lens], cu, T, causal, window,
                                   scale or D ** -0.5)
    ds = ((D + 8) * 2.0 ** -24 * big + 2.0 ** -21)[..., None]    # error of a score
    for out, ls in results:
        got = f64(out[:, :heads])[:cu[-1]]
        bound = u * np.abs(o) + (2.0 ** -10 + 2 * ds) * mag + 2.0 ** -24
        fine = within(got, o[:cu[-1]], bound[:cu[-1]], dt)
        assert fine.all(), (np.argwhere(~fine)[:3], (np.abs(got - o[:cu[-1]]) / bound[:cu[-1]]).max())
        assert (f64(out[cu[-1]:]) == 9).all() and (f64(out[:, heads]) == 9).all()
        if lse:
            gl, l = f64(ls)[:cu[-1]], l[:cu[-1]]
            assert np.array_equal(np.isnan(gl), np.isnan(l))
            empty = np.isinf(l) | np.isnan(l)
            assert (gl[np.isinf(l)] == -np.inf).all()
            lb = ds[:cu[-1], :, 0] + 2.0 ** -20 * (1 + np.abs(np.where(empty, 0, l)))
            assert (np.abs(gl[~empty] - l[~empty]) <= lb[~empty]).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,D,T", [
    (1, 1, 64, 16), (8, 2, 128, 32), (16, 2, 128, 64), (5, 1, 64, 128), (14, 2, 256, 16),
    (32, 1, 128, 16), (40, 2, 64, 32), (6, 6, 256, 64)])
@pytest.mark.parametrize("q", [1, 3])
def test_attention_decode(lib, cuda, kind, heads, kv_heads, D, T, q):
    from yolo11_cu_b200 import runtime as rt
    lens = [(1, 1), (0, 0), (0, 1), (T - 1, q), (T, q), (T + 1, q), (333, q), (16, q), (17, q), (127, q), (2, 5)]
    run_attention(lib, rt, kind, heads, kv_heads, D, T, lens, pad=2)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,D,T", [(4, 2, 64, 16), (3, 1, 128, 64), (2, 2, 256, 32), (8, 1, 128, 128)])
@pytest.mark.parametrize("causal,window", [(1, 0), (1, 1), (1, 37), (0, 0)])
def test_attention_prompt(lib, cuda, kind, heads, kv_heads, D, T, causal, window):
    from yolo11_cu_b200 import runtime as rt
    lens = [(130, 130), (201, 77), (64, 64), (5, 9), (1, 1), (0, 0), (300, 129)]
    run_attention(lib, rt, kind, heads, kv_heads, D, T, lens, causal=causal, window=window, pad=1)


@pytest.mark.parametrize("lens", [[(9000, 1)], [(4097, 1), (70, 1), (6000, 2)], [(5000, 1)] + [(3, 1)] * 40])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 1000])
def test_attention_long(lib, cuda, lens, D, window):
    """Work split along the keys and joined."""
    from yolo11_cu_b200 import runtime as rt
    run_attention(lib, rt, "f16", 4, 2, D, 32, lens, window=window, joint=True, repeat=3)


def test_attention_many_requests(lib, cuda):
    from yolo11_cu_b200 import runtime as rt
    rng = random.Random(2)
    lens = [(rng.randrange(0, 90), 1) if rng.random() < 0.9 else (0, 0) for _ in range(1100)]
    run_attention(lib, rt, "bf16", 2, 1, 64, 16, lens, lse=False)


def test_attention_many_prompts(lib, cuda):
    """More requests than are ordered by their length."""
    from yolo11_cu_b200 import runtime as rt
    rng = random.Random(4)
    lens = []
    for _ in range(150):
        q = rng.choice([0, 1, 20, 66, 130])
        lens.append((q + rng.randrange(0, 70), q))
    assert sum(q for _, q in lens) * 2 >= 64 * len(lens)
    run_attention(lib, rt, "bf16", 2, 1, 64, 32, lens)


@pytest.mark.parametrize("window", [0, 50])
def test_attention_prompt_among_decodes(lib, cuda, window):
    """A long prompt in a batch whose average is a few rows: many row tiles share the split list."""
    from yolo11_cu_b200 import runtime as rt
    run_attention(lib, rt, "f16", 6, 2, 128, 16, [(50, 1)] * 20 + [(300, 200)] + [(33, 1), (0, 0), (700, 2)] * 9,
                  window=window)


@pytest.mark.parametrize("qscale,scale,vspread", [(30.0, 0.0, 0.5), (1.0, 3.0, 0.5), (1.0, 0.0, 9.0),
                                                  (1e-4, 0.0, 0.5), (8.0, 0.5, 9.0)])
@pytest.mark.parametrize("q", [1, 70])
def test_attention_ranges(lib, cuda, qscale, scale, vspread, q):
    """Peaked and flat weights, and value scales that differ by many powers of two."""
    from yolo11_cu_b200 import runtime as rt
    for kind in ("f16", "bf16"):
        run_attention(lib, rt, kind, 4, 2, 128, 16, [(400, q), (90, q), (700, q)], qscale=qscale,
                      scale=scale, vspread=vspread)


@pytest.mark.parametrize("q", [1, 90])
@pytest.mark.parametrize("bad", [(0, 1, -1), (0, 0, 10 ** 6), (1, 2, 2 ** 31 - 1)])
def test_attention_block_outside_pool(lib, cuda, bad, q):
    """Keys of a block id outside the pool are not seen; nothing is read for them."""
    from yolo11_cu_b200 import runtime as rt
    run_attention(lib, rt, "f16", 4, 2, 64, 32, [(100, q), (129, q)], bad_block=bad)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 9])
@pytest.mark.parametrize("lens", [[(40, 20), (90, 6)], [(300, 150), (31, 1)]])
def test_attention_nan_is_seen_only_where_visible(lib, cuda, D, window, lens):
    """A NaN value reaches its channel in the rows that see its token, a NaN key those rows whole;
    rows that do not see the token are as without it."""
    from yolo11_cu_b200 import runtime as rt
    run_attention(lib, rt, "f16", 4, 2, D, 32, lens, window=window,
                  nan=[(0, 35, 1, 3), (0, 33, 1, D - 1), (1, 20, 1, 7)])
    run_attention(lib, rt, "bf16", 3, 1, D, 32, lens, window=window,
                  nan=[(0, 37, 0, 3), (0, 26, 1, 9), (1, 30, 1, 0)])


def attend_one(lib, rt, kind, q, k, v, ks, vs, T, scale):
    """One request of one key head: q [rows, heads, dim] as its last tokens over codes k, v [blocks, T, dim]
    with scales ks, vs [blocks], both kernels against the definition."""
    dt, code, u = TYPES[kind]
    n, heads, D = q.shape
    blocks = k.shape[0]
    q = q.to(dt).cuda()
    k, v = k.to(ref.F8).view(torch.uint8).cuda().contiguous(), v.to(ref.F8).view(torch.uint8).cuda().contiguous()
    ks, vs = ks.float().cuda(), vs.float().cuda()
    c = rt.YkKvCache(k=k.data_ptr(), v=v.data_ptr(), kscale=ks.data_ptr(), vscale=vs.data_ptr(),
                     block_stride=T * D, scale_stride=1, blocks=blocks, heads=1, tokens=T, dim=D)
    out, lse = torch.zeros_like(q), torch.zeros(n, heads, device="cuda")
    size = lib.yk_attn_kv8_workspace_bytes(1, n, heads, 1, D)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    cu, kv, t = i32([0, n]), i32([blocks * T]), i32([list(range(blocks))])
    a = rt.YkAttnKv8(q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), q_row=heads * D, out_row=heads * D,
                     cu=cu.data_ptr(), kv_lens=kv.data_ptr(), table=t.data_ptr(), table_stride=blocks,
                     max_blocks=blocks, requests=1, rows=n, heads=heads, dtype=code, causal=1, scale=scale,
                     ws=ws.data_ptr(), ws_bytes=size)
    o, l, mag, big = ref.attention(f64(q), k[:, None].cpu().numpy(), f64(ks)[:, None], v[:, None].cpu().numpy(),
                                   f64(vs)[:, None], [list(range(blocks))], [blocks * T], [0, n], T, 1, 0, scale)
    ds = ((D + 8) * 2.0 ** -24 * big + 2.0 ** -21)[..., None]
    bound = u * np.abs(o) + (2.0 ** -10 + 2 * ds) * mag + 2.0 ** -24
    for kernel in (1, 2):
        assert lib.yk_test_attn_kv8(kernel) == 0
        out.fill_(9.0)
        ok(lib, lib.yk_attn_kv8(C.byref(c), C.byref(a), stream()))
        fine = within(f64(out), o, bound, dt)
        assert fine.all(), (kernel, np.argwhere(~fine)[:3], np.nanmax(np.abs(f64(out) - o) / bound))
        assert (np.abs(f64(lse) - l) <= ds[..., 0] + 2.0 ** -20 * (1 + np.abs(l))).all()


@pytest.mark.parametrize("rows", [1, 66])
@pytest.mark.parametrize("gap,spread", [(16.0, 1.5), (17.0, 0.5), (18.0, 1.0)])
def test_attention_flat_tail_behind_a_loud_key(lib, cuda, rows, gap, spread):
    """One key far above thousands of others, with a value of zero: the output is the others' alone, though
    each weight is 2^-22 .. 2^-27 of the largest."""
    from yolo11_cu_b200 import runtime as rt
    T, D, blocks = 16, 64, 375
    g = torch.Generator().manual_seed(int(gap * 2))
    k, v = (torch.randn(blocks, T, D, generator=g) * 20 for _ in range(2))
    k[..., 0] = 0
    k[0, 0] = 0
    k[0, 0, 0] = 16
    v[0, 0] = 0
    q = torch.randn(rows, 2, D, generator=g) * (spread / (20 * (D - 1) ** 0.5))    # scores of this spread
    q[..., 0] = gap / 16
    for kind in ("f16", "bf16"):
        attend_one(lib, rt, kind, q, k, v, torch.ones(blocks), torch.ones(blocks), T, 1.0)


@pytest.mark.parametrize("rows", [1, 66])
@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("gap,loud", [(84.0, 11), (95.0, 11), (90.0, 90), (110.0, 110), (70.0, 110), (0.0, 110)])
def test_attention_value_scales_far_apart(lib, cuda, rows, order, gap, loud):
    """A block of zero values has the smallest scale (2^-126); with the highest scores and a block of a large
    scale beside it, the factor between weights and their 16-bit form stays finite."""
    from yolo11_cu_b200 import runtime as rt
    T, D, blocks = 16, 64, 13
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(blocks, T, D, generator=g) * 20 for _ in range(2))
    vs = torch.ones(blocks)
    for b, e in ((0, -126), (1, loud), (2, -20)):
        vs[b] = 2.0 ** e
    k[..., 0] = 0
    k[0, :, 0] = 16
    v[0] = 0
    q = torch.randn(rows, 2, D, generator=g) * (1 / 160)
    q[..., 0] = gap / 16
    if order < 0:
        k, v, vs = k.flip(0), v.flip(0), vs.flip(0)
    attend_one(lib, rt, "bf16", q, k, v, torch.ones(blocks), vs, T, 1.0)


def test_attention_offsets_past_32_bits(lib, cuda):
    """A pool whose code offsets pass 2^31 and 2^32."""
    from yolo11_cu_b200 import runtime as rt
    heads, T, D = 8, 128, 256
    blocks = (2 ** 32) // (heads * T * D) + 9
    pool = torch.zeros(blocks, heads, T, D, dtype=torch.uint8, device="cuda")
    sc = torch.ones(blocks, heads, device="cuda")
    c = rt.YkKvCache(k=pool.data_ptr(), v=pool.data_ptr(), kscale=sc.data_ptr(), vscale=sc.data_ptr(),
                     block_stride=heads * T * D, scale_stride=heads, blocks=blocks, heads=heads,
                     tokens=T, dim=D)
    row = [blocks - 1, blocks // 2 + 1, 3]
    slots = [row[0] * T + i for i in range(T)] + [row[1] * T + i for i in range(T)] + [row[2] * T]
    x = torch.randn(len(slots), 2, heads, D, device="cuda").half()
    s = i32(slots)
    a = rt.YkKvRows(k=x.data_ptr(), v=x.data_ptr(), slots=s.data_ptr(), k_row=2 * heads * D,
                    v_row=2 * heads * D, k_head=D, v_head=D, rows=len(slots), dtype=0)
    ok(lib, lib.yk_kv_append(C.byref(c), C.byref(a), stream()))
    mine = pool[row].cpu().numpy()
    ids = {b: i for i, b in enumerate(row)}
    val, want = ref.append(f64(x[:, 0]), [ids[t // T] * T + t % T for t in slots],
                           np.zeros_like(mine), np.ones((3, heads)), T)
    same_values(mine, val)
    assert int((pool != 0).any(-1).any(-1).any(-1).sum()) == 3
    for q, kernel in ((1, 1), (65, 1), (65, 2)):
        lib.yk_test_attn_kv8(kernel)
        qs = torch.randn(q, heads, D, device="cuda").half()
        out = torch.zeros_like(qs)
        size = lib.yk_attn_kv8_workspace_bytes(1, q, heads, heads, D)
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        cu, kv, t = i32([0, q]), i32([len(slots)]), i32([row])
        b = rt.YkAttnKv8(q=qs.data_ptr(), out=out.data_ptr(), lse=None, q_row=heads * D,
                         out_row=heads * D, cu=cu.data_ptr(), kv_lens=kv.data_ptr(),
                         table=t.data_ptr(), table_stride=3, max_blocks=3, requests=1, rows=q,
                         heads=heads, dtype=0, causal=1, window=0, scale=0.0, ws=ws.data_ptr(),
                         ws_bytes=size)
        ok(lib, lib.yk_attn_kv8(C.byref(c), C.byref(b), stream()))
        o, _, mag, big = ref.attention(f64(qs), mine, f64(sc[row]), mine, f64(sc[row]), [[0, 1, 2]],
                                       [len(slots)], [0, q], T, 1, 0, D ** -0.5)
        ds = ((D + 8) * 2.0 ** -24 * big + 2.0 ** -21)[..., None]
        assert (np.abs(f64(out) - o) <= 2.0 ** -11 * np.abs(o) + (2.0 ** -10 + 2 * ds) * mag + 2.0 ** -24).all()


# ---------------------------------------------------------------- norm

def run_norm(lib, rt, kind, rows, cols, group, add=True, sum_=True, out=True, codes=True, extra=0,
             inplace=None, x=None, eps=1e-5, shift=0):
    dt, code, u = TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if x is None:
        x = new(rows, cols) * torch.exp(new(cols))
    xb = torch.zeros(rows * (cols + extra) + shift, dtype=dt, device="cuda")[shift:].view(rows, cols + extra)
    xb[:, :cols] = x
    ab = torch.zeros(rows, cols + 2 * extra, dtype=dt, device="cuda")
    ab[:, :cols] = new(rows, cols)
    w = (1 + 0.3 * new(cols)).to(dt)
    x64, a64 = f64(xb[:, :cols]), f64(ab[:, :cols])
    groups = -(-cols // (group or cols))
    sb = {None: torch.full((rows, cols + extra), 7.0, dtype=dt, device="cuda"), "x": xb, "add": ab}[inplace]
    ob = torch.full((rows, cols + extra), 7.0, dtype=dt, device="cuda")
    cb = torch.full((rows, cols + extra), 7, dtype=torch.uint8, device="cuda")
    sc = torch.full((rows, groups + 1), 7.0, device="cuda")
    p = lambda t, on: t.data_ptr() if on else None  # noqa: E731
    a = rt.YkRmsNorm8(x=xb.data_ptr(), add=p(ab, add), sum=p(sb, sum_), weight=w.data_ptr(), out=p(ob, out),
                      codes=p(cb, codes), scales=p(sc, codes), x_row=xb.stride(0), add_row=ab.stride(0),
                      sum_row=sb.stride(0), out_row=ob.stride(0), codes_row=cb.stride(0),
                      scales_row=groups + 1, rows=rows, cols=cols, group=group, dtype=code, eps=eps)
    ok(lib, lib.yk_rmsnorm8(C.byref(a), stream()))
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        h = x64 + (a64 if add else 0)
        y = h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * f64(w)
    # fp32: cols additions of squares (half of that in the root), a handful of roundings
    rel = (cols + 16) * 2.0 ** -25 + 2.0 ** -21
    tiny = 2.0 ** -24 if kind == "f16" else 2.0 ** -133
    fine = np.isfinite(y)
    if sum_:
        assert (np.abs(f64(sb[:, :cols])[fine] - h[fine]) <= (u * np.abs(h[fine]) * 1.001 + tiny)).all()
    if out:
        got = f64(ob[:, :cols])
        assert np.array_equal(np.isnan(got), np.isnan(y))
        assert (np.abs(got[fine] - y[fine]) <= (u + rel) * np.abs(y[fine]) * 1.001 + tiny).all()
        assert (f64(ob[:, cols:]) == 7).all()
    if codes:
        assert (f64(cb[:, cols:]) == 7).all() and (f64(sc[:, groups:]) == 7).all()
        got, s = ref.e4m3_values(cb[:, :cols].cpu().numpy()), f64(sc)
        for i in range(groups):
            at = slice(i * (group or cols), min(cols, (i + 1) * (group or cols)))
            yy = y[:, at]
            amax = np.where(np.isfinite(yy), np.abs(yy), 0).max(1)
            want = np.maximum(amax / 448, 2.0 ** -126)
            assert (np.abs(s[:, i] - want) <= rel * want).all()
            q = yy / s[:, i:i + 1]
            # half a step of e4m3: 2^-4 of the value, 2^-10 among the subnormals
            assert np.array_equal(np.isnan(got[:, at]), np.isnan(q))
            f = np.isfinite(q)
            assert (np.abs(got[:, at] - q)[f] <= (np.abs(q) * (2.0 ** -4 + rel) + 2.0 ** -10)[f]).all()
    return sb, ob, cb, sc


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,cols,group", [
    (1, 1, 0), (1, 2048, 0), (3, 4096, 128), (5, 5120, 128), (2, 777, 0), (7, 1000, 64), (300, 129, 32),
    (2, 16384, 0), (2, 32768, 16), (1, 32760, 48), (9, 255, 128), (4, 8, 16), (1000, 512, 0), (33, 2056, 200)])
def test_norm(lib, cuda, kind, rows, cols, group):
    from yolo11_cu_b200 import runtime as rt
    run_norm(lib, rt, kind, rows, cols, group)
    run_norm(lib, rt, kind, rows, cols, group, extra=8)
    run_norm(lib, rt, kind, rows, cols, group, extra=3, inplace="x")
    run_norm(lib, rt, kind, rows, cols, group, inplace="add", out=False)
    run_norm(lib, rt, kind, rows, cols, group, add=False, sum_=False, codes=False, shift=1)
    run_norm(lib, rt, kind, rows, cols, group, add=False, sum_=False, out=False, extra=1)


def test_norm_special_rows(lib, cuda):
    """Zero rows (smallest scale), huge and tiny rows, rows with an infinity or NaN."""
    from yolo11_cu_b200 import runtime as rt
    x = torch.randn(6, 640, device="cuda")
    x[0] = 0
    x[1] *= 1e18
    x[2] *= 1e-20
    x[3, 5] = math.nan
    x[4, 7] = math.inf
    x[5, 3:] = 0
    sb, ob, cb, sc = run_norm(lib, rt, "bf16", 6, 640, 128, add=False, x=x, eps=0.0 + 1e-30)
    assert (f64(sc[0, :5]) == 2.0 ** -126).all() and (f64(sc[3, :5]) == 2.0 ** -126).all()


# ---------------------------------------------------------------- gemv

def run_gemv(lib, rt, kind, rows, n, k, group, zero=False, bias=False, xgroup=None, extra=0, seed=0, shift=0):
    """xgroup: None for 16-bit x, else e4m3 with that group (0: a scale a row)."""
    dt, code, u = TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(seed + rows + n + k)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = torch.randint(0, 256, (n, k // 2 + 16 * extra), generator=g, device="cuda", dtype=torch.uint8)
    ws = (0.02 * torch.exp(new(n, k // group + extra))).to(dt)
    wz = torch.randint(0, 16, (n, k // group + extra), generator=g, device="cuda", dtype=torch.uint8)
    b = new(n)
    xs = torch.exp(new(rows, (-(-k // xgroup) if xgroup else 1) + extra))
    if xgroup is None:
        x = new(rows * (k + extra) + shift).to(dt)[shift:].view(rows, k + extra)
        x64 = f64(x[:, :k])
    else:
        x = (new(rows * (k + extra) + shift) * 100).clamp(-448, 448).to(ref.F8).view(torch.uint8)[shift:].view(rows, k + extra)
        x64 = ref.e4m3_values(x[:, :k].cpu().numpy()) * np.repeat(f64(xs), xgroup or k, 1)[:, :k]
    y = torch.full((rows, n + extra), 7.0, dtype=dt, device="cuda")
    a = rt.YkGemv4(x=x.data_ptr(), xscale=xs.data_ptr() if xgroup is not None else None, w=w.data_ptr(),
                   wscale=ws.data_ptr(), wzero=wz.data_ptr() if zero else None,
                   bias=b.data_ptr() if bias else None, y=y.data_ptr(), x_row=x.stride(0),
                   xscale_row=xs.stride(0), w_row=w.stride(0), group_row=k // group + extra,
                   y_row=n + extra, rows=rows, n=n, k=k, group=group, xgroup=xgroup or 0,
                   xtype=code if xgroup is None else rt.YK_E4M3, dtype=code)
    ok(lib, lib.yk_gemv4(C.byref(a), stream()))
    torch.cuda.synchronize()
    first = y.clone()
    ok(lib, lib.yk_gemv4(C.byref(a), stream()))
    torch.cuda.synchronize()
    assert torch.equal(first, y)
    wb = w[:, :k // 2].cpu().numpy()
    q = np.stack([wb & 15, wb >> 4], 2).reshape(n, k).astype(np.float64)
    z = np.repeat(wz[:, :k // group].cpu().numpy().astype(np.float64), group, 1) if zero else 8.0
    w64 = (q - z) * np.repeat(f64(ws[:, :k // group]), group, 1)
    want = x64 @ w64.T + (f64(b) if bias else 0)
    # fp32 sums of k products, each scaled in fp32
    bound = u * np.abs(want) + (k + 16) * 2.0 ** -24 * (np.abs(x64) @ np.abs(w64.T) + (np.abs(f64(b)) if bias else 0)) + 2.0 ** -24
    fine = within(f64(y[:, :n]), want, bound, dt)
    assert fine.all(), (np.argwhere(~fine)[:3], (np.abs(f64(y[:, :n]) - want) / bound).max())
    assert (f64(y[:, n:]) == 7).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n,k,group", [
    (1, 1, 32, 32), (1, 4096, 4096, 128), (2, 100, 96, 32), (3, 1000, 1024, 64), (7, 333, 640, 128),
    (8, 512, 2048, 32), (9, 77, 4096, 128), (16, 256, 8192, 64), (17, 1030, 384, 128), (33, 65, 320, 64),
    (64, 200, 1536, 128), (40, 16, 12288, 64), (5, 48, 160, 32), (1, 7, 28672, 64)])
def test_gemv(lib, cuda, kind, rows, n, k, group):
    from yolo11_cu_b200 import runtime as rt
    run_gemv(lib, rt, kind, rows, n, k, group)
    run_gemv(lib, rt, kind, rows, n, k, group, zero=True, bias=True, extra=1)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=0, bias=True, shift=1)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=group, zero=True, extra=8)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=2 * group, shift=3)
    run_gemv(lib, rt, kind, rows, n, k, group, shift=1)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n,k,group", [
    (1, 9472, 128, 128), (5, 9500, 1024, 64), (16, 9473, 672, 32), (17, 9600, 1280, 128), (33, 9472, 576, 64),
    (64, 9489, 288, 32), (64, 9475, 640, 128), (40, 9472, 1152, 64), (2, 9472, 32, 32), (9, 9601, 4224, 128)])
def test_gemv_many_outputs(lib, cuda, kind, rows, n, k, group):
    from yolo11_cu_b200 import runtime as rt
    run_gemv(lib, rt, kind, rows, n, k, group)
    run_gemv(lib, rt, kind, rows, n, k, group, zero=True, bias=True, extra=1)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=0, bias=True, shift=1)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=128, zero=True, extra=8)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=384, shift=8)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=3 * group, shift=3)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n,k,group", [
    (8, 4737, 128, 128), (9, 14209, 128, 32), (16, 14208, 320, 64), (16, 14300, 672, 32), (12, 18950, 256, 128),
    (17, 9473, 96, 32), (32, 9472, 384, 128), (33, 4737, 576, 64), (64, 4736, 288, 32), (64, 4750, 640, 128),
    (64, 48, 2048, 64), (33, 100, 2176, 128), (64, 130, 2048, 32), (40, 333, 1984, 64)])
def test_gemv_either_side_of_the_rule(lib, cuda, kind, rows, n, k, group):
    from yolo11_cu_b200 import runtime as rt
    run_gemv(lib, rt, kind, rows, n, k, group)
    run_gemv(lib, rt, kind, rows, n, k, group, zero=True, bias=True, extra=1)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=0, bias=True, shift=1)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=128, zero=True, extra=8)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=384, shift=8)
    run_gemv(lib, rt, kind, rows, n, k, group, xgroup=group, shift=3)


def test_gemv_large_values(lib, cuda):
    """fp16 x near its largest value: sums stay in 32 bits; x of infinities gives no finite sum."""
    from yolo11_cu_b200 import runtime as rt
    n, k = 64, 256
    x = torch.full((2, k), 60000.0, device="cuda").half()
    x[1, 3] = math.inf
    w = torch.full((n, k // 2), 0x99, dtype=torch.uint8, device="cuda")
    ws = torch.full((n, 2), 2.0 ** -10, device="cuda").half()
    y = torch.zeros(2, n, device="cuda").half()
    a = rt.YkGemv4(x=x.data_ptr(), w=w.data_ptr(), wscale=ws.data_ptr(), y=y.data_ptr(), x_row=k,
                   w_row=k // 2, group_row=2, y_row=n, rows=2, n=n, k=k, group=128, xtype=0, dtype=0)
    ok(lib, lib.yk_gemv4(C.byref(a), stream()))
    assert (f64(y[0]) == 15000.0).all() and (f64(y[1]) == math.inf).all()


# ---------------------------------------------------------------- streams and graphs

def test_side_stream_and_graph(lib, cuda):
    """The operators run in order on the stream they are given, and in a captured graph."""
    from yolo11_cu_b200 import runtime as rt
    x = torch.zeros(64, 2048, device="cuda").half()
    src = torch.randn(64, 2048, device="cuda").half()
    w = torch.ones(2048, device="cuda").half()
    codes, sc = torch.zeros(64, 2048, dtype=torch.uint8, device="cuda"), torch.zeros(64, 1, device="cuda")
    q4 = torch.randint(0, 256, (512, 1024), device="cuda", dtype=torch.uint8)
    ws = torch.full((512, 16), 0.01, device="cuda").half()
    y = torch.zeros(64, 512, device="cuda").half()
    a = rt.YkRmsNorm8(x=x.data_ptr(), weight=w.data_ptr(), codes=codes.data_ptr(), scales=sc.data_ptr(),
                      x_row=2048, codes_row=2048, scales_row=1, rows=64, cols=2048, dtype=0, eps=1e-6)
    b = rt.YkGemv4(x=codes.data_ptr(), xscale=sc.data_ptr(), w=q4.data_ptr(), wscale=ws.data_ptr(),
                   y=y.data_ptr(), x_row=2048, xscale_row=1, w_row=1024, group_row=16, y_row=512, rows=64,
                   n=512, k=2048, group=128, xtype=rt.YK_E4M3, dtype=0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def step():
        x.copy_(src)
        ok(lib, lib.yk_rmsnorm8(C.byref(a), stream()))
        ok(lib, lib.yk_gemv4(C.byref(b), stream()))

    with torch.cuda.stream(s):
        step()
    s.synchronize()
    want = y.clone()
    assert want.abs().sum() > 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    y.zero_()
    codes.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, y)
