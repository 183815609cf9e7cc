"""The text operators check their arguments on the host: a bad one is refused with a reason and
nothing is launched (so these run without a GPU)."""
import ctypes as C

import pytest

PTR = 1 << 20        # stands for device memory; never read


def cache(rt, **kw):
    d = dict(k=PTR, v=PTR, kscale=PTR, vscale=PTR, block_stride=2 * 32 * 128, scale_stride=2, blocks=10, heads=2,
             tokens=32, dim=128)
    return rt.YkKvCache(**(d | kw))


def plan(rt, **kw):
    d = dict(past=PTR, fresh=PTR, free_blocks=PTR, table=PTR, kv_lens=PTR + 4096, cu=PTR, slots=PTR, table_stride=8,
             requests=4, rows=10, free_count=5, blocks=20, max_blocks=8, tokens=16)
    return rt.YkKvPlan(**(d | kw))


def rows(rt, **kw):
    d = dict(k=PTR, v=PTR, slots=PTR, k_row=256, v_row=256, k_head=128, v_head=128, rows=3, dtype=0)
    return rt.YkKvRows(**(d | kw))


def attn(rt, **kw):
    d = dict(q=PTR, out=PTR, q_row=512, out_row=512, cu=PTR, kv_lens=PTR, table=PTR, ws=PTR, ws_bytes=1 << 30,
             table_stride=4, max_blocks=4, requests=2, rows=5, heads=4, dtype=0, causal=1)
    return rt.YkAttnKv8(**(d | kw))


def norm(rt, **kw):
    d = dict(x=PTR, weight=PTR, codes=PTR, scales=PTR, x_row=64, codes_row=64, scales_row=1, rows=2, cols=64, eps=1e-6)
    return rt.YkRmsNorm8(**(d | kw))


def gemv(rt, **kw):
    d = dict(x=PTR, w=PTR, wscale=PTR, y=PTR, x_row=128, w_row=64, group_row=1, y_row=16, rows=1, n=16, k=128,
             group=128, xtype=0, dtype=0)
    return rt.YkGemv4(**(d | kw))


EINVAL, EUNSUP = -1, -4
CACHE = [(dict(k=None), EINVAL), (dict(vscale=None), EINVAL), (dict(tokens=24), EUNSUP), (dict(dim=96), EUNSUP),
         (dict(blocks=0), EINVAL), (dict(blocks=1 << 27), EINVAL), (dict(k=PTR + 8), EINVAL),
         (dict(block_stride=100), EINVAL), (dict(block_stride=2 * 32 * 128 + 8), EINVAL), (dict(scale_stride=1), EINVAL)]
PLAN = [(dict(past=None), EINVAL), (dict(cu=None), EINVAL), (dict(slots=None), EINVAL), (dict(requests=0), EINVAL),
        (dict(requests=16385), EUNSUP), (dict(rows=-1), EINVAL), (dict(table_stride=7), EINVAL), (dict(tokens=10), EUNSUP),
        (dict(free_blocks=None), EINVAL), (dict(blocks=1 << 28), EINVAL), (dict(max_blocks=0), EINVAL)]
ROWS = [(dict(k=None), EINVAL), (dict(slots=None), EINVAL), (dict(rows=-1), EINVAL), (dict(dtype=2), EUNSUP),
        (dict(k=PTR + 2), EINVAL), (dict(k_row=12), EINVAL), (dict(v_head=4), EINVAL)]
ATTN = [(dict(cu=None), EINVAL), (dict(ws=None), EINVAL), (dict(ws_bytes=100), EINVAL), (dict(ws=PTR + 4), EINVAL),
        (dict(heads=3), EINVAL), (dict(heads=0), EINVAL), (dict(dtype=2), EUNSUP), (dict(requests=0), EINVAL),
        (dict(requests=20000), EUNSUP), (dict(rows=1 << 30), EUNSUP), (dict(q=None), EINVAL), (dict(out=PTR + 2), EINVAL), (dict(q_row=513), EINVAL),
        (dict(out_row=256), EINVAL), (dict(window=5, causal=0), EINVAL), (dict(window=-1), EINVAL),
        (dict(scale=-1.0), EINVAL), (dict(scale=float("nan")), EINVAL), (dict(table_stride=3), EINVAL)]
NORM = [(dict(x=None), EINVAL), (dict(codes=None), EINVAL), (dict(scales=None), EINVAL), (dict(dtype=2), EUNSUP),
        (dict(cols=0), EINVAL), (dict(cols=40000, codes_row=40000), EUNSUP), (dict(group=8), EUNSUP),
        (dict(group=-1), EINVAL), (dict(eps=-1.0), EINVAL), (dict(codes_row=63), EINVAL),
        (dict(group=32, scales_row=1), EINVAL), (dict(rows=-2), EINVAL), (dict(x_row=-1), EINVAL),
        (dict(add=PTR, sum=PTR, sum_row=3), EINVAL)]
GEMV = [(dict(x=None), EINVAL), (dict(w=None), EINVAL), (dict(rows=0), EINVAL), (dict(rows=65), EUNSUP),
        (dict(group=48), EUNSUP), (dict(k=96), EINVAL), (dict(dtype=2), EUNSUP), (dict(xtype=1), EUNSUP),
        (dict(xtype=2), EINVAL), (dict(xtype=2, xscale=PTR, xgroup=64, xscale_row=2), EINVAL),
        (dict(xtype=2, xscale=PTR, xgroup=128, xscale_row=0), EINVAL), (dict(w=PTR + 4), EINVAL),
        (dict(w_row=72), EINVAL), (dict(w_row=32), EINVAL), (dict(group_row=0), EINVAL), (dict(y_row=8), EINVAL)]


def refused(lib, code, want):
    assert code == want
    assert lib.yk_last_cuda_error().decode()


@pytest.mark.parametrize("kw,want", CACHE)
def test_cache(lib, kw, want):
    from yolo11_cu_b200 import runtime as rt
    before = lib.yk_launch_count()
    c, x, a = cache(rt, **kw), rows(rt), attn(rt)
    refused(lib, lib.yk_kv_append(C.byref(c), C.byref(x), None), want)
    refused(lib, lib.yk_attn_kv8(C.byref(c), C.byref(a), None), want)
    assert lib.yk_launch_count() == before


@pytest.mark.parametrize("name,make,kw,want", [("yk_kv_plan", plan, *p) for p in PLAN] +
                         [("yk_rmsnorm8", norm, *p) for p in NORM] + [("yk_gemv4", gemv, *p) for p in GEMV])
def test_arguments(lib, name, make, kw, want):
    from yolo11_cu_b200 import runtime as rt
    before = lib.yk_launch_count()
    a = make(rt, **kw)
    refused(lib, getattr(lib, name)(C.byref(a), None), want)
    refused(lib, getattr(lib, name)(None, None), EINVAL)
    assert lib.yk_launch_count() == before


@pytest.mark.parametrize("name,make,kw,want", [("yk_kv_append", rows, *p) for p in ROWS] +
                         [("yk_attn_kv8", attn, *p) for p in ATTN])
def test_arguments_with_cache(lib, name, make, kw, want):
    from yolo11_cu_b200 import runtime as rt
    before = lib.yk_launch_count()
    c, a = cache(rt), make(rt, **kw)
    refused(lib, getattr(lib, name)(C.byref(c), C.byref(a), None), want)
    refused(lib, getattr(lib, name)(C.byref(c), None, None), EINVAL)
    refused(lib, getattr(lib, name)(None, C.byref(a), None), EINVAL)
    assert lib.yk_launch_count() == before


def test_no_rows_is_no_launch(lib):
    from yolo11_cu_b200 import runtime as rt
    before = lib.yk_launch_count()
    c, x, a, n = cache(rt), rows(rt, rows=0), attn(rt, rows=0), norm(rt, rows=0)
    assert lib.yk_kv_append(C.byref(c), C.byref(x), None) == 0
    assert lib.yk_attn_kv8(C.byref(c), C.byref(a), None) == 0
    assert lib.yk_rmsnorm8(C.byref(n), None) == 0
    assert lib.yk_launch_count() == before


def test_workspace_size(lib):
    sizes = [lib.yk_attn_kv8_workspace_bytes(4, 100, 8, 2, d) for d in (64, 128, 256)]
    assert sizes == sorted(sizes) and sizes[0] > 0
