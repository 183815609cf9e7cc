"""The decoder's rotation, 4-bit float and sampling operators check their arguments on the host: a bad one is
refused with a reason and nothing is launched (so these run without a GPU)."""
import ctypes as C
import math

import pytest

PTR = 1 << 20        # stands for device memory; never read
EINVAL, EUNSUP = -1, -4
NAN = math.nan


def rotate(rt, sections=(0, 0, 0, 0), **kw):
    d = dict(q=PTR, k=PTR, q_out=PTR, k_out=PTR, q_weight=PTR, k_weight=PTR, pos=PTR, freqs=PTR, q_row=256, k_row=128,
             q_out_row=256, k_out_row=128, pos_axis=3, rows=3, heads=4, kv_heads=2, dim=64, rot=64, axes=1, eps=1e-6)
    return rt.YkQkRotate(sections=(C.c_int * 4)(*sections), **(d | kw))


def quant(rt, **kw):
    d = dict(x=PTR, codes=PTR, scales=PTR, x_row=64, codes_row=32, rows=3, cols=64)
    return rt.YkQuantFp4(**(d | kw))


def gemm(rt, **kw):
    d = dict(x=PTR, xscale=PTR, w=PTR, wscale=PTR, y=PTR, x_row=64, w_row=64, y_row=10, rows=3, n=10, k=128)
    return rt.YkGemmFp4(**(d | kw))


def sample(rt, **kw):
    d = dict(logits=PTR, u=PTR, token=PTR, row=100, rows=3, n=100)
    return rt.YkSample(**(d | kw))


ROTATE = [(dict(q=None), EINVAL), (dict(k=None), EINVAL), (dict(k_out=None), EINVAL), (dict(pos=None), EINVAL),
          (dict(freqs=None), EINVAL), (dict(dtype=2), EUNSUP), (dict(dtype=3), EUNSUP), (dict(dim=96, rot=96), EUNSUP),
          (dict(dim=16, rot=16), EUNSUP), (dict(rows=-1), EINVAL), (dict(heads=0), EINVAL), (dict(kv_heads=-1), EINVAL),
          (dict(heads=1000, q_row=64000, q_out_row=64000, kv_heads=100, k_row=6400, k_out_row=6400), EUNSUP),
          (dict(heads=2 ** 31 - 1, kv_heads=2 ** 31 - 1), EUNSUP), (dict(rot=0), EINVAL), (dict(rot=24), EINVAL),
          (dict(rot=80), EINVAL), (dict(axes=0), EINVAL), (dict(axes=5), EINVAL), (dict(sections=(16, 0, 0, 0)), EINVAL),
          (dict(sections=(16, 16, 0, 0)), EINVAL), (dict(axes=2, sections=(16, 15, 0, 0)), EINVAL), (dict(axes=2), EINVAL),
          (dict(axes=2, sections=(40, -8, 0, 0)), EINVAL), (dict(axes=2, sections=(16, 16, 0, 0), pos_axis=2), EINVAL),
          (dict(q_row=255), EINVAL), (dict(q_row=248), EINVAL), (dict(k_out_row=120), EINVAL), (dict(q_out_row=260), EINVAL),
          (dict(q=PTR + 8), EINVAL), (dict(k_out=PTR + 2), EINVAL), (dict(q_weight=PTR + 4), EINVAL), (dict(pos=PTR + 2), EINVAL),
          (dict(eps=-1.0), EINVAL), (dict(eps=NAN), EINVAL)]
QUANT = [(dict(x=None), EINVAL), (dict(codes=None), EINVAL), (dict(scales=None), EINVAL), (dict(format=2), EUNSUP),
         (dict(dtype=3), EUNSUP), (dict(rows=-1), EINVAL), (dict(cols=0), EINVAL), (dict(scale=-1.0), EINVAL),
         (dict(scale=NAN), EINVAL), (dict(scale=1e-10), EINVAL), (dict(scale=2e9), EINVAL), (dict(codes=PTR + 8), EINVAL),
         (dict(scales=PTR + 4), EINVAL), (dict(codes_row=16), EINVAL), (dict(codes_row=40), EINVAL), (dict(x_row=-64), EINVAL),
         (dict(values=PTR, values_row=63), EINVAL), (dict(x=PTR + 1), EINVAL), (dict(rows=1 << 24), EUNSUP),
         (dict(cols=2 ** 31 - 1, codes_row=1 << 30), EUNSUP)]
GEMM = [(dict(x=None), EINVAL), (dict(xscale=None), EINVAL), (dict(w=None), EINVAL), (dict(wscale=None), EINVAL),
        (dict(y=None), EINVAL), (dict(w2=PTR), EINVAL), (dict(w2scale=PTR), EINVAL),
        (dict(w2=PTR, w2scale=PTR, bias=PTR), EINVAL), (dict(format=-1), EUNSUP), (dict(dtype=2), EUNSUP),
        (dict(rows=-1), EINVAL), (dict(n=0), EINVAL), (dict(k=0), EINVAL), (dict(x_row=48), EINVAL), (dict(w_row=72), EINVAL),
        (dict(x_row=-64), EINVAL), (dict(y_row=9), EINVAL), (dict(k=129, x_row=64), EINVAL), (dict(x=PTR + 8), EINVAL),
        (dict(wscale=PTR + 8), EINVAL), (dict(y=PTR + 1), EINVAL), (dict(bias=PTR + 2), EINVAL), (dict(alpha=NAN), EINVAL),
        (dict(alpha2=NAN), EINVAL), (dict(k=2 ** 31 - 1, x_row=1 << 30, w_row=1 << 30), EUNSUP), (dict(w_row=1 << 40), EINVAL)]
SAMPLE = [(dict(logits=None), EINVAL), (dict(token=None), EINVAL), (dict(dtype=2), EUNSUP), (dict(rows=-1), EINVAL),
          (dict(n=0), EINVAL), (dict(row=99), EINVAL), (dict(n=262145, row=262145), EUNSUP), (dict(logits=PTR + 1), EINVAL),
          (dict(logits=PTR + 2, dtype=3), EINVAL), (dict(u=PTR + 2), EINVAL), (dict(token=PTR + 1), EINVAL),
          (dict(top_k=PTR + 3), EINVAL), (dict(rows=1 << 25), EUNSUP)]


@pytest.mark.parametrize("name,make,kw,want", [("yk_qk_rotate", rotate, *p) for p in ROTATE] + [("yk_quant_fp4", quant, *p) for p in QUANT] +
                         [("yk_gemm_fp4", gemm, *p) for p in GEMM] + [("yk_sample", sample, *p) for p in SAMPLE])
def test_arguments(lib, name, make, kw, want):
    from yolo11_cu_b200 import runtime as rt
    before = lib.yk_launch_count()
    a = make(rt, **kw)
    assert getattr(lib, name)(C.byref(a), None) == want
    assert lib.yk_last_cuda_error().decode()
    assert getattr(lib, name)(None, None) == EINVAL
    assert lib.yk_launch_count() == before


def test_no_rows_is_no_launch(lib):
    from yolo11_cu_b200 import runtime as rt
    before = lib.yk_launch_count()
    for name, make in (("yk_qk_rotate", rotate), ("yk_quant_fp4", quant), ("yk_gemm_fp4", gemm), ("yk_sample", sample)):
        a = make(rt, rows=0)
        assert getattr(lib, name)(C.byref(a), None) == 0
    assert lib.yk_launch_count() == before


def test_scale_bytes(lib):
    size = lib.yk_fp4_scale_bytes
    assert size(1, 1, 0) == 512 and size(128, 64, 0) == 512 and size(129, 65, 0) == 4 * 512
    assert size(128, 128, 1) == 512 and size(1, 129, 1) == 1024
    assert size(2 ** 31 - 1, 2 ** 31 - 1, 0) == 2 ** 24 * 2 ** 25 * 512
    assert [size(0, 1, 0), size(1, 0, 0), size(-1, 1, 1), size(1, 1, 2), size(1, 1, -1)] == [0] * 5


def test_hooks_refuse(lib):
    assert lib.yk_test_gemm_fp4(3, 0) == EINVAL and lib.yk_test_gemm_fp4(1, 3) == EINVAL
    assert lib.yk_test_sample(16) == EINVAL and lib.yk_test_sample(-1) == EINVAL
    assert lib.yk_test_gemm_fp4(0, 0) == 0 and lib.yk_test_sample(0) == 0


def test_kernel_hook_of_sampling():
    from yolo11_cu_b200 import runtime as rt
    lib = rt.load()
    assert lib.yk_test_sample_kernel(-1) == EINVAL and lib.yk_test_sample_kernel(3) == EINVAL
    assert lib.yk_test_sample_kernel(2) == 0 and lib.yk_test_sample_kernel(0) == 0
