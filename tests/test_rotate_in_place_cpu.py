"""yk_qk_rotate turns rows in place or from one place to another; the same start with another row stride is neither (a row's
output would cover rows that are still to be read), and is refused."""
import ctypes as C

import pytest

from test_decode_refusals_cpu import EINVAL, PTR, rotate


@pytest.mark.parametrize("kw", [dict(k_out=2 * PTR, q_out_row=512), dict(q_out=2 * PTR, k_out_row=256),
                                dict(k_out=2 * PTR, q_row=512, rows=2)])
def test_in_place_with_two_strides(lib, kw):
    from yolo11_cu_b200 import runtime as rt
    before = lib.yk_launch_count()
    a = rotate(rt, **(dict(pos_axis=3) | kw))
    assert lib.yk_qk_rotate(C.byref(a), None) == EINVAL
    assert b"in place" in lib.yk_last_cuda_error()
    assert lib.yk_launch_count() == before
