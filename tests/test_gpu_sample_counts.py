"""A CTA of the kernel that counts 16-bit scores by place, with as many equal scores as it can have: rows of one CTA's and two CTAs'
most scores and one more, at every alignment of their start (which moves the CTAs' parts)."""
import math

import pytest
import torch

from test_gpu_decode import ok, run_sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [65023, 65024, 65025, 130047, 130048, 130049])
def test_equal_scores(lib, cuda, n):
    from yolo11_cu_b200 import runtime as rt
    for kernel in (0, 2):
        ok(lib, lib.yk_test_sample_kernel(kernel))
        for lead in (0, 1, 7):
            rows = torch.zeros(2, n + 16, dtype=torch.float16, device="cuda")
            x = rows[:, lead:lead + n]
            x[1] = 1.0009765625                      # (an odd place: the upper half of a word)
            for kw in (dict(top_k=[n - 1] * 2), dict(top_p=[0.75] * 2)):
                got = run_sample(lib, rt, x, u=[0.5] * 2, check=False, **kw)
                stay = n - 1 if "top_k" in kw else math.ceil(0.75 * n)
                assert got[2] == [stay] * 2 and got[0] == [stay // 2] * 2
                assert all(math.isclose(p, -math.log(stay), rel_tol=2.0 ** -23) for p in got[1])
