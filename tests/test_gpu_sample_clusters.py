"""Rows of scores shared by the CTAs of a cluster, most of which have no score: they reach the first exchange at once, so
that it may not begin before all have started.  Results are those of one CTA a row, bit for bit."""
import pytest
import torch

from test_gpu_decode import TYPES, ok, run_sample, the_librarys_rules  # noqa: F401 (a fixture of every test here)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("n", [1, 9, 300, 2049])
def test_ctas_without_scores(lib, cuda, n, kernel, t):
    from yolo11_cu_b200 import runtime as rt
    g = torch.Generator().manual_seed(n)
    m = 1500
    x = torch.randn(m, n + 1, generator=g).to(TYPES[t][0]).cuda()[:, :n]
    u = torch.rand(m, generator=g).tolist()
    runs = []
    try:
        ok(lib, lib.yk_test_sample_kernel(kernel))
        for split in (1, 2, 4, 8):
            ok(lib, lib.yk_test_sample(split))
            runs.append(run_sample(lib, rt, x, u=u, top_p=[0.9] * m, top_k=[0, n // 2 + 1] * (m // 2), check=False))
            runs.append(run_sample(lib, rt, x, check=False))
    finally:
        ok(lib, lib.yk_test_sample_kernel(0))
    assert all(r == runs[0] for r in runs[2::2]) and all(r == runs[1] for r in runs[3::2])
    want = x.float().argmax(1).tolist()
    assert runs[1][0] == want and runs[1][1] == [0.0] * m
