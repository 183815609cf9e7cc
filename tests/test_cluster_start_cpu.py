"""A CTA may touch another CTA's shared memory only once that one has started, which a barrier of the cluster tells: read
from the sources of the kernels that write to a cluster's other CTAs (a miss shows on a GPU only now and then)."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yolo11.cu_b200", "csrc")


def kernel(source, name):
    text = open(os.path.join(CSRC, source)).read()
    text = re.sub(r"//[^\n]*", "", text)
    start = re.search(r"\b" + name + r"\(const __grid_constant__[^{]*\{", text).end()
    depth, at = 1, start
    while depth:
        depth += {"{": 1, "}": -1}.get(text[at], 0)
        at += 1
    return text[start:at]


@pytest.mark.parametrize("source,name", [("sample.cu", "sample_kernel"), ("sample16.cuh", "sample16_kernel")])
def test_sampling_waits_for_its_cluster_before_it_writes_there(source, name):
    body = kernel(source, name)
    first = body.index("tell(0,")                    # the first call of the lambda that writes to the other CTAs
    before = body[:first]
    assert before.count("cluster_arrive()") == 1 and before.count("cluster_wait()") == 1
    assert before.index("cluster_arrive()") < before.index("cluster_wait()")
    # neither half hides in a lambda, behind a return or in a branch that only some threads of a CTA take
    for half in ("cluster_arrive()", "cluster_wait()"):
        head = before[:before.index(half)]
        assert re.search(r"if \((a\.)?split > 1\)\s*(\{\s*__syncwarp\(\);\s*)?$", head), half
        assert "return;" not in head
    # what stands between the definitions and this wait meets no other CTA
    assert not re.search(r"(?<!\w)meet\(\);", before[before.index("cluster_arrive()"):].split("const auto tell")[0])


@pytest.mark.parametrize("source,name", [("gemm_fp4.cu", "gemm_fp4_pair_kernel"), ("gemm_fp4.cu", "gemm_fp4_split_kernel")])
def test_products_meet_before_they_reach_across(source, name):
    body = kernel(source, name)
    assert body.index("cluster_barrier()") < body.index("cluster_map(")
