"""TextDecoder at its ends: a new capture on request."""
import pytest
import torch

from test_gpu_textdec_modes import make, rows_of

pytestmark = pytest.mark.gpu


def test_a_new_capture_on_request(lib, cuda, pkg):
    dec, eager = make(pkg), make(pkg)
    for d in (dec, eager):
        d.prompt(rows_of(d, 40), [10, 10, 10, 10])
    got = [dec.decode(2)]
    old = dec.graph
    dec.graph = None
    assert dec.graph is None
    got.append(dec.decode(3))
    assert dec.graph is not None and dec.graph is not old
    assert torch.equal(torch.cat(got), eager.decode(5, graph=False))
