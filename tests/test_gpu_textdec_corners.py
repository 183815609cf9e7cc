"""TextDecoder at its ends: a new capture on request, scores without a choice."""
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


@pytest.mark.parametrize("weights", ["int4", "nvfp4"])
@pytest.mark.parametrize("graph", [False, True])
def test_scores_without_a_choice(lib, cuda, pkg, weights, graph):
    """A request whose scores are NaN keeps a token of its own and says so; the others do not notice."""
    def run(poison):
        dec = make(pkg, weights=weights)
        dec.set_sampling(0.8, top_k=50, seed=4)
        dec.prompt(rows_of(dec, 40), [10, 10, 10, 10])
        first = dec.decode(3, graph=graph)
        assert not dec.unscored.any()
        if poison:
            dec.res[1].fill_(float("nan"))
            dec.embed[dec.next[1]] = float("nan")
            assert (dec.next == dec.next[1]).sum() == 1
        mine = int(dec.next[1])
        after = [dec.decode(1, graph=graph)[0].tolist() + dec.unscored.tolist() for _ in range(3)]
        return mine, first, after, dec

    _, clean_first, clean, _ = run(False)
    mine, first, after, dec = run(True)
    assert torch.equal(first, clean_first)
    assert torch.isnan(dec.logits[1]).all() and not torch.isnan(dec.logits[[0, 2, 3]]).any()
    for a, b in zip(after, clean):
        assert [a[i] for i in (0, 2, 3)] == [b[i] for i in (0, 2, 3)]
        assert a[1] == mine                          # it went in (-1 would say that the plan refused it)
        assert a[4:] == [False, True, False, False] and b[4:] == [False] * 4
    assert int(dec.next[1]) == mine and dec.placed.all()
