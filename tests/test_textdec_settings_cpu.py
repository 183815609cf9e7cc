"""What TextDecoder keeps on the host's side of its calls: sampling settings, the captured step, the places of a prompt's rows
(plain tensor arithmetic, so it runs without a GPU)."""
import pytest
import torch


@pytest.fixture
def dec(pkg):
    """A decoder's state without its weights, cache and buffers."""
    from yolo11_cu_b200 import textdec
    d = textdec.TextDecoder.__new__(textdec.TextDecoder)
    d.requests, d.device, d.sampling, d.gen, d.graphs = 3, "cpu", None, None, {}
    d.unscored = torch.zeros(3, dtype=torch.bool)
    d.lens, d.shift = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    return d


def test_refused_settings_change_nothing(dec):
    dec.set_sampling([0.5, 1.0, 2.0], top_k=7, top_p=[0.9, 0.8, 0.7], min_p=0.1, seed=3)
    want = {k: v.clone() for k, v in dec.sampling.items()}
    state = dec.gen.get_state()
    for bad in (dict(top_p=[0.1, 0.2]), dict(top_k=[1, 2, 3, 4]), dict(min_p=[[0.1, 0.2, 0.3]])):
        with pytest.raises(ValueError):
            dec.set_sampling(3.0, **bad, seed=9)
        assert dec.sampling.keys() == want.keys() and all(torch.equal(dec.sampling[k], v) for k, v in want.items())
        assert torch.equal(dec.gen.get_state(), state)
    dec.set_sampling(None)
    with pytest.raises(ValueError):
        dec.set_sampling([1.0, 2.0])
    assert dec.sampling is None


def test_the_captured_step_can_be_let_go(dec):
    dec.graphs = {False: "greedy", True: "drawn"}
    assert dec.graph == "greedy"
    dec.set_sampling(1.0)
    assert dec.graph == "drawn"
    dec.graph = None                                 # what was captured is out of date, in both ways
    assert dec.graph is None and dec.graphs == {}
    dec.set_sampling(None)
    assert dec.graph is None
    dec.graph = "another"
    assert dec.graphs == {False: "another"}
