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


def behind(dec, places, lens):
    counts = torch.tensor(lens)
    owner = torch.repeat_interleave(torch.arange(3), counts)
    return dec._behind(torch.tensor(places, dtype=torch.int32).reshape(3, -1), owner, counts, sum(lens)).tolist(), dec._shift.tolist()


def test_places_behind_an_image(dec):
    """Text follows the image rows before it in the call by one place; where there are none, its token's number and its request's
    shift.  Image rows lie where the caller puts them."""
    dec.lens.copy_(torch.tensor([0, 5, 9]))
    dec.shift.copy_(torch.tensor([0, 0, -4]))
    t, r, c = [-1, 2, 2, -1, -1, -1], [-1, 2, 3, -1, -1, -1], [-1, 2, 6, -1, -1, -1]
    got, shift = behind(dec, [t, r, c], [5, 0, 1])
    assert got == [[0, 2, 2, 7, 8, 5], [0, 2, 3, 7, 8, 5], [0, 2, 6, 7, 8, 5]]
    assert shift == [7 - 3, 0, -4]                   # the next token, number 5, lies at 9
    # an image that the caller puts before earlier places: text follows that image
    got, shift = behind(dec, [[-1, 0, 1, -1], [-1, 0, 0, -1], [-1, 1, 0, -1]], [0, 4, 0])
    assert got[0] == [5, 0, 1, 2] and shift == [0, 2 - 8, -4]
    # two images in one call: the larger places count
    got, shift = behind(dec, [[10, 3, -1]] * 3, [0, 0, 3])
    assert got[0] == [10, 3, 11] and shift == [0, 0, 11 - 11]


def test_places_of_no_rows(dec):
    dec.shift.copy_(torch.tensor([1, 2, 3]))
    got, shift = behind(dec, [], [0, 0, 0])
    assert got == [[], [], []] and shift == [1, 2, 3]
