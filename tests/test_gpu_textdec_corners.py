"""TextDecoder at its ends: scores without a choice, a new capture on request, 4-bit rows of every size, 4-bit weights beside the
16-bit ones.

Bounds.  A scale of e4m3 is within 2^-4 of a group's largest value over 6, so it is at most 17/96 of that value, and a code is off by
at most one unit of it (between 4 and 6; what exceeds 6 exceeds it by 0.4).  A power-of-two scale is at most twice a sixth: 1/3.  The
16-bit weights are 2^-11 off the seed's."""
import numpy as np
import pytest
import torch

import decode_ref as ref
from test_gpu_textdec_modes import f64, make, matrix, rows_of

pytestmark = pytest.mark.gpu
UNIT = {"nvfp4": 17 / 96, "mxfp4": 1 / 3}


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


@pytest.mark.parametrize("weights", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("size", [2.0 ** -6, 0.1, 1.0, 16.0])
def test_rows_of_every_size_in_four_bits(lib, cuda, pkg, weights, size):
    """Attention over a long cache is small, a norm's rows are about one, a gate's product may be large."""
    dec = make(pkg, weights=weights)
    for cols, m in dec.x4.items():
        x = (torch.randn(40, cols, generator=torch.Generator().manual_seed(cols)).cuda() * size).half()
        dec._ok(m.fill(dec.lib, x, 40))
        v = f64(x)
        g = ref.GROUP[dec.fp4]
        largest = np.repeat(np.abs(v).reshape(40, -1, g).max(-1), g, 1)
        assert largest.min() >= 6 * 2.0 ** -6 * m.scale or weights == "mxfp4", "below the scale's normal range"
        assert (np.abs(matrix(m)[:40] - v) <= UNIT[weights] * largest).all()


@pytest.mark.parametrize("weights", ["nvfp4", "mxfp4"])
def test_weights_are_the_seeds_in_four_bits(lib, cuda, pkg, weights):
    dec = make(pkg, weights=weights)
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = (dec.heads + 2 * dec.kv_heads) * dec.dim
    sizes = dict(qkv=(wide, dec.width), out=(dec.width, dec.heads * dec.dim), up=(dec.hidden, dec.width),
                 down=(dec.width, dec.hidden), gate=(dec.hidden, dec.width))
    seen = [(w[k], torch.randn(*s, generator=g, device="cuda") * s[1] ** -0.5) for w in dec.w for k, s in sizes.items()]
    for _ in dec.norms:                              # (drawn whole for each of them)
        torch.randn(2 * dec.layers + 1, dec.width, generator=g, device="cuda")
    seen.append((dec.head, torch.randn(dec.vocab, dec.width, generator=g, device="cuda") * dec.width ** -0.5))
    for m, w in seen:
        v = f64(w)
        n = ref.GROUP[dec.fp4]
        largest = np.repeat(np.abs(v).reshape(m.rows, -1, n).max(-1), n, 1)
        # (the group's largest is rounded to 16 bits, too)
        assert (np.abs(matrix(m) - v) <= (UNIT[weights] + 2.0 ** -10) * largest + 2.0 ** -25).all()
