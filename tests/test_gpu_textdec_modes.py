"""TextDecoder with 4-bit float products, rotary places and sampling: its stages against their definitions on the same
inputs, and the captured step against the eager one.

Bounds: one rounding to fp16 of a product is 2^-11 of the value (2-norms), of a norm's output likewise; tokens are exact."""
import numpy as np
import pytest
import torch

import decode_ref as ref

pytestmark = pytest.mark.gpu


def f64(t):
    return t.double().cpu().numpy()


def rel(a, b):
    return np.linalg.norm(a - b) / np.linalg.norm(b)


def make(pkg, **kw):
    from yolo11_cu_b200 import textdec
    kw = dict(rows=256, max_tokens=512, pool=64, seed=3) | kw
    return textdec.TextDecoder(kw.pop("requests", 4), **kw)


def matrix(m):
    """64-bit values of an Fp4."""
    codes = m.codes.cpu().numpy()
    q = np.stack([codes & 15, codes >> 4], 2).reshape(m.rows, -1)[:, :m.cols]
    g = -(-m.cols // ref.GROUP[m.fmt])
    s = m.scales.cpu().numpy()[ref.scale_at(m.rows, g)]
    return ref.values(q, s, m.cols, m.fmt) * m.scale


def rows_of(dec, n, seed=2):
    return torch.randn(n, dec.width, generator=torch.Generator().manual_seed(seed)).cuda().half()


@pytest.mark.parametrize("weights", ["nvfp4", "mxfp4"])
def test_products(lib, cuda, pkg, weights):
    dec = make(pkg, weights=weights)
    n = 37
    x = rows_of(dec, n)
    w = dec.w[1]
    dec._linear4(x, w["qkv"], dec.qkv, n)
    q, s, v = ref.quant(x.float().cpu().numpy(), dec.fp4, dec.x4[dec.width].scale)
    assert rel(f64(dec.qkv[:n]), v @ matrix(w["qkv"]).T) <= 2.0 ** -11
    dec._linear4(x, w["up"], dec.act, n, gate=w["gate"])
    assert rel(f64(dec.act[:n]), ref.silu(v @ matrix(w["gate"]).T) * (v @ matrix(w["up"]).T)) <= 2.0 ** -11
    y = dec.act[:n].clone()
    dec._linear4(dec.act, w["down"], dec.delta, n)
    v = ref.quant(y.float().cpu().numpy(), dec.fp4, dec.x4[dec.hidden].scale)[2]
    assert rel(f64(dec.delta[:n]), v @ matrix(w["down"]).T) <= 2.0 ** -11


def test_four_bit_weights_are_near_the_sixteen_bit_ones(lib, cuda, pkg):
    """A group's values are rounded by at most 1 / 6 of its largest and the scale's 2^-4; the weights are the seed's in all formats."""
    mats = [make(pkg, weights=w).w[0]["qkv"] for w in ("nvfp4", "mxfp4")]
    assert rel(matrix(mats[0]), matrix(mats[1])) < 0.25


@pytest.mark.parametrize("weights", ["int4", "nvfp4"])
def test_places_of_image_and_text(lib, cuda, pkg, weights):
    dec = make(pkg, weights=weights, rotary=True, requests=3)
    grid = torch.stack([torch.zeros(20), torch.arange(20) // 5, torch.arange(20) % 5]).int()     # 4 x 5 tokens
    text = torch.full((3, 3), -1, dtype=torch.int32)
    lens = [26, 0, 4]
    dec.prompt(rows_of(dec, 30), lens, torch.cat([text, grid + 3, text, text, text[:, :1]], 1))
    want = [[0, 1, 2] + [3] * 20 + [8, 9, 10], [0, 1, 2] + [3 + i // 5 for i in range(20)] + [8, 9, 10],
            [0, 1, 2] + [3 + i % 5 for i in range(20)] + [8, 9, 10]]
    for a in range(3):
        assert dec.at[a, :30].tolist() == want[a] + [0, 1, 2, 3]
    assert dec.shift.tolist() == [8 - 23, 0, 0]
    dec.decode(2, graph=False)
    assert dec.at[:, :3].tolist() == [[12, 1, 5]] * 3
    # rows are turned by these places
    before = rows_of(dec, 3, seed=9)[:, :1].repeat(1, dec.qkv.shape[1]) * torch.arange(1, dec.qkv.shape[1] + 1, device="cuda").half() * 0.01
    dec.qkv[:3] = before
    dec._rotate(0, 3)
    h, d, k = dec.heads, dec.dim, dec.kv_heads
    for lo, heads, w in ((0, h, 0), (h * d, k, 1)):
        x = f64(before[:, lo:lo + heads * d]).reshape(3, heads, d)
        y, big = ref.rotate(x, f64(dec.head_norms[0][w]), dec.at[:, :3].cpu().numpy(), dec.freqs.cpu().numpy(), dec.sections[:3], d,
                            False, dec.eps)
        got = f64(dec.qkv[:3, lo:lo + heads * d]).reshape(3, heads, d)
        assert (np.abs(got - y) <= 2.0 ** -11 * np.abs(y) + 2.0 ** -19 * big + 2.0 ** -25).all()
    assert torch.equal(dec.qkv[:3, (h + k) * d:], before[:, (h + k) * d:])
    # a second image in the same request; a request that is refused keeps its shift
    dec.prompt(rows_of(dec, 25), [25, 0, 0], torch.cat([text, grid, text[:, :2]], 1))
    assert dec.at[0, :25].tolist() == [13, 14, 15] + [0] * 20 + [5, 6]
    shift = dec.shift.tolist()
    dec.free.fill_(0)
    dec.taken.fill_(dec.pool)
    dec.prompt(rows_of(dec, 60), [0, 0, 60], torch.cat([grid] * 3, 1))
    assert dec.shift.tolist() == shift and dec.placed.tolist() == [False] * 3


@pytest.mark.parametrize("kw", [dict(rotary=True), dict(weights="nvfp4"), dict(weights="mxfp4", rotary=True)])
@pytest.mark.parametrize("temperature", [None, 0.8])
def test_captured_steps_equal_eager_steps(lib, cuda, pkg, kw, temperature):
    out = []
    for graph in (False, True):
        dec = make(pkg, **kw)
        dec.set_sampling(temperature, top_k=50, top_p=0.9, seed=5)
        dec.prompt(rows_of(dec, 60), [30, 0, 29, 1])
        out.append((dec.decode(30, graph=graph), dec.logits.clone(), dec.taken.clone(), dec.lens.clone()))
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("graph", [False, True])
def test_sampled_tokens_are_the_definitions(lib, cuda, pkg, graph):
    dec = make(pkg)
    settings = dict(temperature=[0.7, 0.0, 1.5, 1.0], top_k=[0, 5, 40, 3], top_p=[0.9, 1.0, 0.8, 1.0], min_p=[0.0, 0.0, 0.05, 0.0])
    dec.set_sampling(**settings, seed=11)
    dec.prompt(rows_of(dec, 40), [10, 10, 10, 10])
    near = []
    for _ in range(12):
        given = dec.next.clone()
        assert torch.equal(dec.decode(1, graph=graph)[0], given)
        scores, u = f64(dec.logits), f64(dec.u)
        for r in range(4):
            want = ref.sample(scores[r], *(float(np.float32(settings[k][r])) if k != "top_k" else settings[k][r]
                                           for k in ("temperature", "top_k", "top_p", "min_p")), u[r])
            near.append(want[3])
            assert int(dec.next[r]) == want[0]
            assert abs(float(dec.logprob[r]) - want[1]) <= 2.0 ** -23 * abs(want[1]) + 1e-9
    assert min(near) > 1e-9


def test_settings_change_without_a_new_capture(lib, cuda, pkg):
    dec, best = make(pkg), make(pkg)
    for d in (dec, best):
        d.prompt(rows_of(d, 40), [10, 10, 10, 10])
    dec.set_sampling(5.0, seed=1)
    drawn = dec.decode(8)
    captured = dec.graph
    want = best.decode(8)
    assert captured is not None and not torch.equal(drawn, want)
    dec = make(pkg)
    dec.prompt(rows_of(dec, 40), [10, 10, 10, 10])
    dec.set_sampling(3.0, seed=1)
    dec.decode(2)
    captured = dec.graph
    for d in (dec, best):
        d.next.copy_(torch.tensor([1, 2, 3, 4]))
        d.lens.fill_(10)
    dec.set_sampling(0.0)
    assert dec.graph is captured
    got, want = dec.decode(6), best.decode(6)
    assert torch.equal(got, want)
    dec.set_sampling(None)
    assert dec.graph is None


def test_refusals(lib, cuda, pkg):
    from yolo11_cu_b200 import textdec
    with pytest.raises(ValueError, match="weights"):
        textdec.TextDecoder(1, weights="int3")
    dec = make(pkg)
    with pytest.raises(ValueError, match="temperature"):
        dec.set_sampling([0.1, 0.2])
    with pytest.raises(ValueError, match="rotary"):
        dec.prompt(rows_of(dec, 4), [1] * 4, torch.zeros(3, 4))
    dec = make(pkg, rotary=True)
    with pytest.raises(ValueError, match="places"):
        dec.prompt(rows_of(dec, 4), [1] * 4, torch.zeros(2, 4))


@pytest.mark.parametrize("flags", [["--weights", "nvfp4", "--rotary", "--temperature", "0.8", "--top-k", "40", "--top-p", "0.95"],
                                   ["--weights", "mxfp4", "--min-p", "0.1", "--temperature", "1"]])
def test_example_runs(lib, cuda, pkg, capsys, flags):
    from yolo11_cu_b200 import textdec
    textdec.main(["--frames", "2", "--steps", "4"] + flags)
    assert "400 image tokens" in capsys.readouterr().out
