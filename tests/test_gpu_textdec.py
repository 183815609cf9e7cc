"""The text operators together, as TextDecoder runs them: every stage of a prompt and of the steps
after it against its plain form on the same inputs, and the captured step against the eager one.

Bounds on the relative error of a stage's whole output (2-norms): one rounding to fp16 is at most
2^-11 of each value (products, residual rows); attention rounds its weights too (2^-10 in all); norm
outputs compare as code * scale, whose scales carry fp32 errors (2^-20) while single codes may fall
to the other side of a rounding boundary: at most one in a thousand."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def dequant(w, group):
    q, s = w
    v = torch.stack([q & 15, q >> 4], 2).view(q.shape[0], -1).float() - 8
    return v * s.float().repeat_interleave(group, 1)


def norm8(x, w, eps):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()
    s = y.abs().amax(-1, keepdim=True) / 448
    return (y / s).clamp(-448, 448).to(F8).float() * s


def rel(a, b):
    return ((a.float() - b).norm() / b.norm()).item()


def check_norm(dec, weight, n):
    want = dec.res[:n].float() + dec.delta[:n].float()
    dec._norm(dec.delta, dec.res, weight, n)
    assert rel(dec.res[:n], want) <= 2.0 ** -11
    want = norm8(want, weight, dec.eps)
    x = dec.x8[:n].view(F8).float() * dec.xs[:n]
    assert ((x - want).abs() > 2.0 ** -20 * want.abs()).float().mean() <= 1e-3
    return x


def check_product(dec, x, given, w, y, n, scales=None):
    dec._matmul(given, w, y, n, scales)
    assert rel(y[:n], x @ dequant(w, dec.group).t()) <= 2.0 ** -11


def check_attention(dec, layer, n):
    dec._attend(layer, n)
    h, k, d = dec.heads, dec.kv_heads, dec.dim
    codes, scales = dec.codes[layer]
    cu, lens = dec.cu.tolist(), dec.lens.tolist()
    want = torch.zeros(n, h, d, device="cuda")
    for r in range(dec.requests):
        q0, q1, kv = cu[r], cu[r + 1], lens[r]
        if q1 == q0:
            continue
        ids = dec.table[r, :-(-kv // dec.block)].long()

        def held(part):
            v = codes[ids, part].view(F8).float() * scales[part][ids][..., None, None]
            return v.transpose(1, 2).reshape(-1, k, d)[:kv].repeat_interleave(h // k, 1)

        # what the cache holds is what was written: e4m3 of a power-of-two scale, 2^-4 of a value
        new = dec.qkv[q0:q1, h * d:].float().view(q1 - q0, 2, k, d)
        for part in (0, 1):
            err = (held(part)[kv - (q1 - q0):, ::h // k] - new[:, part]).abs()
            step = scales[part][ids][torch.arange(kv - (q1 - q0), kv, device="cuda") // dec.block][..., None]
            assert (err <= 2.0 ** -4 * new[:, part].abs() + 2.0 ** -10 * step).all()
        q = dec.qkv[q0:q1, :h * d].float().view(q1 - q0, h, d)
        a = torch.einsum("qhd,khd->hqk", q, held(0)) * d ** -0.5
        pos = torch.arange(kv - (q1 - q0), kv, device="cuda")
        a = a.masked_fill(torch.arange(kv, device="cuda")[None] > pos[:, None], float("-inf")).softmax(-1)
        want[q0:q1] = torch.einsum("hqk,khd->qhd", a, held(1))
    assert rel(dec.att[:n].view(n, h, d), want) <= 2.0 ** -10


def check_layers(dec, n):
    """TextDecoder._layers, each stage checked."""
    dec._plan(n)
    dec.res[:n] += dec.place[dec.pos[:n].clamp(min=0).long()]
    dec.delta[:n].zero_()
    for i, w in enumerate(dec.w):
        x = check_norm(dec, dec.norms[2 * i], n)
        check_product(dec, x, dec.x8, w["qkv"], dec.qkv, n, dec.xs)
        check_attention(dec, i, n)
        check_product(dec, dec.att[:n].float(), dec.att, w["out"], dec.delta, n)
        x = check_norm(dec, dec.norms[2 * i + 1], n)
        check_product(dec, x, dec.x8, w["up"], dec.up, n, dec.xs)
        dec.act[:n] = torch.nn.functional.silu(dec.up[:n, :dec.hidden]) * dec.up[:n, dec.hidden:]
        check_product(dec, dec.act[:n].float(), dec.act, w["down"], dec.delta, n)
    return check_norm(dec, dec.norms[-1], n)


def test_every_stage_matches_plain(lib, cuda, pkg):
    from yolo11_cu_b200 import textdec
    torch.backends.cuda.matmul.allow_tf32 = False
    lens = [37, 0, 5, 130]
    dec, ref = (textdec.TextDecoder(4, rows=256, max_tokens=512, pool=64) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = torch.randn(sum(lens), dec.width, generator=g, device="cuda").half()
    ref.prompt(rows, lens)
    for step in range(4):               # the prompt, then three tokens, one by one
        n = sum(lens) if step == 0 else 4
        if step == 0:
            dec.fresh.copy_(torch.tensor(lens, dtype=torch.int32))
            dec.res[:n].copy_(rows)
        else:
            dec.fresh.fill_(1)
            dec.res[:n].copy_(dec.embed[ref.next])
            ref.decode(1, graph=False)
        x = check_layers(dec, n)
        last = (dec.cu[1:].long() - 1).clamp(min=0)
        assert rel(ref.logits, x[last] @ dequant(dec.head, dec.group).t()) <= 2.0 ** -11
        assert dec.lens.tolist() == [m + step for m in lens]
    assert int(dec.counts[2]) == 0


def test_captured_steps_equal_eager_steps(lib, cuda, pkg):
    from yolo11_cu_b200 import textdec
    out = []
    for graph in (False, True):
        dec = textdec.TextDecoder(4, rows=128, max_tokens=256, pool=40, seed=3)
        rows = torch.randn(60, dec.width, generator=torch.Generator().manual_seed(2)).cuda().half()
        dec.prompt(rows, [30, 0, 29, 1])
        out.append((dec.decode(40, graph=graph), dec.logits.clone(), dec.taken.clone(), dec.lens.clone()))
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_pool_runs_dry(lib, cuda, pkg):
    """Too few blocks: the last request is refused, its length stays, the others go on."""
    from yolo11_cu_b200 import textdec
    dec = textdec.TextDecoder(3, rows=128, max_tokens=256, pool=3, seed=3)
    rows = torch.randn(96, dec.width, generator=torch.Generator().manual_seed(2)).cuda().half()
    dec.prompt(rows, [32, 32, 32])
    dec.decode(2, graph=False)
    assert dec.lens.tolist() == [32, 32, 32] and int(dec.counts[2]) == 3
    with pytest.raises(ValueError):
        dec.prompt(rows, [32, 32])


def test_example_runs(lib, cuda, pkg, capsys):
    from yolo11_cu_b200 import textdec
    textdec.main(["--frames", "2", "--steps", "4"])
    assert "400 image tokens" in capsys.readouterr().out


@pytest.mark.parametrize("graph", [False, True])
def test_full_requests_stop(lib, cuda, pkg, graph):
    """A request that holds all the blocks of its table is refused from then on and keeps its length;
    the others go on.  max_tokens is no multiple of the block: the last block is used to its end."""
    from yolo11_cu_b200 import textdec
    dec = textdec.TextDecoder(2, rows=300, max_tokens=100, pool=16, seed=3)
    rows = torch.randn(300, dec.width, generator=torch.Generator().manual_seed(2)).cuda().half()
    dec.prompt(rows[:216], [90, 126])
    dec.decode(2, graph=graph)
    assert dec.lens.tolist() == [92, 128] and int(dec.counts[2]) == 0
    for step in range(1, 4):
        dec.decode(1, graph=graph)
        assert dec.lens.tolist() == [92 + step, 128] and int(dec.counts[2]) == 1
    dec.prompt(rows[:200], [200, 0])            # a prompt past the table's end
    assert dec.lens.tolist() == [95, 128] and int(dec.counts[2]) == 1
    torch.cuda.synchronize()


@pytest.mark.parametrize("graph", [False, True])
def test_admission_leaves_other_requests_alone(lib, cuda, pkg, graph):
    """Prompts of other requests in the middle of a request's generation: its pending token stays, and
    its tokens are those of a run without them."""
    from yolo11_cu_b200 import textdec
    rows = torch.randn(71, 512, generator=torch.Generator().manual_seed(2)).cuda().half()
    runs = []
    for admit in (False, True):
        dec = textdec.TextDecoder(3, rows=64, max_tokens=256, pool=30, seed=3)
        dec.prompt(rows[:30], [0, 30, 0])
        ids = [dec.decode(3, graph=graph)]
        pending = int(dec.next[1])
        if admit:
            dec.prompt(rows[30:], [20, 0, 21])
            assert int(dec.next[1]) == pending
            dec.prompt(rows[:0], [0, 0, 0])
            assert int(dec.next[1]) == pending
        ids.append(dec.decode(5, graph=graph))
        runs.append(torch.cat(ids)[:, 1].tolist())
    assert runs[0] == runs[1]


@pytest.mark.parametrize("lens,last", [([5, 0, 7], [4, None, 11]), ([0, 3, 0], [None, 2, None]), ([0, 0, 1], [None, None, 0])])
def test_a_prompt_picks_from_its_own_last_row(lib, cuda, pkg, lens, last):
    from yolo11_cu_b200 import textdec
    dec = textdec.TextDecoder(3, rows=64, max_tokens=256, pool=30, seed=3)
    dec.next.copy_(torch.tensor([11, 22, 33]))
    rows = torch.randn(sum(lens), dec.width, generator=torch.Generator().manual_seed(2)).cuda().half()
    dec.prompt(rows, lens)
    for r, row in enumerate(last):
        if row is None:
            assert int(dec.next[r]) == [11, 22, 33][r]
            continue
        x = dec.x8[row].view(F8).float() * dec.xs[row]
        want = dequant(dec.head, dec.group) @ x
        # fp16 scores: the picked one is the largest but for two roundings
        assert want[dec.next[r]] >= want.max() - 2 * 2.0 ** -11 * want.abs().max()


@pytest.mark.parametrize("graph", [False, True])
def test_refused_requests_keep_their_token(lib, cuda, pkg, graph):
    """A step that the pool refuses a request gives it no token (-1) and keeps the one that waits; once there
    are blocks again, that one goes in."""
    from yolo11_cu_b200 import textdec
    rows = torch.randn(95, 512, generator=torch.Generator().manual_seed(2)).cuda().half()
    free, dec = (textdec.TextDecoder(3, rows=128, max_tokens=256, pool=p, seed=3) for p in (30, 4))
    for d in (free, dec):
        d.prompt(rows, [32, 31, 32])
        assert d.placed.tolist() == [True] * 3
    start = dec.next.tolist()
    want = free.decode(3, graph=graph).tolist()
    assert want[0] == start
    assert dec.decode(1, graph=graph).tolist() == [[start[0], start[1], -1]]      # the last block goes to request 0
    assert dec.placed.tolist() == [True, True, False] and dec.lens.tolist() == [33, 32, 32]
    assert int(dec.next[2]) == start[2]
    waits = int(dec.next[1])
    assert dec.decode(2, graph=graph).tolist() == [[want[1][0], -1, -1], [want[2][0], -1, -1]]
    assert dec.next.tolist()[1:] == [waits, start[2]] and dec.lens.tolist() == [35, 32, 32]
    # request 0 leaves; its two blocks are free again
    dec.lens[0] = 0
    dec.free[2:4] = dec.table[0, :2]
    dec.taken.fill_(2)
    got = dec.decode(1, graph=graph).tolist()
    assert got[0][1:] == [waits, -1] and dec.lens.tolist() == [1, 33, 32]
    # a prompt that does not fit changes nothing either
    dec.prompt(rows[:60], [0, 0, 60])
    assert dec.placed.tolist() == [False] * 3 and int(dec.next[2]) == start[2] and int(dec.lens[2]) == 32
