"""Measured cases of the decoder's rotation, 4-bit float and sampling operators: inputs, plain forms, 64-bit definitions.

Four operators of the text decoder: the norm and rotary position of queries and keys
(``yk_qk_rotate``), the quantisation of rows to 4-bit floats with a scale for each small group of
columns (``yk_quant_fp4``), the product of two such matrices, plain or gated (``yk_gemm_fp4``), and
the choice of the next token (``yk_sample``).  ``run`` computes a case in elementary torch operations,
or, with ``own`` set, through the library's C ABI as a C or Python caller does: descriptors filled
once over buffers that the program keeps, one call a pass.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_F8 = torch.float8_e4m3fn
_E8 = torch.float8_e8m0fnu
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_GROUP = {"nv": 16, "mx": 32}       # columns of a scale: e4m3 scales, power-of-two scales
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _runtime():
    """The package's ctypes binding (the package directory's name has a dot: loaded by path)."""
    if "yolo11_cu_b200" not in sys.modules:
        pkg = os.path.join(_ROOT, "yolo11.cu_b200")
        spec = importlib.util.spec_from_file_location(
            "yolo11_cu_b200", os.path.join(pkg, "__init__.py"), submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["yolo11_cu_b200"] = mod
        spec.loader.exec_module(mod)
    from yolo11_cu_b200 import runtime
    return runtime


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a full batch: new tokens at far positions of a long cache
        {"name": "rotate decode 64", "op": "rotate", "rows": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "axes": 1, "inter": 0, "norm": 1, "far": 262143, "type": "f16"},
        # the 400 image tokens of 30 frames, each at its frame, row and column
        {"name": "rotate 30 frames", "op": "rotate", "rows": 12000, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "axes": 3, "inter": 0, "norm": 1, "far": 5000, "type": "bf16"},
        # a small model's ragged prompt: half of each head rotates, neighbouring pairs, odd head counts
        {"name": "rotate 3001 partial", "op": "rotate", "rows": 3001, "heads": 7, "kv_heads": 1, "dim": 64,
         "rot": 32, "axes": 1, "inter": 1, "norm": 0, "far": 40000, "type": "f16"},
        # rows of a decode batch before a product
        {"name": "quant 16 x 4096", "op": "quant", "rows": 16, "cols": 4096, "fmt": "nv", "type": "f16"},
        # rows of a large batch of prompts
        {"name": "quant 12000 x 5120", "op": "quant", "rows": 12000, "cols": 5120, "fmt": "mx", "type": "bf16"},
        # one token through a square projection: the smallest product, latency counts
        {"name": "gemm 1 x 4096 x 4096", "op": "gemm", "rows": 1, "n": 4096, "k": 4096, "gated": 0, "bias": 1,
         "fmt": "nv", "type": "f16"},
        # a decode batch through a wide projection: the weights' bytes count
        {"name": "gemm 16 x 28672 x 8192", "op": "gemm", "rows": 16, "n": 28672, "k": 8192, "gated": 0, "bias": 0,
         "fmt": "nv", "type": "bf16"},
        # prompts through a projection: operations count
        {"name": "gemm 2048 x 8192 x 8192", "op": "gemm", "rows": 2048, "n": 8192, "k": 8192, "gated": 0, "bias": 0,
         "fmt": "nv", "type": "bf16"},
        # ragged prompts through the gated half of a feed-forward block, sizes off every tile
        {"name": "gated 777 x 11000 x 4000", "op": "gemm", "rows": 777, "n": 11000, "k": 4000, "gated": 1, "bias": 0,
         "fmt": "mx", "type": "f16"},
        # one request's next token
        {"name": "sample 1 x 32000", "op": "sample", "rows": 1, "n": 32000, "top_k": 50, "top_p": 0.95, "min_p": 0.0,
         "mixed": 0, "type": "f16"},
        # a decode batch, one setting for all
        {"name": "sample 64 x 128000", "op": "sample", "rows": 64, "n": 128000, "top_k": 0, "top_p": 0.9, "min_p": 0.0,
         "mixed": 0, "type": "bf16"},
        # a large batch, every request with settings of its own (some greedy)
        {"name": "sample 200 x 151000", "op": "sample", "rows": 200, "n": 151000, "top_k": 200, "top_p": 0.95,
         "min_p": 0.02, "mixed": 1, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["rotate", "quant", "gemm", "gemm", "sample"])
        c = {"op": op}
        if op == "rotate":
            kvh = rng.choice([1, 2, 4, 8])
            dim = rng.choice([64, 128, 128, 256])
            c |= {"rows": _log(rng, 1, 12000), "heads": kvh * rng.choice([1, 2, 4, 5, 7]), "kv_heads": kvh, "dim": dim,
                  "rot": rng.choice([dim, dim, dim // 2]), "axes": rng.choice([1, 3]), "inter": rng.choice([0, 0, 1]),
                  "norm": rng.choice([0, 1, 1]), "far": _log(rng, 64, 262143), "type": rng.choice(["f16", "bf16"])}
        elif op == "quant":
            c |= {"rows": _log(rng, 1, 12000), "cols": _log(rng, 64, 16384), "fmt": rng.choice(["nv", "mx"]),
                  "type": rng.choice(["f16", "bf16"])}
        elif op == "gemm":
            c |= {"rows": _log(rng, 1, 2048), "n": _log(rng, 64, 28672), "k": _log(rng, 128, 8192),
                  "gated": rng.choice([0, 0, 1]), "fmt": rng.choice(["nv", "mx"]), "type": rng.choice(["f16", "bf16"])}
            c["bias"] = 0 if c["gated"] else rng.choice([0, 1])
        else:
            c |= {"rows": _log(rng, 1, 200), "n": _log(rng, 1000, 250000), "top_k": rng.choice([0, 0, _log(rng, 1, 1000)]),
                  "top_p": rng.choice([1.0, 0.95, 0.9, 0.6]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]),
                  "mixed": rng.choice([0, 1]), "type": rng.choice(["f16", "bf16", "f32"])}
        w = work(c)
        if w["bytes"] <= {"rotate": 2.5e8, "quant": 2.9e8, "gemm": 1.6e8, "sample": 1.3e8}[op] and w["flops"] < 2.8e11:
            return c


def _cdiv(a, b):
    return -(-a // b)


def work(c):
    if c["op"] == "rotate":
        n = c["rows"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        return {"bytes": 4.0 * n + 4.0 * c["rows"] * c["axes"] + 4.0 * c["dim"] * c["norm"] + 2.0 * c["rot"],
                "flops": 6.0 * n}
    if c["op"] == "quant":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (2.0 + 0.5 + 2.0) + c["rows"] * _cdiv(c["cols"], _GROUP[c["fmt"]]), "flops": 3.0 * n}
    if c["op"] == "gemm":
        m, n, k = c["rows"], c["n"] * (1 + c["gated"]), c["k"]
        return {"bytes": (m + n) * (k / 2 + _cdiv(k, _GROUP[c["fmt"]])) + 2.0 * m * c["n"] + 4.0 * c["n"] * c["bias"],
                "flops": 2.0 * m * n * k}
    n = c["rows"] * c["n"]
    return {"bytes": n * (4.0 if c["type"] == "f32" else 2.0) + 28.0 * c["rows"], "flops": 4.0 * n}


# ---------------------------------------------------------------- 4-bit floats

def _tiled_at(rows, groups):
    """Places of the scales [rows, groups]: blocks of 128 rows x 4 groups, 512 bytes each, along the groups first."""
    r = torch.arange(rows, device="cuda")[:, None]
    g = torch.arange(groups, device="cuda")[None]
    return (r // 128 * _cdiv(groups, 4) + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4


def _tiled_size(rows, groups):
    return _cdiv(rows, 128) * _cdiv(groups, 4) * 512


def _pitch(cols):
    """Bytes from row to row of the codes of `cols` columns."""
    return _cdiv(_cdiv(cols, 2), 16) * 16


def _quantise(x, fmt, scale):
    """fp32 rows to e2m1 codes (one a byte, rows padded to whole groups) and scale values [rows, groups]."""
    m, n = x.shape
    g = _GROUP[fmt]
    k = _cdiv(n, g)
    full = torch.zeros(m, k * g, device=x.device)
    full[:, :n] = x
    full = full.view(m, k, g)
    t = full.abs().amax(2) / (6.0 * scale)
    if fmt == "nv":
        s = t.clamp(2.0 ** -9, 448.0).to(_F8).float()
    else:
        f, e = torch.frexp(t)
        e = (e - (f == 0.5).to(e.dtype)).clamp(-96, 96)
        s = torch.ldexp(torch.ones_like(t), torch.where(t > 0, e, -96))
    v = full / (s * scale)[..., None]
    a = v.abs()
    code = (a > 0.25).to(torch.uint8)
    for edge, closed in ((0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):   # ties to the even code
        code += (a >= edge) if closed else (a > edge)
    code += torch.signbit(v).to(torch.uint8) * 8
    return code.view(m, k * g), s


def _value4(code):
    lut = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=code.device)
    return lut[code.long()]


def _pack(code, cols):
    """Codes [rows, >= cols], one a byte, as bytes of two [rows, pitch]."""
    m, p = code.shape[0], _pitch(cols)
    full = torch.zeros(m, 2 * p, dtype=torch.uint8, device=code.device)
    full[:, :cols] = code[:, :cols]
    return full[:, 0::2] | (full[:, 1::2] << 4)


def _scale_bytes(s, fmt):
    """Scale values [rows, groups] as bytes in their tiled places, zeros elsewhere."""
    m, k = s.shape
    out = torch.zeros(_tiled_size(m, k), dtype=torch.uint8, device=s.device)
    b = s.to(_F8).view(torch.uint8) if fmt == "nv" else (torch.frexp(s)[1] + 126).to(torch.uint8)
    out[_tiled_at(m, k)] = b
    return out


def _matrix(codes, scales, rows, cols, fmt):
    """fp32 values [rows, cols] of packed codes and tiled scales."""
    g = _GROUP[fmt]
    k = _cdiv(cols, g)
    c = torch.stack([codes & 15, codes >> 4], 2).view(rows, -1)[:, :cols]
    s = scales.view(_F8 if fmt == "nv" else _E8)[_tiled_at(rows, k)].float()
    return _value4(c) * s.repeat_interleave(g, 1)[:, :cols]


# ---------------------------------------------------------------- inputs

def _sections(c):
    """Pairs of each axis: time, row, column."""
    p = c["rot"] // 2
    if c["axes"] == 1:
        return [p, 0, 0, 0]
    s = 3 * p // 8
    return [p - 2 * s, s, s, 0]


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(1000 + seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
    dt = _TYPES[c["type"]]
    s = {"case": c}
    if c["op"] == "rotate":
        n, h, d = c["rows"], c["heads"] + 2 * c["kv_heads"], c["dim"]
        # rows of a fused projection: queries, keys, values; some channels are loud
        s["qkv"] = (randn(n, h, d) * torch.exp(0.5 * randn(h, d))).to(dt)
        if c["norm"]:
            s["q_weight"], s["k_weight"] = (1 + 0.2 * randn(d)).to(dt), (1 + 0.2 * randn(d)).to(dt)
        i = torch.arange(c["rot"] // 2, dtype=torch.float64)
        s["freqs"] = (10000.0 ** (-2 * i / c["rot"])).float().cuda()
        if c["axes"] == 1:
            pos = (rand(1, n) * c["far"]).int()
        else:                                  # frames of 20 x 20 tokens behind a first part of text
            at = torch.arange(n, device="cuda") + random.Random(seed).randrange(400)
            t = at // 400 + c["far"] // 2
            pos = torch.stack([t, t + at % 400 // 20, t + at % 20]).int()
        s["pos"] = pos.contiguous()
    elif c["op"] == "quant":
        s["x"] = (randn(c["rows"], c["cols"]) * torch.exp(0.7 * randn(c["cols"]))).to(dt)
        s["scale"] = 2.0 ** -6 if c["fmt"] == "nv" else 1.0
    elif c["op"] == "gemm":
        m, n, k, f = c["rows"], c["n"], c["k"], c["fmt"]
        s["alpha"] = 1.0
        for name, rows, size in (("x", m, 1.0), ("w", n, k ** -0.5)) + ((("w2", n, k ** -0.5),) if c["gated"] else ()):
            v = randn(rows, k) * size
            if name == "x":
                v *= torch.exp(0.5 * randn(k))
            scale = 1.0 if f == "mx" else 0.02 * size        # of the whole matrix: goes into the product's factor
            code, sc = _quantise(v, f, scale)
            s[name], s[name + "scale"] = _pack(code, k), _scale_bytes(sc, f)
            if name != "w2":
                s["alpha"] *= scale
        if c["bias"]:
            s["bias"] = randn(n)
    else:
        m, n = c["rows"], c["n"]
        x = randn(m, n) * (1.5 + 2 * rand(m, 1))
        s["logits"] = x.to(dt)
        s["u"] = rand(m)
        s["temperature"] = 0.3 + rand(m)
        s["top_k"] = torch.full((m,), c["top_k"], dtype=torch.int32, device="cuda")
        s["top_p"] = torch.full((m,), c["top_p"], device="cuda")
        s["min_p"] = torch.full((m,), c["min_p"], device="cuda")
        if c["mixed"]:
            i = torch.arange(m, device="cuda")
            s["temperature"][i % 5 == 4] = 0.0               # greedy
            s["top_k"][i % 3 == 1] = 0
            s["top_p"][i % 4 == 2] = 1.0
            s["min_p"][i % 2 == 0] = 0.0
    if own:
        _bind(s)
    return s


# ---------------------------------------------------------------- the library's calls

def _bind(s):
    """Output buffers and descriptors over the state's tensors, kept by the program."""
    rt = _runtime()
    lib, c = rt.load(), s["case"]
    code = {"f16": rt.YK_F16, "bf16": rt.YK_BF16, "f32": rt.YK_F32}[c["type"]]
    fmt = {"nv": rt.YK_NVFP4, "mx": rt.YK_MXFP4}.get(c.get("fmt"))
    dt = _TYPES[c["type"]]
    new = lambda *shape, dtype=dt: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "rotate":
        n, h, k, d = c["rows"], c["heads"], c["kv_heads"], c["dim"]
        o = {"q": new(n, h, d), "k": new(n, k, d)}
        row = (h + 2 * k) * d
        a = rt.YkQkRotate(q=p(s["qkv"]), k=s["qkv"].data_ptr() + 2 * h * d, q_out=p(o["q"]), k_out=p(o["k"]),
                          q_weight=p(s.get("q_weight")), k_weight=p(s.get("k_weight")), pos=p(s["pos"]),
                          freqs=p(s["freqs"]), q_row=row, k_row=row, q_out_row=h * d, k_out_row=k * d, pos_axis=n,
                          rows=n, heads=h, kv_heads=k, dim=d, rot=c["rot"], axes=c["axes"],
                          sections=(C.c_int * 4)(*_sections(c)), interleaved=c["inter"], dtype=code, eps=1e-6)
        s["call"] = (lib.yk_qk_rotate, (C.byref(a), stream))
    elif c["op"] == "quant":
        m, n = s["x"].shape
        o = {"values": new(m, n), "scales": new(_tiled_size(m, _cdiv(n, _GROUP[c["fmt"]])), dtype=torch.uint8)}
        s["codes"] = new(m, _pitch(n), dtype=torch.uint8)
        a = rt.YkQuantFp4(x=p(s["x"]), codes=p(s["codes"]), scales=p(o["scales"]), values=p(o["values"]), x_row=n,
                          codes_row=_pitch(n), values_row=n, rows=m, cols=n, format=fmt, dtype=code, scale=s["scale"])
        o["scales"] = o["scales"].view(_F8 if c["fmt"] == "nv" else _E8)
        s["call"] = (lib.yk_quant_fp4, (C.byref(a), stream))
    elif c["op"] == "gemm":
        m, n, k = c["rows"], c["n"], c["k"]
        o = {"y": new(m, n)}
        a = rt.YkGemmFp4(x=p(s["x"]), xscale=p(s["xscale"]), w=p(s["w"]), wscale=p(s["wscale"]), w2=p(s.get("w2")),
                         w2scale=p(s.get("w2scale")), bias=p(s.get("bias")), y=p(o["y"]), x_row=_pitch(k),
                         w_row=_pitch(k), y_row=n, rows=m, n=n, k=k, format=fmt, dtype=code, alpha=s["alpha"],
                         alpha2=s["alpha"])
        s["call"] = (lib.yk_gemm_fp4, (C.byref(a), stream))
    else:
        m, n = s["logits"].shape
        o = {"token": new(m, dtype=torch.int32), "logprob": new(m, dtype=torch.float32)}
        a = rt.YkSample(logits=p(s["logits"]), temperature=p(s["temperature"]), top_k=p(s["top_k"]), top_p=p(s["top_p"]),
                        min_p=p(s["min_p"]), u=p(s["u"]), token=p(o["token"]), logprob=p(o["logprob"]), kept=None,
                        row=n, rows=m, n=n, dtype=code)
        s["call"] = (lib.yk_sample, (C.byref(a), stream))
    s["outputs"] = o


def run(s):
    if own:
        f, args = s["call"]
        if f(*args) != 0:
            raise RuntimeError(_runtime().load().yk_last_cuda_error().decode())
        return s["outputs"]
    return {"rotate": _rotate, "quant": _quant, "gemm": _gemm, "sample": _sample}[s["case"]["op"]](s)


# ---------------------------------------------------------------- plain forms

def _rotate(s):
    c = s["case"]
    h, k, d, p = c["heads"], c["kv_heads"], c["dim"], c["rot"] // 2
    axis = torch.repeat_interleave(torch.arange(4, device="cuda"), torch.tensor(_sections(c), device="cuda"), output_size=p)
    angle = s["pos"].double()[axis].t() * s["freqs"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b = (x[..., 0:2 * p:2], x[..., 1:2 * p:2]) if c["inter"] else (x[..., :p], x[..., p:2 * p])
        u, v = a * cos - b * sin, b * cos + a * sin
        r = torch.stack([u, v], -1).flatten(-2) if c["inter"] else torch.cat([u, v], -1)
        return torch.cat([r, x[..., 2 * p:]], -1).to(s["qkv"].dtype)

    return {"q": turn(s["qkv"][:, :h], s.get("q_weight")), "k": turn(s["qkv"][:, h:h + k], s.get("k_weight"))}


def _quant(s):
    c = s["case"]
    m, n = s["x"].shape
    code, sc = _quantise(s["x"].float(), c["fmt"], s["scale"])
    s["codes"] = _pack(code, n)
    v = _value4(code) * (sc * s["scale"]).repeat_interleave(_GROUP[c["fmt"]], 1)
    return {"values": v[:, :n].to(s["x"].dtype), "scales": _scale_bytes(sc, c["fmt"]).view(_F8 if c["fmt"] == "nv" else _E8)}


def _gemm(s):
    c = s["case"]
    m, n, k, f = c["rows"], c["n"], c["k"], c["fmt"]
    x = _matrix(s["x"], s["xscale"], m, k, f)
    y = (x @ _matrix(s["w"], s["wscale"], n, k, f).t()) * s["alpha"]
    if c["bias"]:
        y = y + s["bias"]
    if c["gated"]:
        y = y / (1 + torch.exp(-y)) * ((x @ _matrix(s["w2"], s["w2scale"], n, k, f).t()) * s["alpha"])
    return {"y": y.to(_TYPES[c["type"]])}


def _sample(s):
    m, n = s["logits"].shape
    x = s["logits"].double()
    top, best = x.max(1, keepdim=True)
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((x - top) / torch.where(greedy, 1.0, t))
    order = torch.argsort(x, dim=1, descending=True, stable=True)       # ties: the lowest index first
    ws = w.gather(1, order)
    k = s["top_k"][:, None]
    rank = torch.arange(n, device=x.device)[None]
    ws = torch.where((rank < k) | (k <= 0), ws, 0.0)
    cum = ws.cumsum(1)
    p = s["top_p"].double()[:, None]
    stay = (ws > 0) & ((cum - ws < p * cum[:, -1:]) | (p >= 1)) & (ws >= s["min_p"].double()[:, None])
    keep = torch.zeros_like(stay).scatter_(1, order, stay)
    w = torch.where(keep, w, 0.0)
    cum = w.cumsum(1)
    total = cum[:, -1:]
    token = (cum <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    last = n - 1 - keep.flip(1).to(torch.uint8).argmax(1, keepdim=True)
    token = torch.where(greedy, best, torch.minimum(token, last))
    logprob = torch.where(greedy, 0.0, torch.log(w.gather(1, token) / total))
    return {"token": token[:, 0].int(), "logprob": logprob[:, 0].float()}


# ---------------------------------------------------------------- definitions in 64 bits

def exact(case, seed):
    return {"rotate": _exact_rotate, "quant": _exact_quant, "gemm": _exact_gemm, "sample": _exact_sample}[
        case["op"]](prepare(case, seed))


def _exact_rotate(s):
    c = s["case"]
    p, out = c["rot"] // 2, {}
    first = 0
    angle = torch.empty(c["rows"], p, dtype=torch.float64, device="cuda")
    for a, count in enumerate(_sections(c)):
        for i in range(first, first + count):
            angle[:, i] = s["pos"][a].double() * s["freqs"][i].double()
        first += count
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    for name, lo, hi in (("q", 0, c["heads"]), ("k", c["heads"], c["heads"] + c["kv_heads"])):
        x = s["qkv"][:, lo:hi].double()
        if c["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + 1e-6).sqrt() * s[name + "_weight"].double()
        at = torch.arange(p, device="cuda")
        a, b = (2 * at, 2 * at + 1) if c["inter"] else (at, at + p)
        z = torch.complex(x[..., a], x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
        out[name] = x
    return out


def _exact_quant(s):
    c, x = s["case"], s["x"].double()
    m, n = x.shape
    g, scale = _GROUP[c["fmt"]], float(torch.tensor(s["scale"], dtype=torch.float32))
    grid = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")
    near = (grid[1:] + grid[:-1]) / 2
    even = torch.arange(7, device="cuda") % 2 == 0             # a tie goes down to an even code
    out, scales = torch.empty_like(x), torch.zeros(_tiled_size(m, _cdiv(n, g)), dtype=torch.float64, device="cuda")
    if c["fmt"] == "mx":
        scales += 2.0 ** -127                                  # code 0
    places = _tiled_at(m, _cdiv(n, g))
    for i in range(_cdiv(n, g)):
        v = x[:, i * g:i * g + g]
        t = v.abs().amax(1) / 6 / scale
        if c["fmt"] == "nv":
            t = t.clamp(2.0 ** -9, 448)
            step = torch.exp2(torch.floor(torch.log2(t)).clamp(min=-6) - 3)
            t = torch.round(t / step) * step
        else:
            t = torch.exp2(torch.ceil(torch.log2(t.clamp(min=2.0 ** -96))))
        scales[places[:, i]] = t
        a = v.abs() / (t * scale)[:, None]
        code = torch.bucketize(a, near)                        # midpoints themselves go down ..
        tie = (a[..., None] == near) & ~even
        code += tie.any(-1).long()                             # .. or up to an even code
        out[:, i * g:i * g + g] = torch.copysign(grid[code], v) * (t * scale)[:, None]
    return {"values": out, "scales": scales}


def _exact_gemm(s):
    c = s["case"]
    m, n, k, g = c["rows"], c["n"], c["k"], _GROUP[c["fmt"]]
    alpha = float(torch.tensor(s["alpha"], dtype=torch.float32))

    def wide(name, r0, r1):
        b = s[name][r0:r1, :_cdiv(k, 2)]
        v = torch.empty(r1 - r0, 2 * b.shape[1], dtype=torch.float64, device="cuda")
        for half, q in enumerate((b % 16, b // 16)):
            e, f = (q % 8 // 2).double(), (q % 2).double()
            mag = torch.where(e == 0, f / 2, torch.exp2(e - 1) * (1 + f / 2))
            v[:, half::2] = torch.where(q >= 8, -mag, mag)
        kind = _F8 if c["fmt"] == "nv" else _E8
        at = _tiled_at(n if name != "x" else m, _cdiv(k, g))[r0:r1]
        return v[:, :k] * s[name + "scale"].view(kind)[at].double().repeat_interleave(g, 1)[:, :k]

    x, y = wide("x", 0, m), torch.empty(m, n, dtype=torch.float64, device="cuda")
    for a in range(0, n, 4096):
        b = min(n, a + 4096)
        v = x @ wide("w", a, b).t() * alpha
        if c["bias"]:
            v += s["bias"][a:b].double()
        if c["gated"]:
            v = v * torch.sigmoid(v) * (x @ wide("w2", a, b).t() * alpha)
        y[:, a:b] = v
    return {"y": y}


def _exact_sample(s):
    """Tokens are whole numbers and have no such value; the probability is that of the token that the definition takes."""
    out = []
    for r in range(s["case"]["rows"]):
        x = s["logits"][r].double()
        t, k = float(s["temperature"][r]), int(s["top_k"][r])
        if t <= 0:
            out.append(0.0)
            continue
        v, index = torch.sort(x, descending=True, stable=True)
        w = torch.exp((v - v[0]) / t)
        if k > 0:
            w = w[:k]
        if float(s["top_p"][r]) < 1:
            w = w[:1 + int((w.cumsum(0)[:-1] < float(s["top_p"][r]) * w.sum()).sum())]
        w = w[w >= float(s["min_p"][r])]
        w = w[w > 0]
        by_index = torch.argsort(index[:w.numel()])
        cum = w[by_index].cumsum(0)
        i = min(int((cum <= float(s["u"][r]) * cum[-1]).sum()), w.numel() - 1)
        out.append(math.log(float(w[by_index][i] / cum[-1])))
    return {"token": None, "logprob": torch.tensor(out, dtype=torch.float64, device="cuda")}
