"""Measured cases of the text-decoder operators: their inputs, plain forms and 64-bit definitions.

Five operators of one decode step: the block plan of a paged cache (``yk_kv_plan``), the write
of new keys and values into the 8-bit cache (``yk_kv_append``), attention over it
(``yk_attn_kv8``), the residual addition with RMS norm and 8-bit output (``yk_rmsnorm8``) and
the product with a 4-bit weight matrix (``yk_gemv4``).  ``run`` computes a case in elementary
torch operations, or, with ``own`` set, through the library's C ABI as a C or Python caller
does: descriptors filled once over buffers that the program keeps, one call a pass.

Lengths of a ragged batch follow from the case alone; the seed orders them and draws the values.
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
_FMAX = 448.0          # largest e4m3 value
_TINY = 2.0 ** -126    # smallest scale
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


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
        # a decode step of a full batch: one new token a request, latency counts
        {"name": "plan decode 64", "op": "plan", "requests": 64, "past_min": 1, "past_max": 4096,
         "fresh_min": 1, "fresh_max": 1, "block": 32, "short": 0, "mix": 1},
        # admission of a large ragged batch of prompts, with too few free blocks for the last ones
        {"name": "plan prompts 2048", "op": "plan", "requests": 2048, "past_min": 0,
         "past_max": 8192, "fresh_min": 0, "fresh_max": 700, "block": 16, "short": 5, "mix": 2},
        # one new token a request goes into partly filled blocks
        {"name": "append decode 64", "op": "append", "requests": 64, "past_min": 1,
         "past_max": 2048, "fresh_min": 1, "fresh_max": 1, "block": 32, "kv_heads": 8, "dim": 128,
         "type": "f16", "mix": 3},
        # ragged prompts (400 image tokens and longer) go into the cache
        {"name": "append prompts", "op": "append", "requests": 24, "past_min": 0, "past_max": 100,
         "fresh_min": 400, "fresh_max": 2100, "block": 64, "kv_heads": 8, "dim": 128,
         "type": "bf16", "mix": 4},
        # one request just after its prompt of 400 image tokens: the smallest call
        {"name": "attn one request", "op": "attn", "requests": 1, "kv_min": 431, "kv_max": 431,
         "q_min": 1, "q_max": 1, "heads": 16, "kv_heads": 4, "dim": 64, "block": 16, "window": 0,
         "type": "f16", "mix": 5},
        # a full ragged decode batch with shared key heads, an idle slot and an empty row
        {"name": "attn decode 64", "op": "attn", "requests": 64, "kv_min": 64, "kv_max": 8192,
         "q_min": 1, "q_max": 1, "heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "window": 0,
         "type": "bf16", "mix": 6},
        # two requests over a long cache: work is split along the keys
        {"name": "attn long cache", "op": "attn", "requests": 2, "kv_min": 131075,
         "kv_max": 262147, "q_min": 1, "q_max": 1, "heads": 16, "kv_heads": 2, "dim": 128,
         "block": 64, "window": 0, "type": "f16", "mix": 7},
        # ragged prompts attend to themselves and to what the cache held before
        {"name": "attn prompts", "op": "attn", "requests": 8, "kv_min": 700, "kv_max": 4096,
         "q_min": 400, "q_max": 2048, "heads": 16, "kv_heads": 4, "dim": 128, "block": 64,
         "window": 0, "type": "bf16", "mix": 8},
        # norm of a small decode batch, 8-bit rows with one scale
        {"name": "norm 8 x 2048", "op": "norm", "rows": 8, "cols": 2048, "group": 0, "add": 1,
         "out16": 0, "type": "f16"},
        # norm of a prompt batch, 8-bit rows with a scale for each 128 channels
        {"name": "norm 12000 x 5120", "op": "norm", "rows": 12000, "cols": 5120, "group": 128,
         "add": 1, "out16": 0, "type": "bf16"},
        # one token through a square projection
        {"name": "gemv 1 x 4096 x 4096", "op": "gemv", "rows": 1, "n": 4096, "k": 4096,
         "group": 128, "zero": 0, "bias": 1, "x8": 0, "xgroup": 0, "type": "f16"},
        # a batch of 8-bit rows (from the norm) through a wide projection with zero points
        {"name": "gemv 16 x 28672 x 8192", "op": "gemv", "rows": 16, "n": 28672, "k": 8192,
         "group": 64, "zero": 1, "bias": 0, "x8": 1, "xgroup": 128, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["plan", "append", "attn", "attn", "attn", "norm", "gemv", "gemv"])
        c = {"op": op}
        if op != "plan":
            c["type"] = rng.choice(["f16", "bf16"])
        if op == "plan":
            c |= {"requests": _log(rng, 1, 2048), "past_min": 0, "past_max": _log(rng, 16, 8192),
                  "fresh_min": rng.choice([0, 1]), "fresh_max": _log(rng, 1, 700),
                  "block": rng.choice([16, 32, 64, 128]), "short": rng.choice([0, 0, 5, 50]),
                  "mix": rng.randrange(1 << 20)}
        elif op == "append":
            lo = _log(rng, 1, 500)
            c |= {"requests": _log(rng, 1, 128), "past_min": 0, "past_max": _log(rng, 1, 2048),
                  "fresh_min": lo, "fresh_max": lo * rng.choice([1, 2, 4]),
                  "block": rng.choice([16, 32, 64, 128]), "kv_heads": rng.choice([1, 2, 4, 8]),
                  "dim": rng.choice([64, 128, 256]), "mix": rng.randrange(1 << 20)}
        elif op == "attn":
            kvh = rng.choice([1, 2, 4, 8])
            q = rng.choice([1, 1, 1, 4, _log(rng, 16, 1500)])
            kv = _log(rng, max(q, 8), 200000 if q == 1 else 8192)
            c |= {"requests": _log(rng, 1, 128 if q <= 4 else 8), "kv_min": max(q, kv // 8),
                  "kv_max": kv, "q_min": q if q <= 4 else max(1, q // 4), "q_max": q,
                  "heads": kvh * rng.choice([1, 2, 4, 5, 7, 8]), "kv_heads": kvh,
                  "dim": rng.choice([64, 128, 128, 256]), "block": rng.choice([16, 32, 64, 128]),
                  "window": rng.choice([0, 0, 0, 1000]), "mix": rng.randrange(1 << 20)}
        elif op == "norm":
            c |= {"rows": _log(rng, 1, 12000), "cols": _log(rng, 64, 16384),
                  "group": rng.choice([0, 32, 128]), "add": rng.choice([0, 1, 1]),
                  "out16": rng.choice([0, 1])}
            c["cols"] += rng.choice([0, 0, 0, -1]) - c["cols"] % 8 + 8
        else:
            g = rng.choice([32, 64, 128])
            c |= {"rows": _log(rng, 1, 64), "n": _log(rng, 64, 28672),
                  "k": 128 * _log(rng, 2, 64), "group": g, "zero": rng.choice([0, 1]),
                  "bias": rng.choice([0, 1]), "x8": rng.choice([0, 0, 1]), "xgroup": 0}
            if c["x8"]:
                c["xgroup"] = rng.choice([0, 128])
        if _affordable(c):
            return c


def _affordable(c):
    """Whether a drawn case stays within the largest listed ones, the plain form's padding
    included."""
    w = work(c)
    if c["op"] == "plan":
        return sum(f for _, f in _lens(c)) >= 1
    if c["op"] == "append":
        return w["bytes"] < 1.2e8
    if c["op"] == "attn":
        r, kv, q = c["requests"], c["kv_max"], c["q_max"]
        return (w["bytes"] < 2.2e8 and w["flops"] < 1.0e11 and r * kv * c["kv_heads"] * c["dim"] < 6e8
                and r * q * kv * c["heads"] < 1.1e9)
    if c["op"] == "norm":
        return w["bytes"] < 4.3e8
    return w["bytes"] < 1.3e8


def _lens(c):
    """(past, fresh) of every request, from the case alone."""
    r, n = random.Random(c["mix"]), c["requests"]
    between = lambda lo, hi: _log(r, lo + 1, hi + 1) - 1  # noqa: E731
    if c["op"] == "attn":
        out = []
        for _ in range(n):
            q = between(c["q_min"], c["q_max"])
            out.append((max(between(c["kv_min"], c["kv_max"]) - q, 0), q))
        if n >= 8:
            out[1] = (0, 0)       # an idle slot
            out[2] = (-1, 1)      # a row whose cache is empty
        return out
    return [(between(c["past_min"], c["past_max"]), r.randint(c["fresh_min"], c["fresh_max"]))
            for _ in range(n)]


def _cdiv(a, b):
    return -(-a // b)


def work(c):
    if c["op"] == "plan":
        t, lens = c["block"], _lens(c)
        rows = sum(f for _, f in lens)
        blocks = sum(_cdiv(p + f, t) - _cdiv(p, t) for p, f in lens)
        return {"bytes": 4.0 * (4 * len(lens) + 1 + 2 * rows + 2 * blocks), "flops": 0.0}
    if c["op"] == "append":
        t, lens = c["block"], _lens(c)
        rows = sum(f for _, f in lens)
        units = sum(_cdiv(p + f, t) - p // t for p, f in lens if f)
        return {"bytes": 6.0 * rows * c["kv_heads"] * c["dim"] + 4.0 * rows
                + 16.0 * units * c["kv_heads"], "flops": 6.0 * rows * c["kv_heads"] * c["dim"]}
    if c["op"] == "attn":
        tokens = pairs = rows = 0
        for p, q in _lens(c):
            kv = p + q
            rows += q
            if q and kv:
                w = c["window"] or kv
                tokens += min(kv, w + q - 1)
                full = max(0, min(q, w - p - 1))   # queries that still see all keys before them
                pairs += full * p + full * (full + 1) // 2 + (q - full) * min(w, kv)
        d = c["dim"]
        return {"bytes": 2.0 * tokens * c["kv_heads"] * d + rows * c["heads"] * (4.0 * d + 4),
                "flops": 4.0 * pairs * c["heads"] * d}
    if c["op"] == "norm":
        n, g = c["rows"] * c["cols"], c["group"] or c["cols"]
        return {"bytes": n * (2.0 + 4 * c["add"] + 1 + 2 * c["out16"]) + 2.0 * c["cols"]
                + 4.0 * c["rows"] * _cdiv(c["cols"], g), "flops": 6.0 * n}
    m, n, k, g = c["rows"], c["n"], c["k"], c["group"]
    x = m * k * (1 if c["x8"] else 2) + (4.0 * m * (_cdiv(k, c["xgroup"]) if c["xgroup"] else 1)
                                         if c["x8"] else 0)
    return {"bytes": n * k / 2 + n * (k // g) * (2.0 + c["zero"]) + 4.0 * n * c["bias"] + x
            + 2.0 * m * n, "flops": 2.0 * m * n * k}


# ---------------------------------------------------------------- inputs

def _pow2_scale(amax):
    """The smallest power of two s >= 2^-126 with 448 s >= amax."""
    f, e = torch.frexp(amax)
    k = (e - 9 + (f > 0.875).to(e.dtype)).clamp(min=-126)
    k = torch.where(amax > 0, k, torch.full_like(k, -126))
    return torch.ldexp(torch.ones_like(amax), k)


def _cache(blocks, heads, t, d, gen):
    """An 8-bit pool [blocks, heads, t, d] of normal values with a few loud channels."""
    gain = torch.exp(0.5 * torch.randn(heads, 1, d, generator=gen, device="cuda"))
    x = torch.empty(blocks, heads, t, d, dtype=torch.float16, device="cuda").normal_(generator=gen)
    x *= gain.half()
    s = _pow2_scale(x.abs().amax((2, 3)).float())
    x *= (1 / s)[..., None, None]
    return x.clamp_(-_FMAX, _FMAX).to(_F8).view(torch.uint8), s


def _ragged(c, seed):
    """Lengths in the seed's order, and a table whose blocks lie anywhere in the pool."""
    lens = _lens(c)
    r = random.Random(seed)
    r.shuffle(lens)
    t = c["block"]
    kv = [max(p + f, 0) for p, f in lens]
    fresh = [f for _, f in lens]
    need = [_cdiv(k, t) for k in kv]
    pool = sum(need) + 3
    ids = list(range(pool))
    r.shuffle(ids)
    cols = max(need + [1])
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (cols - n))
        at += n
    cu = [0]
    for f in fresh:
        cu.append(cu[-1] + f)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    slots = [table[i][p // t] * t + p % t for i, f in enumerate(fresh)
             for p in range(kv[i] - f, kv[i]) if p >= 0]
    return {"kv": i32(kv), "cu": i32(cu), "table": i32(table), "slots": slots, "pool": pool,
            "rows": cu[-1], "cols": cols, "q_max": max(fresh)}


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(1000 + seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    dt = _TYPES.get(c.get("type"))
    s = {"case": c}
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["op"] == "plan":
        lens, r, t = _lens(c), random.Random(seed), c["block"]
        r.shuffle(lens)
        held = [_cdiv(p, t) for p, _ in lens]
        want = sum(_cdiv(p + f, t) for p, f in lens) - sum(held)
        s["cols"] = _cdiv(c["past_max"] + c["fresh_max"], t)
        s["rows"], s["blocks"] = sum(f for _, f in lens), sum(held) + want + 1
        ids = list(range(s["blocks"]))
        r.shuffle(ids)
        table, at = [], 0
        for h in held:
            table.append(ids[at:at + h] + [-1] * (s["cols"] - h))
            at += h
        s["free"] = i32(ids[at:at + max(1, want - want * c["short"] // 100)])
        s["past"], s["fresh"] = i32([p for p, _ in lens]), i32([f for _, f in lens])
        s["table"] = i32(table)
    elif c["op"] == "append":
        g = _ragged(c, seed)
        n, h, d = g["rows"], c["kv_heads"], c["dim"]
        s["slots"] = i32(g["slots"])
        # fused projection rows: keys and values are slices of one buffer
        kv = randn(n, 2, h, d)
        kv *= torch.exp(0.5 * randn(n, 1, h, 1))
        s["kv"] = kv.to(dt)
        s["k"], s["kscale"] = _cache(g["pool"], h, c["block"], d, gen)
        s["v"], s["vscale"] = _cache(g["pool"], h, c["block"], d, gen)
        t = c["block"]
        s["units"] = sum(1 for i, x in enumerate(g["slots"])
                         if i == 0 or x % t == 0 or x != g["slots"][i - 1] + 1)
    elif c["op"] == "attn":
        g = _ragged(c, seed)
        s |= {k: g[k] for k in ("cu", "table", "rows", "q_max")}
        s["kv_lens"] = g["kv"]
        s["q"] = (randn(g["rows"], c["heads"], c["dim"]) * 0.7).to(dt)
        s["k"], s["kscale"] = _cache(g["pool"], c["kv_heads"], c["block"], c["dim"], gen)
        s["v"], s["vscale"] = _cache(g["pool"], c["kv_heads"], c["block"], c["dim"], gen)
    elif c["op"] == "norm":
        m, n = c["rows"], c["cols"]
        s["x"] = (randn(m, n) * torch.exp(randn(n) * 0.5)).to(dt)
        if c["add"]:
            s["add"] = randn(m, n).to(dt)
        s["weight"] = (1 + 0.2 * randn(n)).to(dt)
    else:
        m, n, k, g = c["rows"], c["n"], c["k"], c["group"]
        s["w"] = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["wscale"] = (0.01 * torch.exp(0.3 * randn(n, k // g))).to(dt)
        if c["zero"]:
            s["wzero"] = torch.randint(4, 12, (n, k // g), generator=gen, device="cuda",
                                       dtype=torch.uint8)
        if c["bias"]:
            s["bias"] = randn(n)
        x = randn(m, k) * torch.exp(randn(k) * 0.5)
        if c["x8"]:
            xg = c["xgroup"] or k
            a = x.view(m, k // xg, xg)
            s["xscale"] = (a.abs().amax(2) / _FMAX).contiguous()
            s["x"] = (a / s["xscale"][..., None]).clamp(-_FMAX, _FMAX).to(_F8).view(m, k).view(torch.uint8)
        else:
            s["x"] = x.to(dt)
    if own:
        _bind(s)
    return s


# ---------------------------------------------------------------- the library's calls

def _bind(s):
    """Output buffers, workspace and descriptors over the state's tensors, kept by the program."""
    rt = _runtime()
    lib, c = rt.load(), s["case"]
    code = {"f16": rt.YK_F16, "bf16": rt.YK_BF16}.get(c.get("type"))
    dt = _TYPES.get(c.get("type"))
    new = lambda *shape, dtype=torch.int32: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] in ("append", "attn"):
        pool, h, t, d = s["k"].shape
        cache = rt.YkKvCache(k=p(s["k"]), v=p(s["v"]), kscale=p(s["kscale"]), vscale=p(s["vscale"]),
                             block_stride=h * t * d, scale_stride=h, blocks=pool, heads=h, tokens=t,
                             dim=d)
    if c["op"] == "plan":
        n = c["requests"]
        o = {"table": s["table"], "kv_lens": new(n), "cu": new(n + 1), "slots": new(s["rows"]),
             "pos": new(s["rows"]), "counts": new(4)}
        a = rt.YkKvPlan(past=p(s["past"]), fresh=p(s["fresh"]), free_blocks=p(s["free"]),
                        free_head=None, table=p(o["table"]), kv_lens=p(o["kv_lens"]), cu=p(o["cu"]),
                        slots=p(o["slots"]), pos=p(o["pos"]), counts=p(o["counts"]),
                        table_stride=s["cols"], requests=n, rows=s["rows"],
                        free_count=s["free"].numel(), blocks=s["blocks"], max_blocks=s["cols"],
                        tokens=c["block"])
        s["call"] = (lib.yk_kv_plan, (C.byref(a), stream))
    elif c["op"] == "append":
        o = {"k": s["k"].view(_F8), "v": s["v"].view(_F8), "kscale": s["kscale"],
             "vscale": s["vscale"]}
        n, _, h, d = s["kv"].shape
        a = rt.YkKvRows(k=p(s["kv"]), v=s["kv"].data_ptr() + 2 * h * d, slots=p(s["slots"]),
                        k_row=2 * h * d, v_row=2 * h * d, k_head=d, v_head=d, rows=n, dtype=code)
        s["call"] = (lib.yk_kv_append, (C.byref(cache), C.byref(a), stream))
    elif c["op"] == "attn":
        o = {"out": torch.zeros_like(s["q"]), "lse": new(s["rows"], c["heads"], dtype=torch.float32)}
        n, h, d = s["q"].shape
        size = lib.yk_attn_kv8_workspace_bytes(c["requests"], n, h, c["kv_heads"], d)
        s["ws"] = new(size, dtype=torch.uint8)
        a = rt.YkAttnKv8(q=p(s["q"]), out=p(o["out"]), lse=p(o["lse"]), q_row=h * d, out_row=h * d,
                         cu=p(s["cu"]), kv_lens=p(s["kv_lens"]), table=p(s["table"]),
                         table_stride=s["table"].shape[1], max_blocks=s["table"].shape[1],
                         requests=c["requests"], rows=n, heads=h, dtype=code, causal=1,
                         window=c["window"], scale=0.0, ws=p(s["ws"]), ws_bytes=size)
        s["call"] = (lib.yk_attn_kv8, (C.byref(cache), C.byref(a), stream))
    elif c["op"] == "norm":
        m, n = s["x"].shape
        g = _cdiv(n, c["group"] or n)
        o = {"codes": new(m, n, dtype=torch.uint8), "scales": new(m, g, dtype=torch.float32)}
        if c["add"]:
            o["sum"] = new(m, n, dtype=dt)
        if c["out16"]:
            o["out"] = new(m, n, dtype=dt)
        a = rt.YkRmsNorm8(x=p(s["x"]), add=p(s.get("add")), sum=p(o.get("sum")),
                          weight=p(s["weight"]), out=p(o.get("out")), codes=p(o["codes"]),
                          scales=p(o["scales"]), x_row=n, add_row=n, sum_row=n, out_row=n,
                          codes_row=n, scales_row=g, rows=m, cols=n, group=c["group"], dtype=code,
                          eps=1e-6)
        o["codes"] = o["codes"].view(_F8)
        s["call"] = (lib.yk_rmsnorm8, (C.byref(a), stream))
    else:
        m, k, n = c["rows"], c["k"], c["n"]
        o = {"y": new(m, n, dtype=dt)}
        a = rt.YkGemv4(x=p(s["x"]), xscale=p(s.get("xscale")), w=p(s["w"]), wscale=p(s["wscale"]),
                       wzero=p(s.get("wzero")), bias=p(s.get("bias")), y=p(o["y"]), x_row=k,
                       xscale_row=_cdiv(k, c["xgroup"] or k), w_row=k // 2, group_row=k // c["group"],
                       y_row=n, rows=m, n=n, k=k, group=c["group"], xgroup=c["xgroup"],
                       xtype=rt.YK_E4M3 if c["x8"] else code, dtype=code)
        s["call"] = (lib.yk_gemv4, (C.byref(a), stream))
    s["outputs"] = o


def run(s):
    if own:
        f, args = s["call"]
        if f(*args) != 0:
            raise RuntimeError(_runtime().load().yk_last_cuda_error().decode())
        return s["outputs"]
    return {"plan": _plan, "append": _append, "attn": _attn, "norm": _norm, "gemv": _gemv}[
        s["case"]["op"]](s)


# ---------------------------------------------------------------- plain forms

def _finite_amax(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dims)


def _plan(s):
    t, rows, cols = s["case"]["block"], s["rows"], s["cols"]
    past, fresh = s["past"].long(), s["fresh"].long()
    n, dev = past.numel(), past.device
    held, want = (past + t - 1) // t, (past + fresh + t - 1) // t
    need = torch.where(past + fresh <= cols * t, want - held, 0)
    off = need.cumsum(0) - need
    ok = (past + fresh <= cols * t) & ((need == 0) | (off + need <= s["free"].numel()))
    j = torch.arange(cols, device=dev)[None] - held[:, None]
    taken = ok[:, None] & (j >= 0) & (j < need[:, None])
    ids = s["free"][(off[:, None] + j).clamp(0, s["free"].numel() - 1)]
    table = torch.where(taken, ids, s["table"])
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), fresh.cumsum(0)])
    req = torch.repeat_interleave(torch.arange(n, device=dev), fresh, output_size=rows)
    pos = past[req] + torch.arange(rows, device=dev) - cu[req]
    slots = table[req, (pos // t).clamp(max=cols - 1)].long() * t + pos % t
    slots = torch.where(ok[req], slots, -1)
    counts = torch.stack([torch.where(ok, need, 0).sum(), torch.where(ok, fresh, 0).sum(),
                          (~ok).sum(), cu[-1]])
    return {"table": table, "kv_lens": (past + torch.where(ok, fresh, 0)).int(), "cu": cu.int(),
            "slots": slots.int(), "pos": pos.int(), "counts": counts.int()}


def _append(s):
    t, units = s["case"]["block"], s["units"]
    slots = s["slots"].long()
    block, off = slots // t, slots % t
    prev = torch.cat([slots[:1] - 2, slots[:-1]])
    lead = (off == 0) | (slots != prev + 1)
    unit = lead.long().cumsum(0) - 1
    first = torch.argsort(~lead, stable=True)[:units]
    ub, uo = block[first], off[first]
    new = torch.zeros(units, t, dtype=torch.bool, device=slots.device)
    new[unit, off] = True
    old = torch.arange(t, device=slots.device)[None] < uo[:, None]
    return _append_one(s["kv"][:, 0], s["k"], s["kscale"], ub, uo, unit, off, new, old, "k") | \
        _append_one(s["kv"][:, 1], s["v"], s["vscale"], ub, uo, unit, off, new, old, "v")


def _append_one(x, codes, scales, ub, uo, unit, off, new, old, name):
    units, (_, h, t, d) = ub.numel(), codes.shape
    put = torch.zeros(units, t, h, d, device=x.device)
    put[unit, off] = x.float()
    put = put.transpose(1, 2)
    need = _pow2_scale(_finite_amax(put, (2, 3)))
    before = scales[ub]
    scale = torch.where(uo[:, None] > 0, torch.maximum(before, need), need)
    fresh = (put * (1 / scale)[..., None, None]).clamp(-_FMAX, _FMAX).to(_F8).view(torch.uint8)
    tile = codes[ub]
    again = (tile.view(_F8).float() * (before / scale)[..., None, None]).clamp(-_FMAX, _FMAX)
    tile = torch.where(old[:, None, :, None], again.to(_F8).view(torch.uint8), tile)
    codes[ub] = torch.where(new[:, None, :, None], fresh, tile)
    scales[ub] = scale
    return {name: codes.view(_F8), name + "scale": scales}


def _attn(s):
    c = s["case"]
    n, hq, d = s["q"].shape
    r, hk, t = c["requests"], c["kv_heads"], c["block"]
    g, qm, dev = hq // hk, s["q_max"], s["q"].device
    cu, kv = s["cu"].long(), s["kv_lens"].long()
    qlen = cu[1:] - cu[:-1]
    table = s["table"].long().clamp(min=0)
    m = table.shape[1] * t
    j = torch.arange(m, device=dev)
    there = (j[None] < kv[:, None])[:, None, :, None]

    def rows(codes, scales):
        x = codes[table].view(_F8).float() * scales[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(r, hk, m, d).masked_fill(~there, 0.0)

    i = torch.arange(qm, device=dev)
    at = (cu[:-1, None] + i[None]).clamp(max=n - 1)
    q = s["q"][at].float().view(r, qm, hk, g, d).permute(0, 2, 3, 1, 4).reshape(r, hk, g * qm, d)
    w = (q @ rows(s["k"], s["kscale"]).transpose(2, 3)).view(r, hk, g, qm, m) * (d ** -0.5)
    pos = (kv - qlen)[:, None] + i[None]
    see = (j <= pos[..., None]) & (j < kv[:, None, None])
    if c["window"]:
        see &= j > pos[..., None] - c["window"]
    w = w.masked_fill(~see[:, None, None], float("-inf"))
    top = w.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    w = (w - top).exp_()
    total = w.sum(-1)
    o = (w.view(r, hk, g * qm, m) @ rows(s["v"], s["vscale"])).view(r, hk, g, qm, d)
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    lse = top[..., 0] + total.log()
    req = torch.repeat_interleave(torch.arange(r, device=dev), qlen, output_size=n)
    mine = torch.arange(n, device=dev) - cu[req]
    return {"out": o[req, :, :, mine].reshape(n, hq, d).to(s["q"].dtype),
            "lse": lse[req, :, :, mine].reshape(n, hq)}


def _norm(s):
    c = s["case"]
    x, dt = s["x"].float(), s["x"].dtype
    m, n = x.shape
    o = {}
    if c["add"]:
        x = x + s["add"].float()
        o["sum"] = x.to(dt)
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6) * s["weight"].float()
    g = c["group"] or n
    k = _cdiv(n, g)
    full = torch.zeros(m, k * g, device=x.device)
    full[:, :n] = y
    full = full.view(m, k, g)
    o["scales"] = (_finite_amax(full, 2) / _FMAX).clamp(min=_TINY)
    q = (full * (1 / o["scales"])[..., None]).clamp(-_FMAX, _FMAX).to(_F8).view(torch.uint8)
    o["codes"] = q.view(m, k * g)[:, :n].contiguous().view(_F8)
    if c["out16"]:
        o["out"] = y.to(dt)
    return o


def _gemv(s):
    c = s["case"]
    m, n, k, g = c["rows"], c["n"], c["k"], c["group"]
    w = torch.stack([s["w"] & 15, s["w"] >> 4], 2).view(n, k // g, g).float()
    w = (w - (s["wzero"].float()[..., None] if c["zero"] else 8.0)) * s["wscale"].float()[..., None]
    if c["x8"]:
        x = s["x"].view(_F8).float().view(m, -1, c["xgroup"] or k) * s["xscale"][..., None]
    else:
        x = s["x"].float()
    y = x.view(m, k) @ w.view(n, k).t()
    if c["bias"]:
        y = y + s["bias"]
    return {"y": y.to(s["wscale"].dtype)}


# ---------------------------------------------------------------- definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": lambda s: None, "append": _exact_append, "attn": _exact_attn,
            "norm": _exact_norm, "gemv": _exact_gemv}[case["op"]](s)


def _value(codes):
    return codes.view(_F8).to(torch.float32).double()


def _exact_append(s):
    """Codes before their rounding; scales as they are."""
    t, slots, out = s["case"]["block"], s["slots"].tolist(), {}
    runs = []
    for i, x in enumerate(slots):
        if i and x % t and x == slots[i - 1] + 1:
            runs[-1][2] += 1
        else:
            runs.append([i, x, 1])
    for part, name in enumerate(("k", "v")):
        codes, scales = _value(s[name]), s[name + "scale"].double()
        for row, slot, count in runs:
            b, o = divmod(slot, t)
            x = s["kv"][row:row + count, part].double().transpose(0, 1)   # [heads, count, dim]
            a = x.abs().amax((1, 2))
            f, e = torch.frexp(a / 448)                                   # 2^(e-1) <= a / 448 < 2^e
            e = torch.where(f == 0.5, e - 1, e).clamp(min=-126)
            new = torch.ldexp(torch.ones_like(a), torch.where(a > 0, e, torch.full_like(e, -126)))
            if o:
                new = torch.maximum(new, scales[b])
                codes[b, :, :o] *= (scales[b] / new)[:, None, None]
            codes[b, :, o:o + count] = x / new[:, None, None]
            scales[b] = new
        out[name], out[name + "scale"] = codes, scales
    return out


def _exact_attn(s):
    c, t = s["case"], s["case"]["block"]
    n, hq, d = s["q"].shape
    g = hq // c["kv_heads"]
    out = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq), float("-inf"), dtype=torch.float64, device="cuda")
    cu, lens = s["cu"].tolist(), s["kv_lens"].tolist()
    for r in range(c["requests"]):
        q0, q1, kv = cu[r], cu[r + 1], lens[r]
        if q1 == q0 or kv == 0:
            continue
        ids = s["table"][r, :_cdiv(kv, t)].long()
        first = kv - (q1 - q0)
        at = torch.arange(kv, device="cuda")[None]
        pos = torch.arange(first, kv, device="cuda")[:, None]
        hide = at > pos
        if c["window"]:
            hide |= at <= pos - c["window"]
        for h in range(c["kv_heads"]):
            key = (_value(s["k"][ids, h]) * s["kscale"][ids, h].double()[:, None, None]).view(-1, d)[:kv]
            val = (_value(s["v"][ids, h]) * s["vscale"][ids, h].double()[:, None, None]).view(-1, d)[:kv]
            for a in range(h * g, h * g + g):
                w = (s["q"][q0:q1, a].double() @ key.t() / math.sqrt(d)).masked_fill(hide, float("-inf"))
                lse[q0:q1, a] = torch.logsumexp(w, 1)
                out[q0:q1, a] = torch.softmax(w, 1) @ val
    return {"out": out, "lse": lse}


def _exact_norm(s):
    """Codes before their rounding."""
    c, x = s["case"], s["x"].double()
    m, n = x.shape
    o = {}
    if c["add"]:
        x = x + s["add"].double()
        o["sum"] = x
    y = x / (x.pow(2).sum(1, keepdim=True) / n + 1e-6).sqrt() * s["weight"].double()
    g = c["group"] or n
    o["codes"] = torch.empty_like(y)
    o["scales"] = torch.empty(m, _cdiv(n, g), dtype=torch.float64, device="cuda")
    for i, a in enumerate(range(0, n, g)):
        o["scales"][:, i] = y[:, a:a + g].abs().amax(1) / 448
        o["codes"][:, a:a + g] = y[:, a:a + g] / o["scales"][:, i:i + 1]
    if c["out16"]:
        o["out"] = y
    return o


def _exact_gemv(s):
    c = s["case"]
    m, n, k, g = c["rows"], c["n"], c["k"], c["group"]
    x = _value(s["x"]) if c["x8"] else s["x"].double()
    if c["x8"]:
        x = x * s["xscale"].double().repeat_interleave(c["xgroup"] or k, 1)
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for a in range(0, n, 4096):
        w = torch.empty(min(4096, n - a), k, dtype=torch.float64, device="cuda")
        w[:, 0::2] = (s["w"][a:a + 4096] % 16).double()
        w[:, 1::2] = (s["w"][a:a + 4096] // 16).double()
        z = s["wzero"][a:a + 4096].double() if c["zero"] else torch.full_like(s["wscale"][a:a + 4096], 8).double()
        w -= z.repeat_interleave(g, 1)
        w *= s["wscale"][a:a + 4096].double().repeat_interleave(g, 1)
        y[:, a:a + 4096] = x @ w.t()
    return {"y": y + (s["bias"].double() if c["bias"] else 0.0)}
