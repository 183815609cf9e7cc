"""A small text decoder over the library's text operators, answering about frames: image tokens
from a detector's deepest feature map and a prompt fill a paged 8-bit key/value cache, then every
request gets one token a step.

    python yolo11.cu_b200/textdec.py [--frames 4] [--steps 16] [--model yolo11n] [--weights nvfp4] [--rotary]
                                     [--temperature 0.8 --top-k 40 --top-p 0.95]

``TextDecoder`` owns seeded random-init 4-bit weights, a pool of cache blocks and the buffers of a
step; ``prompt`` runs ragged rows, ``decode`` one row a request as one captured CUDA graph.  A layer
is: yk_rmsnorm8 (adds the last block's output to the residual, 8-bit rows) -> yk_gemv4 (queries,
keys, values) -> yk_kv_append -> yk_attn_kv8 -> yk_gemv4 -> yk_rmsnorm8 -> yk_gemv4 (gate, up) ->
SiLU product -> yk_gemv4.  yk_kv_plan places the step's rows once, before the layers.  Nothing is read
back between kernels: lengths, tables and the free list stay on the device.

With weights="nvfp4" or "mxfp4" the products are of 4-bit floats on both sides: the norm's rows go through
yk_quant_fp4 into yk_gemm_fp4, and the gated half of the feed-forward block is one product.  With rotary=True
yk_qk_rotate norms and turns queries and keys by their place (time, row, column: an image token has its
row and column, text follows behind) in place of a learned position table.  set_sampling() draws tokens
(yk_sample) instead of taking the best.
"""
from __future__ import annotations

import argparse
import ctypes as C
import importlib.util
import os
import sys

PKG = os.path.dirname(os.path.abspath(__file__))


def _pkg():
    if "yolo11_cu_b200" not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            "yolo11_cu_b200", os.path.join(PKG, "__init__.py"), submodule_search_locations=[PKG])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["yolo11_cu_b200"] = mod
        spec.loader.exec_module(mod)


_pkg()
import torch  # noqa: E402
from yolo11_cu_b200 import runtime as rt  # noqa: E402


def quantize_w4(w, group: int = 128):
    """fp32 [n, k] -> (codes [n, k / 2] uint8, scales [n, k / group] fp16): symmetric, zero point 8,
    scale = the group's largest |w| / 7."""
    n, k = w.shape
    g = w.view(n, k // group, group)
    s = (g.abs().amax(2) / 7).clamp(min=1e-7).half()
    q = (torch.round(g / s.float()[..., None]) + 8).clamp(0, 15).to(torch.uint8).view(n, k)
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), s


class Fp4:
    """A matrix of 4-bit floats: codes, scales in their blocks, the scale of all (yk_quant_fp4's layout)."""

    def __init__(self, lib, rows, cols, fmt, device, scale=1.0):
        self.rows, self.cols, self.fmt, self.scale = rows, cols, fmt, scale
        self.codes = torch.zeros(rows, -(-cols // 256) * 128, dtype=torch.uint8, device=device)   # (rows on L2 lines)
        self.scales = torch.zeros(lib.yk_fp4_scale_bytes(rows, cols, fmt), dtype=torch.uint8, device=device)

    def fill(self, lib, x, n, cols=None):
        """The first n rows of x (fp16), whose rows may be shorter than the matrix's."""
        a = rt.YkQuantFp4(x=x.data_ptr(), codes=self.codes.data_ptr(), scales=self.scales.data_ptr(), x_row=x.stride(0),
                          codes_row=self.codes.stride(0), rows=n, cols=cols or self.cols, format=self.fmt, dtype=rt.YK_F16,
                          scale=self.scale)
        return lib.yk_quant_fp4(C.byref(a), torch.cuda.current_stream().cuda_stream)


class TextDecoder:
    def __init__(self, requests: int, *, layers=2, width=512, heads=8, kv_heads=2, dim=64, hidden=1024,
                 vocab=1000, group=128, block=32, pool=256, max_tokens=2048, rows=1024, seed=0, eps=1e-6,
                 device="cuda", weights="int4", rotary=False):
        self.lib = rt.load()
        if weights not in ("int4", "nvfp4", "mxfp4"):
            raise ValueError(f"weights must be int4, nvfp4 or mxfp4, not {weights!r}")
        self.fp4 = {"int4": None, "nvfp4": rt.YK_NVFP4, "mxfp4": rt.YK_MXFP4}[weights]
        self.rotary = rotary
        self.requests, self.layers, self.width, self.heads, self.kv_heads = requests, layers, width, heads, kv_heads
        self.dim, self.hidden, self.vocab, self.group, self.block = dim, hidden, vocab, group, block
        self.pool, self.rows, self.eps, self.device = pool, max(rows, requests), eps, device
        self.max_blocks = -(-max_tokens // block)
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
        qkv = (heads + 2 * kv_heads) * dim
        sizes = {"qkv": (qkv, width), "out": (width, heads * dim), "up": (2 * hidden, width), "down": (width, hidden)}
        if self.fp4 is not None:
            sizes["up"], sizes["gate"] = (hidden, width), (hidden, width)
        self.w = [{k: self._weight(rand(n, m) * m ** -0.5) for k, (n, m) in sizes.items()} for _ in range(layers)]
        self.norms = [(1 + 0.1 * rand(2 * layers + 1, width)).half()[i] for i in range(2 * layers + 1)]
        self.head = self._weight(rand(vocab, width) * width ** -0.5)
        self.embed = rand(vocab, width).half()
        self.place = (0.3 * rand(self.max_blocks * block, width)).half()
        new = lambda *s, dtype=torch.half: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
        i32 = torch.int32
        n = self.rows
        self.cache, self.codes = [], []
        for _ in range(layers):
            kv = new(pool, 2, kv_heads, block, dim, dtype=torch.uint8)
            sc = torch.ones(2, pool, kv_heads, device=device)
            self.codes.append((kv, sc))
            self.cache.append(rt.YkKvCache(
                k=kv[:, 0].data_ptr(), v=kv[:, 1].data_ptr(), kscale=sc[0].data_ptr(), vscale=sc[1].data_ptr(),
                block_stride=kv.stride(0), scale_stride=kv_heads, blocks=pool, heads=kv_heads, tokens=block, dim=dim))
        # the plan's arrays; lens is past and kv_lens in one
        self.lens, self.fresh, self.cu = new(requests, dtype=i32), new(requests, dtype=i32), new(requests + 1, dtype=i32)
        self.table = torch.full((requests, self.max_blocks), -1, dtype=i32, device=device)
        self.free, self.taken = torch.arange(pool, dtype=i32, device=device), new(1, dtype=i32)
        self.slots, self.pos, self.counts = new(n, dtype=i32), new(n, dtype=i32), new(4, dtype=i32)
        # a step's buffers
        self.res, self.delta = new(n, width), new(n, width)
        self.x8, self.xs = new(n, width, dtype=torch.uint8), new(n, 1, dtype=torch.float32)
        self.qkv, self.att = new(n, qkv), new(n, heads * dim)
        self.up, self.act = new(n, 2 * hidden), new(n, hidden)
        self.last8, self.lasts = new(requests, width, dtype=torch.uint8), new(requests, 1, dtype=torch.float32)
        self.logits = new(requests, vocab)
        # next: the token that goes in with the next step; given: the one that went in with the last (-1: refused)
        self.next, self.given = new(requests, dtype=torch.long), new(requests, dtype=torch.long)
        self.held, self.placed = new(requests, dtype=i32), new(requests, dtype=torch.bool)
        size = self.lib.yk_attn_kv8_workspace_bytes(requests, n, heads, kv_heads, dim)
        self.ws = new(size, dtype=torch.uint8)
        if self.fp4 is not None:
            self.x16, self.last16 = new(n, width), new(requests, width)
            # e4m3 scales keep their three bits from 2^-6 to 448, so that groups of rows do whose largest value lies between 6 / 64
            # and 2688 of the whole matrix's scale: 0.003 to 84 with 2^-5 (rows of deviation 1/64: a value
            # is off by up to 0.17 of its group's largest one; 0.33 with 1).  A norm's rows are about one (at most the square root of
            # their width), an average over a long cache is small.  Powers of two have the whole range.
            scale = 2.0 ** -5 if self.fp4 == rt.YK_NVFP4 else 1.0
            self.x4 = {c: Fp4(self.lib, n, c, self.fp4, device, scale) for c in {width, heads * dim, hidden}}
        if rotary:
            self.head_norms = [(1 + 0.1 * rand(2, dim)).half() for _ in range(layers)]       # of queries, of keys
            pairs = torch.arange(dim // 2, dtype=torch.float64)
            self.freqs = (10000.0 ** (-2 * pairs / dim)).float().to(device)
            self.sections = (dim // 2 - 2 * (3 * dim // 16), 3 * dim // 16, 3 * dim // 16, 0)  # time, row, column
            # places of a step's rows, and by how much a request's lie from its tokens' numbers
            self.at, self.shift = torch.full((3, n), -1, dtype=i32, device=device), new(requests, dtype=i32)
        # sampling: None (the best token), or the requests' settings; `u` is drawn before each step
        self.sampling, self.gen = None, None
        self.unscored = new(requests, dtype=torch.bool)       # requests that had no score to draw from in the last step
        self.u, self.picked, self.logprob = new(requests, dtype=torch.float32), new(requests, dtype=i32), new(requests, dtype=torch.float32)
        self.graphs = {}

    @property
    def graph(self):
        """The captured step of the present way to choose tokens, if there is one."""
        return self.graphs.get(self.sampling is not None)

    @graph.setter
    def graph(self, captured):
        """None lets go of what was captured, in every way to choose tokens: the next step is captured anew."""
        if captured is None:
            self.graphs.clear()
        else:
            self.graphs[self.sampling is not None] = captured

    def _weight(self, w):
        """A weight matrix in the decoder's format."""
        if self.fp4 is None:
            return quantize_w4(w, self.group)
        m = Fp4(self.lib, *w.shape, self.fp4, w.device, scale=2.0 ** -8)
        self._ok(m.fill(self.lib, w.half().contiguous(), m.rows))
        return m

    # ---- one call of each operator over the decoder's buffers ----
    def _ok(self, code):
        if code != 0:
            raise RuntimeError(f"text operator refused ({code}): {self.lib.yk_last_cuda_error().decode()}")

    @property
    def _stream(self):
        return torch.cuda.current_stream().cuda_stream

    def _plan(self, n):
        a = rt.YkKvPlan(past=self.lens.data_ptr(), fresh=self.fresh.data_ptr(), free_blocks=self.free.data_ptr(),
                        free_head=self.taken.data_ptr(), table=self.table.data_ptr(), kv_lens=self.lens.data_ptr(),
                        cu=self.cu.data_ptr(), slots=self.slots.data_ptr(), pos=self.pos.data_ptr(),
                        counts=self.counts.data_ptr(), table_stride=self.max_blocks, requests=self.requests,
                        rows=n, free_count=self.pool, blocks=self.pool, max_blocks=self.max_blocks,
                        tokens=self.block)
        self._ok(self.lib.yk_kv_plan(C.byref(a), self._stream))

    def _norm(self, x, add, weight, n):
        a = rt.YkRmsNorm8(x=x.data_ptr(), add=add.data_ptr(), sum=self.res.data_ptr(), weight=weight.data_ptr(),
                          codes=self.x8.data_ptr(), scales=self.xs.data_ptr(), x_row=self.width, add_row=self.width,
                          sum_row=self.width, codes_row=self.width, scales_row=1, rows=n, cols=self.width,
                          group=0, dtype=rt.YK_F16, eps=self.eps)
        if self.fp4 is not None:
            a.codes, a.scales, a.out, a.out_row = None, None, self.x16.data_ptr(), self.width
        self._ok(self.lib.yk_rmsnorm8(C.byref(a), self._stream))

    def _linear4(self, x, w, y, n, gate=None):
        """y = x w^T of 4-bit floats (with gate: silu(x gate^T) * (x w^T)); x fp16, to 4 bits first."""
        x4 = self.x4[w.cols]
        self._ok(x4.fill(self.lib, x, n))
        g = gate or w
        a = rt.YkGemmFp4(x=x4.codes.data_ptr(), xscale=x4.scales.data_ptr(), w=g.codes.data_ptr(), wscale=g.scales.data_ptr(),
                         w2=w.codes.data_ptr() if gate else None, w2scale=w.scales.data_ptr() if gate else None, y=y.data_ptr(),
                         x_row=x4.codes.stride(0), w_row=w.codes.stride(0), y_row=y.stride(0), rows=n, n=w.rows, k=w.cols,
                         format=self.fp4, dtype=rt.YK_F16, alpha=x4.scale * g.scale, alpha2=x4.scale * w.scale)
        self._ok(self.lib.yk_gemm_fp4(C.byref(a), self._stream))

    def _rotate(self, layer, n):
        """Queries and keys of the step's rows: norm of each head, then the turn by the row's place."""
        h, k, d, row = self.heads, self.kv_heads, self.dim, self.qkv.stride(0)
        q, kk, norms = self.qkv.data_ptr(), self.qkv.data_ptr() + 2 * h * d, self.head_norms[layer]
        a = rt.YkQkRotate(q=q, k=kk, q_out=q, k_out=kk, q_weight=norms[0].data_ptr(), k_weight=norms[1].data_ptr(),
                          pos=self.at.data_ptr(), freqs=self.freqs.data_ptr(), q_row=row, k_row=row, q_out_row=row, k_out_row=row,
                          pos_axis=self.at.stride(0), rows=n, heads=h, kv_heads=k, dim=d, rot=d, axes=3,
                          sections=(C.c_int * 4)(*self.sections), dtype=rt.YK_F16, eps=self.eps)
        self._ok(self.lib.yk_qk_rotate(C.byref(a), self._stream))

    def _sample(self):
        s = self.sampling
        a = rt.YkSample(logits=self.logits.data_ptr(), temperature=s["temperature"].data_ptr(), top_k=s["top_k"].data_ptr(),
                        top_p=s["top_p"].data_ptr(), min_p=s["min_p"].data_ptr(), u=self.u.data_ptr(), token=self.picked.data_ptr(),
                        logprob=self.logprob.data_ptr(), row=self.vocab, rows=self.requests, n=self.vocab, dtype=rt.YK_F16)
        self._ok(self.lib.yk_sample(C.byref(a), self._stream))
        # a row without any weight (all NaN or -infinity) gives -1, which is no row of the embedding: the token stays
        none = self.picked < 0
        torch.logical_and(none, self.placed, out=self.unscored)
        return torch.where(none, self.next, self.picked)

    def _matmul(self, x, w, y, n, scales=None):
        """y = x w^T; 64 rows a call.  scales: x is e4m3 codes."""
        q, s = w
        for m in range(0, n, 64):
            a = rt.YkGemv4(x=x[m:].data_ptr(), xscale=scales[m:].data_ptr() if scales is not None else None,
                           w=q.data_ptr(), wscale=s.data_ptr(), y=y[m:].data_ptr(), x_row=x.stride(0),
                           xscale_row=1, w_row=q.stride(0), group_row=s.stride(0), y_row=y.stride(0),
                           rows=min(64, n - m), n=q.shape[0], k=2 * q.shape[1], group=self.group,
                           xtype=rt.YK_F16 if scales is None else rt.YK_E4M3, dtype=rt.YK_F16)
            self._ok(self.lib.yk_gemv4(C.byref(a), self._stream))

    def _attend(self, layer, n):
        h, k, d, row = self.heads, self.kv_heads, self.dim, self.qkv.stride(0)
        c = self.cache[layer]
        a = rt.YkKvRows(k=self.qkv.data_ptr() + 2 * h * d, v=self.qkv.data_ptr() + 2 * (h + k) * d,
                        slots=self.slots.data_ptr(), k_row=row, v_row=row, k_head=d, v_head=d, rows=n,
                        dtype=rt.YK_F16)
        self._ok(self.lib.yk_kv_append(C.byref(c), C.byref(a), self._stream))
        b = rt.YkAttnKv8(q=self.qkv.data_ptr(), out=self.att.data_ptr(), q_row=row, out_row=h * d,
                         cu=self.cu.data_ptr(), kv_lens=self.lens.data_ptr(), table=self.table.data_ptr(),
                         table_stride=self.max_blocks, max_blocks=self.max_blocks, requests=self.requests,
                         rows=n, heads=h, dtype=rt.YK_F16, causal=1, ws=self.ws.data_ptr(),
                         ws_bytes=self.ws.numel())
        self._ok(self.lib.yk_attn_kv8(C.byref(c), C.byref(b), self._stream))

    def _places(self, n):
        """The position rows of a step.  The plan writes the positions of refused rows too (past the last
        block) and -1 for rows of no request; both take the nearest row, which nothing reads."""
        return self.place[self.pos[:n].long().clamp(0, self.place.shape[0] - 1)]

    def _turns(self, n, owner, places=None):
        """The places of a step's rows for the rotation: as given, else the token's number and its request's shift
        on every axis; -1 for rows of no request."""
        at = self.pos[:n] + self.shift[owner]
        self.at[:, :n] = torch.where(self.pos[:n] < 0, -1, at if places is None else torch.where(places[0] < 0, at, places))

    def _layers(self, n, owner=None, places=None):
        """The residual rows self.res[:n] through every layer, then the scores of each request's last row and
        the next token.  A request whose rows the plan refused, or that has none in the step, keeps the token
        that it has (its row of `logits` is then none of its own); `placed` says which have theirs in the cache."""
        self.held.copy_(self.lens)
        self._plan(n)
        torch.gt(self.lens, self.held, out=self.placed)
        if self.rotary:
            self._turns(n, owner, places)
        else:
            self.res[:n] += self._places(n)
        self.delta[:n].zero_()
        for i, w in enumerate(self.w):
            self._norm(self.delta, self.res, self.norms[2 * i], n)
            if self.fp4 is None:
                self._matmul(self.x8, w["qkv"], self.qkv, n, self.xs)
            else:
                self._linear4(self.x16, w["qkv"], self.qkv, n)
            if self.rotary:
                self._rotate(i, n)
            self._attend(i, n)
            if self.fp4 is None:
                self._matmul(self.att, w["out"], self.delta, n)
            else:
                self._linear4(self.att, w["out"], self.delta, n)
            self._norm(self.delta, self.res, self.norms[2 * i + 1], n)
            if self.fp4 is None:
                self._matmul(self.x8, w["up"], self.up, n, self.xs)
                torch.mul(torch.nn.functional.silu(self.up[:n, :self.hidden]), self.up[:n, self.hidden:], out=self.act[:n])
                self._matmul(self.act, w["down"], self.delta, n)
            else:
                self._linear4(self.x16, w["up"], self.act, n, gate=w["gate"])
                self._linear4(self.act, w["down"], self.delta, n)
        self._norm(self.delta, self.res, self.norms[-1], n)
        last = (self.cu[1:].long() - 1).clamp(min=0)
        if self.fp4 is None:
            self.last8.copy_(self.x8[last])
            self.lasts.copy_(self.xs[last])
            self._matmul(self.last8, self.head, self.logits, self.requests, self.lasts)
        else:
            self.last16.copy_(self.x16[last])
            self._linear4(self.last16, self.head, self.logits, self.requests)
        best = self.logits.argmax(1) if self.sampling is None else self._sample()
        self.next.copy_(torch.where(self.placed, best, self.next))

    def _draw(self):
        """The step's random numbers (outside the captured step, which reads them)."""
        if self.sampling is not None:
            self.u.uniform_(generator=self.gen)

    # ---- what a caller uses ----
    def set_sampling(self, temperature=None, top_k=0, top_p=1.0, min_p=0.0, seed=0):
        """How the next tokens are chosen from now on: drawn with these settings (each one for all requests, or one a
        request; a temperature of 0 takes the best), or without a temperature the best token, as at the start.  New
        settings are written where a captured step reads them."""
        if temperature is None:
            self.sampling = None
            self.unscored.zero_()
            return
        want = dict(temperature=(temperature, torch.float32), top_k=(top_k, torch.int32), top_p=(top_p, torch.float32),
                    min_p=(min_p, torch.float32))
        for k, (v, t) in want.items():
            v = torch.as_tensor(v, dtype=t)
            if v.dim() and v.shape != (self.requests,):
                raise ValueError(f"{k}: one value, or one for each of {self.requests} requests")
            want[k] = v.expand(self.requests)
        if not hasattr(self, "_settings"):
            self._settings = {k: torch.zeros(self.requests, dtype=v.dtype, device=self.device) for k, v in want.items()}
            self.gen = torch.Generator(device=self.device)
        for k, v in want.items():
            self._settings[k].copy_(v)
        self.sampling = self._settings
        self.gen.manual_seed(seed)

    def prompt(self, rows, lens, places=None):
        """rows [sum(lens), width]: each request's new rows one after another (embeddings of prompt
        tokens, image tokens); lens[r] may be 0.  Fills the cache and picks the next token of each request
        whose rows went in (`placed`); the others, without rows or refused, keep theirs.
        places [3][sum(lens)] (rotary): time, row and column of each row, which lies there whatever came before it, or -1 for
        rows of text.  Text behind such rows, and every later token, goes on from one place behind the largest place given
        in this call before it; without any it goes on as before.  So an image given places below those that its request has
        had takes the text behind it back there, too: the next token of request r lies at lens[r] + shift[r]."""
        n = sum(lens)
        if n > self.rows or n != rows.shape[0] or len(lens) != self.requests:
            raise ValueError(f"{n} rows in {len(lens)} requests, {rows.shape[0]} given: at most {self.rows} "
                             f"rows in {self.requests} requests")
        owner = None
        if places is not None:
            if not self.rotary:
                raise ValueError("places are for a decoder with rotary=True")
            if tuple(places.shape) != (3, n):
                raise ValueError(f"places are [3][{n}], not {tuple(places.shape)}")
            places = places.to(self.device, torch.int32)
        if self.rotary:
            counts = torch.tensor(lens, device=self.device)
            owner = torch.repeat_interleave(torch.arange(self.requests, device=self.device), counts, output_size=n)
        if places is not None:
            places = self._behind(places, owner, counts, n)
        self.fresh.copy_(torch.tensor(lens, dtype=torch.int32))
        self.res[:n].copy_(rows)
        self._draw()
        shift = self.shift.clone() if self.rotary else None
        if places is not None:
            self.shift.copy_(self._shift)
        self._layers(n, owner, places)
        if places is not None:                       # a refused request's places did not happen
            self.shift.copy_(torch.where(self.placed, self.shift, shift))
        return self.next

    def _behind(self, places, owner, counts, n):
        """places with rows of text (-1) put behind the largest place given before them in their request's rows here (text rows
        themselves do not count), or by their request's shift; the requests' shifts after it go to self._shift."""
        start = self.lens.long()[owner] + torch.arange(n, device=self.device) - (counts.cumsum(0) - counts)[owner]   # token numbers
        text = places[0] < 0
        # a row of text lies at its token's number + shift; the shift is that of the image rows before it: one behind their
        # largest place, less the number of the token that follows the last of them
        big = torch.where(text, torch.full_like(places[0], -1), places.amax(0)).long()
        key = owner * (1 << 32)
        run = (key + big + 1).cummax(0).values - key                                 # 1 + largest place so far in the request (0: none)
        seen = (key + torch.where(text, 0, start + 1)).cummax(0).values - key        # 1 + number of the last image token so far
        shift = torch.where(run > 0, run - seen, self.shift.long()[owner])
        out = torch.where(text, (start + shift).int(), places)
        after = self.shift.clone()
        has = counts > 0
        ends = (counts.cumsum(0) - 1).clamp(min=0)
        if n:
            after = torch.where(has, shift[ends].int(), after)
        self._shift = after
        return out

    def _step(self):
        self.given.copy_(self.next)
        self.res[:self.requests].copy_(self.embed[self.next])
        self._layers(self.requests, torch.arange(self.requests, device=self.device) if self.rotary else None)
        self.given.masked_fill_(~self.placed, -1)

    def decode(self, steps: int, graph: bool = True):
        """`steps` tokens for every request, the best ones or as set_sampling says; [steps, requests].  Where the plan
        refuses a request a step (no free block, or its table is full) it gives -1, and its token waits for the next step.
        A request whose scores leave nothing to draw (all NaN or -infinity) keeps its token, which goes in again, and is true in
        `unscored` until a step draws one for it.
        The first call (of each way to choose tokens), and the first after `graph` was set to None, captures the step."""
        out = torch.empty(steps, self.requests, dtype=torch.long, device=self.device)
        self.fresh.fill_(1)
        for i in range(steps):
            self._draw()
            if not graph:
                self._step()
            elif self.graph is None:
                # a step before the capture (libraries and allocations settle), which counts
                self._step()
                torch.cuda.synchronize()
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured):
                    self._step()
                self.graphs[self.sampling is not None] = captured
            else:
                self.graph.replay()
            out[i] = self.given
        return out


def image_tokens(model: str, frames: int, S: int = 640):
    """The deepest feature map of `frames` synthetic frames as fp16 rows [frames, positions, channels]."""
    from yolo11_cu_b200 import export, frames as fr
    d = export.ensure_model_dir(model, os.path.join(os.path.dirname(PKG), "models"), S)
    eng = rt.Engine(d, frames)
    for i in range(frames):
        eng.preprocess_host(fr.synthetic_bgr(720, 1280, seed=i), i)
    eng.run(frames)
    eng._check()
    best, t = None, 0
    while True:
        try:
            _, h, w, _, _, ch = eng.tensor_view(t)
        except IndexError:
            break
        if h == S // 32 and w == S // 32 and (best is None or ch >= best[1]):
            best = (t, ch)
        t += 1
    x = torch.from_numpy(eng.read(best[0], frames)).cuda()
    eng.close()
    return x.reshape(frames, -1, best[1])


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--frames", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--model", default="yolo11n")
    ap.add_argument("--weights", default="int4", choices=["int4", "nvfp4", "mxfp4"])
    ap.add_argument("--rotary", action="store_true")
    ap.add_argument("--temperature", type=float)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    a = ap.parse_args(argv)
    x = image_tokens(a.model, a.frames)
    n = x.shape[1]
    dec = TextDecoder(a.frames, rows=a.frames * (n + 8), weights=a.weights, rotary=a.rotary)
    dec.set_sampling(a.temperature, a.top_k, a.top_p, a.min_p)
    proj = torch.randn(x.shape[2], dec.width, generator=torch.Generator().manual_seed(1)).cuda().half()
    img = torch.nn.functional.layer_norm(x.float(), x.shape[-1:]).half() @ proj * x.shape[2] ** -0.5
    words = torch.arange(8, device="cuda")                       # the same short prompt for every frame
    rows = torch.cat([torch.cat([img[i], dec.embed[words]]) for i in range(a.frames)])
    places = None
    if a.rotary:
        side = int(n ** 0.5)
        t = torch.arange(n)
        one = torch.cat([torch.stack([0 * t, t // side, t % side]), torch.full((3, 8), -1)], 1)
        places = one.repeat(1, a.frames)
    dec.prompt(rows, [n + 8] * a.frames, places)
    ids = dec.decode(a.steps)
    torch.cuda.synchronize()
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    dec.decode(a.steps)
    t1.record()
    torch.cuda.synchronize()
    for i in range(a.frames):
        print(f"frame {i}: {n} image tokens ->", ids[:, i].tolist())
    print(f"{t0.elapsed_time(t1) / a.steps * 1e3:.1f} us a step of {a.frames} requests, "
          f"{int(dec.counts[2])} refused, {int(dec.taken)} of {dec.pool} blocks in use")


if __name__ == "__main__":
    main()
