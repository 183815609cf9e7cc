"""A small text decoder over the library's text operators, answering about frames: image tokens
from a detector's deepest feature map and a prompt fill a paged 8-bit key/value cache, then every
request gets one token a step.

    python yolo11.cu_b200/textdec.py [--frames 4] [--steps 16] [--model yolo11n]

``TextDecoder`` owns seeded random-init 4-bit weights, a pool of cache blocks and the buffers of a
step; ``prompt`` runs ragged rows, ``decode`` one row a request as one captured CUDA graph.  A layer
is: yk_rmsnorm8 (adds the last block's output to the residual, 8-bit rows) -> yk_gemv4 (queries,
keys, values) -> yk_kv_append -> yk_attn_kv8 -> yk_gemv4 -> yk_rmsnorm8 -> yk_gemv4 (gate, up) ->
SiLU product -> yk_gemv4.  yk_kv_plan places the step's rows once, before the layers.  Nothing is read
back between kernels: lengths, tables and the free list stay on the device.
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


class TextDecoder:
    def __init__(self, requests: int, *, layers=2, width=512, heads=8, kv_heads=2, dim=64, hidden=1024,
                 vocab=1000, group=128, block=32, pool=256, max_tokens=2048, rows=1024, seed=0, eps=1e-6,
                 device="cuda"):
        self.lib = rt.load()
        self.requests, self.layers, self.width, self.heads, self.kv_heads = requests, layers, width, heads, kv_heads
        self.dim, self.hidden, self.vocab, self.group, self.block = dim, hidden, vocab, group, block
        self.pool, self.rows, self.eps, self.device = pool, max(rows, requests), eps, device
        self.max_blocks = -(-max_tokens // block)
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
        qkv = (heads + 2 * kv_heads) * dim
        sizes = {"qkv": (qkv, width), "out": (width, heads * dim), "up": (2 * hidden, width), "down": (width, hidden)}
        self.w = [{k: quantize_w4(rand(n, m) * m ** -0.5, group) for k, (n, m) in sizes.items()}
                  for _ in range(layers)]
        self.norms = [(1 + 0.1 * rand(2 * layers + 1, width)).half()[i] for i in range(2 * layers + 1)]
        self.head = quantize_w4(rand(vocab, width) * width ** -0.5, group)
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
        self.graph = None

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
        self._ok(self.lib.yk_rmsnorm8(C.byref(a), self._stream))

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

    def _layers(self, n):
        """The residual rows self.res[:n] through every layer, then the scores of each request's last row and
        the next token.  A request whose rows the plan refused, or that has none in the step, keeps the token
        that it has (its row of `logits` is then none of its own); `placed` says which have theirs in the cache."""
        self.held.copy_(self.lens)
        self._plan(n)
        torch.gt(self.lens, self.held, out=self.placed)
        self.res[:n] += self._places(n)
        self.delta[:n].zero_()
        for i, w in enumerate(self.w):
            self._norm(self.delta, self.res, self.norms[2 * i], n)
            self._matmul(self.x8, w["qkv"], self.qkv, n, self.xs)
            self._attend(i, n)
            self._matmul(self.att, w["out"], self.delta, n)
            self._norm(self.delta, self.res, self.norms[2 * i + 1], n)
            self._matmul(self.x8, w["up"], self.up, n, self.xs)
            torch.mul(torch.nn.functional.silu(self.up[:n, :self.hidden]), self.up[:n, self.hidden:], out=self.act[:n])
            self._matmul(self.act, w["down"], self.delta, n)
        self._norm(self.delta, self.res, self.norms[-1], n)
        last = (self.cu[1:].long() - 1).clamp(min=0)
        self.last8.copy_(self.x8[last])
        self.lasts.copy_(self.xs[last])
        self._matmul(self.last8, self.head, self.logits, self.requests, self.lasts)
        self.next.copy_(torch.where(self.placed, self.logits.argmax(1), self.next))

    # ---- what a caller uses ----
    def prompt(self, rows, lens):
        """rows [sum(lens), width]: each request's new rows one after another (embeddings of prompt
        tokens, image tokens); lens[r] may be 0.  Fills the cache and picks the next token of each request
        whose rows went in (`placed`); the others, without rows or refused, keep theirs."""
        n = sum(lens)
        if n > self.rows or n != rows.shape[0] or len(lens) != self.requests:
            raise ValueError(f"{n} rows in {len(lens)} requests, {rows.shape[0]} given: at most {self.rows} "
                             f"rows in {self.requests} requests")
        self.fresh.copy_(torch.tensor(lens, dtype=torch.int32))
        self.res[:n].copy_(rows)
        self._layers(n)
        return self.next

    def _step(self):
        self.given.copy_(self.next)
        self.res[:self.requests].copy_(self.embed[self.next])
        self._layers(self.requests)
        self.given.masked_fill_(~self.placed, -1)

    def decode(self, steps: int, graph: bool = True):
        """`steps` tokens for every request, greedily; [steps, requests].  Where the plan refuses a request
        a step (no free block, or its table is full) it gives -1, and its token waits for the next step.
        The first call captures the step."""
        out = torch.empty(steps, self.requests, dtype=torch.long, device=self.device)
        self.fresh.fill_(1)
        for i in range(steps):
            if not graph:
                self._step()
            elif self.graph is None:
                # a step before the capture (libraries and allocations settle), which counts
                self._step()
                torch.cuda.synchronize()
                self.graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(self.graph):
                    self._step()
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
    a = ap.parse_args(argv)
    x = image_tokens(a.model, a.frames)
    n = x.shape[1]
    dec = TextDecoder(a.frames, rows=a.frames * (n + 8))
    proj = torch.randn(x.shape[2], dec.width, generator=torch.Generator().manual_seed(1)).cuda().half()
    img = torch.nn.functional.layer_norm(x.float(), x.shape[-1:]).half() @ proj * x.shape[2] ** -0.5
    words = torch.arange(8, device="cuda")                       # the same short prompt for every frame
    rows = torch.cat([torch.cat([img[i], dec.embed[words]]) for i in range(a.frames)])
    dec.prompt(rows, [n + 8] * a.frames)
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
