"""A model's attention layer over a paged cache, from the library's calls (attentionForward, src/model.zig:918-979, for
a batch of requests instead of one):

    quantized_matmul_group   q (with its gate beside each head), k and v from one x
    rope_cache               head norms, rotary positions, k and v into their pages
    paged_attention          every request's new tokens over its pages, times the gate's sigmoid
    quantized_matmul         the output projection

With cache="e4m3" the pages hold 8 bits a value and the two calls between are `rope_cache_fp8` and `paged_attention_fp8`;
`cache_read_fp8` gives rows of them back.

A step's tables come from `block_tables`, once for all layers of a model.  `python attention_layer.py` prefills
requests of different lengths and decodes a few tokens of each, the decode step as a captured graph: lengths and page
ids live on the GPU and nothing is planned on the host, so every replay follows them.  `python attention_layer.py e4m3`
does the same over a cache held in 8 bits.
"""
from __future__ import annotations

import math
import sys

import torch

import qmm as Q


class Pages:
    """The requests' lengths, pages and a step's tables, all on the GPU; shared by the layers of a model."""

    def __init__(self, requests: int, pages: int, block: int, width: int):
        def ints(*shape):
            return torch.zeros(shape, dtype=torch.int32, device="cuda")

        self.block = block
        self.table, self.head, self.lens = ints(requests, width), ints(1), ints(requests)
        self.free = torch.randperm(pages).to(torch.int32).cuda()
        self.new, self.starts = ints(requests), ints(requests + 1)

    def step(self, tokens: int, stream):
        """Tables of a step of `tokens` tokens, self.new[r] of them request r's; the lengths move on."""
        self.positions = torch.empty(tokens, dtype=torch.int32, device="cuda")
        self.slots = torch.empty_like(self.positions)
        a = {n: Q.Array.from_torch(getattr(self, n), Q.INT32)
             for n in ("table", "head", "lens", "free", "new", "starts", "positions", "slots")}
        Q.block_tables(a["table"], a["head"], a["lens"], a["new"], a["free"], self.block, tokens, table_out=a["table"],
                       head_out=a["head"], q_starts=a["starts"], kv_lens=a["lens"], positions=a["positions"],
                       slots=a["slots"], stream=stream)
        return a


class AttentionLayer:
    """Hq query heads (each with a gate) over Hkv key heads of D values; `rot` of them turn with the position."""

    def __init__(self, K: int, Hq: int, Hkv: int, D: int, rot: int, pages: int, block: int, *, mode: str = "nvfp4",
                 base: float = 1e7, seed: int = 0, cache: str = "bfloat16"):
        if cache not in ("bfloat16", "e4m3"):
            raise ValueError(f"cache must be 'bfloat16' or 'e4m3', not {cache!r}")
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape):
            return torch.randn(shape, generator=g, device="cuda")

        self.Hq, self.Hkv, self.D, self.mode = Hq, Hkv, D, mode
        rows = [2 * Hq * D, Hkv * D, Hkv * D]
        # q, k and v back to back: their three products are one launch
        w = (normal(sum(rows), K) / math.sqrt(K)).to(torch.bfloat16)
        self.w, self.s = self._quantize(w)
        self.ws = [Q.Array.from_torch(x, Q.UINT32) for x in self.w.split(rows)]
        self.ss = [Q.Array.from_torch(x, Q.UINT8) for x in self.s.split(rows)]
        w = (normal(K, Hq * D) / math.sqrt(Hq * D)).to(torch.bfloat16)
        self.wo, self.so = self._quantize(w)
        self.o_proj = Q.Array.from_torch(self.wo, Q.UINT32), Q.Array.from_torch(self.so, Q.UINT8)
        self.q_norm, self.k_norm = ((1 + 0.1 * normal(D)).to(torch.bfloat16) for _ in range(2))
        self.norms = Q.Array.from_torch(self.q_norm), Q.Array.from_torch(self.k_norm)
        freqs, self.amplitude = Q.rope_frequencies(rot, base)
        self.freqs = torch.from_numpy(freqs).cuda()
        self.eight = cache == "e4m3"
        dtype = torch.uint8 if self.eight else torch.bfloat16
        self.k_cache, self.v_cache = (torch.zeros(pages, Hkv, block, D, dtype=dtype, device="cuda") for _ in range(2))
        self.caches = Q.Array.from_torch(self.k_cache), Q.Array.from_torch(self.v_cache)
        if self.eight:  # a scale for each page and head
            self.k_scales, self.v_scales = (torch.zeros(pages, Hkv, dtype=torch.uint8, device="cuda") for _ in range(2))
            self.caches += Q.Array.from_torch(self.k_scales), Q.Array.from_torch(self.v_scales)

    def _quantize(self, w):
        wq, s = Q.quantize(Q.Array.from_torch(w), self.mode, stream=Q.Stream.torch_current())
        return tuple(torch.from_numpy(a.numpy(Q.Stream.torch_current()).view("int32" if a is wq else "uint8")).cuda()
                     for a in (wq, s))

    def __call__(self, x: torch.Tensor, step: dict, stream) -> torch.Tensor:
        """x [T, K] bfloat16 -> [T, K]; `step`: the arrays of Pages.step."""
        T, D = x.shape[0], self.D

        def empty(*shape):
            return torch.empty(shape, dtype=torch.bfloat16, device="cuda")

        q, k, v = empty(T, self.Hq, 2 * D), empty(T, self.Hkv, D), empty(T, self.Hkv, D)
        turned, o, y = empty(T, self.Hq, D), empty(T, self.Hq, D), empty(T, x.shape[1])
        A = Q.Array.from_torch
        Q.quantized_matmul_group(A(x), self.ws, self.ss, self.mode, outs=[A(t.view(T, -1)) for t in (q, k, v)], stream=stream)
        write, attend = (Q.rope_cache_fp8, Q.paged_attention_fp8) if self.eight else (Q.rope_cache, Q.paged_attention)
        write(A(q), A(k), A(v), *self.caches, step["positions"], step["slots"], A(self.freqs),
              amplitude=self.amplitude, q_norm=self.norms[0], k_norm=self.norms[1], q_out=A(turned), stream=stream)
        attend(A(turned), *self.caches, step["table"], step["starts"], step["lens"], gate=A(q), scale=D ** -0.5,
               out=A(o), stream=stream)
        Q.quantized_matmul(A(o.view(T, -1)), *self.o_proj, self.mode, out=A(y), stream=stream)
        return y

    def read(self, slots: torch.Tensor, stream, dtype: torch.dtype = torch.float32):
        """The keys and values in the rows `slots` (int32) of a cache held in 8 bits: two [T, Hkv, D], exact in float32."""
        if not self.eight:
            raise ValueError("only a layer of cache='e4m3' is read back")
        k, v = (torch.empty(slots.numel(), self.Hkv, self.D, dtype=dtype, device="cuda") for _ in range(2))
        A = Q.Array.from_torch
        Q.cache_read_fp8(*self.caches, A(slots, Q.INT32), dtype=A(k).dtype, k_out=A(k), v_out=A(v), stream=stream)
        return k, v


def main(prompts=(700, 96, 1, 2048), tokens: int = 16, K: int = 5120, cache: str = "bfloat16"):
    R, block = len(prompts), 16
    width = -(-(max(prompts) + tokens) // block)
    pages = Pages(R, R * width, block, width)
    layer = AttentionLayer(K, 24, 4, 256, 64, R * width, block, cache=cache)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        s = Q.Stream.torch_current()
        x = torch.randn(sum(prompts), K, device="cuda").to(torch.bfloat16)
        pages.new.copy_(torch.tensor(prompts, dtype=torch.int32))
        layer(x, pages.step(x.shape[0], s), s)
        pages.new.fill_(1)
        x = torch.randn(R, K, device="cuda").to(torch.bfloat16)
        layer(x, pages.step(R, s), s)  # (the workspaces are there before the capture)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = layer(x, pages.step(R, s), s)
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(tokens - 1):
            graph.replay()
        end.record()
        stream.synchronize()
    print(f"{R} requests, {pages.lens.tolist()} tokens each: decode step {begin.elapsed_time(end) / (tokens - 1) * 1e3:.1f} us"
          f", |y| {y.float().abs().mean().item():.4f}")


if __name__ == "__main__":
    main(cache=sys.argv[1] if len(sys.argv) > 1 else "bfloat16")
