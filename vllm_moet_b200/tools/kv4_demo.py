"""A grouped-query draft layer over the 4-bit paged K/V cache, from prompt to decode.

    python -m vllm_moet_b200.tools.kv4_demo [--hidden 4096 --heads 32 --kv-heads 8 --head-dim 128]
        [--streams 8] [--prompt 8192] [--chunk 2048] [--tokens 32] [--budget 32]

One grouped-query attention layer, as a drafter of a user's own may have it (q / k / v projections, RMS-normed
q and k heads, RoPE, output projection; random weights) runs as such a layer runs in serving:
each stream's prompt in chunks (append the chunk's rows, attend to the whole context), then one
token per stream and step over all pages, and once more with ``--budget`` pages chosen per token
and K/V head.  Prints bytes per position against bf16, device time per step (CUDA events after
warm-up), and how far the outputs are from the same layer with unquantised keys and values.
"""
from __future__ import annotations

import argparse
import json
import math
from dataclasses import dataclass
from typing import Optional

import torch

from ..ops.kv4 import PAGE, KV4Cache


def rms(x: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    x = x.float()
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)


def rope(x: torch.Tensor, pos: torch.Tensor, theta: float = 10000.0) -> torch.Tensor:
    """Rotate the halves of x [T, heads, D] by the positions' angles."""
    D = x.shape[-1]
    inv = theta ** (-torch.arange(0, D, 2, device=x.device) / D)
    a = pos[:, None].float() * inv
    c, s = a.cos()[:, None], a.sin()[:, None]
    u, v = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([u * c - v * s, u * s + v * c], -1)


@dataclass
class GQALayer:
    """Attention of one grouped-query layer."""
    qkv: torch.Tensor          # [(heads + 2 kv_heads) * D, hidden]
    o: torch.Tensor            # [hidden, heads * D]
    heads: int
    kv_heads: int
    head_dim: int

    @classmethod
    def random(cls, hidden: int, heads: int, kv_heads: int, head_dim: int, device, seed: int = 0) -> "GQALayer":
        g = torch.Generator(device=device).manual_seed(seed)

        def w(n, k):
            return (torch.randn(n, k, generator=g, device=device) / math.sqrt(k)).to(torch.bfloat16)
        return cls(w((heads + 2 * kv_heads) * head_dim, hidden), w(hidden, heads * head_dim), heads, kv_heads, head_dim)

    def project(self, x: torch.Tensor, pos: torch.Tensor):
        """x [T, hidden] at positions pos -> (q, k, v) rows in bf16."""
        y = (x @ self.qkv.T).unflatten(1, (-1, self.head_dim))
        H, K = self.heads, self.kv_heads
        q, k = (rope(rms(t), pos).to(torch.bfloat16) for t in (y[:, :H], y[:, H:H + K]))
        return q, k, y[:, H + K:]

    def forward(self, cache: KV4Cache, x, pos, slots, cu_q, seq_lens, table, max_q: int,
                budget: int = 0) -> torch.Tensor:
        """One step: the rows' keys and values into the cache, attention over what it then holds."""
        q, k, v = self.project(x, pos)
        cache.append(k, v, slots)
        pages = cache.select(q, cu_q, seq_lens, table, budget, max_q=max_q) if budget else None
        out = cache.attend(q, cu_q, seq_lens, table, self.head_dim ** -0.5, max_q=max_q, pages=pages)
        return out.flatten(1) @ self.o.T


class Streams:
    """Page tables of a fixed set of streams, pages handed out as they grow."""

    def __init__(self, n: int, max_len: int, device):
        self.width = -(-max_len // PAGE)
        self.table = torch.randperm(n * self.width, device=device).to(torch.int32).view(n, self.width).contiguous()
        self.lens = [0] * n
        self.device = device

    def rows(self, streams, count: int):
        """Append `count` positions to each of `streams`: (positions, slots, cu_q, seq_lens, table)."""
        pos, slots, lens = [], [], []
        for b in streams:
            p = torch.arange(self.lens[b], self.lens[b] + count, device=self.device)
            pos.append(p)
            slots.append(self.table[b, p // PAGE].long() * PAGE + p % PAGE)
            self.lens[b] += count
            lens.append(self.lens[b])
        cu = torch.arange(0, (len(lens) + 1) * count, count, dtype=torch.int32, device=self.device)
        return (torch.cat(pos), torch.cat(slots), cu, torch.tensor(lens, dtype=torch.int32, device=self.device),
                self.table[list(streams)].contiguous())

    def back(self, streams, count: int) -> None:
        for b in streams:
            self.lens[b] -= count


def attention_bf16(layer: GQALayer, q, k, v) -> torch.Tensor:
    """The last row of q [heads, D] over unquantised keys / values [n, kv_heads, D], in f32."""
    G = layer.heads // layer.kv_heads
    s = torch.einsum("hgd,nhd->hgn", q.float().unflatten(0, (-1, G)), k.float()) * layer.head_dim ** -0.5
    return torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v.float()).flatten()


def run(hidden=4096, heads=32, kv_heads=8, head_dim=128, streams=8, prompt=8192, chunk=2048, tokens=32, budget=32,
        seed=0, device="cuda", sink: Optional[callable] = print) -> dict:
    layer = GQALayer.random(hidden, heads, kv_heads, head_dim, device, seed)
    book = Streams(streams, prompt + 2 * tokens + 8, device)
    cache = KV4Cache(streams * book.width, kv_heads, head_dim, device=device)
    g = torch.Generator(device=device).manual_seed(seed + 1)
    x0 = torch.randn(prompt, hidden, generator=g, device=device).to(torch.bfloat16)       # stream 0's inputs are kept
    events = lambda: torch.cuda.Event(enable_timing=True)  # noqa: E731
    t0, t1 = events(), events()
    t0.record()
    for b in range(streams):
        for c in range(0, prompt, chunk):
            n = min(chunk, prompt - c)
            pos, slots, cu, lens, table = book.rows([b], n)
            x = x0[c:c + n] if b == 0 else torch.randn(n, hidden, generator=g, device=device).to(torch.bfloat16)
            layer.forward(cache, x, pos, slots, cu, lens, table, n)
    t1.record()
    torch.cuda.synchronize()
    got = {"bytes_per_position": cache.bytes_per_token, "bf16_bytes_per_position": kv_heads * head_dim * 4,
           "prompt_ms": t0.elapsed_time(t1)}
    everyone = range(streams)
    x = torch.randn(streams, hidden, generator=g, device=device).to(torch.bfloat16)
    q, k0, v0 = layer.project(torch.cat([x0, x[:1]]), torch.arange(prompt + 1, device=device))
    want = attention_bf16(layer, q[-1], k0, v0) @ layer.o.float().T
    for name, n_pages in (("all_pages", 0), ("chosen_pages", budget)):
        times = []
        for i in range(tokens):
            pos, slots, cu, lens, table = book.rows(everyone, 1)
            a, b = events(), events()
            a.record()
            y = layer.forward(cache, x, pos, slots, cu, lens, table, 1, n_pages)
            b.record()
            times.append((a, b))
            if i == 0:
                got[name + "_rel_err"] = float((y[0].float() - want).norm() / want.norm())
            if i < 3:
                book.back(everyone, 1)             # warm-up steps write the same position again
        torch.cuda.synchronize()
        got[name + "_step_us"] = sorted(a.elapsed_time(b) for a, b in times[3:])[len(times[3:]) // 2] * 1e3
        book.back(everyone, tokens - 3)
    cache.check()
    if sink:
        sink(json.dumps({k: round(v, 4) if isinstance(v, float) else v for k, v in got.items()}))
    return got


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("hidden", 4096), ("heads", 32), ("kv-heads", 8), ("head-dim", 128), ("streams", 8),
                          ("prompt", 8192), ("chunk", 2048), ("tokens", 32), ("budget", 32), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=default)
    ap.add_argument("--device", default="cuda")
    run(**{k.replace("-", "_"): v for k, v in vars(ap.parse_args(argv)).items()})
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
