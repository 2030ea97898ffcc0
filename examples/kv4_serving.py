"""A small serving loop over a 4-bit key-value cache: W8A8 projections, norm and
rotation, append, attention, and pages that are forked, released and compacted.

    python examples/kv4_serving.py

Random weights of a few layers; two prompts are read in, one of them is sampled
three times from its end on, a row is given back, the pages are compacted, and
decoding goes on.  All arithmetic is the library's; torch holds the tensors.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from baracuda_amd import kv4, plans as P  # noqa: E402


class Linear:
    """y = x W^T with int8 weights and per-token int8 activations."""

    def __init__(self, c_out: int, k: int, g: torch.Generator, dev):
        self.w = torch.randint(-127, 128, (c_out, k), generator=g, dtype=torch.int8).to(dev)
        self.scale = torch.full((c_out,), 1.0 / (73.0 * k ** 0.5), device=dev)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        (m, k), n = x.shape, self.w.shape[0]
        out = torch.empty(m, n, dtype=torch.bfloat16, device=x.device)
        P.QuantizedLinearPlan.select(P.QuantizedLinearDescriptor(m, n, k)).run(
            x, self.w, self.scale, out, torch.empty(m, k, dtype=torch.int8, device=x.device),
            torch.empty(m, dtype=torch.float32, device=x.device))
        return out


class Server:
    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, dim=128, page_size=16, pages=64, rows=8, max_pages=32,
                 max_positions=512, dev="cuda:0", seed=0):
        self.__dict__.update(layers=layers, hidden=hidden, heads=heads, kv_heads=kv_heads, dim=dim, ps=page_size, pages=pages,
                             rows=rows, max_pages=max_pages, dev=dev)
        g = torch.Generator().manual_seed(seed)
        self.qkv = [Linear((heads + 2 * kv_heads) * dim, hidden, g, dev) for _ in range(layers)]
        self.proj = [Linear(hidden, heads * dim, g, dev) for _ in range(layers)]
        self.norms = [[(1 + 0.1 * torch.randn(dim, generator=g)).to(torch.bfloat16).to(dev) for _ in range(2)]
                      for _ in range(layers)]
        angle = torch.arange(max_positions)[:, None] * 1e4 ** (-torch.arange(dim // 2) / (dim // 2))
        self.cos, self.sin = angle.cos().to(dev), angle.sin().to(dev)
        self.page_bytes = kv_heads * kv4.head_bytes(page_size, dim)
        self.cache = torch.zeros(layers, pages, self.page_bytes, dtype=torch.uint8, device=dev)
        self.tables = torch.full((rows, max_pages), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.manage = kv4.KvPagesPlan.select(kv4.KvPagesDescriptor(layers, pages, self.page_bytes, page_size, rows, max_pages))

    def grow(self, rows, counts) -> list[int]:
        """Room for `counts` more tokens of the rows: the lengths before, pages taken where needed."""
        tables, lens, refs = self.tables.cpu(), self.lens.cpu(), self.refs.cpu()
        before = [int(lens[r]) for r in rows]
        for r, n in zip(rows, counts):
            for j in range(-(-int(lens[r]) // self.ps), -(-(int(lens[r]) + n) // self.ps)):
                page = int((refs == 0).nonzero()[0])
                tables[r, j], refs[page] = page, 1
            lens[r] += n
        self.tables.copy_(tables)
        self.lens.copy_(lens)
        self.refs.copy_(refs)
        return before

    def step(self, rows, x: list[torch.Tensor]) -> list[torch.Tensor]:
        """New tokens x[i] [n_i, hidden] of the rows through all layers."""
        counts = [len(t) for t in x]
        before = self.grow(rows, counts)
        total, dev = sum(counts), self.dev
        pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, counts)])
        row = torch.tensor(rows).repeat_interleave(torch.tensor(counts))
        slots = (self.tables.cpu()[row, pos // self.ps].long() * self.ps + pos % self.ps).to(dev)
        pos = pos.to(torch.int32)[None].to(dev)
        cu = torch.cumsum(torch.tensor([0] + counts), 0).to(torch.int32).to(dev)
        at = torch.tensor(rows, device=dev)
        tables, lens = self.tables[at].contiguous(), self.lens[at].contiguous()
        most = max(b + n for b, n in zip(before, counts))
        append = kv4.Kv4AppendPlan.select(kv4.Kv4AppendDescriptor(total, self.heads, self.kv_heads, self.dim, self.ps, self.pages,
                                                                  self.dim))
        attend = kv4.Kv4AttentionPlan.select(kv4.Kv4AttentionDescriptor(
            len(rows), total, max(counts), most, self.heads, self.kv_heads, self.dim, self.ps, self.pages, self.max_pages))
        ws = torch.empty(attend.workspace_size(), dtype=torch.uint8, device=dev)
        h = torch.cat(x)
        for i in range(self.layers):
            qkv = self.qkv[i](h).view(total, self.heads + 2 * self.kv_heads, self.dim)
            q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 1)
            cache = self.cache[i].view(self.pages, self.kv_heads, -1)
            append.run(k, v, cache, slots, q=q, q_out=q, q_weight=self.norms[i][0], k_weight=self.norms[i][1], positions=pos,
                       cos=self.cos, sin=self.sin)
            out = torch.empty(total, self.heads, self.dim, dtype=torch.bfloat16, device=dev)
            attend.run(q, cache, tables, lens, out, cu_q=cu, workspace=ws)
            h = h + self.proj[i](out.view(total, -1))
        return list(h.split(counts))

    def fork(self, parents, children) -> torch.Tensor:
        fresh = torch.empty(len(parents), dtype=torch.int32, device=self.dev)
        ids = [torch.tensor(t, dtype=torch.int32, device=self.dev) for t in (parents, children)]
        self.manage.fork(self.cache, self.tables, self.lens, self.refs, *ids, fresh)
        return fresh

    def release(self, rows) -> None:
        self.manage.release(self.tables, self.lens, self.refs, torch.tensor(rows, dtype=torch.int32, device=self.dev))

    def compact(self) -> int:
        refs, remap = torch.empty_like(self.refs), torch.empty_like(self.refs)
        live = torch.empty(1, dtype=torch.int32, device=self.dev)
        ws = torch.empty(self.manage.workspace_size(), dtype=torch.uint8, device=self.dev)
        self.manage.compact(self.cache, self.tables, self.refs, self.tables, refs, remap, live, workspace=ws)
        self.refs = refs
        return int(live)


def main(steps: int = 3) -> dict:
    s = Server()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randn(n, s.hidden, generator=g).to(torch.bfloat16).to(s.dev) for n in (45, 20)]
    first = s.step([0, 1], prompts)
    print(f"prompts of {[len(p) for p in prompts]} tokens hold {int((s.refs > 0).sum())} pages")
    fresh = s.fork([0, 0], [2, 3])
    print(f"row 0 forked twice: {int((s.refs > 0).sum())} pages, {int((s.refs > 1).sum())} of them shared, new {fresh.tolist()}")
    samples = []
    for i in range(steps):
        token = torch.randn(1, s.hidden, generator=g).to(torch.bfloat16).to(s.dev)
        other = torch.randn(1, s.hidden, generator=g).to(torch.bfloat16).to(s.dev)
        samples.append(s.step([0, 1, 2, 3], [token, other, token, other]))   # row 2 is given what row 0 is
    s.release([1])
    live = s.compact()
    print(f"row 1 given back, compacted to {live} pages")
    token = torch.randn(1, s.hidden, generator=g).to(torch.bfloat16).to(s.dev)
    last = s.step([0, 2, 3], [token] * 3)
    torch.cuda.synchronize()
    return {"server": s, "first": first, "samples": samples, "last": last, "live": live}


if __name__ == "__main__":
    out = main()
    print("last outputs:", [float(t.float().norm()) for t in out["last"]])
