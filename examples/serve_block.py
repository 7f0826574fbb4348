"""A decoder block serving many requests: the block's seven projections are
OrthoLinear layers, everything between them the library's serving operators.

    python examples/serve_block.py [--hidden 4096 --heads 32 --kv-heads 8 ...]

Each step takes whatever tokens the requests bring (a prompt, one token, or
none), with no word from the GPU in between:

  page_step        pages, cache slots and positions from the requests' lengths
  forward_group    q, k and v of all tokens in one call
  adapter_add      each request's low-rank adapter beside q and v
  cache_append     rotary positions; keys and values to their slots
  paged_attention  every token over its own request's pages

The block's weights are random: the point is the calls and their order.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from libortho_amd import OrthoLinear, _C_ops  # noqa: E402


def rotary_table(positions, rot, base=10000.0, device="cuda"):
    """cos_sin [positions, rot] for cache_append: cosines, then sines."""
    freq = base ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


class PagedCache:
    """One layer's keys and values, the pages' owners, and the requests' lengths."""

    def __init__(self, requests, pages, page_size, kv_heads, dim, width, dtype, device="cuda"):
        self.page_size = page_size
        self.k = torch.zeros(pages, page_size, kv_heads, dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.table = torch.zeros(requests, width, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.pool = torch.zeros(2, dtype=torch.int32, device=device)

    def step(self, new_tokens, tokens):
        """Rows, positions and slots of a step's `tokens` tokens."""
        self.lengths, self.pool, _, rows, positions, slots = _C_ops.page_step(
            self.lengths, new_tokens, self.table, self.free, self.pool, self.page_size, tokens)
        return rows, positions, slots

    def release(self, request):
        """A finished request's pages go back to the free ones (between steps)."""
        used, n = int(self.pool[0]), -(-int(self.lengths[request]) // self.page_size)
        self.free = torch.cat([self.free[used:], self.table[request, :n]])
        self.pool = torch.zeros_like(self.pool)
        self.lengths[request] = 0


class Block(nn.Module):
    def __init__(self, hidden, heads, kv_heads, dim, ffn, adapters, rank, density=0.01, dtype=torch.float16, seed=0):
        super().__init__()
        g = torch.Generator(device="cuda").manual_seed(seed)

        def linear(k, n):
            layer = OrthoLinear(k, n, group_size=128 if k % 128 == 0 else None).cuda()
            w = torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
            keep = torch.rand(n, k, generator=g, device="cuda") < density
            layer.load_from_weights(w, torch.where(keep, 0.1 * w, torch.zeros_like(w)))
            return layer

        def lowrank(k, n):
            return (torch.randn(adapters, rank, k, generator=g, device="cuda").mul_(k ** -0.5).to(dtype),
                    torch.randn(adapters, n, rank, generator=g, device="cuda").mul_(0.3 * rank ** -0.5).to(dtype))

        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.q, self.k, self.v = linear(hidden, heads * dim), linear(hidden, kv_heads * dim), linear(hidden, kv_heads * dim)
        self.o, self.down = linear(heads * dim, hidden), linear(ffn, hidden)
        self.gate, self.up = linear(hidden, ffn), linear(hidden, ffn)
        self.q_lora, self.v_lora = lowrank(hidden, heads * dim), lowrank(hidden, kv_heads * dim)
        self.scales = torch.full((adapters,), 2.0, device="cuda")

    @staticmethod
    def norm(h):
        return (h.float() * (h.float().square().mean(-1, keepdim=True) + 1e-5).rsqrt()).to(h.dtype)

    def projections(self, h, adapters):
        x = self.norm(h)
        q, k, v = OrthoLinear.forward_group([self.q, self.k, self.v], x)
        _C_ops.adapter_add(q, x, *self.q_lora, adapters, self.scales, out=q)
        _C_ops.adapter_add(v, x, *self.v_lora, adapters, self.scales, out=v)
        return (q.view(-1, self.heads, self.dim), k.view(-1, self.kv_heads, self.dim), v.view(-1, self.kv_heads, self.dim))

    def after(self, h, attended):
        h = h + self.o(attended.reshape(h.shape[0], -1))
        gate, up = OrthoLinear.forward_group([self.gate, self.up], self.norm(h))
        return h + self.down(nn.functional.silu(gate.float()).to(up.dtype) * up)

    @torch.no_grad()
    def forward(self, h, cache, cos_sin, rows, positions, slots, adapters):
        q, k, v = self.projections(h, adapters)
        q = _C_ops.cache_append(k, v, cache.k, cache.v, slots, q=q, positions=positions, cos_sin=cos_sin, q_out=q)
        return self.after(h, _C_ops.paged_attention(q, cache.k, cache.v, cache.table, positions, rows=rows))


def main():
    p = argparse.ArgumentParser()
    for name, value in (("hidden", 4096), ("heads", 32), ("kv-heads", 8), ("dim", 128), ("ffn", 11008), ("requests", 8),
                        ("prompt", 100), ("steps", 20), ("page-size", 16), ("adapters", 4), ("rank", 16)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args()
    R, width = a.requests, -(-(a.prompt + a.steps) // a.page_size)
    block = Block(a.hidden, a.heads, a.kv_heads, a.dim, a.ffn, a.adapters, a.rank)
    cache = PagedCache(R, R * width, a.page_size, a.kv_heads, a.dim, width, torch.float16)
    cos_sin = rotary_table(width * a.page_size, a.dim)
    of_request = (torch.arange(R, device="cuda") % (a.adapters + 1) - 1).int()  # -1: a request without an adapter
    prompts = [1 + (a.prompt - 1) * (r + 1) // R for r in range(R)]
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(a.steps):
        counts = prompts if i == 0 else [1] * R
        new = torch.tensor(counts, dtype=torch.int32, device="cuda")
        if i == 2:  # (the first steps lay out the layers' ortho entries)
            begin.record()
        rows, positions, slots = cache.step(new, sum(counts))
        h = torch.randn(sum(counts), a.hidden, device="cuda").half()
        out = block(h, cache, cos_sin, rows, positions, slots, of_request[rows.long()])
    end.record()
    torch.cuda.synchronize()
    print(f"{R} requests, {sum(prompts)} prompt tokens, {a.steps - 1} tokens each after them; "
          f"lengths {cache.lengths.tolist()}, status {int(cache.pool[1])}, finite {bool(out.isfinite().all())}")
    if a.steps > 2:
        print(f"{begin.elapsed_time(end) / (a.steps - 2) * 1e3:.0f} us a step of {R} tokens")


if __name__ == "__main__":
    main()
