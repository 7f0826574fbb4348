"""The serving operators together, as examples/serve_block.py uses them:
prompts, single tokens, a request that ends and one that takes its pages, each
step against the same block whose cache is a plain list of keys and values per
request and whose attention, rotary positions and adapters are torch
operations in FP32.

Tolerance, derived: the two differ in the roundings to FP16 of the values the
operators return (adapters twice, rotary twice, attention) and in what those
carry through two projections and the products between: fewer than 16
roundings of 2^-11 of the largest value at each stage, none amplified (every
projection keeps the size of its input), so 2^-7 of the output's largest."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("serve_block", os.path.join(ROOT, "examples", "serve_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


class Plain:
    """The block over plain caches."""

    def __init__(self, block, requests, cos_sin):
        self.b, self.cos_sin = block, cos_sin
        self.keys = [[] for _ in range(requests)]
        self.values = [[] for _ in range(requests)]

    def adapted(self, y, x, lora, ids):
        a, b = lora
        y = y.float()
        for m, i in enumerate(ids.tolist()):
            if i >= 0:
                y[m] += self.b.scales[i] * (b[i].float() @ (a[i].float() @ x[m].float()))
        return y.half()

    def turned(self, x, pos):
        half = x.shape[-1] // 2
        c, s = self.cos_sin[pos, :half], self.cos_sin[pos, half:]
        u, w = x[..., :half].float(), x[..., half:].float()
        return torch.cat([u * c - w * s, w * c + u * s], -1).half()

    @torch.no_grad()
    def __call__(self, h, counts, ids):
        b = self.b
        x = b.norm(h)
        q, k, v = b.q(x), b.k(x), b.v(x)
        q, v = self.adapted(q, x, b.q_lora, ids), self.adapted(v, x, b.v_lora, ids)
        out, m = torch.zeros(h.shape[0], b.heads, b.dim, device="cuda"), 0
        for r, n in enumerate(counts):
            for _ in range(n):
                pos = len(self.keys[r])
                self.keys[r].append(self.turned(k[m].view(b.kv_heads, b.dim), pos))
                self.values[r].append(v[m].view(b.kv_heads, b.dim))
                K, V = torch.stack(self.keys[r]).float(), torch.stack(self.values[r]).float()
                Q = self.turned(q[m].view(b.heads, b.dim), pos).float()
                for i in range(b.heads):
                    j = i // (b.heads // b.kv_heads)
                    out[m, i] = torch.softmax(K[:, j] @ Q[i] * b.dim ** -0.5, 0) @ V[:, j]
                m += 1
        return b.after(h, out.half())


def test_block_steps(gpu):
    ex = example()
    R, hidden, heads, kv, dim = 4, 512, 8, 2, 64
    block = ex.Block(hidden, heads, kv, dim, 1024, adapters=3, rank=8)
    cache = ex.PagedCache(R, 24, 8, kv, dim, 10, torch.float16)
    cos_sin = ex.rotary_table(80, dim)
    plain = Plain(block, R, cos_sin)
    of_request = torch.tensor([0, 2, -1, 1], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for i, counts in enumerate([[5, 0, 33, 1], [1, 17, 1, 1], [1, 1, 0, 1], [1, 1, 1, 1], [1, 1, 9, 1], [1, 1, 1, 0]]):
        if i == 4:  # request 2 ends; another takes its row, and its pages
            cache.release(2)
            plain.keys[2], plain.values[2] = [], []
        T = sum(counts)
        rows, positions, slots = cache.step(torch.tensor(counts, dtype=torch.int32, device="cuda"), T)
        assert int(cache.pool[1]) == 0
        ids = of_request[rows.long()]
        h = torch.randn(T, hidden, generator=g, device="cuda").half()
        got = block(h, cache, cos_sin, rows, positions, slots, ids)
        want = plain(h, counts, ids)
        err = float((got.float() - want.float()).abs().max())
        assert err <= 2.0 ** -7 * float(want.float().abs().max()), (i, err)
    assert cache.lengths.tolist() == [10, 21, 10, 5]


def test_block_decode_step_in_a_graph(gpu):
    ex = example()
    R, hidden, heads, kv, dim = 5, 512, 8, 8, 64
    block = ex.Block(hidden, heads, kv, dim, 1024, adapters=2, rank=8, seed=3)
    cache = ex.PagedCache(R, 60, 4, kv, dim, 12, torch.float16)
    cos_sin = ex.rotary_table(48, dim)
    of_request = torch.tensor([0, 1, -1, 1, 0], dtype=torch.int32, device="cuda")
    new = torch.ones(R, dtype=torch.int32, device="cuda")
    h = torch.randn(R, hidden, device="cuda").half()
    lengths, pool = torch.tensor([3, 0, 9, 20, 7], dtype=torch.int32, device="cuda"), cache.pool.clone()
    free = torch.arange(59, -1, -1, dtype=torch.int32, device="cuda")
    cache.free = free

    def step():
        cache.lengths, cache.pool = lengths, pool
        rows, positions, slots = cache.step(new, R)
        return block(h, cache, cos_sin, rows, positions, slots, of_request), cache.lengths, cache.pool

    cache.table[:, :6] = torch.arange(30, dtype=torch.int32, device="cuda").view(R, 6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, L, p = step()
    for _ in range(4):
        h.copy_(torch.randn(h.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, L, p)]
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got[1:], want[1:]):
            assert torch.equal(a, b)
        # (a captured call reads the ortho entries through the same plan or the
        # CSR: sums of another order, one FP16 step at each of the projections)
        assert float((got[0].float() - want[0].float()).abs().max()) <= 2.0 ** -7 * float(want[0].float().abs().max())
        lengths.copy_(got[1])
        pool.copy_(got[2])
