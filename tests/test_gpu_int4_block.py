"""examples/serve_block.py over a cache in 4 bits: prompts, single tokens and a
request that ends, each step against the block whose keys and values are the
oracle's quantised ones and whose attention is the formula in 64 bits.

The block's own q, k and v go through both, so what is compared is attention
and what follows it.  Tolerance, derived: q is rounded to FP16 once more when
it is turned (2^-11 of its largest) and moves a weight by at most that of the
scores' size, below 8 here, twice; attention is rounded once; the products
that follow keep the size of their input and round to FP16 fewer than eight
times: fewer than 32 roundings of 2^-11 of the largest value, 2^-6 of it.  A
code differs by a step where the reference's turned key, in 64 bits from the
same FP16 elements, is the same number: not at all."""
import numpy as np
import pytest
import torch

from oracle import cache_oracle as O
from test_gpu_serve_block import example

pytestmark = pytest.mark.gpu


class Quantised:
    """What the cache should hold of each request, and attention over it."""

    def __init__(self, requests, group, cos_sin):
        self.group, self.cos_sin = group, cos_sin.double().cpu().numpy()
        self.keys, self.values = [[] for _ in range(requests)], [[] for _ in range(requests)]

    def held(self, x):
        u, s, low = O.quantise(x, self.group)
        return O.values(O.pack(u), np.stack([s, low], -1), x.shape[-1])

    def __call__(self, q, k, v, counts):
        q, k, v = (t.double().cpu().numpy() for t in (q, k, v))
        out, m, half = np.zeros(q.shape), 0, q.shape[-1] // 2
        for r, n in enumerate(counts):
            for _ in range(n):
                cs = self.cos_sin[len(self.keys[r])][None]
                self.keys[r].append(self.held(O.turn(k[m:m + 1], cs[:, :half], cs[:, half:], False)[0]))
                self.values[r].append(self.held(v[m]))
                K, V, Q = np.stack(self.keys[r]), np.stack(self.values[r]), O.turn(q[m:m + 1], cs[:, :half], cs[:, half:], False)[0]
                for i in range(Q.shape[0]):
                    j = i // (Q.shape[0] // K.shape[1])
                    s = K[:, j] @ Q[i] * Q.shape[1] ** -0.5
                    p = np.exp(s - s.max())
                    out[m, i] = p @ V[:, j] / p.sum()
                m += 1
        return torch.from_numpy(out).half().cuda()


@pytest.mark.parametrize("kv,dim,group", [(2, 64, 32), (8, 64, 64)])
def test_block_steps_over_an_int4_cache(gpu, kv, dim, group):
    ex = example()
    R, hidden, heads = 4, 512, 8
    block = ex.Block(hidden, heads, kv, dim, 1024, adapters=3, rank=8)
    cache = ex.PagedInt4Cache(R, 24, 8, kv, dim, 10, torch.float16, group_size=group)
    cos_sin = ex.rotary_table(80, dim)
    plain = Quantised(R, group, cos_sin)
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
        with torch.no_grad():
            want = block.after(h, plain(*block.projections(h, ids), counts))
        got = block(h, cache, cos_sin, rows, positions, slots, ids)
        err = float((got.float() - want.float()).abs().max())
        assert err <= 2.0 ** -6 * float(want.float().abs().max()), (i, err)
    assert cache.lengths.tolist() == [10, 21, 10, 5]


def test_the_example_runs_over_either_cache(gpu, monkeypatch, capsys):
    ex = example()
    base = ["serve_block.py", "--hidden", "512", "--heads", "8", "--kv-heads", "2", "--dim", "64", "--ffn", "1024",
            "--requests", "3", "--prompt", "20", "--steps", "4"]
    for more in ([], ["--int4", "32"]):
        monkeypatch.setattr("sys.argv", base + more)
        ex.main()
        assert "finite True" in capsys.readouterr().out
