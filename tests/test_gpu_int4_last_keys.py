"""paged_attention_int4 at the end of the widest table there is (2^31 - 512
keys): the last places of the table have pages of their own, so a key that is
missed, taken twice or read from another place changes the result.

Reference: the formula in 64 bits over the keys in sight, with the tolerance
of test_gpu_int4_sums.py, against which every key's weight is large: the test
looks that the output without any one of them is outside."""
import numpy as np
import pytest
import torch

from libortho_amd import _C_ops
from oracle import cache_oracle as O
from test_gpu_int4 import TINY, U, i32, np64, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("P", [32, 28])
@pytest.mark.parametrize("tokens", [1, 3])
def test_every_key_at_the_last_numbers(gpu, P, tokens):
    W, own, D, group, H = ((1 << 31) - 512) // P, 45, 64, 32, 2
    table = torch.zeros(1, W, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(P + tokens)
    order = 1 + torch.randperm(own, generator=g, device="cuda").to(torch.int32)
    table[0, -own:] = order
    cache = random_cache(g, own + 1, P, 1, D, group)
    K, V = (O.values(cache[i].cpu().numpy(), cache[i + 1].cpu().numpy(), D)[:, :, 0] for i in (0, 2))
    mags = [np.repeat(np.abs(s[..., 1]) + 15 * s[..., 0], group, -1)[:, :, 0] for s in (cache[i].double().cpu().numpy() for i in (1, 3))]
    page_of, q = order.cpu().numpy(), (0.3 * torch.randn(tokens, H, D, generator=g, device="cuda")).half()
    scale, held = 0.5 * D ** -0.5, W * P  # (weights near to one another)
    for back, window in ((1, 1), (1, 2), (1, 33), (1, 300), (40, 1000), (7, 1000), (0, 70), (0, 300), (P, 500)):
        # (back 0: the last token's key lies past the table and is not seen)
        last = [held - back - (tokens - 1 - i) for i in range(tokens)]
        rows = i32([0] * tokens) if tokens > 1 else None
        got = np64(_C_ops.paged_attention_int4(q, *cache, table, i32(last), rows=rows, scale=scale, window=window))
        for t in range(tokens):
            j = np.arange(max(0, last[t] + 1 - window), min(last[t] + 1, held))
            place = j // P - (W - own)
            assert place.min() >= 0
            (k, kr), (v, vr) = ((x[page_of[place], j % P], r[page_of[place], j % P]) for x, r in zip((K, V), mags))
            qq = np64(q[t])
            s = qq @ k.T * scale
            d = (np.abs(qq) @ kr.T).max(-1, keepdims=True) * (D + 16) * 2.0 ** -24 * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            want = p @ v
            bound = U[torch.float16] * 1.01 * np.abs(want) + TINY[torch.float16] + 2 * d * (p @ np.abs(v)) + \
                (2.0 ** -20 + len(j) * 2.0 ** -24) * (p @ vr)
            assert (np.abs(got[t] - want) <= bound).all(), (back, window, t, float((np.abs(got[t] - want) - bound).max()))
            if len(j) > 1:
                # the output without key i is (want - p_i v_i) / (1 - p_i): off by p_i (want - v_i) / (1 - p_i)
                off = p[:, :, None] * (want[:, None] - v[None]) / (1 - p[:, :, None])
                assert (np.abs(off) > bound[:, None]).any((0, 2)).all()
