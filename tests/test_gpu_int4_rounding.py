"""How cache_append_int4 rounds, at numbers where one rounding to FP16 and two
(64 bits to FP32, FP32 to FP16, each to nearest even) differ: turned keys and
scales go through FP32, as the header says.  Whole numbers, no tolerance."""
import numpy as np
import pytest
import torch

from libortho_amd import _C_ops
from oracle import cache_oracle as O

pytestmark = pytest.mark.gpu


def append(k, v, cos_sin, interleaved, group):
    T, G, D = k.shape
    cache = _C_ops.int4_cache(T, 1, G, D, group)
    _C_ops.cache_append_int4(k, v, *cache, torch.arange(T, device="cuda"), positions=torch.zeros(T, dtype=torch.int32, device="cuda"),
                             cos_sin=cos_sin, interleaved=interleaved)
    return cache


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,group", [(64, 32), (128, 128), (80, 80), (256, 64)])
def test_turned_keys_are_rounded_through_fp32(gpu, D, group, dtype, interleaved):
    # a = b = -1: a c - b s = -(c - s).  Each token's first elements are small parts (2^-26) to either side of a border
    # between two FP16 numbers, which FP32 does not hold: two roundings are the even neighbour's, one the nearer's
    borders = [1 + (2 * i + 1) * 2.0 ** -11 for i in (0, 1, 5, 6, 511, 1022)]
    half = D // 2
    keys = torch.full((len(borders) * 2, 1, D), 0.0, dtype=dtype, device="cuda")
    a, b = (0, 1) if interleaved else (0, half)
    keys[:, 0, a] = keys[:, 0, b] = -1
    differ = 0
    for i, c in enumerate(borders):
        for j, s in enumerate((2.0 ** -26, -2.0 ** -26)):
            cs = torch.zeros(1, D, device="cuda")
            cs[0, 0], cs[0, half] = c, s
            cache = append(keys[:1], keys[:1], cs, interleaved, group)
            angles = cs.double().cpu().numpy()
            turned = O.turn(keys[:1].double().cpu().numpy(), angles[:, :half], angles[:, half:], interleaved)
            u, scale, low = O.quantise(turned, group)
            np.testing.assert_array_equal(cache[0][0].cpu().numpy(), O.pack(u))
            np.testing.assert_array_equal(cache[1][0].cpu().numpy(), np.stack([scale, low], -1))
            exact = -(c - s)  # (a sum of 27 bits, exact in 64)
            assert turned[0, 0, a] == exact and float(cache[1][0, 0, 0, 0, 1]) <= np.float16(np.float32(exact))
            differ += np.float16(np.float32(exact)) != np.float16(exact)
    assert differ == len(borders)  # (of the two sides of each border, the even neighbour's is one)


def scales_of_two_roundings():
    """Pairs of FP16 numbers (low, high) whose (high - low) / 15 is rounded to another FP16 number through FP32 than at once."""
    rng = np.random.default_rng(0)
    low = (rng.standard_normal(4_000_000) * 2.0 ** -rng.integers(8, 14, 4_000_000)).astype(np.float16)  # (differences of many bits)
    high = (9 * rng.standard_normal(4_000_000)).astype(np.float16)
    s = (high.astype(np.float64) - low.astype(np.float64)) / 15
    at = np.nonzero((s > 0) & (s.astype(np.float32).astype(np.float16) != s.astype(np.float16)))[0]
    return low[at], high[at]


def test_scales_are_rounded_through_fp32(gpu):
    low, high = scales_of_two_roundings()
    assert len(low) >= 20
    low, high, D = low[:200], high[:200], 32
    x = np.linspace(0, 1, D)[None] * (high - low)[:, None].astype(np.float64) + low[:, None]
    x[:, 3], x[:, 7] = low, high
    x = x.clip(low[:, None], high[:, None]).astype(np.float16)
    v = torch.from_numpy(x)[:, None].cuda()
    cache = append(v, v, torch.zeros(1, 0, device="cuda"), False, D)
    u, scale, lows = O.quantise(x.astype(np.float64)[:, None], D)
    once = ((high.astype(np.float64) - low.astype(np.float64)) / 15).astype(np.float16)
    assert (scale[:, 0, 0] != once).all()
    for codes, pairs in (cache[:2], cache[2:]):
        np.testing.assert_array_equal(codes[:, 0].cpu().numpy(), O.pack(u))
        np.testing.assert_array_equal(pairs[:, 0].cpu().numpy(), np.stack([scale, lows], -1))


def test_reading_rounds_to_fp16_once_and_to_bf16_from_fp32(gpu):
    # low + u scale whose FP32 number lies on a border between two BF16 ones, or FP16 ones, and the exact number beside it
    D = 8
    rng = np.random.default_rng(1)
    s, m = rng.uniform(2.0 ** -14, 1, (200000, 1)).astype(np.float16), (rng.standard_normal((200000, 1)) * 300).astype(np.float16)
    u = rng.integers(0, 16, (200000, D)).astype(np.uint8)
    exact = m.astype(np.float64) + u * s.astype(np.float64)
    f32 = torch.from_numpy(exact.astype(np.float32))
    rows = torch.from_numpy(O.pack(u)).cuda()[:, None, None]
    held = torch.from_numpy(np.concatenate([s, m], 1)).cuda()[:, None, None, None]
    slots = torch.arange(len(u), device="cuda")
    for dtype in (torch.bfloat16, torch.float16):
        got, _ = _C_ops.cache_read_int4(rows, held, rows, held, slots, D, dtype)
        want = f32.bfloat16() if dtype == torch.bfloat16 else torch.from_numpy(exact.astype(np.float16))
        assert torch.equal(got[:, 0].cpu(), want), dtype
