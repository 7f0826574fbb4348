"""paged_attention_int4 keeps FP32's bits in its sums: parts that cancel leave
what is small beside them, in scores and in outputs.

References are the formula in 64 bits over the values that the codes stand
for.  Tolerances, derived: FP32 sums of n products are off by n 2^-24 of the
sum of their magnitudes, here of the products that there are (code times
scale, and low) and not of the largest codes there could be.  A score of D
products, and a scale and a low for each group, is off by d = (D + 16) 2^-24
sum |q| (u scale + |low|) |softmax scale|: weights moved by d of themselves
move the output by sum p d |v - output|, 2 d sum p |v| at the most (both parts
of a value have the same weight).  Sums over n keys add n 2^-24, exponentials,
quotients and the weights' parts less than 2^-20, of sum p (u scale + |low|);
and the output is rounded once."""
import numpy as np
import pytest
import torch

from libortho_amd import _C_ops
from oracle import cache_oracle as O
from test_gpu_int4 import DT, TINY, U, i32, np64

pytestmark = pytest.mark.gpu

LAYOUTS = [(128, 128), (128, 32), (64, 64), (80, 80), (96, 32), (256, 64), (8, 8)]


def cache_of(codes, scales, lows, pages, P):
    """One request's keys or values: codes [keys, D], scale and low [keys, groups], in `pages` pages."""
    n, D = codes.shape
    rows, pairs = np.zeros((pages * P, 1, O.row_bytes(D)), np.uint8), np.zeros((pages * P, 1, scales.shape[1], 2), np.float16)
    rows[:n, 0], pairs[:n, 0] = O.pack(codes.astype(np.uint8)), np.stack([scales, lows], -1)
    return [torch.from_numpy(rows.reshape(pages, P, 1, -1)).cuda(), torch.from_numpy(pairs.reshape(pages, P, 1, -1, 2)).cuda()]


def check(q, key, value, P, scale, more=0.0, hidden=(), lost=0.0):
    """q [H, D] in its type; key and value (codes, scales, lows) of one request, which q's heads share.  more: added to d;
    hidden: elements in which every key is 0, which add nothing to d;
    lost: added to the bound."""
    n, D = key[0].shape
    pages, dt = -(-n // P), q.dtype
    cache = cache_of(*key, pages, P) + cache_of(*value, pages, P)
    table = torch.arange(pages, device="cuda", dtype=torch.int32)[None].contiguous()
    got = np64(_C_ops.paged_attention_int4(q[None].contiguous(), *cache, table, i32([n - 1]), scale=scale))[0]

    def numbers(x):
        codes, scales, lows = (np.asarray(a, np.float64) for a in x)
        wide = lambda a: np.repeat(a.astype(np.float16).astype(np.float64), D // scales.shape[1], -1)
        return wide(lows) + codes * wide(scales), np.abs(wide(lows)) + codes * np.abs(wide(scales))

    (k, kmag), (v, vmag), qq = numbers(key), numbers(value), np64(q)
    kmag[:, list(hidden)] = 0
    s, d = qq @ k.T * scale, (np.abs(qq) @ kmag.T).max(-1, keepdims=True) * (D + 16) * 2.0 ** -24 * abs(scale) + more
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    want = p @ v
    bound = U[dt] * 1.01 * np.abs(want) + TINY[dt] + 2 * d * (p @ np.abs(v)) + (2.0 ** -20 + n * 2.0 ** -24) * (p @ vmag) + lost
    err = np.abs(got - want)
    assert (err <= bound).all(), (float((err - bound).max()), float(np.abs(want).max()), float(bound.max()))
    return want, bound


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("P", [16, 5])
@pytest.mark.parametrize("D,group", LAYOUTS)
def test_scores_whose_large_products_cancel(gpu, D, group, P, dtype):
    # +X and -X in every group, all codes 1: what is left of a score is the
    # others' 2^-18 X, by which the first key's value outweighs the second's
    X, G = 64.0, D // group
    q = np.full((2, D), X * 2.0 ** -18)
    q[0, ::group], q[0, 1::group] = X, -X
    q[1, 2::group], q[1, group - 1::group] = -X, X  # (D - 1: a high nibble where vectors have any)
    one, none = np.ones((1, D)), np.zeros((1, D))
    key = (np.concatenate([one, none]), np.ones((2, G)), np.zeros((2, G)))
    value = (np.zeros((2, D)), np.zeros((2, G)), np.repeat([[1.0], [-1.0]], G, 1))
    want, bound = check(torch.tensor(q).to(DT[dtype]).cuda(), key, value, P, 1 / (X * 2.0 ** -18 * (D - 2 * G)))
    # a sum without the small products gives 0, off by tanh(1/2) = 0.46; of four groups of 32 the bound is
    # 2 d = 2 (144 2^-24) (8 2^18 / 120) = 0.30, of the others less
    assert (np.abs(want) > bound).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("P", [16, 5])
@pytest.mark.parametrize("D,group", LAYOUTS)
def test_outputs_whose_largest_value_is_zero(gpu, D, group, P, dtype):
    # a key of nearly all the weight, whose value is -1 + 1, and thirty with 2^-18 of it: they are the output
    G, n = D // group, 31
    q = np.zeros((3, D))
    q[:, 0] = 1
    lows = np.zeros((n, G))
    lows[0, 0] = 18 * np.log(2)
    key = (np.zeros((n, D)), np.zeros((n, G)), lows)
    first = np.zeros((n, G))
    first[0] = -1
    codes = np.ones((n, D))
    want, bound = check(torch.tensor(q).to(DT[dtype]).cuda(), key, (codes, np.ones((n, G)), first), P, 1.0)
    assert (np.abs(want) > bound).all()  # (30 2^-18, beside (16 + 31) 2^-24 of 2 and a hundredth of itself)


@pytest.mark.parametrize("P", [16, 5])
@pytest.mark.parametrize("D,group", LAYOUTS)
def test_queries_whose_elements_sum_past_the_largest_number(gpu, D, group, P):
    # finite BF16 elements of up to 2^127.9, all of one sign and mixed, whose sums pass FP32's largest number: scores are of ordinary size
    rng = np.random.default_rng(D + group)
    q = rng.uniform(1, 3.9, (4, D)) * 2.0 ** 126
    q[1] = -q[1]
    q[2, ::2] = -q[2, ::2]
    q[3, 1:] *= 2.0 ** -rng.integers(0, 12, D - 1)
    n, G = 40, D // group

    def side():
        return rng.integers(0, 16, (n, D)), rng.uniform(0.01, 0.02, (n, G)), rng.uniform(-0.2, -0.1, (n, G))
    check(torch.tensor(q).bfloat16().cuda(), side(), side(), P, 2.0 ** -126)


@pytest.mark.parametrize("dtype,k", [("fp16", 24), ("fp16", 27), ("fp16", 30), ("fp16", 34), ("bf16", 24), ("bf16", 30), ("bf16", 33), ("bf16", 36)])
@pytest.mark.parametrize("D,group", LAYOUTS)
def test_small_elements_beside_a_querys_largest(gpu, D, group, dtype, k):
    """The largest element meets a 0 in every key, the others are 2^-k of it.
    Down to 2^-28 (BF16: 2^-31) of the largest they keep all their bits, below
    that each is off by at most 2^-39 of it; a matrix product of such
    elements alone adds less than a hundredth of that."""
    rng = np.random.default_rng(D + group + k)
    X, G, n = 2.0 ** 15, D // group, 20
    q = rng.uniform(1, 2, (6, D)) * X * 2.0 ** -k * rng.choice([-1, 1], (6, D))
    at = [0, D - 1, 5]  # (and a high nibble where vectors have any)
    codes = rng.integers(0, 16, (n, D))
    codes[:, at] = 8
    for h in range(6):
        q[h, at] = 0
        q[h, at[h % 3]] = X
    q = torch.tensor(q).to(DT[dtype]).cuda()
    key = (codes, np.ones((n, G)), np.full((n, G), -8.0))
    value = (np.zeros((n, D)), np.zeros((n, G)), rng.standard_normal((n, G)))
    scale = 1 / (X * 2.0 ** -k * 8 * D ** 0.5)
    exact = k <= (28 if dtype == "fp16" else 31)
    check(q, key, value, 16, scale, more=0 if exact else 1.01 * 2.0 ** -39 * X * scale * np.abs(codes - 8).sum(-1).max(), hidden=at)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("ratio", [-20, -28, -32])
@pytest.mark.parametrize("D,group,P", [(128, 32, 16), (128, 64, 5), (96, 32, 16), (256, 128, 16), (64, 32, 8)])
def test_groups_of_values_of_very_different_scales(gpu, D, group, P, ratio, dtype):
    """The second group's scales are 2^ratio of the others'.  A weight times a
    scale is off by 2^-24 of itself or by 2^-39 of the largest of its token
    and head, whichever is more: a group of 2^-20 of the largest keeps 2^-19
    of its own sums, one of 2^-28 2^-11, in the formula and in what is tested."""
    rng = np.random.default_rng(D - ratio)
    n, G, H = 70, D // group, 3
    q = torch.tensor(rng.standard_normal((H, D))).to(DT[dtype]).cuda()
    key = (rng.integers(0, 16, (n, D)), rng.uniform(0.1, 0.3, (n, G)), rng.uniform(-2, -1, (n, G)))
    scales = rng.uniform(2048, 4096, (n, G))  # (from 2^11 on, so that FP16 holds 2^-32 of them)
    scales[:, 1] = 2.0 ** np.maximum(11 + ratio, -24) * rng.integers(1, 4, n)
    lows = -8 * scales
    value = (rng.integers(0, 16, (n, D)), scales, lows)
    scale = D ** -0.5
    # what the smallest group may lose: 2^-39 of the largest product of a weight and a scale, for each key's |u - 8|
    qq, wide = np64(q), lambda a: np.repeat(np.asarray(a).astype(np.float16).astype(np.float64), group, -1)
    s = qq @ (wide(key[2]) + key[0] * wide(key[1])).T * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    lost = 1.01 * 2.0 ** -39 * (p * scales.astype(np.float16).astype(np.float64).max(-1)).max(-1)[:, None] * np.abs(value[0] - 8).sum(0)
    check(q, key, value, P, scale, lost=lost)
