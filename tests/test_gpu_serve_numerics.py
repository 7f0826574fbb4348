"""What the serving operators keep of their intermediate values, and what they
make of infinite ones, against the formulas in 64 bits.

Tolerances, derived: the output's own rounding, 2^-11 (FP16) or 2^-8 (BF16) of
its value plus half the least subnormal; what precedes it in FP32 is stated at
each test."""
import pytest
import torch

from libortho_amd import _C_ops

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,n", [(64, 3), (128, 3), (80, 600), (256, 34), (128, 9000)])
def test_attention_weights_keep_their_bits(gpu, D, n, dtype):
    # Key 0 has the largest score, keys 1 and 2 weights of about a half that
    # nearly agree and opposite values, all others the value zero: the output
    # is the difference of two weights, far below both.  The scores (one
    # product each) are exact; what is made of keys 1 and 2 (magnitude below 1)
    # errs by 2^-24 in the scaling, the subtraction and 2^-23 in the
    # exponential of a weight, below 2^-21 in the difference of the two over a
    # sum of at least 2.
    dt = DT[dtype]
    rng = torch.Generator().manual_seed(D + n)
    H = 16
    k = torch.zeros(n, D)
    k[:, 0] = -30.0
    k[0, 0], k[1, 0], k[2, 0] = 1.0, 0.125, 0.125 - 2.0 ** -10
    v = torch.zeros(n, D)
    v[1], v[2] = 1.0, -1.0
    q = torch.zeros(1, H, D)
    q[0, :, 0] = torch.randint(128, 256, (H,), generator=rng) / 256.0
    q, k, v = q.to(dt).cuda(), k.to(dt).cuda(), v.to(dt).cuda()
    P = 16
    pages = -(-n // P)
    kc, vc = (torch.zeros(pages * P, 1, D, dtype=dt, device="cuda") for _ in range(2))
    kc[:n, 0], vc[:n, 0] = k, v
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    for scale in (1.0, 0.75, 0.5):
        got = _C_ops.paged_attention(q, kc.view(pages, P, 1, D), vc.view(pages, P, 1, D), table, i32([n - 1]),
                                     scale=scale)[0].double().cpu()
        s = q[0].double().cpu() @ k.double().cpu().T.contiguous() * scale
        want = torch.softmax(s, -1) @ v.double().cpu()
        bound = U[dt] * 1.01 * want.abs() + TINY[dt] + 2.0 ** -21
        err = (got - want).abs()
        assert bool((err <= bound).all()), (scale, float(err.max()), float(want.abs().max()))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,r", [(3, 16), (40, 40), (600, 64), (70, 256), (900, 200), (520, 20)])
def test_adapter_keeps_the_bits_of_its_low_rank_values(gpu, M, r, dtype):
    # Ranks in pairs: A's rows differ in one element's last bit, B's are 1 and
    # -1, so an output is the difference of low-rank values near 1, far below
    # them.  They are single products times a scale of 8 bits: exact in FP32,
    # as is their difference; the output has only its own rounding (and the
    # sums of a pair's parts in FP32, 2^-22 of 2 a pair at most).
    dt = DT[dtype]
    rng = torch.Generator().manual_seed(M + r)
    K, N, n = 64, 72, 3
    x = torch.zeros(M, K)
    x[:, 5] = 1.0 + torch.randint(0, 128, (M,), generator=rng) / 128.0
    a = torch.zeros(n, r, K)
    a[:, 0::2, 5] = 1.0
    a[:, 1::2, 5] = 1.0 - 2.0 ** -8
    b = torch.zeros(n, N, r)
    pair = torch.arange(N) % (r // 2)
    for i in range(n):
        b[i, torch.arange(N), 2 * pair] = 1.0
        b[i, torch.arange(N), 2 * pair + 1] = -1.0
    scales = 1.0 + torch.randint(0, 2 ** 7, (n,), generator=rng) / 128.0
    ids = torch.randint(-1, n, (M,), generator=rng).int()
    y = torch.zeros(M, N, dtype=dt, device="cuda")
    x, a, b = x.to(dt).cuda(), a.to(dt).cuda(), b.to(dt).cuda()
    got = _C_ops.adapter_add(y, x, a, b, ids.cuda(), scales.cuda()).double().cpu()
    want = torch.zeros(M, N, dtype=torch.float64)
    for m, i in enumerate(ids.tolist()):
        if i >= 0:
            want[m] = float(scales[i]) * (b[i].double().cpu() @ (a[i].double().cpu() @ x[m].double().cpu()))
    bound = U[dt] * 1.01 * want.abs() + TINY[dt] + 2.0 ** -21
    assert float(want.abs().max()) > 2.0 ** -8
    err = (got - want).abs()
    assert bool((err <= bound).all()), (float((err - bound).max()), float(err.max()))


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,P,n", [(128, 16, 300), (64, 7, 90), (80, 16, 40), (256, 8, 33), (128, 16, 9000), (128, 32, 20)])
def test_attention_of_infinite_values_in_sight(gpu, D, P, n, dtype):
    # a value of a key in sight that is infinite makes its element infinite for
    # every query head of that key head, two of opposite signs or a NaN a NaN;
    # all other elements stay as they are without them
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(D + n)
    G, H = 2, 6
    pages = -(-n // P)
    q = (2 * torch.randn(1, H, D, generator=g, device="cuda")).to(dt)
    kc, vc = (torch.randn(pages, P, G, D, generator=g, device="cuda").to(dt) for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    pos = i32([n - 1])
    plain = _C_ops.paged_attention(q, kc, vc, table, pos)
    flat = vc.flatten(0, 1)  # (a view)
    put = {(0, 3): {0: INF}, (0, 4): {n - 1: -INF}, (0, 5): {0: INF, n // 2: INF}, (1, 3): {n // 3: NAN},
           (1, 0): {1: INF, n - 1: -INF}, (1, D - 1): {n // 2: -INF}}
    for (h, d), keys in put.items():
        for j, v in keys.items():
            flat[j, h, d] = v
    got = _C_ops.paged_attention(q, kc, vc, table, pos)
    for h in range(H):
        for d in range(D):
            vals = put.get((h // (H // G), d))
            if vals is None:
                continue
            want = sum(vals.values())
            x = float(got[0, h, d])
            assert (x != x) if want != want else x == want, (h, d, x, want)
            plain[0, h, d] = got[0, h, d] = 0
    assert torch.equal(got, plain)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,r,N", [(3, 16, 264), (40, 40, 100), (600, 64, 264), (70, 200, 72), (900, 20, 130), (530, 3, 33)])
def test_adapters_of_infinite_weights(gpu, M, r, N, dtype):
    # an infinite element of B makes its output infinite (with the sign of the
    # low-rank value), of A whatever the formula says, one of the adapter's low-rank
    # values infinite and the others as large as they were
    dt = DT[dtype]
    K, n = 72, 2
    g = torch.Generator(device="cuda").manual_seed(M + r)
    x = (torch.rand(M, K, generator=g, device="cuda") + 0.5).to(dt)
    a = (torch.rand(n, r, K, generator=g, device="cuda") + 0.5).to(dt)
    b = (torch.rand(n, N, r, generator=g, device="cuda") + 0.5).to(dt)
    y = torch.randn(M, N, generator=g, device="cuda").to(dt)
    ids = (torch.arange(M, device="cuda") % n).int()
    plain = _C_ops.adapter_add(y, x, a, b, ids)
    b[0, 5, 0], b[0, 6, r - 1], b[0, 7, 1] = INF, -INF, NAN
    got = _C_ops.adapter_add(y, x, a, b, ids)
    of = (ids == 0).nonzero().flatten()
    assert bool((got[of, 5] == INF).all()) and bool((got[of, 6] == -INF).all()) and bool(got[of, 7].isnan().all())
    got[of, 5:8] = plain[of, 5:8] = 0
    assert torch.equal(got, plain)
    # one infinite low-rank value, the others past FP16's largest number
    big = 200.0
    x2, a2 = (x * big).to(dt), (a * big).to(dt)
    a2[1, 0, 3] = INF
    b2 = torch.ones_like(b)
    b2[:, :, 1:] = -1.0
    got = _C_ops.adapter_add(y, x2, a2, b2, ids)
    of = (ids == 1).nonzero().flatten()
    assert bool((got[of] == INF).all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n", [1, 64, 40000])
def test_attention_of_the_types_largest_and_smallest_values(gpu, n, dtype):
    # equal weights over equal values: the value, however many
    dt, P, D = DT[dtype], 16, 64
    pages = -(-n // P)
    kc = torch.zeros(pages, P, 1, D, dtype=dt, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    q = torch.ones(1, 3, D, dtype=dt, device="cuda")
    for v in (torch.finfo(dt).max, torch.finfo(dt).min):
        got = _C_ops.paged_attention(q, kc, torch.full_like(kc, v), table, i32([n - 1]))
        assert bool((got == v).all()), (v, float(got[0, 0, 0]))
    least = 4 * TINY[dt]  # two of the smallest steps
    got = _C_ops.paged_attention(q, kc, torch.full_like(kc, least), table, i32([n - 1])).double()
    # (FP32 steps of 2^-149 a key in BF16: with the weights' 2^16 half a step of the type)
    assert bool(((got - least).abs() <= 2 * TINY[dt]).all())
