"""adapter_add against the formula in 64 bits.

Tolerance, derived: the output's own rounding (u = 2^-11 of its value in FP16,
2^-8 in BF16, half the least subnormal); FP32 sums of the K products of each
low-rank value and of the rank products of each output, 2^-24 of the sum of
magnitudes a term; the low-rank values split in two 16-bit parts, 2^-15 of
their largest one at most."""
import pytest
import torch

from libortho_amd import _C_ops, _lib

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def case(M, K, N, r, n, dt, seed=0, sigma=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + M + K + r)
    x = (sigma * torch.randn(M, K, generator=g, device="cuda")).to(dt)
    y = torch.randn(M, N, generator=g, device="cuda").to(dt)
    a = (K ** -0.5 * torch.randn(n, r, K, generator=g, device="cuda")).to(dt)
    b = (0.5 * r ** -0.5 * torch.randn(n, N, r, generator=g, device="cuda")).to(dt)
    ids = torch.randint(-1, n, (M,), generator=g, device="cuda", dtype=torch.int32)
    scales = torch.rand(n, generator=g, device="cuda") * 2
    return y, x, a, b, ids, scales


def check(y, x, a, b, ids, scales=None, out=None):
    y0 = y.double().cpu()
    got = _C_ops.adapter_add(y, x, a, b, ids, scales, out=out)
    K, r, dt = x.shape[1], a.shape[1], x.dtype
    want, bound = y0.clone(), torch.zeros_like(y0)
    for m, i in enumerate(ids.tolist()):
        if not 0 <= i < a.shape[0]:
            assert torch.equal(got[m].cpu(), y0[m].to(dt))
            continue
        X, A, B = x[m].double().cpu(), a[i].double().cpu(), b[i].double().cpu()
        s = 1.0 if scales is None else float(scales[i])
        low = A @ X
        want[m] += s * (B @ low)
        sums = (K + r + 8) * 2.0 ** -24 * (B.abs() @ (A.abs() @ X.abs()))
        split = 2.0 ** -15 * B.abs().sum(1) * float(low.abs().max())
        bound[m] = s * (sums + split)
    bound += U[dt] * 1.01 * want.abs() + TINY[dt] + 2.0 ** -23 * y0.abs()
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())
    return got


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,N,r,n", [
    (1, 4096, 4096, 16, 1), (3, 512, 700, 8, 2), (16, 256, 256, 32, 5), (33, 1024, 1000, 64, 3), (64, 512, 1536, 16, 64),
    (65, 512, 512, 128, 1), (130, 264, 333, 20, 7), (257, 1000, 999, 4, 4), (70, 96, 64, 256, 3), (40, 128, 130, 1, 3),
    (9, 33, 17, 5, 2), (12, 1, 1, 3, 2), (300, 2048, 512, 24, 2), (5, 11008, 4096, 40, 9), (600, 1000, 200, 64, 1),
    (577, 512, 264, 16, 3), (700, 264, 128, 32, 4), (513, 320, 130, 20, 5), (1000, 128, 136, 8, 64), (530, 200, 72, 200, 2),
    (640, 96, 80, 100, 20), (520, 77, 40, 12, 3), (515, 40, 33, 7, 9),
    (400, 128, 96, 16, 120), (512, 64, 72, 8, 511), (65, 64, 64, 8, 30), (48, 160, 64, 32, 24), (900, 64, 50, 8, 30)])
def test_adapters(gpu, M, K, N, r, n, dtype):
    check(*case(M, K, N, r, n, DT[dtype]))


def test_no_scales_in_place_and_runs(gpu):
    y, x, a, b, ids, _ = case(200, 512, 640, 16, 3, torch.float16)
    ids = torch.sort(ids).values.contiguous()
    want = check(y, x, a, b, ids)
    # runs that end inside tiles of many tokens
    wide = case(900, 512, 640, 32, 5, torch.bfloat16)
    runs = torch.sort(wide[4]).values.contiguous()
    check(*wide[:4], runs, wide[5])
    y2 = y.clone()
    got = _C_ops.adapter_add(y2, x, a, b, ids, out=y2)
    assert got.data_ptr() == y2.data_ptr() and torch.equal(y2, want)


def test_uneven_use_of_the_stack(gpu):
    # most tokens on one adapter, the others' tokens on one each: more
    # adapters in a tile than on average; and one token between others
    for M, n in ((300, 90), (60, 40), (200, 3)):
        y, x, a, b, ids, s = case(M, 128, 136, 16, n, torch.float16)
        ids.fill_(n - 1)
        ids[:min(n, M // 2)] = torch.arange(min(n, M // 2), device="cuda", dtype=torch.int32)
        check(y, x, a, b, ids, s)
        ids.fill_(-1)
        ids[M // 2] = 1
        check(y, x, a, b, ids, s)


def test_adapters_outside_the_stack_add_nothing(gpu):
    y, x, a, b, ids, s = case(20, 256, 256, 16, 3, torch.bfloat16)
    for bad in (-1, 3, 2 ** 31 - 1, -2 ** 31):
        ids.fill_(bad)
        assert torch.equal(_C_ops.adapter_add(y, x, a, b, ids, s), y)
    for M in (20, 100, 300, 600):  # an empty stack
        y, x, _, _, ids, _ = case(M, 256, 256, 16, 3, torch.bfloat16)
        assert torch.equal(_C_ops.adapter_add(y, x, a[:0], b[:0], ids, s[:0]), y)
    assert _C_ops.adapter_add(y[:0], x[:0], a, b, ids[:0], s).shape == (0, 256)  # and no token


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_strided_and_unaligned(gpu, dtype):
    y, x, a, b, ids, s = case(50, 512, 768, 16, 4, DT[dtype])
    want = check(y, x, a, b, ids, s)
    wx = torch.zeros(50, 1025, dtype=x.dtype, device="cuda")
    wx[:, 1:513] = x
    wy = torch.zeros(50, 2000, dtype=x.dtype, device="cuda")
    wy[:, 3:771] = y
    out = torch.zeros(50, 801, dtype=x.dtype, device="cuda")
    got = _C_ops.adapter_add(wy[:, 3:771], wx[:, 1:513], a, b, ids, s, out=out[:, 5:773])
    check(wy[:, 3:771], wx[:, 1:513], a, b, ids, s, out=out[:, 5:773])
    assert bool((out[:, :5] == 0).all()) and bool((out[:, 773:] == 0).all())
    # the stacks at an odd element offset
    a2 = torch.empty(a.numel() + 1, dtype=a.dtype, device="cuda")[1:].view(a.shape).copy_(a)
    b2 = torch.empty(b.numel() + 1, dtype=b.dtype, device="cuda")[1:].view(b.shape).copy_(b)
    check(y, x, a2, b2, ids, s)


def test_large_and_small_values(gpu):
    # low-rank values past FP16's range, and far below its normal one
    for scale in (300.0, 1e-4):
        y, x, a, b, ids, s = case(20, 2048, 256, 16, 3, torch.float16)
        a = (a * (scale if scale > 1 else 1)).half()
        check(y, (x * scale).half(), a, (b * 1e-4 if scale > 1 else b).half(), ids, s)
    # one value of a row far larger than the others
    y, x, a, b, ids, s = case(20, 512, 256, 16, 3, torch.float16)
    a[:, 3] *= 100
    check(y, x, a, b, ids, s)


@pytest.mark.parametrize("M", [40, 600])
def test_infinities_and_nan_stay_in_their_tokens(gpu, M):
    y, x, a, b, ids, s = case(M, 512, 256, 16, 3, torch.float16)
    ids.fill_(1)
    want = _C_ops.adapter_add(y, x, a, b, ids, s)
    x[7, 3] = float("inf")
    x[9, 5] = float("nan")
    got = _C_ops.adapter_add(y, x, a, b, ids, s)
    keep = [m for m in range(M) if m not in (7, 9)]
    assert torch.equal(got[keep], want[keep])
    assert not bool(got[7].isfinite().any()) and bool(got[9].isnan().all())


@pytest.mark.parametrize("M,n", [(30, 3), (600, 3), (600, 9)])
def test_an_adapter_of_infinities_reaches_its_own_tokens_only(gpu, M, n):
    y, x, a, b, ids, s = case(M, 256, 264, 16, n, torch.float16)
    want = _C_ops.adapter_add(y, x, a, b, ids, s)
    a[1, 3, 5] = float("inf")
    b[2 % n, 7] = float("nan")
    got = _C_ops.adapter_add(y, x, a, b, ids, s)
    rest = (ids != 1) & (ids != 2)
    assert torch.equal(got[rest], want[rest])
    two = got[ids == 2]
    assert bool(two[:, 7].isnan().all()) and bool(two[:, :7].isfinite().all())
    assert not bool(got[ids == 1].isfinite().any())


def test_same_bits_every_time_other_streams_and_replays(gpu):
    y, x, a, b, ids, s = case(48, 4096, 1024, 32, 10, torch.bfloat16)
    want = check(y, x, a, b, ids, s)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        assert torch.equal(_C_ops.adapter_add(y, x, a, b, ids, s), want)
        with torch.cuda.stream(st):
            got = _C_ops.adapter_add(y, x, a, b, ids, s)
        st.synchronize()
        assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _C_ops.adapter_add(y, x, a, b, ids, s)
    for i in range(4):
        x.copy_(torch.randn(x.shape, device="cuda"))
        ids.copy_(torch.randint(-1, 10, (48,), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.clone(), _C_ops.adapter_add(y, x, a, b, ids, s)), i


def test_past_32_bit_offsets(gpu):
    # stacks of more than 2^31 elements, the last adapter used
    K, N, r = 16384, 512, 64
    n = (1 << 31) // (K * r) + 2
    a = torch.empty(n, r, K, dtype=torch.float16, device="cuda")
    b = torch.empty(n, N, r, dtype=torch.float16, device="cuda")
    a[-1].normal_(0, K ** -0.5)
    b[-1].normal_(0, 0.1)
    x, y = torch.randn(3, K, device="cuda").half(), torch.randn(3, N, device="cuda").half()
    ids = torch.full((3,), n - 1, dtype=torch.int32, device="cuda")
    got = _C_ops.adapter_add(y, x, a, b, ids)
    assert torch.equal(got, check(y, x, a[-1:].clone(), b[-1:].clone(), torch.zeros_like(ids)))


def test_refusals(gpu):
    y, x, a, b, ids, s = case(4, 64, 32, 8, 2, torch.float16)
    F = _C_ops.adapter_add
    for args, msg in [
            ((y, x.float(), a, b, ids), "float16 or bfloat16"), ((y, x.cpu(), a, b, ids), "GPU"),
            ((y, x.bfloat16(), a, b, ids), "one dtype"), ((y[:3], x, a, b, ids), "x and y"),
            ((y, x, a[:, :4], b, ids), "rank"), ((y, x, a, b.transpose(1, 2), ids), "rank"),
            ((y, x, a[:, :, ::2], b, ids), "rank"), ((y, x, a, b, ids.long()), "adapters"), ((y, x, a, b, ids[:2]), "adapters"),
            ((y, x, a, b, ids, s.half()), "scales"), ((y, x, a, b, ids, s[:1]), "scales"),
            ((y.t().contiguous().t(), x, a, b, ids), "rows of x and y")]:
        with pytest.raises(RuntimeError, match=msg):
            F(*args)
    with pytest.raises(RuntimeError, match="rank"):
        F(y, x, torch.zeros(1, 257, 64, dtype=x.dtype, device="cuda"), torch.zeros(1, 32, 257, dtype=x.dtype, device="cuda"), ids)
    with pytest.raises(RuntimeError, match="out"):
        F(y, x, a, b, ids, out=y[:, :16])
    with pytest.raises(RuntimeError, match="overlap"):
        F(y, x, a, b, ids, out=y[:1].expand(4, 32))


def test_ctypes_binding_gives_the_same(gpu, monkeypatch):
    args = case(20, 512, 256, 16, 3, torch.bfloat16)
    want = _C_ops.adapter_add(*args)
    monkeypatch.setattr(_lib, "torch_ops", lambda: None)
    assert torch.equal(_C_ops.adapter_add(*args), want)
    test_refusals(gpu)
