"""What the serving operators refuse, or keep apart, beyond shapes and types."""
import pytest
import torch

from libortho_amd import _C_ops, _lib

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def half(*shape):
    return torch.randn(*shape, device="cuda").half()


def attend_args():
    return dict(q=half(2, 4, 64), k_cache=half(4, 16, 2, 64), v_cache=half(4, 16, 2, 64),
                block_table=i32([[0, 1], [2, 3]]), positions=i32([20, 31]))


def append_args():
    return dict(k=half(2, 2, 64), v=half(2, 2, 64), k_cache=half(4, 16, 2, 64), v_cache=half(4, 16, 2, 64),
                slots=torch.tensor([3, 40], device="cuda"), q=half(2, 4, 64), positions=i32([5, 6]),
                cos_sin=torch.randn(9, 64, device="cuda"))


def adapter_args():
    return dict(y=half(3, 32), x=half(3, 64), a=half(2, 8, 64), b=half(2, 32, 8), adapters=i32([0, 1, -1]),
                scales=torch.rand(2, device="cuda"))


@pytest.mark.parametrize("binding", ["compiled", "ctypes"])
@pytest.mark.parametrize("name,args,takes", [
    ("paged_attention", attend_args, ["q", "k_cache", "v_cache", "out"]),
    ("cache_append", append_args, ["k", "v", "k_cache", "v_cache", "q", "cos_sin", "q_out"]),
    ("adapter_add", adapter_args, ["y", "x", "a", "b", "scales", "out"])])
def test_no_gradient_is_lost_without_a_word(gpu, monkeypatch, binding, name, args, takes):
    if binding == "ctypes":
        monkeypatch.setattr(_lib, "torch_ops", lambda: None)
    f = getattr(_C_ops, name)
    for t in takes:
        kw = args()
        if t in ("out", "q_out"):
            kw[t] = torch.empty_like(kw["y"] if name == "adapter_add" else kw["q"])
        kw[t].requires_grad_()
        with pytest.raises(RuntimeError, match=f"{name} has no gradient.*{t} "):
            f(**kw)
        with torch.no_grad():
            got = f(**kw)
        assert got is not None and not (got.requires_grad and t not in ("out", "q_out"))
        kw[t] = kw[t].detach()
        f(**kw)


def test_append_of_more_heads_than_a_grid_has_rows(gpu):
    # unaligned vectors of 256: two heads a workgroup
    H, D = 140000, 256
    flat = torch.randn(H * D + 1, device="cuda").half()[1:].view(1, H, D)
    kc, vc = (torch.zeros(1, 1, 1, D, dtype=torch.float16, device="cuda") for _ in range(2))
    k, cs = half(1, 1, D), torch.ones(1, D, device="cuda")
    cs[:, D // 2:] = 0
    out = _C_ops.cache_append(k, k, kc, vc, torch.zeros(1, dtype=torch.int64, device="cuda"), q=flat, positions=i32([0]), cos_sin=cs)
    assert torch.equal(out, flat) and torch.equal(kc[0], k) and torch.equal(vc[0], k)


def test_append_of_more_tokens_than_one_grid_holds(gpu):
    # 2^24 workgroups of 256 threads are 2^32 threads, more than a launch takes
    T, D, P, pages = (1 << 24) + 77, 8, 16, 8
    k = torch.zeros(T, 1, D, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    slots = torch.full((T,), -1, dtype=torch.int64, device="cuda")
    at = [0, 5, (1 << 23) - 1, 1 << 23, (1 << 23) + 9, (1 << 24) - 1, 1 << 24, T - 1]
    for i, t in enumerate(at):
        k[t], v[t], slots[t] = i + 1, -i - 1, 7 * i + 3
    kc, vc = (torch.zeros(pages, P, 1, D, dtype=torch.float16, device="cuda") for _ in range(2))
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    pos[1 << 24] = 1
    q = torch.ones(T, 1, D, dtype=torch.float16, device="cuda")
    cs = torch.tensor([[1.0] * 4 + [0.0] * 4, [0.0] * 4 + [1.0] * 4], device="cuda")  # none, and a quarter turn
    out = _C_ops.cache_append(k, v, kc, vc, slots, q=q, positions=pos, cos_sin=cs)
    want = torch.zeros_like(kc).flatten(0, 1)
    for i, t in enumerate(at):
        want[7 * i + 3] = i + 1
    assert torch.equal(vc.flatten(0, 1), -want)
    turned = want[7 * at.index(1 << 24) + 3, 0]
    turned[:4] *= -1
    assert torch.equal(kc.flatten(0, 1), want)
    q[1 << 24, 0, :4] = -1
    assert torch.equal(out, q)


def test_adapters_of_more_tokens_than_one_grid_holds(gpu):
    M, K, N, r = (1 << 28) + 77, 8, 8, 1
    x = torch.ones(M, K, dtype=torch.float16, device="cuda")
    y = torch.zeros(M, N, dtype=torch.float16, device="cuda")
    ids = torch.full((M,), -1, dtype=torch.int32, device="cuda")
    at = [0, 63, (1 << 24) - 1, 1 << 24, (1 << 26) + 9, (1 << 28) - 1, 1 << 28, M - 1]
    for t in at:
        ids[t] = t % 2
    a = torch.ones(2, r, K, dtype=torch.float16, device="cuda")
    b = torch.ones(2, N, r, dtype=torch.float16, device="cuda")
    b[1] = 2.0
    got = _C_ops.adapter_add(y, x, a, b, ids, out=y)
    for t in at:
        assert got[t].tolist() == [8.0 * (1 + t % 2)] * N, t
        got[t] = 0
    assert not bool(got.any())


def test_what_a_server_keeps_between_steps_does_not_hold_the_step(gpu):
    n, T = 2, 70000
    z = torch.zeros(n, dtype=torch.int32, device="cuda")
    lengths, pool, *_ = _C_ops.page_step(z, i32([T - 1, 1]), torch.zeros(n, 5000, dtype=torch.int32, device="cuda"),
                                         torch.arange(8000, dtype=torch.int32, device="cuda"), i32([0, 0]), 16, T)
    assert lengths.tolist() == [T - 1, 1] and pool.tolist() == [-(-(T - 1) // 16) + 1, 0]
    assert lengths.untyped_storage().nbytes() <= 64 and pool.untyped_storage().nbytes() <= 64
