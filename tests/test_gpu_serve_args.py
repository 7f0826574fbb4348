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
