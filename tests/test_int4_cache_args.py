"""int4_cache refuses, before it allocates, what every operator over such a
cache refuses, with their words (CPU: nothing is launched)."""
import pytest
import torch

from libortho_amd import _C_ops

REFUSED = [((4, 16, 2, 60), "head_dim must be a multiple of 8, at most 256"), ((4, 16, 2, 264), "head_dim must be"),
           ((4, 16, 2, 512), "head_dim must be"), ((4, 16, 2, 0), "head_dim must be"), ((4, 16, 2, -8), "head_dim must be"),
           ((4, 16, 2, 64, 16), "group_size must be head_dim, or 32, 64 or 128 where that divides it"),
           ((4, 16, 2, 64, 0), "group_size must be"), ((4, 16, 2, 64, -32), "group_size must be"),
           ((4, 16, 2, 64, 128), "group_size must be"), ((4, 16, 2, 96, 64), "group_size must be"),
           ((4, 16, 2, 80, 40), "group_size must be"), ((4, 16, 2, 256, 8), "group_size must be"),
           ((0, 16, 2, 64), "pages must be positive, at most 2\\^31 - 1"), ((-1, 16, 2, 64), "pages must be"),
           ((1 << 31, 16, 2, 64), "pages must be"), ((4, 0, 2, 64), "page_size must be positive"), ((4, 16, 0, 64), "kv_heads must be positive"),
           ((4, 1 << 31, 2, 64), "page_size or kv_heads is too large"), ((4, 16, 1 << 31, 64), "page_size or kv_heads is too large")]


@pytest.mark.parametrize("args,message", REFUSED)
def test_int4_cache_refuses_before_it_allocates(monkeypatch, args, message):
    def allocated(*a, **kw):
        raise AssertionError("allocated")
    monkeypatch.setattr(torch, "zeros", allocated)
    with pytest.raises(RuntimeError, match=message):
        _C_ops.int4_cache(*args, device="cpu")


@pytest.mark.parametrize("D,group", [(8, None), (8, 8), (40, 40), (64, None), (64, 32), (96, 32), (96, 96), (96, None), (128, 128),
                                     (160, 32), (192, 64), (200, None), (256, 128), (256, 256)])
def test_int4_cache_gives_what_operators_take(D, group):
    k_codes, k_scales, v_codes, v_scales = _C_ops.int4_cache(3, 5, 2, D, group, device="cpu")
    held = group or (64 if D % 64 == 0 else D)
    for codes, scales in ((k_codes, k_scales), (v_codes, v_scales)):
        assert codes.shape == (3, 5, 2, _C_ops._int4_row_bytes(D)) and codes.dtype == torch.uint8 and not codes.any()
        assert scales.shape == (3, 5, 2, D // held, 2) and scales.dtype == torch.float16 and not scales.any()
