"""The cache in 4 bits through views that documents allow and the attention's
fast loads do not take: keys and values of unlike strides, and strides that
pass 32 bits.  References and tolerances are those of test_gpu_int4.py; what
views hold is compared whole."""
import numpy as np
import pytest
import torch

from libortho_amd import _C_ops
from test_gpu_int4 import LENS, append_inputs, attend_case, attend_check, check_read, check_written, i32, np64, random_cache

pytestmark = pytest.mark.gpu


def spread(t, before, behind):
    """t's contents as a view of a tensor with other slots' bytes before and behind each of its slots."""
    wide = torch.randint(0, 100, (*t.shape[:2], before + t.shape[2] + behind, *t.shape[3:]), device="cuda").to(t.dtype)
    view = wide[:, :, before:before + t.shape[2]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,group", [(128, 64), (64, 64), (96, 32), (256, 64), (80, 80)])
@pytest.mark.parametrize("which", [(2,), (3,), (0, 1), (0, 3)])
def test_attention_over_keys_and_values_of_unlike_strides(gpu, D, group, which, dtype):
    q, cache, table, pos = attend_case(LENS, 4, 2, D, group, 16, dtype)
    views = [spread(t, 1, i) if i in which else t for i, t in enumerate(cache)]
    got = attend_check(q, views, table, pos)
    if D <= 128:  # (the same cut of the work: the same sums)
        assert torch.equal(got, _C_ops.paged_attention_int4(q, *cache, table, pos))
    rows = i32([r for r in range(len(LENS) - 1) for _ in range(3)])
    q = torch.randn(len(rows), 4, D, device="cuda").to(dtype)
    attend_check(q, views, table, i32([max(LENS[r] - 3, -1) + i if LENS[r] else -1 for r in range(len(LENS) - 1) for i in range(3)]), rows=rows)


@pytest.mark.parametrize("which", [(2,), (1, 3), (0, 1)])
def test_append_and_read_through_unlike_strides(gpu, which):
    q, k, v, cache, slots = append_inputs(21, 4, 2, 128, 32, 16, torch.float16)
    views = [spread(t, 1, i) if i in which else t for i, t in enumerate(cache)]
    before = [t.clone() for t in views]
    assert _C_ops.cache_append_int4(k, v, *views, slots) is None
    check_written(views, before, slots, np64(k), np64(v), 32)
    check_read(views, torch.arange(-1, views[0].shape[0] * 16 + 1, device="cuda"), 128, torch.float16)


@pytest.mark.parametrize("big", ["codes", "scales", "both"])
def test_pages_that_lie_2_to_the_31_bytes_apart(gpu, big):
    P, G, D, group, pages = 16, 2, 128, 64, 3
    small = random_cache(torch.Generator(device="cuda").manual_seed(5), pages, P, G, D, group)

    def apart(t, on):
        if not on:
            return t
        stride = (1 << 31) // t.element_size() + 16
        flat = torch.empty((pages - 1) * stride + t[0].numel(), dtype=t.dtype, device="cuda")
        view = flat.as_strided(t.shape, (stride, *t.stride()[1:]))
        view.copy_(t)
        return view

    cache = [apart(t, big in ("both", "codes" if i % 2 == 0 else "scales")) for i, t in enumerate(small)]
    table, q = i32([[2, 0, 1]]), torch.randn(1, 8, D, device="cuda").half()
    got = _C_ops.paged_attention_int4(q, *cache, table, i32([44]))
    assert torch.equal(got, attend_check(q, small, table, i32([44])))
    k = torch.randn(4, G, D, device="cuda").half()
    slots = torch.tensor([0, 17, 47, 33], device="cuda")
    for c in (cache, small):
        _C_ops.cache_append_int4(k, -k, *c, slots)
    for a, b in zip(cache, small):
        assert np.array_equal(a.cpu().numpy(), b.cpu().numpy())
    everything = torch.arange(pages * P, device="cuda")
    for a, b in zip(_C_ops.cache_read_int4(*cache, everything, D), _C_ops.cache_read_int4(*small, everything, D)):
        assert torch.equal(a, b)
