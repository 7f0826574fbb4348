"""More refusals of the serving entry points' host checks, without a GPU."""
import ctypes

import pytest

from libortho_amd import _lib
from test_serve_capi import UNSUPPORTED, L, append, cache, refused  # noqa: F401 (L: fixture)


@pytest.mark.parametrize("c,a", [({}, {"q_heads": 1 << 30}), ({"kv_heads": 1 << 30}, {})])
def test_append_refuses_more_heads_than_it_counts(L, c, a):  # noqa: F811
    args = append(q_strides=(1 << 40, 64), q_out_strides=(1 << 40, 64), k_strides=(1 << 40, 64), v_strides=(1 << 40, 64), **a)
    args.tokens = 1
    held = cache(k_strides=(1 << 40, 1 << 36, 64), v_strides=(1 << 40, 1 << 36, 64), **c)
    held.pages, held.page_size = 1, 1
    refused(L, L.orth_cache_append_hip(ctypes.byref(held), ctypes.byref(args), None), UNSUPPORTED, "2^30")
