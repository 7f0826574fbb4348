"""The entry points over the cache in 4 bits without a GPU: struct layouts as
gcc sees them, the host's refusals (no pointer is followed), and the oracle of
the format against its definition."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from libortho_amd import _C_ops, _lib
from oracle import cache_oracle as O
from test_serve_capi import INVALID, L, UNSUPPORTED, append, attend, refused  # noqa: F401 (L: a fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_header(tmp_path):
    lines, want = [], []
    for c, py in {"orth_hip_int4_cache_t": _lib.OrthHipInt4Cache, "orth_hip_read_t": _lib.OrthHipRead}.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(ctypes.sizeof(py))
        for f, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {f}));')
            want.append(getattr(py, f).offset)
    dims = list(range(8, 257, 8))
    lines += [f'printf("%d\\n", ORTH_INT4_ROW_BYTES({d}));' for d in dims]
    want += [O.row_bytes(d) for d in dims]
    assert [_C_ops._int4_row_bytes(d) for d in dims] == [O.row_bytes(d) for d in dims]
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"orth_hip.h\"\nint main(void) {\n" +
                   "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == want


def cache(**kw):
    c = _lib.OrthHipInt4Cache(0x10000, 0x20000, 0x30000, 0x40000, 16, 2, 64, 32, 8, (1024, 64, 32), (1024, 64, 32),
                              (128, 8, 4), (128, 8, 4))
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def read(**kw):
    r = _lib.OrthHipRead(0x1000, 0x2000, (128, 64), (128, 64), 0x3000, 5)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def calls(L, c=None, a=None, t=None, r=None, dtype=_lib.DT_F16):
    ref = lambda x: ctypes.byref(x) if x is not None else None
    c = ref(c)
    return (lambda: L.orth_cache_append_int4_hip(c, ref(a or append()), dtype, None),
            lambda: L.orth_cache_read_int4_hip(c, ref(r or read()), dtype, None),
            lambda: L.orth_paged_attention_int4_hip(c, ref(t or attend()), dtype, None))


@pytest.mark.parametrize("kw,status,needle", [
    ({"page_size": 0}, INVALID, "page_size"), ({"kv_heads": 0}, INVALID, "kv_heads"), ({"head_dim": 60}, UNSUPPORTED, "head_dim"),
    ({"head_dim": 264}, UNSUPPORTED, "head_dim"), ({"head_dim": 0}, UNSUPPORTED, "head_dim"), ({"pages": 0}, INVALID, "pages"),
    ({"pages": 1 << 31}, INVALID, "pages"), ({"group_size": 16}, UNSUPPORTED, "group_size"), ({"group_size": 0}, UNSUPPORTED, "group_size"),
    ({"group_size": -32}, UNSUPPORTED, "group_size"), ({"group_size": 128}, UNSUPPORTED, "group_size"),
    ({"head_dim": 96, "group_size": 64}, UNSUPPORTED, "group_size"), ({"k_codes": None}, INVALID, "NULL"),
    ({"v_scales": None}, INVALID, "NULL"), ({"v_codes": 0x20008}, INVALID, "16-byte"), ({"k_scales": 0x30002}, INVALID, "4-byte"),
    ({"k_code_strides": (1024, 56, 32)}, INVALID, "multiples of 16"), ({"v_scale_strides": (128, 7, 4)}, INVALID, "even"),
    ({"v_code_strides": (-1024, 64, 32)}, INVALID, "negative"), ({"k_scale_strides": (1 << 60, 8, 4)}, INVALID, "too large")])
def test_cache_refusals(L, kw, status, needle):  # noqa: F811
    for call in calls(L, cache(**kw)):
        refused(L, call(), status, needle)


def test_dtype_and_null_refusals(L):  # noqa: F811
    for call in calls(L, cache(), dtype=_lib.DT_F32):
        refused(L, call(), UNSUPPORTED, "dtype")
    for call in calls(L, None):
        refused(L, call(), INVALID, "cache is NULL")
    for f in (L.orth_cache_append_int4_hip, L.orth_cache_read_int4_hip, L.orth_paged_attention_int4_hip):
        refused(L, f(ctypes.byref(cache()), None, _lib.DT_F16, None), INVALID, "NULL")


@pytest.mark.parametrize("kw,needle", [
    ({"count": -1}, "count"), ({"count": 1 << 31}, "count"), ({"k_out": None}, "NULL"), ({"slots": None}, "NULL"),
    ({"v_out": 0x2001}, "aligned"), ({"k_strides": (-1, 64)}, "stride of k_out"), ({"v_strides": (1 << 60, 64)}, "stride of v_out"),
    ({"v_strides": (128, 32)}, "overlap"), ({"k_strides": (64, 64)}, "overlap")])
def test_read_refusals(L, kw, needle):  # noqa: F811
    refused(L, calls(L, cache(), r=read(**kw))[1](), INVALID, needle)


@pytest.mark.parametrize("kw,status,needle", [
    ({"tokens": -1}, INVALID, "tokens"), ({"rot": 66}, INVALID, "rot"), ({"cos_sin": None}, INVALID, "without cos_sin"),
    ({"k": None}, INVALID, "NULL"), ({"q_out": 0x1000, "q_out_strides": (512, 64)}, INVALID, "other strides"),
    ({"q_out_strides": (128, 64)}, INVALID, "overlap"), ({"q_heads": (1 << 30) - 3}, UNSUPPORTED, "2^30")])
def test_append_refusals(L, kw, status, needle):  # noqa: F811
    refused(L, calls(L, cache(), a=append(**kw))[0](), status, needle)


@pytest.mark.parametrize("kw,status,needle", [
    ({"tokens": -1}, INVALID, "tokens"), ({"q_heads": 3}, INVALID, "q_heads"), ({"window": -1}, INVALID, "window"),
    ({"scale": float("nan")}, INVALID, "scale"), ({"table_stride": 4}, INVALID, "table_stride"),
    ({"table_rows": 4}, INVALID, "more tokens"), ({"out_strides": (256, 0)}, INVALID, "overlap"),
    ({"table_width": 1 << 28, "table_stride": 1 << 28}, UNSUPPORTED, "2^31 - 512")])
def test_attention_refusals(L, kw, status, needle):  # noqa: F811
    refused(L, calls(L, cache(), t=attend(**kw))[2](), status, needle)


def test_nothing_to_do_and_valid_arguments(L):  # noqa: F811
    import torch
    for call in calls(L, cache(), a=append(tokens=0), t=attend(tokens=0), r=read(count=0)):
        assert call() == _lib.OK
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the pointers here are made up")
    for kw in ({}, {"group_size": 64}, {"head_dim": 256, "group_size": 128}, {"head_dim": 160}, {"head_dim": 40, "group_size": 40}):
        a = append(rot=16, q_strides=(1024, 256), q_out_strides=(1024, 256), k_strides=(512, 256), v_strides=(512, 256))
        t = attend(q_strides=(1024, 256), out_strides=(1024, 256))
        r = read(k_strides=(512, 256), v_strides=(512, 256))
        for call in calls(L, cache(**kw), a, t, r):
            assert call() == _lib.ERR_NO_DEVICE, _lib.last_error()


# ---------------------------------------------------------------- the format

@pytest.mark.parametrize("D,group", [(128, 32), (128, 128), (80, 80), (96, 32), (8, 8), (256, 64), (200, 200)])
def test_the_format_keeps_values_within_half_a_step(D, group):
    rng = np.random.default_rng(D)
    x = O.to_fp16(rng.standard_normal((50, D)) * 10.0 ** rng.uniform(-3, 3, (50, 1)))
    u, s, low = O.quantise(x, group)
    assert np.array_equal(O.unpack(O.pack(u), D), u) and O.pack(u).shape == (50, O.row_bytes(D))
    got = O.values(O.pack(u), np.stack([s, low], -1), D)
    step = np.repeat(s.astype(np.float64), group, -1)
    # half a step, and at the top what 15 roundings of the scale leave (2^-11 of it each, or 2^-25)
    assert (np.abs(got - x) <= step * (0.5 + 15 * 2.0 ** -11) + 15 * 2.0 ** -25).all()
    assert np.array_equal(got.reshape(50, -1, group).min(-1), x.reshape(50, -1, group).min(-1))


def test_the_format_at_its_edges():
    for row in ([-65504, 65504], [65504, 65472], [0, 0], [-65504, -65504], [2.0 ** -24, 0]):
        u, s, low = O.quantise(np.array([row * 4], np.float64), 8)
        v = O.values(O.pack(u), np.stack([s, low], -1), 8)
        assert np.isfinite(v).all() and (np.abs(v) <= 65504).all()
    u, s, low = O.quantise(np.array([[0, 15, 7.5, 7.25, 0.5, 14.5, 0.25, 3.0]]), 8)
    assert u.tolist() == [[0, 15, 8, 7, 1, 15, 0, 3]] and s[0, 0] == 1 and low[0, 0] == 0
    u, s, low = O.quantise(np.array([[1e9, -1e9, 0, 0, 0, 0, 0, np.inf]]), 8)
    assert np.isnan(s).all() and np.isnan(low).all() and not u.any()
