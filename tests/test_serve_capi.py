"""The serving entry points of the C ABI without a GPU: struct layouts as gcc
sees them, and the refusals of the host's checks (no pointer is followed)."""
import ctypes
import os
import subprocess

import pytest

from libortho_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"orth_hip_cache_t": _lib.OrthHipCache, "orth_hip_step_t": _lib.OrthHipStep,
           "orth_hip_append_t": _lib.OrthHipAppend, "orth_hip_attend_t": _lib.OrthHipAttend,
           "orth_hip_adapter_t": _lib.OrthHipAdapter}
INVALID, UNSUPPORTED = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libortho_amd.so not built (run __graft_entry__.build())")
    return _lib.lib()


def test_struct_layouts_match_the_header(tmp_path):
    lines, want = [], []
    for c, py in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(ctypes.sizeof(py))
        for f, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {f}));')
            want.append(getattr(py, f).offset)
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"orth_hip.h\"\nint main(void) {\n" +
                   "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == want


def cache(**kw):
    c = _lib.OrthHipCache(0x10000, 0x20000, _lib.DT_F16, 16, 2, 64, 8, (2048, 128, 64), (2048, 128, 64))
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def step(**kw):
    s = _lib.OrthHipStep(*[0x1000 * (i + 1) for i in range(11)], 4, 8, 8, 100, 6, 16, 0)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def append(**kw):
    a = _lib.OrthHipAppend(0x1000, 0x2000, 0x3000, 0x4000, (256, 64), (128, 64), (128, 64), (256, 64), 0x5000, 0x6000,
                           0x7000, 32, 5, 4, 64, 0, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attend(**kw):
    a = _lib.OrthHipAttend(0x1000, 0x2000, (256, 64), (256, 64), 0x3000, 0x4000, None, 5, 8, 8, 5, 4, 0, 0.125, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def adapter(**kw):
    a = _lib.OrthHipAdapter(0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, None, 64, 32, 32, 5, 64, 32, 3, 8, _lib.DT_F16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(L, rc, status, needle):
    assert rc == status, (rc, _lib.last_error())
    assert needle in _lib.last_error()


@pytest.mark.parametrize("kw,status,needle", [
    ({"requests": -1}, INVALID, "negative"), ({"tokens": -1}, INVALID, "negative"),
    ({"requests": 8193}, UNSUPPORTED, "8192"), ({"tokens": 1 << 31}, INVALID, "2^31"),
    ({"page_size": 0}, INVALID, "page_size"), ({"table_stride": 7}, INVALID, "table_stride"),
    ({"lengths": None}, INVALID, "lengths"), ({"pool": None}, INVALID, "pool"), ({"block_table": None}, INVALID, "block_table"),
    ({"free_pages": None}, INVALID, "free_pages"), ({"slots": None}, INVALID, "slots"),
    ({"lengths_out": 0x1000}, INVALID, "lengths_out"), ({"pool_out": 0x5000}, INVALID, "pool_out")])
def test_page_step_refusals(L, kw, status, needle):
    refused(L, L.orth_page_step_hip(ctypes.byref(step(**kw)), None), status, needle)


BAD_CACHES = [
    ({"dtype": _lib.DT_F32}, UNSUPPORTED, "F16 or BF16"), ({"page_size": 0}, INVALID, "page_size"),
    ({"kv_heads": 0}, INVALID, "kv_heads"), ({"head_dim": 60}, UNSUPPORTED, "head_dim"),
    ({"head_dim": 264}, UNSUPPORTED, "head_dim"), ({"pages": 0}, INVALID, "pages"), ({"k_cache": None}, INVALID, "NULL"),
    ({"v_cache": 0x20008}, INVALID, "16-byte"), ({"k_strides": (2048, 124, 64)}, INVALID, "multiples of 8"),
    ({"v_strides": (-2048, 128, 64)}, INVALID, "negative"), ({"k_strides": (1 << 60, 128, 64)}, INVALID, "too large")]


@pytest.mark.parametrize("kw,status,needle", BAD_CACHES)
def test_cache_refusals(L, kw, status, needle):
    refused(L, L.orth_paged_attention_hip(ctypes.byref(cache(**kw)), ctypes.byref(attend()), None), status, needle)
    refused(L, L.orth_cache_append_hip(ctypes.byref(cache(**kw)), ctypes.byref(append()), None), status, needle)


@pytest.mark.parametrize("kw,status,needle", [
    ({"tokens": -1}, INVALID, "tokens"), ({"rot": 63}, INVALID, "rot"), ({"rot": 66}, INVALID, "rot"),
    ({"cos_sin": None}, INVALID, "without cos_sin"), ({"positions": None}, INVALID, "positions"),
    ({"q_heads": 0}, INVALID, "q_heads"), ({"k": None}, INVALID, "NULL"), ({"q_out": None}, INVALID, "q_out"),
    ({"v": 0x3001}, INVALID, "aligned"), ({"k_strides": (-1, 64)}, INVALID, "stride of k"),
    ({"q_out": 0x1000, "q_out_strides": (512, 64)}, INVALID, "other strides"),
    ({"q_out_strides": (256, 32)}, INVALID, "overlap"), ({"q_out_strides": (128, 64)}, INVALID, "overlap"),
    ({"cos_sin_rows": -1}, INVALID, "cos_sin_rows")])
def test_append_refusals(L, kw, status, needle):
    refused(L, L.orth_cache_append_hip(ctypes.byref(cache()), ctypes.byref(append(**kw)), None), status, needle)


@pytest.mark.parametrize("kw,status,needle", [
    ({"tokens": -1}, INVALID, "tokens"), ({"q_heads": 3}, INVALID, "q_heads"), ({"q_heads": 0}, INVALID, "q_heads"),
    ({"window": -1}, INVALID, "window"), ({"scale": float("nan")}, INVALID, "scale"), ({"q": None}, INVALID, "NULL"),
    ({"block_table": None}, INVALID, "block_table"), ({"table_stride": 4}, INVALID, "table_stride"),
    ({"table_rows": 4}, INVALID, "more tokens"), ({"out_strides": (256, 0)}, INVALID, "overlap"),
    ({"tokens": 1 << 30, "table_rows": 1 << 30}, UNSUPPORTED, "q_heads")])
def test_attention_refusals(L, kw, status, needle):
    refused(L, L.orth_paged_attention_hip(ctypes.byref(cache()), ctypes.byref(attend(**kw)), None), status, needle)


def test_attention_refuses_tables_of_more_keys_than_its_numbers_hold(L):
    def call(width, page):
        return L.orth_paged_attention_hip(ctypes.byref(cache(page_size=page)),
                                          ctypes.byref(attend(table_width=width, table_stride=width)), None)
    refused(L, call(2, 1 << 30), UNSUPPORTED, "2^31 - 512")
    refused(L, call((1 << 31) - 1, (1 << 31) - 1), UNSUPPORTED, "2^31 - 512")
    refused(L, call((1 << 26) - 15, 32), UNSUPPORTED, "2^31 - 512")
    # the most it takes: no complaint about the table (a null query ends the call)
    a = attend(table_width=(1 << 26) - 16, table_stride=(1 << 26) - 16, q=None)
    refused(L, L.orth_paged_attention_hip(ctypes.byref(cache(page_size=32)), ctypes.byref(a), None), INVALID, "NULL")


@pytest.mark.parametrize("kw,status,needle", [
    ({"dtype": _lib.DT_F32}, UNSUPPORTED, "F16 or BF16"), ({"rank": 0}, UNSUPPORTED, "rank"),
    ({"rank": 257}, UNSUPPORTED, "rank"), ({"in_features": 0}, INVALID, "in_features"), ({"tokens": -1}, INVALID, "tokens"),
    ({"count": -1}, INVALID, "count"), ({"x": None}, INVALID, "NULL"), ({"a": None}, INVALID, "a or b"),
    ({"out_stride": 31}, INVALID, "overlap"), ({"out": 0x2000, "out_stride": 64}, INVALID, "another stride"),
    ({"x_stride": -64}, INVALID, "stride"), ({"b": 0x5001}, INVALID, "aligned"), ({"count": 1 << 31}, INVALID, "count")])
def test_adapter_refusals(L, kw, status, needle):
    refused(L, L.orth_adapter_add_hip(ctypes.byref(adapter(**kw)), None), status, needle)


def test_null_structs_and_valid_calls(L):
    assert L.orth_page_step_hip(None, None) == INVALID
    assert L.orth_paged_attention_hip(None, ctypes.byref(attend()), None) == INVALID
    assert L.orth_paged_attention_hip(ctypes.byref(cache()), None, None) == INVALID
    assert L.orth_cache_append_hip(ctypes.byref(cache()), None, None) == INVALID
    assert L.orth_adapter_add_hip(None, None) == INVALID
    # nothing to do: no device is asked for
    assert L.orth_cache_append_hip(ctypes.byref(cache()), ctypes.byref(append(tokens=0)), None) == _lib.OK
    assert L.orth_paged_attention_hip(ctypes.byref(cache()), ctypes.byref(attend(tokens=0)), None) == _lib.OK
    assert L.orth_adapter_add_hip(ctypes.byref(adapter(tokens=0)), None) == _lib.OK


def test_valid_arguments_reach_the_device_check(L):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the pointers here are made up")
    for rc in (L.orth_page_step_hip(ctypes.byref(step()), None),
               L.orth_cache_append_hip(ctypes.byref(cache()), ctypes.byref(append()), None),
               L.orth_paged_attention_hip(ctypes.byref(cache()), ctypes.byref(attend()), None),
               L.orth_adapter_add_hip(ctypes.byref(adapter()), None)):
        assert rc == _lib.ERR_NO_DEVICE
