"""The host side of the entry points over a cache in 4 bits, without a GPU:
argument checks under AddressSanitizer and UBSan (on the host pass only,
-Xarch_host), driven through the edges of every field by
tests/sanitize/int4_driver.c; and threads that call at the same time, over
stand-ins for the GPU (tests/sanitize/int4_threads_driver.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SAN = os.path.join(ROOT, "tests", "sanitize")
CSRC = os.path.join(ROOT, "libortho_amd", "csrc")
INCLUDE = os.path.join(ROOT, "include")


def run(cmd, **kw):
    r = subprocess.run(cmd, capture_output=True, text=True, **kw)
    assert r.returncode == 0, f"{' '.join(cmd)}\n{r.stdout}\n{r.stderr}"
    return r


@pytest.fixture
def hipcc():
    found = "/opt/rocm/bin/hipcc" if os.path.exists("/opt/rocm/bin/hipcc") else shutil.which("hipcc")
    if not found:
        pytest.skip("hipcc not found")
    return found


def compiled(hipcc, tmp_path, sources):
    objs = []
    for src, more in sources:
        obj = str(tmp_path / (os.path.basename(src) + ".o"))
        run([hipcc, "--offload-arch=gfx950", "-O1", "-g", "-fPIC", "-std=c++17", "-Xclang", "-target-feature",
             "-Xclang", "-packed-fp32-ops", *more, "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj])
        objs.append(obj)
    return objs


def linked(hipcc, tmp_path, objs, *more):
    exe = str(tmp_path / "exe")
    rocm_lib = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(hipcc))), "lib")
    run(["g++", *more, *objs, "-o", exe, "-L", rocm_lib, f"-Wl,-rpath,{rocm_lib}", "-lamdhip64", "-lpthread"])
    return exe


def test_int4_host_side_under_asan_ubsan(hipcc, tmp_path):
    san = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
           "-Xarch_host", "-fno-sanitize-recover=all", "-Xarch_host", "-fno-omit-frame-pointer"]
    objs = compiled(hipcc, tmp_path, [(src, san) for src in (
        os.path.join(CSRC, "orth_capi.hip"), os.path.join(CSRC, "orth_serve4.hip"),
        os.path.join(SAN, "capi_stubs.hip"), os.path.join(SAN, "int4_stubs.hip"))])
    drv = str(tmp_path / "int4_driver.o")
    run(["gcc", "-O1", "-g", "-std=c11", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
         "-I", INCLUDE, "-c", os.path.join(SAN, "int4_driver.c"), "-o", drv])
    exe = linked(hipcc, tmp_path, [drv, *objs], "-fsanitize=address,undefined")
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=1", HIP_VISIBLE_DEVICES="-1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1", ROCR_VISIBLE_DEVICES="-1")
    assert "int4 ok" in run([exe], env=env, timeout=300).stdout


def test_int4_attention_of_several_threads_keeps_its_workspaces(hipcc, tmp_path):
    # (the split-K launcher of capi_stubs.hip gives way to the recording one)
    other = [f"-D{n}=other_{n}" for n in ("skinny_supported", "skinny_workspace_bytes", "launch_skinny")]
    objs = compiled(hipcc, tmp_path, [
        (os.path.join(CSRC, "orth_capi.hip"), []), (os.path.join(CSRC, "orth_serve.hip"), []),
        (os.path.join(CSRC, "orth_serve4.hip"), []), (os.path.join(SAN, "capi_stubs.hip"), other),
        (os.path.join(SAN, "threads_stubs.hip"), []), (os.path.join(SAN, "int4_threads_stubs.hip"), []),
        (os.path.join(SAN, "int4_threads_driver.cpp"), ["-D__HIP_PLATFORM_AMD__"])])
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    assert "threads ok" in run([linked(hipcc, tmp_path, objs)], env=env, timeout=120).stdout
