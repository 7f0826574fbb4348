"""The serving entry points' host side under AddressSanitizer and UBSan (no
GPU): argument checks up to the device check, driven through the edges of
every field by tests/sanitize/serve_driver.c.  The sanitizers are on the host
pass only (-Xarch_host)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SAN = os.path.join(ROOT, "tests", "sanitize")


def run(cmd, **kw):
    r = subprocess.run(cmd, capture_output=True, text=True, **kw)
    assert r.returncode == 0, f"{' '.join(cmd)}\n{r.stdout}\n{r.stderr}"
    return r


def test_serving_host_side_under_asan_ubsan(tmp_path):
    hipcc = "/opt/rocm/bin/hipcc" if os.path.exists("/opt/rocm/bin/hipcc") else shutil.which("hipcc")
    if not hipcc:
        pytest.skip("hipcc not found")
    csrc = os.path.join(ROOT, "libortho_amd", "csrc")
    inc = ["-I", os.path.join(ROOT, "include"), "-I", csrc]
    san = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
           "-Xarch_host", "-fno-sanitize-recover=all", "-Xarch_host", "-fno-omit-frame-pointer"]
    objs = []
    for src in (os.path.join(csrc, "orth_capi.hip"), os.path.join(csrc, "orth_serve.hip"),
                os.path.join(SAN, "capi_stubs.hip"), os.path.join(SAN, "serve_stubs.hip")):
        obj = str(tmp_path / (os.path.basename(src) + ".o"))
        run([hipcc, "--offload-arch=gfx950", "-O1", "-g", "-fPIC", "-std=c++17", "-Xclang", "-target-feature",
             "-Xclang", "-packed-fp32-ops", *san, *inc, "-c", src, "-o", obj])
        objs.append(obj)
    drv = str(tmp_path / "serve_driver.o")
    run(["gcc", "-O1", "-g", "-std=c11", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
         "-I", os.path.join(ROOT, "include"), "-c", os.path.join(SAN, "serve_driver.c"), "-o", drv])
    exe = str(tmp_path / "serve_san")
    rocm_lib = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(hipcc))), "lib")
    run(["g++", "-fsanitize=address,undefined", drv, *objs, "-o", exe, "-L", rocm_lib,
         f"-Wl,-rpath,{rocm_lib}", "-lamdhip64", "-lpthread"])
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=1", HIP_VISIBLE_DEVICES="-1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1", ROCR_VISIBLE_DEVICES="-1")
    assert "serve ok" in run([exe], env=env, timeout=300).stdout
