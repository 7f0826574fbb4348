"""Host threads that call on one stream at the same time (no GPU): the host
side of the C ABI over stand-ins for the GPU (tests/sanitize/threads_stubs.hip)
that record which launches were inside together."""
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


def test_calls_of_several_threads_keep_their_workspaces(tmp_path):
    hipcc = "/opt/rocm/bin/hipcc" if os.path.exists("/opt/rocm/bin/hipcc") else shutil.which("hipcc")
    if not hipcc:
        pytest.skip("hipcc not found")
    csrc = os.path.join(ROOT, "libortho_amd", "csrc")
    flags = [hipcc, "--offload-arch=gfx950", "-O1", "-g", "-fPIC", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
             "-packed-fp32-ops", "-I", os.path.join(ROOT, "include"), "-I", csrc]
    # (the split-K launcher of capi_stubs.hip gives way to the recording one)
    other = [f"-D{n}=other_{n}" for n in ("skinny_supported", "skinny_workspace_bytes", "launch_skinny")]
    objs = []
    for src, more in ((os.path.join(csrc, "orth_capi.hip"), []), (os.path.join(csrc, "orth_serve.hip"), []),
                      (os.path.join(SAN, "capi_stubs.hip"), other), (os.path.join(SAN, "threads_stubs.hip"), []),
                      (os.path.join(SAN, "threads_driver.cpp"), ["-D__HIP_PLATFORM_AMD__"])):
        obj = str(tmp_path / (os.path.basename(src) + ".o"))
        run([*flags, *more, "-c", src, "-o", obj])
        objs.append(obj)
    exe = str(tmp_path / "threads")
    rocm_lib = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(hipcc))), "lib")
    run(["g++", *objs, "-o", exe, "-L", rocm_lib, f"-Wl,-rpath,{rocm_lib}", "-lamdhip64", "-lpthread"])
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    assert "threads ok" in run([exe], env=env, timeout=120).stdout
