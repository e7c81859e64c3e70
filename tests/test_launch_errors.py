"""The status of a launch that fails, without a device: a HIP runtime of a few lines stands in for the real one in a
child process, and one of its launches reports an error."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIP = "/opt/rocm/include"

RUNTIME = r"""
#include <hip/hip_runtime_api.h>
#include <string.h>
static int left = -1, error = 0;  // launches until one fails, and how
extern "C" {
void fail_launch(int after, int e) { left = after; error = e; }
hipError_t hipGetLastError(void) { return left >= 0 && left-- == 0 ? (hipError_t)error : hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "an error"; }
hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
  memset(p, 0, sizeof *p);
  strcpy(p->gcnArchName, "gfx950");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetSymbolAddress(void** p, const void*) { *p = (void*)0x1000; return hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { *s = (hipStream_t)0x1000; return hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t) { *p = (void*)0x1000; return hipSuccess; }
hipError_t hipFree(void*) { return hipSuccess; }
hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3*, dim3*, size_t*, hipStream_t*) { return hipSuccess; }
void** __hipRegisterFatBinary(const void*) { static void* x; return &x; }
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*, void*, int*) {}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
void __hipUnregisterFatBinary(void**) {}
}
"""

CALLS = r"""
import ctypes, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path[:0] = [sys.argv[2], sys.argv[2] + "/tests"]
import __graft_entry__ as e
pkg = e.load_package()
import test_pages as t
lib, ctx = pkg.lib(), pkg.Context(0)
w, ptr = t._window(pkg), ctypes.byref
a = pkg.PagedAttentionDesc(**{n: getattr(w, n) for n, _ in pkg.PagedAttentionDesc._fields_})
big = t._planes(pkg, *[4096] * 129)  # two launches
calls = dict(attention=(lib.qa_attention_paged, a, 1), window=(lib.qa_attention_paged_window, w, 1),
             copy=(lib.qa_pages_copy, t._copy(pkg, nplanes=129, src=big, dst=big), 2), fork=(lib.qa_pages_fork, t._fork(pkg), 2),
             compact=(lib.qa_pages_compact, t._compact(pkg), 2), beam=(lib.qa_beam_select, t._beam(pkg), 1))
for name, (fn, d, launches) in calls.items():
    for at in range(launches + 1):
        for error in (2, 719):  # out of memory, a failed launch
            stub.fail_launch(at, error)
            rc = fn(ctx.handle, ptr(d))
            print(name, at, error, rc, pkg.last_error().split(":")[0].replace(" ", "_") if rc else "-")
"""


@pytest.fixture(scope="module")
def lines(pkg, tmp_path_factory):
    if not shutil.which("g++") or not os.path.exists(os.path.join(HIP, "hip", "hip_runtime_api.h")):
        pytest.skip("g++ or the HIP headers are not there")
    d = tmp_path_factory.mktemp("hip")
    src, so = d / "hip.cpp", d / "hip.so"
    src.write_text(RUNTIME)
    subprocess.run(["g++", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I", HIP, str(src), "-o", str(so)], check=True)
    run = subprocess.run([sys.executable, "-c", CALLS, str(so), ROOT], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    return [x.split() for x in run.stdout.splitlines()]


@pytest.mark.parametrize("name,launches", [("attention", 1), ("window", 1), ("copy", 2), ("fork", 2), ("compact", 2), ("beam", 1)])
def test_a_failed_launch(pkg, lines, name, launches):
    """Out of memory is QA_ENOMEM, whichever launch of the call it is, anything else QA_EDEVICE; behind the last all is well."""
    got = {(int(at), int(e)): (int(rc), text) for n, at, e, rc, text in lines if n == name}
    assert len(got) == 2 * (launches + 1)
    fn = {"attention": "qa_attention_paged", "window": "qa_attention_paged_window", "beam": "qa_beam_select"}.get(name, "qa_pages_" + name)
    for at in range(launches):
        assert got[at, 2] == (pkg.QA_ENOMEM, fn + "_launch"), (at, got)
        assert got[at, 719] == (pkg.QA_EDEVICE, fn + "_launch"), (at, got)
    assert got[launches, 2][0] == got[launches, 719][0] == 0
