"""What the attention entry asks of the HIP runtime before its launches, on the CPU: the
library runs in a process of its own against a stand-in for the runtime's launch functions
that records them and launches nothing."""
import json
import os
import shutil
import subprocess
import sys
from importlib import import_module

import pytest

STAND_IN = r"""
#define __HIP_PLATFORM_AMD__
#include <hip/hip_runtime_api.h>
#include <cstdio>
#include <cstring>
#include <map>
#include <string>

namespace {
struct Config { dim3 grid, block; size_t lds; hipStream_t stream; } config;
std::map<const void*, int> limit, names;
std::string text;
}

extern "C" {
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipGetDeviceProperties(hipDeviceProp_t* p, int) {
    memset(p, 0, sizeof *p);
    strcpy(p->gcnArchName, "gfx950");
    return hipSuccess;
}
hipError_t hipGetSymbolAddress(void** p, const void*) {
    static char memory[256];
    *p = memory;
    return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "none"; }
hipError_t hipFuncSetAttribute(const void* f, hipFuncAttribute, int v) {
    limit[f] = v;
    return hipSuccess;
}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t s) {
    config = {g, b, lds, s};
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* s) {
    *g = config.grid; *b = config.block; *lds = config.lds; *s = config.stream;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3 g, dim3, void**, size_t lds, hipStream_t) {
    char line[200];
    const int id = names.emplace(f, (int)names.size()).first->second;
    snprintf(line, sizeof line, "%d %zu %d %u %u\n", id, lds, limit.count(f) ? limit[f] : -1, g.x, g.y);
    text += line;
    return hipSuccess;
}
const char* recorded() { return text.c_str(); }
void forget() { text.clear(); }
}
"""

CHILD = r"""
import ctypes, json, sys
stand_in = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)  # found before the real runtime
lib = ctypes.CDLL(sys.argv[2])
stand_in.recorded.restype = ctypes.c_char_p
I, P, F = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
size = lib.fni8_paged_attention_workspace_bytes
size.argtypes, size.restype = [I] * 7, I
call = lib.fni8_paged_attention_f16
call.argtypes = [P, I, I, I, I, I, I, P, P, P, P, I, I, P, I, I, P, P, I, I, F, I, P, P, I, P]
out = []
for c in json.loads(sys.argv[3]):
    T, Hq, Hk, D, B, most, width, page = (c[k] for k in ("T", "Hq", "Hk", "D", "B", "most", "width", "page"))
    f = 0x10000  # read by no one
    scale = f if c.get("int8") else None
    n = size(T, Hq, Hk, D, B, most, width * page) if c.get("work", True) else 0
    stand_in.forget()
    rc = call(f, Hq * D, D, T, Hq, Hk, D, f, f, scale, scale, 1 << 10, page, f, width, width, f,
              None if c.get("cu") is False else f, B, most, 0.1, c.get("window", 0), f,
              f if n else None, n + (c.get("more", 0) if n else 0), None)
    lines = [[int(x) for x in l.split()] for l in stand_in.recorded().decode().splitlines()]
    out.append({"rc": rc, "work": n, "launches": lines})
print(json.dumps(out))
"""


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    """launches(calls): for each of the calls in turn, its return code, its workspace and its
    launches as [kernel, LDS bytes, LDS limit that was set for it or -1, grid x, grid y]."""
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    home = tmp_path_factory.mktemp("stand_in")
    (home / "stand_in.cpp").write_text(STAND_IN)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-isystem", "/opt/rocm/include",
                    str(home / "stand_in.cpp"), "-o", str(home / "stand_in.so")], check=True)
    lib = import_module("fni8serve_amd._lib").LIB_PATH
    if not os.path.exists(lib):
        pytest.skip("the library is not built")

    def run(calls):
        p = subprocess.run([sys.executable, "-c", CHILD, str(home / "stand_in.so"), lib,
                            json.dumps(calls)], capture_output=True, text=True, timeout=120)
        assert p.returncode == 0, p.stderr
        return json.loads(p.stdout.splitlines()[-1])
    return run


def _call(D, T, B, most, **kw):
    return dict(dict(T=T, Hq=32, Hk=8, D=D, B=B, most=most, width=64, page=64), **kw)


def test_each_kernel_gets_its_own_lds_limit(pkg, launches):
    """Every kernel with more than 64 KB of LDS has had its limit raised, whichever kernel
    came first."""
    kinds = [_call(D, T, B, most, int8=int8) for D in (64, 128, 256) for int8 in (False, True)
             for T, B, most in ((4, 4, 1), (28, 4, 7), (500, 1, 500), (501, 2, 500))]
    seen = set()
    for order in (kinds, kinds[::-1]):
        for c, r in zip(order, launches(order)):
            assert r["rc"] == 0 and r["launches"], c
            for kernel, lds, limit, x, y in r["launches"]:
                if lds > 64 * 1024:
                    assert limit >= lds, (c, lds, limit)
                    seen.add((c["D"], lds))
    assert {D for D, _ in seen} == {128, 256}  # those of 64 elements take less


def test_the_workspace_is_enough(pkg, launches):
    """The size that the library names is all that a call can use: more changes no launch.
    Decoded tokens without cu_seqlens are one a sequence; their keys are split."""
    calls = [_call(D, B * most if cu else B, B, most, Hk=Hk, cu=cu, width=width, page=16, window=w)
             for D in (64, 128, 256) for Hk in (2, 8) for B in (1, 5, 64, 256, 512)
             for cu, most in ((False, 1), (True, 1), (True, 6), (True, 40)) for width in (20, 32, 1000)
             for w in (0, 100)]
    exact, more = launches(calls), launches([dict(c, more=1 << 40) for c in calls])
    for c, a, b in zip(calls, exact, more):
        assert a["rc"] == 0 and a["launches"] == b["launches"], c
        if not c["cu"] and c["width"] > 24:
            assert a["work"] and len(a["launches"]) == 2, c


def test_the_sum_of_units_and_workers_stays_in_32_bits(pkg, launches):
    """Units close to 2^31: the workgroups' run of units, their number rounded up, is computed
    from the sum of both."""
    call = _call(64, 40438, 40438, 1, Hq=1, Hk=1, cu=False, page=128, width=49979)
    items, units = 40438 + 1 + 40438 // 16, 49979 + 2
    assert 2 ** 31 - 768 <= items * units < 2 ** 31
    few = dict(call, width=49979 - 20)  # a million units fewer
    refused, taken = launches([call, few])
    assert refused["rc"] == -2 and not refused["launches"]
    assert taken["rc"] == 0 and len(taken["launches"]) == 2
