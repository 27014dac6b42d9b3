"""The host side of the operators around the paged cache over host memory (host/operators_host.cpp)."""
import ctypes
import os
import subprocess

from host_cache import CLANG, ROOT, Cache, Refused  # noqa: F401
from tang_amd import capi


def build(folder):
    lib = os.path.join(str(folder), "operators_host.so")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-g", "-O1", "-fPIC", "-shared", "-fopenmp", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), "-o", lib,
                    os.path.join(ROOT, "tests", "host", "operators_host.cpp")], check=True, capture_output=True)
    L = ctypes.CDLL(lib)
    for name, (args, res) in capi.SIGNATURES.items():
        if hasattr(L, name):
            f = getattr(L, name)
            f.argtypes, f.restype = args, res
    L.host_fail.argtypes, L.host_fail.restype = [ctypes.c_long], None
    L.host_allocs.restype = ctypes.c_long
    return L


class Refusals:
    """Calls of one entry point with some of its good arguments changed."""

    def __init__(self, cache, name, **good):
        self.c, self.name, self.good = cache, name, good

    def call(self, **over):
        self.c.call(self.name, *{**self.good, **over}.values())

    def refused(self, match, code=capi.TH_ERR_INVALID, **over):
        import pytest
        with pytest.raises(Refused, match=match) as e:
            self.call(**over)
        assert e.value.code == code, e.value
