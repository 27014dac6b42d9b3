"""The paged cache's host side over host memory (host/kvcache_host.cpp), by its C entry points. Handles are not freed by themselves."""
import ctypes
import os
import subprocess

import numpy as np

from tang_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/llvm/bin/clang++"


def build(folder):
    lib = os.path.join(str(folder), "kvcache_host.so")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-g", "-O1", "-fPIC", "-shared", "-fopenmp", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), "-o", lib,
                    os.path.join(ROOT, "tests", "host", "kvcache_host.cpp")], check=True, capture_output=True)
    L = ctypes.CDLL(lib)
    for name, (args, res) in capi.SIGNATURES.items():
        if hasattr(L, name):
            f = getattr(L, name)
            f.argtypes, f.restype = args, res
    L.host_fail.argtypes, L.host_fail.restype = [ctypes.c_long], None
    L.host_allocs.restype = L.host_launches.restype = ctypes.c_long
    L.host_bytes.restype = ctypes.c_size_t
    return L


class Refused(Exception):
    def __init__(self, code, text):
        super().__init__("%d: %s" % (code, text))
        self.code = code


class Cache:
    """A cache (f16) of one device handle; beside it, the bits that its sequences hold."""

    def __init__(self, L, layers=1, kh=1, hd=8, page=16, pages=100, seqs=8, max_len=4096):
        self.L, self.layers, self.kh, self.hd = L, layers, kh, hd
        self.dev = self.new("th_device_create", 0)
        cfg = capi.KvCacheConfig(capi.F16, layers, kh, hd, page, pages, seqs, max_len)
        self.c = self.new("th_kv_cache_create", self.dev, ctypes.byref(cfg))
        self.rows = {}  # sequence -> [layers][2][len][kh][hd]

    def call(self, name, *args):
        rc = getattr(self.L, name)(*args)
        if rc:
            raise Refused(rc, self.L.th_last_error().decode())

    def new(self, name, *args):
        h = ctypes.c_void_p()
        self.call(name, *args, ctypes.byref(h))
        return h

    def buffer(self, n, dt=capi.F16):
        return self.new("th_buffer_alloc", self.dev, dt, n)

    def create(self):
        return self.created(1)[0]

    def created(self, n):
        s = (ctypes.c_int32 * n)()
        self.call("th_kv_seq_create", self.c, n, s)
        for x in s:
            self.rows[x] = np.zeros((self.layers, 2, 0, self.kh, self.hd), np.uint16)
        return list(s)

    def fork(self, s, n, length):
        out = (ctypes.c_int32 * n)()
        self.call("th_kv_seq_fork", self.c, s, length, n, out)
        for x in out:
            self.rows[x] = self.rows[s][:, :, :length]
        return list(out)

    def free(self, seqs):
        self.call("th_kv_seq_free", self.c, (ctypes.c_int32 * len(seqs))(*seqs), len(seqs))
        for s in seqs:
            del self.rows[s]

    def resize(self, s, n):
        self.call("th_kv_seq_resize", self.c, s, n)

    def select(self, s, positions):
        p = np.ascontiguousarray(positions, np.uint32)
        self.call("th_kv_seq_select", self.c, s, capi.ptr(p), p.size)

    def compact(self):
        n = ctypes.c_size_t()
        self.call("th_kv_cache_compact", self.c, ctypes.byref(n))
        return n.value

    def info(self):
        p, s = ctypes.c_size_t(), ctypes.c_size_t()
        self.call("th_kv_cache_info", self.c, ctypes.byref(p), ctypes.byref(s))
        return p.value, s.value

    def length(self, s):
        n = ctypes.c_size_t()
        self.call("th_kv_seq_len", self.c, s, ctypes.byref(n))
        return n.value

    def batch(self, max_seqs, max_rows, heads=None):
        return self.new("th_kv_batch_create", self.c, max_seqs, max_rows, heads or self.kh)

    def begin(self, b, seqs, news):
        self.call("th_kv_batch_begin", b, (ctypes.c_int32 * len(seqs))(*seqs), (ctypes.c_uint32 * len(seqs))(*news), len(seqs))

    def fill(self, rng, b, seqs, news):
        """A begun batch's new rows, at random."""
        n = sum(news)
        t = rng.integers(0, 1 << 15, (self.layers, 2, n, self.kh, self.hd)).astype(np.uint16)
        bufs = [self.buffer(max(1, n * self.kh * self.hd)) for _ in range(2)]
        for l in range(self.layers):
            for w in range(2):
                x = np.ascontiguousarray(t[l, w])
                self.call("th_buffer_upload", bufs[w], capi.ptr(x), x.size)
            self.call("th_kv_append", b, l, None, *bufs, None, None, None, 0, 0, None)
        for x in bufs:
            self.call("th_buffer_free", x)
        at = 0
        for s, m in zip(seqs, news):
            self.rows[s] = np.concatenate((self.rows[s], t[:, :, at:at + m]), 2)
            at += m

    def grow(self, rng, b, seqs, news):
        self.begin(b, seqs, news)
        self.fill(rng, b, seqs, news)

    def attend(self, b, rows, heads=None, window=0, sinks=0):
        """An attention call of a begun batch (which only makes its plan here)."""
        q, o = (self.buffer(max(1, rows * (heads or self.kh) * self.hd)) for _ in range(2))
        try:
            self.call("th_kv_batch_attention", b, 0, q, window, sinks, 0.0, o)
        finally:
            self.call("th_buffer_free", q)
            self.call("th_buffer_free", o)

    def plan(self, rows):
        """(tokens, rows items, tile items, joined tokens) of the last attention call; items as {tok0, ntok, seq, j0, j1, sink_end, gap, rec},
        tokens as {row, pos, rec, own_n}."""
        n = (ctypes.c_int * 3)()
        self.L.host_plan_sizes(n)
        out = [np.zeros((m, w), np.int32) for m, w in ((rows, 4), (n[0], 8), (n[1], 8), (n[2], 4))]
        self.L.host_plan(rows, *[capi.ptr(x) for x in out])
        return out

    def check(self, what=""):
        for s, want in self.rows.items():
            assert self.length(s) == want.shape[2], (what, s)
            n = want.shape[2]
            if n == 0:
                continue
            bufs = [self.buffer(n * self.kh * self.hd) for _ in range(2)]
            for l in range(self.layers):
                self.call("th_kv_seq_read", self.c, s, l, 0, n, *bufs)
                for w in range(2):
                    got = np.empty((n, self.kh, self.hd), np.uint16)
                    self.call("th_buffer_download", bufs[w], capi.ptr(got), got.size)
                    assert np.array_equal(got, want[l, w]), (what, s, l, w)
            for x in bufs:
                self.call("th_buffer_free", x)

    def close(self):
        self.call("th_kv_cache_destroy", self.c)
        self.call("th_device_destroy", self.dev)
