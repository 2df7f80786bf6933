"""Calls of the key-value cache on a machine without a GPU, in child processes
of the CPU tests under tests/hip_stub's stand-in for the HIP runtime (which
counts launches and drops them).  The argument says which."""
import ctypes as C
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from rocshmem_amd import lib as L  # noqa: E402

P, HEAP = 4, 8 << 20


class Calls:
    def __init__(self):
        self.l = l = L.load()
        assert l.init(P, HEAP) == 0
        self.stub = C.CDLL("libamdhip64.so.7")
        self.stub.hip_stub_counts.argtypes = [C.POINTER(C.c_ulonglong), C.POINTER(C.c_ulonglong)]
        self.pages = l.malloc(l.kv_page_bytes(L.BF16, 16, 2, 64) * 4)
        self.end = self.pages + l.heap_size()  # not symmetric memory from here on
        self.d = l.dev_alloc(1 << 20)
        self.cache = L.KvCache(pages=self.pages, dtype=L.BF16, pages_per_pe=4, page_tokens=16, kv_heads=2, head_dim=64)

    def launches(self):
        n = C.c_ulonglong()
        self.stub.hip_stub_counts(C.byref(n), None)
        return n.value

    def put(self):
        d = self.d
        return self.l.kv_put(self.cache, L.BF16, d, 128, d + 4096, 128, d + 65536, 4, 0, None)

    def get(self):
        d = self.d
        return self.l.kv_get(self.cache, L.BF16, d, 128, d + 4096, 128, d + 65536, 4, 0, None)

    def attend(self, n=3, max_len=64, window=0, ws=None, ws_bytes=0, scale=0.125):
        d = self.d  # the buffers are not looked at: nothing runs
        return self.l.kv_attend(self.cache, L.BF16, d, 512, 8, L.BF16, d + 8192, 512, d + 32768, d + 40000, 1 << 12,
                                d + 50000, n, max_len, window, scale, 0.0, 0, ws, ws_bytes, 0, None)

    def join(self):
        return self.l.kv_join(L.FLOAT, self.pages, self.pages + 8192, 8, 64, L.BF16, self.d, self.d + 8192, 0, 0, P, 0,
                              None)


def workspace(c):
    need = c.l.kv_attend_bytes(c.cache, 256, 8, 1 << 16)
    assert need > 0
    ws = c.l.dev_alloc(need + 16)
    for n in range(1, 257):
        for max_len in (1, 500, 769, 1200, 30000, 1 << 16):
            for window in (0, 1000, 5000):
                before = c.launches()
                assert c.attend(n, max_len, window, ws, need) == 0, (n, max_len, window)
                assert c.launches() > before
    for n in (1, 3, 256):
        need = c.l.kv_attend_bytes(c.cache, n, 8, 1 << 16)
        assert need > 0
        # (a batch smaller than n may be what needs all of it: none of this size is enough for any)
        for other in [dict(ws=None, ws_bytes=need), dict(ws=ws, ws_bytes=0), dict(ws=ws, ws_bytes=n * 8 * 66 * 4),
                      dict(ws=ws + 8, ws_bytes=need), dict(ws=c.end - 64, ws_bytes=need)]:
            before = c.launches()
            assert c.attend(n, 1 << 16, **other) == -1, (n, other)
            assert c.launches() == before
    need = c.l.kv_attend_bytes(c.cache, 1, 8, 1 << 16)
    assert c.attend(1, 1 << 16, ws=ws, ws_bytes=need) == 0 and c.attend(1, 1 << 16, ws=ws, ws_bytes=need - 1) == -1


def stale(c):
    """An error of an earlier call, which nobody has fetched, is not these calls'."""
    c.stub.hipPointerGetAttributes.argtypes = [C.c_void_p, C.c_void_p]
    about = C.create_string_buffer(256)
    for call in (c.put, c.get, c.attend, c.join):
        assert c.stub.hipPointerGetAttributes(about, 8) != 0  # no device memory
        before = c.launches()
        assert call() == 0 and c.launches() == before + 1
        assert c.stub.hipGetLastError() != 0 and c.stub.hipGetLastError() == 0  # still there, once


def scales(c):
    """A scale whose product with log2 e has no 32 bits is refused."""
    for scale in (2.0 ** 127, -2.0 ** 127, 2.4e38, 3.4028234663852886e38):
        before = c.launches()
        assert c.attend(scale=scale) == -1 and c.launches() == before, scale
    for scale in (0.0, -1.0, 2.0 ** 126, 1.7e38, 1e-45):
        assert c.attend(scale=scale) == 0, scale


if __name__ == "__main__":
    calls = Calls()
    {"workspace": workspace, "stale": stale, "scales": scales}[sys.argv[1]](calls)
    calls.l.finalize()
    print(sys.argv[1], "ok")
