"""Refusals of the key-value cache's entry points on a machine without a GPU: a
child process of tests/test_kv_cache_host.py, run with tests/hip_stub's
stand-in for the HIP runtime, which counts launches and drops them."""
import ctypes as C
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from rocshmem_amd import lib as L  # noqa: E402

P, HEAP = 4, 8 << 20
BIG = (1 << 64) - 1


def main():
    l = L.load()
    cache = L.KvCache(pages=0, dtype=L.BF16, pages_per_pe=4, page_tokens=16, kv_heads=2, head_dim=64)
    assert l.kv_refused(0) == -1
    assert l.kv_put(cache, L.BF16, None, 0, None, 0, None, 0, 0, None) == -1  # before init
    assert l.init(P, HEAP) == 0
    stub = C.CDLL("libamdhip64.so.7")
    stub.hip_stub_counts.argtypes = [C.POINTER(C.c_ulonglong), C.POINTER(C.c_ulonglong)]
    stub.hip_stub_alloc_calls.restype = C.c_ulonglong

    def launches():
        n = C.c_ulonglong()
        stub.hip_stub_counts(C.byref(n), None)
        return n.value

    size = l.kv_page_bytes(L.BF16, 16, 2, 64) * 4
    pages = l.malloc(size)
    end = pages + l.heap_size()  # not symmetric memory from here on
    d = l.dev_alloc(1 << 20)
    assert pages and d and l.kv_refused(0) == 0

    def kv(**other):
        f = dict(pages=pages, dtype=L.BF16, pages_per_pe=4, page_tokens=16, kv_heads=2, head_dim=64)
        return L.KvCache(**{**f, **other})

    def rows(call, **other):
        a = dict(cache=kv(), dtype=L.BF16, k=d, k_row=128, v=d + 4096, v_row=128, slots=d + 65536, n=4, pe=0)
        a.update(other)
        return lambda: call(a["cache"], a["dtype"], a["k"], a["k_row"], a["v"], a["v_row"], a["slots"], a["n"],
                            a["pe"], None)

    def attend(**other):
        a = dict(cache=kv(), dtype=L.BF16, q=d, q_row=512, heads=8, out_dtype=L.BF16, out=d + 8192, out_row=512,
                 lse=d + 32768, table=d + 40000, table_row=4, lengths=d + 50000, n=3, max_len=64, window=0, scale=0.125,
                 softcap=0.0, pages_from=0, ws=d + 65536, ws_bytes=1 << 19, pe=0)
        a.update(other)
        return lambda: l.kv_attend(a["cache"], a["dtype"], a["q"], a["q_row"], a["heads"], a["out_dtype"], a["out"],
                                   a["out_row"], a["lse"], a["table"], a["table_row"], a["lengths"], a["n"],
                                   a["max_len"], a["window"], a["scale"], a["softcap"], a["pages_from"], a["ws"],
                                   a["ws_bytes"], a["pe"], None)

    def join(**other):
        a = dict(dtype=L.FLOAT, partial=pages, lse_in=pages + 8192, rows=8, dim=64, out_dtype=L.BF16, out=d,
                 lse=d + 8192, start=0, log_stride=0, size=P, pe=0)
        a.update(other)
        return lambda: l.kv_join(a["dtype"], a["partial"], a["lse_in"], a["rows"], a["dim"], a["out_dtype"], a["out"],
                                 a["lse"], a["start"], a["log_stride"], a["size"], a["pe"], None)

    bad_caches = [kv(dtype=L.FLOAT), kv(dtype=L.INT), kv(dtype=99), kv(pages=0), kv(pages=pages + 8), kv(pages=d),
                  kv(pages=l.pe_ptr(pages, 1)), kv(pages=end - 4096), kv(page_tokens=0), kv(page_tokens=24),
                  kv(page_tokens=-16), kv(page_tokens=1 << 17), kv(kv_heads=0), kv(kv_heads=5000), kv(head_dim=0),
                  kv(head_dim=40), kv(head_dim=272), kv(pages_per_pe=0), kv(pages_per_pe=1 << 20),
                  kv(pages_per_pe=(1 << 31) - 1)]
    calls = []
    for c in bad_caches:
        calls += [rows(l.kv_put, cache=c), rows(l.kv_get, cache=c), attend(cache=c)]
    for call in (l.kv_put, l.kv_get):
        for other in [dict(cache=None), dict(dtype=L.INT), dict(dtype=L.E4M3), dict(dtype=-1), dict(pe=P), dict(pe=-1),
                      dict(k=None), dict(v=None), dict(slots=None), dict(k=d + 1), dict(v=d + 1), dict(slots=d + 4),
                      dict(dtype=L.FLOAT, k=d + 2), dict(n=1 << 62), dict(k_row=BIG), dict(v_row=1 << 62),
                      dict(k=end - 64), dict(v=end - 64), dict(slots=end - 8)]:
            calls.append(rows(call, **other))
    calls += [rows(l.kv_get, k_row=127), rows(l.kv_get, v_row=0)]
    for other in [dict(cache=None), dict(dtype=L.FLOAT), dict(dtype=L.HALF), dict(cache=kv(dtype=L.HALF)),
                  dict(dtype=L.E4M3, cache=kv(dtype=L.E4M3)), dict(out_dtype=L.HALF), dict(out_dtype=L.E4M3),
                  dict(q=None), dict(q=d + 1), dict(out=None), dict(out=d + 1), dict(out_dtype=L.FLOAT, out=d + 2),
                  dict(lse=d + 2), dict(table=None), dict(table=d + 2), dict(lengths=None), dict(lengths=d + 1),
                  dict(heads=0), dict(heads=7), dict(heads=-8), dict(heads=1 << 20), dict(n=-1), dict(n=70000),
                  dict(max_len=-1), dict(window=-1), dict(scale=float("inf")), dict(scale=float("nan")),
                  dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(softcap=1e-38), dict(pages_from=2),
                  dict(pages_from=-1), dict(out_row=511), dict(q_row=BIG), dict(out_row=1 << 62),
                  dict(table_row=1 << 40), dict(pe=P), dict(pe=-1), dict(q=end - 64), dict(out=end - 64),
                  dict(lse=end - 8), dict(lengths=end - 4), dict(table=end - 4)]:
        calls.append(attend(**other))
    for other in [dict(dtype=L.E4M3), dict(dtype=L.INT), dict(out_dtype=L.E4M3), dict(partial=None), dict(partial=d),
                  dict(partial=pages + 8), dict(partial=l.pe_ptr(pages, 2)), dict(partial=end - 1024), dict(lse_in=None),
                  dict(lse_in=d), dict(lse_in=pages + 2), dict(lse_in=end - 16), dict(rows=1 << 60), dict(dim=0),
                  dict(dim=12), dict(dim=-8), dict(out=None), dict(out=d + 1), dict(out=end - 8), dict(lse=d + 1),
                  dict(lse=end - 8), dict(out=pages + 1024), dict(lse=pages + 4), dict(out=pages + 8176), dict(start=-1), dict(start=P), dict(size=0), dict(size=P + 1), dict(log_stride=-1),
                  dict(log_stride=40), dict(log_stride=1, size=3), dict(start=1, size=P), dict(pe=P), dict(pe=-1)]:
        calls.append(join(**other))
    for i, call in enumerate(calls):
        before = launches()
        assert call() == -1, i
        assert launches() == before, (i, "launched something")
    # the same calls unspoiled launch, and allocate nothing
    allocations = stub.hip_stub_alloc_calls()
    for call in [rows(l.kv_put), rows(l.kv_get), attend(), join(), rows(l.kv_put, k_row=0), attend(lse=None),
                 attend(dtype=L.HALF, cache=kv(dtype=L.E4M3), out_dtype=L.FLOAT, out_row=512), join(lse=None),
                 join(start=1, log_stride=1, size=2, pe=2, partial=l.pe_ptr(pages, 2), lse_in=l.pe_ptr(pages, 2) + 8192)]:
        before = launches()
        assert call() == 0
        assert launches() > before
    assert stub.hip_stub_alloc_calls() == allocations
    for call in [rows(l.kv_put, n=0), rows(l.kv_get, n=0), attend(n=0), join(rows=0)]:
        before = launches()
        assert call() == 0 and launches() == before
    # the workspace, for a call that wants one
    long = dict(max_len=1 << 16, table_row=1 << 12, table=d + 40000, n=1)
    need = l.kv_attend_bytes(kv(), 1, 8, 1 << 16)
    if need:
        for other in [dict(ws=None), dict(ws_bytes=need - 1), dict(ws=d + 8), dict(ws=end - 64)]:
            before = launches()
            assert attend(**long, **other)() == -1, other
            assert launches() == before
    assert attend(**long, ws_bytes=need)() == 0
    l.finalize()
    print("refusals ok", len(calls))


if __name__ == "__main__":
    main()
