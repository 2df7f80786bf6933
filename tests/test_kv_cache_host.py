"""The key-value cache without a GPU: where rows lie (the kernels' own
arithmetic, exported as rocshmem_amd_kv_row) against plain Python integers, and
the entry points' refusals under tests/hip_stub's stand-in for the HIP runtime."""
import ctypes as C
import os
import random
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
STUB_DIR = os.path.join(HERE, "hip_stub")
STUB = os.path.join(STUB_DIR, "_build", "libamdhip64.so.7")
ES = {"BF16": 2, "HALF": 2, "E4M3": 1}


def place(dtype, page, heads, dim, per_pe, slot, head, value):
    part = heads * page * dim * ES[dtype]
    used = 2 * part + (2 * heads * page if dtype == "E4M3" else 0)
    page_bytes = -(-used // 128) * 128
    number, at = divmod(slot, page)
    start = number % per_pe * page_bytes
    offset = start + value * part + (head * page + at) * dim * ES[dtype]
    scale = start + 2 * part + (value * heads + head) * page + at if dtype == "E4M3" else offset
    return number // per_pe, offset, scale, page_bytes


def test_rows_lie_where_the_layout_says(L):
    l, rng = L.load(), random.Random(5)
    pe, offset, scale = C.c_int(), C.c_uint64(), C.c_uint64()
    for _ in range(300):
        dtype = rng.choice(list(ES))
        page, heads, dim = 16 * rng.choice([1, 2, 3, 5, 7, 64, 4096]), rng.randint(1, 40), 16 * rng.randint(1, 16)
        npes = rng.choice([1, 2, 3, 8, 16, 256])
        most = (2 ** 31 - 1) // (page // 16) // npes
        if most < 1:
            continue
        per_pe = rng.choice([1, 2, 3, 1000, most, max(1, most - 1)])
        per_pe = min(per_pe, most)
        cache = L.KvCache(pages=None, dtype=getattr(L, dtype), pages_per_pe=per_pe, page_tokens=page, kv_heads=heads,
                          head_dim=dim)
        slots = npes * per_pe * page
        for slot in {0, 1, page - 1, page % slots, slots - 1, slots // 2, rng.randrange(slots), rng.randrange(slots)}:
            head, value = rng.randrange(heads), rng.randrange(2)
            assert l.kv_row(cache, npes, slot, head, value, C.byref(pe), C.byref(offset), C.byref(scale)) == 0
            want = place(dtype, page, heads, dim, per_pe, slot, head, value)
            assert (pe.value, offset.value, scale.value) == want[:3], (dtype, page, heads, dim, per_pe, npes, slot)
            assert l.kv_page_bytes(getattr(L, dtype), page, heads, dim) == want[3]
        for bad in [(slots, 0), (-1, 0), (0, heads), (0, -1), (1 << 62, 0)]:
            assert l.kv_row(cache, npes, bad[0], bad[1], 0, C.byref(pe), C.byref(offset), C.byref(scale)) == -1
        cache.pages_per_pe = most + 1
        assert l.kv_row(cache, npes, 0, 0, 0, C.byref(pe), C.byref(offset), C.byref(scale)) == -1


def test_caches_that_there_are_not(L):
    l = L.load()
    assert l.kv_page_bytes(L.BF16, 16, 1, 16) == 16 * 16 * 2 * 2
    for bad in [(L.FLOAT, 16, 1, 16), (L.INT, 16, 1, 16), (L.BF16, 8, 1, 16), (L.BF16, 16, 0, 16), (L.BF16, 16, 1, 8),
                (L.BF16, 16, 1, 24), (L.BF16, 16, 1, 512), (L.E4M3, 17, 1, 16), (L.E4M3, -16, 1, 16), (77, 16, 1, 16)]:
        assert l.kv_page_bytes(*bad) == 0


def test_refused_calls_launch_nothing_and_accepted_ones_allocate_nothing(L):
    r = subprocess.run(["make", "-C", STUB_DIR], capture_output=True, text=True)
    if r.returncode != 0 or not os.path.exists(STUB):
        pytest.skip("the HIP stand-in does not build here: " + r.stderr[-300:])
    env = dict(os.environ)
    env["LD_LIBRARY_PATH"] = os.path.dirname(STUB) + os.pathsep + env.get("LD_LIBRARY_PATH", "")
    for name in ("ROCSHMEM_EMU_NPES", "ROCSHMEM_EMU_SPREAD", "ROCSHMEM_EMU_HEAP_CACHED", "ROCSHMEM_HEAP_SIZE"):
        env.pop(name, None)
    r = subprocess.run([sys.executable, os.path.join(HERE, "kv_stub_worker.py")], env=env, capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0, (r.stdout[-800:], r.stderr[-1500:])
    assert "refusals ok" in r.stdout
