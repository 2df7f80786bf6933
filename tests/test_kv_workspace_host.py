"""kv_attend's workspace without a GPU: what rocshmem_amd_kv_attend_bytes says
against a plain count of the splits, that it serves every smaller call, and what
kv_attend then takes and refuses under tests/hip_stub's stand-in for the HIP
runtime."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
STUB_DIR = os.path.join(HERE, "hip_stub")
STUB = os.path.join(STUB_DIR, "_build", "libamdhip64.so.7")

CACHES = [  # cache type, cache heads, query heads, head_dim
    ("BF16", 8, 64, 128), ("E4M3", 1, 8, 256), ("BF16", 1, 48, 128), ("HALF", 24, 24, 64), ("E4M3", 4, 16, 256),
    ("BF16", 2, 2, 16), ("BF16", 1, 71, 128), ("HALF", 5, 5, 80), ("BF16", 512, 512, 64), ("E4M3", 600, 600, 16),
]


def cache_of(L, dtype, heads, dim, page=16):
    return L.KvCache(pages=None, dtype=getattr(L, dtype), pages_per_pe=4, page_tokens=page, kv_heads=heads, head_dim=dim)


@pytest.mark.parametrize("dtype,heads,q_heads,dim", CACHES)
def test_a_workspace_serves_every_smaller_call(L, dtype, heads, q_heads, dim):
    """Never less for more sequences or longer ones."""
    l, c = L.load(), cache_of(L, dtype, heads, dim)
    lengths = [1, 700, 760, 768, 769, 1100, 1152, 1153, 2000, 5000, 20000, 131072, 1 << 22, 1 << 25]
    before = [0] * len(lengths)
    for n in list(range(1, 300)) + [511, 512, 513, 600, 1000, 4097, 65535]:
        now = [l.kv_attend_bytes(c, n, q_heads, x) for x in lengths]
        assert now == sorted(now), (n, now)
        assert all(a <= b for a, b in zip(before, now)), (n, before, now)
        before = now


def ceil(a, b):
    return -(-a // b)


def splits_of_a_call(units, work_groups, dim, longest):
    """How many work-groups share a sequence of `longest` units, the longest of
    its call, where `units` is the bound: whole steps of eight units; the
    first half as for `wanted` equal splits, the second in thirds of those."""
    each, least = ceil(512, work_groups), 3 if work_groups < 512 and dim <= 128 else 2
    wanted = max(each, least)
    if longest <= 48:
        return 1
    big = max(ceil(ceil(longest, wanted), 8) * 8, 24)
    small = max(16, ceil(big // 3, 8) * 8)
    n_big = max(1, longest // 2 // big)
    return ceil(longest, big) if longest <= n_big * big else n_big + ceil(longest - n_big * big, small)


@pytest.mark.parametrize("dtype,heads,q_heads,dim", CACHES)
def test_it_holds_what_the_splits_write(L, dtype, heads, q_heads, dim):
    l, c = L.load(), cache_of(L, dtype, heads, dim)
    group = q_heads // heads
    columns = 1 if dim > 128 else min(4, ceil(group, 16))
    tiles = ceil(group, 16 * columns)
    row = dim * (1 if dtype == "E4M3" else 2)
    for n in (1, 2, 3, 7, 16, 17, 60, 64, 200, 1000):
        for bound in (1, 700, 768, 769, 1153, 3000, 10007, 131072, 1 << 21):
            units, work_groups = ceil(bound, 16) + 1, n * heads * tiles
            got = l.kv_attend_bytes(c, n, q_heads, bound)
            if units <= (72 if work_groups >= 128 and row <= 256 else 48):
                continue  # not split
            most = max(splits_of_a_call(units, work_groups, dim, x)
                       for x in set(list(range(1, min(units, 400))) + [units - 1, units, units // 2, units * 3 // 4]))
            assert got >= n * q_heads * most * (dim + 2) * 4 and got > 0, (n, bound, most, got)


def test_none_for_calls_that_are_not_split_and_for_invalid_ones(L):
    l, c = L.load(), cache_of(L, "BF16", 8, 128)
    assert l.kv_attend_bytes(c, 1, 64, 1) == 0 and l.kv_attend_bytes(c, 1, 64, 48 * 16 - 16) == 0
    assert l.kv_attend_bytes(c, 1, 64, 48 * 16 + 1) > 0  # (a window may touch one unit more)
    assert l.kv_attend_bytes(c, 64, 64, 72 * 16 + 1) > 0
    for bad in [(c, 0, 64, 4096), (c, -1, 64, 4096), (c, 65536, 64, 4096), (c, 4, 0, 4096), (c, 4, 63, 4096),
                (c, 4, -64, 4096), (c, 4, 65536, 4096), (c, 4, 64, 0), (c, 4, 64, -1), (c, 4, 64, (1 << 25) + 1),
                (None, 4, 64, 4096), (cache_of(L, "FLOAT", 8, 128), 4, 64, 4096),
                (cache_of(L, "BF16", 8, 24), 4, 64, 4096), (cache_of(L, "BF16", 8, 128, 8), 4, 64, 4096)]:
        assert l.kv_attend_bytes(*bad) == 0, bad[1:]


def run_under_the_stub(which):
    r = subprocess.run(["make", "-C", STUB_DIR], capture_output=True, text=True)
    if r.returncode != 0 or not os.path.exists(STUB):
        pytest.skip("the HIP stand-in does not build here: " + r.stderr[-300:])
    env = dict(os.environ)
    env["LD_LIBRARY_PATH"] = os.path.dirname(STUB) + os.pathsep + env.get("LD_LIBRARY_PATH", "")
    for name in ("ROCSHMEM_EMU_NPES", "ROCSHMEM_EMU_SPREAD", "ROCSHMEM_EMU_HEAP_CACHED", "ROCSHMEM_HEAP_SIZE"):
        env.pop(name, None)
    r = subprocess.run([sys.executable, os.path.join(HERE, "kv_calls_stub_worker.py"), which], env=env,
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.stdout[-800:], r.stderr[-1500:])
    assert which + " ok" in r.stdout


def test_kv_attend_takes_a_larger_batchs_workspace(L):
    run_under_the_stub("workspace")


def test_an_earlier_calls_error_does_not_end_the_program(L):
    run_under_the_stub("stale")


def test_scales_that_32_bits_do_not_hold_in_base_2_are_refused(L):
    run_under_the_stub("scales")
