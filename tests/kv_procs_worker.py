"""One PE of a job with a process per PE, started by
tests/test_gpu_kv_cache_cuts.py: every process puts its share of the tokens
into pages of all PEs, reads others' rows back, attends to all pages and to its
own, and joins what the processes reached.  Prints "ok <pe>" at the end."""
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from rocshmem_amd import lib as L  # noqa: E402
from tests import kv_reference as ref  # noqa: E402

HEADS, GROUP, DIM, PAGE, LENGTHS = 2, 4, 64, 16, [1000, 33, 0, 250]


def main():
    npes, me = int(os.environ["ROCSHMEM_EMU_PROCS"]), int(os.environ["ROCSHMEM_EMU_RANK"])
    l = L.load()
    assert l.init(0, 64 << 20) == 0

    def dev(a):
        a = np.ascontiguousarray(a)
        p = l.dev_alloc(a.nbytes)
        assert l.copy_in(p, a.ctypes.data, a.nbytes) == 0
        return p

    def host(p, shape, dtype):
        out = np.empty(shape, dtype)
        assert l.copy_out(out.ctypes.data, p, out.nbytes) == 0
        return out

    rng = np.random.default_rng(9)  # the same in every process
    need = [-(-n // PAGE) for n in LENGTHS]
    per_pe = -(-sum(need) // npes)
    order = rng.permutation(npes * per_pe).astype(np.int32)
    table = np.full((len(LENGTHS), max(need)), -1, np.int32)
    for b in range(len(LENGTHS)):
        table[b, :need[b]] = order[sum(need[:b]):sum(need[:b + 1])]
    slots = np.concatenate([ref.tokens_of(n, n, table[b], PAGE, npes * per_pe) for b, n in enumerate(LENGTHS)])
    slots = slots.astype(np.int64)
    raw = ref.encode(rng.standard_normal((len(slots), 2 * HEADS, DIM)).astype(np.float32), "bf16")
    q_raw = ref.encode(rng.standard_normal((len(LENGTHS), HEADS * GROUP, DIM)).astype(np.float32), "bf16")
    x, q = ref.decode(raw, "bf16"), ref.decode(q_raw, "bf16")
    m = ref.Cache("e4m3", npes, per_pe, PAGE, HEADS, DIM)
    m.put(slots, x[:, :HEADS], x[:, HEADS:])

    pages = l.malloc(m.page_bytes * per_pe)
    rows = len(LENGTHS) * HEADS * GROUP
    partial, partial_lse = l.malloc(rows * DIM * 4), l.malloc(rows * 4)
    assert pages and partial and partial_lse
    c = L.KvCache(pages=pages, dtype=L.E4M3, pages_per_pe=per_pe, page_tokens=PAGE, kv_heads=HEADS, head_dim=DIM)
    assert l.barrier_all() == 0
    mine = np.arange(len(slots)) % npes == me
    kv = dev(raw[mine])
    row = 2 * HEADS * DIM
    assert l.kv_put(c, L.BF16, kv, row, kv + HEADS * DIM * 2, row, dev(slots[mine]), int(mine.sum()), me, None) == 0
    l.stream_sync(None)
    assert l.barrier_all() == 0

    back = [l.dev_alloc(len(slots) * HEADS * DIM * 4) for _ in range(2)]
    assert l.kv_get(c, L.FLOAT, back[0], HEADS * DIM, back[1], HEADS * DIM, dev(slots), len(slots), me, None) == 0
    d_q, d_table, d_len = dev(q_raw), dev(table), dev(np.array(LENGTHS, np.int32))
    nbytes = l.kv_attend_bytes(c, len(LENGTHS), HEADS * GROUP, max(LENGTHS))
    ws, out, lse = l.dev_alloc(max(nbytes, 16)), l.dev_alloc(rows * DIM * 4), l.dev_alloc(rows * 4)
    joined, joined_lse = l.dev_alloc(rows * DIM * 4), l.dev_alloc(rows * 4)
    for own, to, to_lse in ((0, out, lse), (1, partial, partial_lse)):
        assert l.kv_attend(c, L.BF16, d_q, HEADS * GROUP * DIM, HEADS * GROUP, L.FLOAT, to, HEADS * GROUP * DIM, to_lse,
                           d_table, table.shape[1], d_len, len(LENGTHS), max(LENGTHS), 0, 0.125, 0.0, own, ws, nbytes, me,
                           None) == 0
    l.stream_sync(None)
    assert l.barrier_all() == 0
    assert l.kv_join(L.FLOAT, partial, partial_lse, rows, DIM, L.FLOAT, joined, joined_lse, 0, 0, npes, me, None) == 0
    l.stream_sync(None)

    for value in (0, 1):
        want = m.rows(slots, value).astype(np.float32)
        assert np.array_equal(host(back[value], want.shape, np.float32), want), value
    for got, got_lse in ((out, lse), (joined, joined_lse)):
        got = host(got, (len(LENGTHS), HEADS * GROUP, DIM), np.float32).astype(np.float64)
        got_lse = host(got_lse, (len(LENGTHS), HEADS * GROUP), np.float32)
        for b, n in enumerate(LENGTHS):
            s = ref.tokens_of(n, n, table[b], PAGE, npes * per_pe)
            k, v = (m.rows(s, value) for value in (0, 1))
            for h in range(HEADS * GROUP):
                want, want_lse, d, dlse = ref.attend(q[b, h], k[:, h // GROUP], v[:, h // GROUP], 0.125, 0.0)
                assert (np.abs(got[b, h] - want) <= d + ref.U["fp32"] * (np.abs(want) + d)).all(), (b, h)
                assert got_lse[b, h] == want_lse if not n else abs(got_lse[b, h] - want_lse) <= dlse
    assert l.kv_refused(0) == 0
    assert l.barrier_all() == 0
    l.finalize()
    print("ok %d" % me)


if __name__ == "__main__":
    main()
