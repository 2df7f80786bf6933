"""The key-value cache where the work is cut in other ways than in
tests/test_gpu_kv_cache.py: many splits and runs, many sequences, bounds far
above the lengths, query heads by the dozens, graphs on two streams at once,
caches beyond 32 bits of bytes, a cached heap, one process per PE."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

from tests import kv_reference as ref
from tests.test_gpu_kv_cache import HEAP, P, Dev, OnHeap, Run, dev, type_of, values  # noqa: F401

pytestmark = pytest.mark.gpu


CUTS = [  # source, cache, cache heads, query heads each, dim, page, lengths, bound
    # the longest in splits of more than 256 units, which a work-group's wavefronts take in two runs
    ("bf16", "bf16", 1, 3, 16, 16, [9000] + [1, 17, 0] * 100, None),
    ("bf16", "bf16", 1, 2, 32, 16, [9001] + [1, 17, 0, 5] * 150, None),
    ("bf16", "e4m3", 1, 1, 16, 32, [14000] + [3] * 299, 14100),
    ("fp16", "e4m3", 1, 2, 32, 48, [11111] + [40] * 270, 12000),
    # more sequences than a wavefront looks at
    ("bf16", "bf16", 1, 2, 16, 16, [3, 0, 16, 33] * 260 + [9000, 1400, 770, 2], None),
    ("bf16", "bf16", 1, 2, 16, 16, [3, 0, 1500, 33, 800] * 40 + [2100], 6000),
    # query heads in two to four tiles, whole and split
    ("bf16", "bf16", 1, 32, 128, 64, [601, 5], None),
    ("fp16", "fp16", 1, 48, 128, 16, [1300, 0, 33], None),
    ("bf16", "bf16", 1, 64, 96, 32, [1301, 90], None),
    ("bf16", "e4m3", 1, 71, 128, 64, [700, 1], None),
    ("fp16", "e4m3", 1, 64, 112, 48, [1700], None),
    ("bf16", "e4m3", 2, 48, 128, 16, [1200, 40], 131072),
    ("bf16", "bf16", 1, 40, 256, 16, [900, 1100], None),
    # bounds far above the lengths, and just above
    ("bf16", "bf16", 2, 4, 128, 64, [400, 1, 0, 65], 1 << 25),
    ("fp16", "fp16", 8, 1, 64, 16, [2011, 300], 2600),
    ("fp16", "fp16", 8, 1, 64, 16, [2011, 300], 4000),
    ("bf16", "e4m3", 1, 8, 80, 16, [1, 0, 0], 100000),
    # on either side of one split
    ("bf16", "bf16", 1, 4, 64, 16, [768], None),
    ("bf16", "bf16", 1, 4, 64, 16, [769], None),
    ("bf16", "bf16", 8, 1, 16, 16, [1152] * 16, None),
    ("bf16", "bf16", 8, 1, 16, 16, [1153] + [30] * 15, None),
]


@pytest.mark.parametrize("src,cache,heads,group,dim,page,lengths,bound", CUTS)
def test_attention_however_it_is_cut(rt, L, dev, src, cache, heads, group, dim, page, lengths, bound):
    r = Run(rt, L, dev, src, cache, heads, group, dim, page, lengths, max_len=bound)
    if bound:  # a table that holds as much as the bound says
        wide = min(-(-bound // page), 4096)
        r.table = np.concatenate([r.table, np.full((len(lengths), wide - r.table.shape[1]), -1, np.int32)], 1)
    rt.l.kv_refused(1)
    r.call().check()
    for window in (100, max(lengths) * 3 // 4):
        r.call(window=window, softcap=20.0, out="fp32").check()
    assert rt.l.kv_refused(1) == 0
    r.free()


@pytest.mark.parametrize("cap", [2.0 ** -100, 1e-3, 0.5, 1e4, 1e30])
def test_caps_of_any_size(rt, L, dev, cap):
    """Far below a large cap a capped score is off by a few roundings relative
    to itself (of the cap's reciprocal, the quotient, the series, the cap in
    base 2, the product; 16 half steps allow twice that); the oracle's own
    allowance counts steps of the cap instead, which is right for the small ones."""
    r = Run(rt, L, dev, "bf16", "bf16", 2, 3, 48, 16, [40, 300], spread=0.7)
    if cap > 100:
        r.call(softcap=cap, out="fp32")
        rt.l.stream_sync(None)
        out, lse = r.got()
        for b, n in enumerate(r.lengths):
            slots = ref.tokens_of(int(n), r.max_len, r.table[b], 16, r.n_pages)
            k, v = (r.m.rows(slots, value) for value in (0, 1))
            for h in range(6):
                s = k[:, h // 3] @ r.q[b, h] * r.scale
                more = 16 * 2.0 ** -24 * np.abs(s).max()
                want, want_lse, d, dlse = ref.attend(r.q[b, h], k[:, h // 3], v[:, h // 3], r.scale, 0.0)
                s = cap * np.tanh(s / cap)
                p = np.exp(s - s.max())
                want, want_lse = p @ v[:, h // 3] / p.sum(), s.max() + np.log(p.sum())
                d += 4 * more * (p @ np.abs(v[:, h // 3]) / p.sum())
                assert (np.abs(out[b, h] - want) <= d + ref.U["fp32"] * (np.abs(want) + d)).all()
                assert abs(lse[b, h] - want_lse) <= dlse + more
    else:
        r.call(softcap=cap).check()
    r.free()


def test_infinite_keys_of_rows_narrower_than_the_products(rt, L, dev):
    """A key whose score is -infinity takes no part, though a row of 80 elements
    is multiplied as 128; one whose score is +infinity makes its sequence NaN and no other."""
    r = Run(rt, L, dev, "bf16", "bf16", 1, 2, 80, 16, [40, 33, 900])
    r.q_raw = r.q_raw & 0x7FFF
    r.q = ref.decode(r.q_raw, "bf16")
    for b, at, x in ((0, 7, -np.inf), (2, 850, -np.inf), (1, 3, np.inf)):
        slot = ref.tokens_of(1000, 1000, r.table[b], 16, r.n_pages)[at]
        k = r.m.rows([slot], 0)
        k[..., 0] = x
        r.m.put([slot], k, r.m.rows([slot], 1))
    r.h.upload()
    r.call(out="fp32")
    rt.l.stream_sync(None)
    out, lse = r.got()
    assert np.isnan(out[1]).all() and not np.isfinite(lse[1]).any()
    for b in (0, 2):
        slots = ref.tokens_of(int(r.lengths[b]), 1000, r.table[b], 16, r.n_pages)
        k, v = (r.m.rows(slots, value)[:, 0] for value in (0, 1))
        there = np.isfinite(k[:, 0])
        for h in range(2):
            want, want_lse, d, dlse = ref.attend(r.q[b, h], k[there], v[there], r.scale, 0.0)
            assert (np.abs(out[b, h] - want) <= d + ref.U["fp32"] * (np.abs(want) + d)).all()
            assert abs(lse[b, h] - want_lse) <= dlse
    r.free()


def test_no_tokens_by_bound_or_by_table(rt, L, dev):
    l = rt.l
    r = Run(rt, L, dev, "bf16", "bf16", 2, 3, 64, 16, [20, 5])
    r.max_len = 1
    r.lengths[:] = 0
    r.call().check()
    out, lse = dev.blank(2 * 6 * 64 * 2), dev.blank(2 * 6 * 4)
    lengths = dev(np.array([20, 5], np.int32))
    for max_len, table, table_row in ((0, dev(r.table), r.table.shape[1]), (64, None, 0)):
        l.kv_refused(1)
        l.fill(out, 0x55, 2 * 6 * 64 * 2)
        assert l.kv_attend(r.h.c, L.BF16, dev(r.q_raw), 9 * 64, 6, L.BF16, out, 6 * 64, lse, table, table_row, lengths, 2,
                           max_len, 0, 0.1, 0.0, 0, None, 0, 0, None) == 0
        l.stream_sync(None)
        assert (dev.read(out, 2 * 6 * 64 * 2) == 0).all()
        assert np.isneginf(dev.read(lse, 2 * 6 * 4).view(np.float32)).all()
        assert l.kv_refused(1) == 2
    r.free()


def test_sequences_share_pages(rt, L, dev):
    """A common prefix is held once; a page may also come twice in a sequence."""
    r = Run(rt, L, dev, "fp16", "e4m3", 2, 2, 64, 16, [64, 900, 40])
    r.table[2, :3] = r.table[1, :3]
    r.table[0, 3] = r.table[0, 1]
    r.call().check()
    r.free()


def test_two_graphs_and_eager_calls_at_once(rt, L, dev):
    """Two captured calls with a workspace each, replayed on streams of their
    own at the same time and beside eager calls on a third, while the lengths
    go through everything that decides how the work is cut."""
    from tests.test_gpu_graph_capture import hip
    l, h = rt.l, hip()
    bound = 20000
    runs = [Run(rt, L, dev, "bf16", "bf16", 2, 4, 64, 16, [6000, 700, 1], max_len=bound),
            Run(rt, L, dev, "fp16", "e4m3", 1, 20, 128, 32, [5000, 5200, 30, 0], max_len=bound, seed=1)]
    eager = Run(rt, L, dev, "bf16", "bf16", 1, 2, 32, 16, [3000, 100], seed=2)
    streams, graphs, exes = ([C.c_void_p() for _ in range(n)] for n in (3, 2, 2))
    for s in streams:
        assert h.hipStreamCreate(C.byref(s)) == 0
    try:
        full = [r.lengths.copy() for r in runs]
        for i, r in enumerate(runs):
            q, table, r.d_len = dev(r.q_raw), dev(r.table), dev(r.lengths)
            n, hq = len(r.lengths), r.heads * r.group
            r.window, r.softcap, r.scale, r.out_type, r.out_row = 0, 0.0, r.dim ** -0.5, r.src, hq * r.dim
            r.out, r.lse = dev.blank(n * hq * r.dim * 2), dev.blank(n * hq * 4)
            r.ws_bytes = l.kv_attend_bytes(r.h.c, n, hq, bound)
            assert r.ws_bytes > 0
            r.ws = dev.blank(r.ws_bytes)
            assert h.hipStreamBeginCapture(streams[i], 0) == 0
            rc = l.kv_attend(r.h.c, type_of(L, r.src), q, r.q_raw.shape[1] * r.dim, hq, type_of(L, r.src), r.out, hq * r.dim,
                             r.lse, table, r.table.shape[1], r.d_len, n, bound, 0, r.scale, 0.0, 0, r.ws, r.ws_bytes, 0,
                             streams[i])
            assert h.hipStreamEndCapture(streams[i], C.byref(graphs[i])) == 0 and rc == 0
            assert h.hipGraphInstantiate(C.byref(exes[i]), graphs[i], None, None, 0) == 0
        for part in (0.0, 0.001, 0.1, 1.0, 0.25, 0.6):
            for r, most in zip(runs, full):
                r.lengths = np.ceil(most * part).astype(np.int32)
                rt.put_bytes(r.d_len, r.lengths)
                l.fill(r.ws, 0x77, r.ws_bytes)
            for i in range(2):
                assert h.hipGraphLaunch(exes[i], streams[i]) == 0
            eager.call(window=500, stream=streams[2])
            for s in streams:
                assert h.hipStreamSynchronize(s) == 0
            for r in runs + [eager]:
                r.check()
    finally:
        for x, g in zip(exes, graphs):
            if x.value:
                h.hipGraphExecDestroy(x)
                h.hipGraphDestroy(g)
        for s in streams:
            h.hipStreamDestroy(s)
        for r in runs + [eager]:
            r.free()


@pytest.mark.parametrize("src,cache", [("bf16", "bf16"), ("fp16", "e4m3")])
def test_a_step_over_all_pes_from_one_graph(rt, L, dev, src, cache):
    """What a step of answering does when each PE attends to its own pages: new
    rows put, every PE's attention, the join for every PE; captured once and
    replayed with new rows and queries while the sequences grow."""
    from tests.test_gpu_graph_capture import hip
    l, h = rt.l, hip()
    heads, group, dim, page, n = 2, 3, 64, 16, 3
    hq, row = heads * group, 2 * heads * dim
    r = Run(rt, L, dev, src, cache, heads, group, dim, page, [900, 1, 130])
    r.window, r.softcap, r.scale, r.out_type, r.out_row = 0, 0.0, 0.125, "fp32", hq * dim
    r.max_len = r.table.shape[1] * page
    most = r.lengths.copy()
    r.lengths = np.maximum(most - 4, 0).astype(np.int32)
    kv, slots, lengths = dev(np.zeros((n, row), np.uint16)), dev(np.zeros(n, np.int64)), dev(r.lengths)
    q, table = dev(r.q_raw), dev(r.table)
    r.ws_bytes = l.kv_attend_bytes(r.h.c, n, hq, r.max_len)
    ws = [dev.blank(r.ws_bytes) for _ in range(P)]
    partial, partial_lse = l.malloc(n * hq * dim * 4), l.malloc(n * hq * 4)
    joined = [(dev.blank(n * hq * dim * 4), dev.blank(n * hq * 4)) for _ in range(P)]
    stream, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert h.hipStreamCreate(C.byref(stream)) == 0
    try:
        assert h.hipStreamBeginCapture(stream, 0) == 0
        rc = [l.kv_put(r.h.as_of(L, 2), type_of(L, src), kv, row, kv + row, row, slots, n, 2, stream)]
        for pe in range(P):
            rc.append(l.kv_attend(r.h.as_of(L, pe), type_of(L, src), q, r.q_raw.shape[1] * dim, hq, L.FLOAT,
                                  l.pe_ptr(partial, pe), hq * dim, l.pe_ptr(partial_lse, pe), table, r.table.shape[1],
                                  lengths, n, r.max_len, 0, 0.125, 0.0, L.KV_OWN_PAGES, ws[pe], r.ws_bytes, pe, stream))
        for pe in range(P):
            rc.append(l.kv_join(L.FLOAT, l.pe_ptr(partial, pe), l.pe_ptr(partial_lse, pe), n * hq, dim, L.FLOAT,
                                *joined[pe], 0, 0, P, pe, stream))
        assert h.hipStreamEndCapture(stream, C.byref(graph)) == 0 and not any(rc)
        assert h.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
        for _ in range(4):
            at = r.lengths.copy()
            r.lengths = np.minimum(at + 1, most).astype(np.int32)
            new = np.array([int(r.table[b, i // page]) * page + i % page if i < r.lengths[b] else -1
                            for b, i in enumerate(at)], np.int64)
            raw, x = values(r.rng, (n, 2 * heads, dim), src, 0.3)
            r.q_raw, r.q = values(r.rng, r.q_raw.shape, src, 0.3)
            r.m.put(new, x[:, :heads], x[:, heads:])
            for ptr, a in ((kv, raw), (slots, new), (lengths, r.lengths), (q, r.q_raw)):
                rt.put_bytes(ptr, a)
            assert h.hipGraphLaunch(exe, stream) == 0 and h.hipStreamSynchronize(stream) == 0
            for pe in range(P):
                r.ws, (r.out, r.lse) = ws[pe], joined[pe]
                r.check()  # the join's roundings are far inside the bound for the sums over the tokens
    finally:
        if exe.value:
            h.hipGraphExecDestroy(exe)
            h.hipGraphDestroy(graph)
        h.hipStreamDestroy(stream)
        l.free(partial)
        l.free(partial_lse)
        r.free()


def test_join_refuses_to_write_over_what_it_reads(rt, L, dev):
    l = rt.l
    part, lse = l.malloc(8 * 64 * 4), l.malloc(32)
    out = dev.blank(8 * 64 * 4)
    for o, s in ((part, None), (part + 8 * 64 * 4 - 4, None), (lse - 4, None), (out, lse), (out, part + 64)):
        assert l.kv_join(L.FLOAT, part, lse, 8, 64, L.FLOAT, o, s, 0, 0, P, 0, None) == -1
    l.free(part)
    l.free(lse)


def test_a_cache_of_more_than_four_gigabytes_on_a_pe(rt, L):
    """Rows whose bytes lie beyond 32 bits, on both of two PEs; nothing around them changes."""
    per_pe, page, heads, dim = 70000, 64, 4, 64
    rt.down()
    l = rt.up(2, 8 << 30)
    d = Dev(rt)
    try:
        m = ref.Cache("bf16", 2, 1, page, heads, dim)  # a page's model
        assert m.page_bytes * per_pe > 1 << 32
        ptr = l.malloc(m.page_bytes * per_pe)
        assert ptr
        c = L.KvCache(pages=ptr, dtype=L.BF16, pages_per_pe=per_pe, page_tokens=page, kv_heads=heads, head_dim=dim)
        rng = np.random.default_rng(4)
        pages = np.array([per_pe - 1, 2 * per_pe - 1, 66000, per_pe + 1, 2 * per_pe - 2], np.int32)
        around = {n for p in pages for n in (p - 1, p, p + 1) if n < 2 * per_pe}
        where = lambda n: l.pe_ptr(ptr, int(n) // per_pe) + int(n) % per_pe * m.page_bytes  # noqa: E731
        for n in around:
            l.fill(where(n), 0xA5, m.page_bytes)
        tokens = 5 * page - 3
        slots = (pages[:, None].astype(np.int64) * page + np.arange(page)).reshape(-1)[:tokens]
        raw, x = values(rng, (tokens, 2 * heads, dim), "bf16", 0.3)
        kv, row, d_slots = d(raw), 2 * heads * dim, d(slots)
        assert l.kv_put(c, L.BF16, kv, row, kv + heads * dim * 2, row, d_slots, tokens, 0, None) == 0
        back = [d.blank(tokens * heads * dim * 2) for _ in range(2)]
        assert l.kv_get(c, L.BF16, back[0], heads * dim, back[1], heads * dim, d_slots, tokens, 0, None) == 0
        q_raw, q = values(rng, (heads, dim), "bf16", 0.3)
        out, lse = d.blank(heads * dim * 4), d.blank(heads * 4)
        nbytes = l.kv_attend_bytes(c, 1, heads, tokens)
        lengths, ws = d(np.array([tokens], np.int32)), d.blank(nbytes)
        assert l.kv_attend(c, L.BF16, d(q_raw), 0, heads, L.FLOAT, out, heads * dim, lse, d(pages), len(pages),
                           lengths, 1, tokens, 0, 0.125, 0.0, 0, ws, nbytes, 0, None) == 0
        l.stream_sync(None)
        for value in (0, 1):
            got = d.read(back[value], tokens * heads * dim * 2).view(np.uint16).reshape(tokens, heads, dim)
            assert np.array_equal(got, raw[:, value * heads:(value + 1) * heads])
        for n in around:
            if n in pages:
                m.raw[:] = 0xA5
                mine = slots // page == n
                m.put(slots[mine] % page, x[mine][:, :heads], x[mine][:, heads:])
                assert np.array_equal(rt.get_bytes(where(n), m.page_bytes), m.raw[0, 0])
            else:
                assert (rt.get_bytes(where(n), m.page_bytes) == 0xA5).all()
        got = d.read(out, heads * dim * 4).view(np.float32).reshape(heads, dim).astype(np.float64)
        for h in range(heads):
            want, _, bound, _ = ref.attend(q[h], x[:, h], x[:, heads + h], 0.125, 0.0)
            assert (np.abs(got[h] - want) <= bound + ref.U["fp32"] * (np.abs(want) + bound)).all()
    finally:
        l.stream_sync(None)
        d.free()
        rt.down()


def test_on_a_cached_heap(rt, L):
    """Rows put by one call and read by the next, again and again to the same
    slots, where the L2s may hold the heap's lines."""
    rt.down()
    os.environ["ROCSHMEM_EMU_HEAP_CACHED"] = "1"
    try:
        l = rt.up(P, HEAP)
        assert l.heap_is_uncached() == 0
        d = Dev(rt)
        r = Run(rt, L, d, "bf16", "e4m3", 2, 4, 64, 16, [1500, 40, 0, 333])
        for step in range(4):
            for b, n in enumerate(r.lengths):
                slots = np.array(ref.tokens_of(int(n), int(n), r.table[b], 16, r.n_pages), np.int64)
                raw, x = values(r.rng, (len(slots), 4, 64), "bf16", 0.3)
                kv = d(raw)
                if len(slots):
                    assert l.kv_put(r.h.as_of(L, b), L.BF16, kv, 256, kv + 256, 256, d(slots), len(slots), b, None) == 0
                r.m.put(slots, x[:, :2], x[:, 2:])
            r.call(pe=step).check()
            r.call(pe=step, own=True).check(owner=step)
        l.stream_sync(None)
        r.free()
        d.free()
    finally:
        rt.down()
        os.environ.pop("ROCSHMEM_EMU_HEAP_CACHED", None)


@pytest.mark.parametrize("npes", [1, 3])
def test_other_numbers_of_pes(rt, L, npes):
    rt.down()
    l = rt.up(npes, HEAP)
    d = Dev(rt)
    try:
        m = ref.Cache("e4m3", npes, 5, 16, 3, 48)
        h = OnHeap(rt, L, m)
        rng = np.random.default_rng(npes)
        slots = rng.permutation(m.slots)[:m.slots - 3].astype(np.int64)
        slots = np.append(slots, m.slots)  # the one that is not there
        raw, x = values(rng, (len(slots), 6, 48), "fp16")
        kv, d_slots = d(raw), d(slots)
        l.kv_refused(1)
        assert l.kv_put(h.as_of(L, npes - 1), L.HALF, kv, 288, kv + 288, 288, d_slots, len(slots), npes - 1, None) == 0
        l.stream_sync(None)
        m.put(slots, x[:, :3], x[:, 3:])
        assert np.array_equal(h.download(), m.raw) and l.kv_refused(1) == 1
        table = rng.permutation(5 * npes).astype(np.int32)
        length = 5 * npes * 16 - 16
        seen = ref.tokens_of(length, length, table, 16, 5 * npes)
        filled = np.isin(seen, slots)
        m.put(np.array(seen)[~filled], np.ones(((~filled).sum(), 3, 48)), np.ones(((~filled).sum(), 3, 48)))
        h.upload()
        q_raw, q = values(rng, (6, 48), "fp16", 0.3)
        out, lse = d.blank(6 * 48 * 4), d.blank(24)
        assert l.kv_attend(h.c, L.HALF, d(q_raw), 0, 6, L.FLOAT, out, 288, lse, d(table), len(table),
                           d(np.array([length], np.int32)), 1, length, 0, 0.1, 0.0, 0, None, 0, 0, None) == 0
        l.stream_sync(None)
        got = d.read(out, 6 * 48 * 4).view(np.float32).reshape(6, 48).astype(np.float64)
        k, v = (m.rows(seen, value) for value in (0, 1))
        for i in range(6):
            want, _, bound, _ = ref.attend(q[i], k[:, i // 2], v[:, i // 2], 0.1, 0.0)
            assert (np.abs(got[i] - want) <= bound + ref.U["fp32"] * (np.abs(want) + bound)).all()
        h.free()
    finally:
        l.stream_sync(None)
        d.free()
        rt.down()


@pytest.mark.parametrize("nprocs", [2, 3])
def test_between_processes(rt, nprocs):
    from rocshmem_amd import launch
    rt.down()
    env = dict(os.environ)
    env.pop("ROCSHMEM_EMU_NPES", None)
    worker = [sys.executable, os.path.join(os.path.dirname(os.path.abspath(__file__)), "kv_procs_worker.py")]
    status, outs = launch.run(nprocs, worker, timeout=100, env=env, capture=True)
    assert status == 0, [o[-1500:] for o in outs]
    for pe, o in enumerate(outs):
        assert "ok %d" % pe in o, o[-1500:]
