"""The key-value cache where PEs' slices lie further apart than they are large
(ROCSHMEM_EMU_SPREAD), with three PEs, so that no stride is a power of two of anything."""
import os

import numpy as np
import pytest

from tests import kv_reference as ref
from tests.test_gpu_kv_cache import Dev, OnHeap, type_of, values

pytestmark = pytest.mark.gpu

NPES, HEAP = 3, 48 << 20


@pytest.mark.parametrize("src,cache", [("bf16", "bf16"), ("fp16", "e4m3")])
def test_on_a_spread_heap(rt, L, src, cache):
    rt.down()
    os.environ["ROCSHMEM_EMU_SPREAD"] = "1"
    try:
        l = rt.up(NPES, HEAP)
        assert l.pe_stride() > l.heap_size()
        d = Dev(rt)
        heads, hq, dim, page, per_pe, length = 3, 6, 48, 32, 11, 900
        rng = np.random.default_rng(8)
        m = ref.Cache(cache, NPES, per_pe, page, heads, dim, fill=0xFF)
        h = OnHeap(rt, L, m)
        n_pages = NPES * per_pe
        table = rng.permutation(n_pages).astype(np.int32)
        slots = np.array(ref.tokens_of(length, length, table, page, n_pages), np.int64)
        raw, x = values(rng, (length, 2 * heads, dim), src, 0.3)
        kv, row, d_slots = d(raw), 2 * heads * dim, d(slots)
        assert l.kv_put(h.as_of(L, 1), type_of(L, src), kv, row, kv + heads * dim * 2, row, d_slots, length, 1, None) == 0
        l.stream_sync(None)
        m.put(slots, x[:, :heads], x[:, heads:])
        assert np.array_equal(h.download(), m.raw)
        back = [d.blank(length * heads * dim * 2) for _ in range(2)]
        assert l.kv_get(h.as_of(L, 2), type_of(L, src), back[0], heads * dim, back[1], heads * dim, d_slots, length, 2,
                        None) == 0
        l.stream_sync(None)
        for value in (0, 1):
            got = d.read(back[value], length * heads * dim * 2).view(np.uint16).reshape(length, heads, dim)
            assert np.array_equal(got, ref.encode(m.rows(slots, value).astype(np.float32), src))
        # every PE over its own pages, joined by each
        q_raw, q = values(rng, (hq, dim), src, 0.3)
        partial, lses = l.malloc(hq * dim * 4), l.malloc(hq * 4)
        nbytes = l.kv_attend_bytes(h.c, 1, hq, length)
        q_dev, d_table, d_len = d(q_raw), d(table), d(np.array([length], np.int32))
        for pe in range(NPES):
            ws = d.blank(nbytes)
            assert l.kv_attend(h.as_of(L, pe), type_of(L, src), q_dev, 0, hq, L.FLOAT, l.pe_ptr(partial, pe), hq * dim,
                               l.pe_ptr(lses, pe), d_table, n_pages, d_len, 1, length, 0, 0.125, 0.0,
                               L.KV_OWN_PAGES, ws, nbytes, pe, None) == 0
        k, v = (m.rows(slots, value) for value in (0, 1))
        for pe in range(NPES):
            out, lse = d.blank(hq * dim * 4), d.blank(hq * 4)
            assert l.kv_join(L.FLOAT, l.pe_ptr(partial, pe), l.pe_ptr(lses, pe), hq, dim, L.FLOAT, out, lse, 0, 0, NPES,
                             pe, None) == 0
            l.stream_sync(None)
            got = d.read(out, hq * dim * 4).view(np.float32).reshape(hq, dim).astype(np.float64)
            got_lse = d.read(lse, hq * 4).view(np.float32)
            for i in range(hq):  # (the join's few roundings are far inside the bound for the sums over the tokens)
                want, want_lse, bound, dlse = ref.attend(q[i], k[:, i // 2], v[:, i // 2], 0.125, 0.0)
                assert (np.abs(got[i] - want) <= bound + ref.U["fp32"] * (np.abs(want) + bound)).all()
                assert abs(got_lse[i] - want_lse) <= dlse
        l.free(partial)
        l.free(lses)
        h.free()
        d.free()
    finally:
        l.stream_sync(None)
        rt.down()
        os.environ.pop("ROCSHMEM_EMU_SPREAD", None)
