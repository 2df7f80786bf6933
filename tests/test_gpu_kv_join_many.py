"""The join of more members than its kernel has on their way at once (two,
four or eight): where the largest lse comes late, batches without tokens,
strided active sets."""
import numpy as np
import pytest

from tests import kv_reference as ref
from tests.test_gpu_kv_cache import HEAP, Dev, type_of, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("npes", [5, 8, 9, 16])
@pytest.mark.parametrize("src,out", [("fp32", "bf16"), ("bf16", "fp32"), ("fp16", "fp16")])
def test_join_of_many_members(rt, L, npes, src, out):
    rt.down()
    l = rt.up(npes, HEAP // 4)
    d = Dev(rt)
    try:
        rows, dim, es = 70, 72, ref.SIZE[src]
        rng = np.random.default_rng([npes, es])
        partial, lses = l.malloc(rows * dim * es), l.malloc(rows * 4)
        raw, x = values(rng, (npes, rows, dim), src)
        lse = (rng.standard_normal((npes, rows)) * 3 + 5).astype(np.float32)
        lse[rng.random((npes, rows)) < 0.2] = -np.inf
        lse[:, 0] = np.linspace(-10, 10, npes)          # the largest last
        lse[:, 1] = np.linspace(10, -10, npes)          # and first
        lse[:-1, 2], lse[-1, 2] = -np.inf, 3.0          # the last member's tokens only
        lse[:8, 3] = -np.inf                            # nothing in the first eight
        lse[-max(1, npes - 8):, 4] = -np.inf            # nothing behind them
        lse[:, 5] = -np.inf                             # nothing at all
        lse[:-1, 6], lse[-1, 6] = -200.0, 200.0         # all weight on the last
        raw[np.isneginf(lse)] = np.uint32(0xFFFFFFFF).astype(raw.dtype) if es == 4 else 0xFFFF  # NaN where nothing counts
        for pe in range(npes):
            rt.put_bytes(l.pe_ptr(partial, pe), raw[pe])
            rt.put_bytes(l.pe_ptr(lses, pe), lse[pe])
        sets = [(0, 0, npes), (1, 0, npes - 1), (0, 1, (npes + 1) // 2), (1, 1, npes // 2), (npes - 5, 0, 5)]
        for first, log_stride, size in sets:
            pes = [first + (i << log_stride) for i in range(size)]
            want, want_lse, around = ref.join(x[pes], lse[pes].astype(np.float64))
            o, s = d.blank(rows * dim * ref.SIZE[out]), d.blank(rows * 4)
            my_pe = npes - 1
            assert l.kv_join(type_of(L, src), l.pe_ptr(partial, my_pe), l.pe_ptr(lses, my_pe), rows, dim,
                             type_of(L, out), o, s, first, log_stride, size, my_pe, None) == 0
            l.stream_sync(None)
            got = ref.decode(d.read(o, rows * dim * ref.SIZE[out]).view({2: np.uint16, 4: np.uint32}[ref.SIZE[out]]),
                             out).reshape(rows, dim)
            got_lse = d.read(s, rows * 4).view(np.float32).astype(np.float64)
            none = np.isneginf(want_lse)
            assert np.array_equal(np.isneginf(got_lse), none) and none[5]
            assert (got[none] == 0).all()
            # a weight: the difference of two lse's rounds to 2^-24 of at most 25 (beyond,
            # the weight is below 2^-36 of the whole), times log2 e to as much, the
            # exponential 2^-22, twice with a second batch; sums of up to 16 terms, a
            # quotient and a product, each 2^-24
            dw = 2 * (25 * 2.0 ** -23 + 2.0 ** -22)
            bound = 2 * dw * around + (2 * size + 4) * 2.0 ** -24 * around + 2.0 ** -32 * np.abs(x[pes]).max()
            off = np.abs(got - want) - ref.U[out] * (np.abs(want) + bound) - ref.LEAST[out]
            assert (off <= bound)[~none].all(), (first, log_stride, size)
            # the same and a logarithm (2^-22 of up to log2(16)), and the last sum
            assert (np.abs(got_lse - want_lse)[~none] <= dw + size * 2.0 ** -24 + 2.0 ** -20 +
                    np.abs(want_lse[~none]) * 2.0 ** -23).all()
        l.free(partial)
        l.free(lses)
    finally:
        l.stream_sync(None)
        d.free()
        rt.down()
