"""What the key-value cache's attention holds in 32 bits, and a NaN on its way
through out, lse and join.  Where tolerances are stated scores are exact (queries
and keys with one element that is not 0), so that they count the roundings of
one quantity at a time, each 2^-24 of it at most unless said otherwise."""
import numpy as np
import pytest

from tests import kv_reference as ref
from tests.test_gpu_kv_cache import HEAP, P, Dev, OnHeap, dev, type_of  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "e4m3")]
HALF_STEP = 2.0 ** -24


class Given:
    """Sequences with given keys and values, [b] -> [tokens, dim], one cache head."""

    def __init__(self, rt, L, dev, src, cache, keys, values, page=16):
        self.l, self.L, self.dev, self.src = rt.l, L, dev, src
        dim = keys[0].shape[1]
        need = [-(-len(k) // page) for k in keys]
        per_pe = -(-sum(need) // P)
        self.m = ref.Cache(cache, P, per_pe, page, 1, dim, fill=0xFF)
        self.table = np.full((len(keys), max(need)), -1, np.int32)
        self.lengths = np.array([len(k) for k in keys], np.int32)
        order = np.random.default_rng(len(keys)).permutation(P * per_pe)
        at = 0
        for b, (k, v) in enumerate(zip(keys, values)):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            slots = ref.tokens_of(len(k), len(k), self.table[b], page, P * per_pe)
            self.m.put(slots, k[:, None], v[:, None])
        self.h = OnHeap(rt, L, self.m)
        self.dim = dim

    def attend(self, q, scale=1.0, softcap=0.0, own_of=None):
        """q: [sequences, heads, dim], values that the type holds; fp32 results."""
        l, n, hq = self.l, len(self.lengths), q.shape[1]
        bound = int(self.lengths.max())
        out, lse = self.dev.blank(n * hq * self.dim * 4), self.dev.blank(n * hq * 4)
        nbytes = l.kv_attend_bytes(self.h.c, n, hq, bound)
        pe = own_of or 0
        raw = ref.encode(q.astype(np.float32), self.src)
        assert np.array_equal(ref.decode(raw, self.src), q)
        assert l.kv_attend(self.h.as_of(self.L, pe), type_of(self.L, self.src), self.dev(raw), hq * self.dim, hq,
                           self.L.FLOAT, out, hq * self.dim, lse, self.dev(self.table), self.table.shape[1],
                           self.dev(self.lengths), n, bound, 0, scale, softcap, 0 if own_of is None else 1,
                           self.dev.blank(nbytes), nbytes, pe, None) == 0
        l.stream_sync(None)
        return (self.dev.read(out, n * hq * self.dim * 4).view(np.float32).reshape(n, hq, self.dim).astype(np.float64),
                self.dev.read(lse, n * hq * 4).view(np.float32).reshape(n, hq).astype(np.float64))


def held(x, name):
    """The nearest values that a format holds."""
    return ref.decode(ref.encode(np.asarray(x, np.float32), name), name)


@pytest.mark.parametrize("src,cache", TYPES)
def test_weights_keep_32_bits(rt, L, dev, src, cache):
    """Two tokens, one with score 0 and one with -x, values 1 in a column each:
    out is 1 / (1 + w) and w / (1 + w) with w = exp(-x)."""
    n, hq, dim, dim_v = 24, 32, 16, 16
    rng = np.random.default_rng(6)
    x = held(rng.uniform(0.01, 3.0, (n, hq)), "bf16")
    x = held(x, src)
    k, v = np.zeros((2, dim)), np.zeros((2, dim_v))
    k[1, 0], v[0, 3], v[1, 5] = -1.0, 1.0, 1.0
    g = Given(rt, L, dev, src, cache, [k] * n, [v] * n)
    q = np.zeros((n, hq, dim))
    q[..., 0] = x
    out, lse = g.attend(q)
    w = np.exp(-x)
    # w: its argument by two roundings (log2 e, the product) of x each, the exponential 2;
    # a weight kept as two 16-bit parts of fp16 another 4.  out: the sums over the
    # tokens and of the weights, up to 4 additions each, a quotient (2) and a product.
    of_w = (2 * x + 2 + (4 if cache == "fp16" else 0)) * HALF_STEP
    bound = of_w + 11 * HALF_STEP
    assert (np.abs(out[..., 5] / (w / (1 + w)) - 1) <= bound).all(), np.abs(out[..., 5] / (w / (1 + w)) - 1).max()
    assert (np.abs(out[..., 3] / (1 / (1 + w)) - 1) <= bound).all()
    # log(1 + w) <= log 2: the sum's roundings, the logarithm's 2^-22, and (fp16: weights
    # lie 2^7 above the exponentials) a sum of at most 8
    assert (np.abs(lse - np.log1p(w)) <= of_w + 2.0 ** -21 + (8 * 2.0 ** -23 if cache == "fp16" else 0)).all()
    rest = np.delete(out, (3, 5), axis=-1)
    assert (rest == 0).all()
    g.h.free()


def one_token_each(rt, L, dev, src, cache):
    """Sequences of one token whose scores are 1280 values from 2^-10 to 3008 of
    either sign: (sequences, queries, scores, the tokens' value as it is held)."""
    n, hq, dim = 32, 40, 16
    s = np.exp(np.linspace(np.log(2.0 ** -10), np.log(3e3), n * hq // 2))
    s = held(held(np.stack([s, -s]), "bf16"), src).reshape(n, hq)
    k = np.zeros((1, dim))
    k[0, 0] = 1.0
    v = held(np.random.default_rng(1).standard_normal((1, dim)), "bf16")
    v[:, 0] = 2.0
    g = Given(rt, L, dev, src, cache, [k] * n, [v] * n)
    q = np.zeros((n, hq, dim))
    q[..., 0] = s
    return g, q, s, g.m.rows(ref.tokens_of(1, 1, g.table[0], 16, 1 << 20), 1)[0, 0]


@pytest.mark.parametrize("src,cache", TYPES)
def test_caps_up_to_the_largest(rt, L, dev, src, cache):
    """A cap near or at the largest 32-bit value is none."""
    g, q, s, v = one_token_each(rt, L, dev, src, cache)
    for cap in (2.3e38, 2.4e38, float(np.finfo(np.float32).max)):
        cap = float(np.float32(cap))
        out, lse = g.attend(q, softcap=cap)
        # a few roundings, of a quotient by the cap (below the normal numbers: of 2^-149),
        # products by it and by log2 e and ln 2; fp16 caches add and take off 7
        bound = 16 * HALF_STEP * np.abs(s) + 2.0 ** -149 * cap + (8 * 2.0 ** -23 if cache == "fp16" else 0)
        assert (np.abs(lse - s) <= bound).all(), cap
        assert (np.abs(out - v) <= 4 * HALF_STEP * np.abs(v)).all(), cap
    g.h.free()


@pytest.mark.parametrize("src,cache", TYPES)
def test_capped_scores_keep_32_bits(rt, L, dev, src, cache):
    g, q, s, v = one_token_each(rt, L, dev, src, cache)
    for cap in (2.0 ** -100, 1e-3, 1.0, 20.0, 30.0, 50.0, 63.0, 65.0, 1000.0, 1e30, 2.4e38,
                float(np.finfo(np.float32).max)):
        cap = float(np.float32(cap))
        out, lse = g.attend(q, softcap=cap)
        want = cap * np.tanh(s / cap)
        # The quotient by the cap 2, which tanh passes on by at most 0.8 of that; tanh
        # by an exponential and a reciprocal 6, by a polynomial less; the factors log2 e,
        # cap and ln 2 with their products 4: 12, and 16 allowed.
        bound = 16 * HALF_STEP * np.abs(want)
        if cache == "fp16":  # weights lie 2^7 above the exponentials: 7 is taken off and added again
            bound = bound + 8 * 2.0 ** -23
        off = np.abs(lse - want)
        assert (off <= bound).all(), (cap, float((off / bound).max()), s.ravel()[(off / bound).argmax()])
        assert (np.abs(out - v) <= 4 * HALF_STEP * np.abs(v)).all(), cap  # its only token's value
    g.h.free()


@pytest.mark.parametrize("src,cache", TYPES)
def test_a_nan_score_reaches_out_and_lse(rt, L, dev, src, cache):
    """A sequence with NaN among the scores of its tokens, or with nothing else,
    is NaN in out and in lse, so that a join does not take it for one without
    tokens; its neighbours are not."""
    rng, dim = np.random.default_rng(2), 32
    lengths = [1, 1, 40, 40, 40, 900, 900, 2000, 17]
    bad = [[0], [], range(40), [39], [], range(900), [450], [], range(17)]
    keys = [held(rng.standard_normal((n, dim)), "bf16") for n in lengths]
    values = [held(rng.standard_normal((n, dim)), "bf16") for n in lengths]
    for k, at in zip(keys, bad):
        k[list(at), 3] = np.nan
    g = Given(rt, L, dev, src, cache, keys, values)
    q = held(held(rng.standard_normal((len(lengths), 3, dim)), "bf16"), src)
    spoiled = np.array([len(at) > 0 for at in bad])
    for softcap in (0.0, 20.0):
        out, lse = g.attend(q, scale=0.25, softcap=softcap)
        assert np.isnan(out[spoiled]).all() and np.isnan(lse[spoiled]).all(), lse
        assert np.isfinite(out[~spoiled]).all() and np.isfinite(lse[~spoiled]).all()
    # each PE over its own pages, and the join of all
    l, n = rt.l, len(lengths) * 3
    partial, lses = l.malloc(n * dim * 4), l.malloc(n * 4)
    for pe in range(P):
        out, lse = g.attend(q, scale=0.25, own_of=pe)
        rt.put_bytes(l.pe_ptr(partial, pe), out.astype(np.float32))
        rt.put_bytes(l.pe_ptr(lses, pe), lse.astype(np.float32))
    o, s = dev.blank(n * dim * 4), dev.blank(n * 4)
    assert l.kv_join(L.FLOAT, partial, lses, n, dim, L.FLOAT, o, s, 0, 0, P, 0, None) == 0
    l.stream_sync(None)
    out = dev.read(o, n * dim * 4).view(np.float32).reshape(-1, 3, dim)
    lse = dev.read(s, n * 4).view(np.float32).reshape(-1, 3)
    assert np.isnan(out[spoiled]).all() and np.isnan(lse[spoiled]).all()
    assert np.isfinite(out[~spoiled]).all() and np.isfinite(lse[~spoiled]).all()
    l.free(partial)
    l.free(lses)
    g.h.free()
