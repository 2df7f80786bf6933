"""The key-value cache on the symmetric heap (include/rocshmem_amd.h,
rocshmem_amd_kv_*): rows put and read back bit for bit, attention of one new
token and the join of partial results against a 64-bit computation in numpy
(tests/kv_reference.py), with the tolerance of every value derived there."""
import ctypes as C

import numpy as np
import pytest

from tests import kv_reference as ref

pytestmark = pytest.mark.gpu

P, HEAP = 4, 64 << 20
GUARD = 256


def type_of(L, name):
    return {"bf16": L.BF16, "fp16": L.HALF, "fp32": L.FLOAT, "e4m3": L.E4M3}[name]


class OnHeap:
    """A ref.Cache's bytes on the symmetric heap, with guard bytes behind them."""

    def __init__(self, rt, L, model):
        self.rt, self.l, self.m = rt, rt.l, model
        self.n = model.raw[0].nbytes
        self.ptr = self.l.malloc(self.n + GUARD)
        assert self.ptr
        assert self.l.kv_page_bytes(type_of(L, model.dtype), model.page, model.heads, model.dim) == model.page_bytes
        self.c = L.KvCache(pages=self.ptr, dtype=type_of(L, model.dtype), pages_per_pe=model.pages_per_pe,
                           page_tokens=model.page, kv_heads=model.heads, head_dim=model.dim)
        self.upload()

    def upload(self):
        for p in range(self.m.npes):
            self.l.fill(self.l.pe_ptr(self.ptr, p), 0x5B, self.n + GUARD)
            self.rt.put_bytes(self.l.pe_ptr(self.ptr, p), self.m.raw[p])

    def as_of(self, L, pe):
        """The same cache as PE `pe` names it."""
        c = self.c
        return L.KvCache(pages=self.l.pe_ptr(self.ptr, pe), dtype=c.dtype, pages_per_pe=c.pages_per_pe,
                         page_tokens=c.page_tokens, kv_heads=c.kv_heads, head_dim=c.head_dim)

    def download(self):
        got = np.stack([self.rt.get_bytes(self.l.pe_ptr(self.ptr, p), self.n + GUARD) for p in range(self.m.npes)])
        assert (got[:, self.n:] == 0x5B).all(), "wrote past the cache"
        return got[:, :self.n].reshape(self.m.raw.shape)

    def free(self):
        self.l.free(self.ptr)


class Dev:
    """Device buffers that a test frees together."""

    def __init__(self, rt):
        self.rt, self.ptrs = rt, []

    def __call__(self, array):
        self.ptrs.append(self.rt.dev_array(array))
        return self.ptrs[-1]

    def blank(self, nbytes):
        """nbytes of 0x77 between guards of the same."""
        return self(np.full(nbytes + 2 * GUARD, 0x77, np.uint8)) + GUARD

    def read(self, ptr, nbytes):
        got = self.rt.get_bytes(ptr - GUARD, nbytes + 2 * GUARD)
        assert (got[:GUARD] == 0x77).all() and (got[GUARD + nbytes:] == 0x77).all(), "wrote outside the buffer"
        return got[GUARD:GUARD + nbytes]

    def free(self):
        for p in self.ptrs:
            self.rt.l.dev_free(p)


@pytest.fixture
def dev(rt):
    rt.up(P, HEAP)
    d = Dev(rt)
    yield d
    rt.l.stream_sync(None)
    d.free()


def values(rng, shape, name, spread=1.0):
    """Random values that the format holds, sizes differing from row to row: (raw integers, 64-bit values)."""
    x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal(shape[:-1] + (1,)))
    raw = ref.encode(x.astype(np.float32), name)
    return raw, ref.decode(raw, name)


# ---------------------------------------------------------------- put and get

ROWS = [  # source, cache, tokens, heads, dim, page, pages per PE, extra elements between tokens
    ("bf16", "bf16", 1, 1, 16, 16, 1, 0),
    ("bf16", "bf16", 37, 3, 128, 64, 2, 24),
    ("fp16", "fp16", 130, 5, 96, 48, 3, 8),
    ("fp16", "bf16", 20, 2, 64, 16, 2, 0),
    ("fp32", "fp16", 20, 2, 256, 16, 1, 4),
    ("bf16", "e4m3", 61, 4, 128, 32, 2, 40),
    ("fp16", "e4m3", 33, 3, 80, 16, 3, 1),
    ("fp32", "e4m3", 100, 1, 256, 112, 1, 3),
    ("fp32", "e4m3", 5, 7, 16, 16, 1, 0),
    ("bf16", "e4m3", 700, 8, 128, 64, 4, 0),
]


@pytest.mark.parametrize("src,cache,tokens,heads,dim,page,pages,extra", ROWS)
def test_put_writes_its_rows_and_nothing_else(rt, L, dev, src, cache, tokens, heads, dim, page, pages, extra):
    l, rng = rt.l, np.random.default_rng([tokens, heads, dim])
    m = ref.Cache(cache, P, pages, page, heads, dim)
    h = OnHeap(rt, L, m)
    es, row = ref.SIZE[src], heads * dim + extra
    slots = rng.permutation(m.slots)[:tokens].astype(np.int64)
    slots[2::5] = -1
    if tokens > 4:
        slots[1], slots[3] = m.slots, -7      # out of range: left out and counted
    raw, x = zip(*(values(rng, (tokens, row), src) for _ in range(2)))
    x = [a[:, :heads * dim].reshape(tokens, heads, dim) for a in x]
    ptr = [dev(np.concatenate([np.zeros(3, a.dtype), a.reshape(-1)])) + 3 * es for a in raw]  # an odd start
    for pe in (0, P - 1):
        h.upload()
        l.kv_refused(1)
        assert l.kv_put(h.as_of(L, pe), type_of(L, src), ptr[0], row, ptr[1], row, dev(slots), tokens, pe, None) == 0
        l.stream_sync(None)
        want = ref.Cache(cache, P, pages, page, heads, dim)
        want.put(slots, *x)
        assert np.array_equal(h.download(), want.raw)
        assert l.kv_refused(1) == (2 if tokens > 4 else 0) and l.kv_refused(0) == 0
    h.free()


@pytest.mark.parametrize("dst,cache,tokens,heads,dim,page,pages,extra", ROWS)
def test_get_reads_rows_back_and_leaves_the_others(rt, L, dev, dst, cache, tokens, heads, dim, page, pages, extra):
    l, rng = rt.l, np.random.default_rng([tokens, heads, dim, 1])
    m = ref.Cache(cache, P, pages, page, heads, dim)
    all_slots = np.arange(m.slots)
    m.put(all_slots, *(values(rng, (m.slots, heads, dim), "fp32" if cache == "e4m3" else cache)[1] for _ in range(2)))
    h = OnHeap(rt, L, m)
    es, row = ref.SIZE[dst], heads * dim + extra
    slots = rng.integers(0, m.slots, tokens).astype(np.int64)  # reading a slot twice is fine
    slots[2::5] = -1
    if tokens > 4:
        slots[1], slots[3] = 1 << 40, -(1 << 40)
    out = [dev.blank(tokens * row * es) for _ in range(2)]
    l.kv_refused(1)
    assert l.kv_get(h.as_of(L, 1), type_of(L, dst), out[0], row, out[1], row, dev(slots), tokens, 1, None) == 0
    l.stream_sync(None)
    assert l.kv_refused(1) == (2 if tokens > 4 else 0)
    good = (slots >= 0) & (slots < m.slots)
    for value in (0, 1):
        raw = dev.read(out[value], tokens * row * es).view({2: np.uint16, 4: np.uint32}[es]).reshape(tokens, row)
        blank = np.full(row, 0x77777777, np.uint32).view(raw.dtype)[:row]
        assert (raw[~good] == blank).all() and (raw[:, heads * dim:] == blank[heads * dim:]).all()
        x = m.rows(slots[good], value).reshape(-1, heads * dim)
        assert np.array_equal(raw[good][:, :heads * dim], ref.encode(x.astype(np.float32), dst))
    h.free()


def test_e4m3_rows_at_the_edges_of_the_format(rt, L, dev):
    """Zeros, a single tiny value, the border of a scale (448 and its
    neighbours), ties between codes, the largest and smallest magnitudes of
    32 bits, infinities and NaN beside ordinary values."""
    l, dim = rt.l, 32
    rows = [np.zeros(dim), np.r_[2.0 ** -149, np.zeros(dim - 1)], np.r_[2.0 ** -126, 2.0 ** -130, np.zeros(dim - 2)]]
    for top in (448.0, np.nextafter(np.float32(448), np.float32(500)), 449.0, 447.9, 1.75, 1.7500001, 3.4e38, 1e-37, 7.0 * 2 ** -127):
        r = np.linspace(-1, 1, dim) * top
        r[0] = top
        rows.append(r)
    ties = np.array([17, 18, 19, 21, 23, 25, 27, 29, 31, 8.5, 9.5, 1.0625, 1.1875]) / 16
    rows.append(np.r_[448.0, ties, -ties, np.zeros(dim - 1 - 2 * len(ties))])
    rows.append(np.r_[448.0, np.arange(1, 16) * 2.0 ** -10, np.zeros(dim - 16)])  # around the smallest code
    rows.append(np.r_[np.inf, 3.0, -np.inf, np.nan, 1e-3, np.zeros(dim - 5)])
    rows.append(np.full(dim, np.nan))
    rows.append(np.full(dim, -np.inf))
    x = np.array(rows, np.float32)
    m = ref.Cache("e4m3", P, 1, 16, 1, dim)
    h = OnHeap(rt, L, m)
    slots = np.arange(len(x), dtype=np.int64) + 5
    kv = dev(x)
    assert l.kv_put(h.c, L.FLOAT, kv, dim, kv, dim, dev(slots), len(x), 0, None) == 0
    out = [dev.blank(x.nbytes) for _ in range(2)]
    assert l.kv_get(h.c, L.FLOAT, out[0], dim, out[1], dim, dev(slots), len(x), 0, None) == 0
    l.stream_sync(None)
    m.put(slots, *(x.astype(np.float64)[:, None],) * 2)
    got = h.download()
    nan_codes = (m.raw & 127) == 127  # the sign of a NaN is not said
    codes = np.zeros(m.raw.shape, bool)
    codes[..., :2 * m.part] = True
    loose = nan_codes & codes
    assert np.array_equal(got[~loose], m.raw[~loose]) and ((got[loose] & 127) == 127).all()
    for value in (0, 1):
        y = dev.read(out[value], x.nbytes).view(np.float32).reshape(x.shape)
        want = m.rows(slots, value)[:, 0]
        assert np.array_equal(np.isnan(y), np.isnan(want)) and np.array_equal(np.isnan(y), ~np.isfinite(x))
        fine = np.isfinite(x)
        with np.errstate(over="ignore"):  # a code may stand for slightly more than 32 bits hold
            assert np.array_equal(y[fine], want[fine].astype(np.float32))
    h.free()


def test_put_of_no_tokens_does_nothing(rt, L, dev):
    l = rt.l
    m = ref.Cache("bf16", P, 1, 16, 1, 16)
    h = OnHeap(rt, L, m)
    assert l.kv_put(h.c, L.BF16, None, 0, None, 0, None, 0, 0, None) == 0
    assert l.kv_get(h.c, L.BF16, None, 0, None, 0, None, 0, 0, None) == 0
    l.stream_sync(None)
    assert np.array_equal(h.download(), m.raw)
    h.free()


def test_a_source_row_may_serve_every_token(rt, L, dev):
    """A stride of 0 puts one row to many slots."""
    l, rng = rt.l, np.random.default_rng(3)
    m = ref.Cache("fp16", P, 1, 16, 2, 48)
    h = OnHeap(rt, L, m)
    raw, x = values(rng, (1, 96), "fp16")
    slots = np.arange(40, dtype=np.int64)
    p = dev(raw)
    assert l.kv_put(h.c, L.HALF, p, 0, p, 0, dev(slots), 40, 0, None) == 0
    l.stream_sync(None)
    x = np.broadcast_to(x.reshape(1, 2, 48), (40, 2, 48))
    m.put(slots, x, x)
    assert np.array_equal(h.download(), m.raw)
    h.free()


# ------------------------------------------------------------------- attention

class Run:
    """A cache with sequences in it, and a call of kv_attend on them."""

    def __init__(self, rt, L, dev, src, cache, heads, group, dim, page, lengths, max_len=None, seed=0, spread=0.3,
                 gain=1.0):
        self.rt, self.l, self.L, self.dev, self.src = rt, rt.l, L, dev, src
        rng = self.rng = np.random.default_rng([seed, heads, group, dim, page, len(lengths)])
        self.lengths = np.array(lengths, np.int32)
        self.max_len = max(max(lengths), 0) if max_len is None else max_len
        each = max(1, -(-max(max(lengths), 1) // page))
        used = sum(-(-max(n, 0) // page) for n in lengths)
        per_pe = -(-max(used, 1) // P)
        self.m = ref.Cache(cache, P, per_pe, page, heads, dim, fill=0xFF)  # 0xFF: NaN in every format
        order = rng.permutation(P * per_pe)
        self.table = np.full((len(lengths), each), -1, np.int32)
        at = 0
        for b, n in enumerate(lengths):
            need = -(-max(n, 0) // page)
            self.table[b, :need] = order[at:at + need]
            at += need
        self.n_pages = P * per_pe
        # only the tokens that exist are written: all else stays NaN
        for b, n in enumerate(lengths):
            slots = ref.tokens_of(n, n, self.table[b], page, self.n_pages)
            kv = [values(rng, (len(slots), heads, dim), src, spread)[1] for _ in range(2)]
            self.m.put(slots, *kv)
        self.heads, self.group, self.dim = heads, group, dim
        q_raw, q = values(rng, (len(lengths), heads * group + 3, dim), src, spread)
        self.q_raw, self.q = q_raw, q * 1.0
        if gain != 1.0:
            self.q_raw = ref.encode((q * gain).astype(np.float32), src)
            self.q = ref.decode(self.q_raw, src)
        self.h = OnHeap(rt, L, self.m)

    def call(self, window=0, softcap=0.0, out="same", scale=None, pe=0, own=False, stream=None, out_extra=0,
             workspace=None):
        L, l, n = self.L, self.l, len(self.lengths)
        self.out_type = self.src if out == "same" else out
        self.window, self.softcap, self.scale = window, softcap, self.dim ** -0.5 if scale is None else scale
        hq = self.heads * self.group
        es = ref.SIZE[self.out_type]
        self.out_row = hq * self.dim + out_extra
        self.out = self.dev.blank(n * self.out_row * es)
        self.lse = self.dev.blank(n * hq * 4)
        nbytes = l.kv_attend_bytes(self.h.c, n, hq, self.max_len)
        ws = self.dev.blank(nbytes) if workspace is None else workspace
        rc = l.kv_attend(self.h.as_of(L, pe), type_of(L, self.src), self.dev(self.q_raw), self.q_raw.shape[1] * self.dim,
                         hq, type_of(L, self.out_type), self.out, self.out_row, self.lse, self.dev(self.table),
                         self.table.shape[1], self.dev(self.lengths), n, self.max_len, window, self.scale, softcap,
                         L.KV_OWN_PAGES if own else L.KV_ALL_PAGES, ws, nbytes, pe, stream)
        assert rc == 0
        self.ws, self.ws_bytes = ws, nbytes
        return self

    def got(self):
        n, hq, es = len(self.lengths), self.heads * self.group, ref.SIZE[self.out_type]
        raw = self.dev.read(self.out, n * self.out_row * es).view({2: np.uint16, 4: np.uint32}[es])
        raw = raw.reshape(n, self.out_row)
        assert (raw[:, hq * self.dim:].reshape(-1).view(np.uint8) == 0x77).all(), "wrote between the rows"
        self.dev.read(self.ws, self.ws_bytes)
        return (ref.decode(raw[:, :hq * self.dim], self.out_type).reshape(n, hq, self.dim),
                self.dev.read(self.lse, n * hq * 4).view(np.float32).astype(np.float64).reshape(n, hq))

    def check(self, owner=None):
        """Every value within its bound; owner: only that PE's pages take part."""
        self.l.stream_sync(None)
        out, lse = self.got()
        u = ref.U[self.out_type]
        for b, n in enumerate(self.lengths):
            slots = ref.tokens_of(int(n), self.max_len, self.table[b], self.m.page, self.n_pages, self.window)
            if owner is not None:
                slots = [s for s in slots if self.m.where(s)[0][0] == owner]
            k, v = (self.m.rows(slots, value) for value in (0, 1))
            for h in range(self.heads * self.group):
                c = h // self.group
                want, want_lse, d, dlse = ref.attend(self.q[b, h], k[:, c], v[:, c], self.scale, self.softcap)
                bound = d + u * (np.abs(want) + d) + ref.LEAST[self.out_type]
                off = np.abs(out[b, h] - want)
                assert (off <= bound).all(), (b, h, int(n), float(np.max(off / bound)))
                if not slots:
                    assert lse[b, h] == -np.inf and (out[b, h] == 0).all()
                else:
                    assert abs(lse[b, h] - want_lse) <= dlse, (b, h, lse[b, h], want_lse, dlse)
        return self

    def free(self):
        self.h.free()


ATTEND = [  # source, cache, cache heads, query heads each, dim, page, lengths
    ("bf16", "bf16", 1, 1, 16, 16, [1]),
    ("bf16", "bf16", 2, 4, 128, 64, [0, 1, 15, 16, 17, 63, 64, 65, 129, 500]),
    ("fp16", "fp16", 3, 1, 64, 16, [31, 32, 33, 0, 200]),
    ("fp16", "fp16", 1, 16, 96, 48, [47, 48, 49, 300, 5]),
    ("bf16", "bf16", 1, 17, 80, 80, [81, 7]),
    ("bf16", "bf16", 1, 33, 256, 32, [70, 257]),
    ("bf16", "bf16", 1, 71, 64, 16, [100]),
    ("bf16", "e4m3", 2, 8, 128, 32, [1, 31, 33, 400, 0, 64]),
    ("fp16", "e4m3", 2, 6, 256, 48, [95, 96, 97, 2]),
    ("fp16", "e4m3", 1, 40, 112, 16, [150, 33]),
    ("bf16", "e4m3", 5, 1, 48, 16, [3, 130]),
    ("bf16", "e4m3", 1, 64, 16, 16, [257]),
    ("bf16", "bf16", 1, 8, 128, 128, [3001]),
    ("fp16", "e4m3", 1, 4, 64, 64, [5003, 20, 2500]),
]


@pytest.mark.parametrize("src,cache,heads,group,dim,page,lengths", ATTEND)
def test_attention_of_one_token(rt, L, dev, src, cache, heads, group, dim, page, lengths):
    r = Run(rt, L, dev, src, cache, heads, group, dim, page, lengths)
    r.call(out_extra=5).check()
    r.call(out="fp32", pe=P - 1).check()
    rt.l.kv_refused(1)
    r.call(softcap=5.0).check()
    longest = max(lengths)
    for window in {1, 16, 33, max(1, longest - 1), longest + 10}:
        r.call(window=window, softcap=0.0).check()
    assert rt.l.kv_refused(1) == 0
    r.free()


@pytest.mark.parametrize("src,cache", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "e4m3")])
def test_attention_whose_weights_are_anything_but_even(rt, L, dev, src, cache):
    """Large queries: a few tokens take all the weight, the maximum moves along the row."""
    r = Run(rt, L, dev, src, cache, 2, 5, 64, 16, [700, 65, 40], spread=0.7, gain=8.0)
    r.call().check()
    r.call(out="fp32", softcap=30.0).check()
    r.call(scale=-0.1).check()
    r.call(scale=0.0).check()
    r.free()


@pytest.mark.parametrize("src,cache", [("bf16", "bf16"), ("fp16", "e4m3")])
def test_pes_attend_to_their_own_pages_and_the_results_are_joined(rt, L, dev, src, cache):
    """Every PE over its own share of the tokens, the joined result against all
    of them: sequences whose pages all lie on one PE among them."""
    l = rt.l
    r = Run(rt, L, dev, src, cache, 2, 4, 64, 16, [300, 1, 0, 16, 77])
    rows, dim = 5 * 8, 64
    partial, lses = l.malloc(rows * dim * 4), l.malloc(rows * 4)
    for pe in range(P):
        r.call(pe=pe, own=True, out="fp32").check(owner=pe)
        assert l.copy_dev(l.pe_ptr(partial, pe), r.out, rows * dim * 4) == 0
        assert l.copy_dev(l.pe_ptr(lses, pe), r.lse, rows * 4) == 0
    for pe in (0, P - 1):
        r.out_type, r.out_row = r.src, 8 * dim
        r.out, r.lse = dev.blank(rows * dim * 2), dev.blank(rows * 4)
        assert l.kv_join(L.FLOAT, l.pe_ptr(partial, pe), l.pe_ptr(lses, pe), rows, dim, type_of(L, src), r.out, r.lse,
                         0, 0, P, pe, None) == 0
        # the join's own arithmetic is a few roundings of 2^-24: far inside the
        # bound that check() allows for the sums over the tokens
        r.check()
    l.free(partial)
    l.free(lses)
    r.free()


def test_pages_and_lengths_out_of_range_are_left_out_and_counted(rt, L, dev):
    l = rt.l
    r = Run(rt, L, dev, "bf16", "bf16", 2, 2, 32, 16, [100, 50, 33])
    r.table[0, 2], r.table[0, 5], r.table[1, 0] = r.n_pages, -1, 1 << 30
    l.kv_refused(1)
    r.call().check()
    assert l.kv_refused(1) == 3
    r.table[1, :] = -5
    r.call().check()
    assert l.kv_refused(1) == 2 + 4  # the second sequence has four pages
    r.call(window=10).check()
    assert l.kv_refused(1) == 1 + 2  # only what the window touches: tokens 90 to 99 and 40 to 49
    r.free()
    r = Run(rt, L, dev, "bf16", "e4m3", 1, 2, 32, 16, [112, 50, 33])
    r.lengths = np.array([1 << 30, -3, 33], np.int32)
    r.max_len = 40
    l.kv_refused(1)
    r.call().check()
    assert l.kv_refused(1) == 2
    r.max_len = 2000  # more than the table holds: 7 pages
    r.lengths = np.array([1999, 50, 33], np.int32)
    r.call().check()
    assert l.kv_refused(1) == 1
    r.free()


def test_attention_without_lse_and_without_sequences(rt, L, dev):
    l = rt.l
    r = Run(rt, L, dev, "bf16", "bf16", 1, 2, 32, 16, [20])
    r.call()
    out = dev.blank(2 * 32 * 2)
    args = [L.BF16, dev(r.q_raw), 5 * 32, 2, L.BF16, out, 64, None, dev(r.table), r.table.shape[1], dev(r.lengths)]
    tail = [20, 0, r.scale, 0.0, 0, r.ws, r.ws_bytes, 0, None]
    assert l.kv_attend(r.h.c, *args, 1, *tail) == 0
    l.stream_sync(None)
    assert np.array_equal(dev.read(out, 128), dev.read(r.out, 128))
    again = dev.blank(2 * 32 * 2)
    args[5] = again
    assert l.kv_attend(r.h.c, *args, 0, *tail) == 0
    l.stream_sync(None)
    assert (dev.read(again, 128) == 0x77).all()
    r.free()


# ------------------------------------------------------------------------ join

@pytest.mark.parametrize("src,out,rows,dim,members", [
    ("fp32", "bf16", 1, 8, (0, 0, 4)), ("fp32", "fp32", 37, 128, (0, 0, 4)), ("bf16", "bf16", 300, 64, (1, 0, 3)),
    ("fp16", "fp16", 65, 72, (1, 1, 2)), ("bf16", "fp32", 9, 256, (3, 0, 1)), ("fp16", "bf16", 1000, 96, (0, 1, 2)),
    ("fp32", "fp16", 77, 1000, (0, 0, 4)),
])
def test_join_of_partial_results(rt, L, dev, src, out, rows, dim, members):
    l, rng = rt.l, np.random.default_rng([rows, dim])
    first, log_stride, size = members
    pes = [first + (i << log_stride) for i in range(size)]
    es = ref.SIZE[src]
    partial, lses = l.malloc(rows * dim * es), l.malloc(rows * 4)
    raw, x = values(rng, (P, rows, dim), src)
    lse = (rng.standard_normal((P, rows)) * 3 + 5).astype(np.float32)
    lse[rng.random((P, rows)) < 0.2] = -np.inf
    lse[:, rows // 2] = -np.inf                  # a row that nobody holds
    lse[0, rows // 3], lse[1:, rows // 3] = 200.0, -200.0  # one that takes all the weight
    raw[np.isneginf(lse)] = np.uint32(0xFFFFFFFF).astype(raw.dtype) if es == 4 else 0xFFFF  # NaN where nothing counts
    for pe in range(P):
        rt.put_bytes(l.pe_ptr(partial, pe), raw[pe])
        rt.put_bytes(l.pe_ptr(lses, pe), lse[pe])
    want, want_lse, around = ref.join(x[pes], lse[pes].astype(np.float64))
    for my_pe in (0, 2):
        o, s = dev.blank(rows * dim * ref.SIZE[out]), dev.blank(rows * 4)
        assert l.kv_join(type_of(L, src), l.pe_ptr(partial, my_pe), l.pe_ptr(lses, my_pe), rows, dim, type_of(L, out), o,
                         s if my_pe else None, first, log_stride, size, my_pe, None) == 0
        l.stream_sync(None)
        got = ref.decode(dev.read(o, rows * dim * ref.SIZE[out]).view({2: np.uint16, 4: np.uint32}[ref.SIZE[out]]),
                         out).reshape(rows, dim)
        # a weight: the difference of two lse's rounds to 2^-24 of at most 20 here
        # (beyond, the weight is below 2^-28 of the whole), the exponential 2^-22;
        # sums of at most 4 terms and a quotient
        d = around * (20 * 2.0 ** -23 + 2.0 ** -21 + 8 * 2.0 ** -24) + 2.0 ** -28 * np.abs(want)
        assert (np.abs(got - want) <= d + ref.U[out] * (np.abs(want) + d) + ref.LEAST[out]).all()
        if my_pe:
            got_lse = dev.read(s, rows * 4).view(np.float32).astype(np.float64)
            none = np.isneginf(want_lse)
            assert np.array_equal(np.isneginf(got_lse), none) and (rows == 1 or none[rows // 2])
            # the roundings above, a logarithm of a sum of at most 4, and the last sum
            assert (np.abs(got_lse - want_lse)[~none] <= 20 * 2.0 ** -23 + 2.0 ** -20 +
                    np.abs(want_lse[~none]) * 2.0 ** -23).all()
        else:
            assert (dev.read(s, rows * 4) == 0x77).all()
    l.free(partial)
    l.free(lses)


# ------------------------------------------------------- together, as they are used

@pytest.mark.parametrize("src,cache", [("bf16", "bf16"), ("fp16", "e4m3")])
def test_sequences_grow_token_by_token_eager_and_from_a_graph(rt, L, dev, src, cache):
    """A decoding loop: each step puts one new token per sequence (one of them
    idle in some steps), attends, and reads the rows back; first eagerly, then
    as one captured graph replayed with new inputs, every step checked."""
    from tests.test_gpu_graph_capture import hip
    l, h = rt.l, hip()
    rng = np.random.default_rng(11)
    heads, group, dim, page, n, each, per_pe = 2, 4, 64, 16, 3, 4, 3
    hq = heads * group
    r = Run(rt, L, dev, src, cache, heads, group, dim, page, [1])
    r.free()
    r.table = np.arange(n * each, dtype=np.int32).reshape(n, each)[:, ::-1].copy()  # pages back to front
    r.n_pages = P * per_pe
    r.m = ref.Cache(cache, P, per_pe, page, heads, dim, fill=0xFF)
    r.h = OnHeap(rt, L, r.m)
    src_t, es = type_of(L, src), ref.SIZE[src]
    r.max_len, r.window, r.softcap, r.scale, r.out_type, r.out_row = 64, 0, 0.0, dim ** -0.5, src, hq * dim
    kv_row = 2 * heads * dim
    kv, slots, lengths = dev(np.zeros((n, kv_row), np.uint16)), dev(np.zeros(n, np.int64)), dev(np.zeros(n, np.int32))
    q, table = dev(np.zeros((n, hq * dim), np.uint16)), dev(r.table)
    r.out, r.lse = dev.blank(n * hq * dim * es), dev.blank(n * hq * 4)
    back = [dev.blank(n * heads * dim * es) for _ in range(2)]
    r.ws_bytes = l.kv_attend_bytes(r.h.c, n, hq, r.max_len)
    r.ws = dev.blank(r.ws_bytes)

    def enqueue(stream):
        assert l.kv_put(r.h.c, src_t, kv, kv_row, kv + heads * dim * es, kv_row, slots, n, 0, stream) == 0
        assert l.kv_attend(r.h.c, src_t, q, hq * dim, hq, src_t, r.out, hq * dim, r.lse, table, r.table.shape[1],
                           lengths, n, r.max_len, 0, r.scale, 0.0, 0, r.ws, r.ws_bytes, 0, stream) == 0
        assert l.kv_get(r.h.c, src_t, back[0], heads * dim, back[1], heads * dim, slots, n, 0, stream) == 0

    stream, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert h.hipStreamCreate(C.byref(stream)) == 0
    r.lengths = np.array([0, 0, 0], np.int32)
    try:
        for step in range(40):
            if step == 20:
                assert h.hipStreamBeginCapture(stream, 0) == 0
                enqueue(stream)
                assert h.hipStreamEndCapture(stream, C.byref(graph)) == 0 and graph.value
                assert h.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0 and exe.value
            idle = step % 3 if step % 4 == 3 else None
            new = np.full(n, -1, np.int64)
            for b in range(n):
                if b != idle:
                    at = int(r.lengths[b])
                    new[b] = int(r.table[b, at // page]) * page + at % page
                    r.lengths[b] += 1
            raw, x = values(rng, (n, 2 * heads, dim), src, 0.3)
            r.q_raw, r.q = values(rng, (n, hq, dim), src, 0.3)
            rt.put_bytes(kv, raw)
            rt.put_bytes(q, r.q_raw)
            rt.put_bytes(slots, new)
            rt.put_bytes(lengths, r.lengths)
            r.m.put(new, x[:, :heads], x[:, heads:])
            if exe.value:
                assert h.hipGraphLaunch(exe, stream) == 0
            else:
                enqueue(stream)
            assert h.hipStreamSynchronize(stream) == 0
            r.check()
            for value in (0, 1):
                got = dev.read(back[value], n * heads * dim * es).view(np.uint16).reshape(n, heads * dim)
                want = ref.encode(r.m.rows(new[new >= 0], value).astype(np.float32), src).reshape(-1, heads * dim)
                assert np.array_equal(got[new >= 0], want), step
    finally:
        if exe.value:
            h.hipGraphExecDestroy(exe)
            h.hipGraphDestroy(graph)
        h.hipStreamDestroy(stream)
        r.free()
