"""The key-value cache in numpy: formats by their definitions, pages by the
layout that include/rocshmem_amd.h states, attention and joins in 64 bits.
Test infrastructure; nothing here calls the library."""
import numpy as np

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}  # half a step, relative
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
LEAST = {"bf16": 2.0 ** -133, "fp16": 2.0 ** -24, "fp32": 2.0 ** -149}  # the smallest step


# ---- formats: 64-bit values <-> raw bytes ------------------------------------

def encode(x, name):
    """32-bit values in a format, rounded to nearest even, as an array of its integers."""
    x = np.asarray(x, np.float32)
    if name == "fp32":
        return x.view(np.uint32)
    if name == "fp16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def decode(raw, name):
    raw = np.asarray(raw)
    if name == "fp32":
        return raw.view(np.float32).astype(np.float64)
    if name == "fp16":
        return raw.view(np.float16).astype(np.float64)
    if name == "bf16":
        return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return E4M3[raw]


def _e4m3_table():
    code = np.arange(256)
    power, low = (code >> 3) & 15, code & 7
    v = np.where(power == 0, low * 2.0 ** -9, (8 + low) * 2.0 ** (power - 10.0))
    v = np.where((code & 127) == 127, np.nan, v)
    return np.where(code > 127, -v, v)


E4M3 = _e4m3_table()


def to_e4m3(y):
    """Codes of 64-bit values of magnitude up to 448, to nearest, ties to the even code; NaN for what is not finite."""
    grid = E4M3[:127]
    a = np.abs(np.where(np.isfinite(y), y, 0.0))
    hi = np.clip(np.searchsorted(grid, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - a, a - grid[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.isfinite(y), code, 127)
    return (code | (np.signbit(y).astype(int) << 7)).astype(np.uint8)


def narrow(x):
    """Rows [..., D] of 64-bit values as (codes, scale bytes)."""
    top = np.abs(np.where(np.isfinite(x), x, 0.0)).max(-1)
    e = np.full(top.shape, -126)
    some = top > 0
    m, p = np.frexp(top)  # m in [0.5, 1): top <= 448 * 2^e with 448 = 0.875 * 2^9
    e[some] = np.maximum(np.where(m <= 0.875, p - 9, p - 8), -126)[some]
    with np.errstate(invalid="ignore"):
        return to_e4m3(x * np.exp2(-e.astype(float))[..., None]), (e + 127).astype(np.uint8)


# ---- pages --------------------------------------------------------------------

class Cache:
    """A cache of P PEs as bytes [P, pages_per_pe, page_bytes]."""

    def __init__(self, dtype, npes, pages_per_pe, page, heads, dim, fill=0xA5):
        self.dtype, self.page, self.heads, self.dim, self.npes, self.pages_per_pe = dtype, page, heads, dim, npes, pages_per_pe
        self.part = heads * page * dim * SIZE[dtype]
        used = 2 * self.part + (2 * heads * page if dtype == "e4m3" else 0)
        self.page_bytes = -(-used // 128) * 128
        self.raw = np.full((npes, pages_per_pe, self.page_bytes), fill, np.uint8)
        self.slots = npes * pages_per_pe * page

    def where(self, slot):
        page, at = divmod(int(slot), self.page)
        return (page // self.pages_per_pe, page % self.pages_per_pe), at

    def row_at(self, head, at, value):
        return value * self.part + (head * self.page + at) * self.dim * SIZE[self.dtype]

    def scale_at(self, head, at, value):
        return 2 * self.part + (value * self.heads + head) * self.page + at

    def put(self, slots, k, v):
        """Rows [T, heads, D] of 64-bit values that the source's format holds."""
        for t, slot in enumerate(slots):
            if not 0 <= slot < self.slots:
                continue
            place, at = self.where(slot)
            block = self.raw[place]
            for value, x in enumerate((k[t], v[t])):
                codes, scales = narrow(x) if self.dtype == "e4m3" else (encode(x, self.dtype), None)
                for h in range(self.heads):
                    o = self.row_at(h, at, value)
                    row = np.ascontiguousarray(codes[h]).view(np.uint8)
                    block[o:o + row.size] = row
                    if scales is not None:
                        block[self.scale_at(h, at, value)] = scales[h]

    def rows(self, slots, value):
        """Values of the given slots' rows, in 64 bits: [T, heads, D]."""
        out = np.empty((len(slots), self.heads, self.dim))
        n = self.dim * SIZE[self.dtype]
        for t, slot in enumerate(slots):
            place, at = self.where(slot)
            for h in range(self.heads):
                o = self.row_at(h, at, value)
                raw = self.raw[place][o:o + n]
                if self.dtype == "e4m3":
                    out[t, h] = E4M3[raw] * 2.0 ** (float(self.raw[place][self.scale_at(h, at, value)]) - 127)
                else:
                    out[t, h] = decode(raw.view(np.uint16), self.dtype)
        return out


# ---- attention and joins ---------------------------------------------------------

def tokens_of(length, max_len, table, page, n_pages, window=0):
    """Slots that take part, in order, for one sequence."""
    end = min(max(length, 0), max_len, len(table) * page)
    first = max(0, end - window) if window else 0
    return [int(table[i // page]) * page + i % page for i in range(first, end) if 0 <= table[i // page] < n_pages]


def attend(q, k, v, scale, softcap):
    """One query [D] over [T, D] keys and values in 64 bits: (out, lse, bound on
    out's error, bound on lse's).  The bounds are what 32-bit arithmetic may
    cost, before the last rounding: a score's error is that of a sum of D
    products, (D + 4) roundings of at most sum |q k| scale; capping adds 2^-21 of
    the cap (an exponential and a quotient near 1); a weight exp(s - max) adds
    its argument's rounding and 2^-22 of its own; weights may be held as two
    bf16 parts (2^-17); a sum of T terms rounds T times, the running rescaling
    twice as often at most."""
    if not len(k):
        return np.zeros(q.shape), -np.inf, np.zeros(q.shape), 0.0
    s = k @ q * scale
    ds = (len(q) + 4) * 2.0 ** -24 * np.max(np.abs(k) @ np.abs(q)) * abs(scale)
    if softcap:
        s = softcap * np.tanh(s / softcap)
        ds += softcap * 2.0 ** -21
    top = s.max()
    p = np.exp(s - top)
    total = p.sum()
    out = p @ v / total
    around = p @ np.abs(v) / total
    dp = 2 * ds + 2.0 ** -22 + (np.abs(s).max() + abs(top)) * 2.0 ** -22
    dsum = (2 * len(k) + 16) * 2.0 ** -24
    lse = top + np.log(total)
    return out, lse, around * (2 * dp + 2 * dsum + 2.0 ** -17), ds + dp + dsum + abs(lse) * 2.0 ** -22


def join(outs, lses):
    """[P, rows, D], [P, rows] -> (out, lse, magnitude that the weights spread over)."""
    top = lses.max(0)
    with np.errstate(invalid="ignore", divide="ignore"):
        w = np.exp(lses - np.where(np.isneginf(top), 0.0, top))
        total = w.sum(0)
        x = np.where((lses > -np.inf)[..., None], outs, 0.0)
        safe = np.where(total == 0, 1.0, total)[:, None]
        return (w[..., None] * x).sum(0) / safe, top + np.log(total), (w[..., None] * np.abs(x)).sum(0) / safe
