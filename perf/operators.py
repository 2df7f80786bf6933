"""Timed cases of the operators that serve a key-value cache on the symmetric heap.

A model that answers with a cache keeps, for every token it has seen, one key
and one value row per head.  Here the cache is a symmetric object: pages of a
fixed number of tokens, spread over the slices of P processing elements (PEs),
found through a page table.  Four operators work on it:

  put     writes tokens' key and value rows into their slots of the cache, in
          16 bits or narrowed to e4m3 with one power-of-two scale per row
  get     reads tokens' rows back
  attend  attention of one new token per sequence over its cached tokens
  join    the partial results that P PEs reached over their own shares of the
          tokens, joined into the result over all of them

`run` computes them in plain torch operations where `own` is false and makes
the library's calls where it is true.  Both work on the same page layout:

  page = [keys | values | key scales | value scales | padding to 128 bytes]
  keys, values: [kv_heads][page_tokens][head_dim];  scales (e4m3 only):
  [kv_heads][page_tokens] bytes b, each standing for 2^(b - 127)
"""

import math

import numpy as np
import torch

own = False

PES = 8
HEAP_BYTES = 2 << 30  # per PE
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
         "e4m3": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One decoding step of 64 users: every layer writes 64 rows per head.
        dict(name="put, 64 users' new tokens", op="put", src="bf16", cache="bf16", tokens=64,
             kv_heads=8, head_dim=128, page=64, pages=256),
        # A prompt of odd length enters an 8-bit cache and is read back (as the
        # cached prefix of a next prompt is).
        dict(name="put+get, prompt of 20011", op="put_get", src="bf16", cache="e4m3", tokens=20011,
             kv_heads=8, head_dim=128, page=64, pages=512),
        # Several long prompts at once, activations in 16-bit floating point.
        dict(name="put+get, prompts of 65536", op="put_get", src="fp16", cache="e4m3", tokens=65536,
             kv_heads=8, head_dim=128, page=128, pages=1024),
        # A shared prefix read back, narrower heads, a head count that is no power of two.
        dict(name="get, prefix of 3001", op="get", src="fp16", cache="fp16", tokens=3001,
             kv_heads=5, head_dim=96, page=32, pages=256),
        # One user, a short conversation: latency is all there is.
        dict(name="attend, 1 user of 333", op="attend", src="bf16", cache="bf16", seqs=1, max_len=333,
             q_heads=32, kv_heads=8, head_dim=128, page=64, window=0, softcap=0.0),
        # Many users with ordinary conversations, some just arrived.
        dict(name="attend, 64 users to 4096", op="attend", src="bf16", cache="bf16", seqs=64,
             max_len=4096, q_heads=64, kv_heads=8, head_dim=128, page=64, window=0, softcap=0.0),
        # Two long documents over an 8-bit cache: few rows, a long axis.
        dict(name="attend, 2 users to 131072", op="attend", src="bf16", cache="e4m3", seqs=2,
             max_len=131072, q_heads=64, kv_heads=8, head_dim=128, page=128, window=0, softcap=0.0),
        # Every query head with a cache head of its own, capped scores.
        dict(name="attend, 16 users, own heads", op="attend", src="fp16", cache="fp16", seqs=16,
             max_len=2011, q_heads=24, kv_heads=24, head_dim=64, page=16, window=0, softcap=30.0),
        # A layer that looks back over a window, wide heads, pages that end inside any tile.
        dict(name="attend, window of 1024", op="attend", src="fp16", cache="e4m3", seqs=32,
             max_len=20000, q_heads=16, kv_heads=4, head_dim=256, page=48, window=1024, softcap=0.0),
        # One cache head for all query heads.
        dict(name="attend, one cache head", op="attend", src="bf16", cache="bf16", seqs=24,
             max_len=30011, q_heads=48, kv_heads=1, head_dim=128, page=32, window=0, softcap=0.0),
        # Partial results of a decoding step's 8 x 64 rows, from 8 PEs.
        dict(name="join, 512 rows", op="join", src="fp32", out="bf16", rows=512, head_dim=128),
        # The same for a chunk of a prompt.
        dict(name="join, 65536 rows", op="join", src="fp32", out="bf16", rows=65536, head_dim=128),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["put", "put_get", "get", "attend", "attend", "attend", "join"])
    if op == "join":
        return dict(op=op, src=rng.choice(["fp32", "bf16", "fp16"]), out=rng.choice(["bf16", "fp16"]),
                    rows=_log_between(rng, 1, 60000), head_dim=16 * rng.randint(1, 8))
    src = rng.choice(["bf16", "fp16"])
    cache = "e4m3" if op == "put_get" else rng.choice([src, "e4m3"]) if op == "attend" else src
    page = 16 * rng.randint(1, 8)
    head_dim = 16 * rng.randint(1, 16)
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8])
    if op == "attend":
        group = _log_between(rng, 1, 64 // kv_heads if kv_heads > 1 else 64)
        max_len = min(_log_between(rng, 1, 100000), 120_000_000 // (kv_heads * head_dim))
        most = 120_000_000 // (max_len * kv_heads * head_dim)
        return dict(op=op, src=src, cache=cache, seqs=_log_between(rng, 1, min(96, max(1, most))),
                    max_len=max_len, q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                    page=page, window=rng.choice([0, 0, _log_between(rng, 1, max_len)]),
                    softcap=rng.choice([0.0, 0.0, 20.0, 50.0]))
    tokens = _log_between(rng, 1, max(1, min(60000, 60_000_000 // (kv_heads * head_dim))))
    return dict(op=op, src=src, cache=cache, tokens=tokens, kv_heads=kv_heads, head_dim=head_dim,
                page=page, pages=PES * (-(-tokens // (page * PES)) + rng.randint(0, 4)))


def _lengths(case):
    """Lengths up to max_len in even steps, from 0 where there are more than a few sequences."""
    n, top = case["seqs"], case["max_len"]
    return [round(top * (i + 1) / n) for i in range(n)] if n < 8 else [round(top * i / (n - 1)) for i in range(n)]


def _seen(case):
    """How many tokens each sequence's new token attends to."""
    return [min(x, case["window"]) if case["window"] else x for x in _lengths(case)]


def _row_bytes(case):
    """Bytes of one token's keys and values in the cache."""
    narrow = case["cache"] == "e4m3"
    return 2 * case["kv_heads"] * (case["head_dim"] * SIZE[case["cache"]] + (1 if narrow else 0))


def work(case):
    if case["op"] == "join":
        rows, d = case["rows"], case["head_dim"]
        return dict(bytes=PES * rows * (d * SIZE[case["src"]] + 4) + rows * (d * SIZE[case["out"]] + 4),
                    flops=2 * PES * rows * d)
    if case["op"] == "attend":
        tokens, heads = sum(_seen(case)), case["seqs"] * case["q_heads"]
        return dict(bytes=tokens * _row_bytes(case) + heads * (2 * case["head_dim"] * SIZE[case["src"]] + 4)
                    + 4 * (case["seqs"] + sum(-(-x // case["page"]) for x in _seen(case))),
                    flops=4 * tokens * case["q_heads"] * case["head_dim"])
    wide = 2 * case["kv_heads"] * case["head_dim"] * SIZE[case["src"]]
    times = 2 if case["op"] == "put_get" else 1
    return dict(bytes=times * case["tokens"] * (wide + _row_bytes(case) + 8),
                flops=(4 if case["cache"] == "e4m3" else 1) * case["tokens"] * wide)


# ------------------------------------------------------- pages, in plain torch

def _page_bytes(case):
    n = case["kv_heads"] * case["page"] * (case["head_dim"] * SIZE[case["cache"]] + (1 if case["cache"] == "e4m3" else 0))
    return -(-2 * n // 128) * 128


def _parts(case, pages):
    """Views of the keys, the values and (e4m3) their scale bytes in pages [..., page_bytes]."""
    h, t, d = case["kv_heads"], case["page"], case["head_dim"]
    n, s = h * t * d * SIZE[case["cache"]], h * t
    rows = [pages[..., i * n:(i + 1) * n].view(TYPES[case["cache"]]).unflatten(-1, (h, t, d)) for i in (0, 1)]
    if case["cache"] != "e4m3":
        return rows + [None, None]
    return rows + [pages[..., 2 * n + i * s:2 * n + (i + 1) * s].unflatten(-1, (h, t)) for i in (0, 1)]


def _narrow(x):
    """Rows of 32-bit values as e4m3 codes and one scale byte: the smallest power of two, from
    2^-126 up, that brings the row's largest finite value to at most 448.  What is not finite
    becomes NaN."""
    fine = torch.isfinite(x)
    m, e = torch.frexp(torch.where(fine, x.abs(), 0.0).amax(-1))
    e = torch.where(m == 0, -126, torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126))
    y = torch.where(fine, torch.ldexp(x, -e.unsqueeze(-1)), math.nan)
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _two_to(scale_bytes):
    return (scale_bytes.int() << 23).view(torch.float32)


def _wide(rows, scales):
    x = rows.float()
    return x if scales is None else x * _two_to(scales).unsqueeze(-1)


# --------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def _random_pages(case, n_pages, g):
    """Pages as earlier tokens left them."""
    pages = torch.zeros(n_pages, _page_bytes(case), dtype=torch.uint8, device="cuda")
    parts = _parts(case, pages)
    shape = parts[0].shape
    for i in (0, 1):
        x = _normal(g, *shape)
        if case["cache"] == "e4m3":
            codes, scales = _narrow(x)
            parts[i].view(torch.uint8).copy_(codes.view(torch.uint8))
            parts[2 + i].copy_(scales)
        else:
            parts[i].copy_(x)
    return pages


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case=case)
    if case["op"] == "join":
        rows, d = case["rows"], case["head_dim"]
        s["partial"] = _normal(g, PES, rows, d, dtype=TYPES[case["src"]])
        s["partial_lse"] = 2 * _normal(g, PES, rows) + 8
        # a PE that holds none of a row's tokens
        s["partial_lse"][torch.rand(PES, rows, device="cuda", generator=g) < 0.1] = -math.inf
        if own:
            _place_join(s)
        return s
    if case["op"] == "attend":
        lengths = _lengths(case)
        each = -(-case["max_len"] // case["page"])
        used = sum(-(-x // case["page"]) for x in lengths)
        n_pages = PES * -(-used // PES)
        s["pages"] = _random_pages(case, n_pages, g)
        order = torch.randperm(case["seqs"], device="cuda", generator=g)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")[order]
        at = torch.arange(each, device="cuda")
        mine = at.unsqueeze(0) < (-(-s["lengths"] // case["page"])).unsqueeze(1)
        table = torch.full((case["seqs"], each), -1, dtype=torch.int32, device="cuda")
        table[mine] = torch.randperm(n_pages, device="cuda", generator=g)[:used].int()
        s["table"] = table
        # queries come as the first part of a packed projection
        packed = _normal(g, case["seqs"], case["q_heads"] + 2 * case["kv_heads"], case["head_dim"],
                         dtype=TYPES[case["src"]])
        s["q"] = packed[:, :case["q_heads"]]
        s["out"] = torch.zeros(case["seqs"], case["q_heads"], case["head_dim"], dtype=TYPES[case["src"]], device="cuda")
        s["lse"] = torch.zeros(case["seqs"], case["q_heads"], dtype=torch.float32, device="cuda")
    else:
        s["pages"] = _random_pages(case, case["pages"], g)
        slots = torch.randperm(case["pages"] * case["page"], device="cuda", generator=g)[:case["tokens"]]
        if case["tokens"] > 7:
            slots[::7] = torch.where(torch.arange(len(slots[::7]), device="cuda") % 5 == 0, -1, slots[::7])  # padding
        s["slots"] = slots
        packed = _normal(g, case["tokens"], 6 * case["kv_heads"], case["head_dim"])
        # activations differ in size from token to token
        packed *= torch.exp(_normal(g, case["tokens"], 1, 1))
        packed = packed.to(TYPES[case["src"]])
        s["k"], s["v"] = packed[:, -2 * case["kv_heads"]:-case["kv_heads"]], packed[:, -case["kv_heads"]:]
        s["k_back"], s["v_back"] = (torch.zeros(case["tokens"], case["kv_heads"], case["head_dim"],
                                                dtype=TYPES[case["src"]], device="cuda") for _ in range(2))
    if own:
        _place(s)
    return s


# ------------------------------------------------------------ the plain forms

def _put(s):
    case, parts = s["case"], _parts(s["case"], s["pages"])
    keep = s["slots"] >= 0
    slots = s["slots"][keep]
    page, at = slots // case["page"], slots % case["page"]
    for i, x in enumerate((s["k"], s["v"])):
        x = x[keep].float()
        if case["cache"] == "e4m3":
            codes, scales = _narrow(x)
            parts[i].view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
            parts[2 + i][page, :, at] = scales
        else:
            parts[i][page, :, at] = x.to(TYPES[case["cache"]])


def _get(s):
    case, parts = s["case"], _parts(s["case"], s["pages"])
    slots = s["slots"].clamp(min=0)
    page, at = slots // case["page"], slots % case["page"]
    keep = (s["slots"] >= 0).view(-1, 1, 1)
    for i, to in enumerate((s["k_back"], s["v_back"])):
        rows = parts[i].view(torch.uint8)[page, :, at].view(TYPES[case["cache"]])
        scales = None if parts[2] is None else parts[2 + i][page, :, at]
        to.copy_(torch.where(keep, _wide(rows, scales).to(to.dtype), to))


def _attend(s):
    case = s["case"]
    h, d = case["kv_heads"], case["head_dim"]
    end = s["lengths"].view(-1, 1)
    start = (end - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(end)
    # the pages that may be looked at: all of a sequence's, or as many as a window can touch
    most = s["table"].shape[1]
    count = min(most, -(-case["window"] // case["page"]) + 1) if case["window"] else most
    which = start // case["page"] + torch.arange(count, device=end.device)
    pages = s["pages"][s["table"].gather(1, which.clamp(max=most - 1)).clamp(min=0)]  # [seqs, pages, bytes]
    parts = _parts(case, pages)
    # [seqs, pages, heads, page, dim] -> [seqs, heads, tokens, dim]
    k, v = (_wide(parts[i], parts[2 + i]).transpose(1, 2).flatten(2, 3) for i in (0, 1))
    q = s["q"].float().unflatten(1, (h, -1))
    x = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    at = (which.unsqueeze(-1) * case["page"] + torch.arange(case["page"], device=end.device)).flatten(1)
    seen = (at >= start) & (at < end)
    x = torch.where(seen[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, torch.where(seen[:, None, :, None], v, 0.0)) / torch.where(total == 0, 1.0, total)
    return {"out": out.flatten(1, 2).to(s["q"].dtype), "lse": (top + torch.log(total)).flatten(1, 2).squeeze(-1)}


def _join(s):
    x, lse = s["partial"].float(), s["partial_lse"]
    top = lse.amax(0)
    w = torch.exp(lse - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(0)
    out = (w.unsqueeze(-1) * torch.where((w > 0).unsqueeze(-1), x, 0.0)).sum(0)
    out = out / torch.where(total == 0, 1.0, total).unsqueeze(-1)
    return {"out": out.to(TYPES[s["case"]["out"]]), "lse": top + torch.log(total)}


def run(s):
    if own:
        return _run_own(s)
    op = s["case"]["op"]
    if op == "attend":
        return _attend(s)
    if op == "join":
        return _join(s)
    if op != "get":
        _put(s)
    if op == "put":
        return {"cache": s["pages"].view(PES, -1).view(TYPES[s["case"]["cache"]])}
    _get(s)
    return {"k": s["k_back"], "v": s["v_back"]}


# ---------------------------------------------------------- the library's calls

class _Symmetric:
    """A symmetric object of `nbytes` per PE, and all its copies as one tensor."""

    def __init__(self, lib, rows):
        self.lib, nbytes = lib, rows.shape[1] * rows.element_size()
        self.ptr = lib.malloc(nbytes)
        if not self.ptr:
            raise RuntimeError("the symmetric heap is full")
        self.__cuda_array_interface__ = dict(data=(self.ptr, False), shape=(PES, nbytes), typestr="|u1",
                                             strides=(lib.pe_stride(), 1), version=3)
        torch.as_tensor(self, device="cuda").copy_(rows.view(torch.uint8))
        torch.cuda.synchronize()

    def __del__(self):
        self.lib.free(self.ptr)


def _library():
    from rocshmem_amd import lib
    loaded = lib.load()
    if not loaded.heap_size() and loaded.init(PES, HEAP_BYTES) != 0:
        raise RuntimeError("rocshmem_amd_init failed")
    return lib, loaded


def _type_of(lib, name):
    return {"bf16": lib.BF16, "fp16": lib.HALF, "fp32": lib.FLOAT, "e4m3": lib.E4M3}[name]


def _place(s):
    """The cache onto the symmetric heap, and what a program keeps from call to call."""
    lib, loaded = _library()
    case = s["case"]
    s["symmetric"] = _Symmetric(loaded, s.pop("pages").view(PES, -1))
    s["cache"] = lib.KvCache(pages=s["symmetric"].ptr, dtype=_type_of(lib, case["cache"]),
                             pages_per_pe=s["symmetric"].__cuda_array_interface__["shape"][1] // _page_bytes(case),
                             page_tokens=case["page"], kv_heads=case["kv_heads"], head_dim=case["head_dim"])
    s["lib"], s["type"] = loaded, _type_of(lib, case["src"])
    if case["op"] == "attend":
        n = loaded.kv_attend_bytes(s["cache"], case["seqs"], case["q_heads"], case["max_len"])
        s["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda")


def _place_join(s):
    lib, loaded = _library()
    s["lib"], s["type"], s["out_type"] = loaded, _type_of(lib, s["case"]["src"]), _type_of(lib, s["case"]["out"])
    s["partial"] = _Symmetric(loaded, s["partial"].view(PES, -1))
    s["partial_lse"] = _Symmetric(loaded, s["partial_lse"].view(PES, -1))
    s["out"] = torch.empty(s["case"]["rows"], s["case"]["head_dim"], dtype=TYPES[s["case"]["out"]], device="cuda")
    s["lse"] = torch.empty(s["case"]["rows"], dtype=torch.float32, device="cuda")


def _checked(status):
    if status != 0:
        raise RuntimeError("the call was refused: %d" % status)


def _run_own(s):
    case, lib = s["case"], s["lib"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "join":
        _checked(lib.kv_join(s["type"], s["partial"].ptr, s["partial_lse"].ptr, case["rows"], case["head_dim"],
                             s["out_type"], s["out"].data_ptr(), s["lse"].data_ptr(), 0, 0, PES, 0, stream))
        return {"out": s["out"], "lse": s["lse"]}
    if case["op"] == "attend":
        _checked(lib.kv_attend(s["cache"], s["type"], s["q"].data_ptr(), s["q"].stride(0), case["q_heads"],
                               s["type"], s["out"].data_ptr(), s["out"].stride(0), s["lse"].data_ptr(),
                               s["table"].data_ptr(), s["table"].stride(0), s["lengths"].data_ptr(),
                               case["seqs"], case["max_len"], case["window"], case["head_dim"] ** -0.5,
                               case["softcap"], 0, s["workspace"].data_ptr(), s["workspace"].numel(), 0, stream))
        return {"out": s["out"], "lse": s["lse"]}
    if case["op"] != "get":
        _checked(lib.kv_put(s["cache"], s["type"], s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(),
                            s["v"].stride(0), s["slots"].data_ptr(), case["tokens"], 0, stream))
    if case["op"] == "put":
        return {"cache": torch.as_tensor(s["symmetric"], device="cuda").view(TYPES[case["cache"]])}
    _checked(lib.kv_get(s["cache"], s["type"], s["k_back"].data_ptr(), s["k_back"].stride(0), s["v_back"].data_ptr(),
                        s["v_back"].stride(0), s["slots"].data_ptr(), case["tokens"], 0, stream))
    return {"k": s["k_back"], "v": s["v_back"]}


# ------------------------------------------------------- the definition, 64 bits

def _bytes_as_values(raw, cache):
    """Values of 16-bit or e4m3 bytes, in 64 bits, from the formats' definitions."""
    if cache == "bf16":
        return (raw.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if cache == "fp16":
        return raw.view(np.float16).astype(np.float64)
    code = np.arange(256)
    power, low = (code >> 3) & 15, code & 7
    value = np.where(power == 0, low * 2.0 ** -9, (8 + low) * 2.0 ** (power - 10.0))
    value = np.where((code & 127) == 127, np.nan, np.where(code > 127, -value, value))
    return value[raw]


def _token_rows(case, page, which):
    """Keys (which = 0) or values (1) of one page's bytes: [kv_heads, page, head_dim]."""
    h, t, d = case["kv_heads"], case["page"], case["head_dim"]
    n = h * t * d * SIZE[case["cache"]]
    x = _bytes_as_values(page[..., which * n:(which + 1) * n], case["cache"]).reshape(*page.shape[:-1], h, t, d)
    if case["cache"] == "e4m3":
        b = page[..., 2 * n + which * h * t:2 * n + (which + 1) * h * t].astype(np.float64)
        x = x * np.exp2(b - 127).reshape(*page.shape[:-1], h, t, 1)
    return x


def _nearest_e4m3(x):
    """x, rows of 64-bit values, as e4m3 with a power-of-two scale per row stands for them."""
    one = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448)).clamp(min=-126))
    step = torch.exp2(torch.floor(torch.log2(x.abs() / one)).clamp(min=-6) - 3) * one
    return torch.round(x / step) * step


def _exact_attend(case, s):
    """Sequence by sequence on the GPU, in 64 bits."""
    h, d, n = case["kv_heads"], case["head_dim"], case["page"]
    group = case["q_heads"] // h
    out = torch.zeros(case["seqs"], case["q_heads"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((case["seqs"], case["q_heads"]), -math.inf, dtype=torch.float64, device="cuda")
    wide = torch.arange(256, device="cuda").to(torch.uint8).view(torch.float8_e4m3fn).double()
    for b, end in enumerate(s["lengths"].tolist()):
        start = max(0, end - case["window"]) if case["window"] else 0
        if start == end:
            continue
        raw = s["pages"][s["table"][b, start // n:-(-end // n)].long()]
        part = h * n * d * SIZE[case["cache"]]
        for i in range(h):  # one head at a time: a long cache is large in 64 bits
            kv = []
            for which in (0, 1):
                lo = which * part + i * n * d * SIZE[case["cache"]]
                x = raw[:, lo:lo + n * d * SIZE[case["cache"]]]
                if case["cache"] == "e4m3":
                    lo = 2 * part + which * h * n + i * n
                    x = wide[x.long()].view(-1, n, d) * torch.exp2(raw[:, lo:lo + n].double() - 127).unsqueeze(-1)
                else:
                    x = x.contiguous().view(TYPES[case["cache"]]).double().view(-1, n, d)
                kv.append(x.reshape(-1, d)[start % n:start % n + end - start])
            x = (s["q"][b, i * group:(i + 1) * group].double() @ kv[0].T) / math.sqrt(d)
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            lse[b, i * group:(i + 1) * group] = torch.logsumexp(x, -1)
            out[b, i * group:(i + 1) * group] = torch.softmax(x, -1) @ kv[1]
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    if case["op"] == "join":
        x, lse = s["partial"].double(), s["partial_lse"].double()
        total = torch.logsumexp(lse, 0)
        return {"out": (torch.softmax(lse, 0).nan_to_num(0.0).unsqueeze(-1) * x).sum(0), "lse": total}
    if case["op"] == "put_get":
        keep = (s["slots"] >= 0).view(-1, 1, 1)
        return {name: torch.where(keep, _nearest_e4m3(s[name].double()), 0.0) for name in ("k", "v")}
    slots, pages = s["slots"].cpu().numpy(), s["pages"].cpu().numpy()
    keep, page, at = slots >= 0, slots // case["page"], slots % case["page"]
    if case["op"] == "put":
        values = _bytes_as_values(pages.view(np.uint8), case["cache"]).reshape(len(pages), -1)
        n = case["kv_heads"] * case["page"] * case["head_dim"]
        for which, x in enumerate((s["k"], s["v"])):
            rows = values[:, which * n:(which + 1) * n].reshape(len(pages), case["kv_heads"], case["page"], -1)
            rows[page[keep], :, at[keep]] = x.double().cpu().numpy()[keep]
            values[:, which * n:(which + 1) * n] = rows.reshape(len(pages), n)
        return {"cache": values.reshape(PES, -1)}
    return {name: np.where(keep[:, None, None], _token_rows(case, pages, which)[page, :, at], 0.0)
            for which, name in enumerate(("k", "v"))}
