"""The operators of a paged key-value cache held in 8 and 4 bits, as timed cases.

A server's cache is what fills its memory and what a decode step reads. Here the pages
hold whole numbers with scales instead of floating-point rows: rows that come from
elsewhere are quantised as they are written and read back (kind "store"), a step's new
keys and values are normalised, rotated and quantised into their pages and read back, as
a prompt's attention does that continues on them (kind "produce"), one new token of every
sequence attends over the pages (kind "attend"), and a cached prefix is copied out in
order (kind "gather").

A row is one token's key or value of one head, of dh values x.
8 bits: x = S n, n from -127 to 127, S the least bfloat16 with 127 S >= max |x|.
4 bits: x = S sub n in groups of 32 dims, n from -8 to 7, S the least bfloat16 with
1016 S >= max |x| of the row, |sub| the least whole number with 8 |sub| S >= max |x| of the
group and its sign such that the group's extreme (the positive of two equal ones) is at -8.
S is at least 2^-126, |sub| at least 1; n is rounded to nearest, halves to even.

A page: for each head its rows, dh bits / 8 bytes a token, n + 2^(bits - 1) stored (4 bits:
even dims in the low half of a byte); then for each head and 16 tokens, in 4 bits sub + 128
of the tokens' groups (keys token by token, group 4 j + i at i dh / 128 + j; values group by
group), and in both S. The whole is rounded up to 128 bytes.

The widths are Gemma-4-E2B's (8 query heads over 1 kv head; head_dim 256 with a
512-key window, 512 with full context) and groups of other counts. Token counts,
contexts and page sizes are free. What is not in the pages is in 32 bits.

`own` False: the operators in elementary torch operations. `own` True: the calls
a program makes of this library on the same buffers.
"""
from __future__ import annotations

import functools
import math
import os
import sys

import numpy as np
import torch

own = False

EPS = float(np.float32(1e-6))
NO_PAGE = -1
WINDOW = 512
LEAST = 2.0 ** -126
ROPE = {64: (10000.0, 64), 128: (10000.0, 128), 256: (10000.0, 256), 512: (1000000.0, 128)}  # head_dim: theta, rotated


def listed():
    return [
        # one chat's step on a sliding layer, its window full: the smallest attention call
        {"name": "attend_one_sliding_i8", "kind": "attend", "dh": 256, "hq": 8, "hkv": 1, "bits": 8, "page": 16,
         "n": 1, "longest": 2048, "window": WINDOW, "cap": 0.0},
        # one chat's step on a global layer, far into a long document
        {"name": "attend_one_32k_i4", "kind": "attend", "dh": 512, "hq": 8, "hkv": 1, "bits": 4, "page": 64,
         "n": 1, "longest": 32768, "window": 0, "cap": 0.0},
        # a server's step over chats of different lengths
        {"name": "attend_batch_i8", "kind": "attend", "dh": 512, "hq": 8, "hkv": 1, "bits": 8, "page": 16,
         "n": 16, "longest": 8192, "window": 0, "cap": 0.0},
        # the sliding layers of a larger batch, their windows in rings of pages
        {"name": "attend_batch_sliding_i4", "kind": "attend", "dh": 256, "hq": 8, "hkv": 1, "bits": 4, "page": 32,
         "n": 64, "longest": 8192, "window": WINDOW, "cap": 0.0},
        # long documents, up to the model's whole context: what a cache in 4 bits is for
        {"name": "attend_long_i4", "kind": "attend", "dh": 512, "hq": 8, "hkv": 1, "bits": 4, "page": 64,
         "n": 8, "longest": 131072, "window": 0, "cap": 0.0},
        # many short chats of a model with several kv heads and a score cap
        {"name": "attend_many_grouped_i4", "kind": "attend", "dh": 128, "hq": 16, "hkv": 4, "bits": 4, "page": 16,
         "n": 128, "longest": 2000, "window": 0, "cap": 30.0},
        # the new tokens of a decode step of 64 chats
        {"name": "produce_step_i4", "kind": "produce", "dh": 512, "hq": 8, "hkv": 1, "bits": 4, "page": 32,
         "n": 64, "tokens": 64, "past": 1024},
        # prompts of several requests, packed
        {"name": "produce_prompts_i8", "kind": "produce", "dh": 256, "hq": 8, "hkv": 1, "bits": 8, "page": 16,
         "n": 7, "tokens": 4099, "past": 0},
        # one short prompt's rows, handed over by the machine that ran it
        {"name": "store_short_i8", "kind": "store", "dh": 256, "hkv": 1, "bits": 8, "page": 16, "n": 1, "tokens": 333},
        # the rows of several long prompts handed over
        {"name": "store_long_i4", "kind": "store", "dh": 512, "hkv": 1, "bits": 4, "page": 64, "n": 5, "tokens": 20011},
        # a short system prompt ahead of a new question
        {"name": "gather_short_i4", "kind": "gather", "dh": 256, "hkv": 1, "bits": 4, "page": 16, "rows": 700},
        # the next turn on a long document
        {"name": "gather_long_i4", "kind": "gather", "dh": 512, "hkv": 1, "bits": 4, "page": 64, "rows": 32768},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "produce", "store", "gather"])
    bits, page = rng.choice([4, 4, 8]), rng.choice([16, 32, 64, 128, 256])
    dh = rng.choice([64, 128, 256, 256, 512, 512])
    hq, hkv = rng.choice([(8, 1), (8, 1), (8, 2), (16, 4), (4, 4), (16, 1), (3, 1)])
    case = {"kind": kind, "dh": dh, "hkv": hkv, "bits": bits, "page": page}
    if kind == "gather":
        return {**case, "rows": _log(rng, 1, 32768 // hkv)}
    if kind == "store":
        tokens = _log(rng, 1, 20000 // hkv)
        return {**case, "n": _log(rng, 1, min(tokens, 256)), "tokens": tokens}
    if kind == "produce":
        tokens = _log(rng, 1, 4096)
        return {**case, "hq": hq, "n": _log(rng, 1, min(tokens, 256)), "tokens": tokens,
                "past": rng.choice([0, _log(rng, 1, 1024)])}
    n, longest = _log(rng, 1, 128), _log(rng, 1, 131072)
    while n * longest * hkv * dh > 1 << 28:  # about a quarter of attend_long_i4's rows, in the plain form's layout
        longest = (longest + 1) // 2
    return {**case, "hq": hq, "n": n, "longest": longest, "window": rng.choice([0, 0, WINDOW, _log(rng, 1, 4096)]),
            "cap": rng.choice([0.0, 0.0, 30.0])}


# ---- the format -----------------------------------------------------------------

def _row_bytes(case):
    return case["dh"] * case["bits"] // 8


def _subs(case):
    """Scaled groups of a row."""
    return case["dh"] // 32 if case["bits"] == 4 else 0


def _page_bytes(case):
    raw = case["hkv"] * (case["page"] * _row_bytes(case) + case["page"] // 16 * (16 * _subs(case) + 32))
    return -(-raw // 128) * 128


def _views(case, pool, values):
    """A pool's parts: rows [pages, hkv, page, bytes], subs [pages, hkv, tile, 16 tokens, groups] and S's two bytes
    [pages, hkv, tile, 16, 2]."""
    hkv, page, G = case["hkv"], case["page"], _subs(case)
    data, meta = page * _row_bytes(case), 16 * G + 32
    rows = pool[:, :hkv * data].unflatten(1, (hkv, page, -1))
    rest = pool[:, hkv * data:hkv * (data + page // 16 * meta)].unflatten(1, (hkv, page // 16, meta))
    subs = rest[..., :16 * G]
    if G:
        subs = subs.unflatten(-1, (G, 16)).transpose(-1, -2) if values else subs.unflatten(-1, (16, G))
    return rows, subs, rest[..., 16 * G:].unflatten(-1, (16, 2))


def _order(case):
    """The place of each group of a key's row among its subs."""
    G = _subs(case)
    return [g % 4 * (G // 4) + g // 4 for g in range(G)] if G >= 4 else list(range(G))


def _encode(case, x):
    """f32 rows [..., dh] to (n, sub, S): whole numbers, and the row's scale as f32."""
    bits = case["bits"]
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], 0.0, x)
    big, most = x.abs().amax(-1), 127.0 if bits == 8 else 1016.0
    s = (((big.double() / most).float().clamp(min=LEAST).view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)
    s = torch.where(s * most < big, (s.view(torch.int32) + 0x10000).view(torch.float32), s)
    if bits == 8:
        n, sub = torch.round(x.double() / s.double()[..., None]), None
    else:
        x = x.unflatten(-1, (-1, 32))
        high, low = x.amax(-1), -x.amin(-1)
        c = torch.ceil(torch.maximum(high, low).double() / (8.0 * s.double()[..., None])).clamp(min=1.0)
        sub = torch.where(high >= low, -c, c)
        n = torch.round(x.double() / (s.double()[..., None] * sub)[..., None]).clamp(-8, 7).flatten(-2)
        sub = sub.int()
    return n.int(), sub, torch.where(bad, math.nan, s)


def _put(case, pool, values, page, row, x):
    """Rows x [N, hkv, dh] into (page, row) [N] of a pool."""
    n, sub, s = _encode(case, x)
    rows, subs, scale = _views(case, pool, values)
    n = n + (1 << case["bits"] - 1)
    if case["bits"] == 4:
        n = n[..., 0::2] | n[..., 1::2] << 4
        place = list(range(_subs(case))) if values else _order(case)
        stored = torch.empty_like(sub, dtype=torch.uint8)
        stored[..., place] = (sub + 128).to(torch.uint8)
        subs[page, :, row // 16, row % 16] = stored
    rows[page, :, row] = n.to(torch.uint8)
    top = s.to(torch.bfloat16).view(torch.int16).int() & 0xFFFF
    scale[page, :, row // 16, row % 16] = torch.stack([top & 255, top >> 8], -1).to(torch.uint8)


def _get(case, pool, values, page, row):
    """Rows [..., hkv, dh] of (page, row) [...] of a pool, as f32."""
    rows, subs, scale = _views(case, pool, values)
    n, s = rows[page, :, row], scale[page, :, row // 16, row % 16].int()
    s = (s[..., 0] << 16 | s[..., 1] << 24).view(torch.float32)
    if case["bits"] == 8:
        return (n.float() - 128.0) * s[..., None]
    sub = subs[page, :, row // 16, row % 16].float() - 128.0
    if not values:
        sub = sub[..., _order(case)]
    n = torch.stack([n & 15, n >> 4], -1).flatten(-2).float() - 8.0
    return ((n.unflatten(-1, (-1, 32)) * sub[..., None]).flatten(-2)) * s[..., None]


# ---- what a program holds -----------------------------------------------------

def _ragged(n, longest):
    """n lengths from `longest` down to about a sixteenth of it."""
    return [max(1, int(longest * 16 ** (-i / max(1, n - 1)))) for i in range(n)]


def _prompts(n, tokens):
    """n token counts that sum to `tokens`, ragged, at least one each."""
    shares = _ragged(n, tokens)
    half = 2 * sum(shares)
    lens = [max(1, x * tokens // half) for x in shares]
    lens[0] += tokens - sum(lens)
    return lens


class _Draws:
    """Seeded device tensors and host shuffles, in a fixed order of calls."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.host = np.random.RandomState(seed % (1 << 32))

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda")

    def unit_rows(self, *shape):
        x = self.normal(*shape)
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)

    def shuffled(self, xs):
        return [xs[i] for i in self.host.permutation(len(xs))]


def _i32(x):
    """Whole numbers as the device's 32-bit words."""
    return torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()


def _tables(d, lens, page, per_seq, spare):
    """Each sequence's pages, out of a pool in shuffled order: (table [n, per_seq], pages)."""
    used = [min(-(-x // page), per_seq) for x in lens]
    total = sum(used) + spare
    order = d.host.permutation(total).astype(np.int64)
    table = np.full((len(lens), per_seq), NO_PAGE, np.int64)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    return table, total


def _pool(d, case, total, values):
    """A pool of full pages: unit-RMS key rows, or plain values."""
    pool = torch.zeros(total, _page_bytes(case), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (case["page"] * case["hkv"] * case["dh"]))
    for i in range(0, total, step):
        n = min(step, total - i) * case["page"]
        x = (d.normal if values else d.unit_rows)(n, case["hkv"], case["dh"])
        at = torch.arange(n, device="cuda")
        _put(case, pool, values, i + at // case["page"], at % case["page"], x)
    return pool


def _prepare_attend(case, seed):
    d, page, n, window = _Draws(seed), case["page"], case["n"], case["window"]
    lens = d.shuffled(_ragged(n, case["longest"]))
    longest = max(lens)
    # a window's pages are a ring; a full context has a page for every token
    per_seq = -(-(window or longest) // page)
    table, total = _tables(d, lens, page, per_seq, 3)
    # a query norm's weight of a quarter: scores of a few units, as trained heads have
    q = 0.25 * d.unit_rows(n, case["hq"], case["dh"])
    return {"case": case, "q": q, "k": _pool(d, case, total, False), "v": _pool(d, case, total, True),
            "table": _i32(table), "len": _i32(lens), "total": total, "per_seq": per_seq, "longest": longest,
            "out": torch.empty(n, case["hq"] * case["dh"], device="cuda")}


def _new_tokens(d, case, past):
    """Positions and slots of a step's packed tokens, in pages of an empty pool."""
    page, n = case["page"], case["n"]
    new = d.shuffled(_prompts(n, case["tokens"]))
    past = d.shuffled(_ragged(n, past)) if past else [0] * n
    per_seq = -(-max(a + b for a, b in zip(past, new)) // page)
    table, total = _tables(d, [a + b for a, b in zip(past, new)], page, per_seq, 3)
    pos = np.concatenate([np.arange(a, a + b) for a, b in zip(past, new)])
    slots = table[np.repeat(np.arange(n), new), pos // page] * page + pos % page
    rows = (case["tokens"], case["hkv"], case["dh"])
    pools = {x: torch.zeros(total, _page_bytes(case), dtype=torch.uint8, device="cuda") for x in ("k_pool", "v_pool")}
    return {"case": case, "pos": _i32(pos), "slots": _i32(slots), "total": total, **pools,
            "k_out": torch.empty(rows, device="cuda"), "v_out": torch.empty(rows, device="cuda")}


def _prepare_produce(case, seed):
    d, dh, T, hq, hkv = _Draws(seed), case["dh"], case["tokens"], case["hq"], case["hkv"]
    return {**_new_tokens(d, case, case["past"]), "q": d.normal(T, hq, dh), "k": 2.0 * d.normal(T, hkv, dh),
            "v": 3.0 * d.normal(T, hkv, dh), "q_norm": 1.0 + 0.1 * d.normal(dh), "k_norm": 1.0 + 0.1 * d.normal(dh),
            "q_out": torch.empty(T, hq, dh, device="cuda")}


def _prepare_store(case, seed):
    d = _Draws(seed)
    rows = (case["tokens"], case["hkv"], case["dh"])
    return {**_new_tokens(d, case, 0), "k": d.unit_rows(*rows) * (1.0 + 0.3 * d.normal(case["dh"])), "v": d.normal(*rows)}


def _prepare_gather(case, seed):
    d, page, rows = _Draws(seed), case["page"], case["rows"]
    lens = [rows // 3, rows, rows // 2]  # the sequence between two others
    per_seq = -(-rows // page)
    table, total = _tables(d, lens, page, per_seq, 3)
    shape = (rows, case["hkv"], case["dh"])
    return {"case": case, "k": _pool(d, case, total, False), "v": _pool(d, case, total, True), "table": _i32(table),
            "len": _i32(lens), "total": total, "per_seq": per_seq, "k_out": torch.empty(shape, device="cuda"),
            "v_out": torch.empty(shape, device="cuda")}


def prepare(case, seed):
    state = {"attend": _prepare_attend, "produce": _prepare_produce, "store": _prepare_store,
             "gather": _prepare_gather}[case["kind"]](case, seed)
    torch.cuda.synchronize()  # torch's stream made the inputs; a library's own stream may read them
    return state


# ---- the library's calls --------------------------------------------------------

@functools.lru_cache(maxsize=1)
def _library():
    sys.path.insert(0, os.path.join(os.getcwd(), "gemma-4-webgpu-kernels_amd"))
    import g4a
    return g4a, g4a.Context(0)


def _calls(state):
    """A state's calls, their argument blocks filled once, as a program keeps them."""
    g4a, ctx = _library()
    case = state["case"]
    kind = case["kind"]

    def cache(k, v, **more):
        return g4a.PagedCache(k_pages=k.data_ptr(), v_pages=v.data_ptr(), page_size=case["page"], Hkv=case["hkv"],
                              Dh=case["dh"], n_pages=state["total"], kv_type=g4a.KV_TYPES["i%d" % case["bits"]], **more)

    if kind in ("produce", "store"):
        pages = cache(state["k_pool"], state["v_pool"])
        slots, T = state["slots"].data_ptr(), case["tokens"]
        read = functools.partial(ctx.kv_read_paged, pages, slots, T, state["k_out"].data_ptr(),
                                 state["v_out"].data_ptr())
        if kind == "store":
            return [functools.partial(ctx.kv_write_paged, pages, state["k"].data_ptr(), state["v"].data_ptr(), slots, T),
                    read]
        theta, rot = ROPE[case["dh"]]
        args = g4a.PagedProducerArgs(**{n: state[n].data_ptr() for n in ("q", "k", "v", "q_norm", "k_norm", "q_out")},
                                     positions=state["pos"].data_ptr(), slots=slots, T=T, Hq=case["hq"],
                                     rotary_dim=rot, theta=theta, eps=EPS)
        return [functools.partial(ctx.attn_producer_paged, pages, args), read]
    pages = cache(state["k"], state["v"], block_table=state["table"].data_ptr(), kv_len=state["len"].data_ptr(),
                  n_seqs=state["len"].numel(), pages_per_seq=state["per_seq"], ring=bool(case.get("window")))
    if kind == "gather":
        return [functools.partial(ctx.kv_gather_paged, pages, 1, 0, case["rows"], state["k_out"].data_ptr(),
                                  state["v_out"].data_ptr())]
    args = g4a.PagedAttnArgs(q=state["q"].data_ptr(), out=state["out"].data_ptr(), Hq=case["hq"], scale=1.0,
                             sliding_window=case["window"], attn_softcap=case["cap"])
    return [functools.partial(ctx.attention_paged, pages, args)]


def _run_own(state):
    if "calls" not in state:
        state["calls"] = _calls(state)
    for call in state["calls"]:
        call()
    kind = state["case"]["kind"]
    if kind == "attend":
        return state["out"]
    rows = {"k": state["k_out"], "v": state["v_out"]}
    return {"q": state["q_out"], **rows} if kind == "produce" else rows


# ---- the same in elementary operations ------------------------------------------

def _attend(state):
    case = state["case"]
    n, hq, hkv, dh, window, page = (case[x] for x in ("n", "hq", "hkv", "dh", "window", "page"))
    lens = state["len"].long()[:, None]
    span = min(state["longest"], window or state["longest"])
    pos = torch.arange(span, device="cuda")[None] + ((lens - span).clamp(min=0) if window else 0)
    seen = (pos < lens) & (pos >= lens - window) if window else pos < lens
    pos = torch.where(seen, pos, (lens - 1).clamp(min=0))
    pages = state["table"].long()[torch.arange(n, device="cuda")[:, None], (pos // page) % state["per_seq"]]
    q = state["q"].view(n, hkv, hq // hkv, dh).transpose(2, 3).contiguous()
    k = _get(case, state["k"], False, pages, pos % page).transpose(1, 2).contiguous()
    s = torch.matmul(k, q)  # [n, hkv, span, group]
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    s = torch.where(seen[:, None, :, None], s, -math.inf)
    e = torch.exp(s - s.amax(2, keepdim=True))
    v = _get(case, state["v"], True, pages, pos % page).transpose(1, 2).contiguous()
    out = torch.matmul(e.transpose(2, 3).contiguous(), v) / e.sum(2)[..., None]
    return out.reshape(n, hq * dh)


def _rms(x, w=None):
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return y if w is None else y * w


def _turn(x, pos, dh):
    """Half-split rotation of the first `rot` dims; an angle is position * frequency, both held in 32 bits."""
    theta, rot = ROPE[dh]
    half = rot // 2
    freq = (theta ** (torch.arange(half, dtype=torch.float64, device="cuda") * (-2.0 / rot))).float()
    ang = (pos.float()[:, None] * freq)[:, None, :].to(x.dtype)
    a, b, c, s = x[..., :half], x[..., half:rot], torch.cos(ang), torch.sin(ang)
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)


def _store(state, k, v):
    """Rows quantised into their slots, and read back from there."""
    case, slots = state["case"], state["slots"].long()
    page, row = slots // case["page"], slots % case["page"]
    _put(case, state["k_pool"], False, page, row, k)
    _put(case, state["v_pool"], True, page, row, v)
    return {"k": _get(case, state["k_pool"], False, page, row), "v": _get(case, state["v_pool"], True, page, row)}


def _produce(state):
    dh, pos = state["case"]["dh"], state["pos"]
    # in 64 bits up to the rounding to a page's numbers: which of two neighbours a value takes is seen in the output
    k = _turn(_rms(state["k"].double(), state["k_norm"].double()), pos, dh).float()
    v = _rms(state["v"].double()).float()
    return {"q": _turn(_rms(state["q"], state["q_norm"]), pos, dh), **_store(state, k, v)}


def _gather(state):
    case = state["case"]
    pos = torch.arange(case["rows"], device="cuda")
    pages = state["table"].long()[1, pos // case["page"]]
    return {x: _get(case, state[x], x == "v", pages, pos % case["page"]) for x in "kv"}


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "store":
        return _store(state, state["k"], state["v"])
    return {"attend": _attend, "produce": _produce, "gather": _gather}[kind](state)


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    kind, hkv, dh = case["kind"], case["hkv"], case["dh"]
    row, values = _row_bytes(case) + _subs(case) + 2.0, 4.0 * dh  # bytes of a row in a page, and as f32
    if kind == "gather":
        return {"bytes": 2.0 * case["rows"] * hkv * (row + values), "flops": 0.0}
    if kind in ("store", "produce"):  # rows in, pages written and read, rows out
        T, hq = case["tokens"], case.get("hq", 0)
        return {"bytes": 4.0 * T * hkv * (row + values) + 2.0 * T * hq * values + 8.0 * T,
                "flops": 8.0 * T * (hq + 2 * hkv) * dh}
    keys = sum(min(x, case["window"] or x) for x in _ragged(case["n"], case["longest"]))
    return {"bytes": 2.0 * keys * hkv * row + 2.0 * case["n"] * case["hq"] * values + 4.0 * keys / case["page"],
            "flops": 4.0 * keys * case["hq"] * dh}


# ---- the definitions in 64 bits --------------------------------------------------

def _exact_rows(case, x):
    """What f32 rows [..., dh] become on a page, in 64 bits, from the definition."""
    x = x.double()

    def scale(most):  # the least number of 8 bits' length with scale * most >= the row's largest
        f, e = torch.frexp(x.abs().amax(-1) / most)
        return torch.ldexp(torch.ceil(f * 256.0) / 256.0, e).clamp(min=LEAST)[..., None]

    if case["bits"] == 8:
        s = scale(127.0)
        return torch.round(x / s) * s
    s = scale(1016.0)[..., None]
    g = x.reshape(*x.shape[:-1], -1, 32)
    top, bottom = g.max(-1, keepdim=True).values, g.min(-1, keepdim=True).values
    far = torch.where(top >= -bottom, top, bottom)
    step = -torch.sign(far + (far == 0)) * torch.ceil(far.abs() / s / 8.0).clamp(min=1.0) * s
    return (torch.clamp(torch.round(g / step), -8.0, 7.0) * step).reshape(x.shape)


def _exact_page(case, pool, table, t, per_seq, h, values):
    """Tokens t of one sequence and head in 64 bits, out of the pages' bytes."""
    page, rb, G = case["page"], _row_bytes(case), _subs(case)
    at = torch.from_numpy(table[(t // page) % per_seq].astype(np.int64)).cuda() * pool.shape[1]
    r = torch.from_numpy((t % page).astype(np.int64)).cuda()
    flat = pool.view(-1)
    n = flat[(at + (h * page + r) * rb)[:, None] + torch.arange(rb, device="cuda")].long()
    meta = at + case["hkv"] * page * rb + (h * (page // 16) + r // 16) * (16 * G + 32)
    low, high = (flat[meta + 16 * G + 2 * (r % 16) + i].int() for i in (0, 1))
    s = (low << 16 | high << 24).view(torch.float32).double()[:, None]
    if case["bits"] == 8:
        return (n.double() - 128.0) * s
    table4 = torch.tensor([[b % 16 - 8, b // 16 - 8] for b in range(256)], dtype=torch.float64, device="cuda")
    g = torch.arange(G, device="cuda")
    place = g * 16 + (r % 16)[:, None] if values else (r % 16)[:, None] * G + (g % 4 * (G // 4) + g // 4 if G >= 4 else g)
    sub = flat[meta[:, None] + place].double() - 128.0
    return (table4[n].reshape(len(t), G, 32) * sub[..., None]).reshape(len(t), -1) * s


def _exact_attend(case, seed):
    st = _prepare_attend(case, seed)
    lens, table = st["len"].cpu().numpy(), st["table"].cpu().numpy()
    group = case["hq"] // case["hkv"]
    out = torch.zeros(case["n"], case["hq"], case["dh"], dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        t = np.arange(max(0, length - case["window"]) if case["window"] else 0, length)
        for h in range(case["hkv"]):
            k, v = (_exact_page(case, st[x], table[b], t, st["per_seq"], h, x == "v") for x in "kv")
            s = st["q"][b, h * group:(h + 1) * group].double() @ k.t()
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            out[b, h * group:(h + 1) * group] = torch.softmax(s, -1) @ v
    return out.view(case["n"], -1)


def _exact_produce(case, seed):
    st = _prepare_produce(case, seed)
    theta, rot = ROPE[case["dh"]]
    half = rot // 2
    freq = np.array([theta ** (-2.0 * j / rot) for j in range(half)]).astype(np.float32)
    ang = st["pos"].cpu().numpy().astype(np.float32)[:, None] * freq  # (32 bits, as the definition says)
    turn = torch.polar(torch.ones(ang.shape, dtype=torch.float64), torch.from_numpy(ang.astype(np.float64))).cuda()

    def norm(x, w):
        x = x.double()
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (w.double() if w is not None else 1.0)

    def rope(x):
        z = torch.complex(x[..., :half].contiguous(), x[..., half:rot].contiguous()) * turn[:, None]
        return torch.cat([z.real, z.imag, x[..., rot:]], -1)

    return {"q": rope(norm(st["q"], st["q_norm"])), "k": _exact_rows(case, rope(norm(st["k"], st["k_norm"])).float()),
            "v": _exact_rows(case, norm(st["v"], None).float())}


def _exact_store(case, seed):
    st = _prepare_store(case, seed)
    return {x: _exact_rows(case, st[x]) for x in "kv"}


def _exact_gather(case, seed):
    st = _prepare_gather(case, seed)
    table, t = st["table"].cpu().numpy()[1], np.arange(case["rows"])
    return {x: torch.stack([_exact_page(case, st[x], table, t, st["per_seq"], h, x == "v") for h in range(case["hkv"])], 1)
            for x in "kv"}


def exact(case, seed):
    return {"attend": _exact_attend, "produce": _exact_produce, "store": _exact_store,
            "gather": _exact_gather}[case["kind"]](case, seed)
