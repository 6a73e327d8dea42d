"""The operators of a paged key-value cache, as timed cases.

A server keeps the keys and values of many sequences in pages of one pool. Each
step maps the step's tokens to pages (kind "map"), writes their keys and values
there beside the queries it makes (kind "produce"), attends with one new token
of every sequence (kind "attend"), and copies a cached prefix out in order for
the prompt attention that continues it (kind "gather").

The widths are Gemma-4-E2B's (8 query heads over 1 kv head; head_dim 256 with a
512-key window, 512 with full context) and groups of other counts. Token counts,
contexts and page sizes are free. Pages are held in 32 bits or in bfloat16; the
rest is in 32 bits.

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

EPS = 1e-6
NO_ROW = -1  # 0xFFFFFFFF: a token row that has no slot, or no token
SEQ_END = -1  # 0xFFFFFFFF as a sequence's new tokens: it ends
WINDOW = 512
ROPE = {64: (10000.0, 64), 128: (10000.0, 128), 256: (10000.0, 256), 512: (1000000.0, 128)}  # head_dim: theta, rotated
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one chat's step on a sliding layer, its window full: the smallest attention call
        {"name": "attend_one_sliding", "kind": "attend", "dh": 256, "hq": 8, "hkv": 1, "type": "f32", "page": 16,
         "n": 1, "longest": 2048, "window": WINDOW, "cap": 0.0},
        # one chat's step on a global layer, far into a long document
        {"name": "attend_one_32k", "kind": "attend", "dh": 512, "hq": 8, "hkv": 1, "type": "f32", "page": 64,
         "n": 1, "longest": 32768, "window": 0, "cap": 0.0},
        # a server's step over chats of different lengths
        {"name": "attend_batch_f32", "kind": "attend", "dh": 512, "hq": 8, "hkv": 1, "type": "f32", "page": 16,
         "n": 16, "longest": 8192, "window": 0, "cap": 0.0},
        # the sliding layers of a larger batch, their windows in rings of pages
        {"name": "attend_batch_sliding", "kind": "attend", "dh": 256, "hq": 8, "hkv": 1, "type": "bf16", "page": 32,
         "n": 64, "longest": 8192, "window": WINDOW, "cap": 0.0},
        # long documents, up to the model's whole context
        {"name": "attend_long_bf16", "kind": "attend", "dh": 512, "hq": 8, "hkv": 1, "type": "bf16", "page": 64,
         "n": 8, "longest": 131072, "window": 0, "cap": 0.0},
        # many short chats of a model with several kv heads and a score cap
        {"name": "attend_many_grouped", "kind": "attend", "dh": 128, "hq": 16, "hkv": 4, "type": "bf16", "page": 16,
         "n": 128, "longest": 2000, "window": 0, "cap": 30.0},
        # the new tokens of a decode step of 64 chats
        {"name": "produce_step", "kind": "produce", "dh": 512, "hq": 8, "hkv": 1, "type": "bf16", "page": 32,
         "n": 64, "tokens": 64, "past": 1024},
        # prompts of several requests, packed
        {"name": "produce_prompts", "kind": "produce", "dh": 256, "hq": 8, "hkv": 1, "type": "f32", "page": 16,
         "n": 7, "tokens": 4099, "past": 0},
        # a decode step's pages and slots
        {"name": "map_step", "kind": "map", "n": 64, "page": 16, "longest": 8192, "tokens": 0, "ring": False},
        # a step that admits prompts, ends sequences and goes on with the others
        {"name": "map_admit", "kind": "map", "n": 512, "page": 32, "longest": 8192, "tokens": 65536, "ring": False},
        # a short system prompt ahead of a new question
        {"name": "gather_short", "kind": "gather", "dh": 256, "hkv": 1, "type": "f32", "page": 16, "rows": 700},
        # the next turn on a long document
        {"name": "gather_long", "kind": "gather", "dh": 512, "hkv": 1, "type": "bf16", "page": 64, "rows": 32768},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "produce", "map", "gather"])
    kv, page = rng.choice(["f32", "bf16"]), rng.choice([16, 32, 64, 128, 256])
    if kind == "map":
        n = _log(rng, 1, 1024)
        return {"kind": kind, "n": n, "page": page, "longest": _log(rng, 16, 16384),
                "tokens": rng.choice([0, _log(rng, n, 65536)]), "ring": rng.choice([False, False, True])}
    dh = rng.choice([64, 128, 256, 256, 512, 512])
    hq, hkv = rng.choice([(8, 1), (8, 1), (8, 2), (16, 4), (4, 4), (16, 1), (3, 1)])
    if kind == "gather":
        return {"kind": kind, "dh": dh, "hkv": hkv, "type": kv, "page": page, "rows": _log(rng, 1, 32768 // hkv)}
    if kind == "produce":
        tokens = _log(rng, 1, 4096)
        n = _log(rng, 1, tokens)
        return {"kind": kind, "dh": dh, "hq": hq, "hkv": hkv, "type": kv, "page": page, "n": n, "tokens": tokens,
                "past": rng.choice([0, _log(rng, 1, 1024)])}
    n, longest = _log(rng, 1, 128), _log(rng, 1, 131072)
    while n * longest * hkv * dh > 1 << 28:  # about a quarter of attend_long_bf16's rows, in the plain form's layout
        longest = (longest + 1) // 2
    return {"kind": kind, "dh": dh, "hq": hq, "hkv": hkv, "type": kv, "page": page, "n": n, "longest": longest,
            "window": rng.choice([0, 0, WINDOW, _log(rng, 1, 4096)]), "cap": rng.choice([0.0, 0.0, 30.0])}


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
    """Whole numbers as the device's 32-bit words (0xFFFFFFFF is -1)."""
    return torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()


def _pages_of(lens, page, per_seq):
    return [min(-(-x // page), per_seq) for x in lens]


def _tables(d, lens, page, per_seq, spare):
    """Each sequence's pages, out of a pool in shuffled order, and the pages left: (table [n, per_seq], free, pages)."""
    used = _pages_of(lens, page, per_seq)
    total = sum(used) + spare
    order = d.host.permutation(total).astype(np.int64)
    table = np.full((len(lens), per_seq), NO_ROW, np.int64)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    return table, order[at:], total


def _pool(d, kv, total, page, hkv, dh, unit):
    """A pool of pages, filled a piece at a time: unit-RMS key rows or plain values."""
    pool = torch.empty((total, page, hkv, dh), dtype=TYPES[kv], device="cuda")
    step = max(1, (1 << 27) // (page * hkv * dh))
    for i in range(0, total, step):
        part = pool[i:i + step]
        part.copy_((d.unit_rows if unit else d.normal)(*part.shape))
    return pool


def _attend_lengths(case):
    return _ragged(case["n"], case["longest"])


def _prepare_attend(case, seed):
    d, page, n, window = _Draws(seed), case["page"], case["n"], case["window"]
    lens = d.shuffled(_attend_lengths(case))
    longest = max(lens)
    # a window's pages are a ring; a full context has a page for every token
    per_seq = -(-(window or longest) // page)
    table, _, total = _tables(d, lens, page, per_seq, 3)
    k = _pool(d, case["type"], total, page, case["hkv"], case["dh"], True)
    v = _pool(d, case["type"], total, page, case["hkv"], case["dh"], False)
    # a query norm's weight of a quarter: scores of a few units, as trained heads have
    q = 0.25 * d.unit_rows(n, case["hq"], case["dh"])
    return {"case": case, "q": q, "k": k, "v": v, "table": _i32(table), "len": _i32(lens), "total": total,
            "per_seq": per_seq, "longest": longest, "out": torch.empty(n, case["hq"] * case["dh"], device="cuda")}


def _prepare_produce(case, seed):
    d, page, n, dh = _Draws(seed), case["page"], case["n"], case["dh"]
    new = d.shuffled(_prompts(n, case["tokens"]))
    past = d.shuffled(_ragged(n, case["past"])) if case["past"] else [0] * n
    lens = [a + b for a, b in zip(past, new)]
    per_seq = -(-max(lens) // page)
    table, _, total = _tables(d, lens, page, per_seq, 3)
    pos = np.concatenate([np.arange(a, a + b) for a, b in zip(past, new)])
    seq = np.repeat(np.arange(n), new)
    slots = table[seq, pos // page] * page + pos % page
    T, hq, hkv = case["tokens"], case["hq"], case["hkv"]
    return {"case": case, "k_pool": _pool(d, case["type"], total, page, hkv, dh, True),
            "v_pool": _pool(d, case["type"], total, page, hkv, dh, False), "q": d.normal(T, hq, dh),
            "k": 2.0 * d.normal(T, hkv, dh), "v": 3.0 * d.normal(T, hkv, dh), "q_norm": 1.0 + 0.1 * d.normal(dh),
            "k_norm": 1.0 + 0.1 * d.normal(dh), "pos": _i32(pos), "slots": _i32(slots), "total": total,
            "q_out": torch.empty(T, hq, dh, device="cuda")}


def _map_step(case):
    """(tokens cached, tokens new) of every sequence. Without `tokens` each gets one; with them an eighth of the
    sequences end, a quarter are prompts that start, and the others get one token."""
    n = case["n"]
    lens = _ragged(n, case["longest"])
    if not case["tokens"]:
        return lens, [1] * n
    ends, starts = n // 8, max(1, n // 4)
    goes_on = n - ends - starts
    prompts = _prompts(starts, max(starts, case["tokens"] - goes_on))
    return lens[:n - starts] + [0] * starts, [SEQ_END] * ends + [1] * goes_on + prompts


def _prepare_map(case, seed):
    d, page, n = _Draws(seed), case["page"], case["n"]
    steps = d.shuffled(list(zip(*_map_step(case))))
    lens, new = [a for a, _ in steps], [b for _, b in steps]
    after = [a + max(0, b) for a, b in steps]
    per_seq = -(-WINDOW // page) + 1 if case["ring"] else -(-max(after) // page) + 1
    more = sum(_pages_of(after, page, per_seq)) - sum(_pages_of(lens, page, per_seq))
    table, free, total = _tables(d, lens, page, per_seq, more + 5)
    ring = np.full(total, 0, np.int64)  # the pages free, in a ring of as many places as there are pages
    first = int(d.host.randint(total))
    ring[(first + np.arange(len(free))) % total] = free
    rows = sum(max(0, b) for b in new)
    rows = rows if not case["tokens"] else -(-rows // 64) * 64  # a packed batch is padded
    return {"case": case, "table": _i32(table), "len": _i32(lens), "new": _i32(new), "free": _i32(ring),
            "state": _i32([first, len(free)]), "rows": rows, "total": total, "per_seq": per_seq,
            "out": {"slots": _i32(np.zeros(rows)), "positions": _i32(np.zeros(rows)),
                    "row_start": _i32(np.zeros(n + 1)), "added": _i32(np.zeros(n)), "len": _i32(np.zeros(n)),
                    "state": _i32(np.zeros(2))}}


def _prepare_gather(case, seed):
    d, page, rows = _Draws(seed), case["page"], case["rows"]
    lens = [rows // 3, rows, rows // 2]  # the sequence between two others
    per_seq = -(-rows // page)
    table, _, total = _tables(d, lens, page, per_seq, 3)
    hkv, dh = case["hkv"], case["dh"]
    return {"case": case, "k": _pool(d, case["type"], total, page, hkv, dh, True),
            "v": _pool(d, case["type"], total, page, hkv, dh, False), "table": _i32(table), "len": _i32(lens),
            "total": total, "per_seq": per_seq, "k_out": torch.empty(rows, hkv, dh, device="cuda"),
            "v_out": torch.empty(rows, hkv, dh, device="cuda")}


def prepare(case, seed):
    state = {"attend": _prepare_attend, "produce": _prepare_produce, "map": _prepare_map,
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
    """The argument blocks of a state's call, which a program fills once and keeps."""
    g4a, ctx = _library()
    case = state["case"]
    kind = case["kind"]

    def cache(k, v, **more):
        return g4a.PagedCache(k_pages=k.data_ptr(), v_pages=v.data_ptr(), page_size=case["page"], Hkv=case["hkv"],
                              Dh=case["dh"], n_pages=state["total"], kv_type=g4a.KV_TYPES[case["type"]], **more)

    if kind == "map":
        o = state["out"]
        pages = g4a.PagedCache(block_table=state["table"].data_ptr(), kv_len=state["len"].data_ptr(),
                               n_seqs=case["n"], pages_per_seq=state["per_seq"], n_pages=state["total"],
                               page_size=case["page"], ring=case["ring"])
        args = g4a.PageMapArgs(new_len=state["new"].data_ptr(), free_pages=state["free"].data_ptr(),
                               free_state=state["state"].data_ptr(), free_cap=state["total"], rows=state["rows"],
                               slots=o["slots"].data_ptr(), positions=o["positions"].data_ptr(),
                               row_start=o["row_start"].data_ptr(), added=o["added"].data_ptr(),
                               kv_len_out=o["len"].data_ptr(), free_state_out=o["state"].data_ptr())
        return functools.partial(ctx.page_map, pages, args)
    if kind == "produce":
        theta, rot = ROPE[case["dh"]]
        args = g4a.PagedProducerArgs(**{n: state[n].data_ptr() for n in ("q", "k", "v", "q_norm", "k_norm", "q_out")},
                                     positions=state["pos"].data_ptr(), slots=state["slots"].data_ptr(),
                                     T=case["tokens"], Hq=case["hq"], rotary_dim=rot, theta=theta, eps=EPS)
        return functools.partial(ctx.attn_producer_paged, cache(state["k_pool"], state["v_pool"]), args)
    pages = cache(state["k"], state["v"], block_table=state["table"].data_ptr(), kv_len=state["len"].data_ptr(),
                  n_seqs=state["len"].numel(), pages_per_seq=state["per_seq"], ring=bool(case.get("window")))
    if kind == "gather":
        return functools.partial(ctx.kv_gather_paged, pages, 1, 0, case["rows"], state["k_out"].data_ptr(),
                                 state["v_out"].data_ptr())
    args = g4a.PagedAttnArgs(q=state["q"].data_ptr(), out=state["out"].data_ptr(), Hq=case["hq"], scale=1.0,
                             sliding_window=case["window"], attn_softcap=case["cap"])
    return functools.partial(ctx.attention_paged, pages, args)


def _run_own(state):
    if "call" not in state:
        state["call"] = _calls(state)
    state["call"]()
    kind = state["case"]["kind"]
    if kind == "attend":
        return state["out"]
    if kind == "produce":
        return {"q": state["q_out"], "k": state["k_pool"], "v": state["v_pool"]}
    if kind == "gather":
        return {"k": state["k_out"], "v": state["v_out"]}
    return {**state["out"], "table": state["table"], "free": state["free"]}


# ---- the same in elementary operations ------------------------------------------

def _rows(state, seq, pos):
    """Row of the pool that holds token `pos` of sequence `seq`."""
    page = state["case"]["page"]
    return state["table"].long()[seq, (pos // page) % state["per_seq"]] * page + pos % page


def _attend(state):
    case = state["case"]
    n, hq, hkv, dh, window = case["n"], case["hq"], case["hkv"], case["dh"], case["window"]
    lens = state["len"].long()[:, None]
    span = min(state["longest"], window or state["longest"])
    pos = torch.arange(span, device="cuda")[None] + ((lens - span).clamp(min=0) if window else 0)
    seen = (pos < lens) & (pos >= lens - window) if window else pos < lens
    rows = _rows(state, torch.arange(n, device="cuda")[:, None], torch.where(seen, pos, (lens - 1).clamp(min=0)))
    k, v = (state[x].view(-1, hkv, dh)[rows].float().transpose(1, 2).contiguous() for x in "kv")  # [n, hkv, span, dh]
    q = state["q"].view(n, hkv, hq // hkv, dh).transpose(2, 3).contiguous()
    s = torch.matmul(k, q)  # [n, hkv, span, group]
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    seen = seen[:, None, :, None]
    s = torch.where(seen, s, -math.inf)
    e = torch.exp(s - s.amax(2, keepdim=True))
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


def _produce(state):
    dh, pos, slots = state["case"]["dh"], state["pos"], state["slots"].long()
    k, v = state["k_pool"], state["v_pool"]
    k.view(-1, *k.shape[2:])[slots] = _turn(_rms(state["k"], state["k_norm"]), pos, dh).to(k.dtype)
    v.view(-1, *v.shape[2:])[slots] = _rms(state["v"]).to(v.dtype)
    return {"q": _turn(_rms(state["q"], state["q_norm"]), pos, dh), "k": k, "v": v}


def _map(state):
    case = state["case"]
    n, page, per_seq, cap, rows = case["n"], case["page"], state["per_seq"], state["total"], state["rows"]
    lens, new, table, free = (state[x].long() for x in ("len", "new", "table", "free"))
    first, count = state["state"].long()
    ends = new == SEQ_END
    want = torch.where(ends, 0, new)
    fits = (lens + want <= per_seq * page) | case["ring"]

    def pages(x):
        return ((x + page - 1) // page).clamp(max=per_seq)

    had = pages(lens)
    need = torch.where(fits, pages(lens + want) - had, 0)
    taken = need.cumsum(0)
    goes = fits & ((need == 0) | (taken <= count))
    goes = goes & (torch.where(goes, want, 0).cumsum(0) <= rows)
    added = torch.where(goes, want, 0)
    need = torch.where(goes, need, 0)
    start = torch.cat([added.new_zeros(1), added.cumsum(0)])
    base = need.cumsum(0) - need
    # new pages into the tables, in order of the ring
    col = torch.arange(per_seq, device="cuda")[None]
    fresh = (col >= had[:, None]) & (col < (had + need)[:, None])
    out_table = torch.where(fresh, free[(first + base[:, None] + col - had[:, None]) % cap], table)
    # the pages of ended sequences to the ring's end, sequence by sequence
    gone = ends[:, None] & (col < had[:, None])
    at = torch.where(gone, (first + count + gone.flatten().cumsum(0).view(n, per_seq) - 1) % cap, cap)
    out_free = torch.cat([free, free.new_zeros(1)]).scatter(0, at.flatten(), table.flatten())[:cap]
    # token rows
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(start[1:].contiguous(), row, right=True).clamp(max=n - 1)
    pos = lens[seq] + row - start[seq]
    slots = out_table[seq, (pos // page) % per_seq] * page + pos % page
    live = row < start[-1]
    # a ring keeps the last of a sequence's tokens
    kept = live & (pos + per_seq * page >= (lens + added)[seq]) if case["ring"] else live
    return {"slots": torch.where(kept, slots, NO_ROW).int(), "positions": torch.where(live, pos, NO_ROW).int(),
            "row_start": start.int(), "added": added.int(), "len": torch.where(ends, 0, lens + added).int(),
            "state": torch.stack([(first + need.sum()) % cap, count - need.sum() + gone.sum()]).int(),
            "table": out_table.int(), "free": out_free.int()}


def _gather(state):
    case = state["case"]
    rows = _rows(state, 1, torch.arange(case["rows"], device="cuda"))
    return {x: state[x].view(-1, case["hkv"], case["dh"])[rows].float() for x in "kv"}


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend, "produce": _produce, "map": _map, "gather": _gather}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "map":
        lens, new = _map_step(case)
        tokens = sum(max(0, x) for x in new)
        # lengths, new counts, added counts; a slot and a position a token; a page's number read and written
        return {"bytes": 16.0 * len(lens) + 8.0 * tokens + 8.0 * tokens / case["page"], "flops": float(tokens)}
    hkv, dh, width = case["hkv"], case["dh"], 4 if case["type"] == "f32" else 2
    if kind == "gather":
        return {"bytes": 2.0 * case["rows"] * hkv * dh * (width + 4), "flops": 0.0}
    if kind == "produce":
        T, hq = case["tokens"], case["hq"]
        values = T * (hq + 2 * hkv) * dh
        return {"bytes": 4.0 * (values + T * hq * dh) + 2.0 * width * T * hkv * dh + 8.0 * T, "flops": 8.0 * values}
    keys = sum(min(x, case["window"] or x) for x in _attend_lengths(case))
    return {"bytes": 2.0 * width * keys * hkv * dh + 8.0 * case["n"] * case["hq"] * dh + 4.0 * keys / case["page"],
            "flops": 4.0 * keys * case["hq"] * dh}


# ---- the definitions in 64 bits --------------------------------------------------

def _exact_attend(case, seed):
    st = _prepare_attend(case, seed)
    lens, table = st["len"].cpu().numpy(), st["table"].cpu().numpy()
    group, page = case["hq"] // case["hkv"], case["page"]
    out = torch.zeros(case["n"], case["hq"], case["dh"], dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        t = np.arange(max(0, length - case["window"]) if case["window"] else 0, length)
        rows = torch.from_numpy(table[b, (t // page) % st["per_seq"]].astype(np.int64) * page + t % page).cuda()
        for h in range(case["hkv"]):
            k, v = (st[x].view(-1, case["hkv"], case["dh"])[:, h][rows].double() for x in "kv")
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

    slots = st["slots"].long()
    k, v = st["k_pool"].double(), st["v_pool"].double()
    k.view(-1, *k.shape[2:])[slots] = rope(norm(st["k"], st["k_norm"]))
    v.view(-1, *v.shape[2:])[slots] = norm(st["v"], None)
    return {"q": rope(norm(st["q"], st["q_norm"])), "k": k, "v": v}


def _exact_gather(case, seed):
    st = _prepare_gather(case, seed)
    table, page = st["table"].cpu().numpy()[1], case["page"]
    whole = [st[x][torch.from_numpy(table[:-(-case["rows"] // page)].astype(np.int64)).cuda()] for x in "kv"]
    return {x: p.reshape(-1, case["hkv"], case["dh"])[:case["rows"]].double() for x, p in zip("kv", whole)}


def exact(case, seed):
    if case["kind"] == "map":  # whole numbers
        return None
    return {"attend": _exact_attend, "produce": _exact_produce, "gather": _exact_gather}[case["kind"]](case, seed)
