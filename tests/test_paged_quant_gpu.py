"""Pages of 8 and 4 bits on the GPU, through the C-ABI: rows written and read back to the byte, by slot and by the
producer; attention and the gather against 64-bit forms on what the pages stand for, at the lengths, windows, tables and
values where they can go wrong; together as a server runs them, eagerly and as replayed graphs. Bytes that hold no token
are random (NaN and infinite scales among them) and stay as they are."""
import numpy as np
import pytest

import g4a
import paged_ref as ref
import quant_ref as quant
from test_paged_gpu import EDGES, Server, _close, say

pytestmark = pytest.mark.gpu

TYPES = ["i8", "i4"]


class Paged:
    """Pools of seeded tokens for sequences of the given lengths, on shuffled pages, random bytes elsewhere.
    `spread`: rows of magnitudes 2^-spread to 2^spread."""

    def __init__(self, ctx, lens, *, dh, hkv=1, kv_type="i4", page=16, ring=False, per_seq=None, stride=0, seed=0, unit=0.25,
                 spread=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.page, self.ring, self.type, self.hkv, self.dh = ctx, page, ring, kv_type, hkv, dh
        lens = [int(x) for x in lens]
        per_seq = per_seq or max(1, -(-max(lens + [1]) // page))
        used = [min(-(-x // page), per_seq) for x in lens]
        self.n_pages = sum(used) + 3
        order = rng.permutation(self.n_pages).astype(np.uint32)
        self.table = np.full((len(lens), per_seq), ref.NO_ROW, np.uint32)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = order[at:at + u]
            at += u
        self.lens = np.array(lens, np.uint32)
        size = quant.page_bytes(dh, hkv, page, kv_type)
        self.bytes = [rng.integers(0, 256, (self.n_pages, stride or size), dtype=np.uint8) for _ in range(2)]
        for i, buf in enumerate(self.bytes):
            for b, n in enumerate(lens):
                t = np.arange(max(0, n - per_seq * page) if ring else 0, n if ring else min(n, per_seq * page))
                x = rng.standard_normal((len(t), hkv, dh))
                if i == 0:
                    x /= np.sqrt((x ** 2).mean(-1, keepdims=True))
                if spread:
                    x *= 2.0 ** rng.uniform(-spread, 0 if i == 0 else spread, (len(t), hkv, 1))
                self.put(i, self.table[b, (t // page) % per_seq], t % page, x)
        self.dev = [ctx.upload(x) for x in self.bytes]
        self.dtable, self.dlen = ctx.upload(self.table), ctx.upload(self.lens)
        self.cache = g4a.PagedCache(k_pages=self.dev[0].ptr, v_pages=self.dev[1].ptr, block_table=self.dtable.ptr,
                                    kv_len=self.dlen.ptr, page_stride=stride, n_seqs=len(lens), pages_per_seq=per_seq,
                                    n_pages=self.n_pages, page_size=page, Hkv=hkv, Dh=dh,
                                    kv_type=g4a.KV_TYPES[kv_type], ring=int(ring))
        self.rng, self.unit = rng, unit

    def put(self, which, pages, rows, x):
        quant.pack(self.bytes[which], pages, rows, x, self.dh, self.hkv, self.page, self.type, which == 1)

    def upload(self):
        for d, x in zip(self.dev, self.bytes):
            self.ctx.h2d(d.ptr, x)

    def values(self):
        """The pools as the host has them, as f32 values [pages, page, hkv, dh]."""
        return [quant.unpack(x, self.dh, self.hkv, self.page, self.type, i == 1) for i, x in enumerate(self.bytes)]

    def queries(self, hq):
        q = self.rng.standard_normal((len(self.lens), hq, self.dh)).astype(np.float32)
        return q * np.float32(self.unit) / np.sqrt((q ** 2).mean(-1, keepdims=True))

    def attend(self, q, window=0, scale=1.0, cap=0.0, ctx=None):
        ctx = ctx or self.ctx
        dq, out = self.ctx.upload(q), self.ctx.upload(np.full((q.shape[0], q[0].size), 7.0, np.float32))
        try:
            ctx.attention_paged(self.cache, g4a.PagedAttnArgs(q=dq.ptr, out=out.ptr, Hq=q.shape[1], scale=scale,
                                                              sliding_window=window, attn_softcap=cap))
            ctx.sync()
            return out.to_host()
        finally:
            dq.free()
            out.free()

    def want(self, q, window=0, scale=1.0, cap=0.0):
        with np.errstate(invalid="ignore"):
            return quant.attention(q, *self.values(), self.table, self.lens, page=self.page, ring=self.ring,
                                   n_pages=self.n_pages, window=window, scale=scale, cap=cap)

    def free(self):
        for d in (*self.dev, self.dtable, self.dlen):
            d.free()


def _check(ctx, lens, hq, what, window=0, scale=1.0, cap=0.0, **kw):
    say(f"{what}: lens {list(lens)[:8]} hq {hq} window {window} cap {cap} {kw}")
    c = Paged(ctx, lens, **kw)
    q = c.queries(hq)
    got = c.attend(q, window, scale, cap)
    want, bound = c.want(q, window, scale, cap)
    _close(got, want, bound, what)
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[b].any(), "a sequence without tokens gives zeros"
    c.free()
    return got


# ---- rows written and read by slot ---------------------------------------------------

def _rows(T, hkv, dh, seed):
    """Rows of all kinds: plain, zero, of one value, with halves of steps, tiny, huge, of mixed magnitudes, not finite."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, hkv, dh)).astype(np.float32)
    kinds = [lambda r: 0 * r, lambda r: np.full_like(r, -2.5), lambda r: -np.abs(r), lambda r: r * 1e-39, lambda r: r * 1e37,
             lambda r: np.rint(r * 8) / 2, lambda r: np.where(np.arange(dh) % 7 == 0, 4.0, np.rint(r * 4) / 4),
             lambda r: (r * 10.0 ** rng.uniform(-30, 30, dh)).astype(np.float32), lambda r: np.where(np.arange(dh) % 32 == 5, r, 0),
             lambda r: np.where(np.arange(dh) == dh // 3, np.nan, r), lambda r: np.where(np.arange(dh) == dh - 1, -np.inf, r),
             lambda r: np.where(np.arange(dh) % 2 == 0, 127.0, rng.integers(-254, 255, dh) / 2),
             lambda r: np.where(np.arange(dh) % 32 < 2, [(-1) ** i * 8.0 for i in range(dh)], rng.integers(-16, 17, dh) / 2)]
    with np.errstate(all="ignore"):
        for i in range(0, T, 3):
            for h in range(hkv):
                x[i, h] = kinds[(i // 3 + h) % len(kinds)](x[i, h])
    return x


def _pools(ctx, n_pages, dh, hkv, page, kv_type, stride, seed):
    rng = np.random.default_rng(seed)
    if kv_type in TYPES:
        bufs = [rng.integers(0, 256, (n_pages, stride or quant.page_bytes(dh, hkv, page, kv_type)), dtype=np.uint8) for _ in "kv"]
    else:
        width = stride or page * hkv * dh
        bufs = [ref.pack(rng.standard_normal((n_pages, width)).astype(np.float32), kv_type) for _ in "kv"]
    dev = [ctx.upload(x) for x in bufs]
    cache = g4a.PagedCache(k_pages=dev[0].ptr, v_pages=dev[1].ptr, page_stride=stride, n_pages=n_pages, page_size=page,
                           Hkv=hkv, Dh=dh, kv_type=g4a.KV_TYPES[kv_type])
    return bufs, dev, cache


def _put(buf, slots, x, dh, hkv, page, kv_type, vals):
    if kv_type in TYPES:
        quant.pack(buf, slots // page, slots % page, x, dh, hkv, page, kv_type, vals)
    else:
        buf[:, :page * hkv * dh].reshape(len(buf), page, hkv, dh)[slots // page, slots % page] = ref.pack(x, kv_type)


def _read(buf, slots, dh, hkv, page, kv_type, vals):
    if kv_type in TYPES:
        return quant.unpack(buf, dh, hkv, page, kv_type, vals)[slots // page, slots % page]
    return ref.unpack(buf[:, :page * hkv * dh].reshape(len(buf), page, hkv, dh)[slots // page, slots % page], kv_type)


@pytest.mark.parametrize("kv_type", ["f32", "bf16", "i8", "i4"])
@pytest.mark.parametrize("dh,hkv,page,stride", [(64, 1, 16, 0), (128, 3, 32, 0), (256, 1, 64, 0), (512, 2, 16, 0), (64, 5, 16, 1),
                                                (512, 1, 16, 1), (256, 8, 16, 0)])
def test_rows_are_written_and_read_by_slot(ctx, dh, hkv, page, stride, kv_type):
    if stride:
        stride = (quant.page_bytes(dh, hkv, page, kv_type) if kv_type in TYPES else page * hkv * dh) + 80
    for T in (1, 2, 3, 67, 301):
        say(f"rows T {T} heads {hkv} dh {dh} page {page} stride {stride} {kv_type}")
        n_pages = -(-T // page) + 2
        bufs, dev, cache = _pools(ctx, n_pages, dh, hkv, page, kv_type, stride, T)
        slots = np.random.default_rng(T).permutation(n_pages * page)[:T].astype(np.uint32)
        if T > 2:
            slots[1], slots[T - 1] = ref.NO_ROW, n_pages * page + 5
        x = [_rows(T, hkv, dh, seed) for seed in (T, T + 1)]
        if kv_type in ("f32", "bf16"):
            x = [np.nan_to_num(y, nan=1.0) for y in x]
        d = [ctx.upload(y) for y in (*x, slots)]
        out = [ctx.upload(np.full((T + 1, hkv, dh), 3.0, np.float32)) for _ in range(2)]
        live = slots < n_pages * page
        for _ in range(2):  # the second time onto rows that stand there
            ctx.kv_write_paged(cache, d[0].ptr, d[1].ptr, d[2].ptr, T)
            ctx.kv_read_paged(cache, d[2].ptr, T, out[0].ptr, out[1].ptr)
        for i in range(2):
            _put(bufs[i], slots[live], x[i][live], dh, hkv, page, kv_type, i == 1)
            got = dev[i].to_host()
            assert np.array_equal(got, bufs[i]), (i, np.argwhere(got != bufs[i])[:5])
            want = np.zeros((T + 1, hkv, dh), np.float32)
            want[T] = 3.0
            want[:T][live] = _read(bufs[i], slots[live], dh, hkv, page, kv_type, i == 1)
            assert np.array_equal(out[i].to_host(), want, equal_nan=True)
        for y in (*d, *out, *dev):
            y.free()


@pytest.mark.parametrize("kv_type", TYPES)
def test_reads_of_any_bytes(ctx, kv_type):
    """Whatever stands in a page reads as its definition says."""
    for dh, hkv, page in ((64, 2, 16), (128, 1, 32), (256, 1, 16), (512, 1, 16)):
        bufs, dev, cache = _pools(ctx, 6, dh, hkv, page, kv_type, 0, dh)
        slots = np.arange(6 * page, dtype=np.uint32)
        d, out = ctx.upload(slots), [ctx.empty((len(slots), hkv, dh)) for _ in range(2)]
        ctx.kv_read_paged(cache, d.ptr, len(slots), out[0].ptr, out[1].ptr)
        for i in range(2):
            assert np.array_equal(out[i].to_host(), _read(bufs[i], slots, dh, hkv, page, kv_type, i == 1), equal_nan=True)
        for y in (d, *out, *dev):
            y.free()


@pytest.mark.parametrize("kv_type", TYPES)
def test_long_writes(ctx, kv_type):
    for T, hkv, dh in ((5003, 2, 64), (3001, 1, 128), (2999, 1, 256), (1501, 1, 512)):
        say(f"long write {T} {hkv} {dh} {kv_type}")
        page, n_pages = 64, 90
        bufs, dev, cache = _pools(ctx, n_pages, dh, hkv, page, kv_type, 0, 1)
        slots = np.random.default_rng(T).permutation(n_pages * page)[:T].astype(np.uint32)
        x = [np.random.default_rng(i).standard_normal((T, hkv, dh)).astype(np.float32) for i in range(2)]
        d, out = [ctx.upload(y) for y in (*x, slots)], [ctx.empty((T, hkv, dh)) for _ in range(2)]
        ctx.kv_write_paged(cache, d[0].ptr, d[1].ptr, d[2].ptr, T)
        ctx.kv_read_paged(cache, d[2].ptr, T, out[0].ptr, out[1].ptr)
        for i in range(2):
            assert np.array_equal(out[i].to_host(), quant.values(x[i], kv_type))
        for y in (*d, *out, *dev):
            y.free()


# ---- the producer ---------------------------------------------------------------------

def _produce(ctx, T, hq, hkv, dh, kv_type, rot, theta, seed, *, norms=True, kv=True, page=16, stride=0, pos=None, skip=()):
    rng = np.random.default_rng(seed)
    n_pages = -(-T // page) + 4
    bufs, dev, cache = _pools(ctx, n_pages, dh, hkv, page, kv_type, stride, seed)
    q, k, v = (rng.standard_normal((T, h, dh)).astype(np.float32) * s for h, s in ((hq, 1), (hkv, 2), (hkv, 3)))
    wq, wk = (1 + 0.1 * rng.standard_normal(dh).astype(np.float32) for _ in range(2))
    slots = rng.permutation(n_pages * page)[:T].astype(np.uint32)
    pos = rng.integers(0, 40000, T).astype(np.uint32) if pos is None else np.asarray(pos, np.uint32)
    for i, what in skip:  # rows without a slot, past the pool, or without a token
        if what == "pos":
            pos[i] = ref.NO_ROW
        else:
            slots[i] = ref.NO_ROW if what == "slot" else n_pages * page + 3
    d = {n: ctx.upload(x) for n, x in dict(q=q, k=k, v=v, wq=wq, wk=wk, slots=slots, pos=pos,
                                           out=np.full(q.shape, 5.0, np.float32)).items()}
    args = g4a.PagedProducerArgs(q=d["q"].ptr, k=d["k"].ptr if kv else None, v=d["v"].ptr if kv else None,
                                 q_norm=d["wq"].ptr if norms else None, k_norm=d["wk"].ptr if norms else None,
                                 q_out=d["out"].ptr, positions=d["pos"].ptr, slots=d["slots"].ptr if kv else None, T=T,
                                 Hq=hq, rotary_dim=rot, theta=theta, eps=1e-6)
    ctx.attn_producer_paged(cache, args)
    live = pos != ref.NO_ROW
    writes = live & (slots < n_pages * page) & kv
    at = np.where(live, pos, 0)
    eps = float(np.float32(1e-6))

    want_q = np.where(live[:, None, None], ref.rope(ref.rms(q, wq, eps) if norms else q.astype(np.float64), at, rot, theta), 5.0)
    # (the bound of the same rows for f32 pages)
    _close(d["out"].to_host(), want_q, 24 * ref.HALF * np.abs(want_q).max(-1, keepdims=True) + 0 * want_q, "q")
    new = [ref.rope(ref.rms(k, wk, eps) if norms else k.astype(np.float64), at, rot, theta), ref.rms(v, None, eps)]
    for i in range(2):
        # 64-bit rows on both sides: apart by some 2^-52, so that hardly one in 2^20 rounds to another f32, and to another
        # whole number one in 2^40
        _put(bufs[i], slots[writes], new[i][writes].astype(np.float32), dh, hkv, page, kv_type, i == 1)
        got = dev[i].to_host()
        assert np.array_equal(got, bufs[i]), ("kv"[i], np.argwhere(got != bufs[i])[:5])
    for x in (*d.values(), *dev):
        x.free()


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,rot,theta", [(64, 64, 1e4), (128, 128, 1e4), (256, 256, 1e4), (512, 128, 1e6), (512, 512, 1e4),
                                          (256, 6, 1e4), (128, 0, 1e4), (512, 250, 1e4)])
def test_producer_rows(ctx, dh, rot, theta, kv_type):
    for T, hq, hkv in ((1, 8, 1), (3, 3, 2), (65, 8, 1), (37, 16, 5)):
        say(f"producer T {T} heads {hq}/{hkv} dh {dh} rot {rot} {kv_type}")
        _produce(ctx, T, hq, hkv, dh, kv_type, rot, theta, T + dh)


@pytest.mark.parametrize("T,hq,hkv,dh,kv_type", [(1500, 3, 2, 64, "i4"), (1030, 8, 1, 256, "i8"), (1100, 5, 1, 128, "i4"),
                                                 (1024, 2, 1, 512, "i4"), (8200, 4, 1, 64, "i8"), (8193, 1, 1, 256, "i4")])
def test_producer_of_long_calls(ctx, T, hq, hkv, dh, kv_type):
    _produce(ctx, T, hq, hkv, dh, kv_type, dh // 2, 1e4, T, skip=[(1, "slot"), (T // 2, "pos"), (T - 2, "past")])


def test_producer_variants(ctx):
    for kv_type in TYPES:
        _produce(ctx, 9, 8, 1, 256, kv_type, 256, 1e4, 1, norms=False)
        _produce(ctx, 9, 8, 1, 512, kv_type, 128, 1e6, 2, kv=False)
        _produce(ctx, 20, 8, 2, 128, kv_type, 128, 1e4, 3, stride=quant.page_bytes(128, 2, 16, kv_type) + 48)
        _produce(ctx, 12, 8, 1, 256, kv_type, 256, 1e4, 4, skip=[(0, "pos"), (3, "slot"), (7, "past"), (11, "pos")])
        _produce(ctx, 4, 8, 1, 512, kv_type, 128, 1e6, 5, pos=[0, 131071, (1 << 20) + 1, (1 << 24) + 2])


@pytest.mark.parametrize("kv_type", TYPES)
def test_the_same_rows_make_the_same_pages(ctx, kv_type):
    """A token's row does not depend on the batch that it is produced in."""
    T, dh, page = 70, 256, 16
    rng = np.random.default_rng(2)
    d = {n: ctx.upload(rng.standard_normal((T, h, dh)).astype(np.float32)) for n, h in (("q", 8), ("k", 1), ("v", 1))}
    slots, pos = (ctx.upload(np.arange(T, dtype=np.uint32) + x) for x in (0, 3000))
    q_out = ctx.empty((T, 8, dh))
    got = []
    for step in (T, 1, 9):
        _, dev, cache = _pools(ctx, 5, dh, 1, page, kv_type, 0, 1)
        for t in range(0, T, step):
            n, row = min(step, T - t), 4 * dh * t
            ctx.attn_producer_paged(cache, g4a.PagedProducerArgs(
                q=d["q"].ptr + 8 * row, k=d["k"].ptr + row, v=d["v"].ptr + row, q_out=q_out.ptr, positions=pos.ptr + 4 * t,
                slots=slots.ptr + 4 * t, T=n, Hq=8, rotary_dim=dh, theta=1e4, eps=1e-6))
        got.append([x.to_host() for x in dev])
        for x in dev:
            x.free()
    for other in got[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(got[0], other))
    for x in (*d.values(), slots, pos, q_out):
        x.free()


# ---- attention -------------------------------------------------------------------------

@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh", [64, 128, 256, 512])
def test_attention_at_the_edges_of_pages_and_tiles(ctx, dh, kv_type):
    _check(ctx, EDGES, 8, f"edges dh {dh} {kv_type}", dh=dh, kv_type=kv_type, seed=dh)
    _check(ctx, EDGES[::-1], 8, f"edges, page 64, dh {dh} {kv_type}", dh=dh, kv_type=kv_type, page=64, seed=dh + 1)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (4, 4), (8, 2), (5, 1), (16, 1), (16, 4), (24, 1), (40, 2), (12, 3)])
@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_of_head_groups(ctx, hq, hkv, kv_type):
    for dh in (64, 128, 256):
        _check(ctx, [70, 0, 5, 333], hq, f"{hq} over {hkv} dh {dh} {kv_type}", dh=dh, hkv=hkv, kv_type=kv_type,
               seed=hq * 10 + hkv)
    _check(ctx, [41, 200], hq, f"{hq} over {hkv} dh 512 {kv_type}", dh=512, hkv=hkv, kv_type=kv_type, seed=hq + hkv)


@pytest.mark.parametrize("window", [1, 7, 16, 100, 512])
@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_windows_and_rings(ctx, window, kv_type):
    lens = [0, 1, 5, window, window + 1, window + 15, 2 * window + 3, 1000, 2003]
    _check(ctx, lens, 8, f"window {window}", window=window, dh=256, kv_type=kv_type, seed=window)
    for more in (0, 1):
        _check(ctx, lens, 8, f"window {window} in a ring", window=window, dh=256, kv_type=kv_type, ring=True,
               per_seq=-(-window // 16) + more, seed=window + 1)
    _check(ctx, lens, 8, "a ring alone", dh=512, kv_type=kv_type, ring=True, per_seq=3, page=32, seed=window + 2)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("page,per_seq", [(16, 4), (32, 2), (64, 1), (16, 3), (16, 5)])
def test_attention_over_rings_of_about_a_part(ctx, page, per_seq, kv_type):
    for lens in ([65], [0, 1, 48, 49, 63, 64, 65, 70, 79, 80, 100, 1000]):
        for window in (0, 63, 64, 100):
            _check(ctx, lens, 8, f"ring {page} x {per_seq}", window=window, dh=256, kv_type=kv_type, page=page, ring=True,
                   per_seq=per_seq, seed=per_seq + window)


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_long_and_ragged(ctx, kv_type):
    _check(ctx, [9011], 8, "one long", dh=512, kv_type=kv_type, page=64, seed=1)
    _check(ctx, [5001, 3, 0, 4097, 1, 700, 3000], 8, "ragged", dh=256, kv_type=kv_type, seed=2)
    _check(ctx, [1 + 37 * i % 150 for i in range(300)], 4, "300 short", dh=64, hkv=2, kv_type=kv_type, seed=3)
    _check(ctx, [2000] * 5 + [1] * 40 + [900] * 5, 16, "mixed groups", dh=128, hkv=4, kv_type=kv_type, seed=4, cap=20.0)


@pytest.mark.parametrize("n,hq,hkv,dh,kv_type,longest", [
    (2100, 2, 1, 64, "i4", 40), (1025, 8, 1, 64, "i8", 20), (300, 8, 8, 64, "i4", 40), (150, 40, 5, 128, "i8", 40),
    (260, 8, 1, 512, "i4", 100), (140, 8, 1, 512, "i8", 100), (129, 4, 1, 512, "i4", 100), (65, 9, 1, 256, "i8", 300),
    (150, 8, 2, 512, "i4", 60), (257, 7, 1, 512, "i8", 60), (256, 3, 1, 512, "i8", 60)])
def test_attention_of_many_sequences(ctx, n, hq, hkv, dh, kv_type, longest):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, longest + 1, n)
    lens[[0, n // 2, n - 1]] = [5 * longest, 0, longest]
    for window in (0, 37):
        _check(ctx, lens, hq, "many", window=window, hkv=hkv, dh=dh, kv_type=kv_type, seed=n)


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_scale_softcap_and_page_stride(ctx, kv_type):
    _check(ctx, [100, 513, 31], 8, "scale", dh=256, scale=0.0625, unit=1.0, kv_type=kv_type, seed=1)
    _check(ctx, [100, 513, 31], 8, "a negative scale", dh=128, scale=-0.1, unit=1.0, kv_type=kv_type, seed=1)
    _check(ctx, [100, 513, 31], 8, "softcap", dh=512, cap=5.0, unit=1.0, kv_type=kv_type, seed=2)
    for cap in (0.7, 40.0, 1000.0):  # scores far beyond the cap, about it and far below
        _check(ctx, [100, 513, 31], 4, "softcap", dh=128, cap=cap, unit=1.0, kv_type=kv_type, seed=2)
    _check(ctx, [100, 513, 31], 8, "stride", dh=128, hkv=2, stride=quant.page_bytes(128, 2, 16, kv_type) + 48, kv_type=kv_type,
           seed=3)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,hq", [(64, 8), (128, 3), (256, 16), (512, 8), (512, 16)])
def test_attention_of_rows_of_all_magnitudes(ctx, kv_type, dh, hq):
    """Keys from 2^-20 to 1 and values from 2^-20 to 2^20 of the usual size, in parts that one wave and many take; queries
    of tiny and of huge size, with scores of the usual one."""
    for seed, lens in enumerate(([700, 33, 16], [3000], [5])):
        _check(ctx, lens, hq, "spread", dh=dh, kv_type=kv_type, spread=20, seed=seed)
    for unit, scale in ((2.0 ** -100, 2.0 ** 98), (2.0 ** 100, 2.0 ** -102)):
        _check(ctx, [100, 33], hq, "queries", dh=dh, kv_type=kv_type, unit=unit, scale=scale, seed=4)


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_leaves_out_tokens_without_a_page(ctx, kv_type):
    c = Paged(ctx, [200, 64, 90, 48], dh=256, kv_type=kv_type, seed=4)
    c.table[0, 3], c.table[0, 12], c.table[1, :], c.table[2, 0] = ref.NO_ROW, c.n_pages, 0x80000000, c.n_pages + 7
    ctx.h2d(c.dtable.ptr, c.table)
    q = c.queries(8)
    got = c.attend(q)
    want, bound = c.want(q)
    _close(got, want, bound, f"bad pages {kv_type}")
    assert not got[1].any()
    c.lens[3] = 4000  # a length past the table's end counts what the table holds
    ctx.h2d(c.dlen.ptr, c.lens)
    _close(c.attend(q), want, bound, f"a long length {kv_type}")
    c.free()


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,hq,hkv", [(64, 16, 1), (128, 3, 1), (256, 8, 2), (512, 8, 1)])
def test_attention_shows_rows_that_are_not_finite_where_visible(ctx, dh, hq, hkv, kv_type):
    """A row written with a NaN or an infinity makes its kv head's outputs NaN where it is visible, and none where it is
    behind the length or before the window."""
    bad = np.ones((1, hkv, dh), np.float32)
    bad[0, hkv - 1, 3] = np.inf
    for which in range(2):
        c = Paged(ctx, [50, 700, 120], dh=dh, hkv=hkv, kv_type=kv_type, seed=6)
        c.put(which, c.table[0:1, 1], np.array([3]), bad)       # token 19 of sequence 0
        c.put(which, c.table[1:2, 5], np.array([0]), bad * np.nan)  # token 80 of sequence 1, outside the window
        c.put(which, c.table[2:3, 7], np.array([9]), bad * np.nan)  # token 121 of sequence 2: behind its length
        c.upload()
        q = c.queries(hq)
        with np.errstate(invalid="ignore"):
            want, bound = (x.reshape(3, hq, dh) for x in c.want(q, window=100))
        got = c.attend(q, window=100).reshape(3, hq, dh)
        heads = np.arange(hq) // (hq // hkv) == hkv - 1
        assert np.isnan(got[0, heads]).all()
        rest = np.isfinite(want)
        assert rest[0, ~heads].all() and rest[1:].all()
        _close(got[rest], want[rest], bound[rest], f"not finite, {'kv'[which]}")
        c.free()


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,hq,hkv", [(64, 16, 1), (128, 3, 1), (256, 8, 1), (512, 9, 1)])
def test_attention_of_queries_that_are_not_finite(ctx, dh, hq, hkv, kv_type):
    """A NaN or an infinity in a query makes its head's row NaN and no other's, in sequences of one part and of many;
    a sequence without tokens stays zero."""
    c = Paged(ctx, [50, 700, 17, 0, 2000], dh=dh, hkv=hkv, kv_type=kv_type, seed=dh)
    q = c.queries(hq)
    want, bound = (x.reshape(5, hq, dh) for x in c.want(q))
    bad = np.zeros((5, hq), bool)
    q[1, 0, dh - 1], q[2, :, 40], q[4, hq - 1, 3], q[3] = np.nan, -np.inf, np.inf, np.nan
    bad[1, 0] = bad[2] = bad[4, hq - 1] = True
    got = c.attend(q).reshape(5, hq, dh)
    assert np.isnan(got[bad]).all() and not got[3].any()
    _close(got[~bad], want[~bad], bound[~bad], "the others")
    c.free()


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,hq", [(64, 16), (128, 3), (256, 8), (512, 9)])
def test_attention_of_queries_of_nothing(ctx, kv_type, dh, hq):
    """All zeros, the smallest numbers there are, and one value among zeros."""
    c = Paged(ctx, [50, 700, 17, 33], dh=dh, kv_type=kv_type, seed=dh)
    q = c.queries(hq)
    q[0], q[1] = 0.0, q[1] * np.float32(1e-40)
    q[2, :, 1:], q[3, 0] = 0.0, -0.0
    got = c.attend(q)
    want, bound = c.want(q)
    _close(got, want, bound, "nothing")
    c.free()


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,hq", [(64, 16), (128, 3), (256, 8), (512, 9)])
def test_attention_of_soft_caps_at_the_ends_of_f32(ctx, kv_type, dh, hq):
    """Caps beyond any score, up to f32's largest, leave scores as they are; caps down to its smallest make every score
    about 0, one of exactly 0 among them."""
    c = Paged(ctx, [100, 513, 31, 0, 7], dh=dh, kv_type=kv_type, seed=dh)
    q = c.queries(hq)
    q[2], q[4, 0] = 0.0, 0.0
    for cap in (2.0 ** 126, 2.4e38, float(np.finfo(np.float32).max), 2.0 ** -126, 2e-39, 1e-45):
        got = c.attend(q, cap=cap)
        want, bound = c.want(q, cap=cap)
        _close(got, want, bound, f"soft-cap {cap} dh {dh} {kv_type}")
    c.free()


def _values(c, b, x):
    """Sequence b's V rows are x."""
    t = np.arange(len(x))
    c.put(1, c.table[b, t // c.page], t % c.page, x[:, None])


def _sharp(c, q):
    return quant.attention_sharp(q, *c.values(), c.table, c.lens, page=c.page, n_pages=c.n_pages)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,hq", [(64, 16), (128, 3), (256, 8), (512, 9)])
def test_attention_of_values_at_the_ends_of_f32(ctx, kv_type, dh, hq):
    """V rows of 2^-110 or 2^-92 throughout, of 2^-110 ahead of 2^60 and behind it, and of 2^100, in parts that are their
    whole unit and in those that are merged."""
    c = Paged(ctx, [16, 60, 1100, 700, 900, 2000], dh=dh, kv_type=kv_type, seed=dh)
    q = c.queries(hq)
    for what, first, second in (("tiny", -110, -110), ("small", -92, -92), ("tiny, then large", -110, 60),
                                ("large, then tiny", 60, -110), ("huge", 100, 100)):
        for b, n in enumerate(c.lens):
            power = np.where(np.arange(n) < n // 2, first, second)[:, None]
            _values(c, b, c.rng.standard_normal((n, dh)) * 2.0 ** power)
        c.upload()
        _close(c.attend(q), *_sharp(c, q), f"{what} dh {dh} {kv_type}")
    c.free()


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_of_huge_values_under_rising_scores(ctx, kv_type):
    """A maximum that lags behind the scores leaves weights above 1, by up to 2^8, and no sum of 32768 tokens' V rows of
    2^108 passes f32's largest number for it. Two pages by turns: scores of 0, which a wave meets first, and of 5.4."""
    dh, page, n = 256, 64, 32768
    c = Paged(ctx, [2 * page], dh=dh, kv_type=kv_type, page=page, per_seq=n // page, seed=1)
    low, high = c.table[0, :2]
    c.table[0], c.lens[0] = np.tile([low, high], n // page // 2), n
    c.put(0, np.full(page, low), np.arange(page), np.zeros((page, 1, dh)))
    c.put(0, np.full(page, high), np.arange(page), np.full((page, 1, dh), 5.4))
    for p in (low, high):
        c.put(1, np.full(page, p), np.arange(page), c.rng.uniform(1, 2, (page, 1, dh)) * 2.0 ** 108)
    c.upload()
    ctx.h2d(c.dtable.ptr, c.table)
    ctx.h2d(c.dlen.ptr, c.lens)
    q = np.full((1, 2, dh), 1 / dh, np.float32)
    _close(c.attend(q), *_sharp(c, q), f"rising scores {kv_type}")
    c.free()


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,hq", [(64, 3), (256, 8), (512, 16)])
def test_attention_holds_the_low_parts_of_probabilities_in_long_contexts(ctx, kv_type, dh, hq):
    """9000 tokens whose weights, but for one of a tile's, lie between two fp16 numbers alike: without their low parts
    the result would be off by some ten times its bound, as the host's form shows."""
    n = 9000
    c = Paged(ctx, [n], dh=dh, kv_type=kv_type, seed=dh)
    t = np.arange(n)
    k = np.zeros((n, 1, dh))
    k[t % 16 == 0, 0, 0] = 127 / 128  # (a row of 8 bits has S = 2^-7, one of 4 bits S sub n = 1: scores of 0.677 are by q)
    c.put(0, c.table[0, t // 16], t % 16, k)
    v = c.rng.uniform(0.5, 1, (n, dh))
    v[:, 1] = 1.0  # one S for all rows, 1.015625 times a power of two
    _values(c, 0, v)
    c.upload()
    weight = (33 + 0.0146) / 65  # a weight times S and its power of two (to [64, 128)): a half step of fp16 off at 33
    q = np.zeros((1, hq, dh), np.float32)
    q[:, :, 0] = -np.log(weight) / c.values()[0][c.table[0, 0], 0, 0, 0]
    want, bound = _sharp(c, q)
    rows = c.values()[1][c.table[0, t // 16], t % 16, 0].astype(np.float64)
    p = np.where(t % 16 == 0, 1.0, weight)
    cut = (p * 65).astype(np.float16).astype(np.float64) @ rows / (65 * p.sum())
    assert np.abs(cut - want[0, :dh]).min() > 5 * bound.max(), "a form that drops the low parts would pass"
    _close(c.attend(q), want, bound, f"low parts dh {dh} {kv_type}")
    c.free()


def test_attention_is_repeatable_and_shares_pages(ctx):
    for kv_type in TYPES:
        c = Paged(ctx, [3000, 3000, 17], dh=512, page=32, kv_type=kv_type, seed=7)
        c.table[1] = c.table[0]
        ctx.h2d(c.dtable.ptr, c.table)
        q = c.queries(8)
        q[1] = q[0]
        one, two = c.attend(q), c.attend(q)
        assert np.array_equal(one, two)
        want, bound = c.want(q)
        _close(one, want, bound, "shared pages")
        c.free()


# ---- the gather ---------------------------------------------------------------------------

@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,hkv,page", [(64, 1, 16), (128, 3, 32), (256, 1, 256), (512, 2, 16)])
def test_gather_gives_tokens_in_order(ctx, dh, hkv, page, kv_type):
    for ring in (False, True):
        c = Paged(ctx, [5, 700, 90], dh=dh, hkv=hkv, kv_type=kv_type, page=page, ring=ring, seed=dh,
                  per_seq=max(1, 192 // page) if ring else None,
                  stride=0 if ring else quant.page_bytes(dh, hkv, page, kv_type) + 16)
        if not ring:
            c.table[1, 1] = c.n_pages  # a hole
            ctx.h2d(c.dtable.ptr, c.table)
        for pos0, n in ((0, 700), (0, 1), (699, 1), (17, 301), (690, 40), (800, 9)):
            say(f"gather {pos0} + {n} page {page} ring {ring}")
            out = [ctx.upload(np.full((n + 1, hkv, dh), 3.0, np.float32)) for _ in range(2)]
            ctx.kv_gather_paged(c.cache, 1, pos0, n, out[0].ptr, out[1].ptr)
            for d, pool in zip(out, c.values()):
                want = np.zeros((n + 1, hkv, dh), np.float32)
                want[n] = 3.0
                t, rows = ref.tokens(pool, c.table, 1, 700, page=page, ring=ring, n_pages=c.n_pages)
                keep = (t >= pos0) & (t < pos0 + n)
                want[t[keep] - pos0] = rows[keep]
                assert np.array_equal(d.to_host(), want)
                d.free()
        c.free()


# ---- together, as a server runs them -------------------------------------------------------

class QuantServer(Server):
    """The server's steps on pages of 8 and 4 bits; the host's mirror holds what its 64-bit rows stand for once written."""

    def __init__(self, ctx, n, dh, kv_type, window, seed):
        super().__init__(ctx, n, dh, "f32", window, seed)
        size = quant.page_bytes(dh, 1, 16, kv_type)
        for i, name in enumerate(("k_pool", "v_pool")):
            self.d[name].free()
            self.d[name] = ctx.upload(np.random.default_rng(i).integers(0, 256, (self.n_pages, size), dtype=np.uint8))
        self.cache.k_pages, self.cache.v_pages = self.d["k_pool"].ptr, self.d["v_pool"].ptr
        self.cache.kv_type = g4a.KV_TYPES[kv_type]
        self.quant = kv_type

    def check(self, rows_per_seq, attend=True):
        seen = [len(t[0]) for t in self.tokens]
        ended = self.new == ref.NO_ROW
        super().check(rows_per_seq, attend=False)  # (appends this step's rows in 64 bits, held as f32)
        for b in range(self.n):
            first = 0 if ended[b] else seen[b]
            self.tokens[b] = [np.concatenate([t[:first], quant.values(t[first:], self.quant)]) for t in self.tokens[b]]
        if not attend:
            return
        added, lens = self.d["added"].to_host(), self.d["lens"].to_host()
        got, q = self.d["out"].to_host(), self.d["q_out"].to_host()  # (queries have tests of their own)
        for b in range(self.n):
            k, v = self.tokens[b]
            if not len(k):
                assert not got[b].any()
            elif added[b]:
                row = b if rows_per_seq else int(np.sum(added[:b + 1])) - 1
                table, page = np.zeros((1, 1), np.uint32), 1 << 16
                want, bound = quant.attention(q[row:row + 1], k[None], v[None], table, lens[b:b + 1], page=page, n_pages=1,
                                              window=self.window, scale=0.1)
                _close(got[b:b + 1], want, bound, f"sequence {b} of {len(k)}")


@pytest.mark.parametrize("dh,kv_type,window", [(256, "i8", 100), (512, "i4", 0), (512, "i8", 0), (256, "i4", 100), (64, "i4", 0)])
def test_a_server_steps_eagerly_and_replayed(ctx, dh, kv_type, window):
    """Prompts of one step, then decode steps with sequences that end and start again, eagerly and as replays of one
    captured step, each checked against the definition."""
    say(f"server dh {dh} {kv_type} window {window}")
    n = 6
    s = QuantServer(ctx, n, dh, kv_type, window, dh)
    s.rows(128, 0)
    s.feed([30, 0, 17, 1, 40, 16], 128)
    s.step(attend=False)
    s.check(0, attend=False)
    s.rows(n, 1)
    s.feed([1, 1, 1, 0, 1, 1], n)
    s.step()
    s.check(1)
    ctx.capture_begin()
    s.step()
    graph = ctx.capture_end()
    for new in ([1] * 6, [1, ref.NO_ROW, 1, 1, 1, 1], [1, 1, 0, 1, ref.NO_ROW, 1], [0, 1, 1, 1, 1, ref.NO_ROW], [1] * 6):
        s.feed(new, n)
        graph.launch()
        s.check(1)
        s.feed(new if new[0] else [1] * 6, n)  # an eager step between the replays
        s.step()
        s.check(1)
    graph.free()
    for d in s.d.values():
        d.free()


def test_two_graphs_replay_beside_a_larger_call(ctx):
    """Two captured calls share the context's workspace, and a later call that needs more of it leaves theirs."""
    c = g4a.Context(0)
    small, big = (Paged(c, lens, dh=256, kv_type=t, seed=3) for lens, t in (([700, 33, 0], "i4"), ([90, 2000, 17, 5], "i8")))
    huge = Paged(c, [1500] * 24, dh=256, hkv=2, seed=4)
    runs = []
    for x in (small, big):
        q = x.queries(8)
        dq, out = c.upload(q), c.empty((len(q), 8 * 256))
        runs.append((x, q, dq, out, g4a.PagedAttnArgs(q=dq.ptr, out=out.ptr, Hq=8, scale=1.0)))
    for x, _, _, _, args in runs:
        c.attention_paged(x.cache, args)
    graphs = []
    for x, _, _, _, args in runs:
        c.capture_begin()
        c.attention_paged(x.cache, args)
        graphs.append(c.capture_end())
    for turn, (i, cut) in enumerate([(0, 0), (1, 0), (0, 200), (1, 500), (1, 0), (0, 0)]):
        x, q, _, out, args = runs[i]
        full = x.lens
        x.lens = np.maximum(full.astype(np.int64) - cut, 0).astype(np.uint32)
        c.h2d(x.dlen.ptr, x.lens)
        if turn == 2:  # a larger workspace, in between
            hq = huge.queries(16)
            want, bound = huge.want(hq)
            _close(huge.attend(hq), want, bound, "the larger call")
        c.h2d(out.ptr, np.full((len(q), 8 * 256), 7.0, np.float32))
        graphs[i].launch()
        want, bound = x.want(q)
        got = out.to_host()
        _close(got, want, bound, f"replay {turn}")
        c.attention_paged(x.cache, args)
        assert np.array_equal(out.to_host(), got), "the eager call's bits"
        x.lens = full
    for g in graphs:
        g.free()
    c.close()


def test_two_contexts_read_one_cache(ctx):
    """Two contexts, each with a stream and a workspace of its own, attend over the same pages at once."""
    c = Paged(ctx, [2000, 300, 1, 900], dh=512, kv_type="i4", seed=11)
    ctx.sync()
    other = g4a.Context(0)
    q = c.queries(8)
    alone = c.attend(q)
    dq, outs = ctx.upload(q), [ctx.empty((4, 8 * 512)) for _ in range(2)]
    ctx.sync()
    args = [g4a.PagedAttnArgs(q=dq.ptr, out=o.ptr, Hq=8, scale=1.0) for o in outs]
    for _ in range(20):
        ctx.attention_paged(c.cache, args[0])
        other.attention_paged(c.cache, args[1])
    other.sync()
    for o in outs:
        assert np.array_equal(o.to_host(), alone)
        o.free()
    other.close()
    dq.free()
    c.free()


@pytest.mark.parametrize("kv_type", TYPES)
def test_pages_past_four_gib(ctx, kv_type):
    """The same tokens in pages side by side and more than 2^32 bytes apart: produced, written, gathered, read and attended
    alike, bit for bit."""
    T, page, dh, hkv = 90, 32, 256, 2
    rng = np.random.default_rng(8)
    x = {m: ctx.upload(rng.standard_normal((T, h, dh)).astype(np.float32)) for m, h in (("q", 8), ("k", hkv), ("v", hkv))}
    table, t = np.array([[2, 0, 1]], np.uint32), np.arange(T)
    slots = (table[0, t // page] * page + t % page).astype(np.uint32)
    d = dict(table=ctx.upload(table), len=ctx.upload(np.array([T], np.uint32)), slots=ctx.upload(slots),
             pos=ctx.upload(t.astype(np.uint32)))
    got = []
    size = quant.page_bytes(dh, hkv, page, kv_type)
    for stride in (size, (1 << 32) + 64):
        pools = [ctx.empty((2 * stride + size,), np.uint8) for _ in range(2)]
        q, out, k, v, k2, v2 = (ctx.empty(s) for s in ((T, 8, dh), (1, 8 * dh), *[(T, hkv, dh)] * 4))
        cache = g4a.PagedCache(k_pages=pools[0].ptr, v_pages=pools[1].ptr, block_table=d["table"].ptr, kv_len=d["len"].ptr,
                               page_stride=stride, n_seqs=1, pages_per_seq=3, n_pages=3, page_size=page, Hkv=hkv, Dh=dh,
                               kv_type=g4a.KV_TYPES[kv_type])
        say(f"stride {stride} {kv_type}")
        ctx.attn_producer_paged(cache, g4a.PagedProducerArgs(q=x["q"].ptr, k=x["k"].ptr, v=x["v"].ptr, q_out=q.ptr,
                                                             positions=d["pos"].ptr, slots=d["slots"].ptr, T=T, Hq=8,
                                                             rotary_dim=dh, theta=1e4, eps=1e-6))
        ctx.kv_gather_paged(cache, 0, 0, T, k.ptr, v.ptr)
        ctx.attention_paged(cache, g4a.PagedAttnArgs(q=q.ptr, out=out.ptr, Hq=8, scale=0.1))
        ctx.kv_write_paged(cache, x["k"].ptr, x["v"].ptr, d["slots"].ptr, T)
        ctx.kv_read_paged(cache, d["slots"].ptr, T, k2.ptr, v2.ptr)
        got.append([y.to_host() for y in (k, v, out, k2, v2)])
        for y in (*pools, q, out, k, v, k2, v2):
            y.free()
    assert all(np.isfinite(y).all() and y.any() for y in got[0])
    assert all(np.array_equal(a, b) for a, b in zip(*got))
    for y in (*x.values(), *d.values()):
        y.free()


@pytest.mark.parametrize("kv_type", TYPES)
def test_a_prompt_continues_a_prefix_that_was_handed_over(ctx, kv_type):
    """A prefix's rows arrive in f32 and are written into slots of a page map; a prompt's second part is produced behind
    them; both are gathered and attended by g4a_attention, whose last row is what the decode attention gives."""
    rng = np.random.default_rng(9)
    dh, T0, T1, page = 512, 70, 45, 16
    n = T0 + T1
    x = [rng.standard_normal((n, h, dh)).astype(np.float32) for h in (8, 1, 1)]
    d = {m: ctx.upload(a) for m, a in dict(q=x[0], k=x[1], v=x[2]).items()}
    size = quant.page_bytes(dh, 1, page, kv_type)
    pool = [ctx.upload(rng.integers(0, 256, (12, size), dtype=np.uint8)) for _ in range(2)]
    m = {a: ctx.upload(np.asarray(b, np.uint32)) for a, b in dict(
        table=np.full((1, 10), ref.NO_ROW), lens=[0], new=[0], free=rng.permutation(12), state=[0, 12], slots=np.zeros(128),
        pos=np.zeros(128)).items()}
    cache = g4a.PagedCache(k_pages=pool[0].ptr, v_pages=pool[1].ptr, block_table=m["table"].ptr, kv_len=m["lens"].ptr,
                           n_seqs=1, pages_per_seq=10, n_pages=12, page_size=page, Hkv=1, Dh=dh, kv_type=g4a.KV_TYPES[kv_type])
    assert ctx.kv_page_bytes(cache) == size
    q_out, k_all, v_all, out, last = (ctx.empty(s) for s in ((T1, 8, dh), (n, 1, dh), (n, 1, dh), (T1, 8 * dh), (1, 8 * dh)))
    for t0, T in ((0, T0), (T0, T1)):
        ctx.h2d(m["new"].ptr, np.array([T], np.uint32))
        ctx.page_map(cache, g4a.PageMapArgs(new_len=m["new"].ptr, free_pages=m["free"].ptr, free_state=m["state"].ptr,
                                            free_cap=12, rows=T, slots=m["slots"].ptr, positions=m["pos"].ptr))
        at = t0 * dh * 4
        if t0 == 0:
            ctx.kv_write_paged(cache, d["k"].ptr, d["v"].ptr, m["slots"].ptr, T)
        else:
            ctx.attn_producer_paged(cache, g4a.PagedProducerArgs(
                q=d["q"].ptr + 8 * at, k=d["k"].ptr + at, v=d["v"].ptr + at, q_out=q_out.ptr, positions=m["pos"].ptr,
                slots=m["slots"].ptr, T=T, Hq=8, rotary_dim=128, theta=1e6, eps=1e-6))
    ctx.kv_gather_paged(cache, 0, 0, n, k_all.ptr, v_all.ptr)
    pos = np.arange(T0, n)
    k = np.concatenate([x[1][:T0], ref.rope(x[1][T0:].astype(np.float64), pos, 128, 1e6).astype(np.float32)])
    v = np.concatenate([x[2][:T0], ref.rms(x[2][T0:], None, float(np.float32(1e-6))).astype(np.float32)])
    assert np.array_equal(k_all.to_host(), quant.values(k, kv_type)) and np.array_equal(v_all.to_host(), quant.values(v, kv_type))
    ctx.attention(q_out.ptr, k_all.ptr, v_all.ptr, out.ptr, T=T1, S=n, Hq=8, Hkv=1, Dh=dh, Dv=dh, q_pos0=T0, scale=0.05)
    ctx.attention_paged(cache, g4a.PagedAttnArgs(q=q_out.ptr + (T1 - 1) * 8 * dh * 4, out=last.ptr, Hq=8, scale=0.05))
    q = q_out.to_host()[-1:]
    want, bound = quant.attention(q, quant.values(k, kv_type)[None], quant.values(v, kv_type)[None], np.zeros((1, 1), np.uint32),
                                  [n], page=1 << 16, n_pages=1, scale=0.05)
    _close(last.to_host(), want, bound, "the decode step")
    _close(out.to_host()[-1:], want, bound, "the prompt's last row")
    for a in (*d.values(), *pool, *m.values(), q_out, k_all, v_all, out, last):
        a.free()


@pytest.mark.parametrize("kv_type", TYPES)
def test_rows_move_between_caches_in_a_graph(ctx, kv_type):
    """Rows read from a cache of one type and written into one of another, captured and replayed with other slots."""
    T, dh, page, hkv = 33, 128, 16, 2
    rng = np.random.default_rng(3)
    src_buf, src, a = _pools(ctx, 5, dh, hkv, page, "bf16", 0, 1)
    dst_buf, dst, b = _pools(ctx, 6, dh, hkv, page, kv_type, 0, 2)
    slots = [ctx.empty((T,), np.uint32) for _ in range(2)]
    k, v = ctx.empty((T, hkv, dh)), ctx.empty((T, hkv, dh))

    def move():
        ctx.kv_read_paged(a, slots[0].ptr, T, k.ptr, v.ptr)
        ctx.kv_write_paged(b, k.ptr, v.ptr, slots[1].ptr, T)

    ctx.capture_begin()
    move()
    graph = ctx.capture_end()
    for turn in range(4):
        at = [rng.permutation(n * page)[:T].astype(np.uint32) for n in (5, 6)]
        for s, x in zip(slots, at):
            ctx.h2d(s.ptr, x)
        graph.launch() if turn != 2 else move()
        for i in range(2):
            _put(dst_buf[i], at[1], _read(src_buf[i], at[0], dh, hkv, page, "bf16", i == 1), dh, hkv, page, kv_type, i == 1)
            assert np.array_equal(dst[i].to_host(), dst_buf[i])
    graph.free()
    for x in (*src, *dst, *slots, k, v):
        x.free()
