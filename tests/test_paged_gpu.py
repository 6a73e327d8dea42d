"""The paged KV cache on the GPU, through the C-ABI: page maps equal to a walk over
the sequences; attention, the producer and the gather against 64-bit forms, at the
lengths, windows, tables and values where they can go wrong; the three of them as a
server runs them, eagerly and as a replayed graph. Rows of the pools that hold no
token are NaN throughout."""
import numpy as np
import pytest

import g4a
import paged_ref as ref

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[gpu] {msg}", flush=True)


class Paged:
    """Pools of seeded tokens for sequences of the given lengths, on shuffled pages, NaN elsewhere."""

    def __init__(self, ctx, lens, *, dh, hkv=1, kv_type="f32", page=16, ring=False, per_seq=None, stride=None, seed=0,
                 unit=0.25):
        rng = np.random.default_rng(seed)
        self.ctx, self.page, self.ring, self.type = ctx, page, ring, kv_type
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
        pools = []
        for _ in range(2):
            pool = np.full((self.n_pages, page, hkv, dh), np.nan, np.float32)
            for b, n in enumerate(lens):
                t = np.arange(max(0, n - per_seq * page) if ring else 0, n if ring else min(n, per_seq * page))
                pool[self.table[b, (t // page) % per_seq], t % page] = rng.standard_normal((len(t), hkv, dh))
            pools.append(pool)
        pools[0] /= np.sqrt((pools[0] ** 2).mean(-1, keepdims=True))
        self.k, self.v = (ref.unpack(ref.pack(x, kv_type), kv_type) for x in pools)
        self.stride = stride or 0
        self.dev = [ctx.upload(self._spread(ref.pack(x, kv_type))) for x in (self.k, self.v)]
        self.dtable, self.dlen = ctx.upload(self.table), ctx.upload(self.lens)
        self.cache = g4a.PagedCache(k_pages=self.dev[0].ptr, v_pages=self.dev[1].ptr, block_table=self.dtable.ptr,
                                    kv_len=self.dlen.ptr, page_stride=self.stride, n_seqs=len(lens),
                                    pages_per_seq=per_seq, n_pages=self.n_pages, page_size=page, Hkv=hkv, Dh=dh,
                                    kv_type=g4a.KV_TYPES[kv_type], ring=int(ring))
        self.rng, self.unit = rng, unit

    def _spread(self, x):
        """Pages page_stride values apart, with NaN words between."""
        if not self.stride:
            return x
        flat = np.full((len(x), self.stride), 0x7FC0 if x.dtype == np.uint16 else np.nan, x.dtype)
        flat[:, :x[0].size] = x.reshape(len(x), -1)
        return flat

    def pools(self):
        """The pools as the GPU has them now, as f32 values [pages, page, hkv, dh]."""
        out = []
        for d, like in zip(self.dev, (self.k, self.v)):
            x = d.to_host()
            x = x[:, :like[0].size].reshape(like.shape) if self.stride else x
            out.append(ref.unpack(x, self.type))
        return out

    def queries(self, hq):
        q = self.rng.standard_normal((len(self.lens), hq, self.k.shape[3])).astype(np.float32)
        return q * np.float32(self.unit) / np.sqrt((q ** 2).mean(-1, keepdims=True))

    def attend(self, q, window=0, scale=1.0, cap=0.0):
        dq, out = self.ctx.upload(q), self.ctx.upload(np.full((q.shape[0], q[0].size), 7.0, np.float32))
        try:
            self.ctx.attention_paged(self.cache, g4a.PagedAttnArgs(q=dq.ptr, out=out.ptr, Hq=q.shape[1], scale=scale,
                                                                   sliding_window=window, attn_softcap=cap))
            return out.to_host()
        finally:
            dq.free()
            out.free()

    def want(self, q, window=0, scale=1.0, cap=0.0):
        return ref.attention(q, self.k, self.v, self.table, self.lens, page=self.page, ring=self.ring,
                             n_pages=self.n_pages, window=window, scale=scale, cap=cap)

    def free(self):
        for d in (*self.dev, self.dtable, self.dlen):
            d.free()


def _close(got, want, bound, what):
    off = np.abs(got.astype(np.float64) - want)
    share = np.divide(off, bound, out=np.zeros_like(off), where=bound > 0).max()
    say(f"{what}: max-abs {off.max():.2e}, at most {share:.2f} of the bound")
    assert np.all(off <= bound), (what, float(share))


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


EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65, 127, 130, 255, 257, 500]


@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
@pytest.mark.parametrize("dh", [64, 128, 256, 512])
def test_attention_at_the_edges_of_pages_and_tiles(ctx, dh, kv_type):
    _check(ctx, EDGES, 8, f"edges dh {dh} {kv_type}", dh=dh, kv_type=kv_type, seed=dh)
    _check(ctx, EDGES[::-1], 8, f"edges, page 64, dh {dh} {kv_type}", dh=dh, kv_type=kv_type, page=64, seed=dh + 1)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (4, 4), (8, 2), (5, 1), (16, 1), (16, 4), (24, 1), (40, 2), (12, 3)])
@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
def test_attention_of_head_groups(ctx, hq, hkv, kv_type):
    for dh in (64, 256):
        _check(ctx, [70, 0, 5, 333], hq, f"{hq} over {hkv} dh {dh} {kv_type}", dh=dh, hkv=hkv, kv_type=kv_type,
               seed=hq * 10 + hkv)
    _check(ctx, [41, 200], hq, f"{hq} over {hkv} dh 512 {kv_type}", dh=512, hkv=hkv, kv_type=kv_type, seed=hq + hkv)


@pytest.mark.parametrize("window", [1, 7, 16, 100, 512])
@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
def test_attention_windows_and_rings(ctx, window, kv_type):
    lens = [0, 1, 5, window, window + 1, window + 15, 2 * window + 3, 1000, 5003]
    _check(ctx, lens, 8, f"window {window}", window=window, dh=256, kv_type=kv_type, seed=window)
    # a ring of just the window's pages, whose unwritten slots are NaN, and of one page more
    for more in (0, 1):
        _check(ctx, lens, 8, f"window {window} in a ring", window=window, dh=256, kv_type=kv_type, ring=True,
               per_seq=-(-window // 16) + more, seed=window + 1)
    # a ring without a window shows what it holds
    _check(ctx, lens, 8, "a ring alone", dh=512, kv_type=kv_type, ring=True, per_seq=3, page=32, seed=window + 2)


@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
@pytest.mark.parametrize("page,per_seq", [(16, 4), (32, 2), (64, 1), (16, 3), (16, 5)])
def test_attention_over_rings_of_about_a_part(ctx, page, per_seq, kv_type):
    """A ring of four tiles, the smallest part, shows 64 tokens that touch five where they start inside one."""
    for lens in ([65], [0, 1, 48, 49, 63, 64, 65, 70, 79, 80, 100, 1000]):
        for window in (0, 63, 64, 100):
            _check(ctx, lens, 8, f"ring {page} x {per_seq}", window=window, dh=256, kv_type=kv_type, page=page, ring=True,
                   per_seq=per_seq, seed=per_seq + window)


@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
def test_attention_long_and_ragged(ctx, kv_type):
    _check(ctx, [20011], 8, "one long", dh=512, kv_type=kv_type, page=64, seed=1)
    _check(ctx, [9001, 3, 0, 4097, 1, 700, 12000], 8, "ragged", dh=256, kv_type=kv_type, seed=2)
    _check(ctx, [1 + 37 * i % 150 for i in range(300)], 4, "300 short", dh=64, hkv=2, kv_type=kv_type, seed=3)
    _check(ctx, [4000] * 9 + [1] * 40 + [900] * 5, 16, "mixed groups", dh=128, hkv=4, kv_type=kv_type, seed=4, cap=20.0)


@pytest.mark.parametrize("n,hq,hkv,dh,kv_type,longest", [
    (2100, 2, 1, 64, "f32", 40), (1025, 8, 1, 64, "bf16", 20), (300, 8, 8, 64, "f32", 70), (150, 40, 5, 128, "bf16", 90),
    (260, 8, 1, 512, "bf16", 300), (140, 8, 1, 512, "f32", 400), (129, 4, 1, 512, "bf16", 400), (65, 9, 1, 256, "f32", 900)])
def test_attention_of_many_sequences(ctx, n, hq, hkv, dh, kv_type, longest):
    """More sequences and head groups than one launch takes, and about as many as run at once; lengths
    from none to a few parts, one sequence far longer than the others."""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, longest + 1, n)
    lens[[0, n // 2, n - 1]] = [5 * longest, 0, longest]
    for window in (0, 37):
        _check(ctx, lens, hq, "many", window=window, hkv=hkv, dh=dh, kv_type=kv_type, seed=n)


def test_attention_scale_softcap_and_page_stride(ctx):
    _check(ctx, [100, 513, 31], 8, "scale", dh=256, scale=0.0625, unit=1.0, seed=1)
    _check(ctx, [100, 513, 31], 8, "softcap", dh=512, cap=5.0, unit=1.0, seed=2)
    for kv_type in ("f32", "bf16"):
        _check(ctx, [100, 513, 31], 8, "stride", dh=128, hkv=2, stride=16 * 256 + 64, kv_type=kv_type, seed=3)


def test_attention_leaves_out_tokens_without_a_page(ctx):
    """Entries that name no page, at and beyond n_pages, in the middle and for a whole sequence."""
    for kv_type in ("f32", "bf16"):
        c = Paged(ctx, [200, 64, 90, 48], dh=256, kv_type=kv_type, seed=4)
        c.table[0, 3], c.table[0, 12], c.table[1, :], c.table[2, 0] = ref.NO_ROW, c.n_pages, 0x80000000, c.n_pages + 7
        ctx.h2d(c.dtable.ptr, c.table)
        q = c.queries(8)
        got = c.attend(q)
        want, bound = c.want(q)
        _close(got, want, bound, f"bad pages {kv_type}")
        assert not got[1].any()
        # a length past the table's end counts what the table holds
        c.lens[3] = 4000
        ctx.h2d(c.dlen.ptr, c.lens)
        _close(c.attend(q), want, bound, f"a long length {kv_type}")
        c.free()


def test_attention_shows_infinities_and_nan_of_visible_tokens_only(ctx):
    """V = inf at a visible token reaches its head's output; the rows behind the length and
    before the window hold NaN and infinities and reach nothing."""
    c = Paged(ctx, [50, 120], dh=256, hkv=2, seed=6)
    c.v[c.table[0, 1], 3, 0, 17] = np.inf  # token 19 of sequence 0, kv head 0, dim 17
    c.k[c.table[1, 0]] = np.inf            # tokens 0 .. 15 of sequence 1, outside the window
    c.v[c.table[1, 0]] = -np.inf
    for d, x in zip(c.dev, (c.k, c.v)):
        ctx.h2d(d.ptr, x)
    q = c.queries(8)
    got = c.attend(q, window=100).reshape(2, 8, 256)
    assert np.isposinf(got[0, :4, 17]).all()
    want, bound = (x.reshape(2, 8, 256) for x in c.want(q, window=100))
    rest = np.isfinite(want)
    assert rest.sum() == want.size - 4
    assert np.all(np.abs(got[rest] - want[rest]) <= bound[rest])
    c.free()


def _same(got, want, bound, what):
    """Infinities and NaN where the definition has them, the rest within the bound."""
    got, rest = got.astype(np.float64), np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~rest & ~np.isnan(want)], want[~rest & ~np.isnan(want)]), what
    _close(got[rest], want[rest], bound[rest], what)


@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
@pytest.mark.parametrize("dh,hq,hkv", [(64, 4, 1), (64, 8, 1), (64, 16, 1), (128, 3, 1), (128, 16, 2), (128, 12, 1),
                                       (256, 4, 1), (256, 8, 1), (256, 20, 1), (512, 2, 1), (512, 16, 2), (512, 9, 1)])
def test_attention_of_infinite_values(ctx, dh, hq, hkv, kv_type):
    """Visible infinities and NaN act as in f32 arithmetic whatever the pages hold, in sequences of one part and of
    many: V's reach their dim of their kv head's output; a key of minus infinity has weight 0 where a query's value
    there is positive, and makes the row NaN where it is negative; a query's value near f32's largest times a key's
    near its smallest is a score like any other."""
    say(f"infinite values: dh {dh} heads {hq}/{hkv} {kv_type}")
    opts = dict(dh=dh, hkv=hkv, kv_type=kv_type, unit=0.05 * np.sqrt(256 / dh), seed=dh + hq)
    c = Paged(ctx, [50, 700, 17, 0], **opts)
    q = c.queries(hq)

    def attend(q=q):
        for d, x in zip(c.dev, (c.k, c.v)):
            ctx.h2d(d.ptr, ref.pack(x, kv_type))
        return c.attend(q)

    plain = [c.want(q), c.k.copy(), c.v.copy()]
    for b, e in ((0, 1), (1, 20), (2, 0)):  # V, infinite and NaN
        c.v[c.table[b, e], 3, hkv - 1, 17] = np.inf
        c.v[c.table[b, e], 5, 0, dh - 1] = -np.inf
        c.v[c.table[b, e], 7, 0, 2] = np.nan
    c.v[c.table[1, 30], 1, hkv - 1, 17] = -np.inf
    with np.errstate(all="ignore"):
        want, bound = c.want(q)
    assert np.isnan(want).any() and np.isposinf(want).any() and np.isneginf(want).any()
    _same(attend(), want, bound, "V")

    c.k, c.v = plain[1].copy(), plain[2].copy()
    pages = [c.table[0, 1], c.table[1, 20]]  # K of whole pages: as if they were not there, for a query positive there
    c.k[pages, :, :, 33] = -np.inf
    got = attend()
    held = c.table.copy()
    c.table[0, 1] = c.table[1, 20] = ref.NO_ROW
    want, bound = (x.reshape(4, hq, dh).copy() for x in c.want(q))
    c.table = held
    want[:2][q[:2, :, 33] < 0] = np.nan
    _same(got.reshape(want.shape), want, bound, "K")

    # products as of 2^-120 of the query's value and 2^120 of the key's, which the bound is taken of
    c.k, c.v = plain[1].copy(), plain[2].copy()
    far, far_q, live = c.k.copy(), q.copy(), np.isfinite(c.k[..., 5])
    c.k[..., 5][live], far[..., 5][live] = 2.0 ** -6, 2.0 ** -126
    far_q[:, :, 5] = np.where(q[:, :, 5] > 0, 3.4e38, -3.4e38)
    q2 = far_q.copy()
    q2[:, :, 5] *= 2.0 ** -120
    want, bound = c.want(q2)
    c.k = far
    _same(attend(far_q), want, bound, "the query")
    c.free()


@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
@pytest.mark.parametrize("dh,hq,hkv", [(64, 16, 1), (128, 3, 1), (256, 8, 1), (512, 9, 1)])
def test_attention_of_queries_that_are_nan(ctx, dh, hq, hkv, kv_type):
    """A NaN in a query makes its head's row NaN and no other's, beside an infinity in V or not."""
    say(f"NaN queries: dh {dh} heads {hq}/{hkv} {kv_type}")
    c = Paged(ctx, [50, 700, 17, 90], dh=dh, hkv=hkv, kv_type=kv_type, seed=dh)
    q = c.queries(hq)
    q[1, 0, dh - 1] = q[2, :, 40] = q[3, hq - 1, 3] = np.nan
    for poison in (False, True):
        if poison:
            c.v[c.table[1, 20], 3, 0, 17] = c.v[c.table[3, 1], 2, 0, 5] = -np.inf
            ctx.h2d(c.dev[1].ptr, ref.pack(c.v, kv_type))
        with np.errstate(all="ignore"):
            want, bound = c.want(q)
        assert np.isnan(want.reshape(4, hq, dh)).all(-1).sum() == 1 + hq + 1 and np.isinf(want).any() == poison
        _same(c.attend(q), want, bound, f"NaN queries, infinities {poison}")
    c.free()


def test_attention_is_repeatable_and_shares_pages(ctx):
    """Two sequences over the same pages, twice: the same bits."""
    c = Paged(ctx, [3000, 3000, 17], dh=512, page=32, seed=7)
    c.table[1] = c.table[0]
    ctx.h2d(c.dtable.ptr, c.table)
    q = c.queries(8)
    q[1] = q[0]
    one, two = c.attend(q), c.attend(q)
    assert np.array_equal(one, two)
    want, bound = c.want(q)
    _close(one, want, bound, "shared pages")
    c.free()


# ---- page maps -------------------------------------------------------------------

def _run_map(ctx, lens, new, table, free, first, count, *, page, ring, rows, rows_per_seq=0, shared=None, apart=False,
             n_pages=None, new_null=False, lean=False):
    n, per_seq = table.shape
    d = {k: ctx.upload(np.ascontiguousarray(v, np.uint32)) for k, v in dict(
        lens=lens, new=new, table=table, free=free, state=[first, count], slots=np.full(max(rows, 1) + 5, 9),
        pos=np.full(max(rows, 1) + 5, 9), start=np.full(n + 1, 9), added=np.full(n, 9), lens2=np.full(n, 9),
        state2=[9, 9], shared=np.zeros(n) if shared is None else shared).items()}
    cache = g4a.PagedCache(block_table=d["table"].ptr, kv_len=d["lens"].ptr, n_seqs=n, pages_per_seq=per_seq,
                           n_pages=n_pages or len(free), page_size=page, ring=int(ring))
    args = g4a.PageMapArgs(new_len=None if new_null else d["new"].ptr, shared_pages=None if shared is None else d["shared"].ptr,
                           free_pages=d["free"].ptr, free_state=d["state"].ptr, slots=d["slots"].ptr,
                           positions=d["pos"].ptr, row_start=None if lean else d["start"].ptr,
                           added=None if lean else d["added"].ptr, kv_len_out=d["lens2"].ptr if apart else None,
                           free_state_out=d["state2"].ptr if apart else None, free_cap=len(free), rows=rows,
                           rows_per_seq=rows_per_seq)
    ctx.page_map(cache, args)
    got = {k: v.to_host() for k, v in d.items()}
    for v in d.values():
        v.free()
    return got


def _check_map(ctx, what, lens, new, table, free, first, count, **kw):
    say(f"map {what}: {len(lens)} sequences, {kw}")
    opts = {k: kw.pop(k) for k in ("apart", "n_pages", "new_null", "lean") if k in kw}
    got = _run_map(ctx, lens, new, table, free, first, count, **kw, **opts)
    slots, pos, start, added, out, table2, free2, first2, count2 = ref.page_map(
        lens, new, table, free, first, count, **kw)
    rows = kw["rows"]
    apart = opts.get("apart")
    assert np.array_equal(got["slots"][:rows], slots), what
    assert np.array_equal(got["pos"][:rows], pos), what
    assert (got["slots"][max(rows, 1):] == 9).all() and (got["pos"][max(rows, 1):] == 9).all(), "rows behind the last"
    if not opts.get("lean"):
        assert np.array_equal(got["start"], start) and np.array_equal(got["added"], added), what
    assert np.array_equal(got["table"], table2) and np.array_equal(got["free"], free2), what
    assert np.array_equal(got["lens2" if apart else "lens"], out), what
    assert list(got["state2" if apart else "state"]) == [first2, count2], what
    if apart:
        assert np.array_equal(got["lens"], lens) and list(got["state"]) == [first, count]
    return out, table2, free2, first2, count2, added


@pytest.mark.parametrize("n,page,ring,rows_per_seq", [(1, 16, False, 0), (5, 16, True, 0), (64, 16, False, 1),
                                                      (256, 32, False, 0), (257, 16, False, 3), (700, 16, True, 0),
                                                      (1024, 64, False, 1), (2500, 16, False, 0), (2500, 16, True, 2)])
@pytest.mark.parametrize("apart", [False, True])
def test_maps_of_random_steps(ctx, n, page, ring, rows_per_seq, apart):
    """Steps in a row, each on what the one before left: starts, ends, refusals for want of pages, rows
    and table entries, rings that wrap."""
    rng = np.random.default_rng(n + page + 7 * ring)
    per_seq = 3 if ring else 6
    cap = max(4, int(n * per_seq * 0.6))
    lens, table = np.zeros(n, np.uint32), np.full((n, per_seq), ref.NO_ROW, np.uint32)
    free, first, count = rng.permutation(cap).astype(np.uint32), int(rng.integers(cap)), cap
    refused = 0
    for step in range(6):
        most = rows_per_seq + 1 if rows_per_seq else 3 * page
        new = rng.integers(0, most + 1, n).astype(np.uint32)
        if step % 2:
            new[rng.random(n) < 0.3] = ref.NO_ROW
        elif step:
            new[:] = 1
        rows = n * rows_per_seq if rows_per_seq else int(np.where(new == ref.NO_ROW, 0, new).sum() * (0.8 if step == 4 else 1)) + 3
        lens, table, free, first, count, added = _check_map(
            ctx, f"step {step}", lens, new, table, free, first, count, page=page, ring=ring, rows=rows,
            rows_per_seq=rows_per_seq, apart=apart, lean=step == 3)
        refused += int(((new != ref.NO_ROW) & (new != added)).sum())
    assert refused or n == 1 or ring


def test_maps_of_long_prompts(ctx):
    """Prompts of thousands of tokens, over many workgroups, in place and apart; a ring keeps each prompt's end."""
    rng = np.random.default_rng(3)
    for ring, per_seq in ((False, 800), (True, 33)):
        lens = np.array([0, 700, 3, 0, 16, 511], np.uint32)
        new = np.array([12345, 1, 5000, ref.NO_ROW, 9999, ref.NO_ROW], np.uint32)
        free = rng.permutation(5000).astype(np.uint32)
        table = np.full((6, per_seq), ref.NO_ROW, np.uint32)
        for b in range(6):
            u = min(-(-int(lens[b]) // 16), per_seq)
            table[b, :u] = 4000 + 100 * b + np.arange(u)
        for apart in (False, True):
            _check_map(ctx, "prompts", lens, new, table, free, 4900, 4000, page=16, ring=ring, rows=28000, apart=apart)


def test_maps_keep_shared_pages_and_take_single_tokens(ctx):
    rng = np.random.default_rng(4)
    lens, new = np.array([50, 64, 10, 0], np.uint32), np.array([ref.NO_ROW, ref.NO_ROW, 7, ref.NO_ROW], np.uint32)
    table = np.full((4, 5), ref.NO_ROW, np.uint32)
    table[0, :4], table[1, :4], table[2, :1] = [20, 21, 22, 23], [20, 21, 24, 25], [26]
    free = rng.permutation(30).astype(np.uint32)
    _check_map(ctx, "shared", lens, new, table, free, 28, 9, page=16, ring=False, rows=10,
               shared=np.array([0, 2, 9, 4], np.uint32))
    _check_map(ctx, "one each", lens, np.ones(4, np.uint32), table, free, 0, 3, page=16, ring=False, rows=4,
               rows_per_seq=1, new_null=True)
    _check_map(ctx, "no rows", lens, np.zeros(4, np.uint32), table, free, 0, 3, page=16, ring=False, rows=0)


@pytest.mark.parametrize("apart", [False, True])
def test_maps_refuse_rows_over_thousands_of_sequences(ctx, apart):
    """Once the rows asked for have passed those there are, no later sequence gets one, however far behind."""
    n = 2600
    lens, new = np.zeros(n, np.uint32), np.zeros(n, np.uint32)
    table = np.full((n, 4), ref.NO_ROW, np.uint32)
    new[[3, 700, 900, 1030, 1500, 2590]] = [10, 45, 3, 2, 1, 7]
    free = np.arange(n, dtype=np.uint32)
    *_, added = _check_map(ctx, "rows", lens, new, table, free, 5, n, page=16, ring=False, rows=50, apart=apart)
    assert added.sum() == 10


def test_maps_in_place_replay_over_many_workgroups(ctx):
    """One captured step of thousands of rows, lengths and free ring in place, replayed with other demands, an
    eager step between the replays: each leaves what a walk over the sequences leaves."""
    rng = np.random.default_rng(12)
    n, per_seq, page, rows, cap = 300, 12, 16, 6000, 2500
    lens, table = np.zeros(n, np.uint32), np.full((n, per_seq), ref.NO_ROW, np.uint32)
    free, first, count = rng.permutation(cap).astype(np.uint32), 7, cap
    d = {k: ctx.upload(np.ascontiguousarray(v, np.uint32)) for k, v in dict(
        lens=lens, new=np.zeros(n), table=table, free=free, state=[first, count], slots=np.zeros(rows),
        pos=np.zeros(rows), start=np.zeros(n + 1), added=np.zeros(n)).items()}
    cache = g4a.PagedCache(block_table=d["table"].ptr, kv_len=d["lens"].ptr, n_seqs=n, pages_per_seq=per_seq, n_pages=cap,
                           page_size=page)
    args = g4a.PageMapArgs(new_len=d["new"].ptr, free_pages=d["free"].ptr, free_state=d["state"].ptr, slots=d["slots"].ptr,
                           positions=d["pos"].ptr, row_start=d["start"].ptr, added=d["added"].ptr, free_cap=cap, rows=rows)
    ctx.capture_begin()
    ctx.page_map(cache, args)
    graph = ctx.capture_end()
    for step in range(8):
        new = rng.integers(0, 40, n).astype(np.uint32)
        new[rng.random(n) < 0.2] = ref.NO_ROW if step % 3 else 1
        ctx.h2d(d["new"].ptr, new)
        if step % 4 == 2:
            ctx.page_map(cache, args)
        else:
            graph.launch()
        say(f"step {step}")
        slots, pos, start, added, lens, table, free, first, count = ref.page_map(
            lens, new, table, free, first, count, page=page, ring=False, rows=rows)
        want = dict(slots=slots, pos=pos, start=start, added=added, lens=lens, table=table, free=free,
                    state=np.array([first, count]))
        for k, v in want.items():
            assert np.array_equal(d[k].to_host(), v), (step, k)
    graph.free()
    for v in d.values():
        v.free()


def test_maps_of_bad_device_values_stay_inside(ctx):
    """Lengths past the table, a free ring that claims more than it holds, page numbers that do not exist:
    no slot past the pool, nothing written behind the buffers."""
    lens, new = np.array([0xFFFFFF00, 70, 0], np.uint32), np.array([5, 3, 20], np.uint32)
    table = np.full((3, 4), 0xFFFFFFF0, np.uint32)
    got = _run_map(ctx, lens, new, table, np.array([3, 0xFFFFFFFF, 900], np.uint32), 0xFFFFFFFF, 0xFFFFFFFF, page=16,
                   ring=False, rows=40, n_pages=8)
    assert list(got["added"]) == [0, 0, 20]  # (a table of 4 pages holds 64 tokens)
    live = got["slots"][got["slots"] != ref.NO_ROW]
    assert (live < 8 * 16).all() and (got["slots"][40:] == 9).all()


@pytest.mark.parametrize("apart", [False, True])
def test_a_map_of_no_sequence(ctx, apart):
    """Without a sequence no row has a token: row_start is its end alone, 0, and the ring's state goes on."""
    for rows in (0, 5, 70000):
        say(f"no sequence, {rows} rows, apart {apart}")
        d = {k: ctx.upload(np.asarray(v, np.uint32)) for k, v in dict(
            free=[4, 2, 7], state=[5, 2], slots=np.full(rows + 5, 9), pos=np.full(rows + 5, 9), start=[9, 9],
            state2=[9, 9, 9]).items()}
        args = g4a.PageMapArgs(free_pages=d["free"].ptr, free_state=d["state"].ptr, slots=d["slots"].ptr,
                               positions=d["pos"].ptr, row_start=d["start"].ptr,
                               free_state_out=d["state2"].ptr if apart else None, free_cap=3, rows=rows)
        ctx.page_map(g4a.PagedCache(n_pages=8, page_size=16), args)
        got = {k: list(v.to_host()) for k, v in d.items()}
        assert got["start"] == [0, 9] and got["free"] == [4, 2, 7]
        assert got["state2" if apart else "state"][:2] == [2, 2]  # (place 5 of a ring of 3 is place 2)
        assert got["state2"][2] == 9 and (not apart or got["state"] == [5, 2])
        for k in ("slots", "pos"):
            assert got[k] == [ref.NO_ROW] * rows + [9] * 5
        for v in d.values():
            v.free()


# ---- the producer ------------------------------------------------------------------

def _produce(ctx, T, hq, hkv, dh, kv_type, rot, theta, seed, *, norms=True, kv=True, page=16, stride=0, pos=None,
             skip=()):
    rng = np.random.default_rng(seed)
    n_pages = -(-T // page) + 4
    pools = [rng.standard_normal((n_pages, page, hkv, dh)).astype(np.float32) for _ in range(2)]
    pools = [ref.unpack(ref.pack(x, kv_type), kv_type) for x in pools]
    q, k, v = (rng.standard_normal((T, h, dh)).astype(np.float32) * s for h, s in ((hq, 1), (hkv, 2), (hkv, 3)))
    wq, wk = (1 + 0.1 * rng.standard_normal(dh).astype(np.float32) for _ in range(2))
    slots = rng.permutation(n_pages * page)[:T].astype(np.uint32)
    pos = rng.integers(0, 40000, T).astype(np.uint32) if pos is None else np.asarray(pos, np.uint32)
    for i, what in skip:  # rows without a slot, past the pool, or without a token
        if what == "pos":
            pos[i] = ref.NO_ROW
        else:
            slots[i] = ref.NO_ROW if what == "slot" else n_pages * page + 3
    c = Paged.__new__(Paged)
    c.stride, c.type, c.k, c.v = stride, kv_type, *pools
    d = {n: ctx.upload(x) for n, x in dict(q=q, k=k, v=v, wq=wq, wk=wk, slots=slots, pos=pos,
                                           out=np.full(q.shape, 5.0, np.float32)).items()}
    c.dev = [ctx.upload(c._spread(ref.pack(x, kv_type))) for x in pools]
    cache = g4a.PagedCache(k_pages=c.dev[0].ptr, v_pages=c.dev[1].ptr, page_stride=stride, n_pages=n_pages,
                           page_size=page, Hkv=hkv, Dh=dh, kv_type=g4a.KV_TYPES[kv_type])
    args = g4a.PagedProducerArgs(q=d["q"].ptr, k=d["k"].ptr if kv else None, v=d["v"].ptr if kv else None,
                                 q_norm=d["wq"].ptr if norms else None, k_norm=d["wk"].ptr if norms else None,
                                 q_out=d["out"].ptr, positions=d["pos"].ptr, slots=d["slots"].ptr if kv else None, T=T,
                                 Hq=hq, rotary_dim=rot, theta=theta, eps=1e-6)
    ctx.attn_producer_paged(cache, args)
    got_q, (got_k, got_v) = d["out"].to_host(), c.pools()
    live = pos != ref.NO_ROW
    writes = live & (slots < n_pages * page) & kv

    def made(x, w, turn=True):
        x = ref.rms(x, w, 1e-6) if w is not None or not turn else x.astype(np.float64)
        return ref.rope(x, np.where(live, pos, 0), rot, theta) if turn else x

    want_q = np.where(live[:, None, None], made(q, wq if norms else None), 5.0)
    # a norm is a few roundings (sum tree, divide, root, two products), a rotation three more; the sine of
    # an f32 angle is right to 2 half steps of 1: all relative to the pair's size, here the row's largest
    _close(got_q, want_q, 24 * ref.HALF * np.abs(want_q).max(-1, keepdims=True) + 0 * want_q, "q")
    half_step = 2.0 ** -8 if kv_type == "bf16" else 0.0
    for name, got, pool, x, w, turn in (("k", got_k, pools[0], k, wk if norms else None, True),
                                        ("v", got_v, pools[1], v, None, False)):
        rows = pool.reshape(-1, hkv, dh).astype(np.float64)
        new = made(x, w, turn)[writes]
        rows[slots[writes]] = new
        bound = np.zeros_like(rows)
        f32 = 24 * ref.HALF * np.abs(new).max(-1, keepdims=True)
        bound[slots[writes]] = f32 + half_step * (np.abs(new) + f32)
        _close(got.reshape(rows.shape), rows, bound + 1e-300, name)  # (rows of other slots: unchanged)
    for x in (*d.values(), *c.dev):
        x.free()


@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
@pytest.mark.parametrize("dh,rot,theta", [(64, 64, 1e4), (128, 128, 1e4), (256, 256, 1e4), (512, 128, 1e6), (512, 512, 1e4),
                                          (256, 6, 1e4), (128, 0, 1e4), (512, 250, 1e4)])
def test_producer_rows(ctx, dh, rot, theta, kv_type):
    for T, hq, hkv in ((1, 8, 1), (3, 3, 2), (65, 8, 1), (37, 16, 4)):
        say(f"producer T {T} heads {hq}/{hkv} dh {dh} rot {rot} {kv_type}")
        _produce(ctx, T, hq, hkv, dh, kv_type, rot, theta, T + dh)


@pytest.mark.parametrize("T,hq,hkv,dh,kv_type", [(1500, 3, 2, 64, "f32"), (1030, 8, 1, 256, "bf16"), (1100, 5, 1, 128, "f32"),
                                                 (1024, 2, 1, 512, "bf16"), (8200, 4, 1, 64, "bf16"), (8193, 1, 1, 256, "f32")])
def test_producer_of_long_calls(ctx, T, hq, hkv, dh, kv_type):
    """Calls whose waves take several rows of a token: numbers of rows that do not divide, tokens without slot or position."""
    _produce(ctx, T, hq, hkv, dh, kv_type, dh // 2, 1e4, T, skip=[(1, "slot"), (T // 2, "pos"), (T - 2, "past")])


def test_producer_variants(ctx):
    for kv_type in ("f32", "bf16"):
        _produce(ctx, 9, 8, 1, 256, kv_type, 256, 1e4, 1, norms=False)
        _produce(ctx, 9, 8, 1, 512, kv_type, 128, 1e6, 2, kv=False)
        _produce(ctx, 20, 8, 2, 128, kv_type, 128, 1e4, 3, stride=16 * 256 + 40)
        _produce(ctx, 12, 8, 1, 256, kv_type, 256, 1e4, 4, skip=[(0, "pos"), (3, "slot"), (7, "past"), (11, "pos")])
        _produce(ctx, 4, 8, 1, 512, kv_type, 128, 1e6, 5, pos=[0, 131071, (1 << 20) + 1, (1 << 24) + 2])


# ---- the gather --------------------------------------------------------------------

@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
@pytest.mark.parametrize("dh,hkv,page", [(64, 1, 16), (128, 3, 32), (256, 1, 256), (512, 2, 16)])
def test_gather_gives_tokens_in_order(ctx, dh, hkv, page, kv_type):
    for ring in (False, True):
        c = Paged(ctx, [5, 700, 90], dh=dh, hkv=hkv, kv_type=kv_type, page=page, ring=ring, seed=dh,
                  per_seq=max(1, 192 // page) if ring else None, stride=0 if ring else page * hkv * dh + 8)
        if not ring:
            c.table[1, 1] = c.n_pages  # a hole
            ctx.h2d(c.dtable.ptr, c.table)
        for pos0, n in ((0, 700), (0, 1), (699, 1), (17, 301), (690, 40), (800, 9)):
            say(f"gather {pos0} + {n} page {page} ring {ring}")
            out = [ctx.upload(np.full((n + 1, hkv, dh), 3.0, np.float32)) for _ in range(2)]
            ctx.kv_gather_paged(c.cache, 1, pos0, n, out[0].ptr, out[1].ptr)
            for d, pool in zip(out, (c.k, c.v)):
                want = np.zeros((n + 1, hkv, dh), np.float32)
                want[n] = 3.0
                t, rows = ref.tokens(pool, c.table, 1, 700, page=page, ring=ring, n_pages=c.n_pages)
                keep = (t >= pos0) & (t < pos0 + n)
                want[t[keep] - pos0] = rows[keep]
                assert np.array_equal(d.to_host(), want)
                d.free()
        c.free()


# ---- together, as a server runs them ----------------------------------------------

class Server:
    """A layer's decode steps of a batch of fixed size over a paged cache: new tokens in, pages mapped,
    rows produced, attention out; the mirror of the cache on the host is checked after every step."""

    def __init__(self, ctx, n, dh, kv_type, window, seed):
        self.ctx, self.n, self.dh, self.type, self.window = ctx, n, dh, kv_type, window
        self.page, self.ring = 16, bool(window)
        self.per_seq = -(-(window + 40) // 16) if window else 20
        self.n_pages = n * self.per_seq
        self.rng = rng = np.random.default_rng(seed)
        z = np.zeros
        host = dict(k_pool=ref.pack(np.full((self.n_pages, 16, 1, dh), np.nan, np.float32), kv_type),
                    v_pool=ref.pack(np.full((self.n_pages, 16, 1, dh), np.nan, np.float32), kv_type),
                    table=np.full((n, self.per_seq), ref.NO_ROW, np.uint32), lens=z(n, np.uint32), new=z(n, np.uint32),
                    free=rng.permutation(self.n_pages).astype(np.uint32), state=np.array([0, self.n_pages], np.uint32),
                    slots=z(512, np.uint32), pos=z(512, np.uint32), start=z(n + 1, np.uint32), added=z(n, np.uint32),
                    q=z((512, 8, dh), np.float32), k=z((512, 1, dh), np.float32), v=z((512, 1, dh), np.float32),
                    q_out=z((512, 8, dh), np.float32), out=z((n, 8 * dh), np.float32))
        self.d = {name: ctx.upload(x) for name, x in host.items()}
        p = {name: x.ptr for name, x in self.d.items()}
        self.cache = g4a.PagedCache(k_pages=p["k_pool"], v_pages=p["v_pool"], block_table=p["table"], kv_len=p["lens"],
                                    n_seqs=n, pages_per_seq=self.per_seq, n_pages=self.n_pages, page_size=16, Hkv=1,
                                    Dh=dh, kv_type=g4a.KV_TYPES[kv_type], ring=int(self.ring))
        self.map = g4a.PageMapArgs(new_len=p["new"], free_pages=p["free"], free_state=p["state"], slots=p["slots"],
                                   positions=p["pos"], row_start=p["start"], added=p["added"], free_cap=self.n_pages)
        self.rot, self.theta = (128, 1e6) if dh == 512 else (dh, 1e4)
        self.prod = g4a.PagedProducerArgs(q=p["q"], k=p["k"], v=p["v"], q_out=p["q_out"], positions=p["pos"],
                                          slots=p["slots"], Hq=8, rotary_dim=self.rot, theta=self.theta, eps=1e-6)
        self.attn = g4a.PagedAttnArgs(q=p["q_out"], out=p["out"], Hq=8, scale=0.1, sliding_window=window)
        self.tokens = [[np.zeros((0, 1, dh), np.float32)] * 2 for _ in range(n)]

    def rows(self, rows, rows_per_seq):
        self.map.rows, self.map.rows_per_seq, self.prod.T = rows, rows_per_seq, rows

    def feed(self, new, rows):
        """New tokens' projections on the device and on the host."""
        self.new = np.asarray(new, np.uint32)
        self.x = [self.rng.standard_normal((rows, h, self.dh)).astype(np.float32) for h in (8, 1, 1)]
        self.ctx.h2d(self.d["new"].ptr, self.new)
        for name, x in zip("qkv", self.x):
            self.ctx.h2d(self.d[name].ptr, x)

    def step(self, attend=True):
        self.ctx.page_map(self.cache, self.map)
        self.ctx.attn_producer_paged(self.cache, self.prod)
        if attend:
            self.ctx.attention_paged(self.cache, self.attn)

    def check(self, rows_per_seq, attend=True):
        q, k, v = self.x
        added, lens = self.d["added"].to_host(), self.d["lens"].to_host()
        start = 0
        qs = np.zeros((self.n, 8, self.dh))
        for b in range(self.n):
            assert added[b] == (0 if self.new[b] == ref.NO_ROW else self.new[b])
            if self.new[b] == ref.NO_ROW:
                self.tokens[b] = [np.zeros((0, 1, self.dh), np.float32)] * 2
            r0 = b * rows_per_seq if rows_per_seq else start
            r, past = np.arange(r0, r0 + added[b]), len(self.tokens[b][0])
            pos = past + np.arange(len(r))
            made = ref.rope(k[r].astype(np.float64), pos, self.rot, self.theta), ref.rms(v[r], None, 1e-6)
            self.tokens[b] = [np.concatenate([t, ref.unpack(ref.pack(x, self.type), self.type)])
                              for t, x in zip(self.tokens[b], made)]
            assert lens[b] == len(self.tokens[b][0])
            if len(r):
                qs[b] = ref.rope(q[r[-1:]].astype(np.float64), pos[-1:], self.rot, self.theta)[0]
            start += added[b]
        if not attend:
            return
        got = self.d["out"].to_host().reshape(self.n, 8, self.dh)
        for b in range(self.n):
            kk, vv = self.tokens[b]
            if not len(kk):
                assert not got[b].any()
                continue
            if added[b] == 0:  # its query was not made this step
                continue
            lo = max(0, len(kk) - self.window) if self.window else 0
            kk, vv = kk[lo:, 0].astype(np.float64), vv[lo:, 0].astype(np.float64)
            s = 0.1 * (qs[b] @ kk.T)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            # as ref.attention's bound, and what the produced rows are off: an f32 rounding (with bf16 pages, now
            # and then a rounding to the other neighbour: a step of 2^-7) of a score's terms and of V
            step = 2.0 ** -7 if self.type == "bf16" else 24 * ref.HALF
            size = 0.1 * np.linalg.norm(qs[b], axis=-1).max() * np.linalg.norm(kk, axis=1).max() / np.sqrt(self.dh)
            size = max(size, np.abs(s).max())
            flips = 8 * step * size * (0.05 if self.type == "bf16" else 1.0)
            tol = (2 * flips + 2 * ref.HALF * (size * 8 * np.sqrt(self.dh) + 64)) * (p @ np.abs(vv)).max() + (
                step * (np.abs(p).max() * np.abs(vv).max()) if self.type == "bf16" else 0)
            off = np.abs(got[b] - p @ vv).max()
            assert off <= tol, (b, len(kk), off, tol)


@pytest.mark.parametrize("dh,kv_type,window", [(256, "f32", 100), (512, "f32", 0), (512, "bf16", 0), (256, "bf16", 100)])
def test_a_server_steps_eagerly_and_replayed(ctx, dh, kv_type, window):
    """Prompts of one step, then decode steps with sequences that end and start again, eagerly and as replays of
    one captured step, each checked against the definition."""
    say(f"server dh {dh} {kv_type} window {window}")
    n = 6
    s = Server(ctx, n, dh, kv_type, window, dh)
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


def test_two_graphs_replay_beside_a_larger_call(ctx):
    """Two captured calls share the context's workspace, and a later call that needs more of it leaves theirs:
    replays in any order give what the eager calls gave, as lengths change between them."""
    c = g4a.Context(0)
    small, big = (Paged(c, lens, dh=256, kv_type=t, seed=3) for lens, t in (([700, 33, 0], "f32"), ([90, 2000, 17, 5], "bf16")))
    huge = Paged(c, [3000] * 24, dh=256, hkv=2, seed=4)
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


@pytest.mark.parametrize("kv_type", ["f32", "bf16"])
def test_pages_past_four_gib(ctx, kv_type):
    """The same tokens in pages side by side and more than 2^32 bytes apart: produced, gathered and attended alike, bit for bit."""
    size = 4 if kv_type == "f32" else 2
    T, page, dh, far = 90, 32, 256, (1 << 32) // size + 64
    rng = np.random.default_rng(8)
    x = {m: ctx.upload(rng.standard_normal((T, h, dh)).astype(np.float32)) for m, h in (("q", 8), ("k", 1), ("v", 1))}
    table, slots = np.array([[2, 0, 1]], np.uint32), np.zeros(T, np.uint32)
    t = np.arange(T)
    slots[:] = table[0, t // page] * page + t % page
    d = dict(table=ctx.upload(table), len=ctx.upload(np.array([T], np.uint32)), slots=ctx.upload(slots),
             pos=ctx.upload(t.astype(np.uint32)))
    got = []
    for stride in (page * dh, far):
        pools = [ctx.empty(((2 * stride + page * dh) * size // 4,)) for _ in range(2)]
        q, out, k, v = (ctx.empty(s) for s in ((T, 8, dh), (1, 8 * dh), (T, 1, dh), (T, 1, dh)))
        cache = g4a.PagedCache(k_pages=pools[0].ptr, v_pages=pools[1].ptr, block_table=d["table"].ptr, kv_len=d["len"].ptr,
                               page_stride=stride, n_seqs=1, pages_per_seq=3, n_pages=3, page_size=page, Hkv=1, Dh=dh,
                               kv_type=g4a.KV_TYPES[kv_type])
        say(f"stride {stride} {kv_type}")
        ctx.attn_producer_paged(cache, g4a.PagedProducerArgs(q=x["q"].ptr, k=x["k"].ptr, v=x["v"].ptr, q_out=q.ptr,
                                                             positions=d["pos"].ptr, slots=d["slots"].ptr, T=T, Hq=8,
                                                             rotary_dim=dh, theta=1e4, eps=1e-6))
        ctx.kv_gather_paged(cache, 0, 0, T, k.ptr, v.ptr)
        ctx.attention_paged(cache, g4a.PagedAttnArgs(q=q.ptr, out=out.ptr, Hq=8, scale=0.1))
        got.append([y.to_host() for y in (k, v, out)])
        for y in (*pools, q, out, k, v):
            y.free()
    assert all(np.isfinite(y).all() and y.any() for y in got[0])
    assert all(np.array_equal(a, b) for a, b in zip(*got))


def test_a_prompt_continues_a_cached_prefix(ctx):
    """A second part of a prompt: produced into pages, gathered in order, attended by g4a_attention; the same
    rows as one attention call over a contiguous cache."""
    rng = np.random.default_rng(9)
    dh, T0, T1, page = 512, 70, 45, 16
    n = T0 + T1
    x = [rng.standard_normal((n, h, dh)).astype(np.float32) for h in (8, 1, 1)]
    w = [1 + 0.1 * rng.standard_normal(dh).astype(np.float32) for _ in range(2)]
    d = {m: ctx.upload(a) for m, a in dict(q=x[0], k=x[1], v=x[2], wq=w[0], wk=w[1]).items()}
    q_ref, k_ref, v_ref = ctx.empty((n, 8, dh)), ctx.empty((n, 1, dh)), ctx.empty((n, 1, dh))
    ctx.attn_producer(q=d["q"].ptr, k=d["k"].ptr, v=d["v"].ptr, q_norm=d["wq"].ptr, k_norm=d["wk"].ptr, q_out=q_ref.ptr,
                      k_cache=k_ref.ptr, v_cache=v_ref.ptr, T=n, Hq=8, Hkv=1, Dh=dh, rotary_dim=128, theta=1e6, eps=1e-6)
    out_ref, out = ctx.empty((T1, 8 * dh)), ctx.empty((T1, 8 * dh))
    row = 8 * dh * 4
    ctx.attention(q_ref.ptr + T0 * row, k_ref.ptr, v_ref.ptr, out_ref.ptr, T=T1, S=n, Hq=8, Hkv=1, Dh=dh, Dv=dh, q_pos0=T0,
                  scale=0.05)
    pool = [ctx.upload(np.full((12, page, 1, dh), np.nan, np.float32)) for _ in range(2)]
    m = {a: ctx.upload(np.asarray(b, np.uint32)) for a, b in dict(
        table=np.full((1, 10), ref.NO_ROW), lens=[0], new=[0], free=rng.permutation(12), state=[0, 12], slots=np.zeros(128),
        pos=np.zeros(128)).items()}
    cache = g4a.PagedCache(k_pages=pool[0].ptr, v_pages=pool[1].ptr, block_table=m["table"].ptr, kv_len=m["lens"].ptr,
                           n_seqs=1, pages_per_seq=10, n_pages=12, page_size=page, Hkv=1, Dh=dh)
    q_out = ctx.empty((n, 8, dh))
    for t0, T in ((0, T0), (T0, T1)):
        ctx.h2d(m["new"].ptr, np.array([T], np.uint32))
        ctx.page_map(cache, g4a.PageMapArgs(new_len=m["new"].ptr, free_pages=m["free"].ptr, free_state=m["state"].ptr,
                                            free_cap=12, rows=T, slots=m["slots"].ptr, positions=m["pos"].ptr))
        ctx.attn_producer_paged(cache, g4a.PagedProducerArgs(
            q=d["q"].ptr + t0 * row, k=d["k"].ptr + t0 * dh * 4, v=d["v"].ptr + t0 * dh * 4, q_norm=d["wq"].ptr,
            k_norm=d["wk"].ptr, q_out=q_out.ptr + t0 * row, positions=m["pos"].ptr, slots=m["slots"].ptr, T=T, Hq=8,
            rotary_dim=128, theta=1e6, eps=1e-6))
    k_all, v_all = ctx.empty((n, 1, dh)), ctx.empty((n, 1, dh))
    ctx.kv_gather_paged(cache, 0, 0, n, k_all.ptr, v_all.ptr)
    for a, b in ((k_all, k_ref), (v_all, v_ref), (q_out, q_ref)):
        x, y = a.to_host(), b.to_host()
        assert np.all(np.abs(x - y) <= 32 * ref.HALF * np.abs(y).max(-1, keepdims=True))
    ctx.attention(q_out.ptr + T0 * row, k_all.ptr, v_all.ptr, out.ptr, T=T1, S=n, Hq=8, Hkv=1, Dh=dh, Dv=dh, q_pos0=T0,
                  scale=0.05)
    # rows 32 half steps apart move a score of up to |q||k| * 0.05 = 26 by a walk of 512 of them over its terms
    assert np.abs(out.to_host() - out_ref.to_host()).max() <= 1e-4
    for a in (*d.values(), *pool, *m.values(), q_ref, k_ref, v_ref, out_ref, out, q_out, k_all, v_all):
        a.free()
