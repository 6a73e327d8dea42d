"""The paged KV cache's entry points on the host side of the library, over a stand-in
for the HIP runtime: what they refuse, with which code, and that a refused call
launches nothing; which kernels the others launch. CPU only."""
import numpy as np
import pytest

import hip_standin as hip
import paged_ref as ref
from hip_standin import PTR

ARG, SHAPE, UNSUPPORTED = -2, -3, -4


@pytest.fixture
def ctx():
    c = hip.binding().Context(0)
    hip.launches()
    yield c
    c.close()


def _cache(**kw):
    base = dict(k_pages=PTR, v_pages=PTR, block_table=PTR, kv_len=PTR, n_seqs=4, pages_per_seq=8, n_pages=64,
                page_size=16, Hkv=1, Dh=256, kv_type=0, ring=0)
    base.update(kw)
    return hip.binding().PagedCache(**base)


def _map(**kw):
    base = dict(free_pages=PTR, free_state=PTR, slots=PTR, positions=PTR, free_cap=64, rows=100)
    base.update(kw)
    return hip.binding().PageMapArgs(**base)


def _producer(**kw):
    base = dict(q=PTR, k=PTR, v=PTR, q_norm=PTR, k_norm=PTR, q_out=PTR, positions=PTR, slots=PTR, T=3, Hq=8,
                rotary_dim=256, theta=1e4, eps=1e-6)
    base.update(kw)
    return hip.binding().PagedProducerArgs(**base)


def _attn(**kw):
    base = dict(q=PTR, out=PTR, Hq=8, scale=1.0)
    base.update(kw)
    return hip.binding().PagedAttnArgs(**base)


def _refused(ctx, code, text, call, *args):
    with pytest.raises(hip.binding().G4aError) as e:
        call(*args)
    assert e.value.code == code and text in str(e.value), str(e.value)
    assert hip.launches() == []


POOLS = [
    (UNSUPPORTED, "page_size", dict(page_size=8)), (UNSUPPORTED, "page_size", dict(page_size=48)),
    (UNSUPPORTED, "page_size", dict(page_size=1 << 17)), (UNSUPPORTED, "page_size", dict(page_size=0)),
    (SHAPE, "slots", dict(n_pages=0)), (SHAPE, "slots", dict(n_pages=1 << 28, page_size=16)),
    (ARG, "ring", dict(ring=2)), (UNSUPPORTED, "head_dim", dict(Dh=96)), (UNSUPPORTED, "head_dim", dict(Dh=0)),
    (UNSUPPORTED, "Hkv", dict(Hkv=0)), (UNSUPPORTED, "Hkv", dict(Hkv=2000)), (ARG, "kv_type", dict(kv_type=2)),
    (ARG, "k_pages", dict(k_pages=None)), (ARG, "v_pages", dict(v_pages=PTR + 8)),
    (SHAPE, "page_stride", dict(page_stride=16 * 256 - 8)), (SHAPE, "page_stride", dict(page_stride=16 * 256 + 4)),
    (SHAPE, "page_stride", dict(page_stride=1 << 41)),
]
TABLES = [
    (ARG, "block_table", dict(block_table=None)), (ARG, "kv_len", dict(kv_len=None)),
    (SHAPE, "tables", dict(pages_per_seq=0)), (SHAPE, "tables", dict(pages_per_seq=1 << 28)),
    (SHAPE, "tables", dict(n_seqs=1 << 31, pages_per_seq=2)),
]


@pytest.mark.parametrize("code,text,kw", POOLS + TABLES)
def test_bad_caches_are_refused(ctx, code, text, kw):
    if text not in ("slots", "page_size", "ring") and (code, text, kw) not in TABLES:  # what page_map does not look at
        ctx.page_map(_cache(**kw), _map())
        assert len(hip.launches()) == 1
    else:
        _refused(ctx, code, text, ctx.page_map, _cache(**kw), _map())
    if (code, text, kw) not in TABLES:  # the producer looks at pools alone
        _refused(ctx, code, text, ctx.attn_producer_paged, _cache(**kw), _producer())
    _refused(ctx, code, text, ctx.attention_paged, _cache(**kw), _attn())
    _refused(ctx, code, text, ctx.kv_gather_paged, _cache(**kw), 0, 0, 5, PTR, PTR)


@pytest.mark.parametrize("code,text,kw", [
    (ARG, "slots", dict(slots=None)), (ARG, "positions", dict(positions=None)), (ARG, "free", dict(free_pages=None)),
    (ARG, "free", dict(free_state=None)), (ARG, "free", dict(free_cap=0)), (SHAPE, "rows", dict(rows=1 << 31)),
    (SHAPE, "rows", dict(rows_per_seq=1)),
])
def test_bad_maps_are_refused(ctx, code, text, kw):
    _refused(ctx, code, text, ctx.page_map, _cache(), _map(**kw))


@pytest.mark.parametrize("code,text,kw", [
    (ARG, "rotary_dim", dict(rotary_dim=3)), (ARG, "rotary_dim", dict(rotary_dim=258)), (ARG, "k and v", dict(k=None)),
    (UNSUPPORTED, "Hq", dict(Hq=0)), (SHAPE, "rows", dict(T=1 << 31)), (ARG, "null", dict(q=None)),
    (ARG, "null", dict(q_out=None)), (ARG, "null", dict(positions=None)), (ARG, "null", dict(slots=None)),
    (ARG, "aligned", dict(q=PTR + 4)), (ARG, "aligned", dict(k_norm=PTR + 8)),
])
def test_bad_producers_are_refused(ctx, code, text, kw):
    _refused(ctx, code, text, ctx.attn_producer_paged, _cache(), _producer(**kw))


@pytest.mark.parametrize("code,text,cache,kw", [
    (SHAPE, "Hq", {}, dict(Hq=0)), (SHAPE, "Hq", dict(Hkv=3), dict(Hq=8)), (SHAPE, "Hq", {}, dict(Hq=1 << 17)),
    (ARG, "softcap", {}, dict(attn_softcap=-1.0)), (ARG, "softcap", {}, dict(attn_softcap=float("nan"))),
    (ARG, "null", {}, dict(q=None)), (ARG, "aligned", {}, dict(out=PTR + 4)),
])
def test_bad_attention_calls_are_refused(ctx, code, text, cache, kw):
    _refused(ctx, code, text, ctx.attention_paged, _cache(**cache), _attn(**kw))


@pytest.mark.parametrize("code,text,args", [
    (ARG, "sequence", (4, 0, 5, PTR, PTR)), (SHAPE, "positions", (0, 0xFFFFFFF0, 32, PTR, PTR)),
    (ARG, "null", (0, 0, 5, None, PTR)), (ARG, "aligned", (0, 0, 5, PTR, PTR + 4)),
])
def test_bad_gathers_are_refused(ctx, code, text, args):
    _refused(ctx, code, text, ctx.kv_gather_paged, _cache(), *args)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_words_off_their_four_bytes_are_refused(ctx, off):
    """Tables, lengths, slots and positions are words at multiples of four bytes."""
    for field in ("block_table", "kv_len"):
        c = _cache(**{field: PTR + off})
        _refused(ctx, ARG, "aligned", ctx.page_map, c, _map())
        _refused(ctx, ARG, "aligned", ctx.attention_paged, c, _attn())
        _refused(ctx, ARG, "aligned", ctx.kv_gather_paged, c, 0, 0, 5, PTR, PTR)
        ctx.attn_producer_paged(c, _producer())  # which looks at the pools alone
        assert len(hip.launches()) == 1
    for field in ("new_len", "shared_pages", "free_pages", "free_state", "slots", "positions", "row_start", "added",
                  "kv_len_out", "free_state_out"):
        _refused(ctx, ARG, "aligned", ctx.page_map, _cache(), _map(**{field: PTR + off}))
    for field in ("positions", "slots"):
        _refused(ctx, ARG, "aligned", ctx.attn_producer_paged, _cache(), _producer(**{field: PTR + off}))
    ctx.page_map(_cache(block_table=PTR + 4, kv_len=PTR + 8), _map(slots=PTR + 4, free_state=PTR + 12))
    assert len(hip.launches()) == 1


def test_calls_past_a_launch_are_refused(ctx):
    """A launch counts its threads in 32 bits: 2^24 - 1 workgroups of 256. At 512 dims a wave takes two rows of a
    token, four waves a workgroup; a gather of 64-dim rows takes a page of 16 a workgroup."""
    most = (1 << 24) - 1
    ctx.attn_producer_paged(_cache(Dh=512), _producer(T=4 * most // 5))
    assert [x.gx for x in hip.launches()] == [(4 * most // 5 * 5 + 3) // 4]
    _refused(ctx, SHAPE, "rows", ctx.attn_producer_paged, _cache(Dh=512), _producer(T=4 * most // 5 + 1))
    ctx.kv_gather_paged(_cache(Dh=64), 0, 0, 16 * most, PTR, PTR)
    assert [x.gx for x in hip.launches()] == [most]
    _refused(ctx, SHAPE, "groups", ctx.kv_gather_paged, _cache(Dh=64), 0, 0, 16 * most + 1, PTR, PTR)


def test_maps_of_more_sequences_than_are_counted_are_refused(ctx):
    """The kernel counts sequences in 32 bits, up to 1024 past the last."""
    ctx.page_map(_cache(n_seqs=(1 << 31) - 1, pages_per_seq=1), _map())
    assert len(hip.launches()) == 1
    for n in (1 << 31, 0xFFFFFC01, 0xFFFFFFFE):
        _refused(ctx, SHAPE, "sequences", ctx.page_map, _cache(n_seqs=n, pages_per_seq=1), _map())


def test_calls_without_work_launch_nothing(ctx):
    ctx.page_map(_cache(n_seqs=0), _map(rows=0))
    ctx.attn_producer_paged(_cache(), _producer(T=0))
    ctx.attention_paged(_cache(n_seqs=0), _attn())
    ctx.kv_gather_paged(_cache(), 0, 7, 0, PTR, PTR)
    assert hip.launches() == []


def test_a_map_of_no_sequence_still_gives_its_end_and_the_ring_state(ctx):
    for kw in (dict(row_start=PTR), dict(free_state_out=PTR + 256)):
        ctx.page_map(_cache(n_seqs=0, block_table=None, kv_len=None), _map(rows=0, **kw))
        assert [x.name for x in hip.launches()] == ["g4a_page_map_t256"]
        _refused(ctx, ARG, "free", ctx.page_map, _cache(n_seqs=0), _map(rows=0, free_state=None, **kw))


def test_a_rotation_is_first_used_outside_a_capture(ctx):
    ctx.capture_begin()
    with pytest.raises(hip.binding().G4aError, match="capture"):
        ctx.attn_producer_paged(_cache(), _producer(theta=777.0))
    with pytest.raises(hip.binding().G4aError):
        ctx.capture_end()
    ctx.attn_producer_paged(_cache(), _producer(theta=777.0))
    ctx.attention_paged(_cache(), _attn())  # (and its workspace)
    ctx.capture_begin()
    ctx.page_map(_cache(), _map(rows=4, rows_per_seq=1))
    ctx.attn_producer_paged(_cache(), _producer(theta=777.0))
    ctx.attention_paged(_cache(), _attn())
    ctx.kv_gather_paged(_cache(), 0, 0, 5, PTR, PTR)
    ctx.capture_end().free()


def test_attention_launches(ctx):
    """What a call launches follows from its arguments: one decode and one merge kernel a launch of up to 1024
    sequences and 2048 head groups, no merge where no sequence can have more than the smallest part."""
    def names(**kw):
        attn = {k: kw.pop(k) for k in ("Hq", "sliding_window") if k in kw}
        ctx.attention_paged(_cache(**kw), _attn(**attn))
        return [x.name for x in hip.launches()]

    assert names(Dh=512) == ["g4a_paged_decode_d512_f32_h2", "g4a_paged_combine16_d512_f32_h2"]
    assert names(n_seqs=9, kv_type=1, Hq=4) == ["g4a_paged_decode_d256_bf16_h1", "g4a_paged_combine64_d256_bf16_h1"]
    assert names(sliding_window=100, Hq=9) == ["g4a_paged_decode_win_d256_f32_h4", "g4a_paged_combine16_d256_f32_h4"]
    # 50 tokens from the last row of a tile of 16 on touch five tiles (1 + 16 + 16 + 16 + 1), 49 at most four
    assert names(sliding_window=50) == ["g4a_paged_decode_win_d256_f32_h2", "g4a_paged_combine16_d256_f32_h2"]
    assert names(sliding_window=49) == ["g4a_paged_decode_win_d256_f32_h2"]
    assert names(pages_per_seq=4) == ["g4a_paged_decode_d256_f32_h2"]
    assert len(names(n_seqs=2100)) == 6 and len(names(n_seqs=1024)) == 2
    assert len(names(n_seqs=600, Hkv=4, Hq=32)) == 4


@pytest.mark.parametrize("window", [0, 64, 100])
@pytest.mark.parametrize("page,per_seq", [(16, 4), (32, 2), (64, 1)])
def test_a_ring_of_four_tiles_is_merged(ctx, page, per_seq, window):
    """64 tokens of a ring touch five tiles where the first of them is inside one; a table that is no ring starts
    with its first tile, and a ring of 48 touches four at most."""
    def names(ring, per_seq):
        ctx.attention_paged(_cache(page_size=page, pages_per_seq=per_seq, ring=ring), _attn(sliding_window=window))
        return [x.name for x in hip.launches()]

    decode = "g4a_paged_decode_win_d256_f32_h2" if window else "g4a_paged_decode_d256_f32_h2"
    assert names(1, per_seq) == [decode, "g4a_paged_combine16_d256_f32_h2"]
    assert names(0, per_seq) == [decode]
    if page == 16:
        assert names(1, 3) == [decode]


def test_attention_grows_its_workspace_outside_a_capture(ctx):
    ctx.attention_paged(_cache(), _attn())
    ctx.capture_begin()
    ctx.attention_paged(_cache(), _attn())
    with pytest.raises(hip.binding().G4aError, match="capture"):
        ctx.attention_paged(_cache(n_seqs=600, Dh=512, pages_per_seq=64), _attn())
    with pytest.raises(hip.binding().G4aError):
        ctx.capture_end()


def test_the_reference_map_keeps_every_page_once():
    """Steps of random demands: pages are owned by one sequence or free, never both, and
    slots of live tokens differ."""
    rng = np.random.default_rng(5)
    n, per_seq, page, cap = 6, 4, 16, 20
    lens, table = np.zeros(n, np.uint32), np.full((n, per_seq), ref.NO_ROW, np.uint32)
    free, first, count = rng.permutation(cap).astype(np.uint32), 3, cap
    for _ in range(60):
        new = np.where(rng.random(n) < 0.15, ref.NO_ROW, rng.integers(0, 30, n)).astype(np.uint32)
        slots, pos, start, added, lens, table, free, first, count = ref.page_map(
            lens, new, table, free, first, count, page=page, ring=False, rows=64)
        owned = [p for b in range(n) for p in table[b, :-(-int(lens[b]) // page)]]
        left = [free[(first + i) % cap] for i in range(count)]
        assert sorted(owned + left) == list(range(cap))
        live = slots[slots != ref.NO_ROW]
        assert len(set(live)) == len(live) == added.sum() == start[n]
