"""Pages of 8 and 4 bits on the host side of the library, over a stand-in for the HIP runtime: sizes, refusals, which
kernels a call launches; and the test's own form of the format against exact fractions. CPU only."""
from fractions import Fraction

import numpy as np
import pytest

import hip_standin as hip
import quant_ref as quant
from hip_standin import PTR
from test_paged_host import ARG, SHAPE, UNSUPPORTED, _attn, _cache, _producer, _refused, ctx  # noqa: F401

TYPES = {"i4": 4, "i8": 8}


# ---- the format --------------------------------------------------------------------

def _bf16_at_least(x):
    """The least bfloat16 >= 2^-126 that is at least the fraction x."""
    f = Fraction(1, 2 ** 126)
    while f * 2 <= x:
        f *= 2
    if x <= f:
        return f
    step = f / 128
    return -(-x // step) * step


@pytest.mark.parametrize("kv_type", TYPES)
def test_the_format_against_fractions(kv_type):
    rng = np.random.default_rng(1)
    rows = [rng.standard_normal(64), np.zeros(64), np.full(64, -3.0), np.arange(64) - 31.5, np.where(np.arange(64) == 40, 1e30, 1e-3),
            rng.standard_normal(64) * 10.0 ** rng.uniform(-20, 20, 64), np.full(64, 1e-40), np.tile([127.5, -127.5, 0.5, 1.5], 16),
            np.tile([2.0, -2.0, 1.0, 0.0], 16)]
    for x in rows:
        x = np.asarray(x, np.float32)
        n, sub, s = quant.encode(x, kv_type)
        exact = [Fraction(float(y)) for y in x]
        most = 127 if kv_type == "i8" else 1016
        S = _bf16_at_least(max(map(abs, exact)) / most)
        assert Fraction(float(s)) == S
        for g in range(2):
            part, step = exact[32 * g:32 * g + 32], S
            if kv_type == "i4":
                high, low = max(part), -min(part)
                c = max(1, -(-max(high, low) // (8 * S)))
                c = int(c)
                assert c <= 127 and sub[g] == (-c if high >= low else c)
                step = S * int(sub[g])
            for i, y in enumerate(part):
                want = round(y / step)  # (halves to even)
                want = want if kv_type == "i8" else min(7, max(-8, want))
                assert n[32 * g + i] == want and abs(want) <= 128
                off = abs(want * step - y)
                assert off <= abs(step) / 2 or (kv_type == "i4" and want == 7 and off <= abs(step))


@pytest.mark.parametrize("kv_type", TYPES)
def test_how_far_a_value_may_be_off(kv_type):
    """A half step against the largest magnitudes of row and group, as the binding's notes state it, in rows with and
    without outliers. S is below its least real number by a factor of at most 1 + 2^-7 (bfloat16), 1016 / 1008 and 127 / 126;
    |sub| is below its least real number + 1. So a step of 4 bits is below group / 8 + row / 1008."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4000, 512)).astype(np.float32)
    x[1000:] *= np.float32(2.0) ** rng.integers(-12, 3, (3000, 16)).repeat(32, axis=1).astype(np.float32)
    x[np.arange(2000, 4000), rng.integers(0, 512, 2000)] = 10.0 ** rng.uniform(0, 4, 2000)
    x[3000:] *= (2.0 ** rng.uniform(-116, 100, 1000)).astype(np.float32)[:, None]
    off = np.abs(quant.values(x, kv_type).astype(np.float64) - x)
    row = np.maximum(np.abs(x).max(-1), np.float32(2.0 ** -116 if kv_type == "i4" else 2.0 ** -119))[:, None].astype(np.float64)
    if kv_type == "i8":
        assert (off <= row / 252).all() and (off / row).max() > 0.98 / 252
        return
    g = x.reshape(4000, 16, 32).astype(np.float64)
    group = np.abs(g).max(-1, keepdims=True)
    half = (group / 16 + row[..., None] / 2016).repeat(32, -1)
    opposite = np.where(g.max(-1, keepdims=True) >= -g.min(-1, keepdims=True), g < 0, g > 0)
    off = off.reshape(g.shape)
    assert (off < np.where(opposite, 2 * half, half)).all()
    inner = np.where(opposite, 0, off / half)
    assert inner.max() > 0.95 and (inner[2000:] > 1 / 16 * (group / half)[2000:]).any(), "not below 1/16 of the group's"
    # a group far below its row's largest value
    x = np.zeros(64, np.float32)
    x[3], x[32:] = 1016.0, 0.45
    assert not quant.values(x, kv_type)[32:].any() and quant.values(x, kv_type)[3] == 1016.0


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("vals", [False, True])
@pytest.mark.parametrize("dh,hkv,page", [(64, 1, 16), (128, 3, 32), (256, 2, 16), (512, 1, 64)])
def test_pages_hold_what_was_packed(kv_type, vals, dh, hkv, page):
    rng = np.random.default_rng(dh)
    buf = rng.integers(0, 256, (3, quant.page_bytes(dh, hkv, page, kv_type)), dtype=np.uint8)
    x = rng.standard_normal((20, hkv, dh)).astype(np.float32)
    at = rng.permutation(3 * page)[:20]
    quant.pack(buf, at // page, at % page, x, dh, hkv, page, kv_type, vals)
    got = quant.unpack(buf, dh, hkv, page, kv_type, vals)
    assert np.array_equal(got[at // page, at % page], quant.values(x, kv_type))


# ---- the library --------------------------------------------------------------------

@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("dh,hkv,page", [(64, 1, 16), (128, 3, 32), (256, 1, 256), (512, 2, 16)])
def test_page_bytes(ctx, kv_type, dh, hkv, page):  # noqa: F811
    def size(**kw):
        return ctx.kv_page_bytes(_cache(Dh=dh, Hkv=hkv, page_size=page, **{"kv_type": TYPES[kv_type], **kw}))

    assert size() == quant.page_bytes(dh, hkv, page, kv_type)
    assert size(k_pages=None, v_pages=None, n_pages=0, n_seqs=0, block_table=None) == size()
    assert size(page_stride=size() + 48) == size() + 48
    assert size(kv_type=0) == 4 * page * hkv * dh and size(kv_type=1, page_stride=page * hkv * dh + 8) == 2 * page * hkv * dh + 16


def test_page_bytes_needs_no_context():
    import ctypes
    lib, n = hip.binding().load_library(), ctypes.c_uint64()
    assert lib.g4a_kv_page_bytes(None, ctypes.byref(_cache(kv_type=4, Dh=512)), ctypes.byref(n)) == 0
    assert n.value == quant.page_bytes(512, 1, 16, "i4")
    assert lib.g4a_kv_page_bytes(None, ctypes.byref(_cache(kv_type=2)), ctypes.byref(n)) == ARG
    assert b"kv_type" in lib.g4a_last_error(None)
    assert lib.g4a_kv_page_bytes(None, None, ctypes.byref(n)) == ARG
    assert lib.g4a_kv_page_bytes(None, ctypes.byref(_cache()), None) == ARG


def test_page_bytes_refuses_and_leaves_a_capture_open(ctx):  # noqa: F811
    ctx.capture_begin()
    for code, text, kw in [(UNSUPPORTED, "page_size", dict(page_size=24)), (UNSUPPORTED, "head_dim", dict(Dh=96)),
                           (UNSUPPORTED, "Hkv", dict(Hkv=0)), (ARG, "kv_type", dict(kv_type=3)),
                           (SHAPE, "16 bytes", dict(kv_type=8, page_stride=1 << 20 | 8))]:
        _refused(ctx, code, text, ctx.kv_page_bytes, _cache(**kw))
    ctx.capture_end().free()


@pytest.mark.parametrize("kv_type", [2, 3, 5, 6, 7, 9, 16, 32, 0xFFFFFFFF])
def test_other_types_are_refused(ctx, kv_type):  # noqa: F811
    c = _cache(kv_type=kv_type)
    for call in (lambda: ctx.attention_paged(c, _attn()), lambda: ctx.attn_producer_paged(c, _producer()),
                 lambda: ctx.kv_gather_paged(c, 0, 0, 5, PTR, PTR), lambda: ctx.kv_write_paged(c, PTR, PTR, PTR, 3),
                 lambda: ctx.kv_read_paged(c, PTR, 3, PTR, PTR)):
        _refused(ctx, ARG, "kv_type", call)


@pytest.mark.parametrize("kv_type", TYPES)
def test_bad_pages_are_refused(ctx, kv_type):  # noqa: F811
    size = quant.page_bytes(256, 1, 16, kv_type)
    for code, text, kw in [(SHAPE, "page_stride", dict(page_stride=size - 16)), (SHAPE, "page_stride", dict(page_stride=size + 8)),
                           (SHAPE, "page_stride", dict(page_stride=1 << 41)), (ARG, "v_pages", dict(v_pages=PTR + 8)),
                           (ARG, "k_pages", dict(k_pages=None)), (UNSUPPORTED, "head_dim", dict(Dh=1024))]:
        c = _cache(kv_type=TYPES[kv_type], **kw)
        for call in (lambda: ctx.attention_paged(c, _attn()), lambda: ctx.attn_producer_paged(c, _producer()),
                     lambda: ctx.kv_gather_paged(c, 0, 0, 5, PTR, PTR), lambda: ctx.kv_write_paged(c, PTR, PTR, PTR, 3),
                     lambda: ctx.kv_read_paged(c, PTR, 3, PTR, PTR)):
            _refused(ctx, code, text, call)


@pytest.mark.parametrize("kv_type", [0, 1, 4, 8])
def test_bad_rows_are_refused(ctx, kv_type):  # noqa: F811
    c = _cache(kv_type=kv_type)
    for args in ((None, PTR, PTR, 3), (PTR, None, PTR, 3), (PTR, PTR, None, 3), (PTR + 4, PTR, PTR, 3), (PTR, PTR + 8, PTR, 3),
                 (PTR, PTR, PTR + 2, 3)):
        _refused(ctx, ARG, "aligned", ctx.kv_write_paged, c, *args)
        _refused(ctx, ARG, "aligned", ctx.kv_read_paged, c, args[2], args[3], args[0], args[1])
    _refused(ctx, ARG, "null cache", ctx.kv_write_paged, None, PTR, PTR, PTR, 3)
    _refused(ctx, SHAPE, "rows", ctx.kv_write_paged, _cache(kv_type=kv_type, Hkv=1024), PTR, PTR, PTR, 1 << 31)
    _refused(ctx, SHAPE, "rows", ctx.kv_read_paged, _cache(kv_type=kv_type, Hkv=1024), PTR, 1 << 31, PTR, PTR)
    ctx.kv_write_paged(c, None, None, None, 0)
    ctx.kv_read_paged(c, None, 0, None, None)
    assert hip.launches() == []


@pytest.mark.parametrize("kv_type", TYPES)
def test_launches(ctx, kv_type):  # noqa: F811
    """One launch each but for the attention's merge; the query rows alone need nothing of the pages' type."""
    def names(call, *args):
        call(*args)
        return [x.name for x in hip.launches()]

    c = _cache(kv_type=TYPES[kv_type], Dh=512)
    assert names(ctx.attn_producer_paged, c, _producer()) == [f"g4a_paged_producer_d512_{kv_type}"]
    assert names(ctx.attn_producer_paged, c, _producer(k=None, v=None, slots=None)) == ["g4a_paged_producer_d512_f32"]
    assert names(ctx.kv_write_paged, c, PTR, PTR, PTR, 3) == [f"g4a_paged_write_d512_{kv_type}"]
    assert names(ctx.kv_read_paged, c, PTR, 3, PTR, PTR) == [f"g4a_paged_read_d512_{kv_type}"]
    assert names(ctx.kv_gather_paged, c, 1, 5, 100, PTR, PTR) == [f"g4a_paged_read_d512_{kv_type}"]
    got = names(ctx.attention_paged, _cache(kv_type=TYPES[kv_type], Dh=512, pages_per_seq=9), _attn())
    assert got == [f"g4a_paged_decode_d512_{kv_type}_h2", f"g4a_paged_combine16_d512_{kv_type}_h2"]
    # eight waves, a tile of 16 tokens each, are the smallest part there
    assert names(ctx.attention_paged, c, _attn()) == got[:1]
    # units for every CU: two workgroups of four waves a CU at 512 dims
    many = _cache(kv_type=TYPES[kv_type], Dh=512, n_seqs=256)
    assert names(ctx.attention_paged, many, _attn())[0] == f"g4a_paged_decode_many_d512_{kv_type}_h2"
    assert names(ctx.attention_paged, many, _attn(Hq=3, sliding_window=90))[0] == f"g4a_paged_decode_many_win_d512_{kv_type}_h1"
    assert names(ctx.attention_paged, many, _attn(Hq=9))[0] == f"g4a_paged_decode_d512_{kv_type}_h4"
    assert names(ctx.attention_paged, _cache(kv_type=TYPES[kv_type], Dh=512, n_seqs=255), _attn())[0] == got[0]
    ctx.capture_begin()
    ctx.attention_paged(c, _attn())
    ctx.kv_write_paged(c, PTR, PTR, PTR, 3)
    ctx.kv_read_paged(c, PTR, 3, PTR, PTR)
    ctx.kv_gather_paged(c, 1, 5, 100, PTR, PTR)
    ctx.capture_end().free()


def test_producers_past_a_launch_are_refused(ctx):  # noqa: F811
    """The waves of the K and V rows count too: at 512 dims and 8 query heads four and a half waves of two turns a token,
    and two of K and V."""
    for kv_type in TYPES.values():
        _refused(ctx, SHAPE, "rows", ctx.attn_producer_paged, _cache(Dh=512, kv_type=kv_type), _producer(T=1 << 25))
        ctx.attn_producer_paged(_cache(Dh=512, kv_type=kv_type), _producer(T=1 << 23))
        assert hip.launches()[0].gx == (4 << 21) + (2 << 21)
