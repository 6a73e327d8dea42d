"""Pages of 8 and 4 bits from their definition (include/g4a.h), on the host: rows to whole numbers and scales and
back, and the bytes of pages. In 64 bits, where every quantity below is exact or far from where it would be rounded
another way: x has 24 bits, S 8 and sub 7, so a quotient that is no whole number (or half of one) is at least 2^-40 of
itself away from it."""
import numpy as np

import paged_ref as ref

BITS = {"i8": 8, "i4": 4}


def page_bytes(dh, hkv, page, kv_type):
    bits = BITS[kv_type]
    raw = hkv * page * (dh * bits // 8 + (dh // 32 if bits == 4 else 0) + 2)
    return -(-raw // 128) * 128


def scale(big, most):
    """The least bfloat16 s >= 2^-126 with most * s >= big."""
    m, e = np.frexp(big / most)
    return np.maximum(np.ldexp(np.ceil(m * 256) / 256, e), 2.0 ** -126)


def encode(x, kv_type):
    """f32 rows [..., dh] as (n [..., dh], sub [..., groups] or None, S [...])."""
    x = np.asarray(x, np.float32).astype(np.float64)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], 0.0, x)
    big = np.abs(x).max(-1)
    if kv_type == "i8":
        s = scale(big, 127.0)
        n, sub = np.rint(x / s[..., None]), None
    else:
        s = scale(big, 1016.0)
        g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
        high, low = g.max(-1), -g.min(-1)
        c = np.maximum(np.ceil(np.maximum(high, low) / (8 * s[..., None])), 1.0)
        sub = np.where(high >= low, -c, c)
        n = np.clip(np.rint(g / (s[..., None] * sub)[..., None]), -8, 7).reshape(x.shape)
        sub = sub.astype(np.int64)
    return n.astype(np.int64), sub, np.where(bad, np.nan, s)


def decode(n, sub, s):
    if sub is not None:
        n = (n.reshape(*sub.shape, 32) * sub[..., None]).reshape(n.shape)
    with np.errstate(over="ignore"):
        return (n * s[..., None]).astype(np.float32)


def values(x, kv_type):
    """What rows stand for once written, as f32."""
    return decode(*encode(x, kv_type))


def _parts(buf, dh, hkv, page, kv_type, vals):
    """Views of pages' bytes [pages, page_bytes]: rows [pages, hkv, page, bytes], subs [pages, hkv, tile, 16, G] in the
    order of groups (a copy's index list for K), S [pages, hkv, tile, 16, 2]."""
    bits = BITS[kv_type]
    rb, G = dh * bits // 8, dh // 32 if bits == 4 else 0
    data = hkv * page * rb
    rows = buf[:, :data].reshape(len(buf), hkv, page, rb)
    meta = buf[:, data:data + hkv * page // 16 * (16 * G + 32)].reshape(len(buf), hkv, page // 16, 16 * G + 32)
    return rows, meta[..., :16 * G], meta[..., 16 * G:].reshape(len(buf), hkv, page // 16, 16, 2)


def _places(dh):
    G = dh // 32
    return np.array([g % 4 * (G // 4) + g // 4 if G >= 4 else g for g in range(G)])


def pack(buf, page_no, row, x, dh, hkv, page, kv_type, vals):
    """Rows x [N, hkv, dh] into (page_no, row) [N] of pages' bytes, in place."""
    for i in range(len(page_no)):  # (a view of a view of `buf` a row: plain assignments)
        n, sub, s = encode(x[i], kv_type)
        rows, subs, scales = (v[page_no[i]] for v in _parts(buf, dh, hkv, page, kv_type, vals))
        if kv_type == "i8":
            rows[:, row[i]] = n + 128
        else:
            rows[:, row[i]] = n[:, 0::2] + 8 | n[:, 1::2] + 8 << 4
            G = dh // 32
            place = np.arange(G) * 16 + row[i] % 16 if vals else row[i] % 16 * G + _places(dh)
            subs[:, row[i] // 16, place] = sub + 128
        word = np.where(np.isnan(s), 0x7FC0, s.astype(np.float32).view(np.uint32) >> 16).astype(np.uint32)
        scales[:, row[i] // 16, row[i] % 16, 0] = word & 255
        scales[:, row[i] // 16, row[i] % 16, 1] = word >> 8


def unpack(buf, dh, hkv, page, kv_type, vals):
    """Every row of pages' bytes as f32 values [pages, page, hkv, dh]."""
    rows, subs, scales = _parts(buf, dh, hkv, page, kv_type, vals)
    word = (scales[..., 0].astype(np.uint32) | scales[..., 1].astype(np.uint32) << 8) << 16
    with np.errstate(invalid="ignore"):
        s = word.view(np.float32).astype(np.float64).reshape(len(buf), hkv, page)
    if kv_type == "i8":
        n, sub = rows.astype(np.int64) - 128, None
    else:
        n = np.stack([rows & 15, rows >> 4], -1).reshape(len(buf), hkv, page, dh).astype(np.int64) - 8
        G = dh // 32
        sub = subs.astype(np.int64) - 128
        sub = sub.reshape(*sub.shape[:3], G, 16).swapaxes(-1, -2) if vals else sub.reshape(*sub.shape[:3], 16, G)[..., _places(dh)]
        sub = sub.reshape(len(buf), hkv, page, G)
    with np.errstate(invalid="ignore"):
        return decode(n, sub, s).swapaxes(1, 2)


def attention(q, k, v, table, lens, *, scale=1.0, ring=False, **kw):
    """paged_ref.attention on the values of the pages, its bound widened by what the queries and probabilities of
    two fp16 parts are off: 2^-22 of a value of a score's terms (|q||k| at most in all) and of a probability's, and 2^-31 of
    the largest value seen for each token: fp16 ends in steps of 2^-24, so a low part is off by 2^-25 at least, where a
    weight e^(s - m) of 1 with the largest S seen stands at 2^6 and more, and the weights' sum is at least 1."""
    out, bound = ref.attention(q, k, v, table, lens, scale=scale, ring=ring, **kw)
    n, hq, dh = q.shape
    group = hq // k.shape[2]
    opts = {x: kw[x] for x in ("page", "n_pages", "window") if x in kw}
    opts["ring"] = ring
    wide = bound.reshape(n, hq, dh).copy()
    for b in range(n):
        _, kk = ref.tokens(k, table, b, int(lens[b]), **opts)
        _, vv = ref.tokens(v, table, b, int(lens[b]), **opts)
        if not len(kk):
            continue
        for h in range(hq):
            kh, vh = (x[:, h // group].astype(np.float64) for x in (kk, vv))
            s = kh @ q[b, h].astype(np.float64) * scale
            if kw.get("cap"):
                s = kw["cap"] * np.tanh(s / kw["cap"])
            p = np.exp(s - s.max())
            p /= p.sum()
            score = 2.0 ** -22 * abs(scale) * np.linalg.norm(q[b, h]) * np.linalg.norm(kh, axis=1).max()
            wide[b, h] += (2 * score + 2.0 ** -22) * (p @ np.abs(vh)) + 2.0 ** -31 * len(kh) * np.abs(vh).max()
    return out, wide.reshape(bound.shape)


def attention_sharp(q, k, v, table, lens, *, page, n_pages, ring=False, window=0, scale=1.0, cap=0.0):
    """attention() for values of any magnitude and for long contexts: what fp16's last step costs a weight (2^-31 of the
    largest value seen, and at least of 2^-90) is divided by the weights' sum, as the weight is, and nothing absolute is
    added. The other terms are those of paged_ref.attention and attention()."""
    n, hq, dh = q.shape
    out, bound = np.zeros((n, hq, dh)), np.zeros((n, hq, dh))
    opts = dict(page=page, ring=ring, n_pages=n_pages, window=window)
    for b in range(n):
        kk, vv = (ref.tokens(x, table, b, int(lens[b]), **opts)[1] for x in (k, v))
        if not len(kk):
            continue
        for h in range(hq):
            kh, vh = (x[:, h // (hq // k.shape[2])].astype(np.float64) for x in (kk, vv))
            s = kh @ q[b, h].astype(np.float64)
            length = np.linalg.norm(q[b, h]) * np.linalg.norm(kh, axis=1).max()
            size = max(np.abs(s).max(), length / np.sqrt(dh))
            s = s * scale
            s = cap * np.tanh(s / cap) if cap else s
            e = np.exp(s - s.max())
            p = e / e.sum()
            out[b, h] = p @ vh
            steps = abs(scale) * size * (8 * np.sqrt(dh / 12) + 8) + 16 + 8 * np.sqrt(len(kh) / 12)
            part = 2.0 ** -22 * (2 * abs(scale) * length + 1)
            bound[b, h] = (2 * ref.HALF * steps + part) * (p @ np.abs(vh)) + 2.0 ** -31 * len(kh) / e.sum() * max(
                np.abs(vh).max(), 2.0 ** -90)
    return out.reshape(n, -1), bound.reshape(n, -1)
