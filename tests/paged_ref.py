"""The paged KV cache's operators from their definitions (include/g4a.h), on the host:
page maps by walking the sequences, attention and the producer in 64 bits."""
import numpy as np

NO_ROW = 0xFFFFFFFF
HALF = 2.0 ** -24  # half a step of f32, relative


def bf16_bits(x):
    """f32 values as bfloat16 words, rounded to nearest even (NaN stays NaN)."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def bf16_values(bits):
    return (np.asarray(bits, np.uint32) << 16).view(np.float32)


def pack(x, kv_type):
    return bf16_bits(x) if kv_type == "bf16" else np.ascontiguousarray(x, np.float32)


def unpack(x, kv_type):
    return bf16_values(x) if kv_type == "bf16" else x


def page_map(lens, new, table, free, first, count, *, page, ring, rows, rows_per_seq=0, shared=None):
    """One step, a sequence after the other: (slots, positions, row_start, added, lens, table, free, first, count)."""
    n, per_seq = table.shape
    table, free, cap = table.copy(), free.copy(), len(free)
    slots, positions = np.full(rows, NO_ROW, np.uint32), np.full(rows, NO_ROW, np.uint32)
    row_start, added, out = np.zeros(n + 1, np.uint32), np.zeros(n, np.uint32), np.zeros(n, np.uint32)
    demand = rows_so_far = row = taken = 0
    given = []

    def pages(tokens):
        return min(-(-tokens // page), per_seq)

    for b in range(n):
        length = int(lens[b])
        ends = int(new[b]) == NO_ROW
        want = 0 if ends else int(new[b])
        fits = (length + want < NO_ROW if ring else length + want <= per_seq * page) and (
            rows_per_seq == 0 or want <= rows_per_seq)
        had = pages(length)
        need = pages(length + want) - had if fits and want else 0
        demand += need
        goes = fits and (need == 0 or demand <= count)
        rows_so_far += want if goes else 0
        goes = goes and (rows_per_seq > 0 or rows_so_far <= rows)
        row_start[b] = b * rows_per_seq if rows_per_seq else row
        if goes:
            for e in range(had, had + need):
                table[b, e] = free[(first + taken) % cap]
                taken += 1
            for i in range(want):
                pos = length + i
                p = table[b, (pos // page) % per_seq]
                r = row_start[b] + i
                positions[r] = pos
                if not ring or pos + per_seq * page >= length + want:
                    slots[r] = p * page + pos % page
            added[b] = want
            row += want
        if ends:
            given += list(table[b, (min(int(shared[b]), had) if shared is not None else 0):had])
        out[b] = 0 if ends else length + added[b]
    row_start[n] = n * rows_per_seq if rows_per_seq else row
    for i, p in enumerate(given):
        free[(first + count + i) % cap] = p
    return slots, positions, row_start, added, out, table, free, (first + taken) % cap, count - taken + len(given)


def tokens(pool, table, b, length, *, page, ring, n_pages, window=0):
    """(positions, rows) of the tokens of sequence b that a query at its end sees, in the pool [pages, page, ...]."""
    per_seq = table.shape[1]
    if not ring:
        length = min(length, per_seq * page)
    lo = max(0, length - (window or length))
    if ring:
        lo = max(lo, length - per_seq * page)
    t = np.arange(lo, length)
    p = table[b, (t // page) % per_seq]
    t, p = t[p < n_pages], p[p < n_pages]
    return t, pool[p, t % page]


def attention(q, k_pool, v_pool, table, lens, *, page, ring=False, n_pages, window=0, scale=1.0, cap=0.0):
    """(out, bound) in 64 bits: bound is what f32 arithmetic may be off by, elementwise. A score is a sum
    of Dh products; its roundings add up as a random walk of Dh steps of at most half a step of the partial
    sums, whose size is |q||k| / sqrt(Dh) or the score itself: 8 standard deviations of it, 8 * sqrt(Dh / 12)
    half steps. The scale, soft-cap, difference and exponential add a few half steps of the score, and the
    sums over N tokens a walk of N."""
    n, hq, dh = q.shape
    hkv = k_pool.shape[2]
    out, bound = np.zeros((n, hq, dh)), np.zeros((n, hq, dh))
    for b in range(n):
        _, k = tokens(k_pool, table, b, int(lens[b]), page=page, ring=ring, n_pages=n_pages, window=window)
        _, v = tokens(v_pool, table, b, int(lens[b]), page=page, ring=ring, n_pages=n_pages, window=window)
        if not len(k):
            continue
        for h in range(hq):
            kh, vh = (x[:, h // (hq // hkv)].astype(np.float64) for x in (k, v))
            s = kh @ q[b, h].astype(np.float64)
            size = max(np.abs(s).max(), np.linalg.norm(q[b, h]) * np.linalg.norm(kh, axis=1).max() / np.sqrt(dh))
            s = s * scale
            s = cap * np.tanh(s / cap) if cap else s
            e = np.exp(s - s.max())
            p = e / e.sum()
            out[b, h] = p @ vh
            steps = abs(scale) * size * (8 * np.sqrt(dh / 12) + 8) + 16 + 8 * np.sqrt(len(kh) / 12)
            bound[b, h] = 2 * HALF * steps * (p @ np.abs(vh)) + 1e-30
    return out.reshape(n, -1), bound.reshape(n, -1)


def rms(x, w, eps):
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return y if w is None else y * w.astype(np.float64)


def rope(x, pos, rot, theta):
    """Half-split rotation of x [T, heads, Dh]; frequency and angle are f32, as the library's are."""
    half = rot // 2
    expo = -(2.0 * np.arange(half, dtype=np.float32)) / np.float32(max(rot, 1))
    freq = (float(np.float32(theta)) ** expo.astype(np.float64)).astype(np.float32)
    ang = (pos.astype(np.float32)[:, None] * freq).astype(np.float64)[:, None]
    a, b = x[..., :half], x[..., half:rot]
    return np.concatenate([a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang), x[..., rot:]], -1)
