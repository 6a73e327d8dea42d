// Decode attention over a paged KV cache for gfx950: one query of every sequence
// over its visible tokens len - window <= t < len (window 0: all of them),
//   out[b, h] = sum_t softmax_t(cap(scale * q[b, h] . K[t])) V[t],
// cap(s) = softcap * tanh(s / softcap) where set; zeros without a visible token.
// Layout: G4aPaged (g4a_params.h); lengths and tables are read on the device, so a
// captured call replays with whatever they hold.
//
// Work. A unit is a sequence and up to 16 query heads of one kv head; its keys are
// tiles of 16 tokens, which lie on one page. A workgroup takes one part of a unit: the
// parts of a unit are even, of at most `quota` tiles, which is the tiles of all units
// over the workgroups there are beside one a unit. Each workgroup finds quota and its
// part from the lengths itself. A part that is its whole unit writes the output, any
// other a partial (O, m, l), which paged_combine merges. (Equal runs of tiles across
// units, with the next unit's first tile loaded behind the last of the one before,
// balanced better and were slower: 16 ragged sequences 52.0 against 48.3 us, 128 of 4 kv
// heads 68.2 against 55.8: several merges a workgroup, and 40 more registers.)
//
// A workgroup is 4 waves, each on every fourth tile of its part, with K and V of
// the next tile in flight in registers (16-byte loads; no LDS in between):
//   scores: K is the B operand of 16x16 MFMAs as it is loaded (lane = key l % 16 and
//           a quarter of the dims), the query rows A, out of LDS: f32 pages on
//           v_mfma_f32_16x16x4_f32, bf16 pages on v_mfma_f32_16x16x32_bf16 with the
//           query as three bf16 parts, whose sum it is exactly;
//   softmax: running maximum and sum in f32, a row of lanes per 4 heads;
//   P.V:    v_mfma_f32_4x4x1_16b_f32, in f32: V is B as it is loaded (a lane's dims are
//           columns of its block), P is A, one key of it broadcast to all blocks by the
//           instruction; bf16 values become f32 by a shift.
// The waves' partials join through LDS at the end.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "g4a_math.h"
#include "g4a_params.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <int DH, typename KV, int NHQ>
struct PagedCfg {
    static constexpr bool BF = sizeof(KV) == 2;
    static constexpr int HR = 4 * NHQ;                       // query heads of a unit
    static constexpr int EL = 16 / (int)sizeof(KV);          // values of a 16-byte load
    static constexpr int LG = DH / EL < 64 ? DH / EL : 64;   // lanes of a V row
    static constexpr int LPK = DH / (EL * LG);               // V loads per row and lane
    static constexpr int NK = 64 / LG;                       // V rows of a load
    static constexpr int KI = 16 / NK;                       // V loads (times LPK) of a tile
    static constexpr int CBSZ = KI == 16 ? 4 : KI == 8 ? 3 : KI == 4 ? 2 : 1;  // log2 KI: blocks a key of P goes to
    static constexpr int NDG = EL * LPK;                     // 4 x 64 accumulators per 4 heads
    static constexpr int KC = DH / (4 * EL);                 // K loads of a tile
    static constexpr int NM = NHQ == 1 ? 1 : NHQ == 2 ? 2 : 3;  // bf16: MFMAs per K load's dims
    // 16-byte query blocks in LDS: [K load][dim group][head], bf16 for each of three parts (half the
    // banks apart, as the lanes of one read take two of them)
    static constexpr int QPART = KC * 4 * HR + 8;
    static constexpr int QS = BF ? 3 * QPART : KC * 4 * HR;
    static constexpr int QL = (HR * DH / EL + 255) / 256;    // 16-byte (bf16: 32-byte) query pieces of a thread
    static constexpr int ITEMS = NHQ * NDG * LG;             // = NHQ * DH: (4 heads, dim) of a partial
    static constexpr int MRG = 4 * NHQ * NDG * 64;           // 16-byte blocks of the waves' accumulators
    static constexpr int SM = (QS > MRG ? QS : MRG) * 16;    // the two never live at once
};

// A sequence's visible tiles: tokens [lo, len), tiles first .. first + n - 1 of 16 tokens.
struct PagedSpan {
    uint32_t lo, len, first, n;
};

__device__ __forceinline__ PagedSpan paged_span(const G4aPagedAttnParams& p, uint32_t len) {
    PagedSpan s;
    s.len = p.c.ring ? len : min(len, p.room);
    s.lo = s.len > p.span ? s.len - p.span : 0u;
    s.first = s.lo / 16;
    s.n = s.len ? (s.len - 1) / 16 + 1 - s.first : 0u;
    return s;
}

// Sums over the lanes up to and with this one: four shifts within the rows of 16 lanes,
// then the rows' last lanes to the rows behind them.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t add_dpp(uint32_t x) {
    return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_incl_sum(uint32_t x) {
    x = add_dpp<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
    x = add_dpp<0x112, 0xf>(x);
    x = add_dpp<0x114, 0xf>(x);
    x = add_dpp<0x118, 0xf>(x);
    x = add_dpp<0x142, 0xa>(x);  // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
    return add_dpp<0x143, 0xc>(x);
}

// A word that no workgroup writes, at an address all lanes share: a scalar load, which no
// vector load in flight delays.
__device__ __forceinline__ uint32_t load_scalar(const uint32_t* p, size_t i) {
    return reinterpret_cast<const __attribute__((address_space(4))) uint32_t*>(reinterpret_cast<uintptr_t>(p))[i];
}

// A 64-bit value that all lanes share, in scalar registers.
__device__ __forceinline__ size_t uniform(size_t x) {
    return (size_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

// N pieces of 16 bytes of a tile of K or V, PER of them `apart` bytes from one another in each
// of N / PER rows that are `step` bytes apart; `off` is the lane's. Buffer loads: the row is a
// scalar offset (as global loads each took a 64-bit vector sum, and registers for it), and what
// lies behind the tile's `bytes` is not read. NT: past the caches.
template <bool NT, int N, int PER, int APART>
__device__ __forceinline__ void load_pieces(u32x4 (&x)[N], const char* tile, uint32_t bytes, uint32_t step, uint32_t off) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(tile), 0, (int)bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < N / PER; ++i)
#pragma unroll
        for (int y = 0; y < PER; ++y)
            x[i * PER + y] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off + APART * y, (int)(i * step), NT ? 2 : 0);
}

// One V row's element as f32.
template <bool BF>
__device__ __forceinline__ float v_value(const u32x4& v, int c) {
    if constexpr (BF) return __uint_as_float(c & 1 ? v[c / 2] & 0xFFFF0000u : v[c / 2] << 16);
    else return __uint_as_float(v[c]);
}

// acc[hq][dg] += P[key II of each block group][4 heads] x V's values of that load.
template <typename C, int II>
__device__ __forceinline__ void pv_step(f4v (&acc)[C::HR / 4][C::NDG], const float (&pa)[C::HR / 4],
                                        const u32x4 (&v)[C::KI * C::LPK]) {
#pragma unroll
    for (int e = 0; e < C::LPK; ++e)
#pragma unroll
        for (int c = 0; c < C::EL; ++c) {
            const float b = v_value<C::BF>(v[II * C::LPK + e], c);
#pragma unroll
            for (int hq = 0; hq < C::HR / 4; ++hq)
                acc[hq][e * C::EL + c] =
                    __builtin_amdgcn_mfma_f32_4x4x1f32(pa[hq], b, acc[hq][e * C::EL + c], C::CBSZ, II, 0);
        }
}

template <typename C, int... II>
__device__ __forceinline__ void pv_tile(f4v (&acc)[C::HR / 4][C::NDG], const float (&pa)[C::HR / 4],
                                        const u32x4 (&v)[C::KI * C::LPK], std::integer_sequence<int, II...>) {
    (pv_step<C, II>(acc, pa, v), ...);
}

// WIN: a window's rows, which stay in the caches until the next step; a whole context's K and V
// are read past them (16 ragged sequences 58.0 -> 55.3 us, eight of up to 131072 keys 163 -> 156;
// 64 windows 31.7 us, read past the caches 32.8).
template <int DH, typename KV, int NHQ, bool WIN>
__device__ __forceinline__ void paged_decode(const G4aPagedAttnParams& p) {
    using C = PagedCfg<DH, KV, NHQ>;
    constexpr bool BF = C::BF;
    constexpr int HR = C::HR, EL = C::EL, LG = C::LG, LPK = C::LPK, KI = C::KI, NDG = C::NDG, KC = C::KC, NM = C::NM,
                  QL = C::QL;
    __shared__ __attribute__((aligned(16))) char smem[C::SM];
    __shared__ __attribute__((aligned(16))) float p_s[4][NHQ * 64];
    __shared__ __attribute__((aligned(16))) float f_s[4][HR];
    __shared__ float m_s[4][HR], l_s[4][HR];
    u32x4* const qs = reinterpret_cast<u32x4*>(smem);
    f4v* const mrg = reinterpret_cast<f4v*>(smem);
    const G4aPaged& c = p.c;
    const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, key = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    // ---- this workgroup's part: every wave sums the lengths, a span of `each` sequences a lane ----
    const uint32_t n = c.n_seqs, each = (n + 63) / 64;
    const uint32_t my_len = lane < (int)n && each == 1 ? c.len[lane] : 0u;
    auto lane_tiles = [&](uint32_t b) { return b < n ? paged_span(p, each == 1 ? my_len : c.len[b]).n : 0u; };
    uint32_t mine = 0;
    for (uint32_t i = 0; i < each; ++i) mine += lane_tiles(lane * each + i);
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane(wave_incl_sum(mine), 63) * p.units;
    uint32_t quota = max((total + p.spread - 1) / p.spread, p.min_part), upto;
    if (quota < 2 * p.min_part) quota = (quota + p.min_part - 1) / p.min_part * p.min_part;  // (whole rounds of the waves)
    // parts of a sequence's units; the first few quotas may give more parts than `fit` holds, the last cannot
    auto parts_of = [&](uint32_t tiles) { return p.units * ((tiles + quota - 1) / quota); };
    for (int tries = 0;; ++tries) {
        mine = 0;
        for (uint32_t i = 0; i < each; ++i) mine += parts_of(lane_tiles(lane * each + i));
        upto = wave_incl_sum(mine);
        if (p.fit == 0 || (uint32_t)__builtin_amdgcn_readlane(upto, 63) <= p.fit) break;
        const uint32_t sure = (total + p.fit - n * p.units - 1) / (p.fit - n * p.units);
        quota = tries < 3 ? min(quota + (quota + 31) / 32, sure) : sure;
    }
    if (blockIdx.x == 0 && w == 0) {  // where each sequence's parts start, for the merge
        if (lane == 0) p.offs[0] = quota;
        uint32_t before = upto - mine;
        for (uint32_t i = 0; i < each; ++i) {
            const uint32_t b = lane * each + i;
            if (b < n) p.offs[1 + b] = before;
            before += parts_of(lane_tiles(b));
        }
    }
    const uint32_t at = blockIdx.x;
    if (at >= (uint32_t)__builtin_amdgcn_readlane(upto, 63)) return;
    // the sequence it is of, and that one's first part
    const int l0 = __builtin_ctzll(__ballot(upto > at));
    uint32_t b = l0 * each, base = __builtin_amdgcn_readlane(upto - mine, l0), len;
    if (each == 1) {
        len = __builtin_amdgcn_readlane(my_len, b);
    } else {
        for (const uint32_t last = min(b + each, n);; b += 64) {
            const uint32_t t = b + lane < last ? parts_of(lane_tiles(b + lane)) : 0u;
            const uint32_t u = wave_incl_sum(t);
            const uint64_t hit = __ballot(base + u > at);
            if (hit) {
                const int l1 = __builtin_ctzll(hit);
                base += __builtin_amdgcn_readlane(u - t, l1);
                b += l1;
                break;
            }
            base += __builtin_amdgcn_readlane(u, 63);
        }
        len = load_scalar(c.len, b);
    }
    const PagedSpan sp = paged_span(p, len);
    const uint32_t parts = (sp.n + quota - 1) / quota, j = (at - base) / parts, part = at - base - j * parts;
    const uint32_t floor = sp.n / parts, more = sp.n % parts;
    const uint32_t s = part * floor + min(part, more), e = s + floor + (part < more ? 1u : 0u);  // its tiles
    const uint32_t kvh = j / p.chunks, h0 = kvh * p.group + (j - kvh * p.chunks) * HR;
    const uint32_t nh = min((uint32_t)HR, p.group - (j - kvh * p.chunks) * HR);

    const uint32_t row_bytes = c.Hkv * DH * sizeof(KV);  // (at most 2 MiB)
    const uint32_t koff = key * row_bytes + 16 * g4, voff = (lane / LG) * KI * row_bytes + 16 * (lane % LG);

    auto page_of = [&](uint32_t t) {
        const uint32_t no = (sp.first + t) >> (c.page_shift - 4);
        return load_scalar(c.table, (size_t)b * c.per_seq + (c.ring ? no % c.per_seq : no));
    };
    auto tile_at = [&](uint32_t page, uint32_t t) {  // byte offset of a tile's first row in the pools
        const uint32_t r = ((sp.first + t) * 16) & ((1u << c.page_shift) - 1);
        return ((size_t)(page < c.n_pages ? page : 0u) * c.page_stride + ((size_t)r * c.Hkv + kvh) * DH) * sizeof(KV);
    };
    u32x4 k[KC], v[KI * LPK];
    const uint32_t tile_bytes = 16 * row_bytes;
    auto load_k = [&](size_t at) {
        load_pieces<!WIN, KC, KC, 64>(k, reinterpret_cast<const char*>(c.k) + uniform(at), tile_bytes, 0, koff);
    };
    auto load_v = [&](size_t at) {
        load_pieces<!WIN, KI * LPK, LPK, 1024>(v, reinterpret_cast<const char*>(c.v) + uniform(at), tile_bytes, row_bytes,
                                               voff);
    };
    // ---- the query rows into LDS, EL dims of a head a piece; their loads go out first ----
    f4v qr[QL][EL / 4];
#pragma unroll
    for (int i = 0; i < QL; ++i) {
        const int x = tid + 256 * i, h = x % HR, d = EL * (x / HR);
        const bool is = h < (int)nh && d < DH;
#pragma unroll
        for (int y = 0; y < EL / 4; ++y)
            qr[i][y] = is ? *reinterpret_cast<const f4v*>(p.q + ((size_t)b * p.Hq + h0 + h) * DH + d + 4 * y)
                          : f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // The first tile's; a wave without one reads the part's last again. No load of K or V stands under a
    // branch that one path leaves out: the compiler counts loads in flight over all paths to a use, and
    // waited for V, the younger, where it needed K (5 us of 17 in a call of 64 windows).
    uint32_t t = s + w;
    uint32_t page = page_of(min(t, e - 1)), page_next = t + 4 < e ? page_of(t + 4) : 0u;
    {
        const size_t off = tile_at(page, min(t, e - 1));
        load_k(off);
        load_v(off);
    }
#pragma unroll
    for (int i = 0; i < QL; ++i) {
        const int x = tid + 256 * i;  // = (K load * 4 + dim group) * HR + head
        if (QL * 256 > HR * DH / EL && x >= HR * DH / EL) break;
        if constexpr (BF) {
            float f[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) f[y] = qr[i][y / 4][y % 4];
#pragma unroll
            for (int z = 0; z < 3; ++z) {
                bf16x8 o;
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    o[y] = (__bf16)f[y];
                    f[y] -= (float)o[y];
                }
                qs[z * C::QPART + x] = __builtin_bit_cast(u32x4, o);
            }
        } else {
            qs[x] = __builtin_bit_cast(u32x4, qr[i][0]);
        }
    }
    // bf16: this lane's query block of the first K load in each MFMA: rows of 4 * NHQ heads, the parts in order
    // (NHQ 1: the fourth repeats the third, and is not summed; NHQ 2: so does the second MFMA's second half)
    int qi[NM];
#pragma unroll
    for (int y = 0; y < NM; ++y) {
        const int part = NHQ == 4 ? y : NHQ == 2 ? (y ? 2 : key / 8) : min(key / 4, 2);
        qi[y] = part * C::QPART + g4 * HR + key % HR;
    }

    barrier_lds();  // (K and V stay in flight across it)

    // lane (g4, key): heads 4 * (g4 % NHQ) + r of the tile's key
    float m[4], l[4];
    f4v acc[NHQ][NDG];
#pragma unroll
    for (int r = 0; r < 4; ++r) m[r] = G4A_NEG_INF, l[r] = 0.0f;
#pragma unroll
    for (int hq = 0; hq < NHQ; ++hq)
#pragma unroll
        for (int d = 0; d < NDG; ++d) acc[hq][d] = f4v{0.0f, 0.0f, 0.0f, 0.0f};

    // one tile; MORE: with the loads of the wave's next
    auto tile = [&](auto last) {
        constexpr bool MORE = !decltype(last)::value;
        const uint32_t page_after = MORE && t + 8 < e ? page_of(t + 8) : 0u;
        const size_t off = MORE ? tile_at(page_next, t + 4) : 0;
        // scores
        float x[4];
        if constexpr (BF) {
            f4v d[NM];
#pragma unroll
            for (int y = 0; y < NM; ++y) d[y] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KC; ++i)
#pragma unroll
                for (int y = 0; y < NM; ++y)
                    d[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, qs[qi[y] + i * 4 * HR]), __builtin_bit_cast(bf16x8, k[i]), d[y], 0, 0,
                        0);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (NHQ == 4) {
                    x[r] = (d[2][r] + d[1][r]) + d[0][r];
                } else if constexpr (NHQ == 2) {
                    const float2 y = g4a_pair32(d[0][r]);  // the first and second parts
                    x[r] = (d[1][r] + y.y) + y.x;
                } else {
                    const float2 y = g4a_pair16(d[0][r]);  // lanes 0 .. 31: first and second part, others: the third
                    const float2 z = g4a_pair32(y.x + (g4 < 2 ? y.y : 0.0f));
                    x[r] = z.x + z.y;
                }
            }
        } else {
            f4v d[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) d[y] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KC; ++i) {
                const u32x4 qa = qs[(i * 4 + g4) * HR + key % HR];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    d[y] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(qa[y]), __uint_as_float(k[i][y]), d[y],
                                                                0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = (d[0][r] + d[1][r]) + (d[2][r] + d[3][r]);
        }
        if constexpr (MORE) load_k(off);

        // running maximum and sum
        const uint32_t t0 = (sp.first + t) * 16;
        const bool hidden = page >= c.n_pages;
        const uint32_t lo = sp.lo > t0 ? sp.lo - t0 : 0u, hi = hidden ? 0u : min(16u, sp.len - t0);
        const bool seen = (uint32_t)key >= lo && (uint32_t)key < hi;
        float corr[4];
        bool moved = false;
        f4v pr;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float y = x[r] * p.scale;
            if (p.softcap > 0.0f) y = p.softcap * tanhf(y / p.softcap);
            y = seen ? y : G4A_NEG_INF;
            const float mn = fmaxf(m[r], g4a_row_max16(y));
            corr[r] = m[r] == G4A_NEG_INF ? 0.0f : expf(m[r] - mn);
            pr[r] = y == G4A_NEG_INF ? 0.0f : expf(y - mn);
            moved |= mn != m[r];
            l[r] = l[r] * corr[r] + pr[r];
            m[r] = mn;
        }
        // P to lane 4 * key + head, the A operand of 4x4x1
        if (g4 < NHQ) *reinterpret_cast<f4v*>(&p_s[w][4 * (16 * g4 + key)]) = pr;
        if (__ballot(moved)) {
#pragma unroll
            for (int hq = 0; hq < NHQ; ++hq)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f = g4a_lane(corr[r], 16 * hq);
#pragma unroll
                    for (int d = 0; d < NDG; ++d) acc[hq][d][r] *= f;
                }
        }
        __builtin_amdgcn_wave_barrier();
        float pa[NHQ];
#pragma unroll
        for (int hq = 0; hq < NHQ; ++hq) pa[hq] = p_s[w][64 * hq + lane];
        __builtin_amdgcn_wave_barrier();
        // what no token was written to may hold anything, and 0 times it is not 0
        if (lo > 0 || hi < 16) {
#pragma unroll
            for (int i = 0; i < KI; ++i) {
                const uint32_t row = i + KI * (lane / LG);
                const uint32_t keep = row >= lo && row < hi ? 0xFFFFFFFFu : 0u;
#pragma unroll
                for (int y = 0; y < LPK; ++y) v[i * LPK + y] &= keep;
            }
        }
        pv_tile<C>(acc, pa, v, std::make_integer_sequence<int, KI>());
        if constexpr (MORE) load_v(off);
        page = page_next;
        page_next = page_after;
    };
    for (; t + 4 < e; t += 4) tile(std::false_type());
    if (t < e) tile(std::true_type());

    // ---- the waves' partials, through LDS ----
#pragma unroll
    for (int r = 0; r < 4; ++r) l[r] = g4a_row_sum16(l[r]);
    if (key == 0 && g4 < NHQ)
#pragma unroll
        for (int r = 0; r < 4; ++r) m_s[w][4 * g4 + r] = m[r], l_s[w][4 * g4 + r] = l[r];
    barrier_lds();  // every wave is done with the query rows, where the accumulators go
#pragma unroll
    for (int hq = 0; hq < NHQ; ++hq)
#pragma unroll
        for (int d = 0; d < NDG; ++d) mrg[((w * NHQ + hq) * NDG + d) * 64 + lane] = acc[hq][d];
    const bool whole = parts == 1;
    if (tid < HR) {
        float M = G4A_NEG_INF, L = 0.0f, f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) M = fmaxf(M, m_s[i][tid]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = m_s[i][tid] == G4A_NEG_INF ? 0.0f : expf(m_s[i][tid] - M);
            L += l_s[i][tid] * f[i];
        }
        const float inv = whole ? (L != 0.0f ? 1.0f / L : 0.0f) : 1.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) f_s[i][tid] = f[i] * inv;
        if (!whole) {
            float* const ml = p.part_ml + (size_t)at * 2 * HR + tid;
            ml[0] = M;
            ml[HR] = L;
        }
    }
    barrier_lds();
    f4v* const dst = reinterpret_cast<f4v*>(p.part) + (size_t)at * C::ITEMS;
    for (int i = tid; i < C::ITEMS; i += 256) {
        const int hq = i / (NDG * LG), d = (i / LG) % NDG, lg = i % LG;
        f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const f4v f = *reinterpret_cast<const f4v*>(&f_s[y][4 * hq]);
            f4v a = mrg[((y * NHQ + hq) * NDG + d) * 64 + lg];
#pragma unroll
            for (int z = 1; z < C::NK; ++z) a += mrg[((y * NHQ + hq) * NDG + d) * 64 + z * LG + lg];
            o += a * f;
        }
        if (whole) {
            const int dim = (d / EL) * LG * EL + lg * EL + d % EL;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (4 * hq + r < (int)nh) p.out[((size_t)b * p.Hq + h0 + 4 * hq + r) * DH + dim] = o[r];
        } else {
            dst[i] = o;
        }
    }
}

// Merges the partials of units that more than one workgroup worked on, and writes the
// zeros of sequences without tokens. A block takes CI items (4 heads, one dim) of a
// unit, 256 / CI groups of threads every such part of it: CI 16 where there are few
// units of many parts, 64 where there are many units. A thread's first partial is
// loaded with the parts' maxima and sums, ahead of the weights e^(m - M), which are
// computed a part a thread and meet in LDS.
constexpr int PAGED_PARTS = 1024;  // of a unit, at most

template <int DH, typename KV, int NHQ, int CI>
__device__ __forceinline__ void paged_combine(const G4aPagedAttnParams& p) {
    using C = PagedCfg<DH, KV, NHQ>;
    constexpr int CG = 256 / CI;
    __shared__ f4v w_s[PAGED_PARTS];
    __shared__ f4v o_s[CG][CI];
    __shared__ f4v r_s[2][4];
    const uint32_t u = blockIdx.x / (C::ITEMS / CI), b = u / p.units, j = u - b * p.units;
    const uint32_t kvh = j / p.chunks, hc = j - kvh * p.chunks;
    const uint32_t h0 = kvh * p.group + hc * C::HR, nh = min((uint32_t)C::HR, p.group - hc * C::HR);
    const int tid = threadIdx.x, it = tid % CI, gr = tid / CI;
    const uint32_t item = blockIdx.x % (C::ITEMS / CI) * CI + it;
    // (the block's items are of one group of 4 heads)
    const int hq = item / (C::NDG * C::LG), d = (item / C::LG) % C::NDG, lg = item % C::LG;
    const int dim = (d / C::EL) * C::LG * C::EL + lg * C::EL + d % C::EL;
    static_assert(C::NDG * C::LG % CI == 0, "a block's items share their heads");
    const uint32_t quota = load_scalar(p.offs, 0), off = load_scalar(p.offs, 1 + b);
    const PagedSpan sp = paged_span(p, load_scalar(p.c.len, b));
    f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (sp.n) {
        const uint32_t parts = (sp.n + quota - 1) / quota, slot0 = off + j * parts;
        if (parts == 1) return;
        const f4v* const part = reinterpret_cast<const f4v*>(p.part) + (size_t)slot0 * C::ITEMS + item;
        const f4v* const ml = reinterpret_cast<const f4v*>(p.part_ml) + (size_t)slot0 * 2 * NHQ + hq;
        const f4v none = {G4A_NEG_INF, G4A_NEG_INF, G4A_NEG_INF, G4A_NEG_INF};
        const bool has = tid < (int)parts;
        const f4v m0 = has ? ml[(size_t)tid * 2 * NHQ] : none, l0 = has ? ml[(size_t)tid * 2 * NHQ + NHQ] : f4v{};
        const f4v o0 = gr < (int)parts ? part[(size_t)gr * C::ITEMS] : f4v{};
        f4v M = m0;
        for (uint32_t i = tid + 256; i < parts; i += 256)
#pragma unroll
            for (int r = 0; r < 4; ++r) M[r] = fmaxf(M[r], ml[(size_t)i * 2 * NHQ][r]);
        // (parts of the first waves only, but for more than 256)
        const int waves = parts >= 256 ? 4 : (int)(parts + 63) / 64, wave = tid / 64;
        if (wave < waves) {
#pragma unroll
            for (int r = 0; r < 4; ++r) M[r] = g4a_wave_max(M[r]);
            if (tid % 64 == 0) r_s[0][wave] = M;
        }
        if (waves > 1) {
            __syncthreads();
            M = r_s[0][0];
            for (int i = 1; i < waves; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) M[r] = fmaxf(M[r], r_s[0][i][r]);
        }
        f4v L = {0.0f, 0.0f, 0.0f, 0.0f};
        if (wave < waves) {
            for (uint32_t i = tid; i < parts; i += 256) {
                const f4v m = i < 256 ? m0 : ml[(size_t)i * 2 * NHQ], l = i < 256 ? l0 : ml[(size_t)i * 2 * NHQ + NHQ];
                f4v f;
#pragma unroll
                for (int r = 0; r < 4; ++r) f[r] = m[r] == G4A_NEG_INF ? 0.0f : expf(m[r] - M[r]);
                w_s[i] = f;
                L += l * f;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) L[r] = g4a_wave_sum(L[r]);
            if (tid % 64 == 0) r_s[1][wave] = L;
        }
        __syncthreads();
        if (gr < (int)parts) o = o0 * w_s[gr];
#pragma unroll 4
        for (uint32_t i = gr + CG; i < parts; i += CG) o += part[(size_t)i * C::ITEMS] * w_s[i];
        o_s[gr][it] = o;
        __syncthreads();
        if (gr) return;
        L = r_s[1][0];
        for (int i = 1; i < waves; ++i) L += r_s[1][i];
        for (int i = 1; i < min(CG, (int)parts); ++i) o += o_s[i][it];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = L[r] != 0.0f ? o[r] / L[r] : 0.0f;
    }
    if (gr) return;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (4 * hq + r < (int)nh) p.out[((size_t)b * p.Hq + h0 + 4 * hq + r) * DH + dim] = o[r];
}

}  // namespace

#define G4A_PAGED_DECODE(dh, type, kv, nhq, occ)                                                              \
    extern "C" __global__ __launch_bounds__(256, occ) void g4a_paged_decode_d##dh##_##type##_h##nhq(          \
        G4aPagedAttnParams p) { paged_decode<dh, kv, nhq, false>(p); }                                        \
    extern "C" __global__ __launch_bounds__(256, occ) void g4a_paged_decode_win_d##dh##_##type##_h##nhq(      \
        G4aPagedAttnParams p) { paged_decode<dh, kv, nhq, true>(p); }                                         \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_combine16_d##dh##_##type##_h##nhq(            \
        G4aPagedAttnParams p) { paged_combine<dh, kv, nhq, 16>(p); }                                          \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_combine64_d##dh##_##type##_h##nhq(            \
        G4aPagedAttnParams p) { paged_combine<dh, kv, nhq, 64>(p); }
#define G4A_PAGED_DECODE_TYPES(dh, nhq, occ_f32, occ_bf16) \
    G4A_PAGED_DECODE(dh, f32, float, nhq, occ_f32)         \
    G4A_PAGED_DECODE(dh, bf16, __bf16, nhq, occ_bf16)
// The second bound: workgroups of a CU, as the registers (and LDS) leave room for.
G4A_PAGED_DECODE_TYPES(64, 1, 4, 4) G4A_PAGED_DECODE_TYPES(64, 2, 3, 2) G4A_PAGED_DECODE_TYPES(64, 4, 2, 1)
G4A_PAGED_DECODE_TYPES(128, 1, 3, 4) G4A_PAGED_DECODE_TYPES(128, 2, 2, 2) G4A_PAGED_DECODE_TYPES(128, 4, 2, 1)
G4A_PAGED_DECODE_TYPES(256, 1, 2, 3) G4A_PAGED_DECODE_TYPES(256, 2, 2, 2) G4A_PAGED_DECODE_TYPES(256, 4, 1, 1)
G4A_PAGED_DECODE_TYPES(512, 1, 1, 2) G4A_PAGED_DECODE_TYPES(512, 2, 1, 1)
G4A_PAGED_DECODE(512, bf16, __bf16, 4, 1)  // (f32: two units of 8 heads, 16 have too many registers)
#undef G4A_PAGED_DECODE_TYPES
#undef G4A_PAGED_DECODE
