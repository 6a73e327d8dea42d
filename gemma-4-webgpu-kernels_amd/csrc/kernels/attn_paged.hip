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
// balanced better and were slower in an early form: 16 ragged sequences 52.0 against
// 48.3 us, 128 of 4 kv heads 68.2 against 55.8: several merges a workgroup, and 40 more
// registers.)
//
// A workgroup is 4 waves, each on every fourth tile of its part, with K and V of
// the next tile in flight in registers (16-byte loads; no LDS in between):
//   scores: K is the A operand of 16x16 MFMAs as it is loaded (lane = key l % 16 and a
//           quarter of the dims), the query rows B, out of LDS: f32 pages on
//           v_mfma_f32_16x16x4_f32, bf16 pages on v_mfma_f32_16x16x32_bf16 with the
//           query as three bf16 parts, whose sum it is exactly. A lane then has four
//           keys of one head;
//   softmax: running maximum and sum in f32, across the four lanes of a head;
//   P.V:    f32 pages on v_mfma_f32_4x4x1_16b_f32: V is B as it is loaded (a lane's dims
//           are columns of its block), P is A, through LDS, one key of it broadcast to all
//           blocks by the instruction. bf16 pages on v_mfma_f32_16x16x16_bf16: P is A as
//           the softmax left it, in three bf16 parts, and a lane's four keys of a dim
//           are B by two byte permutes of its loads. (4x4x1 takes 14 .. 16 cycles: 1.5
//           of the 2.6 us a tile of 512 dims took from bf16 pages on it were its.)
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

// DPP: lane i of a row of 16 reads lane (i - 4 or 8) % 16.
constexpr int ROW_ROR4 = 0x124, ROW_ROR8 = 0x128;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <int DH, typename KV, int NHQ>
struct PagedCfg {
    static constexpr bool BF = sizeof(KV) == 2;
    static constexpr int HR = 4 * NHQ;                       // query heads of a unit
    static constexpr int EL = 16 / (int)sizeof(KV);          // values of a 16-byte load
    static constexpr int KC = DH / (4 * EL);                 // K loads of a tile
    // f32 V: LG lanes of a row, LPK loads of a row and lane, NK rows of a load, KI * LPK loads of a tile
    static constexpr int LG = DH / EL < 64 ? DH / EL : 64;
    static constexpr int LPK = DH / (EL * LG);
    static constexpr int NK = 64 / LG;
    static constexpr int KI = 16 / NK;
    static constexpr int CBSZ = KI == 16 ? 4 : KI == 8 ? 3 : KI == 4 ? 2 : 1;  // log2 KI: blocks a key of P goes to
    // bf16 V: 16 lanes of EV dims of a row, four rows a lane, VB such blocks of dims
    static constexpr int EV = DH / 16 < 8 ? DH / 16 : 8;
    static constexpr int VB = DH / (16 * EV);
    static constexpr int VW = BF ? EV / 2 : 4;               // words of a V load
    static constexpr int VL = BF ? 4 * VB : KI * LPK;        // V loads of a tile
    static constexpr int NM = NHQ == 1 ? 1 : NHQ == 2 ? 2 : 3;  // bf16: MFMAs for the three parts of 4 NHQ heads
    // accumulators of a lane: f32 NHQ x EL LPK of 4 heads (a column a lane), bf16 VB EV of 16 rows
    static constexpr int NA = BF ? VB * EV : NHQ * EL * LPK;
    // 16-byte query blocks in LDS: [K load][dim group][head], bf16 for each of three parts (half the
    // banks apart, as the lanes of one read take two of them)
    static constexpr int QPART = KC * 4 * HR + 8;
    static constexpr int QS = BF ? 3 * QPART : KC * 4 * HR;
    static constexpr int QL = (HR * DH / EL + 255) / 256;    // 16-byte (bf16: 32-byte) query pieces of a thread
    static constexpr int ITEMS = NHQ * DH;                   // (4 heads, dim) of a partial
    static constexpr int ML = BF ? 16 * NHQ : 64;            // lanes that hand accumulators over
    // queries, those and the sequences' lengths never live at once
    static constexpr int SM = (QS > 4 * NA * ML ? QS : 4 * NA * ML) * 16;
    static_assert(SM >= 4096, "the lengths of PAGED_SEQS sequences");
    // Items in the accumulators' order: 4 heads hq, accumulator a, lane n of a row.
    static constexpr int IL = BF ? 16 : LG, IA = DH / IL;
    static __device__ __forceinline__ int hq(int item) { return item / DH; }
    static __device__ __forceinline__ int dim(int item) {
        const int n = item % IL, a = (item / IL) % IA;
        return BF ? (a / EV) * 16 * EV + n * EV + a % EV : (a / EL) * LG * EL + n * EL + a % EL;
    }
};

constexpr uint32_t PAGED_SEQS = 1024;  // of a launch, at most

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

// ceil(tiles / quota) parts of a unit, one of none (it writes zeros), by a reciprocal that is rounded down by 2^-20: exact below
// 2^19 tiles, never more. (An integer division each took 2 us of a call of 128 sequences. Every
// workgroup and the merge compute the same.)
__device__ __forceinline__ uint32_t paged_parts(uint32_t tiles, uint32_t quota) {
    const float inv = __builtin_amdgcn_rcpf((float)quota) * (1.0f - 0x1p-20f);
    return 1u + (uint32_t)fmaxf(((float)tiles - 0.5f) * inv, 0.0f);
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

// A tile of K or V: `bytes` from its first row on, behind which nothing is read. Buffer loads:
// a row is a scalar offset (as global loads each took a 64-bit vector sum, and registers for it).
struct PagedTile {
    __amdgpu_buffer_rsrc_t rsrc;
};

__device__ __forceinline__ PagedTile paged_tile(const void* pool, size_t at, uint32_t bytes) {
    const char* const tile = reinterpret_cast<const char*>(pool) + uniform(at);
    return {__builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(tile), 0, (int)bytes, 0x00020000)};
}

// One load of 16 (or 8) bytes at the scalar offset `row` and the lane's `off`. NT: past the caches.
template <bool NT, typename W>
__device__ __forceinline__ void load_piece(W& x, const PagedTile& t, uint32_t row, uint32_t off) {
    if constexpr (sizeof(W) == 16) x = __builtin_amdgcn_raw_buffer_load_b128(t.rsrc, (int)off, (int)row, NT ? 2 : 0);
    else x = __builtin_amdgcn_raw_buffer_load_b64(t.rsrc, (int)off, (int)row, NT ? 2 : 0);
}

// f32 pages: acc[hq][dims] += P[key II of each block group][4 heads] x V's values of that load.
template <typename C, int II>
__device__ __forceinline__ void pv_step(f4v (&acc)[C::NA], const float (&pa)[C::HR / 4], const u32x4 (&v)[C::VL]) {
    constexpr int ND = C::EL * C::LPK;
#pragma unroll
    for (int e = 0; e < C::LPK; ++e)
#pragma unroll
        for (int c = 0; c < C::EL; ++c)
#pragma unroll
            for (int hq = 0; hq < C::HR / 4; ++hq)
                acc[hq * ND + e * C::EL + c] = __builtin_amdgcn_mfma_f32_4x4x1f32(
                    pa[hq], __uint_as_float(v[II * C::LPK + e][c]), acc[hq * ND + e * C::EL + c], C::CBSZ, II, 0);
}

template <typename C, typename After, int... II>
__device__ __forceinline__ void pv_tile(f4v (&acc)[C::NA], const float (&pa)[C::HR / 4], const u32x4 (&v)[C::VL],
                                        const After& after, std::integer_sequence<int, II...>) {
    ((pv_step<C, II>(acc, pa, v), after(II)), ...);
}

typedef short bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 0x1.fffffep127f; }

// The heads of a unit whose query holds a NaN: their output is NaN in any arithmetic, so paged_part_f32 is not called
// for them (a sequence that pauses may have anything in its row of q; 8 sequences of up to 131072 keys of 512 dims with
// NaN in every query 138 us, with it 4.2 ms).
template <typename C, int DH>
__device__ __forceinline__ uint32_t nan_queries(const G4aPagedAttnParams& p, uint32_t b, uint32_t h0, uint32_t nh) {
    const int ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    uint32_t heads = 0;
#pragma unroll
    for (int q = 0; q < C::HR / 4; ++q) {
        const uint32_t h = h0 + min((uint32_t)(4 * q + ln / 16), nh - 1);
        const f4v* const y = reinterpret_cast<const f4v*>(p.q + ((size_t)b * p.Hq + h) * DH);
        bool is = false;
#pragma unroll
        for (int d = 0; d < DH / 64; ++d) {
            const f4v x = y[ln % 16 + 16 * d];
            is |= x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3];
        }
        const uint64_t lanes = __ballot(is);
#pragma unroll
        for (int g = 0; g < 4; ++g) heads |= (lanes >> (16 * g) & 0xFFFF ? 1u : 0u) << (4 * q + g);
    }
    return heads;
}

// A wave's items of a part of bf16 pages once more, in f32 arithmetic on K and V as they are, where the products of
// the three parts gave a value or a sum that is not finite: 0 times an infinity, or infinities of both signs, stand in
// them where a token's K or V is infinite or a query is beyond bf16's largest value, and f32 products have neither.
// Two passes over the part's tiles, the maxima and then the sums; s[q] is the score of head 4 q + lane / 16 and key
// lane % 16, the items are those of the part's end. Heads whose sums were finite keep their maxima and sums, by which
// the other waves' items go. Slow (8 sequences of up to 131072 keys of 512 dims: 131 us, with one infinity in V 2.7 ms,
// with one in every page 3.6), and no cost where all is finite: such calls take what they took without it.
template <typename C, int DH>
__device__ __forceinline__ void paged_part_f32(const G4aPagedAttnParams& p, const PagedSpan& sp, uint32_t b, uint32_t kvh,
                                               uint32_t h0, uint32_t nh, uint32_t from, uint32_t to, uint32_t at,
                                               bool whole, int w, const float (*m_s)[C::HR], const float (*l_s)[C::HR]) {
    constexpr int HR = C::HR, NQ = HR / 4, NI = (C::ITEMS + 255) / 256;
    const G4aPaged& c = p.c;
    // (the lane, and the divisor of page numbers, anew: nothing is kept for this over the tiles)
    const int ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), id = 64 * w + ln;
    const int g4 = ln >> 4, key = ln & 15;
    uint32_t per_seq = c.per_seq;
    asm volatile("" : "+s"(per_seq));
    const size_t width = (size_t)c.Hkv * DH;
    // each visible tile of the part: its first row in the pools, and its rows [lo, hi)
    auto tiles = [&](auto&& use) {
        for (uint32_t t = from; t < to; ++t) {
            const uint32_t t0 = (sp.first + t) * 16, no = t0 >> c.page_shift;
            const uint32_t page = load_scalar(c.table, (size_t)b * per_seq + (c.ring ? no % per_seq : no));
            if (page >= c.n_pages) continue;
            const uint32_t r = t0 & ((1u << c.page_shift) - 1);
            use((size_t)page * c.page_stride + ((size_t)r * c.Hkv + kvh) * DH, sp.lo > t0 ? sp.lo - t0 : 0u,
                min(16u, sp.len - t0));
        }
    };
    auto scores = [&](f4v& s, size_t row, uint32_t lo, uint32_t hi) {
        const u32x4* const k = reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(c.k) + row + key * width);
#pragma unroll
        for (int q = 0; q < NQ; ++q) s[q] = 0.0f;
#pragma unroll 1
        for (int d = 0; d < DH / 8; ++d) {
            const u32x4 x = k[d];
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const float* const y = p.q + ((size_t)b * p.Hq + h0 + min((uint32_t)(4 * q + g4), nh - 1)) * DH + 8 * d;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    s[q] += __uint_as_float(e & 1 ? x[e / 2] & 0xFFFF0000u : x[e / 2] << 16) * y[e];
            }
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            s[q] *= p.scale;
            if (p.softcap > 0.0f) s[q] = p.softcap * tanhf(s[q] / p.softcap);
            if ((uint32_t)key < lo || (uint32_t)key >= hi) s[q] = G4A_NEG_INF;
        }
    };
    // (vectors: a choice among an array's elements became an index into scratch memory)
    f4v m = {G4A_NEG_INF, G4A_NEG_INF, G4A_NEG_INF, G4A_NEG_INF}, l = {}, s, L_was = {};
    tiles([&](size_t row, uint32_t lo, uint32_t hi) {
        scores(s, row, lo, hi);
#pragma unroll
        for (int q = 0; q < NQ; ++q) m[q] = fmaxf(m[q], s[q]);
    });
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        float M = G4A_NEG_INF;
        for (int i = 0; i < 4; ++i) M = fmaxf(M, m_s[i][4 * q + g4]);
        for (int i = 0; i < 4; ++i)
            L_was[q] += l_s[i][4 * q + g4] * (m_s[i][4 * q + g4] == G4A_NEG_INF ? 0.0f : expf(m_s[i][4 * q + g4] - M));
        m[q] = finite(L_was[q]) ? M : g4a_row_max16(m[q]);
    }
    f4v o[NI];
#pragma unroll
    for (int x = 0; x < NI; ++x) o[x] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    tiles([&](size_t row, uint32_t lo, uint32_t hi) {
        scores(s, row, lo, hi);
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            s[q] = s[q] == G4A_NEG_INF ? 0.0f : expf(s[q] - m[q]);
            l[q] += s[q];
        }
#pragma unroll 1
        for (uint32_t j = lo; j < hi; ++j)
#pragma unroll
            for (int x = 0; x < NI; ++x) {
                const int i = id + 256 * x, hq = __builtin_amdgcn_readfirstlane(C::hq(i));  // (one for a wave's 64 items)
                if (C::ITEMS < 256 && i >= C::ITEMS) continue;
                const uint32_t v = reinterpret_cast<const uint16_t*>(c.v)[row + j * width + C::dim(i)];
                float pw = s[0];
#pragma unroll
                for (int q = 1; q < NQ; ++q)
                    if (hq == q) pw = s[q];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[x][r] += __shfl(pw, 16 * r + (int)j) * __uint_as_float(v << 16);
            }
    });
#pragma unroll
    for (int q = 0; q < NQ; ++q) l[q] = finite(L_was[q]) ? L_was[q] : g4a_row_sum16(l[q]);
    if (!whole && w == 0) {  // (the lanes that wrote these before)
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const float M = __shfl(m[q], 16 * (ln & 3)), L = __shfl(l[q], 16 * (ln & 3));
            if (ln / 4 == q) {
                float* const ml = p.part_ml + (size_t)at * 2 * HR + ln;
                ml[0] = M;
                ml[HR] = L;
            }
        }
    }
#pragma unroll
    for (int x = 0; x < NI; ++x) {
        const int i = id + 256 * x, hq = __builtin_amdgcn_readfirstlane(C::hq(i));
        if (C::ITEMS < 256 && i >= C::ITEMS) continue;
        if (!whole) {
            (reinterpret_cast<f4v*>(p.part) + (size_t)at * C::ITEMS)[i] = o[x];
            continue;
        }
        float L = l[0];
#pragma unroll
        for (int q = 1; q < NQ; ++q)
            if (hq == q) L = l[q];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float sum = g4a_lane(L, 16 * r);
            if (4 * hq + r < (int)nh)
                p.out[((size_t)b * p.Hq + h0 + 4 * hq + r) * DH + C::dim(i)] = o[x][r] * (sum != 0.0f ? 1.0f / sum : 0.0f);
        }
    }
}

// WIN: a window's rows, which stay in the caches until the next step; a whole context's K and V
// are read past them (the other way about: 16 ragged sequences 42.2 us for 40.4, eight of up to 131072 keys 142 for
// 131, 128 of 4 kv heads 45.3 for 41.8, 64 windows 18.3 for 17.0, in f32 pages 23.0 for 21.1; only one sequence of
// 32768 keys, read again and again, gains: 31.6 for 32.5).
template <int DH, typename KV, int NHQ, bool WIN>
__device__ __forceinline__ void paged_decode(const G4aPagedAttnParams& p) {
    using C = PagedCfg<DH, KV, NHQ>;
    constexpr bool BF = C::BF;
    constexpr int HR = C::HR, EL = C::EL, KC = C::KC, NM = C::NM, NA = C::NA, QL = C::QL;
    using VWord = uint32_t __attribute__((ext_vector_type(C::VW)));
    __shared__ __attribute__((aligned(16))) char smem[C::SM];
    __shared__ __attribute__((aligned(16))) float p_s[4][BF ? 4 : NHQ * 64];
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
    // (more than one a lane: through LDS, by every wave alike. Short loops: sixteen lengths a lane in registers,
    // unrolled, took 1.6 us more of a small call, in code that no cache holds yet.)
    uint32_t* const lens = reinterpret_cast<uint32_t*>(smem);
    if (each > 1)
        for (uint32_t b = lane; b < n; b += 64) lens[b] = c.len[b];
    auto lane_tiles = [&](uint32_t b) { return b < n ? paged_span(p, each == 1 ? my_len : lens[b]).n : 0u; };
    uint32_t mine = 0;
    for (uint32_t i = 0; i < each; ++i) mine += lane_tiles(lane * each + i);
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane(wave_incl_sum(mine), 63) * p.units;
    // (not in whole rounds of the waves: 64 windows of 512, hd 256 f32, took 23.4 us so, 21.1 with parts of five tiles)
    uint32_t quota = max((total + p.spread - 1) / p.spread, p.min_part), upto;
    // parts of a sequence's units; the first few quotas may give more parts than `fit` holds, the last cannot
    auto lane_parts = [&](uint32_t b) { return b < n ? p.units * paged_parts(lane_tiles(b), quota) : 0u; };
    for (int tries = 0;; ++tries) {
        mine = 0;
        for (uint32_t i = 0; i < each; ++i) mine += lane_parts(lane * each + i);
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
            before += lane_parts(b);
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
        static_assert(PAGED_SEQS <= 64 * 64, "a lane's span of sequences, a lane each");
        const uint32_t mine_of = lane < (int)min(each, n - b) ? lane_parts(b + lane) : 0u;
        const uint32_t incl = wave_incl_sum(mine_of);
        const int l1 = __builtin_ctzll(__ballot(base + incl > at));
        base += __builtin_amdgcn_readlane(incl - mine_of, l1);
        b += l1;
        len = __builtin_amdgcn_readfirstlane(lens[b]);
        barrier_lds();  // every wave has read the lengths: the query rows go there
    }
    const PagedSpan sp = paged_span(p, len);
    const uint32_t parts = __builtin_amdgcn_readfirstlane(paged_parts(sp.n, quota));
    const uint32_t j = (at - base) / parts, part = at - base - j * parts;
    const uint32_t floor = sp.n / parts, more = sp.n % parts;
    const uint32_t s = part * floor + min(part, more), e = s + floor + (part < more ? 1u : 0u);  // its tiles
    const uint32_t kvh = j / p.chunks, h0 = kvh * p.group + (j - kvh * p.chunks) * HR;
    const uint32_t nh = min((uint32_t)HR, p.group - (j - kvh * p.chunks) * HR);
    if (sp.n == 0) {
        for (uint32_t i = tid; i < nh * DH; i += 256) p.out[((size_t)b * p.Hq + h0) * DH + i] = 0.0f;
        return;
    }

    const uint32_t row_bytes = c.Hkv * DH * sizeof(KV);  // (at most 2 MiB)
    // K: lane (g4, key) its key's dims; V: f32 lane LG r + n row KI r, bf16 lane (g4, n) row 4 g4
    const uint32_t koff = key * row_bytes + 16 * g4;
    const uint32_t voff = BF ? 4 * g4 * row_bytes + 4 * C::VW * key
                             : (lane / C::LG) * C::KI * row_bytes + 16 * (lane % C::LG);

    auto page_of = [&](uint32_t t) {
        const uint32_t no = (sp.first + t) >> (c.page_shift - 4);
        return load_scalar(c.table, (size_t)b * c.per_seq + (c.ring ? no % c.per_seq : no));
    };
    auto tile_at = [&](uint32_t page, uint32_t t) {  // byte offset of a tile's first row in the pools
        const uint32_t r = ((sp.first + t) * 16) & ((1u << c.page_shift) - 1);
        return ((size_t)(page < c.n_pages ? page : 0u) * c.page_stride + ((size_t)r * c.Hkv + kvh) * DH) * sizeof(KV);
    };
    // 512 dims: K and V take turns in one set of registers, V's pieces loaded where K's have been used and
    // K's next where V's have. With 16 heads there is no room for both; with up to 8 a second workgroup of a
    // CU starts while the first ends (256 ragged sequences of up to 1500 tokens in bf16 pages: 68.7 us, and
    // 78.3 with both in flight; one of 32768 in f32 pages 32.4 and 34.6; eight of up to 131072 in bf16 pages
    // 131.2 and 130.4, which runs differ by as well).
    constexpr bool TURNS = DH == 512;
    VWord v[C::VL];  // bf16: [row][block of dims]
    u32x4 k_own[TURNS ? 1 : KC];
    u32x4 (&k)[KC] = [&]() -> u32x4 (&)[KC] {
        if constexpr (TURNS) return v;
        else return k_own;
    }();
    static_assert(C::VL % KC == 0 && (!TURNS || KC == C::VL), "pieces of V for each of K");
    const uint32_t tile_bytes = 16 * row_bytes;
    auto load_k = [&](const PagedTile& t, int i) { load_piece<!WIN>(k[i], t, 0, koff + 64 * i); };
    auto load_v = [&](const PagedTile& t, int i) {  // bf16: row i / VB, block i % VB; f32: rows i / LPK
        constexpr int PER = BF ? C::VB : C::LPK;
        load_piece<!WIN>(v[i], t, i / PER * row_bytes, voff + i % PER * (BF ? 256 : 1024));
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
        const PagedTile kt = paged_tile(c.k, off, tile_bytes);
#pragma unroll
        for (int i = 0; i < KC; ++i) load_k(kt, i);
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
    // bf16: this lane's query block of the first K load in each MFMA: columns of 4 * NHQ heads, the parts in order
    // (NHQ 1: the fourth repeats the third, and is not summed; NHQ 2: so does the second MFMA's second half)
    int qi[NM];
#pragma unroll
    for (int y = 0; y < NM; ++y) {
        const int part = NHQ == 4 ? y : NHQ == 2 ? (y ? 2 : key / 8) : min(key / 4, 2);
        qi[y] = part * C::QPART + g4 * HR + key % HR;
    }

    barrier_lds();  // (K and V stay in flight across it)

    // lane (g4, n): keys 4 g4 + r of the tile, head n % HR of the unit (all of n's repeats alike)
    float m = G4A_NEG_INF, l = 0.0f;
    f4v acc[NA];
#pragma unroll
    for (int d = 0; d < NA; ++d) acc[d] = f4v{0.0f, 0.0f, 0.0f, 0.0f};

    // The lane, and what follows from it, once more where it is used: kept over the loop those were a few
    // registers too many, in scratch memory.
    auto lane_again = [&] {
        int x = lane;
        if constexpr (TURNS && NHQ < 4) asm volatile("" : "+v"(x));
        return x;
    };
    // One tile; MORE: a piece of the wave's next is loaded where this one's has been used; FIRST: V is
    // loaded between the scores' MFMAs, as ahead of them its loads held up the first of them. (The empty
    // scheduling barriers keep the reads of all query rows, and V's permutes, from being gathered ahead of
    // the first MFMA, in more registers than there are.)
    auto tile = [&](auto first, auto more) {
        constexpr bool FIRST = decltype(first)::value || TURNS, MORE = decltype(more)::value;
        const int ln = lane_again(), g4 = ln >> 4, key = ln & 15;
        const uint32_t page_after = MORE && t + 8 < e ? page_of(t + 8) : 0u;
        const size_t next = MORE ? tile_at(page_next, t + 4) : 0;
        const PagedTile kt = paged_tile(c.k, next, tile_bytes);
        const PagedTile vt = paged_tile(c.v, next, tile_bytes), vt0 = paged_tile(c.v, FIRST ? tile_at(page, t) : 0, tile_bytes);
        auto after_k = [&](int i) {
            if constexpr (FIRST)
#pragma unroll
                for (int x = i * C::VL / KC; x < (i + 1) * C::VL / KC; ++x) load_v(vt0, x);
            if constexpr (!TURNS && MORE) load_k(kt, i);
        };
        auto after_v = [&](int i) {
            if constexpr (!MORE) return;
            else if constexpr (TURNS) load_k(kt, i);
            else load_v(vt, i);
        };
        // scores
        float x[4];
        if constexpr (BF) {
            f4v d[NM];
#pragma unroll
            for (int y = 0; y < NM; ++y) d[y] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KC; ++i) {
#pragma unroll
                for (int y = 0; y < NM; ++y)
                    d[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, k[i]), __builtin_bit_cast(bf16x8, qs[qi[y] + i * 4 * HR]), d[y], 0, 0,
                        0);
                after_k(i);
                if (i % 8 == 7) __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {  // the parts of a head are in columns HR apart
                if constexpr (NHQ == 4) {
                    x[r] = (d[2][r] + d[1][r]) + d[0][r];
                } else if constexpr (NHQ == 2) {
                    x[r] = d[1][r] + (d[0][r] + g4a_dpp<ROW_ROR8>(d[0][r]));
                } else {
                    const float y = key < 12 ? d[0][r] : 0.0f, z = y + g4a_dpp<ROW_ROR8>(y);
                    x[r] = z + g4a_dpp<ROW_ROR4>(z);
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
                    d[y] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[i][y]), __uint_as_float(qa[y]), d[y], 0, 0,
                                                                0);
                after_k(i);
                if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = (d[0][r] + d[1][r]) + (d[2][r] + d[3][r]);
        }

        // running maximum and sum
        const uint32_t t0 = (sp.first + t) * 16;
        const bool hidden = page >= c.n_pages;
        const uint32_t lo = sp.lo > t0 ? sp.lo - t0 : 0u, hi = hidden ? 0u : min(16u, sp.len - t0);
        f4v pr;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float y = x[r] * p.scale;
            if (p.softcap > 0.0f) y = p.softcap * tanhf(y / p.softcap);
            const uint32_t row = 4 * g4 + r;
            pr[r] = row >= lo && row < hi ? y : G4A_NEG_INF;
        }
        const float mn = fmaxf(m, g4a_col_max4(fmaxf(fmaxf(pr[0], pr[1]), fmaxf(pr[2], pr[3]))));
        const float corr = m == G4A_NEG_INF ? 0.0f : expf(m - mn);
        const bool moved = mn != m;
        m = mn;
#pragma unroll
        for (int r = 0; r < 4; ++r) pr[r] = pr[r] == G4A_NEG_INF ? 0.0f : expf(pr[r] - mn);
        l = l * corr + ((pr[0] + pr[1]) + (pr[2] + pr[3]));
        if (__ballot(moved)) {
#pragma unroll
            for (int hq = 0; hq < (BF ? 1 : NHQ); ++hq)
#pragma unroll
                for (int r = 0; r < 4; ++r) {  // the lanes of a head hold its factor
                    const float f = BF && NHQ > 1 ? __shfl(corr, 4 * (g4 % NHQ) + r) : g4a_lane(corr, 4 * hq + r);
#pragma unroll
                    for (int d = 0; d < (BF ? NA : NA / NHQ); ++d) acc[hq * (NA / NHQ) + d][r] *= f;
                }
        }
        // what no token was written to may hold anything, and 0 times it is not 0
        if (lo > 0 || hi < 16) {
#pragma unroll
            for (int i = 0; i < C::VL; ++i) {
                const uint32_t row = BF ? 4 * g4 + i / C::VB : i / C::LPK + C::KI * (ln / C::LG);
                v[i] &= row >= lo && row < hi ? 0xFFFFFFFFu : 0u;
            }
        }
        if constexpr (BF) {
            // P's rows as the query's columns: part by part, a head's parts HR rows apart
            bf4 pa[NM];
            bf16x4v part[3];
            f4v rest = pr;
#pragma unroll
            for (int y = 0; y < 3; ++y) {
                part[y] = __builtin_convertvector(rest, bf16x4v);
                rest -= __builtin_convertvector(part[y], f4v);
            }
            const bf4 zero = {0, 0, 0, 0};
            if constexpr (NHQ == 4) {
#pragma unroll
                for (int y = 0; y < 3; ++y) pa[y] = __builtin_bit_cast(bf4, part[y]);
            } else if constexpr (NHQ == 2) {
                pa[0] = key < 8 ? __builtin_bit_cast(bf4, part[0]) : __builtin_bit_cast(bf4, part[1]);
                pa[1] = key < 8 ? __builtin_bit_cast(bf4, part[2]) : zero;
            } else {
                pa[0] = key < 4    ? __builtin_bit_cast(bf4, part[0])
                        : key < 8  ? __builtin_bit_cast(bf4, part[1])
                        : key < 12 ? __builtin_bit_cast(bf4, part[2])
                                   : zero;
            }
#pragma unroll
            for (int y = 0; y < C::VB; ++y) {
#pragma unroll
                for (int e = 0; e < C::EV; ++e) {
                    const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;  // rows i, i + 1 of a dim into a word
                    const uint32_t b0 = __builtin_amdgcn_perm(v[C::VB + y][e / 2], v[y][e / 2], sel);
                    const uint32_t b1 = __builtin_amdgcn_perm(v[3 * C::VB + y][e / 2], v[2 * C::VB + y][e / 2], sel);
                    const bf4 b = __builtin_bit_cast(bf4, (uint64_t)b1 << 32 | b0);
#pragma unroll
                    for (int z = 0; z < NM; ++z)
                        acc[y * C::EV + e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(pa[z], b, acc[y * C::EV + e], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) after_v(i * C::VB + y);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // P to lane 4 * key + head, the A operand of 4x4x1
            if (key < HR) *reinterpret_cast<f4v*>(&p_s[w][16 * key + 4 * g4]) = pr;
            __builtin_amdgcn_wave_barrier();
            float pa[NHQ];
#pragma unroll
            for (int hq = 0; hq < NHQ; ++hq) pa[hq] = p_s[w][16 * (4 * hq + (ln & 3)) + (ln >> 2)];
            __builtin_amdgcn_wave_barrier();
            auto reload = [&](int ii) {
#pragma unroll
                for (int x = 0; x < C::LPK; ++x) after_v(ii * C::LPK + x);
            };
            pv_tile<C>(acc, pa, v, reload, std::make_integer_sequence<int, C::KI>());
        }
        page = page_next;
        page_next = page_after;
    };
    const std::true_type yes;
    const std::false_type no;
    if constexpr (TURNS) {
        for (; t + 4 < e; t += 4) tile(yes, yes);
        if (t < e) tile(yes, no);
    } else if (t + 4 < e) {
        tile(yes, yes);
        for (t += 4; t + 4 < e; t += 4) tile(no, yes);
        tile(no, no);
    } else if (t < e) {
        tile(yes, no);
    }

    // ---- the waves' partials, through LDS ----
    const int ln = lane_again(), id = 64 * w + ln;
    l = g4a_col_sum4(l);
    if (ln < HR) m_s[w][ln] = m, l_s[w][ln] = l;
    barrier_lds();  // every wave is done with the query rows, where the accumulators go
#pragma unroll
    for (int d = 0; d < NA; ++d) {
        if constexpr (BF && NHQ < 4) {  // the rows of a head's parts, in lanes 16 NHQ apart
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float2 y = g4a_pair32(acc[d][r]);
                acc[d][r] = y.x + y.y;
                if constexpr (NHQ == 1) {
                    y = g4a_pair16(acc[d][r]);
                    acc[d][r] = y.x + y.y;
                }
            }
        }
        if (C::ML == 64 || ln < C::ML) mrg[(w * NA + d) * C::ML + ln] = acc[d];
    }
    const bool whole = parts == 1;
    bool sum_bad = false;
    if (id < HR) {
        float M = G4A_NEG_INF, L = 0.0f, f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) M = fmaxf(M, m_s[i][id]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = m_s[i][id] == G4A_NEG_INF ? 0.0f : expf(m_s[i][id] - M);
            L += l_s[i][id] * f[i];
        }
        sum_bad = !finite(L);
        const float inv = whole ? (L != 0.0f ? 1.0f / L : 0.0f) : 1.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) f_s[i][id] = f[i] * inv;
        if (!whole) {
            float* const ml = p.part_ml + (size_t)at * 2 * HR + id;
            ml[0] = M;
            ml[HR] = L;
        }
    }
    uint32_t bad = BF ? (uint32_t)__ballot(sum_bad) : 0u;  // heads with a sum or a value that is not finite
    barrier_lds();
    f4v* const dst = reinterpret_cast<f4v*>(p.part) + (size_t)at * C::ITEMS;
    for (int i = id; i < C::ITEMS; i += 256) {
        const int hq = C::hq(i), n = i % C::IL, a = (i / C::IL) % C::IA;
        f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const f4v f = *reinterpret_cast<const f4v*>(&f_s[y][4 * hq]);
            if constexpr (BF) {
                o += mrg[(y * NA + a) * C::ML + 16 * hq + n] * f;
            } else {
                f4v x = mrg[(y * NA + hq * C::IA + a) * 64 + n];
#pragma unroll
                for (int z = 1; z < C::NK; ++z) x += mrg[(y * NA + hq * C::IA + a) * 64 + z * C::LG + n];
                o += x * f;
            }
        }
        if constexpr (BF)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                bad |= (__ballot(!finite(o[r])) ? 1u : 0u) << (4 * __builtin_amdgcn_readfirstlane(hq) + r);
        if (whole) {
            const int dim = C::dim(i);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (4 * hq + r < (int)nh) p.out[((size_t)b * p.Hq + h0 + 4 * hq + r) * DH + dim] = o[r];
        } else {
            dst[i] = o;
        }
    }
    if constexpr (BF) {
        bad &= (1u << nh) - 1;
        if (bad && (bad & ~nan_queries<C, DH>(p, b, h0, nh)))
            paged_part_f32<C, DH>(p, sp, b, kvh, h0, nh, s, e, at, whole, w, m_s, l_s);
    }
}

// Merges the partials of units that more than one workgroup worked on. A block of W waves takes CI items (4 heads, one
// dim) of a unit, 64 W / CI groups of threads every such part of it: 16 items and 8
// waves where there are few units of many parts (one unit of 256 parts of 512 dims: with
// 64 items and 4 waves a call takes 37.2 us, 32.2 so), 64 items and 4 waves where there are many units (64 of
// up to 4000 tokens 72.1 us, 79.0 with 16). A thread's first partial is loaded with the parts' maxima
// and sums, ahead of the weights e^(m - M), which are computed a part a thread and meet
// in LDS.
constexpr int PAGED_PARTS = 1024;  // of a unit, at most

template <int DH, typename KV, int NHQ, int CI, int W>
__device__ __forceinline__ void paged_combine(const G4aPagedAttnParams& p) {
    using C = PagedCfg<DH, KV, NHQ>;
    constexpr int NT = 64 * W, CG = NT / CI;
    static_assert(CI == 16 || CI == 64, "a wave's groups meet by columns of 16 lanes");
    __shared__ f4v w_s[PAGED_PARTS];
    __shared__ f4v o_s[W][CI];
    __shared__ f4v r_s[2][W];
    const uint32_t u = blockIdx.x / (C::ITEMS / CI), b = u / p.units, j = u - b * p.units;
    const uint32_t kvh = j / p.chunks, hc = j - kvh * p.chunks;
    const uint32_t h0 = kvh * p.group + hc * C::HR, nh = min((uint32_t)C::HR, p.group - hc * C::HR);
    const int tid = threadIdx.x, it = tid % CI, gr = tid / CI;
    const uint32_t item = blockIdx.x % (C::ITEMS / CI) * CI + it;
    // (the block's items are of one group of 4 heads)
    const int hq = C::hq(item), dim = C::dim(item);
    static_assert(DH % CI == 0, "a block's items share their heads");
    const uint32_t quota = load_scalar(p.offs, 0), off = load_scalar(p.offs, 1 + b);
    const PagedSpan sp = paged_span(p, load_scalar(p.c.len, b));
    const uint32_t parts = __builtin_amdgcn_readfirstlane(paged_parts(sp.n, quota)), slot0 = off + j * parts;
    if (parts == 1) return;
    const f4v* const part = reinterpret_cast<const f4v*>(p.part) + (size_t)slot0 * C::ITEMS + item;
    const f4v* const ml = reinterpret_cast<const f4v*>(p.part_ml) + (size_t)slot0 * 2 * NHQ + hq;
    const f4v none = {G4A_NEG_INF, G4A_NEG_INF, G4A_NEG_INF, G4A_NEG_INF};
    const bool has = tid < (int)parts;
    const f4v m0 = has ? ml[(size_t)tid * 2 * NHQ] : none, l0 = has ? ml[(size_t)tid * 2 * NHQ + NHQ] : f4v{};
    const f4v o0 = gr < (int)parts ? part[(size_t)gr * C::ITEMS] : f4v{};
    f4v M = m0;
    for (uint32_t i = tid + NT; i < parts; i += NT)
#pragma unroll
        for (int r = 0; r < 4; ++r) M[r] = fmaxf(M[r], ml[(size_t)i * 2 * NHQ][r]);
    // (parts of the first waves only, but for more than NT)
    const int waves = parts >= NT ? W : (int)(parts + 63) / 64, wave = tid / 64;
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
        for (uint32_t i = tid; i < parts; i += NT) {
            const f4v m = i < NT ? m0 : ml[(size_t)i * 2 * NHQ], l = i < NT ? l0 : ml[(size_t)i * 2 * NHQ + NHQ];
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
    f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (gr < (int)parts) o = o0 * w_s[gr];
#pragma unroll 4
    for (uint32_t i = gr + CG; i < parts; i += CG) o += part[(size_t)i * C::ITEMS] * w_s[i];
    if constexpr (CI == 16)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = g4a_col_sum4(o[r]);
    if (tid % 64 < CI) o_s[wave][it] = o;
    __syncthreads();
    if (gr) return;
    L = r_s[1][0];
    for (int i = 1; i < waves; ++i) L += r_s[1][i];
#pragma unroll
    for (int i = 1; i < W; ++i) o += o_s[i][it];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = L[r] != 0.0f ? o[r] / L[r] : 0.0f;
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
    extern "C" __global__ __launch_bounds__(512) void g4a_paged_combine16_d##dh##_##type##_h##nhq(            \
        G4aPagedAttnParams p) { paged_combine<dh, kv, nhq, 16, 8>(p); }                                      \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_combine64_d##dh##_##type##_h##nhq(            \
        G4aPagedAttnParams p) { paged_combine<dh, kv, nhq, 64, 4>(p); }
#define G4A_PAGED_DECODE_TYPES(dh, nhq, occ_f32, occ_bf16) \
    G4A_PAGED_DECODE(dh, f32, float, nhq, occ_f32)         \
    G4A_PAGED_DECODE(dh, bf16, __bf16, nhq, occ_bf16)
// The second bound: workgroups of a CU, as the registers (and LDS) leave room for.
G4A_PAGED_DECODE_TYPES(64, 1, 4, 4) G4A_PAGED_DECODE_TYPES(64, 2, 4, 4) G4A_PAGED_DECODE_TYPES(64, 4, 2, 4)
G4A_PAGED_DECODE_TYPES(128, 1, 3, 4) G4A_PAGED_DECODE_TYPES(128, 2, 3, 4) G4A_PAGED_DECODE_TYPES(128, 4, 2, 3)
G4A_PAGED_DECODE_TYPES(256, 1, 2, 3) G4A_PAGED_DECODE_TYPES(256, 2, 2, 3) G4A_PAGED_DECODE_TYPES(256, 4, 1, 2)
G4A_PAGED_DECODE_TYPES(512, 1, 2, 2) G4A_PAGED_DECODE_TYPES(512, 2, 2, 2) G4A_PAGED_DECODE_TYPES(512, 4, 1, 1)
#undef G4A_PAGED_DECODE_TYPES
#undef G4A_PAGED_DECODE
