// Decode attention over pages of 8 and 4 bits for gfx950: one query of every sequence over its visible tokens,
//   out[b, h] = sum_t softmax_t(cap(scale * q[b, h] . K[t])) V[t],  K[t] = S_t sub n (8 bits: S_t n), V alike,
// as attn_paged.hip, whose division of the work into parts and merge of their partials these kernels share. Formats:
// paged_quant.h; layout: G4aPaged. The reference has no quantised cache.
//
// No value is ever multiplied out. sub n has 10 bits, so it is an fp16 operand exactly, made by one fma for two of them
// (below); S_t, one number a token, goes to the score and to the probability:
//   scores: K is the A operand of v_mfma_f32_16x16x32_f16 (lane = key l % 16 and a quarter of the dims, as it is loaded, no
//           LDS in between), the query B, out of LDS, as two fp16 parts whose sum it is to 2^-22: 8 heads fill its 16
//           columns. A lane then has four keys of one head; s = (x S) scale;
//   softmax: in powers of two, relative to a maximum that follows the tiles' only when they pass it by LAZY, sum in f32;
//   P.V:    P S_t 2^k is the A operand of v_mfma_f32_16x16x16_f16 as the softmax left it, in two fp16 parts in the rows of 8
//           heads each, V is B: a lane holds four tokens' bytes of the same dims, and a byte permute pairs two
//           tokens in a register. k follows the largest S_t, so that P S_t stays in fp16's range.
// Against 64 bits the results are about as near as the same in f32 operations, or nearer (relative 5e-7 to 2e-6, those 6e-7
// to 7e-6).
//
// A workgroup is 4 waves (8 at 512 dims, unless there are units for every CU), each on every 4th (8th) tile of its part
// with the next tile's K and V in flight in registers, reloaded where they have been used. At 512 dims a wave holds 128
// accumulators, so two waves a SIMD; eight waves that share their queries and one merge in LDS, and not two workgroups
// of four: twice as many parts to start and merge (one sequence of 32768 tokens, 4 bits 17.6 us, 23.6 so; 16 ragged of up to 8192, 8 bits
// 20.7 and 27.1). Where there are units for every CU the parts are there anyway, and two workgroups of four
// overlap their starts and ends (256 sequences of up to 1500 tokens, 4 bits 35.3 us, 43.0 with eight waves).
//
// What bounds it: a tile of 512 dims and 8 heads in 4 bits takes about 450 vector instructions (some 150 each to unpack
// K and V), 48 MFMAs and 8.8 KiB, and 590 instructions with its share of a wave's start and end. Over eight sequences of
// up to 131072 tokens (211 MB, 49 us with the merge, 4.3 TB/s) these are 2430 cycles of a SIMD a tile, two thirds of the
// 3620 for which its waves live and half of the 4740 of the kernel: a quarter of it passes before a wave's start or after
// its end, in the mean. Calls of few tiles a wave are bound by
// the chain of a workgroup's start (lengths, table, queries: 5000 cycles; to the end of the first tile 10000), its end (6000) and
// the merge launch (5 us).
// A merge by the last of a unit's workgroups to end (tickets, partials past the XCD's cache) was slower:
// 16 ragged sequences 26.5 us for 21, one window of 512 tokens 10.0 for 10.0.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "g4a_math.h"
#include "g4a_params.h"
#include "paged_quant.h"

namespace {

template <int DH, int BITS, int NHQ, bool MANY = false>
struct QuantCfg {
    static constexpr int DIMS = DH;
    static __device__ __forceinline__ float exp(float x) { return __builtin_amdgcn_exp2f(x); }  // of the partials' maxima
    static constexpr int HR = 4 * NHQ;                                // query heads of a unit
    static constexpr int EV = DH / 16 < 32 / (BITS / 4) ? DH / 16 : 32 / (BITS / 4);  // dims of a lane and block
    static constexpr int NA = DH / 16;                                // accumulators of a lane, of 16 rows
    static constexpr int ITEMS = NHQ * DH;                            // (4 heads, dim) of a partial
    static constexpr int ML = 16 * NHQ;                               // lanes with a row of heads each, per accumulator
    static constexpr int W = g4a_paged_waves(DH, NHQ, MANY);          // waves
    // the queries (two fp16 parts), the waves' accumulators and the sequences' lengths never live at once
    static constexpr int SM0 = 4 * HR * DH > W * NA * ML * 16 ? 4 * HR * DH : W * NA * ML * 16;
    static constexpr int SM = SM0 > 4096 ? SM0 : 4096;
    static_assert(SM >= 4 * (int)PAGED_SEQS, "the lengths of PAGED_SEQS sequences");
    // Items in the accumulators' order: 4 heads hq, accumulator a, lane n of 16.
    static __device__ __forceinline__ int hq(int item) { return item / DH; }
    static __device__ __forceinline__ int dim(int item) {
        const int n = item % 16, a = item / 16 % NA;
        return a / EV * 16 * EV + n * EV + a % EV;
    }
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int WORDS>
struct WordsOf {
    typedef uint32_t type __attribute__((ext_vector_type(WORDS)));
};
template <>
struct WordsOf<1> {
    typedef uint32_t type;
};

// WORDS 32-bit words of a lane (0: 16 bits) at scalar offset `row` and the lane's `off`. NT: past the caches.
template <bool NT, int WORDS>
__device__ __forceinline__ typename WordsOf<WORDS ? WORDS : 1>::type load_words(const PagedTile& t, uint32_t row, uint32_t off) {
    if constexpr (WORDS == 4) return __builtin_amdgcn_raw_buffer_load_b128(t.rsrc, (int)off, (int)row, NT ? 2 : 0);
    else if constexpr (WORDS == 2) return __builtin_amdgcn_raw_buffer_load_b64(t.rsrc, (int)off, (int)row, NT ? 2 : 0);
    else if constexpr (WORDS == 1) return __builtin_amdgcn_raw_buffer_load_b32(t.rsrc, (int)off, (int)row, NT ? 2 : 0);
    else return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(t.rsrc, (int)off, (int)row, NT ? 2 : 0);
}
template <typename W>
__device__ __forceinline__ uint32_t word(const W& x, int i) {
    if constexpr (sizeof(W) == 4) return x;
    else return x[i];
}

// Whole numbers as fp16 operands. A field of 4 or 8 bits alone in the low part of a 16-bit half is, as fp16, that
// number times 2^-24 (at bit 4: 2^-20), a denormal, and a multiplication by sub and a power of two with the offset's
// subtraction is one exact fma for two of them: (N 2^-24)(sub 2^8) - 8 sub 2^-16. So numbers of 4 bits become
// sub n 2^-16 from a low field, sub n 2^-12 from one at bit 4, and those of 8 bits n 2^-9.
struct SubPair {
    f16x2 mul, low, high;  // sub 2^8, -8 sub 2^-16, -8 sub 2^-12 (finite for any byte that may stand there)
};
// `sel` picks the two bytes (0 .. 3) of stored subs for a perm with 0x64 between: 1024 + byte as fp16.
__device__ __forceinline__ SubPair sub_pair(uint32_t stored, uint32_t sel) {
    const f16x2 sub = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, stored, sel | 0x04000400u)) - (_Float16)1152.0f;
    return {sub * (_Float16)256.0f, sub * (_Float16)-0x1p-13f, sub * (_Float16)-0x1p-9f};
}
__device__ __forceinline__ uint32_t low_fields(uint32_t w, const SubPair& s) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, w & 0x000F000Fu), s.mul, s.low));
}
__device__ __forceinline__ uint32_t high_fields(uint32_t w, const SubPair& s) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, w & 0x00F000F0u), s.mul, s.high));
}
// Bytes a of x and b of y, each alone in a half.
template <int A, int B>
__device__ __forceinline__ uint32_t two_bytes(uint32_t y, uint32_t x) {
    return __builtin_amdgcn_perm(y, x, 0x0C000C00u | (uint32_t)(4 + B) << 16 | A);
}
__device__ __forceinline__ uint32_t byte_fields(uint32_t w) {
    const f16x2 mul = {(_Float16)32768.0f, (_Float16)32768.0f}, add = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, w), mul, add));
}

constexpr float LOG2E = 0x1.715476p+0f;

// tanh to 2 units in the last place or so, in 14 instructions (tanhf is 46; with a soft-cap four of it were half of a
// tile of 128 dims): below 1/2 z + z^3 P(z^2), P fitted to 2^-25 of the result there; else 1 - 2 / (e^2|z| + 1).
__device__ __forceinline__ float quick_tanh(float z) {
    const float u = z * z;
    const float p = fmaf(fmaf(fmaf(0.0172569659f, u, -0.0530529357f), u, 0.133259878f), u, -0.333331496f);
    const float e = __builtin_amdgcn_exp2f(2.0f * LOG2E * fabsf(z));
    const float far = copysignf(fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f), z);
    return fabsf(z) < 0.5f ? fmaf(z * u, p, z) : far;
}
// Scores are relative to a maximum that follows the tiles' by more than this (of 2^x) alone: the accumulators are
// scaled then, which took a fifth of a tile's vector instructions where every new maximum did.
constexpr float LAZY = 8.0f, LEAST = 0x1p-8f;  // 2^-LAZY

template <int DH, int BITS, int NHQ, bool WIN, bool MANY = false>
__device__ __forceinline__ void paged_decode_quant(const G4aPagedAttnParams& p) {
    using C = QuantCfg<DH, BITS, NHQ, MANY>;
    using Q = QuantRow<DH, BITS>;
    constexpr bool I4 = BITS == 4;
    constexpr int HR = C::HR, NA = C::NA, EV = C::EV, ROW = Q::ROW, G = Q::G, ML = C::ML, COLS = 2 * HR, W = C::W;
    constexpr int KL = ROW >= 64 ? ROW / 64 : 1, KW = ROW >= 64 ? 4 : 2;      // K: loads of a lane, words of one
    constexpr int VN = DH / (16 * EV), VBY = EV * BITS / 8, VW = VBY / 4;     // V: blocks of dims, a lane's bytes and words
    __shared__ __attribute__((aligned(16))) char smem[C::SM];
    __shared__ __attribute__((aligned(16))) float f_s[W][HR];
    __shared__ float m_s[W][HR], l_s[W][HR], r_s[W], k_s[HR];
    f16x8* const qs = reinterpret_cast<f16x8*>(smem);
    f4v* const mrg = reinterpret_cast<f4v*>(smem);
    const G4aPaged& c = p.c;
    const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, key = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // (one wave looks its part up, for all: with 16 waves of a CU at it each, of 128 sequences, it took 4 us of a call)
    __shared__ PagedPart found;
    __shared__ bool any;
    if (w == 0) {
        PagedPart x;
        const bool is = paged_find<HR, false>(p, reinterpret_cast<uint32_t*>(smem), lane, 0, x);
        if (lane == 0) found = x, any = is;
    }
    barrier_lds();
    if (!any) return;
    PagedPart mine;
    static_assert(sizeof mine % 4 == 0, "words");
#pragma unroll
    for (int i = 0; i < (int)sizeof mine / 4; ++i)
        reinterpret_cast<uint32_t*>(&mine)[i] = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t*>(&found)[i]);
    const PagedSpan sp = mine.sp;
    const uint32_t at = blockIdx.x, b = mine.b, e = mine.to, h0 = mine.h0, nh = mine.nh, kvh = mine.kvh;
    if (sp.n == 0) {
        for (uint32_t i = tid; i < nh * DH; i += 64 * W) p.out[((size_t)b * p.Hq + h0) * DH + i] = 0.0f;
        return;
    }

    // ---- loads: a tile's rows and its block of subs and scales, in each pool ----
    auto page_of = [&](uint32_t t) {
        const uint32_t no = (sp.first + t) >> (c.page_shift - 4);
        return load_scalar(c.table, (size_t)b * c.per_seq + (c.ring ? no % c.per_seq : no));
    };
    struct Tile {
        PagedTile rows, meta;
    };
    // (`is` false: of no bytes, whose loads go nowhere. One copy of a tile's code, whose loads of a next tile the last
    // makes like that: with a copy of its own for the last tile short parts ran twice the code, most of it not in a cache.)
    auto tile_of = [&](const void* pool, uint32_t page, uint32_t t, bool is) {
        const uint32_t r = ((sp.first + t) * 16) & ((1u << c.page_shift) - 1), no = page < c.n_pages ? page : 0u;
        return Tile{paged_tile(pool, Q::row_at(c, no, kvh, r), is ? 16 * ROW : 0),
                    paged_tile(pool, Q::meta_at(c, no, kvh, r), is ? Q::META : 0)};
    };
    typename WordsOf<KW>::type k[KL];
    typename WordsOf<VW ? VW : 1>::type v[4][VN];  // rows 4 g4 .. 4 g4 + 3
    typename WordsOf<2>::type ks, vs;              // S of tokens 4 g4 .. 4 g4 + 3
    uint32_t ksub = 0, vsub = 0;                   // subs: of the lane's KL groups; of its group, the four rows
    auto load_k = [&](const Tile& t, int j, int key, int g4) {
        k[j] = load_words<!WIN, KW>(t.rows, 0, key * ROW + 4 * KW * g4 + 64 * j);
    };
    auto load_ks = [&](const Tile& t, int key, int g4) {
        ks = load_words<!WIN, 2>(t.meta, 16 * G, 8 * g4);
        if constexpr (I4) {
            if constexpr (G == 16) ksub = load_words<!WIN, 1>(t.meta, 0, 16 * key + 4 * g4);
            else if constexpr (G == 8) ksub = load_words<!WIN, 0>(t.meta, 0, 8 * key + 2 * g4);
            else ksub = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(t.meta.rsrc, G * key + (G == 4 ? g4 : g4 / 2), 0, WIN ? 0 : 2);
        }
    };
    auto load_v = [&](const Tile& t, int key, int g4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int y = 0; y < VN; ++y) v[i][y] = load_words<!WIN, VW>(t.rows, i * ROW, 4 * g4 * ROW + VBY * key + 16 * VBY * y);
        vs = load_words<!WIN, 2>(t.meta, 16 * G, 8 * g4);
        if constexpr (I4) vsub = load_words<!WIN, 1>(t.meta, 0, 16 * (key * EV / 32) + 4 * g4);
    };

    // ---- the query rows into LDS: each head's scaled by a power of two and split into two fp16 parts, whose sum it
    // is to 2^-22; a piece is 8 dims of a head, in the order in which the tiles' whole numbers come out of their words ----
    constexpr int PH = DH / 8, QP = (HR * PH + 64 * W - 1) / (64 * W);  // pieces of a head, of a thread
    f4v qr[QP][2];
#pragma unroll
    for (int i = 0; i < QP; ++i) {
        const int x = tid + 64 * W * i, h = x / PH;
        const bool is = h < (int)nh;
#pragma unroll
        for (int y = 0; y < 2; ++y)
            qr[i][y] = is ? *reinterpret_cast<const f4v*>(p.q + ((size_t)b * p.Hq + h0 + h) * DH + x % PH * 8 + 4 * y)
                          : f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
    uint32_t t = mine.from + w;
    uint32_t page = page_of(min(t, e - 1)), page_next = t + W < e ? page_of(t + W) : 0u;
    {
        const Tile kt = tile_of(c.k, page, min(t, e - 1), t < e);
#pragma unroll
        for (int j = 0; j < KL; ++j) load_k(kt, j, key, g4);
        load_ks(kt, key, g4);
    }
#pragma unroll
    for (int i = 0; i < QP; ++i) {
        const int x = tid + 64 * W * i, h = x / PH, ch = x % PH;
        if (QP * 64 * W > HR * PH && x >= HR * PH) break;
        uint32_t big = 0;
#pragma unroll
        for (int y = 0; y < 8; ++y) big = max(big, __float_as_uint(qr[i][y / 4][y % 4]) & 0x7FFFFFFFu);
        big = g4a_dpp_max<G4A_DPP_XOR1>(big);
        big = g4a_dpp_max<G4A_DPP_XOR2>(big);
        big = g4a_dpp_max<G4A_DPP_HALF_MIRROR>(big);
        if constexpr (PH >= 16) big = g4a_dpp_max<G4A_DPP_ROW_MIRROR>(big);
        if constexpr (PH >= 32) big = g4a_pair16_max(big);
        if constexpr (PH >= 64) big = g4a_pair32_max(big);
        // times 2^(up - 127): the largest to [2^10, 2^11) (8 bits: [2^14, 2^15)), or by 2^122, of which 16 times is a
        // number too: a query may be all zeros
        const uint32_t up = min(249u, 254u + (I4 ? 10u : 14u) - (big >> 23));
        const float f = __uint_as_float(up << 23);
        if (ch == 0) k_s[h] = __uint_as_float((254u - up) << 23) * (I4 ? 0x1p6f : 0x1p3f);
        f16x8 hi, lo;
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            // 4 bits: fields (q, q + 4) of a word are halves of a register; the low ones are 2^-4 too small
            const int d = I4 ? y / 2 + 4 * (y % 2) : y;
            const float z = qr[i][d / 4][d % 4] * (I4 && y / 2 % 2 == 0 ? 16.0f * f : f);
            hi[y] = (_Float16)z;
            lo[y] = (_Float16)(z - (float)hi[y]);
        }
        const int mt = !I4 ? ch / 8 * 2 + ch % 2 : DH == 64 ? ch % 2 : ch / 16 * 4 + ch % 4;
        const int gr = !I4 || DH == 64 ? ch / 2 % 4 : ch / 4 % 4, row = 4 * mt + gr;
        qs[row * COLS + (h ^ (row % COLS))] = hi;  // (the columns turned, or a wave's writes would meet in four banks)
        qs[row * COLS + ((HR + h) ^ (row % COLS))] = lo;
    }
    load_v(tile_of(c.v, page, min(t, e - 1), t < e), key, g4);  // (ahead of the queries it would be ahead of other waves' too)
    barrier_lds();  // (K and V stay in flight across it)

    // lane (g4, n): keys 4 g4 + r of the tile, head n % HR of the unit; part n / HR % 2 of the queries and probabilities
    const bool lower = NHQ < 4 && key / HR % 2;
    const float qf = k_s[key % HR] * p.scale * (p.softcap > 0.0f ? 1.0f : LOG2E);
    const float cap_inv = 1.0f / p.softcap;  // (where there is one: from 2^-126 to 2^126)
    float m = G4A_NEG_INF, l = 0.0f;
    // P V's power of two: 2^6 over the largest S of V so far, rounded down to one (and as for 2^-100 for smaller S:
    // the merge's factors, its reciprocal over a sum of up to 2^29, are not to be denormal)
    float rs = 0x1p106f;
    f4v acc[NA];
#pragma unroll
    for (int d = 0; d < NA; ++d) acc[d] = f4v{0.0f, 0.0f, 0.0f, 0.0f};

    // (the lane, and what follows from it, anew in each tile of 512 dims: kept, those are a few registers too many)
    auto lane_again = [&] {
        int x = lane;
        if constexpr (DH == 512 && NHQ < 4) asm volatile("" : "+v"(x));
        return x;
    };
    for (; t < e; t += W) {
        const int ln = lane_again(), g4 = ln >> 4, key = ln & 15;
        const bool more = t + W < e, first = t == mine.from + w;
        const uint32_t page_after = t + 2 * W < e ? page_of(t + 2 * W) : 0u;
        const Tile kt = tile_of(c.k, page_next, t + W, more);
        // ---- scores ----
        constexpr int KM = I4 ? KW : 2, QN = NHQ == 4 ? 2 : 1;  // MFMA steps of a load; query operands of a step
        f4v d[QN];
#pragma unroll
        for (int y = 0; y < QN; ++y) d[y] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        // (a row's columns are turned by its number modulo COLS: 4 mt and g4, which share no bit)
        const f16x8* const qrow = qs + g4 * COLS;
        const int col = (key ^ g4) % COLS;
        f16x8 qb[2][KM][QN];  // those of a load's steps are read ahead of the load before it
        auto read_q = [&](int j) {
#pragma unroll
            for (int i = 0; i < KM; ++i)
#pragma unroll
                for (int y = 0; y < QN; ++y)
                    qb[j % 2][i][y] = qrow[(col ^ ((4 * (KM * j + i) + 16 * y) % COLS)) + 4 * (KM * j + i) * COLS];
        };
        auto mac = [&](int j, int i, const f16x8& a) {
#pragma unroll
            for (int y = 0; y < QN; ++y) d[y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qb[j % 2][i][y], d[y], 0, 0, 0);
        };
        read_q(0);
#pragma unroll
        for (int j = 0; j < KL; ++j) {
            if (j + 1 < KL) read_q(j + 1);
            if constexpr (I4) {
                const SubPair s = sub_pair(ksub, j | j << 16);
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    const uint32_t x = k[j][i], y = x >> 8;
                    mac(j, i, __builtin_bit_cast(f16x8, (typename WordsOf<4>::type){low_fields(x, s), high_fields(x, s),
                                                                                           low_fields(y, s), high_fields(y, s)}));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                    mac(j, i / 2, __builtin_bit_cast(f16x8, (typename WordsOf<4>::type){
                                           byte_fields(two_bytes<0, 1>(k[j][i], k[j][i])), byte_fields(two_bytes<2, 3>(k[j][i], k[j][i])),
                                           byte_fields(two_bytes<0, 1>(k[j][i + 1], k[j][i + 1])),
                                           byte_fields(two_bytes<2, 3>(k[j][i + 1], k[j][i + 1]))}));
            }
            load_k(kt, j, key, g4);
            __builtin_amdgcn_sched_barrier(0);
        }
        f4v x;
#pragma unroll
        for (int r = 0; r < 4; ++r) {  // the parts' sums, in columns HR apart
            if constexpr (NHQ == 4) x[r] = d[0][r] + d[1][r];
            else if constexpr (NHQ == 2) x[r] = d[0][r] + g4a_dpp<ROW_ROR8>(d[0][r]);
            else x[r] = d[0][r] + g4a_dpp<ROW_ROR4>(d[0][r]);
            const float s = __uint_as_float(r % 2 ? ks[r / 2] & 0xFFFF0000u : ks[r / 2] << 16);
            x[r] *= s * 0x1p6f * qf;
            if (p.softcap > 0.0f) x[r] = p.softcap * LOG2E * quick_tanh(x[r] * cap_inv);
        }
        f4v sv;
#pragma unroll
        for (int r = 0; r < 4; ++r) sv[r] = __uint_as_float(r % 2 ? vs[r / 2] & 0xFFFF0000u : vs[r / 2] << 16);
        const uint32_t t0 = (sp.first + t) * 16;
        const uint32_t lo = sp.lo > t0 ? sp.lo - t0 : 0u, hi = page < c.n_pages ? min(16u, sp.len - t0) : 0u;
        if (lo > 0 || hi < 16) {  // what no token was written to may hold anything
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t row = 4 * g4 + r;
                const bool seen = row >= lo && row < hi;
                x[r] = seen ? x[r] : G4A_NEG_INF;
                sv[r] = seen ? sv[r] : 0.0f;
            }
        }
        load_ks(kt, key, g4);
        // ---- running maximum and sum, in powers of two ----
        const float mt = g4a_col_max4(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        if (__ballot(mt > m + LAZY)) {
            const float mn = mt > m + LAZY ? mt : m;
            const float corr = m == G4A_NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= corr;
            if (!first)
#pragma unroll
                for (int r = 0; r < 4; ++r) {  // the lanes of a head hold its factor
                    const float f = NHQ > 1 ? __shfl(corr, 4 * (g4 % NHQ) + r) : g4a_lane(corr, r);
#pragma unroll
                    for (int a = 0; a < NA; ++a) acc[a][r] *= f;
                }
        }
        // V's scales times rs stay below 2^7, and with the probability, at most 2^LAZY, below 2^15 of fp16's 65504: a
        // probability is held to 2^-22, or 2^-31 (half of fp16's smallest step, over 2^6) of one of 1 at the largest S
        const float top = fmaxf(fmaxf(fabsf(sv[0]), fabsf(sv[1])), fmaxf(fabsf(sv[2]), fabsf(sv[3])));
        if (__ballot(top * rs >= 0x1p7f)) {
            const uint32_t r2 = __float_as_uint(g4a_col_max4(top)) & 0x7F800000u;
            const float now = __uint_as_float((260u << 23) - r2), f = now / rs;
            rs = now;
            if (!first)
#pragma unroll
                for (int a = 0; a < NA; ++a) acc[a] *= f;
        }
        const float from = m == G4A_NEG_INF ? 0.0f : m;
        f4v pr;
#pragma unroll
        for (int r = 0; r < 4; ++r) pr[r] = __builtin_amdgcn_exp2f(x[r] - from);
        l += (pr[0] + pr[1]) + (pr[2] + pr[3]);
        // ---- P V: P is the A operand as it stands, in two parts ----
        f16x4 pa[QN];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float y = pr[r] * (sv[r] * rs);
            // (one f32: the compiler rounds a product on its way to fp16 once, and elsewhere twice, and parts that were
            // made of both were a step of fp16 apart now and then)
            asm("" : "+v"(y));
            const _Float16 high = (_Float16)y;
            if constexpr (NHQ == 4) {
                pa[0][r] = high;
                pa[1][r] = (_Float16)(y - (float)high);
            } else {
                pa[0][r] = (_Float16)(lower ? y - (float)high : y);
            }
        }
        const Tile vt = tile_of(c.v, page_next, t + W, more);
        auto pv = [&](int a, uint32_t b0, uint32_t b1) {
            const f16x4 y = __builtin_bit_cast(f16x4, (typename WordsOf<2>::type){b0, b1});
#pragma unroll
            for (int z = 0; z < QN; ++z) acc[a] = __builtin_amdgcn_mfma_f32_16x16x16f16(pa[z], y, acc[a], 0, 0, 0);
        };
        SubPair s01, s23;
        if constexpr (I4) s01 = sub_pair(vsub, 0x00010000u), s23 = sub_pair(vsub, 0x00030002u);
#pragma unroll
        for (int y = 0; y < VN; ++y)
#pragma unroll
            for (int i = 0; i < (VW ? VW : 1); ++i) {
                const uint32_t w0 = word(v[0][y], i), w1 = word(v[1][y], i), w2 = word(v[2][y], i), w3 = word(v[3][y], i);
                auto dims = [&](int at, uint32_t ab, uint32_t cd) {  // a byte of each of the four rows
                    if constexpr (I4) {
                        pv(at, low_fields(ab, s01), low_fields(cd, s23));
                        pv(at + 1, high_fields(ab, s01), high_fields(cd, s23));
                    } else {
                        pv(at, byte_fields(ab), byte_fields(cd));
                    }
                };
                constexpr int PER = I4 ? 2 : 1;
                const int first = EV * y + 4 * PER * i;
                dims(first, two_bytes<0, 0>(w1, w0), two_bytes<0, 0>(w3, w2));
                dims(first + PER, two_bytes<1, 1>(w1, w0), two_bytes<1, 1>(w3, w2));
                if constexpr (VW > 0) {
                    dims(first + 2 * PER, two_bytes<2, 2>(w1, w0), two_bytes<2, 2>(w3, w2));
                    dims(first + 3 * PER, two_bytes<3, 3>(w1, w0), two_bytes<3, 3>(w3, w2));
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        load_v(vt, key, g4);
        page = page_next;
        page_next = page_after;
    }

    // ---- the waves' partials, through LDS ----
    l = g4a_col_sum4(l);
    if (lane < HR) m_s[w][lane] = m, l_s[w][lane] = l;
    if (lane == 0) r_s[w] = (I4 ? 0x1p12f : 0x1p9f) / rs;
    barrier_lds();  // every wave is done with the query rows, where the accumulators go
    const bool whole = mine.parts == 1;
    if (w == 0) {  // the waves' factors of each head: lane HR i + h for wave i and head h
        const int i = lane / HR, h = lane % HR;
        const bool is = i < W;
        const float mi = is ? m_s[i][h] : G4A_NEG_INF, li = is ? l_s[i][h] : 0.0f;
        auto over_waves = [&](float x, auto op) {  // the lanes of a head are HR apart
            if constexpr (HR == 4) x = op(x, g4a_dpp<ROW_ROR4>(x));
            if constexpr (HR <= 8) x = op(x, g4a_dpp<ROW_ROR8>(x));
            float2 y = g4a_pair16(x);
            x = op(y.x, y.y);
            y = g4a_pair32(x);
            return op(y.x, y.y);
        };
        static_assert(W * HR <= 64, "a lane a wave and head");
        const float M = over_waves(mi, [](float a, float b) { return fmaxf(a, b); });
        float f = mi == G4A_NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(mi - M);
        // (a sum without a maximum: scores that are NaN)
        const float L = over_waves(mi == G4A_NEG_INF ? li : li * f, [](float a, float b) { return a + b; });
        // (a partial's weights and their sum by 2^-LAZY: weights stand above 1 by up to 2^LAZY, where scores rise behind the
        // maximum, and are not to take sums of V rows near f32's largest numbers past them)
        if (!whole && lane < HR) {
            float* const ml = p.part_ml + (size_t)at * 2 * HR + lane;
            ml[0] = M;
            ml[HR] = L * LEAST;
        }
        if (whole) f *= L != 0.0f ? 1.0f / L : 0.0f;
        else f *= LEAST;
        if (is) f_s[i][h] = f * r_s[i];
    }
    if constexpr (NHQ == 4) {
#pragma unroll
        for (int d = 0; d < NA; ++d) mrg[(w * NA + d) * 64 + lane] = acc[d];
    } else {
        // A head's two parts are in lanes 16 NHQ apart. Two accumulators at a time: a swap brings the first parts of both
        // together, and the second parts, and the sums of the one are in the lower of these lanes, of the other in the upper.
#pragma unroll
        for (int d = 0; d < NA / 2; ++d) {
            f4v y;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t one = __float_as_uint(acc[d][r]), two = __float_as_uint(acc[d + NA / 2][r]);
                if constexpr (NHQ == 2) {
                    const auto z = __builtin_amdgcn_permlane32_swap(one, two, false, false);
                    y[r] = __uint_as_float(z[0]) + __uint_as_float(z[1]);
                } else {
                    const auto z = __builtin_amdgcn_permlane16_swap(one, two, false, false);
                    y[r] = __uint_as_float(z[0]) + __uint_as_float(z[1]);
                }
            }
            if (lane < 2 * ML) mrg[(w * NA + d + lane / ML * (NA / 2)) * ML + lane % ML] = y;
        }
    }
    barrier_lds();
    f4v* const dst = reinterpret_cast<f4v*>(p.part) + (size_t)at * C::ITEMS;
#pragma unroll
    for (int i0 = 0; i0 < C::ITEMS; i0 += 64 * W) {
        const int i = i0 + tid;
        if (C::ITEMS % (64 * W) && i >= C::ITEMS) break;
        const int hq = C::hq(i), n = i % 16, a = i / 16 % NA;
        f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int y = 0; y < W; ++y)
            o = __builtin_elementwise_fma(mrg[(y * NA + a) * ML + 16 * hq + n], *reinterpret_cast<const f4v*>(&f_s[y][4 * hq]), o);
        if (I4 && a % 2 == 0) o *= 16.0f;
        if (whole) {
            const int dim = C::dim(i);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (4 * hq + r < (int)nh) p.out[((size_t)b * p.Hq + h0 + 4 * hq + r) * DH + dim] = o[r];
        } else {
            dst[i] = o;
        }
    }
}

}  // namespace

#define G4A_PAGED_QUANT_DECODE(dh, type, bits, nhq, occ)                                                      \
    extern "C" __global__                                                                                     \
        __launch_bounds__((64 * QuantCfg<dh, bits, nhq>::W), (occ * QuantCfg<dh, bits, nhq>::W / 4))          \
        void g4a_paged_decode_d##dh##_##type##_h##nhq(G4aPagedAttnParams p) {                                 \
        paged_decode_quant<dh, bits, nhq, false>(p);                                                          \
    }                                                                                                         \
    extern "C" __global__                                                                                     \
        __launch_bounds__((64 * QuantCfg<dh, bits, nhq>::W), (occ * QuantCfg<dh, bits, nhq>::W / 4))          \
        void g4a_paged_decode_win_d##dh##_##type##_h##nhq(G4aPagedAttnParams p) {                             \
        paged_decode_quant<dh, bits, nhq, true>(p);                                                           \
    }                                                                                                         \
    extern "C" __global__ __launch_bounds__(512) void g4a_paged_combine16_d##dh##_##type##_h##nhq(            \
        G4aPagedAttnParams p) { paged_combine<QuantCfg<dh, bits, nhq>, 16, 8>(p); }                           \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_combine64_d##dh##_##type##_h##nhq(            \
        G4aPagedAttnParams p) { paged_combine<QuantCfg<dh, bits, nhq>, 64, 4>(p); }
#define G4A_PAGED_QUANT_TYPES(dh, nhq, occ_i8, occ_i4) \
    G4A_PAGED_QUANT_DECODE(dh, i8, 8, nhq, occ_i8)     \
    G4A_PAGED_QUANT_DECODE(dh, i4, 4, nhq, occ_i4)
// The second bound: workgroups of a CU, as the registers (and LDS) leave room for.
G4A_PAGED_QUANT_TYPES(64, 1, 4, 4) G4A_PAGED_QUANT_TYPES(64, 2, 4, 4) G4A_PAGED_QUANT_TYPES(64, 4, 4, 4)
G4A_PAGED_QUANT_TYPES(128, 1, 4, 4) G4A_PAGED_QUANT_TYPES(128, 2, 4, 4) G4A_PAGED_QUANT_TYPES(128, 4, 4, 4)
G4A_PAGED_QUANT_TYPES(256, 1, 3, 3) G4A_PAGED_QUANT_TYPES(256, 2, 3, 3) G4A_PAGED_QUANT_TYPES(256, 4, 2, 2)
G4A_PAGED_QUANT_TYPES(512, 1, 1, 1) G4A_PAGED_QUANT_TYPES(512, 2, 1, 1) G4A_PAGED_QUANT_TYPES(512, 4, 1, 1)
// Many units of 512 dims: two workgroups of four waves a CU.
#define G4A_PAGED_QUANT_MANY(type, bits, nhq)                                                                 \
    extern "C" __global__ __launch_bounds__(256, 2) void g4a_paged_decode_many_d512_##type##_h##nhq(          \
        G4aPagedAttnParams p) { paged_decode_quant<512, bits, nhq, false, true>(p); }                         \
    extern "C" __global__ __launch_bounds__(256, 2) void g4a_paged_decode_many_win_d512_##type##_h##nhq(      \
        G4aPagedAttnParams p) { paged_decode_quant<512, bits, nhq, true, true>(p); }
G4A_PAGED_QUANT_MANY(i8, 8, 1) G4A_PAGED_QUANT_MANY(i8, 8, 2) G4A_PAGED_QUANT_MANY(i4, 4, 1) G4A_PAGED_QUANT_MANY(i4, 4, 2)
#undef G4A_PAGED_QUANT_MANY
#undef G4A_PAGED_QUANT_TYPES
#undef G4A_PAGED_QUANT_DECODE
