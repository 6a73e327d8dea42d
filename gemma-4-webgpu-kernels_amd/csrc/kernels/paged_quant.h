// Pages of 8 and 4 bits: where a row stands, and how its values become whole numbers
// and back. A row is one token's K or V of one head, x[0 .. DH).
//
//   8 bits: x ~ S n, |n| <= 127, S the least bfloat16 with 127 S >= max |x|.
//   4 bits: x ~ S sub n in groups of 32 dims, -8 <= n <= 7. S: the least bfloat16 with
//           1016 S >= max |x| of the row (1016 = 127 * 8); |sub| >= 1: the least whole number with
//           8 |sub| S >= max |x| of the group, at most 127; its sign puts the group's extreme
//           at n = -8 (the positive one, of two equal ones).
// S is at least 2^-126. n is x / S (or x / (S sub)) rounded to nearest, halves to even, in
// exact arithmetic, and cut to its range: 4 bits lose up to a step at the end opposite to
// the extreme, all else half a step. A row that holds an infinity or a NaN gets S = NaN.
//
// The two scales are what lets attention work on whole numbers: sub n has 10 bits, an
// fp16 operand of a matrix instruction exactly, and S, one number a row, goes to the
// score or the probability. A row's values S sub n are exact in f32.
//
// A page: rows [Hkv][page size] of DH * BITS / 8 bytes, n + 2^(BITS-1) (4 bits: an even dim
// in a byte's low half), then [Hkv][page size / 16] blocks of 16 tokens: in 4 bits their
// subs + 128 (K: token by token, group g at place g % 4 * (G/4) + g / 4 of G >= 4, as a lane of
// the attention kernel holds them together; V: group by group), and S of each. Heads
// are apart so that a tile of 16 tokens of one head is one run of bytes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "g4a_math.h"
#include "g4a_params.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int DH, int BITS>
struct QuantRow {
    static constexpr int ROW = DH * BITS / 8;              // bytes of a row
    static constexpr int G = BITS == 4 ? DH / 32 : 0;      // groups with a sub of their own
    static constexpr int META = 16 * G + 32;               // bytes of a block of subs and scales
    static constexpr int MOST = BITS == 4 ? 1016 : 127;    // max |x| is at most MOST S
    // Bytes into a pool: row r of a page and head, and that of its block, whose token r % 16 it is.
    static __device__ __forceinline__ size_t row_at(const G4aPaged& c, uint32_t page, uint32_t h, uint32_t r) {
        return (size_t)page * c.page_stride + (((size_t)h << c.page_shift) + r) * ROW;
    }
    static __device__ __forceinline__ size_t meta_at(const G4aPaged& c, uint32_t page, uint32_t h, uint32_t r) {
        return (size_t)page * c.page_stride + ((size_t)c.Hkv << c.page_shift) * ROW +
               (((size_t)h << (c.page_shift - 4)) + r / 16) * META;
    }
    // Place of group g of token r among its block's subs.
    template <bool VALUES>
    static __device__ __forceinline__ uint32_t sub_at(uint32_t g, uint32_t r) {
        if constexpr (VALUES) return 16 * g + r % 16;
        else return r % 16 * G + (G >= 4 ? g % 4 * (G / 4) + g / 4 : g);
    }
};

__device__ __forceinline__ uint32_t g4a_pair16_max(uint32_t x) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ uint32_t g4a_pair32_max(uint32_t x) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}
template <int CTRL>
__device__ __forceinline__ uint32_t g4a_dpp_max(uint32_t x) {
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false));
}

// The largest x of LPR lanes (16, 32 or 64) that hold a row, in each of them.
template <int LPR>
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
    x = g4a_dpp_max<G4A_DPP_XOR1>(x);
    x = g4a_dpp_max<G4A_DPP_XOR2>(x);
    x = g4a_dpp_max<G4A_DPP_HALF_MIRROR>(x);
    x = g4a_dpp_max<G4A_DPP_ROW_MIRROR>(x);
    if constexpr (LPR >= 32) x = g4a_pair16_max(x);
    if constexpr (LPR == 64) x = g4a_pair32_max(x);
    return x;
}

// S of a row whose largest magnitude is `big` (finite): about big / MOST, rounded up to a bfloat16, is it or next to
// it, and MOST S is exact. (Divisions by rule of IEEE were half of a row's instructions, here and below.)
template <int MOST>
__device__ __forceinline__ float quant_scale(float big) {
    const float t = fmaxf(big * (1.0f / MOST), 0x1p-126f);
    const uint32_t up = (__float_as_uint(t) + 0xFFFFu) & 0xFFFF0000u;
    const float s = __uint_as_float(up), less = fmaxf(__uint_as_float(up - 0x10000u), 0x1p-126f);
    if (s * (float)MOST < big) return __uint_as_float(up + 0x10000u);
    return less * (float)MOST >= big ? less : s;
}

// x / step rounded to nearest, halves to even, exactly, for four values: x * inv (inv about 1 / step) rounds to it or next
// to it, and x - n step, exact as it has no more bits than x, says which. That n is not x * inv's, or that x is
// half way between two, is rare and looked for once.
__device__ __forceinline__ f32x4 quant_round(const f32x4& x, float step, float inv) {
    const float half = 0.5f * fabsf(step);
    f32x4 n, r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        n[i] = rintf(x[i] * inv);
        r[i] = fmaf(-n[i], step, x[i]);
    }
    if (__ballot(fmaxf(fmaxf(fabsf(r[0]), fabsf(r[1])), fmaxf(fabsf(r[2]), fabsf(r[3]))) >= half))
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float towards = (r[i] < 0.0f) != (step < 0.0f) ? -1.0f : 1.0f;
            const bool odd = (int)n[i] & 1;
            if (fabsf(r[i]) > half || (fabsf(r[i]) == half && odd)) n[i] += towards;
        }
    return n;
}

// A row into its place, by LPR lanes of which lane l holds dims 4 l .. and, at 512, 256 + 4 l ..; `is`: there is one.
// Every lane of the wave takes part.
template <int DH, int BITS, bool VALUES, int E>
__device__ __forceinline__ void quant_store(const G4aPaged& c, void* pool, uint32_t slot, uint32_t h, int l,
                                            const f32x4 (&x)[E], bool is) {
    using Q = QuantRow<DH, BITS>;
    constexpr int LPR = DH / (4 * E);
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) big = max(big, __float_as_uint(x[e][i]) & 0x7FFFFFFFu);
    big = row_max<LPR>(big);  // (as words: infinities and NaN are above all else)
    const bool bad = big >= 0x7F800000u;
    const float s = bad ? 1.0f : quant_scale<Q::MOST>(__uint_as_float(big));
    const uint32_t page = slot >> c.page_shift, r = slot & ((1u << c.page_shift) - 1);
    uint8_t* const row = static_cast<uint8_t*>(pool) + Q::row_at(c, page, h, r);
    uint8_t* const meta = static_cast<uint8_t*>(pool) + Q::meta_at(c, page, h, r);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        f32x4 y = x[e];
        if (bad) y = f32x4{0, 0, 0, 0};
        if constexpr (BITS == 8) {
            const f32x4 n = quant_round(y, s, __builtin_amdgcn_rcpf(s));
            const uint32_t w = (uint32_t)fmaf(n[1], 256.0f, n[0] + 128.0f * 257.0f) |
                               (uint32_t)fmaf(n[3], 256.0f, n[2] + 128.0f * 257.0f) << 16;
            if (is) *reinterpret_cast<uint32_t*>(row + 4 * l + 256 * e) = w;
        } else {
            const float high = g4a_max8(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
            const float low = g4a_max8(fmaxf(fmaxf(-y[0], -y[1]), fmaxf(-y[2], -y[3])));
            const float most = fmaxf(high, low);
            const float s8 = 8.0f * s;
            float c8 = fmaxf(ceilf(most * __builtin_amdgcn_rcpf(s8)), 1.0f);  // (or next to it; the products are exact)
            if (c8 * s8 < most) c8 += 1.0f;
            else if (c8 > 1.0f && (c8 - 1.0f) * s8 >= most) c8 -= 1.0f;
            const float sub = high >= low ? -c8 : c8, step = s * sub;
            f32x4 n = quant_round(y, step, __builtin_amdgcn_rcpf(step));
#pragma unroll
            for (int i = 0; i < 4; ++i) n[i] = fminf(fmaxf(n[i], -8.0f), 7.0f);
            uint32_t w = (uint32_t)fmaf(n[3], 4096.0f, fmaf(n[2], 256.0f, fmaf(n[1], 16.0f, n[0] + 8.0f * 4369.0f)));
            w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, G4A_DPP_XOR1, 0xf, 0xf, false) << 16;
            if (is && l % 2 == 0) *reinterpret_cast<uint32_t*>(row + 2 * l + 128 * e) = w;
            if (is && l % 8 == 0) meta[Q::template sub_at<VALUES>((4 * l + 256 * e) / 32, r)] = (uint8_t)((int)sub + 128);
        }
    }
    if (is && l == 0)
        *reinterpret_cast<uint16_t*>(meta + 16 * Q::G + 2 * (r % 16)) =
            bad ? (uint16_t)0x7FC0 : (uint16_t)(__float_as_uint(s) >> 16);
}

// Dims 4 l .. and 256 + 4 l .. of the row at `slot`.
template <int DH, int BITS, bool VALUES, int E>
__device__ __forceinline__ void quant_load(const G4aPaged& c, const void* pool, uint32_t slot, uint32_t h, int l,
                                           f32x4 (&x)[E]) {
    using Q = QuantRow<DH, BITS>;
    const uint32_t page = slot >> c.page_shift, r = slot & ((1u << c.page_shift) - 1);
    const uint8_t* const row = static_cast<const uint8_t*>(pool) + Q::row_at(c, page, h, r);
    const uint8_t* const meta = static_cast<const uint8_t*>(pool) + Q::meta_at(c, page, h, r);
    const float s = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(meta + 16 * Q::G + 2 * (r % 16)) << 16);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if constexpr (BITS == 8) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(row + 4 * l + 256 * e);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[e][i] = ((float)(w >> (8 * i) & 255u) - 128.0f) * s;
        } else {
            const uint32_t w = *reinterpret_cast<const uint16_t*>(row + 2 * l + 128 * e);
            const int sub = (int)meta[Q::template sub_at<VALUES>((4 * l + 256 * e) / 32, r)] - 128;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[e][i] = (float)(((int)(w >> (4 * i) & 15u) - 8) * sub) * s;
        }
    }
}
