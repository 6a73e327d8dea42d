// Rows of K and V between f32 arrays and the pages of a paged KV cache, for gfx950: written
// and read by slot in every type of page, a sequence's tokens in order out of pages of 8 and
// 4 bits (paged.hip has those of f32 and bf16), and the attention producer into such pages.
// The reference has neither pages nor a quantised cache (its KVCache grows one f32 buffer
// per layer, rust/src/kvcache.rs:49-62). Formats: paged_quant.h; layout: G4aPaged.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "g4a_math.h"
#include "g4a_params.h"
#include "paged_quant.h"

namespace {

// LPR lanes hold a row, 4 dims each (8 at 512); a wave holds RPW rows.
template <int DH>
struct RowLanes {
    static constexpr int LPR = DH / 4 < 64 ? DH / 4 : 64, E = DH / (4 * LPR), RPW = 64 / LPR;
};

template <int DH, int BITS, bool VALUES, int E>
__device__ __forceinline__ void store_row(const G4aPaged& c, void* pool, uint32_t slot, uint32_t h, int l,
                                          const f32x4 (&x)[E], bool is) {
    if constexpr (BITS <= 8) {
        quant_store<DH, BITS, VALUES>(c, pool, slot, h, l, x, is);
    } else if (is) {
        const size_t at = (size_t)(slot >> c.page_shift) * c.page_stride +
                          ((size_t)(slot & ((1u << c.page_shift) - 1)) * c.Hkv + h) * DH + 4 * l;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if constexpr (BITS == 32) store4(static_cast<float*>(pool) + at + 256 * e, x[e]);
            else store4(static_cast<__bf16*>(pool) + at + 256 * e, x[e]);
        }
    }
}

template <int DH, int BITS, bool VALUES, int E>
__device__ __forceinline__ void load_row(const G4aPaged& c, const void* pool, uint32_t slot, uint32_t h, int l,
                                         f32x4 (&x)[E]) {
    if constexpr (BITS <= 8) {
        quant_load<DH, BITS, VALUES>(c, pool, slot, h, l, x);
    } else {
        const size_t at = (size_t)(slot >> c.page_shift) * c.page_stride +
                          ((size_t)(slot & ((1u << c.page_shift) - 1)) * c.Hkv + h) * DH + 4 * l;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if constexpr (BITS == 32) x[e] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(pool) + at + 256 * e);
            else x[e] = __builtin_convertvector(*reinterpret_cast<const bf16x4*>(static_cast<const __bf16*>(pool) + at + 256 * e), f32x4);
        }
    }
}

// T tokens' rows into their slots: K by the workgroups of blockIdx.y 0, V by those of 1. Row i of a pool's
// rows is head i % Hkv of token i / Hkv. In 4 bits a row is a reduction over its lanes (S), one over groups of eight of them
// (sub) and some 35 instructions a value; bound by HBM and these: 20011 tokens of 512 dims take 21 us (104 MB read and
// written, 4.9 TB/s; 27 with divisions and with halves looked for value by value). More rows a wave, the next ones' loads ahead,
// were slower (written and read 51.5 us for 43.8).
template <int DH, int BITS, bool VALUES>
__device__ __forceinline__ void paged_write(const G4aPagedRowsParams& p) {
    using R = RowLanes<DH>;
    const G4aPaged& c = p.c;
    const int lane = threadIdx.x & 63, g = lane / R::LPR, l = lane % R::LPR;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rows = p.T * c.Hkv, row = (blockIdx.x * 4 + w) * R::RPW + g;
    const bool is = row < rows;
    const uint32_t t = is ? row / c.Hkv : 0u, slot = p.slots[t];
    f32x4 x[R::E];
#pragma unroll
    for (int e = 0; e < R::E; ++e)
        x[e] = is ? __builtin_nontemporal_load(reinterpret_cast<const f32x4*>((VALUES ? p.v_in : p.k_in) + (size_t)row * DH + 4 * l + 256 * e))
                  : f32x4{0, 0, 0, 0};
    store_row<DH, BITS, VALUES>(c, VALUES ? c.v : c.k, slot, row - t * c.Hkv, l, x, is && (slot >> c.page_shift) < c.n_pages);
}

// The slot of token t of a call: given, or that of position pos0 + t of its sequence; G4A_NO_ROW32 where the cache
// holds none.
__device__ __forceinline__ uint32_t paged_slot(const G4aPagedRowsParams& p, uint32_t t) {
    const G4aPaged& c = p.c;
    if (p.slots) {
        const uint32_t slot = p.slots[t];
        return (slot >> c.page_shift) < c.n_pages ? slot : G4A_NO_ROW32;
    }
    const uint32_t pos = p.pos0 + t, no = pos >> c.page_shift, len = c.len[p.seq];
    const uint32_t e = c.ring ? no % c.per_seq : no;
    const uint64_t room = (uint64_t)c.per_seq << c.page_shift;
    if (pos >= len || e >= c.per_seq || (c.ring && pos + room < len)) return G4A_NO_ROW32;
    const uint32_t page = c.table[(size_t)p.seq * c.per_seq + e];
    return page < c.n_pages ? (page << c.page_shift) + (pos & ((1u << c.page_shift) - 1)) : G4A_NO_ROW32;
}

// T tokens' rows as f32, zeros for those that the cache does not hold. The rows go past the caches: 32768 tokens of 512
// dims in 4 bits take 23.3 us (6.5 TB/s read and written), 37.4 with plain stores. (Four rows a wave, their loads side by
// side, 24.5.)
template <int DH, int BITS, bool VALUES>
__device__ __forceinline__ void paged_read(const G4aPagedRowsParams& p) {
    using R = RowLanes<DH>;
    const G4aPaged& c = p.c;
    const int lane = threadIdx.x & 63, g = lane / R::LPR, l = lane % R::LPR;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rows = p.T * c.Hkv, row = (blockIdx.x * 4 + w) * R::RPW + g;
    if (row >= rows) return;
    const uint32_t t = row / c.Hkv, slot = paged_slot(p, t);
    f32x4 x[R::E];
#pragma unroll
    for (int e = 0; e < R::E; ++e) x[e] = f32x4{0, 0, 0, 0};
    if (slot != G4A_NO_ROW32) load_row<DH, BITS, VALUES>(c, VALUES ? c.v : c.k, slot, row - t * c.Hkv, l, x);
#pragma unroll
    for (int e = 0; e < R::E; ++e)
        __builtin_nontemporal_store(x[e], reinterpret_cast<f32x4*>((VALUES ? p.v_out : p.k_out) + (size_t)row * DH + 4 * l + 256 * e));
}

// Sum of the LPR lanes (16, 32 or 64) that hold a row, in each of them: g4a_row_sum16 and the pairs, on two words.
template <int CTRL>
__device__ __forceinline__ double add_dpp64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, false),
                   hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, false);
    return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int LPR>
__device__ __forceinline__ double row_sum64(double x) {
    x = add_dpp64<G4A_DPP_XOR1>(x);
    x = add_dpp64<G4A_DPP_XOR2>(x);
    x = add_dpp64<G4A_DPP_HALF_MIRROR>(x);
    x = add_dpp64<G4A_DPP_ROW_MIRROR>(x);
    auto pair = [](double y, auto swap) {
        const uint64_t u = __builtin_bit_cast(uint64_t, y);
        const auto lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
        return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
    };
    if constexpr (LPR >= 32) x = pair(x, [](uint32_t y) { return __builtin_amdgcn_permlane16_swap(y, y, false, false); });
    if constexpr (LPR == 64) x = pair(x, [](uint32_t y) { return __builtin_amdgcn_permlane32_swap(y, y, false, false); });
    return x;
}

// The K and V rows of the producer into pages of 8 and 4 bits: y = rope(x / sqrt(mean(x^2) + eps) * w) in 64 bits,
// rounded once to f32 and then quantised. In f32, sums in another order (another width of the wave's work, another
// device) would move a value over the border between two steps now and then, which 4 bits show: so the same rows
// give the same pages. The angle is position * frequency in f32, as for the query rows. The lanes hold a row as for
// paged_write; a wave takes one group of K or of V rows of one token, and query rows waves of their own. 4099 tokens of
// 10 rows of 256 (8 bits) take 21 us, 18.4 into f32 pages, whose K and V rows are in f32; 64 of 512 (4 bits) 5.3 and
// 3.7: a chain of the position and slot, behind which the row is loaded (f32 pages load it beside them), its sum, root
// and division in 64 bits, behind which the weights are, then frequencies and sines, then S and the subs.
template <int DH, int BITS>
__device__ __forceinline__ void paged_produce_kv(const G4aPagedQuantProducerParams& qp) {
    using R = RowLanes<DH>;
    constexpr int E = R::E;
    __shared__ double stage[PP_WAVES][R::RPW][DH];
    __shared__ double turn[PP_WAVES][DH / 2][2];
    const G4aPagedProducerParams& p = qp.p;
    const G4aPaged& c = p.c;
    const int lane = threadIdx.x & 63, g = lane / R::LPR, l = lane % R::LPR;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t item = (blockIdx.x - qp.q_wgs) * PP_WAVES + w, t = item / (2 * qp.kv_groups);
    if (t >= p.T) return;
    const uint32_t group = item - t * 2 * qp.kv_groups;
    const bool values = group >= qp.kv_groups;
    const uint32_t h = (values ? group - qp.kv_groups : group) * R::RPW + g;
    const bool is = h < c.Hkv;
    const uint32_t pos = p.positions[t], slot = p.slots[t];
    if (pos == G4A_NO_ROW32 || (slot >> c.page_shift) >= c.n_pages) return;
    double y[4 * E], ss = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        f32x4 x = {0, 0, 0, 0};
        if (is) x = *reinterpret_cast<const f32x4*>((values ? p.vx : p.kx) + ((size_t)t * c.Hkv + h) * DH + 4 * l + 256 * e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[4 * e + i] = x[i];
            ss += y[4 * e + i] * y[4 * e + i];
        }
    }
    ss = row_sum64<R::LPR>(ss);
    if (values || p.k_norm) {
        const double inv = 1.0 / sqrt(ss / DH + (double)p.eps);
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[4 * e + i] = y[4 * e + i] * inv * (values ? 1.0 : (double)p.k_norm[4 * l + 256 * e + i]);
    }
    const int half = p.rotary_dim / 2;
    if (!values && half) {
        for (int j = lane; j < half; j += 64) {
            double sn, cs;
            sincos((double)((float)pos * p.freq[j]), &sn, &cs);
            turn[w][j][0] = sn;
            turn[w][j][1] = cs;
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) stage[w][g][4 * l + 256 * e + i] = y[4 * e + i];
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 4 * l + 256 * e + i;
                if (d >= 2 * half) continue;
                const bool upper = d >= half;
                const int j = upper ? d - half : d;
                const double other = stage[w][g][upper ? j : j + half] * turn[w][j][0];
                y[4 * e + i] = upper ? y[4 * e + i] * turn[w][j][1] + other : y[4 * e + i] * turn[w][j][1] - other;
            }
    }
    f32x4 x[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[e][i] = (float)y[4 * e + i];
    if (values) quant_store<DH, BITS, true>(c, c.v, slot, h, l, x, is);
    else quant_store<DH, BITS, false>(c, c.k, slot, h, l, x, is);
}

template <int DH, int BITS>
__device__ __forceinline__ void paged_quant_producer(const G4aPagedQuantProducerParams& qp) {
    if (blockIdx.x < qp.q_wgs) paged_producer<DH, float>(qp.p);
    else paged_produce_kv<DH, BITS>(qp);
}

}  // namespace

#define G4A_PAGED_ROWS(dh, type, bits)                                                                             \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_write_d##dh##_##type(G4aPagedRowsParams p) {       \
        if (blockIdx.y) paged_write<dh, bits, true>(p);                                                            \
        else paged_write<dh, bits, false>(p);                                                                      \
    }                                                                                                              \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_read_d##dh##_##type(G4aPagedRowsParams p) {        \
        if (blockIdx.y) paged_read<dh, bits, true>(p);                                                             \
        else paged_read<dh, bits, false>(p);                                                                       \
    }
#define G4A_PAGED_QUANT(dh, type, bits)                                                                            \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_producer_d##dh##_##type(                           \
        G4aPagedQuantProducerParams p) { paged_quant_producer<dh, bits>(p); }
#define G4A_PAGED_ROW_TYPES(dh)                                                                                    \
    G4A_PAGED_ROWS(dh, f32, 32) G4A_PAGED_ROWS(dh, bf16, 16) G4A_PAGED_ROWS(dh, i8, 8) G4A_PAGED_ROWS(dh, i4, 4)   \
    G4A_PAGED_QUANT(dh, i8, 8) G4A_PAGED_QUANT(dh, i4, 4)
G4A_PAGED_ROW_TYPES(64) G4A_PAGED_ROW_TYPES(128) G4A_PAGED_ROW_TYPES(256) G4A_PAGED_ROW_TYPES(512)
#undef G4A_PAGED_ROW_TYPES
#undef G4A_PAGED_QUANT
#undef G4A_PAGED_ROWS
