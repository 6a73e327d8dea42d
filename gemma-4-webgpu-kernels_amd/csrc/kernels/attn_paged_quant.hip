// Decode attention over pages of 8 and 4 bits for gfx950: as attn_paged.hip, whose
// division of the work and merge these kernels share, on the whole numbers and
// scales of paged_quant.h.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "g4a_math.h"
#include "g4a_params.h"
#include "paged_quant.h"

namespace {

template <int DH, int BITS, int NHQ>
struct QuantCfg {
    static constexpr int DIMS = DH;
    static constexpr int HR = 4 * NHQ;                                // query heads of a unit
    static constexpr int EV = DH / 16 < 32 / (BITS / 4) ? DH / 16 : 32 / (BITS / 4);  // dims of a lane and block
    static constexpr int NA = DH / 16;                                // accumulators of a lane, of 16 rows
    static constexpr int ITEMS = NHQ * DH;                            // (4 heads, dim) of a partial
    // Items in the accumulators' order: 4 heads hq, accumulator a, lane n of 16.
    static __device__ __forceinline__ int hq(int item) { return item / DH; }
    static __device__ __forceinline__ int dim(int item) {
        const int n = item % 16, a = item / 16 % NA;
        return a / EV * 16 * EV + n * EV + a % EV;
    }
};

// The simple form: a tile at a time by all four waves, 16 lanes a token for the scores, a dim a thread for P.V.
template <int DH, int BITS, int NHQ>
__device__ __forceinline__ void paged_decode_quant(const G4aPagedAttnParams& p) {
    using C = QuantCfg<DH, BITS, NHQ>;
    using Q = QuantRow<DH, BITS>;
    constexpr int HR = C::HR, D = (DH + 255) / 256;
    __shared__ uint32_t lens[PAGED_SEQS];
    __shared__ float q_s[HR][DH], s_s[HR][16], c_s[HR], m_s[HR], l_s[HR];
    const G4aPaged& c = p.c;
    const int tid = threadIdx.x, key = tid / 16, i16 = tid % 16;
    PagedPart x;
    if (!paged_find<HR>(p, lens, tid & 63, __builtin_amdgcn_readfirstlane(tid >> 6), x)) return;
    if (x.sp.n == 0) {
        for (uint32_t i = tid; i < x.nh * DH; i += 256) p.out[((size_t)x.b * p.Hq + x.h0) * DH + i] = 0.0f;
        return;
    }
    for (int i = tid; i < HR * DH; i += 256)
        q_s[i / DH][i % DH] = i / DH < (int)x.nh ? p.q[((size_t)x.b * p.Hq + x.h0) * DH + i] : 0.0f;
    if (tid < HR) m_s[tid] = G4A_NEG_INF, l_s[tid] = 0.0f;
    float acc[HR][D] = {};
    auto value = [&](const void* pool, uint32_t page, uint32_t r, int d, bool values) {
        const uint8_t* const row = static_cast<const uint8_t*>(pool) + Q::row_at(c, page, x.kvh, r);
        const uint8_t* const meta = static_cast<const uint8_t*>(pool) + Q::meta_at(c, page, x.kvh, r);
        const float s = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(meta + 16 * Q::G + 2 * (r % 16)) << 16);
        if constexpr (BITS == 8) return ((float)row[d] - 128.0f) * s;
        const int sub = (int)meta[values ? Q::template sub_at<true>(d / 32, r) : Q::template sub_at<false>(d / 32, r)] - 128;
        return (float)(((int)(row[d / 2] >> (4 * (d % 2)) & 15) - 8) * sub) * s;
    };
    for (uint32_t t = x.from; t < x.to; ++t) {
        const uint32_t t0 = (x.sp.first + t) * 16, no = t0 >> c.page_shift;
        const uint32_t page = c.table[(size_t)x.b * c.per_seq + (c.ring ? no % c.per_seq : no)];
        if (page >= c.n_pages) continue;
        const uint32_t r0 = t0 & ((1u << c.page_shift) - 1);
        const uint32_t lo = x.sp.lo > t0 ? x.sp.lo - t0 : 0u, hi = min(16u, x.sp.len - t0);
        __syncthreads();  // the queries, or the tile before
        const bool seen = key >= (int)lo && key < (int)hi;
        float k[DH / 16];
        for (int d = 0; d < DH / 16; ++d) k[d] = value(c.k, page, r0 + key, i16 + 16 * d, false);
        for (int h = 0; h < HR; ++h) {
            float s = 0.0f;
            for (int d = 0; d < DH / 16; ++d) s += q_s[h][i16 + 16 * d] * k[d];
            s = g4a_row_sum16(s) * p.scale;
            if (p.softcap > 0.0f) s = p.softcap * tanhf(s / p.softcap);
            if (i16 == 0) s_s[h][key] = seen ? s : G4A_NEG_INF;
        }
        __syncthreads();
        if (tid < HR) {
            float m = m_s[tid], l = 0.0f;
            for (int i = 0; i < 16; ++i) m = fmaxf(m, s_s[tid][i]);
            const float corr = m_s[tid] == G4A_NEG_INF ? 0.0f : expf(m_s[tid] - m);
            for (int i = 0; i < 16; ++i) {
                const float e = s_s[tid][i] == G4A_NEG_INF ? 0.0f : expf(s_s[tid][i] - m);
                s_s[tid][i] = e;
                l += e;
            }
            c_s[tid] = corr;
            m_s[tid] = m;
            l_s[tid] = l_s[tid] * corr + l;
        }
        __syncthreads();
        for (int d = 0; d < D; ++d) {
            const int dim = tid + 256 * d;
            if (dim >= DH) continue;
            for (int h = 0; h < HR; ++h) acc[h][d] *= c_s[h];
            for (uint32_t i = lo; i < hi; ++i) {
                const float v = value(c.v, page, r0 + i, dim, true);
                for (int h = 0; h < HR; ++h) acc[h][d] += s_s[h][i] * v;
            }
        }
    }
    __syncthreads();
    const uint32_t at = blockIdx.x;
    const bool whole = x.parts == 1;
    for (int d = 0; d < D; ++d) {
        const int dim = tid + 256 * d;
        if (dim >= DH) continue;
        for (int h = 0; h < HR; ++h) {
            const float l = l_s[h];
            if (!whole) {
                const int n = dim % (16 * C::EV) / C::EV, a = dim / (16 * C::EV) * C::EV + dim % C::EV;
                p.part[((size_t)at * C::ITEMS + h / 4 * DH + a * 16 + n) * 4 + h % 4] = acc[h][d];
            } else if (h < (int)x.nh) {
                p.out[((size_t)x.b * p.Hq + x.h0 + h) * DH + dim] = l != 0.0f ? acc[h][d] / l : 0.0f;
            }
        }
    }
    if (!whole && tid < HR) {
        p.part_ml[(size_t)at * 2 * HR + tid] = m_s[tid];
        p.part_ml[(size_t)at * 2 * HR + HR + tid] = l_s[tid];
    }
}

}  // namespace

#define G4A_PAGED_QUANT_DECODE(dh, type, bits, nhq)                                                           \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_decode_d##dh##_##type##_h##nhq(               \
        G4aPagedAttnParams p) { paged_decode_quant<dh, bits, nhq>(p); }                                       \
    extern "C" __global__ __launch_bounds__(512) void g4a_paged_combine16_d##dh##_##type##_h##nhq(            \
        G4aPagedAttnParams p) { paged_combine<QuantCfg<dh, bits, nhq>, 16, 8>(p); }                           \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_combine64_d##dh##_##type##_h##nhq(            \
        G4aPagedAttnParams p) { paged_combine<QuantCfg<dh, bits, nhq>, 64, 4>(p); }
#define G4A_PAGED_QUANT_TYPES(dh, nhq) G4A_PAGED_QUANT_DECODE(dh, i8, 8, nhq) G4A_PAGED_QUANT_DECODE(dh, i4, 4, nhq)
G4A_PAGED_QUANT_TYPES(64, 1) G4A_PAGED_QUANT_TYPES(64, 2) G4A_PAGED_QUANT_TYPES(64, 4)
G4A_PAGED_QUANT_TYPES(128, 1) G4A_PAGED_QUANT_TYPES(128, 2) G4A_PAGED_QUANT_TYPES(128, 4)
G4A_PAGED_QUANT_TYPES(256, 1) G4A_PAGED_QUANT_TYPES(256, 2) G4A_PAGED_QUANT_TYPES(256, 4)
G4A_PAGED_QUANT_TYPES(512, 1) G4A_PAGED_QUANT_TYPES(512, 2) G4A_PAGED_QUANT_TYPES(512, 4)
#undef G4A_PAGED_QUANT_TYPES
#undef G4A_PAGED_QUANT_DECODE
