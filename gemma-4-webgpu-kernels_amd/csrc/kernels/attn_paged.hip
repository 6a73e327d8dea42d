// Decode attention over a paged KV cache for gfx950: one query of every sequence
// over its visible tokens len - window <= t < len (window 0: all of them),
//   out[b, h] = sum_t softmax_t(cap(scale * q[b, h] . K[t])) V[t],
// cap(s) = softcap * tanh(s / softcap) where set; zeros without a visible token.
// Layout: G4aPaged (g4a_params.h); lengths and tables are read on the device, so a
// captured call replays with whatever they hold.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "g4a_math.h"
#include "g4a_params.h"

namespace {

// The simple form: a workgroup per (sequence, query head), a wave per key, lane l
// holding dims l, l + 64, ...; running maximum and sum; the waves join through LDS.
template <int DH, typename KV>
__device__ __forceinline__ void paged_decode(const G4aPagedAttnParams& p) {
    constexpr int E = DH / 64;
    __shared__ float acc_s[4][DH], m_s[4], l_s[4];
    const G4aPaged& c = p.c;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint32_t b = blockIdx.x, h = blockIdx.y, kvh = h / (p.Hq / c.Hkv);
    const uint64_t room = (uint64_t)c.per_seq << c.page_shift;
    const uint32_t len = c.ring ? c.len[b] : (uint32_t)min((uint64_t)c.len[b], room);
    const uint32_t span = (uint32_t)min(room, (uint64_t)(p.window ? p.window : G4A_NO_ROW32));
    const uint32_t t0 = len > span ? len - span : 0u;
    float q[E], acc[E] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = p.q[((size_t)b * p.Hq + h) * DH + 64 * e + lane];
    float m = G4A_NEG_INF, l = 0.0f;
    for (uint64_t t = (uint64_t)t0 + w; t < len; t += 4) {
        const uint32_t page_no = (uint32_t)t >> c.page_shift;
        const uint32_t page = c.table[(size_t)b * c.per_seq + (c.ring ? page_no % c.per_seq : page_no)];
        if (page >= c.n_pages) continue;
        const size_t at = (size_t)page * c.page_stride +
                          ((size_t)(t & ((1u << c.page_shift) - 1)) * c.Hkv + kvh) * DH + lane;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += q[e] * (float)reinterpret_cast<const KV*>(c.k)[at + 64 * e];
        s = g4a_wave_sum(s) * p.scale;
        if (p.softcap > 0.0f) s = p.softcap * tanhf(s / p.softcap);
        const float mn = fmaxf(m, s), corr = m == G4A_NEG_INF ? 0.0f : expf(m - mn), pr = s == G4A_NEG_INF ? 0.0f : expf(s - mn);
        l = l * corr + pr;
        m = mn;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * corr + pr * (float)reinterpret_cast<const KV*>(c.v)[at + 64 * e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) acc_s[w][64 * e + lane] = acc[e];
    if (lane == 0) m_s[w] = m, l_s[w] = l;
    __syncthreads();
    float M = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3])), L = 0.0f, f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = m_s[i] == G4A_NEG_INF ? 0.0f : expf(m_s[i] - M);
        L += l_s[i] * f[i];
    }
    for (int d = threadIdx.x; d < DH; d += 256) {
        float o = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o += acc_s[i][d] * f[i];
        p.out[((size_t)b * p.Hq + h) * DH + d] = L > 0.0f ? o / L : 0.0f;
    }
}

}  // namespace

#define G4A_PAGED_DECODE(dh)                                                                            \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_decode_d##dh##_f32(G4aPagedAttnParams p) { \
        paged_decode<dh, float>(p);                                                                     \
    }                                                                                                   \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_decode_d##dh##_bf16(G4aPagedAttnParams p) { \
        paged_decode<dh, __bf16>(p);                                                                    \
    }
G4A_PAGED_DECODE(64) G4A_PAGED_DECODE(128) G4A_PAGED_DECODE(256) G4A_PAGED_DECODE(512)
#undef G4A_PAGED_DECODE
