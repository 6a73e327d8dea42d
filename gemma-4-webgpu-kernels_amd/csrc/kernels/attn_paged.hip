// Decode attention over a paged KV cache for gfx950: one query of every sequence
// over its visible tokens len - window <= t < len (window 0: all of them),
//   out[b, h] = sum_t softmax_t(cap(scale * q[b, h] . K[t])) V[t],
// cap(s) = softcap * tanh(s / softcap) where set; zeros without a visible token.
// Layout: G4aPaged (g4a_params.h); lengths and tables are read on the device, so a
// captured call replays with whatever they hold.
//
// Work. A unit is a sequence and up to 16 query heads of one kv head; its keys are
// tiles of 16 tokens, which lie on one page. The tiles of all units in order are
// dealt in equal runs to the launch's workgroups, whatever the lengths are: each
// workgroup finds its run from the lengths itself. A run's part of a unit is a
// segment; a segment that is its whole unit writes the output, any other a partial
// (O, m, l), which paged_combine merges.
//
// A workgroup is 4 waves, each on every fourth tile of the segment, with K and V of
// the next tile in flight in registers (16-byte loads; no LDS in between):
//   scores: K is the B operand of 16x16 MFMAs as it is loaded (lane = key l % 16 and
//           a quarter of the dims), the query rows A, out of LDS: f32 pages on
//           v_mfma_f32_16x16x4_f32, bf16 pages on v_mfma_f32_16x16x32_bf16 with the
//           query as three bf16 parts, whose sum it is exactly;
//   softmax: running maximum and sum in f32, a row of lanes per 4 heads;
//   P.V:    v_mfma_f32_4x4x1_16b_f32, in f32: V is B as it is loaded (a lane's dims are
//           columns of its block), P is A, one key of it broadcast to all blocks by the
//           instruction; bf16 values become f32 by a shift.
// The waves' partials join through LDS at the segment's end.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

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
    static constexpr int NM = BF ? (NHQ == 1 ? 1 : NHQ == 2 ? 2 : 3) : 1;  // MFMAs per K load's dims (bf16)
    static constexpr int QS = BF ? KC * NM * 64 : KC * 4 * HR;  // 16-byte query blocks in LDS
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

__device__ __forceinline__ uint32_t wave_incl_sum(uint32_t x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t u = __shfl_up(x, d);
        if (lane >= d) x += u;
    }
    return x;
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

template <int DH, typename KV, int NHQ>
__device__ __forceinline__ void paged_decode(const G4aPagedAttnParams& p) {
    using C = PagedCfg<DH, KV, NHQ>;
    constexpr bool BF = C::BF;
    constexpr int HR = C::HR, EL = C::EL, LG = C::LG, LPK = C::LPK, KI = C::KI, NDG = C::NDG, KC = C::KC, NM = C::NM;
    __shared__ __attribute__((aligned(16))) char smem[C::SM];
    __shared__ __attribute__((aligned(16))) float p_s[4][NHQ * 64];
    __shared__ float m_s[4][HR], l_s[4][HR], f_s[4][HR];
    u32x4* const qs = reinterpret_cast<u32x4*>(smem);
    f4v* const mrg = reinterpret_cast<f4v*>(smem);
    const G4aPaged& c = p.c;
    const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, key = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    // ---- this workgroup's run: every wave sums the lengths, 64 spans of `each` sequences ----
    const uint32_t n = c.n_seqs, each = (n + 63) / 64;
    auto tiles_of = [&](uint32_t b) { return b < n ? paged_span(p, c.len[b]).n * p.units : 0u; };
    uint32_t mine = 0;
    for (uint32_t i = 0; i < each; ++i) {
        const uint32_t t = tiles_of(lane * each + i);
        if (blockIdx.x == 0 && w == 0 && lane * each + i < n) p.offs[1 + lane * each + i] = mine;
        mine += t;
    }
    const uint32_t upto = wave_incl_sum(mine);
    const uint32_t total = __builtin_amdgcn_readlane(upto, 63);
    const uint32_t quota = max((total + gridDim.x - 1) / gridDim.x, p.min_run);
    if (blockIdx.x == 0 && w == 0) {  // where each sequence's tiles start, for the merge
        if (lane == 0) p.offs[0] = quota;
        for (uint32_t i = 0; i < each; ++i)
            if (lane * each + i < n) p.offs[1 + lane * each + i] += upto - mine;
    }
    uint32_t at = blockIdx.x * quota;
    if (at >= total) return;
    const uint32_t end = min(at + quota, total);
    // the sequence `at` falls into, and where its tiles start
    uint32_t b, base;
    {
        const int l0 = __builtin_ctzll(__ballot(upto > at));
        b = l0 * each;
        base = __builtin_amdgcn_readlane(upto - mine, l0);
        if (each > 1) {
            const uint32_t last = min(b + each, n);
            for (;;) {
                const uint32_t t = b + lane < last ? tiles_of(b + lane) : 0u;
                const uint32_t u = wave_incl_sum(t);
                const uint64_t hit = __ballot(base + u > at);
                if (hit) {
                    const int l1 = __builtin_ctzll(hit);
                    base += __builtin_amdgcn_readlane(u - t, l1);
                    b += l1;
                    break;
                }
                base += __builtin_amdgcn_readlane(u, 63);
                b += 64;
            }
        }
    }

    const size_t row_bytes = (size_t)c.Hkv * DH * sizeof(KV);
    const uint32_t koff = (uint32_t)(key * row_bytes) + 16 * g4;
    const uint32_t voff = (uint32_t)((lane / LG) * KI * row_bytes) + 16 * (lane % LG);
    uint32_t nseg = 0;
    PagedSpan sp = paged_span(p, c.len[b]);

    while (at < end) {
        // ---- the segment: tiles [s, e) of unit j of sequence b ----
        while (at - base >= sp.n * p.units) {  // (also steps over sequences without tokens)
            base += sp.n * p.units;
            sp = paged_span(p, c.len[++b]);
        }
        const uint32_t j = (at - base) / sp.n, s = at - base - j * sp.n, e = min(sp.n, s + end - at);
        const uint32_t kvh = j / p.chunks, hc = j - kvh * p.chunks;
        const uint32_t h0 = kvh * p.group + hc * HR, nh = min((uint32_t)HR, p.group - hc * HR);
        const uint32_t* const table = c.table + (size_t)b * c.per_seq;
        auto page_of = [&](uint32_t t) {
            const uint32_t no = (sp.first + t) >> (c.page_shift - 4);
            return table[c.ring ? no % c.per_seq : no];
        };
        auto tile_base = [&](const void* pool, uint32_t page, uint32_t t) {
            const uint32_t r = ((sp.first + t) * 16) & ((1u << c.page_shift) - 1);
            return reinterpret_cast<const char*>(pool) +
                   ((size_t)(page < c.n_pages ? page : 0u) * c.page_stride + ((size_t)r * c.Hkv + kvh) * DH) * sizeof(KV);
        };
        u32x4 k[KC], v[KI * LPK];
        auto load_k = [&](const char* kb) {
#pragma unroll
            for (int i = 0; i < KC; ++i) k[i] = *reinterpret_cast<const u32x4*>(kb + koff + 64 * i);
        };
        auto load_v = [&](const char* vb) {
#pragma unroll
            for (int i = 0; i < KI; ++i)
#pragma unroll
                for (int x = 0; x < LPK; ++x)
                    v[i * LPK + x] = *reinterpret_cast<const u32x4*>(vb + i * row_bytes + voff + 1024 * x);
        };
        uint32_t t = s + w;
        uint32_t page = t < e ? page_of(t) : 0u, page_next = t + 4 < e ? page_of(t + 4) : 0u;
        if (t < e) {
            load_k(tile_base(c.k, page, t));
            load_v(tile_base(c.v, page, t));
        }

        // ---- the query rows into LDS, in the MFMAs' order ----
        const float* const q = p.q + ((size_t)b * p.Hq + h0) * DH;
        __syncthreads();  // the segment before has read its accumulators
        for (int i = tid; i < C::QS; i += 256) {
            if constexpr (BF) {
                // block i: K load i / (64 NM), MFMA (i / 64) % NM, lane i % 64: a row of 8 dims
                const int m = (i / 64) % NM, row = i & 15, d = 32 * (i / (64 * NM)) + 8 * ((i >> 4) & 3);
                const int part = NHQ == 4 ? m : NHQ == 2 ? (m == 0 ? row / 8 : 2) : row / 4, h = row % HR;
                bf16x8 x;
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    float f = h < (int)nh && part < 3 ? q[(size_t)h * DH + d + y] : 0.0f;
                    if (part > 0) f -= (float)(__bf16)f;
                    if (part > 1) f -= (float)(__bf16)f;
                    x[y] = (__bf16)f;
                }
                qs[i] = __builtin_bit_cast(u32x4, x);
            } else {
                const int h = i % HR, d = 4 * (i / HR);
                qs[i] = h < (int)nh ? *reinterpret_cast<const u32x4*>(q + (size_t)h * DH + d) : u32x4{0, 0, 0, 0};
            }
        }
        __syncthreads();

        // lane (g4, key): heads 4 * (g4 % NHQ) + r of the tile's key
        float m[4], l[4];
        f4v acc[NHQ][NDG];
#pragma unroll
        for (int r = 0; r < 4; ++r) m[r] = G4A_NEG_INF, l[r] = 0.0f;
#pragma unroll
        for (int hq = 0; hq < NHQ; ++hq)
#pragma unroll
            for (int d = 0; d < NDG; ++d) acc[hq][d] = f4v{0.0f, 0.0f, 0.0f, 0.0f};

        for (; t < e; t += 4) {
            const bool more = t + 4 < e;
            const uint32_t page_after = t + 8 < e ? page_of(t + 8) : 0u;
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
                            __builtin_bit_cast(bf16x8, qs[(i * NM + y) * 64 + lane]), __builtin_bit_cast(bf16x8, k[i]), d[y],
                            0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (NHQ == 4) {
                        x[r] = (d[2][r] + d[1][r]) + d[0][r];
                    } else if constexpr (NHQ == 2) {
                        const float2 y = g4a_pair32(d[0][r]);  // the first and second parts
                        x[r] = (d[1][r] + y.y) + y.x;
                    } else {
                        x[r] = g4a_col_sum4(d[0][r]);
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
            if (more) load_k(tile_base(c.k, page_next, t + 4));

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
            if (more) load_v(tile_base(c.v, page_next, t + 4));
            page = page_next;
            page_next = page_after;
        }

        // ---- the waves' partials, through LDS ----
#pragma unroll
        for (int r = 0; r < 4; ++r) l[r] = g4a_row_sum16(l[r]);
        if (key == 0 && g4 < NHQ)
#pragma unroll
            for (int r = 0; r < 4; ++r) m_s[w][4 * g4 + r] = m[r], l_s[w][4 * g4 + r] = l[r];
        __syncthreads();  // every wave is done with the query rows, where the accumulators go
#pragma unroll
        for (int hq = 0; hq < NHQ; ++hq)
#pragma unroll
            for (int d = 0; d < NDG; ++d) mrg[((w * NHQ + hq) * NDG + d) * 64 + lane] = acc[hq][d];
        const bool whole = s == 0 && e == sp.n;
        const uint32_t slot = 2 * blockIdx.x + (nseg ? 1u : 0u);
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
                float* const ml = p.part_ml + ((size_t)slot * HR + tid) * 2;
                ml[0] = M;
                ml[1] = L;
            }
        }
        __syncthreads();
        f4v* const part = reinterpret_cast<f4v*>(p.part) + (size_t)slot * C::ITEMS;
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
                part[i] = o;
            }
        }
        at += e - s;
        ++nseg;
    }
}

// Merges the partials of units that more than one workgroup worked on, and writes the
// zeros of sequences without tokens. A block takes CI items (4 heads, one dim) of a
// unit; CG groups of threads take every CG-th partial each and join through LDS.
constexpr int CI = 16, CG = 16;

template <int DH, typename KV, int NHQ>
__device__ __forceinline__ void paged_combine(const G4aPagedAttnParams& p) {
    using C = PagedCfg<DH, KV, NHQ>;
    __shared__ f4v o_s[CG][CI];
    __shared__ f4v l_s[CG];
    const uint32_t u = blockIdx.x / (C::ITEMS / CI), b = u / p.units, j = u - b * p.units;
    const uint32_t kvh = j / p.chunks, hc = j - kvh * p.chunks;
    const uint32_t h0 = kvh * p.group + hc * C::HR, nh = min((uint32_t)C::HR, p.group - hc * C::HR);
    const PagedSpan sp = paged_span(p, p.c.len[b]);
    const int it = threadIdx.x % CI, gr = threadIdx.x / CI;
    const uint32_t item = blockIdx.x % (C::ITEMS / CI) * CI + it;
    const int hq = item / (C::NDG * C::LG), d = (item / C::LG) % C::NDG, lg = item % C::LG;
    const int dim = (d / C::EL) * C::LG * C::EL + lg * C::EL + d % C::EL;
    f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (sp.n) {
        const uint32_t quota = p.offs[0], start = p.offs[1 + b] + j * sp.n;
        const uint32_t first = start / quota, last = (start + sp.n - 1) / quota;
        if (first == last) return;
        // workgroup `first` holds it in its second slot if it began with another unit
        auto slot = [&](uint32_t wg) { return 2 * wg + (wg == first && first * quota != start ? 1u : 0u); };
        f4v M = {G4A_NEG_INF, G4A_NEG_INF, G4A_NEG_INF, G4A_NEG_INF}, L = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t wg = first; wg <= last; ++wg) {
            const float* const ml = p.part_ml + ((size_t)slot(wg) * C::HR + 4 * hq) * 2;
#pragma unroll
            for (int r = 0; r < 4; ++r) M[r] = fmaxf(M[r], ml[2 * r]);
        }
        for (uint32_t wg = first + gr; wg <= last; wg += CG) {
            const uint32_t sl = slot(wg);
            const float* const ml = p.part_ml + ((size_t)sl * C::HR + 4 * hq) * 2;
            const f4v a = reinterpret_cast<const f4v*>(p.part)[(size_t)sl * C::ITEMS + item];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float f = ml[2 * r] == G4A_NEG_INF ? 0.0f : expf(ml[2 * r] - M[r]);
                o[r] += a[r] * f;
                L[r] += ml[2 * r + 1] * f;
            }
        }
        o_s[gr][it] = o;
        if (it == 0) l_s[gr] = L;
        __syncthreads();
        if (gr) return;
        L = l_s[0];
#pragma unroll
        for (int i = 1; i < CG; ++i) {
            o += o_s[i][it];
            L += l_s[i];
        }
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
        G4aPagedAttnParams p) { paged_decode<dh, kv, nhq>(p); }                                               \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_combine_d##dh##_##type##_h##nhq(              \
        G4aPagedAttnParams p) { paged_combine<dh, kv, nhq>(p); }
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
