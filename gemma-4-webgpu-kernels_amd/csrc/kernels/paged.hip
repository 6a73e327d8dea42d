// The paged KV cache's bookkeeping for gfx950: the page map of a step, the
// attention producer that writes into pages, and the copy of cached tokens in
// order. The reference has no paged cache (its KVCache grows one buffer per
// layer, rust/src/kvcache.rs:49-62). Layout: G4aPaged (g4a_params.h).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "g4a_math.h"
#include "g4a_params.h"
#include "paged_quant.h"

namespace {

// a + b, 2^32 - 1 where that is more (an associative sum).
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// Saturating sums over the lanes up to and with this one (attn_paged.hip has the plain ones).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t add_sat_dpp(uint32_t x) {
    return add_sat(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x = add_sat_dpp<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
    x = add_sat_dpp<0x112, 0xf>(x);
    x = add_sat_dpp<0x114, 0xf>(x);
    x = add_sat_dpp<0x118, 0xf>(x);
    x = add_sat_dpp<0x142, 0xa>(x);  // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
    return add_sat_dpp<0x143, 0xc>(x);
}

// Inclusive saturating sums of two values over a workgroup of T threads; `tot` gets the
// workgroup's. Waves first, then their sums through LDS, which every wave scans again.
// One barrier: `sums` is another set of T / 64 pairs for each call between two others.
template <int T>
__device__ __forceinline__ void block_scan(uint32_t& a, uint32_t& b, uint32_t& tot_a, uint32_t& tot_b,
                                           uint32_t (*sums)[2]) {
    constexpr int W = T / 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    a = wave_scan(a);
    b = wave_scan(b);
    if (lane == 63) {
        sums[w][0] = a;
        sums[w][1] = b;
    }
    __syncthreads();
    const uint32_t wa = wave_scan(lane < W ? sums[lane][0] : 0u), wb = wave_scan(lane < W ? sums[lane][1] : 0u);
    if (w) {
        a = add_sat(a, __builtin_amdgcn_readlane(wa, w - 1));
        b = add_sat(b, __builtin_amdgcn_readlane(wb, w - 1));
    }
    tot_a = __builtin_amdgcn_readlane(wa, W - 1);
    tot_b = __builtin_amdgcn_readlane(wb, W - 1);
}

// Last i in [0, n) with start[i] <= x (start ascending, start[0] <= x).
__device__ __forceinline__ uint32_t last_at_or_before(const uint32_t* start, uint32_t n, uint32_t x) {
    uint32_t lo = 0;
    for (uint32_t step = 512; step > 0; step >>= 1)
        if (lo + step < n && start[lo + step] <= x) lo += step;
    return lo;
}

// A step's page map. With had = ceil(len / page size), capped at the table's entries,
// and need = ceil((len + add) / page size) - had, likewise capped, a sequence takes
// pages first + C - need .. first + C - 1 of the free ring, C the running sum of need:
// it goes on if C <= count or need = 0, if its tokens fit its table and its rows, and,
// packed, if the running sum of rows fits. Token i of it is row start + i at position
// len + i; the row of a page's first token also writes the table entry. Sequences that
// end put their pages at the ring's end.
//
// Every workgroup runs the scans over all sequences, T of them at a time, and writes
// its share of each chunk's rows: the scans are a microsecond of latency, less than a
// second launch. Lengths and ring state are written by workgroup 0 where they have
// buffers of their own, else by the workgroup that draws the last ticket, which is
// after every other's reads of them, in a second pass over the sequences: 512 of them and
// 65536 rows take 10.3 us in place, 6.4 with buffers of their own, 64 of one token (one
// workgroup, one pass) 4.3 and 3.8. The sums are 32 bits wide and their third scan is for
// chunks that refuse rows alone (64 sequences of one token 4.1 us a call; 4.8 with 64-bit
// sums, shuffles and three scans each).
template <int T>
__device__ __forceinline__ void page_map(const G4aPageMapParams& p) {
    __shared__ uint32_t s_start[T], s_len[T], s_had[T], s_base[T], s_added[T], s_rel[T], s_keep[T];
    __shared__ uint32_t s_sums[3][T / 64][2];
    __shared__ uint32_t s_last;
    const G4aPaged& c = p.c;
    const uint32_t tid = threadIdx.x, shift = c.page_shift, low = (1u << shift) - 1, P = c.per_seq;
    const uint32_t room = P << shift;  // (below 2^32)
    const uint32_t cap = p.free_cap, first = p.free_state[0] < cap ? p.free_state[0] : p.free_state[0] % cap;
    const uint32_t count = min(p.free_state[1], cap);
    const bool apart = p.len_out != c.len && p.state_out != p.free_state;
    auto pages = [&](uint32_t tokens) { return min((tokens >> shift) + ((tokens & low) ? 1u : 0u), P); };
    // place i of the ring behind `first`, i below 2 cap (places beyond wrap onto others)
    auto place = [&](uint32_t i) {
        i = i < cap ? i : (i - cap) % cap;
        return i < cap - first ? first + i : i - (cap - first);
    };

    // One pass over all sequences; `rows`: write this workgroup's rows and released
    // pages, `commit`: write the per-sequence outputs and the ring's state.
    auto pass = [&](bool rows, bool commit) {
        uint32_t row0 = 0, asked0 = 0;  // rows of the chunks before, and with those refused
        uint32_t need0 = 0, rel0 = 0;  // pages demanded, pages released
        uint32_t taken = 0;            // pages taken
        for (uint32_t b0 = 0; b0 < c.n_seqs; b0 += T) {
            const uint32_t b = b0 + tid;
            const bool is = b < c.n_seqs;
            const uint32_t len = is ? c.len[b] : 0u;
            const uint32_t add = is ? (p.add ? p.add[b] : 1u) : 0u;
            const bool ends = is && add == G4A_NO_ROW32;
            const uint32_t want = ends ? 0u : add;
            const uint32_t after = add_sat(len, want);
            const bool fits = (c.ring ? after < G4A_NO_ROW32 : after <= room) &&
                              (p.rows_per_seq == 0 || want <= p.rows_per_seq);
            const uint32_t had = pages(len);
            const uint32_t need = fits && want ? pages(after) - had : 0u;
            const uint32_t keep = ends && p.shared ? min(p.shared[b], had) : 0u;
            const uint32_t rel = ends ? had - keep : 0u;
            uint32_t cn = need, cr = rel, tn, tr;
            block_scan<T>(cn, cr, tn, tr, s_sums[0]);
            cn = add_sat(cn, need0);
            const bool goes = fits && (need == 0 || cn <= count);
            uint32_t rn = goes ? want : 0u, gn = goes ? need : 0u, trows, tneed;
            block_scan<T>(rn, gn, trows, tneed, s_sums[1]);
            uint32_t added = goes ? want : 0u, got = goes ? need : 0u;
            const uint32_t asked = add_sat(asked0, trows);
            if (p.rows_per_seq == 0 && asked > p.rows) {
                // some find no rows: from the first of them on, none that wants any goes
                if (add_sat(asked0, rn) > p.rows) added = got = 0u;
                rn = added;
                gn = got;
                block_scan<T>(rn, gn, trows, tneed, s_sums[2]);
            }
            const uint32_t row_end = row0 + rn;  // (at most p.rows, or, by rows_per_seq, not looked at)
            __syncthreads();  // the chunk before has been used
            s_start[tid] = row_end - added;
            s_len[tid] = len;
            s_had[tid] = had;
            s_base[tid] = taken + gn - got;
            s_added[tid] = added;
            s_rel[tid] = cr - rel;
            s_keep[tid] = keep;
            __syncthreads();
            if (commit && is) {
                if (p.added) p.added[b] = added;
                if (p.row_start) p.row_start[b] = p.rows_per_seq ? b * p.rows_per_seq : row_end - added;
                p.len_out[b] = ends ? 0u : len + added;
            }
            if (rows) {
                const uint32_t nb = min((uint32_t)T, c.n_seqs - b0);
                const uint32_t r_lo = p.rows_per_seq ? b0 * p.rows_per_seq : row0;
                const uint32_t r_hi = p.rows_per_seq ? (b0 + nb) * p.rows_per_seq : row0 + trows;
                for (uint32_t r = r_lo + blockIdx.x * T + tid; r < r_hi; r += gridDim.x * T) {
                    const uint32_t i = p.rows_per_seq == 0   ? last_at_or_before(s_start, nb, r)
                                       : p.rows_per_seq == 1 ? r - b0
                                                             : r / p.rows_per_seq - b0;
                    const uint32_t k = p.rows_per_seq ? r - (b0 + i) * p.rows_per_seq : r - s_start[i];
                    uint32_t slot = G4A_NO_ROW32, pos = G4A_NO_ROW32;
                    if (k < s_added[i]) {
                        pos = s_len[i] + k;
                        const uint32_t page_no = pos >> shift, e = c.ring ? page_no % P : page_no;
                        uint32_t* const entry = c.table + (size_t)(b0 + i) * P + e;
                        uint32_t page;
                        if (e < s_had[i]) {
                            page = *entry;
                        } else {
                            page = p.free_pages[place(s_base[i] + e - s_had[i])];
                            if ((pos & low) == 0 && page_no < P) *entry = page;
                        }
                        // a ring keeps its last tokens: the slots of earlier ones are theirs
                        const bool kept = !c.ring || add_sat(pos, room) >= s_len[i] + s_added[i];
                        if (kept && page < c.n_pages) slot = (page << shift) + (pos & low);
                    }
                    p.slots[r] = slot;
                    p.positions[r] = pos;
                }
                for (uint32_t x = blockIdx.x * T + tid; x < tr; x += gridDim.x * T) {
                    const uint32_t i = last_at_or_before(s_rel, nb, x);
                    const uint32_t page = c.table[(size_t)(b0 + i) * P + s_keep[i] + (x - s_rel[i])];
                    p.free_pages[place(add_sat(count, add_sat(rel0, x)))] = page;
                }
            }
            row0 += p.rows_per_seq ? 0u : trows;
            asked0 = asked;
            need0 = add_sat(need0, tn);
            rel0 = add_sat(rel0, tr);
            taken += tneed;
        }
        if (rows && p.rows_per_seq == 0)  // rows behind the last sequence
            for (uint32_t r = row0 + blockIdx.x * T + tid; r < p.rows; r += gridDim.x * T) {
                p.slots[r] = G4A_NO_ROW32;
                p.positions[r] = G4A_NO_ROW32;
            }
        if (commit && tid == 0) {
            if (p.row_start) p.row_start[c.n_seqs] = p.rows_per_seq ? c.n_seqs * p.rows_per_seq : row0;
            p.state_out[0] = place(taken);
            p.state_out[1] = min(add_sat(count - taken, rel0), cap);
        }
    };

    const bool alone = gridDim.x == 1;
    pass(true, alone || (apart && blockIdx.x == 0));
    if (alone || apart) return;
    __syncthreads();  // this workgroup's reads are done
    if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(p.ticket, 1u) == gridDim.x - 1 ? 1u : 0u;
        if (s_last) *p.ticket = 0u;
    }
    __syncthreads();
    if (s_last) pass(false, true);
}

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// Four values of a page's row, rounded to nearest even where the page holds bf16.
__device__ __forceinline__ void store4(float* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }
__device__ __forceinline__ void store4(__bf16* p, const f32x4& v) {
    *reinterpret_cast<bf16x4*>(p) = __builtin_convertvector(v, bf16x4);
}

// y = rope(x / sqrt(mean(x^2) + eps) * w) for the q, k and v rows of T tokens, in f32: v
// without w and rotation, q and k unnormalised where w is null. The angle is position *
// frequency, both f32, as in g4a_norm_rope; its sine and cosine are the device's, once a
// token and wave. The sum of squares is a tree over the row's lanes. K and V rows go to
// their token's slot.
//
// A row takes DH / 4 lanes (two float4 each at 512), so a wave holds 256 / DH of them at a
// time; it takes heads_per_wave rows of one token, the next rows' loads ahead of the work
// on these. Bound by HBM in long calls: 16384 tokens of 10 rows of 256 take 65 us (5.2
// TB/s read and written) with four turns a wave, 87 with one; one token 5.1 us and 3.9.
constexpr int PP_WAVES = 4;

template <int DH, typename KV>
__device__ __forceinline__ void paged_producer(const G4aPagedProducerParams& p) {
    constexpr int LPR = DH / 4 < 64 ? DH / 4 : 64;  // lanes of a row
    constexpr int E = DH / (4 * LPR), RPW = 64 / LPR;
    __shared__ __attribute__((aligned(16))) float stage[PP_WAVES][RPW][DH + 4];
    __shared__ __attribute__((aligned(16))) float2 turn[PP_WAVES][DH / 2];
    const int lane = threadIdx.x & 63, g = lane / LPR, l = lane % LPR;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const G4aPaged& c = p.c;
    const uint32_t item = blockIdx.x * PP_WAVES + w, t = item / p.groups;
    if (t >= p.T) return;
    uint32_t h = (item - t * p.groups) * p.heads_per_wave + g, h_end = min(h - g + p.heads_per_wave, p.heads);
    // (a branch each: for a choice among pointers the compiler moves the arguments to scratch memory)
    auto load4 = [&](f32x4 (&x)[E], const float* src) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = *reinterpret_cast<const f32x4*>(src + 4 * l + 256 * e);
    };
    auto load = [&](f32x4 (&x)[E], uint32_t h) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = f32x4{0, 0, 0, 0};
        if (h >= h_end) return;
        if (h < p.Hq) load4(x, p.q + ((size_t)t * p.Hq + h) * DH);
        else if (h < p.Hq + c.Hkv) load4(x, p.kx + ((size_t)t * c.Hkv + (h - p.Hq)) * DH);
        else load4(x, p.vx + ((size_t)t * c.Hkv + (h - p.Hq - c.Hkv)) * DH);
    };
    f32x4 x[E], next[E];
    load(next, h);  // (beside the token's position and slot, not behind them)
    const uint32_t pos = p.positions[t], slot = p.heads > p.Hq ? p.slots[t] : G4A_NO_ROW32;
    if (pos == G4A_NO_ROW32) return;
    if ((slot >> c.page_shift) >= c.n_pages) h_end = min(h_end, p.Hq);
    const uint32_t half = p.rotary_dim / 2;
    for (uint32_t j = lane; j < half; j += 64) {
        float sn, cs;
        sincosf((float)pos * p.freq[j], &sn, &cs);
        turn[w][j] = make_float2(sn, cs);
    }
    for (; h - g < h_end; h += RPW) {  // (lane groups past the last row work on zeros and write nothing)
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = next[e];
        load(next, h + RPW);
        const bool on_q = h < p.Hq, on_k = !on_q && h < p.Hq + c.Hkv;
        const bool norm = on_q ? p.q_norm != nullptr : on_k ? p.k_norm != nullptr : true;
        f32x4 wv[E];
#pragma unroll
        for (int e = 0; e < E; ++e) wv[e] = f32x4{1, 1, 1, 1};
        if (on_q) {
            if (p.q_norm) load4(wv, p.q_norm);
        } else if (on_k) {
            if (p.k_norm) load4(wv, p.k_norm);
        }
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            ss += (x[e].x * x[e].x + x[e].y * x[e].y) + (x[e].z * x[e].z + x[e].w * x[e].w);
        if constexpr (LPR == 64) {
            ss = g4a_wave_sum(ss);
        } else {
            ss = g4a_row_sum16(ss);
            if constexpr (LPR == 32) {
                const float2 y = g4a_pair16(ss);
                ss = y.x + y.y;
            }
        }
        const float inv = norm ? 1.0f / sqrtf(ss / (float)DH + p.eps) : 1.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = x[e] * inv * wv[e];
        if (half) {
#pragma unroll
            for (int e = 0; e < E; ++e) *reinterpret_cast<f32x4*>(&stage[w][g][4 * l + 256 * e]) = x[e];
            __builtin_amdgcn_wave_barrier();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (on_q || on_k)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const uint32_t d = 4 * l + 256 * e;
                    if (half % 4 == 0) {  // the lane's four dims are on one side of the pairs
                        if (d >= p.rotary_dim) continue;
                        const bool upper = d >= half;
                        const uint32_t j = upper ? d - half : d;
                        const f32x4 other = *reinterpret_cast<const f32x4*>(&stage[w][g][upper ? j : j + half]);
                        const f32x4 sc0 = *reinterpret_cast<const f32x4*>(&turn[w][j]),
                                    sc1 = *reinterpret_cast<const f32x4*>(&turn[w][j + 2]);
                        const f32x4 sn = {sc0.x, sc0.z, sc1.x, sc1.z}, cs = {sc0.y, sc0.w, sc1.y, sc1.w};
                        const f32x4 xc = x[e] * cs, os = other * sn;
                        x[e] = upper ? xc + os : xc - os;
                    } else {
                        auto one = [&](uint32_t d, float y) {
                            if (d >= p.rotary_dim) return y;
                            const bool upper = d >= half;
                            const uint32_t j = upper ? d - half : d;
                            const float os = stage[w][g][upper ? j : j + half] * turn[w][j].x;
                            return upper ? y * turn[w][j].y + os : y * turn[w][j].y - os;
                        };
                        x[e] = f32x4{one(d, x[e].x), one(d + 1, x[e].y), one(d + 2, x[e].z), one(d + 3, x[e].w)};
                    }
                }
            __builtin_amdgcn_wave_barrier();
        }
        if (h >= h_end) continue;
        if (on_q) {
#pragma unroll
            for (int e = 0; e < E; ++e) store4(p.q_out + ((size_t)t * p.Hq + h) * DH + 4 * l + 256 * e, x[e]);
        } else {
            const uint32_t kvh = on_k ? h - p.Hq : h - p.Hq - c.Hkv;
            const uint32_t page = slot >> c.page_shift, r = slot & ((1u << c.page_shift) - 1);
            const size_t at = (size_t)page * c.page_stride + ((size_t)r * c.Hkv + kvh) * DH + 4 * l;
            if (on_k) {
#pragma unroll
                for (int e = 0; e < E; ++e) store4(reinterpret_cast<KV*>(c.k) + at + 256 * e, x[e]);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) store4(reinterpret_cast<KV*>(c.v) + at + 256 * e, x[e]);
            }
        }
    }
}

// Tokens in order from their pages, as f32. A workgroup copies 1 << rows_shift tokens,
// which lie on one page, K (blockIdx.y 0) or V: 16 bytes written a thread and step.
// Tokens the cache does not hold are zeros.
template <typename KV>
__device__ __forceinline__ void paged_gather(const G4aPagedGatherParams& p) {
    typedef KV kv4 __attribute__((ext_vector_type(4)));
    const G4aPaged& c = p.c;
    const uint32_t t0 = ((p.pos0 >> p.rows_shift) + blockIdx.x) << p.rows_shift;  // its first token
    const uint32_t page_no = t0 >> c.page_shift;
    const uint32_t len = c.len[p.seq];
    const uint32_t e = c.ring ? page_no % c.per_seq : page_no;
    const uint32_t page = e < c.per_seq ? c.table[(size_t)p.seq * c.per_seq + e] : c.n_pages;
    const size_t width = (size_t)c.Hkv * c.Dh;
    const uint64_t room = (uint64_t)c.per_seq << c.page_shift;
    // tokens [lo, hi) are asked for, [a, b) of them held
    const uint64_t lo = max(t0, p.pos0), hi = min((uint64_t)t0 + (1u << p.rows_shift), (uint64_t)p.pos0 + p.n);
    const uint64_t b = page < c.n_pages ? max(lo, min(hi, (uint64_t)len)) : lo;
    const uint64_t a = page < c.n_pages && c.ring && len > room ? max(lo, min(b, (uint64_t)len - room)) : lo;
    float* const out = (blockIdx.y ? p.v_out : p.k_out) + (lo - p.pos0) * width;
    const KV* const src = reinterpret_cast<const KV*>(blockIdx.y ? c.v : c.k) + (size_t)page * c.page_stride +
                          (lo & ((1u << c.page_shift) - 1)) * width;
    const uint32_t n = (uint32_t)((hi - lo) * width / 4), from = (uint32_t)((a - lo) * width / 4),
                   to = (uint32_t)((b - lo) * width / 4);
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
        f32x4 x = {0, 0, 0, 0};
        if (i >= from && i < to)
            x = __builtin_convertvector(reinterpret_cast<const kv4*>(src)[i], f32x4);
        reinterpret_cast<f32x4*>(out)[i] = x;
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void g4a_page_map_t256(G4aPageMapParams p) { page_map<256>(p); }
extern "C" __global__ __launch_bounds__(1024) void g4a_page_map_t1024(G4aPageMapParams p) { page_map<1024>(p); }
#define G4A_PAGED_PRODUCER(dh)                                                                         \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_producer_d##dh##_f32(                  \
        G4aPagedProducerParams p) { paged_producer<dh, float>(p); }                                    \
    extern "C" __global__ __launch_bounds__(256) void g4a_paged_producer_d##dh##_bf16(                 \
        G4aPagedProducerParams p) { paged_producer<dh, __bf16>(p); }
G4A_PAGED_PRODUCER(64) G4A_PAGED_PRODUCER(128) G4A_PAGED_PRODUCER(256) G4A_PAGED_PRODUCER(512)
#undef G4A_PAGED_PRODUCER
extern "C" __global__ __launch_bounds__(256) void g4a_paged_gather_f32(G4aPagedGatherParams p) {
    paged_gather<float>(p);
}
extern "C" __global__ __launch_bounds__(256) void g4a_paged_gather_bf16(G4aPagedGatherParams p) {
    paged_gather<__bf16>(p);
}
