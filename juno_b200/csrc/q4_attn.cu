// Decode attention over 4-bit pages, and the weight that cached positions receive.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "bulk.cuh"
#include "cache_ops.cuh"
#include "q4_pages.cuh"
#include "ring.cuh"

namespace juno {

struct Q4AttnParams {
    CacheRows rows;  // first: the row's first split; splits of a row follow one another
    const uint8_t *pool;
    const int32_t *table;
    int max_pages_per_seq, n_pages, n_kv_heads, n_heads, layer, n_layers;
    int n_splits, chunk;  // splits of all rows; positions of one, a multiple of the page
    const float *q;
    int64_t ldq, ldo;
    float *out;
    float *part_o, *part_ml;  // [split][head][hd], [split][head][max, sum]
    float *scores;            // sequences that keep weights: [split][kv_head][chunk][G], log2 domain
    float *weights;
    int track_tokens;
    unsigned *err;
};

__device__ __forceinline__ int row_splits(const Q4AttnParams &p, int i) {
    return (i + 1 < p.rows.n ? cache_row(p.rows, i + 1).first : p.n_splits) - cache_row(p.rows, i).first;
}

constexpr int kQ4MaxGroup = 8, kQ4Warps = 4, kQ4Slots = 4;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {  // an 8 x 8 matrix of halves, a row to four lanes
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// NG words that lie together in shared memory
template <int NG>
__device__ __forceinline__ void lds_words(uint32_t (&v)[NG], uint32_t a) {
    if constexpr (NG == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
    else
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a));
}
__device__ __forceinline__ float factor_m(uint32_t f) { return __half2float(__ushort_as_half((unsigned short)f)); }
__device__ __forceinline__ float factor_d(uint32_t f) { return __uint_as_float(f & 0xffff0000u); }

// One CTA per (split, key/value head), its pages spread over four warps; each warp has a ring of kQ4Slots page blocks that bulk copies fill.  Per page
//   S = K Q   m16n8k16: the 16 positions are the rows, a group's 32 dimensions the k of two MMAs, the columns query heads.  The numbers are not converted: in
//             the low bits of a half they are the subnormal q 2^-24, in the next four 16 q 2^-24, which the query's side takes back; two ANDs
//             and half a shift make a register.  A group's result is multiplied by its step d in FP32 and the offset's part, m times the sum of the query
//             over the group, added.
//   O += V P  rows are dimensions, k the positions, columns heads; a weight is multiplied by the step of its position and group first, and the offsets' part
//             is a sum of their own per lane.  The product is scaled by a power of two that follows the largest step, so that it keeps its digits in FP16.
// Queries and weights are two FP16 limbs.  HPL = 1: up to four heads, columns 2h and 2h + 1 are the limbs of head h, and a lane has one head.  HPL = 2: up to
// eight heads, a column each, the limbs in MMAs of their own; a lane has two heads.
// Scores come out of an MMA with positions in the rows and go into the next with positions along k: movmatrix turns them.
template <int HD, int HPL>
__global__ void __launch_bounds__(kQ4Warps * 32, HPL == 1 ? 4 : 3) q4_attn_kernel(const __grid_constant__ Q4AttnParams p) {
    constexpr int NG = HD / kQ4Group, BLOCK = 20 * HD, FACT = NG * 4;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t = lane & 3;
    const int kvh = blockIdx.x % p.n_kv_heads, id = blockIdx.x / p.n_kv_heads;
    const int i = cache_find(p.rows, id), nsp = row_splits(p, i), G = p.n_heads / p.n_kv_heads, h0 = kvh * G;
    const CacheRow r = cache_row(p.rows, i);
    const int t0 = (id - r.first) * p.chunk, t1 = min(r.upto, t0 + p.chunk);
    const uint32_t ring = smem_u32(smem) + warp * kQ4Slots * BLOCK, bars = smem_u32(smem) + kQ4Warps * kQ4Slots * BLOCK + warp * kQ4Slots * 8;
    if (lane == 0) {
        for (int s = 0; s < kQ4Slots; s++) mbar_init(bars + s * 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async;" ::: "memory");
    }
    __syncwarp();
    // this warp's pages: first, first + kQ4Warps, ...; their places in the pool wait in the lanes, 32 at a time and the next 32 asked for ahead
    const int first = (t0 >> 4) + warp, end = t1 > t0 ? (t1 + 15) >> 4 : 0, n_pages = first < end ? (end - first + kQ4Warps - 1) / kQ4Warps : 0;
    const int32_t *table = p.table + (size_t)r.slot * p.max_pages_per_seq + first;
    const uint8_t *plane = p.pool + ((size_t)p.layer * p.n_pages * p.n_kv_heads + kvh) * BLOCK;
    const size_t page_bytes = (size_t)p.n_kv_heads * BLOCK;
    const uint64_t policy = l2_evict_first_policy();
    auto place = [&](int j) { return j < n_pages ? table[j * kQ4Warps] : 0; };
    int places = place(lane), places_next = place(32 + lane), issued = 0;
    auto issue = [&] {
        const int page = __shfl_sync(0xffffffffu, places, issued & 31);
        if (lane == 0) {
            const uint32_t bar = bars + issued % kQ4Slots * 8;
            mbar_expect_tx(bar, BLOCK);
            bulk_g2s(ring + issued % kQ4Slots * BLOCK, plane + page * page_bytes, BLOCK, bar, policy);
        }
        if ((++issued & 31) == 0) {
            places = places_next;
            places_next = place(issued + 32 + lane);
        }
    };
    while (issued < min(n_pages, kQ4Slots)) issue();

    // The query: lane (g8, t) has dimensions 8t .. 8t + 7 of every group of the head of column g8, as the B operand wants them.
    uint32_t qh[NG][4], ql[HPL == 2 ? NG : 1][4];
    float qsum[HPL][NG], back[HPL];  // of this lane's own heads: sums over the groups, and the scale of the scores
    {
        const int head = HPL == 1 ? g8 >> 1 : g8;
        const float *src = p.q + (size_t)i * p.ldq + (size_t)(h0 + head) * HD + 8 * t;
        const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
        const float scale = (float)(1.0 / sqrt((double)HD)) * 1.4426950408889634f;
        float y[NG][8], top = 0.f, sums[NG];
#pragma unroll
        for (int g = 0; g < NG; g++) {
            if (head >= G) {
#pragma unroll
                for (int e = 0; e < 8; e++) y[g][e] = 0.f;
            } else if (vec) {
                const float4 a = *reinterpret_cast<const float4 *>(src + g * kQ4Group), b = *reinterpret_cast<const float4 *>(src + g * kQ4Group + 4);
                y[g][0] = a.x; y[g][1] = a.y; y[g][2] = a.z; y[g][3] = a.w;
                y[g][4] = b.x; y[g][5] = b.y; y[g][6] = b.z; y[g][7] = b.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) y[g][e] = src[g * kQ4Group + e];
            }
            sums[g] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[g][e] *= scale;
                sums[g] += y[g][e];
                top = fmaxf(top, fabsf(y[g][e]));
            }
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
            for (int g = 0; g < NG; g++) sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], o);
        }
        // the largest element to 2^13 .. 2^14: the second limb then ends at 2^-25, 38 bits below it
        const int up = top > 0.f && top < INFINITY ? 13 - max(-100, min(100, ilogbf(top))) : 0;
        const float shift = scalbnf(1.f, up);
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int b = 0; b < 4; b++) {  // registers: MMA 0 (k low, k high), MMA 1 (k low, k high); k high meets 16 q
                const float s = b & 1 ? shift * 0.0625f : shift, y0 = y[g][2 * b] * s, y1 = y[g][2 * b + 1] * s;
                const uint32_t hi = pack_h2(y0, y1);
                const float2 hf = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                const uint32_t lo = pack_h2(y0 - hf.x, y1 - hf.y);
                if constexpr (HPL == 1) {
                    qh[g][b] = g8 & 1 ? lo : hi;
                } else {
                    qh[g][b] = hi;
                    ql[g][b] = lo;
                }
            }
#pragma unroll
        for (int h = 0; h < HPL; h++) {
            const int from = HPL == 1 ? 8 * t : 8 * t + 4 * h;  // a lane of the column that holds this lane's head
            back[h] = scalbnf(1.f, 24 - __shfl_sync(0xffffffffu, up, from));
#pragma unroll
            for (int g = 0; g < NG; g++) qsum[h][g] = __shfl_sync(0xffffffffu, sums[g], from);
        }
    }
    float o[NG][2][4], omin[HPL][NG], m_run[HPL], l_run[HPL], vscale = 0.f;
    uint32_t limit = 0;  // factors above this one ask for another scale
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int x = 0; x < 4; x++) o[g][0][x] = o[g][1][x] = 0.f;
#pragma unroll
    for (int h = 0; h < HPL; h++) {
        m_run[h] = -INFINITY;
        l_run[h] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; g++) omin[h][g] = 0.f;
    }
    bool failed = false;
    constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;
    for (int j = 0; j < n_pages; j++) {
        mbar_wait_bounded(bars + j % kQ4Slots * 8, (unsigned)(j / kQ4Slots) & 1u, 0, p.err, failed, kErrCacheWait);
        if (__any_sync(0xffffffffu, failed)) {
            failed = true;
            break;
        }
        const uint32_t base = ring + j % kQ4Slots * BLOCK;
        const int pos0 = (first + j * kQ4Warps) << 4;
        float s[HPL][2];  // rows g8 and g8 + 8
        {
            uint32_t k0[NG], k1[NG], f0[NG], f1[NG];
            lds_words<NG>(k0, base + lane * FACT);
            lds_words<NG>(k1, base + 32 * FACT + lane * FACT);
            lds_words<NG>(f0, base + 8 * HD + g8 * FACT);
            lds_words<NG>(f1, base + 8 * HD + (g8 + 8) * FACT);
            float off[HPL][2];
#pragma unroll
            for (int h = 0; h < HPL; h++) s[h][0] = s[h][1] = off[h][0] = off[h][1] = 0.f;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                const uint32_t x0 = k0[g] >> 8, x1 = k1[g] >> 8;
                mma_f16(c, k0[g] & kLow, k1[g] & kLow, k0[g] & kHigh, k1[g] & kHigh, qh[g][0], qh[g][1]);
                mma_f16(c, x0 & kLow, x1 & kLow, x0 & kHigh, x1 & kHigh, qh[g][2], qh[g][3]);
                const float d0 = factor_d(f0[g]), d1 = factor_d(f1[g]), m0 = factor_m(f0[g]), m1 = factor_m(f1[g]);
                if constexpr (HPL == 1) {
                    s[0][0] = fmaf(d0, c[0] + c[1], s[0][0]);
                    s[0][1] = fmaf(d1, c[2] + c[3], s[0][1]);
                } else {
                    mma_f16(c, k0[g] & kLow, k1[g] & kLow, k0[g] & kHigh, k1[g] & kHigh, ql[g][0], ql[g][1]);
                    mma_f16(c, x0 & kLow, x1 & kLow, x0 & kHigh, x1 & kHigh, ql[g][2], ql[g][3]);
#pragma unroll
                    for (int h = 0; h < HPL; h++) {
                        s[h][0] = fmaf(d0, c[h], s[h][0]);
                        s[h][1] = fmaf(d1, c[2 + h], s[h][1]);
                    }
                }
#pragma unroll
                for (int h = 0; h < HPL; h++) {
                    off[h][0] = fmaf(m0, qsum[h][g], off[h][0]);
                    off[h][1] = fmaf(m1, qsum[h][g], off[h][1]);
                }
            }
#pragma unroll
            for (int h = 0; h < HPL; h++) {
                s[h][0] = fmaf(s[h][0], back[h], off[h][0]);
                s[h][1] = fmaf(s[h][1], back[h], off[h][1]);
            }
        }
        const bool tail = pos0 + 16 > t1, on0 = pos0 + g8 < t1, on1 = pos0 + g8 + 8 < t1;
        if (p.scores) {
            float *to = p.scores + (((size_t)id * p.n_kv_heads + kvh) * p.chunk + (pos0 - t0) + g8) * G;
#pragma unroll
            for (int h = 0; h < HPL; h++) {
                const int head = HPL * t + h;
                if (head < G && on0) to[head] = s[h][0];
                if (head < G && on1) to[8 * G + head] = s[h][1];
            }
        }
        uint32_t f0[NG], f1[NG];
        lds_words<NG>(f0, base + 18 * HD + g8 * FACT);
        lds_words<NG>(f1, base + 18 * HD + (g8 + 8) * FACT);
        if (tail) {  // positions behind the end: whatever their place holds
#pragma unroll
            for (int h = 0; h < HPL; h++) {
                if (!on0) s[h][0] = -INFINITY;
                if (!on1) s[h][1] = -INFINITY;
            }
#pragma unroll
            for (int g = 0; g < NG; g++) {
                if (!on0) f0[g] = 0u;
                if (!on1) f1[g] = 0u;
            }
        }
        // a larger score than any before, or a step beyond the scale's range: seldom after the first pages
        uint32_t steps = 0;
#pragma unroll
        for (int g = 0; g < NG; g++) steps = max(steps, max(f0[g], f1[g]));
        steps &= 0xffff0000u;
        bool grown = steps > limit;
#pragma unroll
        for (int h = 0; h < HPL; h++) grown |= s[h][0] > m_run[h] || s[h][1] > m_run[h];
        if (__any_sync(0xffffffffu, grown)) {
            float fix[HPL], vfix = 1.f;
            steps = __reduce_max_sync(0xffffffffu, steps);
            if (steps > limit) {  // the largest step to 2^10 .. 2^11, up to 2^15 in range
                const int e = max((int)(steps >> 23) - 127, -100);
                const float next = scalbnf(1.f, 10 - e);
                vfix = vscale == 0.f ? 0.f : next / vscale;
                vscale = next;
                limit = (uint32_t)(e + 4 + 127) << 23 | 0x7fffffu;
            }
#pragma unroll
            for (int h = 0; h < HPL; h++) {
                float mx = fmaxf(m_run[h], fmaxf(s[h][0], s[h][1]));
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                fix[h] = m_run[h] == -INFINITY ? 0.f : exp2_fast(m_run[h] - mx);
                m_run[h] = mx;
                l_run[h] *= fix[h];
#pragma unroll
                for (int g = 0; g < NG; g++) omin[h][g] *= fix[h];
            }
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const float f = fix[HPL == 1 ? 0 : x & 1] * vfix;
                    o[g][0][x] *= f;
                    o[g][1][x] *= f;
                }
        }
        float w[HPL][2], ws[HPL][2];
#pragma unroll
        for (int h = 0; h < HPL; h++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                w[h][x] = exp2_fast(s[h][x] - m_run[h]);
                ws[h][x] = w[h][x] * vscale;
            }
            l_run[h] += w[h][0] + w[h][1];
        }
        uint32_t v0[NG], v1[NG];
        lds_words<NG>(v0, base + 10 * HD + lane * FACT);
        lds_words<NG>(v1, base + 10 * HD + 32 * FACT + lane * FACT);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const float d0 = factor_d(f0[g]), d1 = factor_d(f1[g]), m0 = factor_m(f0[g]), m1 = factor_m(f1[g]);
            float hi[HPL][2], lo[HPL][2];
#pragma unroll
            for (int h = 0; h < HPL; h++) {
                omin[h][g] = fmaf(w[h][0], m0, omin[h][g]);
                omin[h][g] = fmaf(w[h][1], m1, omin[h][g]);
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const float y = ws[h][x] * (x ? d1 : d0);
                    hi[h][x] = __uint_as_float(__float_as_uint(y) & 0xffffe000u);  // what a half holds
                    lo[h][x] = y - hi[h][x];
                }
            }
            uint32_t b0, b1;
            if constexpr (HPL == 1) {
                b0 = transpose8(pack_h2(hi[0][0], lo[0][0]));
                b1 = transpose8(pack_h2(hi[0][1], lo[0][1]));
            } else {
                b0 = transpose8(pack_h2(hi[0][0], hi[1][0]));
                b1 = transpose8(pack_h2(hi[0][1], hi[1][1]));
            }
            const uint32_t x0 = v0[g] >> 8, x1 = v1[g] >> 8;
            mma_f16(o[g][0], v0[g] & kLow, v0[g] & kHigh, v1[g] & kLow, v1[g] & kHigh, b0, b1);
            mma_f16(o[g][1], x0 & kLow, x0 & kHigh, x1 & kLow, x1 & kHigh, b0, b1);
            if constexpr (HPL == 2) {
                b0 = transpose8(pack_h2(lo[0][0], lo[1][0]));
                b1 = transpose8(pack_h2(lo[0][1], lo[1][1]));
                mma_f16(o[g][0], v0[g] & kLow, v0[g] & kHigh, v1[g] & kLow, v1[g] & kHigh, b0, b1);
                mma_f16(o[g][1], x0 & kLow, x0 & kHigh, x1 & kLow, x1 & kHigh, b0, b1);
            }
        }
        __syncwarp();  // all lanes have read the block before it is filled again
        if (issued < n_pages) issue();
    }
    if (failed)
        for (int j = ring_open(issued, 0, kQ4Slots); j < issued; j++) mbar_wait_bounded(bars + j % kQ4Slots * 8, ring_parity(j, kQ4Slots), 0, p.err, failed, kErrCacheWait);
    // sums over the lanes that share a head, then over the warps
#pragma unroll
    for (int h = 0; h < HPL; h++) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], x);
#pragma unroll
            for (int g = 0; g < NG; g++) omin[h][g] += __shfl_xor_sync(0xffffffffu, omin[h][g], x);
        }
    }
    __syncthreads();  // no copy is under way any more: the rings become the place where the warps meet
    float *mg_o = reinterpret_cast<float *>(smem), *mg_m = mg_o + kQ4Warps * G * HD, *mg_l = mg_m + kQ4Warps * G;  // [warp][head][HD], [warp][head]
    const float unscale = vscale == 0.f ? 0.f : 16777216.f / vscale;
#pragma unroll
    for (int h = 0; h < HPL; h++) {
        const int head = HPL * t + h;
        if (head >= G) continue;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float v[4];  // dimensions 4 g8 .. 4 g8 + 3 of the group
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float *c = &o[g][x >> 1][2 * (x & 1)];
                v[x] = fmaf(HPL == 1 ? c[0] + c[1] : c[h], x & 1 ? unscale * 0.0625f : unscale, omin[h][g]);
            }
            *reinterpret_cast<float4 *>(mg_o + ((size_t)warp * G + head) * HD + g * kQ4Group + 4 * g8) = make_float4(v[0], v[1], v[2], v[3]);
        }
        if (g8 == 0) {
            mg_m[warp * G + head] = m_run[h];
            mg_l[warp * G + head] = l_run[h];
        }
    }
    __syncthreads();
    for (int idx = tid; idx < G * HD; idx += kQ4Warps * 32) {
        const int g = idx / HD, d = idx - g * HD;
        float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < kQ4Warps; w++) M = fmaxf(M, mg_m[w * G + g]);
#pragma unroll
        for (int w = 0; w < kQ4Warps; w++) {
            const float lw = mg_l[w * G + g];
            if (lw == 0.f) continue;  // a warp without pages
            const float f = exp2_fast(mg_m[w * G + g] - M);
            L = fmaf(lw, f, L);
            acc = fmaf(mg_o[((size_t)w * G + g) * HD + d], f, acc);
        }
        const size_t part = (size_t)id * p.n_heads + h0 + g;
        if (nsp == 1)
            p.out[(size_t)i * p.ldo + (h0 + g) * HD + d] = t0 < t1 ? acc / L : 0.f;
        else
            p.part_o[part * HD + d] = acc;
        if (d == 0 && (nsp > 1 || p.scores)) {
            p.part_ml[part * 2] = M;
            p.part_ml[part * 2 + 1] = L;
        }
    }
}

// Blocks [0, rows * n_heads): the splits of one (row, head).  Further blocks, one per (split, kv head): the weight that the split's positions have received.
template <int HD>
__global__ void __launch_bounds__(HD) q4_merge_kernel(const Q4AttnParams p) {
    const int tid = threadIdx.x, merges = p.rows.n * p.n_heads;
    if ((int)blockIdx.x < merges) {
        const int i = blockIdx.x / p.n_heads, h = blockIdx.x - i * p.n_heads, nsp = row_splits(p, i), first = cache_row(p.rows, i).first;
        if (nsp == 1) return;
        float M = -INFINITY, L = 0.f, acc = 0.f;
        for (int s = first; s < first + nsp; s++) M = fmaxf(M, p.part_ml[((size_t)s * p.n_heads + h) * 2]);
        for (int s = first; s < first + nsp; s++) {
            const size_t part = (size_t)s * p.n_heads + h;
            const float f = exp2f(p.part_ml[part * 2] - M);
            L = fmaf(p.part_ml[part * 2 + 1], f, L);
            acc = fmaf(p.part_o[part * HD + tid], f, acc);
        }
        p.out[(size_t)i * p.ldo + h * HD + tid] = acc / L;
        return;
    }
    const int at = blockIdx.x - merges, kvh = at % p.n_kv_heads, id = at / p.n_kv_heads, G = p.n_heads / p.n_kv_heads;
    const int i = cache_find(p.rows, id), nsp = row_splits(p, i);
    const CacheRow r = cache_row(p.rows, i);
    if (r.track < 0) return;
    float M[kQ4MaxGroup], inv[kQ4MaxGroup];
#pragma unroll
    for (int g = 0; g < kQ4MaxGroup; g++) {
        if (g >= G) break;
        M[g] = -INFINITY;
        float L = 0.f;
        for (int s = r.first; s < r.first + nsp; s++) M[g] = fmaxf(M[g], p.part_ml[((size_t)s * p.n_heads + kvh * G + g) * 2]);
        for (int s = r.first; s < r.first + nsp; s++) {
            const float *ml = p.part_ml + ((size_t)s * p.n_heads + kvh * G + g) * 2;
            L = fmaf(ml[1], exp2f(ml[0] - M[g]), L);
        }
        inv[g] = 1.f / L;
    }
    const int t0 = (id - r.first) * p.chunk, t1 = min(r.upto, t0 + p.chunk);
    float *w = p.weights + (((size_t)r.track * p.n_layers + p.layer) * p.n_kv_heads + kvh) * p.track_tokens;
    for (int t = t0 + tid; t < t1; t += HD) {
        const float *s = p.scores + (((size_t)id * p.n_kv_heads + kvh) * p.chunk + (t - t0)) * G;
        float sum = 0.f;
#pragma unroll
        for (int g = 0; g < kQ4MaxGroup; g++)
            if (g < G) sum = fmaf(exp2f(s[g] - M[g]), inv[g], sum);
        w[t] += sum;
    }
}

template <int HD, int HPL>
static int launch_q4_attn(const Q4AttnParams &a, unsigned grid, cudaStream_t st) {
    constexpr int kRing = kQ4Warps * kQ4Slots * (20 * HD + 8);
    static bool set[64] = {false};  // per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!set[dev & 63]) {
        JUNO_CUDA_TRY(cudaFuncSetAttribute(q4_attn_kernel<HD, HPL>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing));
        set[dev & 63] = true;
    }
    q4_attn_kernel<HD, HPL><<<grid, kQ4Warps * 32, kRing, st>>>(a);
    JUNO_CUDA_TRY(cudaGetLastError());
    return JUNO_OK;
}

int q4_attend(juno_ctx *c, juno_kvpool *p, int layer, int n, juno_seq *const *seqs, const int32_t *lens, int n_heads, const float *q, int64_t ldq, float *out,
              int64_t ldo, WaitWord word, cudaStream_t st) {
    const int hd = p->head_dim, H = p->n_kv_heads, G = n_heads / H;
    if (G > kQ4MaxGroup) {
        set_error("attention: query/kv head ratio %d is not supported (up to %d)", G, kQ4MaxGroup);
        return JUNO_ERR_UNSUPPORTED;
    }
    std::vector<CacheRow> rows((size_t)n);
    int64_t pages = 0, bytes = 0;
    int most = 1;
    bool track = false;
    for (int i = 0; i < n; i++) {
        const int len = lens ? lens[i] : seqs[i]->len;
        rows[(size_t)i] = {seqs[i]->slot, len, 0, seqs[i]->track};
        const int pg = std::max(1, (len + kPageTokens - 1) / kPageTokens);
        pages += pg;
        most = std::max(most, pg);
        track |= seqs[i]->track >= 0;
        bytes += len;
    }
    // enough splits for a few CTAs on every SM, none of them below 128 positions
    const int64_t target = (int64_t)c->sm_count * 8;
    int chunk = (int)std::max<int64_t>(8, (pages * H + target - 1) / target);
    chunk = std::max(chunk, (most + 63) / 64);
    int64_t splits = 0;
    for (auto &r : rows) {
        r.first = (int)splits;
        splits += std::max(1, (r.upto + chunk * kPageTokens - 1) / (chunk * kPageTokens));
    }
    Q4AttnParams a;
    auto padded = [](size_t b) { return (b + 255) & ~(size_t)255; };
    const size_t far_b = cache_rows_bytes(n), ml_b = padded((size_t)splits * n_heads * 8), o_b = splits > n ? padded((size_t)splits * n_heads * hd * 4) : 0,
                 s_b = track ? (size_t)splits * n_heads * chunk * kPageTokens * 4 : 0;
    uint8_t *scratch = nullptr;
    JUNO_TRY(cache_scratch(c, far_b + ml_b + o_b + s_b, &scratch));
    JUNO_TRY(cache_rows(c, rows.data(), n, reinterpret_cast<CacheRow *>(scratch), &a.rows, st));
    a.pool = static_cast<const uint8_t *>(p->k);
    a.table = p->d_table;
    a.max_pages_per_seq = p->max_pages_per_seq;
    a.n_pages = p->n_pages;
    a.n_kv_heads = H;
    a.n_heads = n_heads;
    a.layer = layer;
    a.n_layers = p->n_layers;
    a.n_splits = (int)splits;
    a.chunk = chunk * kPageTokens;
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.part_ml = reinterpret_cast<float *>(scratch + far_b);
    a.part_o = reinterpret_cast<float *>(scratch + far_b + ml_b);
    a.scores = track ? reinterpret_cast<float *>(scratch + far_b + ml_b + o_b) : nullptr;
    a.weights = p->weights;
    a.track_tokens = p->track_tokens;
    a.err = c->gemv_scratch.qerr + word;
    ProfScope prof(c, st, PROF_ATTN, (double)bytes * H * p->row_bytes());
    const unsigned grid = (unsigned)(splits * H);
    if (hd == 128)
        JUNO_TRY(G <= 4 ? (launch_q4_attn<128, 1>(a, grid, st)) : (launch_q4_attn<128, 2>(a, grid, st)));
    else
        JUNO_TRY(G <= 4 ? (launch_q4_attn<64, 1>(a, grid, st)) : (launch_q4_attn<64, 2>(a, grid, st)));
    c->kernel_launches++;
    if (splits == n && !track) return JUNO_OK;
    const unsigned merge = (unsigned)(n * n_heads + (track ? splits * H : 0));
    if (hd == 128)
        q4_merge_kernel<128><<<merge, 128, 0, st>>>(a);
    else
        q4_merge_kernel<64><<<merge, 64, 0, st>>>(a);
    JUNO_CUDA_TRY(cudaGetLastError());
    c->kernel_launches++;
    return JUNO_OK;
}

}  // namespace juno

using namespace juno;

extern "C" int juno_attn_decode_device(juno_ctx *c, juno_kvpool *p, int32_t layer, int32_t n, juno_seq *const *seqs, const int32_t *lens, int32_t n_heads,
                                       const float *q_dev, int64_t ldq, float *out_dev, int64_t ldo, void *stream) {
    return guarded([&]() -> int {
        JUNO_TRY(ctx_check(c));
        std::lock_guard<std::recursive_mutex> lk(c->mu);
        JUNO_TRY(cache_call_check(c, p, layer, n, seqs));
        if (p->dtype != kKvQ4) {
            set_error("this entry point serves 4-bit pages; juno_attn_decode and juno_attn_decode_static serve the others");
            return JUNO_ERR_UNSUPPORTED;
        }
        JUNO_REQUIRE(n_heads > 0 && n_heads % p->n_kv_heads == 0, "n_heads %d is not a multiple of n_kv_heads %d", n_heads, p->n_kv_heads);
        JUNO_REQUIRE(ldq >= (int64_t)n_heads * p->head_dim && ldo >= (int64_t)n_heads * p->head_dim, "rows of %lld and %lld elements hold no %d heads of %d",
                     (long long)ldq, (long long)ldo, n_heads, p->head_dim);
        bool track = false;
        for (int i = 0; i < n; i++) {
            JUNO_REQUIRE(!lens || (lens[i] >= 0 && lens[i] <= seqs[i]->len), "sequence %d has %d cached positions, not %d", i, seqs[i]->len, lens ? lens[i] : 0);
            track |= seqs[i]->track >= 0;
        }
        DeviceGuard g(c->device);
        if (track) JUNO_TRY(cache_call_distinct(p, n, seqs));
        JUNO_TRY(device_memory(c, q_dev, "q"));
        JUNO_TRY(device_memory(c, out_dev, "out"));
        CacheStream s(c, stream);
        JUNO_TRY(s.status);
        return q4_attend(c, p, layer, n, seqs, lens, n_heads, q_dev, ldq, out_dev, ldo, WAIT_ENQUEUED, s.st);
    });
}
