// Decode attention over 4-bit pages, and the weight that cached positions receive.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "bulk.cuh"
#include "cache_ops.cuh"
#include "q4_pages.cuh"
#include "ring.cuh"

namespace juno {

// The pages of all rows follow one another (a row without positions counts as one page) and are cut into shares; a CTA takes one share of one key/value
// head, which may hold the end of a row, whole ones and the beginning of another.  What a share has of a row is a part: its number, row + share, is different
// for each (along the cut, each part has a later row or share than the one before), and a row's parts follow one another.
constexpr int kInlineCuts = 160;
struct Q4AttnParams {
    CacheRows rows;  // first: the row's first page among those of all rows; share: the share that has it
    const int32_t *far_cuts;  // null: `cuts`
    int cuts[kInlineCuts];    // share w has the pages [cuts[w], cuts[w + 1])
    const uint8_t *pool;
    const int32_t *table;
    int max_pages_per_seq, n_pages, n_kv_heads, n_heads, layer, n_layers;
    int total, shares;  // pages of all rows
    const float *q;
    int64_t ldq, ldo;
    float *out;
    float *part_o, *part_ml;  // [part][head][hd], [part][head][max, sum]
    float2 *sums;             // sequences that keep weights: [row][head] largest score of all, 1 / sum
    unsigned *arrived;        // [row][kv_head]: parts that are done, zero between launches
    unsigned long long *gave_up, call;  // sequences that keep weights: the last call that gave up a wait; the number of this one
    float *scores;            // sequences that keep weights: [kv_head][position of all rows' pages][G], log2 domain
    float *weights;
    int track_tokens;
    unsigned *err;
};

__device__ __forceinline__ int row_end(const Q4AttnParams &p, int i) { return i + 1 < p.rows.n ? cache_row(p.rows, i + 1).first : p.total; }
__device__ __forceinline__ int cut_at(const Q4AttnParams &p, int w) { return p.far_cuts ? p.far_cuts[w] : p.cuts[w]; }
// How many parts row i has: up to the share that the next row begins in, which has some of this one unless it begins with that one.
__device__ __forceinline__ int row_parts(const Q4AttnParams &p, int i, const CacheRow &r) {
    if (i + 1 >= p.rows.n) return p.shares - r.share;
    const CacheRow next = cache_row(p.rows, i + 1);
    return next.share - r.share + (cut_at(p, next.share) < next.first);
}

constexpr int kQ4MaxGroup = 8, kQ4Slots = 2, kQ4Tile = 2;  // pages of a tile: a warp's step
// Warps of a CTA and CTAs on an SM: 16 warps of 128 registers, 12 of 168 for more than four heads of 128, whose sums need them (48 requests of 8192 positions with
// eight heads a key/value head: 118 us; 16 warps with tiles of one page, so that they fit into 128 registers, 138, 12 with such tiles 131).
template <int HD, int HPL>
constexpr int kQ4Warps = HPL == 1 || HD == 64 ? 8 : 4;
template <int HD, int HPL>
constexpr int kQ4Ctas = HPL == 1 || HD == 64 ? 2 : 3;

// Tiles whose products are added up in an MMA's sums.  An MMA cuts off what lies more than 24 bits below its largest term or sum, always towards zero, so
// that a long chain of them falls behind by some 2^-25 of the sum a time: 48 requests of 8192 positions were 5.8e-6 of the result off without a limit, where one
// request of 2048 is 6e-7 off; they are 1.2e-6 off with chains of 16 to 24 MMAs, whose sums then go to FP32 ones in shared memory (FP32 throughout is 1.0 to 1.8e-6 off).
// Chains twice as long save 0.6 us of 131072 positions.
template <int HD, int HPL>
constexpr int kQ4Chain = HPL == 1 ? 8 : HD == 64 ? 4 : 6;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
constexpr float kLargest = 3.4028234663852886e38f;
// N words that lie together in shared memory
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&v)[N], uint32_t a) {
    if constexpr (N == 1)
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(a));
    else if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
    else
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
// The steps of groups g and g + 1 (g even) lie in one word; a BF16 number is the upper half of an FP32 one.
__device__ __forceinline__ float step_of(const uint32_t *words, int g) { return __uint_as_float(g & 1 ? words[g >> 1] & 0xffff0000u : words[g >> 1] << 16); }
// Two units' numbers, each pair as two halves: q 2^-18.  The third pair of the keys stays where it lies, q 2^-22, and the query's side takes the 16 back: an MMA
// aligns subnormal operands as if they were 2^-14, so that four bits of a score's 24 or more are lost, and two instructions of 300 a page saved.
template <bool KEYS>
__device__ __forceinline__ void numbers_of(uint32_t units, uint32_t (&x)[4]) {
    constexpr uint32_t kTop = 0x03c003c0u;
    x[0] = units & kTop;
    x[1] = units >> 4 & kTop;
    x[2] = KEYS ? units & kTop >> 4 : units << 4 & kTop;
    x[3] = __byte_perm(units, 0, 0x2301) & kTop;
}
// A group's scale and the largest step in its range, both as BF16: scale times step is below 1.
constexpr uint32_t kStepLimits = 0x7eff7effu;
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// FP32 in two halves' worth: what a half holds of x, towards zero, and the rest.
__device__ __forceinline__ float upper_limb(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }

// A share's pages of one row are tiles of two pages, spread over the CTA's warps; each warp has a ring of kQ4Slots tiles that bulk copies fill, the next row's first
// tiles already while this one's results are put together.  Per page
//   S = K Q   m16n8k16: the 16 positions are the rows, a group's 32 dimensions the k of two MMAs, the columns query heads.  The numbers are FP16 numbers as they lie
//             (q4_unit), after an AND.  A group's result is multiplied by its step d in FP32, and the offsets' part, m times the sum of the query over the group,
//             comes from one more MMA, whose operand m is as it lies in the page.
//   O += V P  rows are dimensions, k the positions, columns heads; a weight is multiplied by the step of its position and group first, and the offsets' part
//             is a sum of its own per lane, in FP32.  The product is scaled by a power of two that follows the largest step of its group, so that it keeps its digits in
//             FP16 (one scale for all groups: where one group's values were 10^6 times another's, the smaller ones were 5e-3 of their size off; its own for each
//             takes 43.5 us instead of 42.4 for 131072 positions).  What is left: a position whose step in a group is R times the others' costs them
//             some R 2^-30 (one of 10^4 times their size that weighs nothing: 2e-5 of the result).
//             The numbers of half the positions count from the other end (q4_v_flip), those positions' products have a minus: the sums stay as small as
//             the result, where sums of numbers that are all positive would be larger than it by the root of the number of positions that count.
// Queries and weights are two FP16 limbs.  HPL = 1: up to four heads, columns 2h and 2h + 1 are the limbs of head h, and a lane has one head.  HPL = 2: up to
// eight heads, a column each, the limbs in MMAs of their own; a lane has two heads.  Four heads of 131072 positions took 41 us as the former, 60 as the latter.
// Scores come out of an MMA with positions in the rows and go into the next with positions along k: movmatrix turns them.
// What bounds it: instructions.  A page of a head is 2560 bytes, 1.0 us of an SM's share of 6.55 TB/s for 17 pages, and it takes 368 of them (four heads of 128, of
// which 17 MMAs) or 455 (eight, 34) a warp; with less arithmetic the same kernel streams the pages of 131072 positions in 34 us.  One request of 131072 positions, 32 heads
// over 8 of 128: 43.4 us for 168 MB, 3.9 TB/s (FP16 pages would be 537 MB, 82 us at the rate of a copy); 8 requests of up to 4096 16.5, of which 10 begin and end
// parts; 48 of up to 8192 with eight heads to a key/value head 118 us for 384 MB.
template <int HD, int HPL>
struct Q4Smem {  // bytes
    static constexpr int kRing = kQ4Warps<HD, HPL> * kQ4Slots * kQ4Tile * 20 * HD, kBars = kRing, kMerge = kBars + kQ4Warps<HD, HPL> * kQ4Slots * 8, kMergeRow = HD + 8,  // floats; the pads keep rows on different banks
                         kQuery = kMerge + kQ4Warps<HD, HPL> * 4 * HPL * (kMergeRow + 2) * 4, kQueryRow = HD + 32,  // halves
        kSums = kQuery + 2 * 4 * HPL * kQueryRow * 2, kBack = kSums + 2 * 4 * HPL * 4 * 2, kAll = kBack + 4 * HPL * 4;
};

// A row's parts put together, by the CTA that was last: two dimensions of a head to a thread, a head to a warp, a part's largest score and sum to a lane.
template <int HD, int HPL, bool TRACK>
__device__ __forceinline__ void q4_merge_parts(const Q4AttnParams &p, int i, int share_a, int parts, int kvh) {
    constexpr int W = kQ4Warps<HD, HPL>, HEADS = 4 * HPL;
    const int tid = threadIdx.x, lane = tid & 31, G = p.n_heads / p.n_kv_heads, h0 = kvh * G;
    // The results of 16 parts are asked for at once, or of 8 where a thread has four places: one CTA reads them, and what it waits for is their latency
    // (one row of 16384 positions with eight heads a key/value head, 43 parts: 22 us; 36 with eight parts at a time and one place after the other).
    constexpr int ITEMS = (HEADS * (HD / 2) + W * 32 - 1) / (W * 32), AHEAD = ITEMS == 1 ? 16 : 8;
    const size_t stride = (size_t)p.n_heads * HD;
    const float2 *from_ml = reinterpret_cast<const float2 *>(p.part_ml) + (size_t)(i + share_a) * p.n_heads + h0;
    const float *from_o = p.part_o + (size_t)(i + share_a) * stride + (size_t)h0 * HD;
    float2 v[ITEMS][AHEAD], ml[ITEMS];
    auto ask = [&](int base) {
#pragma unroll
        for (int k = 0; k < ITEMS; k++) {
            const int idx = tid + k * W * 32;
            if (idx >= G * (HD / 2)) continue;
#pragma unroll
            for (int s = 0; s < AHEAD; s++)
                if (base + s < parts) v[k][s] = __ldcg(reinterpret_cast<const float2 *>(from_o + (base + s) * stride) + idx);
        }
    };
    auto largest = [&](int k, int s) {
        const int g = min((tid + k * W * 32) / (HD / 2), G - 1);
        return s < parts ? __ldcg(from_ml + (size_t)s * p.n_heads + g) : make_float2(-INFINITY, 0.f);
    };
#pragma unroll
    for (int k = 0; k < ITEMS; k++) ml[k] = largest(k, lane);
    ask(0);
    float M[ITEMS], L[ITEMS], f[ITEMS], ax[ITEMS], ay[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        M[k] = ml[k].x;
        for (int s = lane + 32; s < parts; s += 32) M[k] = fmaxf(M[k], largest(k, s).x);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) M[k] = fmaxf(M[k], __shfl_xor_sync(0xffffffffu, M[k], x));
        L[k] = ax[k] = ay[k] = 0.f;
    }
    for (int base = 0; base < parts; base += AHEAD) {
        if (base > 0) ask(base);
        if ((base & 31) == 0) {
#pragma unroll
            for (int k = 0; k < ITEMS; k++) {
                if (base > 0) ml[k] = largest(k, base + lane);
                f[k] = exp2_fast(ml[k].x - M[k]);
                L[k] = fmaf(ml[k].y, f[k], L[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < ITEMS; k++)
#pragma unroll
            for (int s = 0; s < AHEAD; s++) {
                const float fs = __shfl_sync(0xffffffffu, f[k], (base + s) & 31);
                if (base + s < parts) {
                    ax[k] = fmaf(v[k][s].x, fs, ax[k]);
                    ay[k] = fmaf(v[k][s].y, fs, ay[k]);
                }
            }
    }
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) L[k] += __shfl_xor_sync(0xffffffffu, L[k], x);
        const int idx = tid + k * W * 32, g = idx / (HD / 2);
        if (g >= G) continue;
        float *to_o = p.out + (size_t)i * p.ldo + h0 * HD + 2 * idx;
        to_o[0] = ax[k] / L[k];
        to_o[1] = ay[k] / L[k];
        if (TRACK && idx == g * (HD / 2)) p.sums[(size_t)i * p.n_heads + h0 + g] = make_float2(M[k], 1.f / L[k]);
    }
}

template <int HD, int HPL, bool TRACK>
__global__ void __launch_bounds__(kQ4Warps<HD, HPL> * 32, kQ4Ctas<HD, HPL>) q4_attn_kernel(const __grid_constant__ Q4AttnParams p) {
    constexpr int NG = HD / kQ4Group, NW = NG / 2, BLOCK = 20 * HD, TILE = kQ4Tile * BLOCK, W = kQ4Warps<HD, HPL>, HEADS = 4 * HPL;
    using Smem = Q4Smem<HD, HPL>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t = lane & 3;
    const int kvh = blockIdx.x % p.n_kv_heads, share = blockIdx.x / p.n_kv_heads, G = p.n_heads / p.n_kv_heads, h0 = kvh * G;
    const uint32_t ring = smem_u32(smem) + warp * kQ4Slots * TILE, bars = smem_u32(smem) + Smem::kBars + warp * kQ4Slots * 8;
    float *mg_o = reinterpret_cast<float *>(smem + Smem::kMerge);  // where the warps meet: [warp][head][kMergeRow], [warp][head], [warp][head]
    float *mg_m = mg_o + W * HEADS * Smem::kMergeRow, *mg_l = mg_m + W * HEADS;
    __half *q_s = reinterpret_cast<__half *>(smem + Smem::kQuery);    // [limb][head][kQueryRow]
    __half *sums_s = reinterpret_cast<__half *>(smem + Smem::kSums);  // [limb][head][4]: the query's sums over groups, scaled
    float *back_s = reinterpret_cast<float *>(smem + Smem::kBack);    // [head]: what takes the scale of the scores back
    int row_a = -1, row_b = -1;             // rows that other shares have parts of, too: the first, the last
    unsigned before_a = 0u, before_b = 0u;  // thread 0: their parts that were done before
    if (lane == 0) {
        for (int s = 0; s < kQ4Slots; s++) mbar_init(bars + s * 8, kQ4Tile);  // an arrival for each page of a tile
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async;" ::: "memory");
    }
    __syncwarp();
    pdl_launch_dependents();
    // What came with the launch is there before the kernels ahead are done; nothing else is.
    if (p.rows.far || p.far_cuts) pdl_wait();
    const int share0 = cut_at(p, share), share1 = cut_at(p, share + 1), row_first = cache_find(p.rows, share0);
    const uint8_t *plane = p.pool + ((size_t)p.layer * p.n_pages * p.n_kv_heads + kvh) * BLOCK;
    const size_t page_bytes = (size_t)p.n_kv_heads * BLOCK;
    const uint64_t policy = l2_evict_first_policy();
    const uint32_t v_piece = q4_v_code(HD, lane & 15, 0, lane >> 4);  // this lane's row of the four matrices of groups 0 and 1; two groups on: 32 bytes flipped
    unsigned issued = 0, used = 0;  // tiles through this warp's ring
    bool failed = false;

    // The part that is copied: its pages in the row's table, and how many of its tiles are this warp's and under way.  The places of 16 tiles' pages (in 16 bytes
    // from `plane`) wait in the lanes, which copy them when it is their turn; the next 16 are asked for ahead.
    constexpr uint32_t kNone = 0xffffffffu;
    int row, part_tiles = 0, part_issued = 0, part_pages = 0;
    uint32_t places = kNone, places_next = kNone;
    CacheRow r;
    const int32_t *table = nullptr;
    int page0 = 0;
    auto place = [&](int tile) {  // of this lane's page among the 16 tiles from `tile`
        const int pg = kQ4Tile * (warp + W * (tile + (lane >> 1))) + (lane & 1);
        return pg < part_pages ? (uint32_t)table[pg] * (uint32_t)(page_bytes >> 4) : kNone;
    };
    auto issue = [&] {
        if ((lane >> 1) == (part_issued & 15)) {
            const uint32_t slot = issued % kQ4Slots, bar = bars + slot * 8;
            mbar_expect_tx(bar, places == kNone ? 0 : BLOCK);  // a part that ends within a tile: no copy
            if (places != kNone) bulk_g2s(ring + slot * TILE + (lane & 1) * BLOCK, plane + (uint64_t)places * 16, BLOCK, bar, policy);
        }
        issued++;
        if ((++part_issued & 15) == 0) {
            places = places_next;
            places_next = place(part_issued + 16);
        }
    };
    constexpr int E = HD / 32, QUERIES = (HEADS + W - 1) / W;  // elements of a lane, heads of a warp
    float query[QUERIES][E];
    auto begin = [&](int i, int from) {  // row i from page `from` of all pages
        row = i;
#pragma unroll
        for (int n = 0; n < QUERIES; n++) {
            const int head = warp + n * W;
            const float *src = p.q + (size_t)i * p.ldq + (size_t)(h0 + head) * HD + E * lane;
#pragma unroll
            for (int e = 0; e < E; e++) query[n][e] = head < G ? src[e] : 0.f;
        }
        r = cache_row(p.rows, i);
        page0 = from - r.first;
        part_pages = r.upto > 0 ? min(share1, row_end(p, i)) - from : 0;
        table = p.table + (size_t)r.slot * p.max_pages_per_seq + page0;
        const int tiles = (part_pages + kQ4Tile - 1) / kQ4Tile;
        part_tiles = tiles > warp ? (tiles - warp + W - 1) / W : 0;
        part_issued = 0;
        places = place(0);
        places_next = place(16);
        while (part_issued < min(part_tiles, kQ4Slots)) issue();
    };
    pdl_wait();
    begin(row_first, share0);

    int from = share0;
    while (from < share1) {
        const int i = row, to = min(share1, row_end(p, i)), n_tiles = part_tiles, pos_first = page0 << 4;
        const int pos_end = min(r.upto, (to - r.first) << 4);  // of this part, in the row
        const bool track = TRACK && r.track >= 0;
        // The query, a head to a warp: times the scale of the scores, brought to 2^13 .. 2^14 by a power of two, those of numbers that stay where they lie; a sixteenth of it the
        // others (the second limb then ends 34 bits below the largest element), in two FP16 limbs; number i of the first unit of eight is next to that of the second.
#pragma unroll
        for (int n = 0; n < QUERIES; n++) {
            const int head = warp + n * W;
            if (head >= HEADS) break;
            const float scale = (float)(1.0 / sqrt((double)HD)) * 1.4426950408889634f;
            float y[E], top = 0.f, sum = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                y[e] = query[n][e] * scale;
                sum += y[e] * 0.03125f;  // 32 elements: five powers of two less, no sum overflows
                top = fmaxf(top, fabsf(y[e]));
            }
#pragma unroll
            for (int x = 1; x < 32; x <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                if (x < kQ4Group / E) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            }
            const int e2 = max(-100, min(127, (int)(__float_as_uint(top) >> 23) - 127)), up = 13 - e2;
            const float shift = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int dim = E * lane + e;
                const float whole = y[e] * ((dim & 3) == 2 ? shift : shift * 0.0625f);
                const __half hi = __float2half_rn(whole);
                __half *to_q = q_s + head * Smem::kQueryRow + (dim & ~7) + (dim & 3) * 2 + (dim >> 2 & 1);
                to_q[0] = hi;
                to_q[HEADS * Smem::kQueryRow] = __float2half_rn(whole - __half2float(hi));
            }
            if (lane % (kQ4Group / E) == 0) {
                const float whole = sum * shift;
                const __half hi = __float2half_rn(whole);
                sums_s[head * 4 + lane / (kQ4Group / E)] = hi;
                sums_s[(HEADS + head) * 4 + lane / (kQ4Group / E)] = __float2half_rn(whole - __half2float(hi));
            }
            if (lane == 0) back_s[head] = __uint_as_float((uint32_t)(127 + 5 - up) << 23);
        }
        __syncthreads();
        // lane (g8, t) has dimensions 8t .. 8t + 7 of every group of the head of column g8
        uint32_t qh[NG][4];
        uint32_t qsum[HPL];  // k: the groups
        float back[HPL];     // of this lane's own heads
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const __half *from_q = q_s + (HPL == 1 ? (g8 & 1) * HEADS + (g8 >> 1) : g8) * Smem::kQueryRow + g * kQ4Group + 8 * t;
            lds_words<4>(qh[g], smem_u32(from_q));
        }
#pragma unroll
        for (int h = 0; h < HPL; h++) {
            const int column = HPL == 1 ? (g8 & 1) * HEADS + (g8 >> 1) : h * HEADS + g8;  // HPL = 2: h is the limb
            qsum[h] = t < NW ? *reinterpret_cast<const uint32_t *>(sums_s + column * 4 + 2 * t) : 0u;
            back[h] = back_s[HPL * t + h];
        }
        float m_run[HPL], l_run[HPL];
        uint32_t vscale[NW];  // of each group, as the steps lie: the power of two that its values are scaled by; at first one that no step but 0 stays below
#pragma unroll
        for (int g = 0; g < NW; g++) vscale[g] = 0x71807180u;  // 2^100; steps are 2^-84 or more
#pragma unroll
        for (int h = 0; h < HPL; h++) {
            m_run[h] = -kLargest;  // finite: scores that overflowed to -infinity weigh nothing, also where a tile has no others
            l_run[h] = 0.f;
        }
        int pos0 = pos_first + warp * kQ4Tile * kPageTokens;
        float *own_row = mg_o + (warp * HEADS + HPL * t) * Smem::kMergeRow + 4 * g8;  // of head HPL * t: dimensions 4 g8 .. 4 g8 + 3 of a group
        int j = 0;
        do {
            float o[NG][2][4], offset[HPL][NG];  // offset: the offsets' part, of this lane's positions
#pragma unroll
            for (int g = 0; g < NG; g++) {
#pragma unroll
                for (int x = 0; x < 4; x++) o[g][0][x] = o[g][1][x] = 0.f;
#pragma unroll
                for (int h = 0; h < HPL; h++) offset[h][g] = 0.f;
            }
            const int first = j, chain_end = min(n_tiles, j + kQ4Chain<HD, HPL>);
            for (; j < chain_end; j++, pos0 += W * kQ4Tile * kPageTokens) {
                mbar_wait_bounded(bars + used % kQ4Slots * 8, used / kQ4Slots & 1u, 0, p.err, failed, kErrCacheWait);
                if (__any_sync(0xffffffffu, failed)) {
                    failed = true;
                    break;
                }
                const uint32_t tile = ring + used % kQ4Slots * TILE;
                used++;
                float s[HPL][kQ4Tile][2];  // rows g8 and g8 + 8 of each page
#pragma unroll
                for (int u = 0; u < kQ4Tile; u++) {
                    const uint32_t base = tile + u * BLOCK;
                    uint32_t k0[NG], k1[NG], d0[NW], d1[NW], m0[1], m1[1];
                    lds_words<NG>(k0, base + lane * NG * 4);
                    lds_words<NG>(k1, base + (32 + lane) * NG * 4);
                    lds_words<NW>(d0, base + 8 * HD + g8 * NG * 2);
                    lds_words<NW>(d1, base + 8 * HD + (g8 + 8) * NG * 2);
                    lds_words<1>(m0, base + 9 * HD + g8 * NG * 2 + (t % NW) * 4);  // k beyond the groups: once more, times the zeros of qsum
                    lds_words<1>(m1, base + 9 * HD + (g8 + 8) * NG * 2 + (t % NW) * 4);
                    float off[4], sum[HPL][2];
                    mma_f16_first(off, m0[0], m1[0], 0u, 0u, qsum[0], 0u);
                    if constexpr (HPL == 1) {
                        off[0] += off[1];
                        off[1] = off[2] + off[3];
                    } else {
                        mma_f16(off, m0[0], m1[0], 0u, 0u, qsum[1], 0u);
                    }
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        float c[4];
                        uint32_t x0[4], x1[4];
                        numbers_of<true>(k0[g], x0);
                        numbers_of<true>(k1[g], x1);
                        mma_f16_first(c, x0[0], x1[0], x0[1], x1[1], qh[g][0], qh[g][1]);
                        mma_f16(c, x0[2], x1[2], x0[3], x1[3], qh[g][2], qh[g][3]);
                        if constexpr (HPL == 1) {
                            c[0] += c[1];
                            c[1] = c[2] + c[3];
                        } else {
                            uint32_t ql[4];  // from shared memory each time: in registers they would push others out (121 us instead of 118, 48 rows of 8192)
                            lds_words<4>(ql, smem_u32(q_s + (HEADS + g8) * Smem::kQueryRow + g * kQ4Group + 8 * t));
                            float low[4];  // sums of their own: the fewer MMAs in a row, the less is cut off
                            mma_f16_first(low, x0[0], x1[0], x0[1], x1[1], ql[0], ql[1]);
                            mma_f16(low, x0[2], x1[2], x0[3], x1[3], ql[2], ql[3]);
#pragma unroll
                            for (int x = 0; x < 4; x++) c[x] += low[x];
                        }
#pragma unroll
                        for (int h = 0; h < HPL; h++) {
                            sum[h][0] = g ? fmaf(step_of(d0, g), c[h], sum[h][0]) : step_of(d0, g) * c[h];
                            sum[h][1] = g ? fmaf(step_of(d1, g), c[HPL + h], sum[h][1]) : step_of(d1, g) * c[HPL + h];
                        }
                    }
                    // 2^22 of the numbers, 2^-up; the sums' 2^5 2^-up
#pragma unroll
                    for (int h = 0; h < HPL; h++)
#pragma unroll
                        for (int x = 0; x < 2; x++) s[h][u][x] = fmaf(sum[h][x], 131072.f, off[x * HPL + h]) * back[h];
                }
                if (track) {
                    float *to_s = p.scores + (((size_t)kvh * p.total + r.first) * kPageTokens + pos0 + g8) * G;
#pragma unroll
                    for (int h = 0; h < HPL; h++)
#pragma unroll
                        for (int u = 0; u < kQ4Tile; u++)
#pragma unroll
                            for (int x = 0; x < 2; x++)
                                if (HPL * t + h < G && pos0 + 16 * u + 8 * x + g8 < pos_end) to_s[(16 * u + 8 * x) * G + HPL * t + h] = s[h][u][x];
                }
                uint32_t d[kQ4Tile][2][NW], vm[kQ4Tile][2][NW], steps[NW];
#pragma unroll
                for (int u = 0; u < kQ4Tile; u++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        lds_words<NW>(d[u][x], tile + u * BLOCK + 18 * HD + (g8 + 8 * x) * NG * 2);
                        lds_words<NW>(vm[u][x], tile + u * BLOCK + 19 * HD + (g8 + 8 * x) * NG * 2);
                    }
                if (pos0 + kQ4Tile * kPageTokens > pos_end) {  // positions behind the end: whatever their place holds
#pragma unroll
                    for (int u = 0; u < kQ4Tile; u++)
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const bool on = pos0 + 16 * u + 8 * x + g8 < pos_end;
#pragma unroll
                            for (int h = 0; h < HPL; h++) s[h][u][x] = on ? s[h][u][x] : -INFINITY;
#pragma unroll
                            for (int g = 0; g < NW; g++) {
                                d[u][x][g] = on ? d[u][x][g] : 0u;
                                vm[u][x][g] = on ? vm[u][x][g] : 0u;
                            }
                        }
                }
                // a score far above the reference, or a step beyond its group's scale: seldom after the first tile
                float top[HPL];
                uint32_t beyond = 0u;
#pragma unroll
                for (int g = 0; g < NW; g++) {
                    const uint32_t limit = kStepLimits - vscale[g];
                    steps[g] = limit;
#pragma unroll
                    for (int u = 0; u < kQ4Tile; u++) steps[g] = __vmaxu2(steps[g], __vmaxu2(d[u][0][g], d[u][1][g]));
                    beyond |= steps[g] ^ limit;
                }
                bool grown = beyond != 0u;
#pragma unroll
                for (int h = 0; h < HPL; h++) {
                    top[h] = s[h][0][0];
#pragma unroll
                    for (int u = 0; u < kQ4Tile; u++) top[h] = fmaxf(fmaxf(top[h], s[h][u][0]), s[h][u][1]);
                    grown |= top[h] > m_run[h] + 15.f;
                }
                if (__any_sync(0xffffffffu, grown)) {
                    float fix[HPL], vfix[NG];
                    uint32_t most[NG];
#pragma unroll
                    for (int g = 0; g < NG; g++) most[g] = __reduce_max_sync(0xffffffffu, steps[g >> 1] >> 16 * (g & 1) & 0xffffu);
#pragma unroll
                    for (int w = 0; w < NW; w++) {
                        uint32_t next = 0u;
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const uint32_t before = vscale[w] >> 16 * x & 0xffffu, step = most[2 * w + x];
                            // the largest step to 2^-5 .. 2^-4, up to 1 in range: times weights of up to 2^15
                            const uint32_t now = step > (kStepLimits & 0xffffu) - before ? (249u - (step >> 7)) << 7 : before;
                            next |= now << 16 * x;
                            vfix[2 * w + x] = __uint_as_float((0x3f80u + now - before) << 16);
                        }
                        vscale[w] = next;
                    }
#pragma unroll
                    for (int h = 0; h < HPL; h++) {
                        float mx = fmaxf(m_run[h] + 11.f, top[h]);
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                        mx -= 11.f;
                        fix[h] = exp2_fast(m_run[h] - mx);
                        m_run[h] = mx;
                        l_run[h] *= fix[h];
                    }
#pragma unroll
                    for (int h = 0; h < HPL; h++)
#pragma unroll
                        for (int g = 0; g < NG; g++) offset[h][g] *= fix[h];
                    if (first > 0) {
#pragma unroll
                        for (int h = 0; h < HPL; h++)
#pragma unroll
                            for (int g = 0; g < NG; g++) {
                                float4 *at = reinterpret_cast<float4 *>(own_row + h * Smem::kMergeRow + g * kQ4Group);
                                const float4 y = *at;
                                *at = make_float4(y.x * fix[h], y.y * fix[h], y.z * fix[h], y.w * fix[h]);
                            }
                    }
#pragma unroll
                    for (int g = 0; g < NG; g++)
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const float y = fix[HPL == 1 ? 0 : x & 1] * vfix[g];
                            o[g][0][x] *= y;
                            o[g][1][x] *= y;
                        }
                }
#pragma unroll
                for (int u = 0; u < kQ4Tile; u++) {
                    uint32_t v0[NG], v1[NG];  // unit g8 of positions 2t, 2t + 1, and of those eight farther
#pragma unroll
                    for (int g = 0; g < NG; g += 2) ldmatrix_x4_trans(v0[g], v1[g], v0[g + 1], v1[g + 1], tile + u * BLOCK + (g == 0 ? v_piece : v_piece ^ 32u));
                    float w[HPL][2];
#pragma unroll
                    for (int h = 0; h < HPL; h++) {
#pragma unroll
                        for (int x = 0; x < 2; x++) w[h][x] = exp2_fast(s[h][u][x] - m_run[h]);
                        l_run[h] += w[h][0] + w[h][1];
                    }
                    // the offsets' part, in FP32: an MMA cuts off what its sum of 22-bit products has below 24 bits, always towards zero, and this part and the
                    // numbers' are often large and of opposite sign
#pragma unroll
                    for (int x = 0; x < 2; x++) {
#pragma unroll
                        for (int g = 0; g < NG; g += 2) {
                            const float2 two = __half22float2(*reinterpret_cast<const __half2 *>(&vm[u][x][g >> 1]));
                            const float m0 = x ? fmaf(step_of(d[u][x], g), 15.f, two.x) : two.x, m1 = x ? fmaf(step_of(d[u][x], g + 1), 15.f, two.y) : two.y;
#pragma unroll
                            for (int h = 0; h < HPL; h++) {
                                offset[h][g] = fmaf(w[h][x], m0, offset[h][g]);
                                offset[h][g + 1] = fmaf(w[h][x], m1, offset[h][g + 1]);
                            }
                        }
                    }
                    // from here on the steps times their group's scale: exact, a power of two
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int g = 0; g < NW; g++) d[u][x][g] = mul_bf16x2(d[u][x][g], vscale[g]);
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        float hi[HPL][2], lo[HPL][2];
#pragma unroll
                        for (int h = 0; h < HPL; h++)
#pragma unroll
                            for (int x = 0; x < 2; x++) {
                                const float y = (x ? -w[h][x] : w[h][x]) * step_of(d[u][x], g);  // positions 8..15: 15 - q
                                hi[h][x] = upper_limb(y);
                                lo[h][x] = y - hi[h][x];
                            }
#pragma unroll
                        for (int limb = 0; limb < HPL; limb++) {
                            uint32_t b0, b1;
                            if constexpr (HPL == 1) {
                                b0 = transpose8(pack_h2(hi[0][0], lo[0][0]));
                                b1 = transpose8(pack_h2(hi[0][1], lo[0][1]));
                            } else {
                                b0 = transpose8(limb ? pack_h2(lo[0][0], lo[1][0]) : pack_h2(hi[0][0], hi[1][0]));
                                b1 = transpose8(limb ? pack_h2(lo[0][1], lo[1][1]) : pack_h2(hi[0][1], hi[1][1]));
                            }
                            uint32_t x0[4], x1[4];
                            numbers_of<false>(v0[g], x0);
                            numbers_of<false>(v1[g], x1);
                            mma_f16(o[g][0], x0[0], x0[1], x1[0], x1[1], b0, b1);
                            mma_f16(o[g][1], x0[2], x0[3], x1[2], x1[3], b0, b1);
                        }
                    }
                }
                __syncwarp();  // all lanes have read the tile before it is filled again
                if (part_issued < part_tiles) issue();
            }
            // a chain's sums, over the lanes that share a head for the offsets' part, to where the warps meet
#pragma unroll
            for (int h = 0; h < HPL; h++)
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const float unscale = __uint_as_float((272u << 23) - __float_as_uint(step_of(vscale, g)));  // 2^18 over the scale
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) offset[h][g] += __shfl_xor_sync(0xffffffffu, offset[h][g], x);
                    float v[4];
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const float *c = &o[g][x >> 1][2 * (x & 1)];
                        v[x] = fmaf(HPL == 1 ? c[0] + c[1] : c[h], unscale, offset[h][g]);
                    }
                    float4 *at = reinterpret_cast<float4 *>(own_row + h * Smem::kMergeRow + g * kQ4Group);
                    const float4 before = first > 0 ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
                    *at = make_float4(v[0] + before.x, v[1] + before.y, v[2] + before.z, v[3] + before.w);
                }
        } while (j < n_tiles && !failed);
        const CacheRow now = r;
        from = to;
        if (from < share1 && !failed) begin(i + 1, from);  // the next row's pages are on their way from here on
        // sums over the lanes that share a head; those over the warps follow
#pragma unroll
        for (int h = 0; h < HPL; h++) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], x);
            const int head = HPL * t + h;
            if (g8 == 0) {
                mg_m[warp * HEADS + head] = m_run[h];
                mg_l[warp * HEADS + head] = l_run[h];
            }
        }
        __syncthreads();
        const int parts = row_parts(p, i, now);
        for (int idx = tid; idx < G * (HD / 2); idx += W * 32) {  // two dimensions of a head; a head to a warp, whose first lanes have the warps' shares of it
            const int g = idx / (HD / 2), d = 2 * (idx - g * (HD / 2));
            float mw = lane < W ? mg_m[lane * HEADS + g] : -INFINITY, lw = lane < W ? mg_l[lane * HEADS + g] : 0.f, M = mw;
#pragma unroll
            for (int x = 1; x < W; x <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
            M = __shfl_sync(0xffffffffu, M, 0);
            const float fw = lw == 0.f ? 0.f : exp2_fast(mw - M);  // a warp without pages has no share
            float L = lw * fw, ax = 0.f, ay = 0.f;
#pragma unroll
            for (int x = 1; x < W; x <<= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
            L = __shfl_sync(0xffffffffu, L, 0);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float f = __shfl_sync(0xffffffffu, fw, w);
                const float2 v = *reinterpret_cast<const float2 *>(mg_o + (w * HEADS + g) * Smem::kMergeRow + d);
                if (f != 0.f) {
                    ax = fmaf(v.x, f, ax);
                    ay = fmaf(v.y, f, ay);
                }
            }
            const size_t part = (size_t)(i + share) * p.n_heads + h0 + g;
            if (parts == 1) {
                float *to_o = p.out + (size_t)i * p.ldo + (h0 + g) * HD + d;
                to_o[0] = pos_end > 0 ? ax / L : 0.f;
                to_o[1] = pos_end > 0 ? ay / L : 0.f;
            } else {
                *reinterpret_cast<float2 *>(p.part_o + part * HD + d) = make_float2(ax, ay);
            }
            if (d == 0 && parts > 1) *reinterpret_cast<float2 *>(p.part_ml + part * 2) = make_float2(M, L);
            if (TRACK && d == 0 && parts == 1) p.sums[(size_t)i * p.n_heads + h0 + g] = make_float2(M, 1.f / L);
        }
        // The rows that this share has with others are its first and its last.  Whoever of a row is last puts its parts together, at the end.
        if (parts > 1) {
            __syncthreads();
            unsigned before = 0u;
            if (tid == 0) {
                __threadfence();
                before = atomicAdd(p.arrived + (size_t)i * p.n_kv_heads + kvh, 1u);
            }
            if (now.first < share0)
                row_a = i, before_a = before;
            else
                row_b = i, before_b = before;
        }
        if (from >= share1) break;
        if (__syncthreads_or(failed)) {  // the warps' results have been read
            failed = true;
            break;
        }
    }
    if (failed) {  // the parts that are left count as done, so that the next launch finds zeros
        if (TRACK && lane == 0) *reinterpret_cast<volatile unsigned long long *>(p.gave_up) = p.call;
        for (unsigned j = ring_open((int)issued, (int)used, kQ4Slots); j < issued; j++)
            mbar_wait_bounded(bars + j % kQ4Slots * 8, j / kQ4Slots & 1u, 0, p.err, failed, kErrCacheWait);
        if (tid == 0)
            for (int i = cache_find(p.rows, min(p.total - 1, from)); from < share1; from = row_end(p, i++)) {
                const int parts = row_parts(p, i, cache_row(p.rows, i));
                unsigned *arrived = p.arrived + (size_t)i * p.n_kv_heads + kvh;
                if (parts > 1 && atomicAdd(arrived, 1u) == (unsigned)parts - 1) *arrived = 0;
            }
    }
    for (int which = 0; which < 2; which++) {
        const int i = which ? row_b : row_a;
        if (i < 0) continue;
        const CacheRow whole = cache_row(p.rows, i);
        const int share_a = whole.share, parts = row_parts(p, i, whole);
        const bool last = tid == 0 && (which ? before_b : before_a) == (unsigned)parts - 1;
        if (last) {
            __threadfence();
            p.arrived[(size_t)i * p.n_kv_heads + kvh] = 0;
        }
        if (!__syncthreads_or(last)) continue;
        q4_merge_parts<HD, HPL, TRACK>(p, i, share_a, parts, kvh);
    }
}

// The weight that positions have received: a thread has four neighbouring positions of all rows' pages and one key/value head, 64 bytes of scores with four heads, which
// come out of L2.  Attention and weights of 16 sequences of up to 8192 positions: 50.2 us, some 1.7 more with one position a thread.
constexpr int kQ4WeightThreads = 128;
__global__ void __launch_bounds__(kQ4WeightThreads) q4_weights_kernel(const __grid_constant__ Q4AttnParams p) {
    pdl_wait();
    const int kvh = blockIdx.y, at = (blockIdx.x * kQ4WeightThreads + threadIdx.x) * 4, G = p.n_heads / p.n_kv_heads;
    if (at >= p.total * kPageTokens) return;
    const int i = cache_find(p.rows, at >> 4);
    const CacheRow r = cache_row(p.rows, i);
    const int pos = at - r.first * kPageTokens, n = min(4, r.upto - pos);
    if (r.track < 0 || n <= 0) return;
    // the sums and scores of a call that gave up a wait are in part those of an earlier one: none of its rows adds anything
    const bool valid = __ldcg(p.gave_up) != p.call;
    const float *scores = p.scores + ((size_t)kvh * p.total * kPageTokens + at) * G;
    const float2 *sums = p.sums + (size_t)i * p.n_heads + kvh * G;
    float4 *w = reinterpret_cast<float4 *>(p.weights + (((size_t)r.track * p.n_layers + p.layer) * p.n_kv_heads + kvh) * p.track_tokens + pos);
    const float4 old = *w;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (G == 4) {  // the scores of a position in one load
        float4 s[4];
#pragma unroll
        for (int x = 0; x < 4; x++) s[x] = x < n ? reinterpret_cast<const float4 *>(scores)[x] : make_float4(0.f, 0.f, 0.f, 0.f);
        const float2 m0 = sums[0], m1 = sums[1], m2 = sums[2], m3 = sums[3];
#pragma unroll
        for (int x = 0; x < 4; x++)
            sum[x] = fmaf(exp2_fast(s[x].w - m3.x), m3.y, fmaf(exp2_fast(s[x].z - m2.x), m2.y, fmaf(exp2_fast(s[x].y - m1.x), m1.y, exp2_fast(s[x].x - m0.x) * m0.y)));
    } else {
        for (int g = 0; g < G; g++) {
            const float2 m = sums[g];
#pragma unroll
            for (int x = 0; x < 4; x++)
                if (x < n) sum[x] = fmaf(exp2_fast(scores[x * G + g] - m.x), m.y, sum[x]);
        }
    }
    // positions behind the row's end keep what they have
    if (valid) *w = make_float4(old.x + sum[0], n > 1 ? old.y + sum[1] : old.y, n > 2 ? old.z + sum[2] : old.z, n > 3 ? old.w + sum[3] : old.w);
}

template <int HD, int HPL, bool TRACK>
static int launch_q4_attn(const Q4AttnParams &a, int shares, cudaStream_t st) {
    static bool set[64] = {false};  // per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!set[dev & 63]) {
        JUNO_CUDA_TRY(cudaFuncSetAttribute(q4_attn_kernel<HD, HPL, TRACK>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4Smem<HD, HPL>::kAll));
        set[dev & 63] = true;
    }
    JUNO_CUDA_TRY(launch_pdl(q4_attn_kernel<HD, HPL, TRACK>, dim3((unsigned)(shares * a.n_kv_heads)), dim3(kQ4Warps<HD, HPL> * 32), Q4Smem<HD, HPL>::kAll, st, a));
    return JUNO_OK;
}

template <int HD, bool TRACK>
static int launch_q4_attn(const Q4AttnParams &a, int G, int shares, cudaStream_t st) {
    return G <= 4 ? launch_q4_attn<HD, 1, TRACK>(a, shares, st) : launch_q4_attn<HD, 2, TRACK>(a, shares, st);
}

// How the pages are cut for `slots` CTAs per key/value head that run at a time.  Either each row into parts of about equal length, no more than `slots` of them:
// then a CTA begins once, and the longest part is waited for; or all pages into equal shares across the rows: no CTA waits for another, but most begin
// a second row (kQ4BeginCost rounds).  A round is `round` pages, a tile for every warp of a CTA.  Parts and shares, 32 heads over 8 of 128: 4 rows of 4096 positions
// 12.5 and 15.8 us, 16 of 8192 35.9 and 37.0, 24 of 8192 63.4 and 49.0, which the rule tells apart; 32 of 4096 38.1 and 39.5, which it does not.
constexpr int kQ4BeginCost = 4;
static void q4_cut(std::vector<CacheRow> &rows, int pages, int slots, int round, std::vector<int32_t> *cuts) {
    const int n = (int)rows.size(), share = std::max(round, (pages + slots - 1) / slots);
    auto end_of = [&](int i) { return i + 1 < n ? rows[(size_t)i + 1].first : pages; };
    int len = 0;
    if (n <= slots) {  // the shortest parts, in whole rounds, that the slots hold
        for (len = (share + round - 1) / round * round;; len += std::max(1, len / (8 * round)) * round) {
            int parts = 0;
            for (int i = 0; i < n; i++) parts += (end_of(i) - rows[(size_t)i].first + len - 1) / len;
            if (parts <= slots) break;
        }
        if (n > 1 && len > share + kQ4BeginCost * round) len = 0;
    }
    for (int i = 0; i < n; i++) {
        const int from = rows[(size_t)i].first, size = end_of(i) - from;
        if (len) {
            const int k = (size + len - 1) / len;
            rows[(size_t)i].share = (int)cuts->size();
            for (int j = 0; j < k; j++) cuts->push_back(from + (int)((int64_t)size * j / k));
        } else {
            rows[(size_t)i].share = from / share;
            while ((int64_t)cuts->size() * share < end_of(i)) cuts->push_back((int32_t)cuts->size() * share);
        }
    }
    cuts->push_back(pages);
}
// Whether every row lies in one share.
static bool q4_whole(const std::vector<CacheRow> &rows, const std::vector<int32_t> &cuts) {
    for (size_t i = 0; i < rows.size(); i++)
        if (cuts[(size_t)rows[i].share + 1] < (i + 1 < rows.size() ? rows[i + 1].first : cuts.back())) return false;
    return true;
}

// Zeros, once; every launch leaves the counts so.
constexpr size_t kArrivedAt = 4;  // words before the counts
static int arrival_words(juno_ctx *c, size_t n, cudaStream_t st) {
    n += kArrivedAt;
    if (c->cache_arrived && c->cache_arrived_bytes >= n * sizeof(unsigned)) return JUNO_OK;
    void *words = c->cache_arrived;
    JUNO_TRY(cache_room(&words, &c->cache_arrived_bytes, n * sizeof(unsigned)));
    c->cache_arrived = static_cast<unsigned *>(words);
    JUNO_CUDA_TRY(cudaMemsetAsync(words, 0, c->cache_arrived_bytes, st));
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
    bool track = false;
    for (int i = 0; i < n; i++) {
        const int len = lens ? lens[i] : seqs[i]->len;
        rows[(size_t)i] = {seqs[i]->slot, len, (int)pages, seqs[i]->track, 0};
        pages += std::max(1, (len + kPageTokens - 1) / kPageTokens);
        track |= seqs[i]->track >= 0;
        bytes += len;
        JUNO_REQUIRE(pages < (1 << 26), "attention over %lld pages in one call", (long long)pages);
    }
    const bool wide = G > 4 && hd == 128;
    const int warps = wide ? kQ4Warps<128, 2> : kQ4Warps<64, 2>, ctas = wide ? kQ4Ctas<128, 2> : kQ4Ctas<64, 2>;
    std::vector<int32_t> cuts;
    q4_cut(rows, (int)pages, std::max(1, c->sm_count * ctas / H), warps * kQ4Tile, &cuts);
    const int shares = (int)cuts.size() - 1;
    const bool whole = shares == 1 || q4_whole(rows, cuts);
    if (track || !whole) JUNO_TRY(arrival_words(c, whole ? 0 : (size_t)n * H, st));
    Q4AttnParams a;
    auto padded = [](size_t b) { return (b + 255) & ~(size_t)255; };
    const size_t parts = whole ? 0 : (size_t)(n + shares), row_b = cache_rows_bytes(n), cut_b = shares + 1 > kInlineCuts ? padded(cuts.size() * sizeof(int32_t)) : 0,
                 far_b = row_b + cut_b, ml_b = padded(parts * n_heads * 8), o_b = padded(parts * n_heads * hd * 4),
                 s_b = track ? padded((size_t)pages * kPageTokens * n_heads * 4) : 0, sum_b = track ? (size_t)n * n_heads * sizeof(float2) : 0;
    uint8_t *scratch = nullptr;
    JUNO_TRY(cache_scratch(c, far_b + ml_b + o_b + s_b + sum_b, &scratch));
    JUNO_TRY(cache_rows(c, rows.data(), n, reinterpret_cast<CacheRow *>(scratch), &a.rows, st));
    a.far_cuts = cut_b ? reinterpret_cast<const int32_t *>(scratch + row_b) : nullptr;
    if (cut_b)
        JUNO_TRY(cache_words(c, cuts.data(), cuts.size(), reinterpret_cast<int32_t *>(scratch + row_b), st));
    else
        std::copy(cuts.begin(), cuts.end(), a.cuts);
    a.pool = static_cast<const uint8_t *>(p->k);
    a.table = p->d_table;
    a.max_pages_per_seq = p->max_pages_per_seq;
    a.n_pages = p->n_pages;
    a.n_kv_heads = H;
    a.n_heads = n_heads;
    a.layer = layer;
    a.n_layers = p->n_layers;
    a.total = (int)pages;
    a.shares = shares;
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.part_ml = reinterpret_cast<float *>(scratch + far_b);
    a.part_o = reinterpret_cast<float *>(scratch + far_b + ml_b);
    a.scores = track ? reinterpret_cast<float *>(scratch + far_b + ml_b + o_b) : nullptr;
    a.sums = track ? reinterpret_cast<float2 *>(scratch + far_b + ml_b + o_b + s_b) : nullptr;
    a.weights = p->weights;
    a.track_tokens = p->track_tokens;
    a.arrived = c->cache_arrived ? c->cache_arrived + kArrivedAt : nullptr;
    a.gave_up = reinterpret_cast<unsigned long long *>(c->cache_arrived);
    a.call = ++c->cache_calls;
    a.err = c->gemv_scratch.qerr + word;
    ProfScope prof(c, st, PROF_ATTN, (double)bytes * H * p->row_bytes());
    if (hd == 128)
        JUNO_TRY((track ? launch_q4_attn<128, true>(a, G, shares, st) : launch_q4_attn<128, false>(a, G, shares, st)));
    else
        JUNO_TRY((track ? launch_q4_attn<64, true>(a, G, shares, st) : launch_q4_attn<64, false>(a, G, shares, st)));
    c->kernel_launches++;
    if (!track) return JUNO_OK;
    JUNO_CUDA_TRY(launch_pdl(q4_weights_kernel, dim3((unsigned)((pages * (kPageTokens / 4) + kQ4WeightThreads - 1) / kQ4WeightThreads), (unsigned)H), dim3(kQ4WeightThreads), 0, st, a));
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
        for (int i = 0; i < n; i++)
            JUNO_REQUIRE(!lens || (lens[i] >= 0 && lens[i] <= seqs[i]->len), "sequence %d has %d cached positions, not %d", i, seqs[i]->len, lens ? lens[i] : 0);
        DeviceGuard g(c->device);
        JUNO_TRY(cache_call_distinct(p, n, seqs, true));
        JUNO_TRY(device_memory(c, q_dev, "q"));
        JUNO_TRY(device_memory(c, out_dev, "out"));
        CacheStream s(c, stream);
        JUNO_TRY(s.status);
        return q4_attend(c, p, layer, n, seqs, lens, n_heads, q_dev, ldq, out_dev, ldo, WAIT_ENQUEUED, s.st);
    });
}
