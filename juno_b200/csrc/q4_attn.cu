// Decode attention over 4-bit pages, and the weight that cached positions receive.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "cache_ops.cuh"
#include "q4_pages.cuh"

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
};

__device__ __forceinline__ int row_splits(const Q4AttnParams &p, int i) {
    return (i + 1 < p.rows.n ? cache_row(p.rows, i + 1).first : p.n_splits) - cache_row(p.rows, i).first;
}

constexpr int kQ4MaxGroup = 8, kQ4Threads = 128;

template <int HD>
__global__ void __launch_bounds__(kQ4Threads) q4_attn_kernel(const Q4AttnParams p) {
    constexpr int LPT = HD / 8, SLOTS = kQ4Threads / LPT;
    const int kvh = blockIdx.x % p.n_kv_heads, id = blockIdx.x / p.n_kv_heads, tid = threadIdx.x, sub = tid % LPT, slot = tid / LPT;
    const int i = cache_find(p.rows, id), nsp = row_splits(p, i), G = p.n_heads / p.n_kv_heads, h0 = kvh * G;
    const CacheRow r = cache_row(p.rows, i);
    const int t0 = (id - r.first) * p.chunk, t1 = min(r.upto, t0 + p.chunk);
    __shared__ float sm_m[SLOTS][kQ4MaxGroup], sm_l[SLOTS][kQ4MaxGroup], sm_o[SLOTS][HD];
    const float scale = (float)(1.0 / sqrt((double)HD)) * 1.4426950408889634f;
    float q[kQ4MaxGroup][8], o[kQ4MaxGroup][8], m[kQ4MaxGroup], l[kQ4MaxGroup];
#pragma unroll
    for (int g = 0; g < kQ4MaxGroup; g++) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            q[g][e] = g < G ? p.q[(size_t)i * p.ldq + (h0 + g) * HD + sub * 8 + e] * scale : 0.f;
            o[g][e] = 0.f;
        }
        m[g] = -INFINITY;
        l[g] = 0.f;
    }
    const int gr = sub >> 2;
    for (int t = t0 + slot; t - slot < t1; t += SLOTS) {
        const bool on = t < t1;
        const int tt = on ? t : t0, pp = tt & 15;
        const uint8_t *b = p.pool + (((size_t)p.layer * p.n_pages + p.table[(size_t)r.slot * p.max_pages_per_seq + (tt >> 4)]) * p.n_kv_heads + kvh) * q4_block_bytes(HD);
        const uint32_t kf = *reinterpret_cast<const uint32_t *>(b + q4_k_factors(HD, pp, gr)), kc = *reinterpret_cast<const uint32_t *>(b + q4_k_code(HD, pp, sub & 3, gr));
        const uint32_t vf = *reinterpret_cast<const uint32_t *>(b + q4_v_factors(HD, pp, gr));
        const uint32_t v0 = *reinterpret_cast<const uint16_t *>(b + q4_v_code(HD, pp, 2 * (sub & 3), gr)), v1 = *reinterpret_cast<const uint16_t *>(b + q4_v_code(HD, pp, 2 * (sub & 3) + 1, gr));
        const float km = __half2float(__ushort_as_half((unsigned short)kf)), kd = __uint_as_float(kf & 0xffff0000u);
        const float vm = __half2float(__ushort_as_half((unsigned short)vf)), vd = __uint_as_float(vf & 0xffff0000u);
        float v[8], k[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            k[e] = fmaf(kd, (float)(kc >> q4_k_shift(e) & 15u), km);
            v[e] = fmaf(vd, (float)((e < 4 ? v0 : v1) >> (4 * (e & 3)) & 15u), vm);
        }
#pragma unroll
        for (int g = 0; g < kQ4MaxGroup; g++) {
            if (g >= G) break;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) s = fmaf(q[g][e], k[e], s);
#pragma unroll
            for (int x = LPT / 2; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            if (!on) continue;
            if (p.scores && sub == 0) p.scores[(((size_t)id * p.n_kv_heads + kvh) * p.chunk + (t - t0)) * G + g] = s;
            const float mn = fmaxf(m[g], s), corr = exp2f(m[g] - mn), pe = exp2f(s - mn);
            l[g] = fmaf(l[g], corr, pe);
#pragma unroll
            for (int e = 0; e < 8; e++) o[g][e] = fmaf(o[g][e], corr, pe * v[e]);
            m[g] = mn;
        }
    }
#pragma unroll
    for (int g = 0; g < kQ4MaxGroup; g++) {
        if (g >= G) break;
        if (sub == 0) {
            sm_m[slot][g] = m[g];
            sm_l[slot][g] = l[g];
        }
#pragma unroll
        for (int e = 0; e < 8; e++) sm_o[slot][sub * 8 + e] = o[g][e];
        __syncthreads();
        if (tid < HD) {
            float M = -INFINITY, L = 0.f, acc = 0.f;
            for (int w = 0; w < SLOTS; w++) M = fmaxf(M, sm_m[w][g]);
            for (int w = 0; w < SLOTS; w++) {
                if (sm_l[w][g] == 0.f) continue;  // a slot without positions
                const float f = exp2f(sm_m[w][g] - M);
                L = fmaf(sm_l[w][g], f, L);
                acc = fmaf(sm_o[w][tid], f, acc);
            }
            const size_t part = (size_t)id * p.n_heads + h0 + g;
            if (nsp == 1)
                p.out[(size_t)i * p.ldo + (h0 + g) * HD + tid] = t0 < t1 ? acc / L : 0.f;
            else
                p.part_o[part * HD + tid] = acc;
            if (tid == 0 && (nsp > 1 || p.scores)) {
                p.part_ml[part * 2] = M;
                p.part_ml[part * 2 + 1] = L;
            }
        }
        __syncthreads();
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

int q4_attend(juno_ctx *c, juno_kvpool *p, int layer, int n, juno_seq *const *seqs, const int32_t *lens, int n_heads, const float *q, int64_t ldq, float *out,
              int64_t ldo, cudaStream_t st) {
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
    ProfScope prof(c, st, PROF_ATTN, (double)bytes * H * p->row_bytes());
    const unsigned grid = (unsigned)(splits * H);
    if (hd == 128)
        q4_attn_kernel<128><<<grid, kQ4Threads, 0, st>>>(a);
    else
        q4_attn_kernel<64><<<grid, kQ4Threads, 0, st>>>(a);
    JUNO_CUDA_TRY(cudaGetLastError());
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
        return q4_attend(c, p, layer, n, seqs, lens, n_heads, q_dev, ldq, out_dev, ldo, s.st);
    });
}
