// Calls on cache pages with device pointers: append, read, weights, eviction.
#include "cache_ops.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <cstring>

#include "q4_pages.cuh"

namespace juno {

// ───────────────────────────── what the calls share ───────────────────────────────────────
CacheStream::CacheStream(juno_ctx *c, void *stream) : st(stream ? (cudaStream_t)stream : c->stream), c_(c) { status = join(); }

int CacheStream::join() {
    auto refuse = [](int rc, const char *what) {
        cudaGetLastError();
        set_error("%s", what);
        return rc;
    };
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(c_->stream, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone)
        return refuse(JUNO_ERR_INVALID_ARG, "the context's stream is being captured: calls on cache pages cannot be part of a graph");
    if (st == c_->stream) return JUNO_OK;
    if (cudaStreamIsCapturing(st, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone)
        return refuse(JUNO_ERR_INVALID_ARG, "the stream is being captured: calls on cache pages cannot be part of a graph");
    int dev = -1;
    if (cudaStreamGetDevice(st, &dev) != cudaSuccess || dev != c_->device)
        return refuse(JUNO_ERR_INVALID_ARG, "the stream belongs to another device than the context");
    for (cudaEvent_t &e : c_->cache_events)
        if (!e && cudaEventCreateWithFlags(&e, cudaEventDisableTiming) != cudaSuccess) return refuse(JUNO_ERR_CUDA, "cudaEventCreateWithFlags failed");
    if (cudaEventRecord(c_->cache_events[0], c_->stream) != cudaSuccess || cudaStreamWaitEvent(st, c_->cache_events[0], 0) != cudaSuccess)
        return refuse(JUNO_ERR_CUDA, "the stream could not be ordered behind the context's");
    joined_ = true;
    return JUNO_OK;
}

CacheStream::~CacheStream() {
    if (!joined_) return;
    if (cudaEventRecord(c_->cache_events[1], st) != cudaSuccess || cudaStreamWaitEvent(c_->stream, c_->cache_events[1], 0) != cudaSuccess) {
        cudaGetLastError();
        cudaStreamSynchronize(st);  // the order holds all the same
    }
}

int device_memory(const juno_ctx *c, const void *p, const char *name) {
    cudaPointerAttributes a;
    const cudaError_t e = cudaPointerGetAttributes(&a, p);
    if (e != cudaSuccess) cudaGetLastError();
    JUNO_REQUIRE(p && e == cudaSuccess && ((a.type == cudaMemoryTypeDevice && a.device == c->device) || a.type == cudaMemoryTypeManaged),
                 "%s is not memory of device %d", name, c->device);
    JUNO_REQUIRE(((uintptr_t)p & 3) == 0, "%s does not lie on a multiple of 4 bytes", name);
    return JUNO_OK;
}

int cache_scratch(juno_ctx *c, size_t bytes, uint8_t **out) {
    JUNO_TRY(ensure_device(&c->cache_scratch, &c->cache_scratch_bytes, bytes));
    *out = static_cast<uint8_t *>(c->cache_scratch);
    return JUNO_OK;
}

// By value: neither the caller's memory nor a staging buffer has to outlive the call.
struct WordsByValue {
    int32_t v[960];
};
static __global__ void words_kernel(int32_t *dst, const WordsByValue w, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) dst[i] = w.v[i];
}
int cache_words(juno_ctx *c, const int32_t *words, size_t n, int32_t *dst, cudaStream_t st) {
    constexpr size_t kMost = sizeof(WordsByValue) / sizeof(int32_t);
    for (size_t at = 0; at < n; at += kMost) {
        WordsByValue w;
        const int part = (int)std::min(kMost, n - at);
        memcpy(w.v, words + at, (size_t)part * sizeof(int32_t));
        words_kernel<<<1, 256, 0, st>>>(dst + at, w, part);
        JUNO_CUDA_TRY(cudaGetLastError());
        c->kernel_launches++;
    }
    return JUNO_OK;
}

int cache_rows(juno_ctx *c, const CacheRow *rows, int n, CacheRow *far, CacheRows *out, cudaStream_t st) {
    out->n = n;
    out->far = nullptr;
    if (n <= kInlineRows) {
        memcpy(out->in, rows, (size_t)n * sizeof(CacheRow));
        return JUNO_OK;
    }
    out->far = far;
    static_assert(sizeof(CacheRow) == 4 * sizeof(int32_t), "rows travel as words");
    return cache_words(c, reinterpret_cast<const int32_t *>(rows), (size_t)n * 4, reinterpret_cast<int32_t *>(far), st);
}

// ───────────────────────────── append and read ────────────────────────────────────────────
struct RowsParams {
    CacheRows rows;
    void *kpool, *vpool;
    const int32_t *table;
    int max_pages_per_seq, n_pages, n_kv_heads, layer, n_layers, n_tokens;
    float *k, *v;  // append only reads them
    int64_t ld;
    float *weights;
    int track_tokens;
};

// Eight lanes' worth of work: one lane has eight neighbouring dimensions of a key or value, four lanes a group.
template <int HD>
__global__ void __launch_bounds__(256) q4_append_kernel(const RowsParams p) {
    constexpr int LPV = HD / 8;  // lanes per vector
    const int H = p.n_kv_heads, sub = threadIdx.x % LPV;
    const int64_t vec = (int64_t)blockIdx.x * (256 / LPV) + threadIdx.x / LPV, n_vec = (int64_t)p.n_tokens * 2 * H;
    const bool on = vec < n_vec;
    const int64_t row = on ? vec / (2 * H) : 0;
    const int which = on ? (int)(vec - row * 2 * H) : 0, is_v = which >= H, h = which - is_v * H;
    float x[8];
    if (on) {
        const float *src = (is_v ? p.v : p.k) + row * p.ld + h * HD + sub * 8;
        if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            const float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + 4);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = src[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = 0.f;
    }
    float lo = INFINITY, hi = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        nan |= x[e] != x[e];
        x[e] = fminf(fmaxf(x[e], -kQ4Most), kQ4Most);
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
    }
    if (nan) hi = INFINITY;  // the group's mark: no clamped value is infinite
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    nan = hi == INFINITY;
    const __half mh = nan ? __ushort_as_half(0x7e00) : __float2half_rn(lo);
    const float reach = hi - lo;
    const __nv_bfloat16 dh = __float2bfloat16_rn(nan || reach < kQ4Nothing ? 0.f : __fdiv_rn(reach, 15.f));
    const float m = __half2float(mh), d = __bfloat162float(dh), inv = __fdiv_rn(1.f, d);
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; e++) q[e] = (uint32_t)q4_number(x[e], m, d, inv);
    if (!on) return;
    const CacheRow r = cache_row(p.rows, cache_find(p.rows, (int)row));
    const int pos = r.upto + (int)row - r.first, pp = pos & 15, g = sub >> 2;
    const int page = p.table[(size_t)r.slot * p.max_pages_per_seq + (pos >> 4)];
    uint8_t *block = static_cast<uint8_t *>(p.kpool) + (((size_t)p.layer * p.n_pages + page) * H + h) * q4_block_bytes(HD);
    if (is_v) {
#pragma unroll
        for (int u = 0; u < 2; u++)
            *reinterpret_cast<uint16_t *>(block + q4_v_code(HD, pp, 2 * (sub & 3) + u, g)) =
                (uint16_t)(q[4 * u] | q[4 * u + 1] << 4 | q[4 * u + 2] << 8 | q[4 * u + 3] << 12);
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) w |= q[e] << q4_k_shift(e);
        *reinterpret_cast<uint32_t *>(block + q4_k_code(HD, pp, sub & 3, g)) = w;
        if (sub == 0 && r.track >= 0)
            p.weights[(((size_t)r.track * p.n_layers + p.layer) * H + h) * p.track_tokens + pos] = 0.f;
    }
    if ((sub & 3) == 0) {
        *reinterpret_cast<uint16_t *>(block + (is_v ? q4_v_step(HD, pp, g) : q4_k_step(HD, pp, g))) = __bfloat16_as_ushort(dh);
        *reinterpret_cast<uint16_t *>(block + (is_v ? q4_v_offset(HD, pp, g) : q4_k_offset(HD, pp, g))) = __half_as_ushort(mh);
    }
}

__device__ __forceinline__ void store8(float *dst, const float (&x)[8]) {
    if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
        reinterpret_cast<float4 *>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) dst[e] = x[e];
    }
}

template <int HD>
__global__ void __launch_bounds__(256) q4_read_kernel(const RowsParams p) {
    constexpr int LPV = HD / 8;
    const int H = p.n_kv_heads, sub = threadIdx.x % LPV;
    const int64_t vec = (int64_t)blockIdx.x * (256 / LPV) + threadIdx.x / LPV;
    if (vec >= (int64_t)p.n_tokens * 2 * H) return;
    const int64_t row = vec / (2 * H);
    const int which = (int)(vec - row * 2 * H), is_v = which >= H, h = which - is_v * H;
    const CacheRow r = cache_row(p.rows, cache_find(p.rows, (int)row));
    const int pos = r.upto + (int)row - r.first, pp = pos & 15, g = sub >> 2;
    const int page = p.table[(size_t)r.slot * p.max_pages_per_seq + (pos >> 4)];
    const uint8_t *block = static_cast<const uint8_t *>(p.kpool) + (((size_t)p.layer * p.n_pages + page) * H + h) * q4_block_bytes(HD);
    const float m = __half2float(*reinterpret_cast<const __half *>(block + (is_v ? q4_v_offset(HD, pp, g) : q4_k_offset(HD, pp, g))));
    const float d = __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(block + (is_v ? q4_v_step(HD, pp, g) : q4_k_step(HD, pp, g))));
    float x[8];
    if (is_v) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t w = *reinterpret_cast<const uint16_t *>(block + q4_v_code(HD, pp, 2 * (sub & 3) + u, g));
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * u + i] = fmaf(d, (float)(w >> (4 * i) & 15u), m);
        }
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(block + q4_k_code(HD, pp, sub & 3, g));
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = fmaf(d, (float)(w >> q4_k_shift(e) & 15u), m);
    }
    store8((is_v ? p.v : p.k) + row * p.ld + h * HD + sub * 8, x);
}

// FP16 and FP32 pages: eight elements a thread, both directions.
template <typename T, bool APPEND>
__global__ void __launch_bounds__(256) rows_kernel(const RowsParams p, int hd) {
    const int H = p.n_kv_heads, per = hd / 8;
    const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)p.n_tokens * 2 * H * per;
    if (item >= n) return;
    const int64_t row = item / (2 * H * per);
    const int rest = (int)(item - row * 2 * H * per), is_v = rest >= H * per, h = (rest - is_v * H * per) / per, sub = rest % per;
    const CacheRow r = cache_row(p.rows, cache_find(p.rows, (int)row));
    const int pos = r.upto + (int)row - r.first;
    const int page = p.table[(size_t)r.slot * p.max_pages_per_seq + (pos >> 4)];
    T *at = static_cast<T *>(is_v ? p.vpool : p.kpool) + ((((size_t)p.layer * p.n_pages + page) * H + h) * kPageTokens + (pos & 15)) * hd + sub * 8;
    float *x = (is_v ? p.v : p.k) + row * p.ld + h * hd + sub * 8;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if constexpr (APPEND)
            at[e] = (T)x[e];
        else
            x[e] = (float)at[e];
    }
}

template <bool APPEND>
static int launch_rows(juno_ctx *c, const juno_kvpool *p, int layer, const CacheRow *rows, int n, int n_tokens, float *k, float *v, int64_t ld, cudaStream_t st) {
    RowsParams a;
    uint8_t *far = nullptr;
    if (cache_rows_bytes(n)) JUNO_TRY(cache_scratch(c, cache_rows_bytes(n), &far));
    JUNO_TRY(cache_rows(c, rows, n, reinterpret_cast<CacheRow *>(far), &a.rows, st));
    a.kpool = p->k;
    a.vpool = p->v;
    a.table = p->d_table;
    a.max_pages_per_seq = p->max_pages_per_seq;
    a.n_pages = p->n_pages;
    a.n_kv_heads = p->n_kv_heads;
    a.layer = layer;
    a.n_layers = p->n_layers;
    a.n_tokens = n_tokens;
    a.k = k;
    a.v = v;
    a.ld = ld;
    a.weights = p->weights;
    a.track_tokens = p->track_tokens;
    const int hd = p->head_dim;
    const int64_t lanes = (int64_t)n_tokens * 2 * p->n_kv_heads * (hd / 8);
    const unsigned blocks = (unsigned)((lanes + 255) / 256);
    ProfScope prof(c, st, APPEND ? PROF_ROPE_APPEND : PROF_OTHER, (double)n_tokens * p->n_kv_heads * (8.0 * hd + p->row_bytes()));
    if (p->dtype == kKvQ4) {
        if (APPEND)
            hd == 128 ? q4_append_kernel<128><<<blocks, 256, 0, st>>>(a) : q4_append_kernel<64><<<blocks, 256, 0, st>>>(a);
        else
            hd == 128 ? q4_read_kernel<128><<<blocks, 256, 0, st>>>(a) : q4_read_kernel<64><<<blocks, 256, 0, st>>>(a);
    } else if (p->dtype == 0) {
        rows_kernel<__half, APPEND><<<blocks, 256, 0, st>>>(a, hd);
    } else {
        rows_kernel<float, APPEND><<<blocks, 256, 0, st>>>(a, hd);
    }
    JUNO_CUDA_TRY(cudaGetLastError());
    c->kernel_launches++;
    return JUNO_OK;
}

int launch_kv_append(juno_ctx *c, const juno_kvpool *p, int layer, const CacheRow *rows, int n, int n_tokens, const float *k, const float *v, int64_t ld,
                     cudaStream_t st) {
    return launch_rows<true>(c, p, layer, rows, n, n_tokens, const_cast<float *>(k), const_cast<float *>(v), ld, st);
}

// ───────────────────────────── weights ────────────────────────────────────────────────────
// w[row][kv_head][ld], the first positions of each row; STORE: into the pool.
template <bool STORE>
__global__ void __launch_bounds__(256) weights_kernel(const CacheRows rows, float *weights, int layer, int n_layers, int n_kv_heads, int track_tokens, float *w, int64_t ld) {
    const int i = blockIdx.z, h = blockIdx.y, pos = blockIdx.x * 256 + threadIdx.x;
    const CacheRow r = cache_row(rows, i);
    if (pos >= r.upto) return;
    float *own = weights + (((size_t)r.track * n_layers + layer) * n_kv_heads + h) * track_tokens + pos;
    float *user = w + ((size_t)i * n_kv_heads + h) * ld + pos;
    if (STORE)
        *own = *user;
    else
        *user = *own;
}

// ───────────────────────────── eviction ───────────────────────────────────────────────────
struct EvictRow {
    int len, keep, recent, track, old_pages, new_pages;  // the last two: offsets into `pages`
};
struct EvictParams {
    const EvictRow *rows;
    const int32_t *pages;
    uint8_t *pool;
    int n, n_pages, n_kv_heads, n_layers, track_tokens, hd;
    float *weights;
    int32_t *kept;  // [layer][row][kv_head][kept_ld]
    int kept_ld;
};

// Order of weights as whole numbers: larger weight, larger key; both zeros alike, a NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvictThreads = 256, kEvictRows = 64;

// One CTA per (sequence, layer, head): the positions that stay, then their rows, in place and in order.  A row moves to the front or stays, so that what a
// step of kEvictRows rows overwrites has been read by it or by an earlier one.
__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const EvictParams p) {
    const int h = blockIdx.x, layer = blockIdx.y, i = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const EvictRow r = p.rows[i];
    float *w = p.weights + (((size_t)r.track * p.n_layers + layer) * p.n_kv_heads + h) * p.track_tokens;
    int32_t *kept = p.kept + (((size_t)layer * p.n + i) * p.n_kv_heads + h) * p.kept_ld;
    for (int j = r.keep + tid; j < p.kept_ld; j += kEvictThreads) kept[j] = -1;
    __shared__ unsigned hist[256];
    __shared__ int sums[kEvictThreads / 32][2];
    __shared__ unsigned sh_key, sh_need;
    if (r.keep == r.len) {
        for (int j = tid; j < r.keep; j += kEvictThreads) kept[j] = j;
        return;
    }
    const int old = r.len - r.recent;  // candidates
    unsigned need = (unsigned)(r.keep - r.recent), key = 0, mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < old; j += kEvictThreads) {
            const uint32_t u = weight_key(w[j]);
            if ((u & mask) == key) atomicAdd(&hist[u >> shift & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            unsigned left = need;
            int b = 255;
            while (b > 0 && hist[b] < left) left -= hist[b--];
            sh_key = key | (unsigned)b << shift;
            sh_need = left;
        }
        __syncthreads();
        key = sh_key;
        need = sh_need;
        mask |= 255u << shift;
    }
    // positions above `key` stay, and the first `need` of those that equal it
    int done = 0, equal = 0;
    for (int base = 0; base < r.len; base += kEvictThreads) {
        const int j = base + tid;
        const uint32_t u = j < old ? weight_key(w[j]) : 0u;
        const bool same = j < old && u == key;
        const unsigned eq = __ballot_sync(0xffffffffu, same);
        if (lane == 0) sums[warp][0] = __popc(eq);
        __syncthreads();
        int before = equal, all = 0;
        for (int k = 0; k < kEvictThreads / 32; k++) {
            if (k < warp) before += sums[k][0];
            all += sums[k][0];
        }
        const int rank = before + __popc(eq & ((1u << lane) - 1u));
        const bool stays = j < r.len && (j >= old || u > key || (same && rank < (int)need));
        const unsigned st = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) sums[warp][1] = __popc(st);
        __syncthreads();
        int at = done, sum = 0;
        for (int k = 0; k < kEvictThreads / 32; k++) {
            if (k < warp) at += sums[k][1];
            sum += sums[k][1];
        }
        if (stays) kept[at + __popc(st & ((1u << lane) - 1u))] = j;
        equal += all;
        done += sum;
        __syncthreads();
    }
    // the rows as half words: keys' numbers, values' numbers, and the four kinds of factors
    extern __shared__ uint16_t rows_s[];  // [kEvictRows][hd * 5 / 8]
    const int hd = p.hd, NG = hd / kQ4Group, halves = hd * 5 / 8;
    __shared__ float w_s[kEvictRows];
    auto block_of = [&](int list, int pos) {
        return p.pool + (((size_t)layer * p.n_pages + p.pages[list + (pos >> 4)]) * p.n_kv_heads + h) * q4_block_bytes(hd);
    };
    auto at = [&](int pos, int i) {  // half word i of a row: where it lies in a block
        const int pp = pos & 15, q = hd / 4;
        if (i < q) return q4_k_code(hd, pp, 0, 0) + 2 * i;
        if ((i -= q) < q) return q4_v_code(hd, pp, i / NG, i % NG);
        i -= q;
        const int kind = i / NG, g = i - kind * NG;
        return kind == 0 ? q4_k_step(hd, pp, g) : kind == 1 ? q4_k_offset(hd, pp, g) : kind == 2 ? q4_v_step(hd, pp, g) : q4_v_offset(hd, pp, g);
    };
    for (int base = 0; base < r.keep; base += kEvictRows) {
        const int n = min(kEvictRows, r.keep - base);
        for (int idx = tid; idx < n * halves; idx += kEvictThreads) {
            const int j = idx / halves, src = kept[base + j];
            rows_s[idx] = *reinterpret_cast<const uint16_t *>(block_of(r.old_pages, src) + at(src, idx - j * halves));
        }
        if (tid < n) w_s[tid] = w[kept[base + tid]];
        __syncthreads();
        for (int idx = tid; idx < n * halves; idx += kEvictThreads) {
            const int j = idx / halves, dst = base + j;
            *reinterpret_cast<uint16_t *>(block_of(r.new_pages, dst) + at(dst, idx - j * halves)) = rows_s[idx];
        }
        if (tid < n) w[base + tid] = w_s[tid];
        __syncthreads();
    }
}

// ───────────────────────────── checks ─────────────────────────────────────────────────────
int cache_call_check(juno_ctx *c, juno_kvpool *p, int layer, int n, juno_seq *const *seqs) {
    JUNO_TRY(ctx_check(c));
    JUNO_REQUIRE(p && seqs, "null argument");
    if (p->magic != kMagicPool) {
        set_error("KV pool is closed");
        return JUNO_ERR_CLOSED;
    }
    JUNO_REQUIRE(p->ctx == c, "pool belongs to another context");
    JUNO_REQUIRE(!p->latent && !p->owned_by_model, "this pool belongs to a model");
    JUNO_REQUIRE(n >= 1 && n <= 4096, "n=%d out of range", n);
    JUNO_REQUIRE(layer >= 0 && layer < p->n_layers, "layer %d out of range", layer);
    for (int i = 0; i < n; i++) {
        JUNO_TRY(seq_check(seqs[i]));
        JUNO_REQUIRE(seqs[i]->pool == p, "sequence %d belongs to another pool", i);
    }
    return JUNO_OK;
}

int cache_call_distinct(const juno_kvpool *p, int n, juno_seq *const *seqs) {
    std::vector<char> seen((size_t)p->max_slots, 0);
    for (int i = 0; i < n; i++) {
        JUNO_REQUIRE(!seen[(size_t)seqs[i]->slot], "sequence %d is there twice", i);
        seen[(size_t)seqs[i]->slot] = 1;
    }
    return JUNO_OK;
}

// The rows of an append or a read.
static int token_rows(int n, juno_seq *const *seqs, const int32_t *positions, const int32_t *counts, std::vector<CacheRow> *rows, int *total) {
    int64_t sum = 0;
    rows->reserve((size_t)n);
    for (int i = 0; i < n; i++) {
        JUNO_REQUIRE(positions[i] >= 0 && counts[i] >= 0, "bad position range of sequence %d", i);
        if (counts[i] == 0) continue;
        rows->push_back({seqs[i]->slot, positions[i], (int)sum, seqs[i]->track});
        sum += counts[i];
    }
    JUNO_REQUIRE(sum <= (1 << 24), "%lld positions in one call", (long long)sum);
    *total = (int)sum;
    return JUNO_OK;
}

}  // namespace juno

using namespace juno;

extern "C" {

int juno_kv_append_device(juno_ctx *c, juno_kvpool *p, int32_t layer, int32_t n, juno_seq *const *seqs, const int32_t *positions, const int32_t *counts,
                          const float *k_dev, const float *v_dev, int64_t ld, void *stream) {
    return guarded([&]() -> int {
        JUNO_TRY(ctx_check(c));
        std::lock_guard<std::recursive_mutex> lk(c->mu);
        JUNO_TRY(cache_call_check(c, p, layer, n, seqs));
        JUNO_REQUIRE(positions && counts, "null argument");
        JUNO_REQUIRE(ld >= (int64_t)p->n_kv_heads * p->head_dim, "rows of %lld elements hold no %d heads of %d", (long long)ld, p->n_kv_heads, p->head_dim);
        DeviceGuard g(c->device);
        JUNO_TRY(cache_call_distinct(p, n, seqs));
        std::vector<CacheRow> rows;
        int total = 0;
        JUNO_TRY(token_rows(n, seqs, positions, counts, &rows, &total));
        for (int i = 0; i < n; i++) {
            JUNO_REQUIRE(positions[i] <= seqs[i]->len, "position %d of sequence %d is not behind its %d cached ones", positions[i], i, seqs[i]->len);
            JUNO_REQUIRE((int64_t)positions[i] + counts[i] <= seqs[i]->max_tokens, "position %lld is beyond the limit of %d of sequence %d",
                         (long long)positions[i] + counts[i] - 1, seqs[i]->max_tokens, i);
        }
        if (total == 0) return JUNO_OK;
        JUNO_TRY(device_memory(c, k_dev, "k"));
        JUNO_TRY(device_memory(c, v_dev, "v"));
        CacheStream s(c, stream);
        JUNO_TRY(s.status);
        for (int i = 0; i < n; i++)
            if (counts[i]) JUNO_TRY(seq_reserve(seqs[i], positions[i], positions[i] + counts[i], s.st));
        JUNO_TRY(launch_kv_append(c, p, layer, rows.data(), (int)rows.size(), total, k_dev, v_dev, ld, s.st));
        for (int i = 0; i < n; i++) seqs[i]->len = std::max(seqs[i]->len, positions[i] + counts[i]);
        return JUNO_OK;
    });
}

int juno_kv_read_device(juno_ctx *c, juno_kvpool *p, int32_t layer, int32_t n, juno_seq *const *seqs, const int32_t *positions, const int32_t *counts, float *k_dev,
                        float *v_dev, int64_t ld, void *stream) {
    return guarded([&]() -> int {
        JUNO_TRY(ctx_check(c));
        std::lock_guard<std::recursive_mutex> lk(c->mu);
        JUNO_TRY(cache_call_check(c, p, layer, n, seqs));
        JUNO_REQUIRE(positions && counts, "null argument");
        JUNO_REQUIRE(ld >= (int64_t)p->n_kv_heads * p->head_dim, "rows of %lld elements hold no %d heads of %d", (long long)ld, p->n_kv_heads, p->head_dim);
        DeviceGuard g(c->device);
        std::vector<CacheRow> rows;
        int total = 0;
        JUNO_TRY(token_rows(n, seqs, positions, counts, &rows, &total));
        for (int i = 0; i < n; i++)
            JUNO_REQUIRE((int64_t)positions[i] + counts[i] <= seqs[i]->len, "sequence %d has %d cached positions, not %lld", i, seqs[i]->len,
                         (long long)positions[i] + counts[i]);
        if (total == 0) return JUNO_OK;
        JUNO_TRY(device_memory(c, k_dev, "k"));
        JUNO_TRY(device_memory(c, v_dev, "v"));
        CacheStream s(c, stream);
        JUNO_TRY(s.status);
        return launch_rows<false>(c, p, layer, rows.data(), (int)rows.size(), total, k_dev, v_dev, ld, s.st);
    });
}

int juno_kv_weights_device(juno_ctx *c, juno_kvpool *p, int32_t layer, int32_t n, juno_seq *const *seqs, const int32_t *counts, float *w_dev, int64_t ld, int32_t store,
                           void *stream) {
    return guarded([&]() -> int {
        JUNO_TRY(ctx_check(c));
        std::lock_guard<std::recursive_mutex> lk(c->mu);
        JUNO_TRY(cache_call_check(c, p, layer, n, seqs));
        JUNO_REQUIRE(counts, "null argument");
        DeviceGuard g(c->device);
        if (store) JUNO_TRY(cache_call_distinct(p, n, seqs));
        std::vector<CacheRow> rows;
        int most = 0;
        for (int i = 0; i < n; i++) {
            JUNO_REQUIRE(seqs[i]->track >= 0, "sequence %d keeps no weights (juno_seq_track)", i);
            JUNO_REQUIRE(counts[i] >= 0 && counts[i] <= seqs[i]->len, "sequence %d has %d cached positions, not %d", i, seqs[i]->len, counts[i]);
            rows.push_back({seqs[i]->slot, counts[i], i, seqs[i]->track});
            most = std::max(most, counts[i]);
        }
        JUNO_REQUIRE(ld >= most, "rows of %lld weights hold no %d", (long long)ld, most);
        if (most == 0) return JUNO_OK;
        JUNO_TRY(device_memory(c, w_dev, "w"));
        CacheStream s(c, stream);
        JUNO_TRY(s.status);
        CacheRows r;
        uint8_t *far = nullptr;
        if (cache_rows_bytes(n)) JUNO_TRY(cache_scratch(c, cache_rows_bytes(n), &far));
        JUNO_TRY(cache_rows(c, rows.data(), n, reinterpret_cast<CacheRow *>(far), &r, s.st));
        const dim3 grid((unsigned)((most + 255) / 256), (unsigned)p->n_kv_heads, (unsigned)n);
        ProfScope prof(c, s.st, PROF_OTHER, 0);
        if (store)
            weights_kernel<true><<<grid, 256, 0, s.st>>>(r, p->weights, layer, p->n_layers, p->n_kv_heads, p->track_tokens, w_dev, ld);
        else
            weights_kernel<false><<<grid, 256, 0, s.st>>>(r, p->weights, layer, p->n_layers, p->n_kv_heads, p->track_tokens, w_dev, ld);
        JUNO_CUDA_TRY(cudaGetLastError());
        c->kernel_launches++;
        return JUNO_OK;
    });
}

int juno_kv_evict(juno_ctx *c, juno_kvpool *p, int32_t n, juno_seq *const *seqs, int32_t keep, int32_t recent, int32_t *kept_dev, void *stream) {
    return guarded([&]() -> int {
        JUNO_TRY(ctx_check(c));
        std::lock_guard<std::recursive_mutex> lk(c->mu);
        JUNO_TRY(cache_call_check(c, p, 0, n, seqs));
        JUNO_REQUIRE(keep >= 1 && recent >= 0 && recent <= keep, "keep %d, recent %d: 1 <= keep and 0 <= recent <= keep", keep, recent);
        DeviceGuard g(c->device);
        JUNO_TRY(cache_call_distinct(p, n, seqs));
        for (int i = 0; i < n; i++) JUNO_REQUIRE(seqs[i]->track >= 0, "sequence %d keeps no weights (juno_seq_track)", i);
        if (kept_dev) JUNO_TRY(device_memory(c, kept_dev, "kept"));
        // Pages of the front that another sequence holds too are left to it: their rows go to fresh pages.
        std::vector<EvictRow> rows;
        std::vector<int32_t> pages;
        size_t fresh = 0;
        for (int i = 0; i < n; i++) {
            const juno_seq *s = seqs[i];
            if (s->len <= keep) continue;
            for (int j = 0; j < (keep + kPageTokens - 1) / kPageTokens; j++) fresh += p->page_refs[(size_t)s->pages[(size_t)j]] > 1;
        }
        if (fresh > p->free_pages.size()) {
            set_error("KV pool exhausted: %zu pages free, %zu needed for rows of shared pages", p->free_pages.size(), fresh);
            return JUNO_ERR_OOM;
        }
        size_t next = p->free_pages.size();
        for (int i = 0; i < n; i++) {
            const juno_seq *s = seqs[i];
            EvictRow r{s->len, std::min(s->len, keep), std::min(s->len, recent), s->track, (int)pages.size(), 0};
            if (s->len > keep) {
                pages.insert(pages.end(), s->pages.begin(), s->pages.end());
                r.new_pages = (int)pages.size();
                for (int j = 0; j < (keep + kPageTokens - 1) / kPageTokens; j++) {
                    const int pg = s->pages[(size_t)j];
                    pages.push_back(p->page_refs[(size_t)pg] > 1 ? p->free_pages[--next] : pg);
                }
            }
            rows.push_back(r);
        }
        CacheStream st(c, stream);
        JUNO_TRY(st.status);
        auto padded = [](size_t b) { return (b + 255) & ~(size_t)255; };
        const size_t row_bytes = padded(rows.size() * sizeof(EvictRow)), page_bytes = padded(pages.size() * 4),
                     kept_bytes = kept_dev ? 0 : (size_t)p->n_layers * n * p->n_kv_heads * keep * 4;
        uint8_t *scratch = nullptr;
        JUNO_TRY(cache_scratch(c, row_bytes + page_bytes + kept_bytes, &scratch));
        JUNO_TRY(cache_words(c, reinterpret_cast<const int32_t *>(rows.data()), rows.size() * sizeof(EvictRow) / 4, reinterpret_cast<int32_t *>(scratch), st.st));
        JUNO_TRY(cache_words(c, pages.data(), pages.size(), reinterpret_cast<int32_t *>(scratch + row_bytes), st.st));
        EvictParams a;
        a.rows = reinterpret_cast<const EvictRow *>(scratch);
        a.pages = reinterpret_cast<const int32_t *>(scratch + row_bytes);
        a.pool = static_cast<uint8_t *>(p->k);
        a.n = n;
        a.n_pages = p->n_pages;
        a.n_kv_heads = p->n_kv_heads;
        a.n_layers = p->n_layers;
        a.track_tokens = p->track_tokens;
        a.hd = p->head_dim;
        a.weights = p->weights;
        a.kept = kept_dev ? kept_dev : reinterpret_cast<int32_t *>(scratch + row_bytes + page_bytes);
        a.kept_ld = keep;
        {
            ProfScope prof(c, st.st, PROF_OTHER, 0);
            evict_kernel<<<dim3((unsigned)p->n_kv_heads, (unsigned)p->n_layers, (unsigned)n), kEvictThreads, (size_t)kEvictRows * p->head_dim * 5 / 4, st.st>>>(a);
        }
        JUNO_CUDA_TRY(cudaGetLastError());
        c->kernel_launches++;
        p->free_pages.resize(next);
        int rc = JUNO_OK;
        for (int i = 0; i < n; i++) {
            juno_seq *s = seqs[i];
            if (s->len <= keep) continue;
            const int np = (keep + kPageTokens - 1) / kPageTokens;
            int32_t *row = p->h_table + (size_t)s->slot * p->max_pages_per_seq;
            int lo = np, hi = -1;
            for (int j = 0; j < (int)s->pages.size(); j++) {
                const int old = s->pages[(size_t)j], now = j < np ? pages[(size_t)rows[(size_t)i].new_pages + j] : -1;
                if (now == old) continue;
                if (--p->page_refs[(size_t)old] == 0) p->free_pages.push_back(old);
                if (now < 0) continue;
                p->page_refs[(size_t)now] = 1;
                s->pages[(size_t)j] = row[j] = now;
                lo = std::min(lo, j);
                hi = j;
            }
            s->pages.resize((size_t)np);
            s->len = keep;
            if (hi >= 0 && rc == JUNO_OK) rc = table_store(p, s->slot, lo, hi, st.st);
        }
        return rc;
    });
}

}  // extern "C"
