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

static int refuse(int rc, const char *what) {
    cudaGetLastError();
    set_error("%s", what);
    return rc;
}

int cache_call_outside_graph(const juno_ctx *c) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    const cudaError_t e = cudaStreamIsCapturing(c->stream, &cap);
    if (e != cudaSuccess) cudaGetLastError();  // but for a capture elsewhere that this stream would join, what is wrong shows in the next call
    if (e == cudaErrorStreamCaptureImplicit || (e == cudaSuccess && cap != cudaStreamCaptureStatusNone))
        return refuse(JUNO_ERR_INVALID_ARG, "the context's stream is being captured: calls on cache pages cannot be part of a graph");
    return JUNO_OK;
}

int CacheStream::join() {
    JUNO_TRY(cache_call_outside_graph(c_));
    if (st == c_->stream) return JUNO_OK;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
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

// Growing waits for the device, so it is done seldom: to twice the room that there was where the device has as much, and 1 MB at first.  A sequence that keeps weights
// asks for more with every page.
int cache_room(void **ptr, size_t *cur, size_t bytes) {
    if (*ptr && *cur >= bytes) return JUNO_OK;
    if (ensure_device(ptr, cur, std::max({bytes, 2 * *cur, (size_t)1 << 20})) == JUNO_OK) return JUNO_OK;
    return ensure_device(ptr, cur, bytes);
}

int cache_scratch(juno_ctx *c, size_t bytes, uint8_t **out) {
    JUNO_TRY(cache_room(&c->cache_scratch, &c->cache_scratch_bytes, bytes));
    *out = static_cast<uint8_t *>(c->cache_scratch);
    return JUNO_OK;
}

static __global__ void words_kernel(int32_t *dst, const __grid_constant__ WordsByValue w, int n) {
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
    constexpr size_t kWords = sizeof(CacheRow) / sizeof(int32_t);
    return cache_words(c, reinterpret_cast<const int32_t *>(rows), (size_t)n * kWords, reinterpret_cast<int32_t *>(far), st);
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

// Where the positions of a block's rows lie: found once per row, by one thread.  A barrier has to follow.
struct RowPlace {
    uint8_t *page;  // this layer's page, or null behind the last row
    int pos, track;
};
template <int R>
__device__ __forceinline__ void find_places(const RowsParams &p, int row0, size_t page_bytes, RowPlace (&places)[R]) {
    pdl_launch_dependents();
    pdl_wait();
    if (threadIdx.x < R) {
        const int row = row0 + threadIdx.x;
        RowPlace at{nullptr, 0, -1};
        if (row < p.n_tokens) {
            const CacheRow r = cache_row(p.rows, cache_find(p.rows, row));
            at.pos = r.upto + row - r.first;
            at.track = r.track;
            at.page = static_cast<uint8_t *>(p.kpool) + ((size_t)p.layer * p.n_pages + p.table[(size_t)r.slot * p.max_pages_per_seq + (at.pos >> 4)]) * page_bytes;
        }
        places[threadIdx.x] = at;
    }
}

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A CTA has R positions, of keys (blockIdx.y = 0) or values.  A lane has eight neighbouring dimensions, four lanes a group: what is stored of a position is
// contiguous.  The arithmetic is what bounds it, so each element costs a dozen instructions: the number is found from an estimate
// (q4_number_near: a saturating product and one sum that rounds), and only where a lane has an estimate too close to half-way are its eight numbers decided
// exactly.  131000 positions of eight heads of 128: 1.24 GB in 235 us, 5.3 TB/s; 8156 of them 77 MB in 23 us.
template <int HD, int R, bool V>
__device__ __forceinline__ void append_rows(const RowsParams &p, const RowPlace (&places)[R], int row0) {
    constexpr int LPV = HD / 8;  // lanes per vector
    const int H = p.n_kv_heads, sub = threadIdx.x % LPV, g = sub >> 2;
    bool found = false;  // the places, by all threads: each of them has a vector
    for (int vec = threadIdx.x / LPV; vec < (H + 3) / 4 * 4; vec += blockDim.x / LPV) {  // whole warps take part in the sums of a group
        const int h = min(vec, H - 1);
        float rows[R][8];  // of all positions: their loads are under way together
        const float *src = (V ? p.v : p.k) + row0 * p.ld + h * HD + sub * 8;
        const bool aligned = (reinterpret_cast<uintptr_t>(src) & 15) == 0 && (p.ld & 3) == 0;
#pragma unroll
        for (int n = 0; n < R; n++) {
            float(&x)[8] = rows[n];
            if (aligned) {
                const float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + 4);
                x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
                x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = src[e];
            }
            if (row0 + n + 1 < p.n_tokens) src += p.ld;  // behind the last row: that one again
        }
        if (!found) __syncthreads();  // the rows are on their way meanwhile
        found = true;
#pragma unroll
        for (int n = 0; n < R; n++) {
            const RowPlace at = places[n];
            float(&x)[8] = rows[n];
            float lo = x[0], hi = x[0];
#pragma unroll
            for (int e = 1; e < 8; e++) {
                lo = min_nan(lo, x[e]);
                hi = max_nan(hi, x[e]);
            }
            if (!(fmaxf(hi, -lo) <= kQ4Most && lo == lo)) {  // seldom: a NaN, or values beyond what FP16 holds
                const bool nan = lo != lo;
                lo = kQ4Most;
                hi = -kQ4Most;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x[e] = fminf(fmaxf(x[e], -kQ4Most), kQ4Most);
                    lo = fminf(lo, x[e]);
                    hi = fmaxf(hi, x[e]);
                }
                if (nan) hi = INFINITY;  // the group's mark of a NaN: no clamped value is infinite
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            const bool nan = hi == INFINITY;
            const __half mh = nan ? __ushort_as_half(0x7e00) : __float2half_rn(lo);
            const float reach = hi - lo;
            // reach / 15 rounded to FP32, then to BF16.  The product with 1/15 is off by an FP32 step or two, which matters only next to the middle of two BF16 numbers.
            float fifteenth = reach * (1.f / 15.f);
            if ((__float_as_uint(fifteenth) + 0x7ffcu & 0xffffu) >= 0xfff8u) fifteenth = __fdiv_rn(reach, 15.f);
            const __nv_bfloat16 dh = __float2bfloat16_rn(nan || reach < kQ4Nothing ? 0.f : fifteenth);
            const float m = __half2float(mh), d = __bfloat162float(dh);
            float inv;  // 1 / (15 d): 15 d has 12 bits
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d * 15.f));
            inv = d > 0.f ? inv : 0.f;
            uint32_t bits[8];
            float worst = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float off;
                bits[e] = q4_number_near(x[e], m, inv, &off);
                worst = fmaxf(worst, off);
            }
            auto word = [](const uint32_t (&q)[8]) { return q4_unit(q[0], q[1], q[2], q[3]) | q4_unit(q[4], q[5], q[6], q[7]) << 16; };
            uint32_t w = word(bits);
            if (worst > kQ4Near) {
                uint32_t q[8];
#pragma unroll
                for (int e = 0; e < 8; e++) q[e] = (uint32_t)q4_number_exact(x[e], m, d, inv * 15.f);
                w = word(q);
            }
            if (vec >= H || !at.page) continue;
            const int pp = at.pos & 15;
            if (V) w ^= q4_v_flip(pp);
            uint8_t *block = at.page + h * q4_block_bytes(HD);
            *reinterpret_cast<uint32_t *>(block + (V ? q4_v_code(HD, pp, 2 * (sub & 3), g) : q4_k_code(HD, pp, sub & 3, g))) = w;
            if (!V && sub == 0 && at.track >= 0) p.weights[(((size_t)at.track * p.n_layers + p.layer) * H + h) * p.track_tokens + at.pos] = 0.f;
            if ((sub & 3) == 0) {
                *reinterpret_cast<uint16_t *>(block + (V ? q4_v_step(HD, pp, g) : q4_k_step(HD, pp, g))) = __bfloat16_as_ushort(dh);
                *reinterpret_cast<uint16_t *>(block + (V ? q4_v_offset(HD, pp, g) : q4_k_offset(HD, pp, g))) = __half_as_ushort(mh);
            }
        }
    }
}
template <int HD, int R>
__global__ void __launch_bounds__(256) q4_append_kernel(const __grid_constant__ RowsParams p) {
    __shared__ RowPlace places[R];
    const int row0 = blockIdx.x * R;
    find_places<R>(p, row0, (size_t)p.n_kv_heads * q4_block_bytes(HD), places);
    if (blockIdx.y == 0)
        append_rows<HD, R, false>(p, places, row0);
    else
        append_rows<HD, R, true>(p, places, row0);
}

// A number that lies in bits of a word below 2^23, as FP32: without a conversion.
__device__ __forceinline__ float bits_as_float(uint32_t w, uint32_t mask) { return __uint_as_float((w & mask) | 0x4b000000u) - 8388608.f; }

// A CTA has kReadRows positions, of keys (blockIdx.y = 0) or values; a lane has eight neighbouring dimensions, which it writes at once where they are aligned, and
// the loads of all positions are under way together.  8156 positions of eight heads of 128, 77 MB, with their append: 32.0 us (0.5 more with four dimensions of two groups a
// lane, 1.2 more of one group).
constexpr int kAppendRows = 4, kReadRows = 4;
__device__ __forceinline__ void store8(float *to, const float (&x)[8], int wide) {
    if (wide == 2) {
        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]) : "memory");
    } else if (wide == 1) {
        *reinterpret_cast<float4 *>(to) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(to + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) to[e] = x[e];
    }
}
template <int HD, bool V>
__device__ __forceinline__ void read_rows(const RowsParams &p, const RowPlace (&places)[kReadRows], int row0) {
    constexpr int LPV = HD / 8;
    const int H = p.n_kv_heads, sub = threadIdx.x % LPV, t = sub & 3, g = sub >> 2, n_rows = min(kReadRows, p.n_tokens - row0);
    for (int h = threadIdx.x / LPV; h < H; h += blockDim.x / LPV) {
        float *to = (V ? p.v : p.k) + row0 * p.ld + h * HD + sub * 8;
        const int wide = (reinterpret_cast<uintptr_t>(to) & 31) == 0 && (p.ld & 7) == 0 ? 2 : (reinterpret_cast<uintptr_t>(to) & 15) == 0 && (p.ld & 3) == 0 ? 1 : 0;
        uint32_t w[kReadRows];
        __half m[kReadRows];
        __nv_bfloat16 d[kReadRows];
#pragma unroll
        for (int n = 0; n < kReadRows; n++) {
            const RowPlace at = places[min(n, n_rows - 1)];
            const int pp = at.pos & 15;
            const uint8_t *block = at.page + h * q4_block_bytes(HD);
            m[n] = *reinterpret_cast<const __half *>(block + (V ? q4_v_offset(HD, pp, g) : q4_k_offset(HD, pp, g)));
            d[n] = *reinterpret_cast<const __nv_bfloat16 *>(block + (V ? q4_v_step(HD, pp, g) : q4_k_step(HD, pp, g)));
            w[n] = *reinterpret_cast<const uint32_t *>(block + (V ? q4_v_code(HD, pp, 2 * t, g) : q4_k_code(HD, pp, t, g)));
            if (V) w[n] ^= q4_v_flip(pp);
        }
#pragma unroll
        for (int n = 0; n < kReadRows; n++) {
            if (n >= n_rows) break;
            const float off = __half2float(m[n]), df = __bfloat162float(d[n]);
            float x[8];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint32_t u = k ? w[n] >> 16 : w[n], turned = __byte_perm(w[n], 0, k ? 0x0023 : 0x0001);
                x[4 * k] = fmaf(df * 0x1p-6f, bits_as_float(u, 0x3c0u), off);
                x[4 * k + 1] = fmaf(df * 0x1p-10f, bits_as_float(u, 0x3c00u), off);
                x[4 * k + 2] = fmaf(df * 0x1p-2f, bits_as_float(u, 0x3cu), off);
                x[4 * k + 3] = fmaf(df * 0x1p-6f, bits_as_float(turned, 0x3c0u), off);
            }
            store8(to, x, wide);
            to += p.ld;
        }
    }
}
template <int HD>
__global__ void __launch_bounds__(256) q4_read_kernel(const __grid_constant__ RowsParams p) {
    __shared__ RowPlace places[kReadRows];
    const int row0 = blockIdx.x * kReadRows;
    find_places<kReadRows>(p, row0, (size_t)p.n_kv_heads * q4_block_bytes(HD), places);
    __syncthreads();
    if (blockIdx.y == 0)
        read_rows<HD, false>(p, places, row0);
    else
        read_rows<HD, true>(p, places, row0);
}

// FP16 and FP32 pages: eight elements a thread, both directions.
template <typename T, bool APPEND>
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ RowsParams p, int hd) {
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
    ProfScope prof(c, st, APPEND ? PROF_ROPE_APPEND : PROF_OTHER, (double)n_tokens * p->n_kv_heads * (8.0 * hd + p->row_bytes()));
    if (p->dtype == kKvQ4 && APPEND) {
        // Several positions to a CTA hide the loads once there are CTAs for every SM many times over, one gives few positions more SMs (eight heads of 128, one
        // and four: 592 positions 6.2 and 12.0 us, 2368 10.6 and 12.8, 4736 both 16.5, 8156 26 and 24).
        const int each = n_tokens >= c->sm_count * 32 ? kAppendRows : 1;
        const dim3 grid((unsigned)((n_tokens + each - 1) / each), 2), block((unsigned)std::min(256, (p->n_kv_heads * (hd / 8) + 31) / 32 * 32));
        if (each == 1)
            JUNO_CUDA_TRY(launch_pdl(hd == 128 ? q4_append_kernel<128, 1> : q4_append_kernel<64, 1>, grid, block, 0, st, a));
        else
            JUNO_CUDA_TRY(launch_pdl(hd == 128 ? q4_append_kernel<128, kAppendRows> : q4_append_kernel<64, kAppendRows>, grid, block, 0, st, a));
    } else if (p->dtype == kKvQ4) {
        const dim3 grid((unsigned)((n_tokens + kReadRows - 1) / kReadRows), 2), block((unsigned)std::min(256, (p->n_kv_heads * (hd / 8) + 31) / 32 * 32));
        JUNO_CUDA_TRY(launch_pdl(hd == 128 ? q4_read_kernel<128> : q4_read_kernel<64>, grid, block, 0, st, a));
    } else {
        const unsigned grid = (unsigned)(((int64_t)n_tokens * 2 * p->n_kv_heads * (hd / 8) + 255) / 256);
        p->dtype == 0 ? rows_kernel<__half, APPEND><<<grid, 256, 0, st>>>(a, hd) : rows_kernel<float, APPEND><<<grid, 256, 0, st>>>(a, hd);
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
__global__ void __launch_bounds__(256) weights_kernel(const __grid_constant__ CacheRows rows, float *weights, int layer, int n_layers, int n_kv_heads, int track_tokens, float *w, int64_t ld) {
    const int i = blockIdx.z, h = blockIdx.y, pos = blockIdx.x * 256 + threadIdx.x;
    pdl_launch_dependents();
    pdl_wait();
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
    int len, keep, recent, track, slot, new_pages;  // new_pages: the first of the row's new pages among those of all rows
};
constexpr int kRowWords = sizeof(EvictRow) / sizeof(int32_t), kEvictWords = 900;
struct EvictParams {
    int32_t in[kEvictWords];  // the rows, then new pages of all of them: in the launch where they fit, else in `far`
    const int32_t *far;
    const int32_t *table;  // as it was before: the rows' old pages
    uint8_t *pool;
    int n, n_pages, n_kv_heads, n_layers, track_tokens, max_pages_per_seq;
    float *weights;
    int32_t *kept;  // [layer][row][kv_head][kept_ld]
    int kept_ld;
};
__device__ __forceinline__ int evict_word(const EvictParams &p, int k) { return p.far ? p.far[k] : p.in[k]; }
__device__ __forceinline__ EvictRow evict_row(const EvictParams &p, int i) {
    const int k = i * kRowWords;
    return {evict_word(p, k), evict_word(p, k + 1), evict_word(p, k + 2), evict_word(p, k + 3), evict_word(p, k + 4), evict_word(p, k + 5)};
}
__device__ __forceinline__ int old_page(const EvictParams &p, const EvictRow &r, int pos) { return p.table[(size_t)r.slot * p.max_pages_per_seq + (pos >> 4)]; }
__device__ __forceinline__ int new_page(const EvictParams &p, const EvictRow &r, int pos) { return evict_word(p, p.n * kRowWords + r.new_pages + (pos >> 4)); }

// Order of weights as whole numbers: larger weight, larger key; both zeros alike, a NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_weight(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }  // 0 becomes a NaN again

constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32, kSelectCached = 24576, kBins = 2048;

// Sum over the threads of the block before this one, in *all the sum over all of them.  `sums`: kSelectWarps words.
__device__ __forceinline__ unsigned block_before(unsigned v, unsigned *sums, unsigned *all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned upto = v;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += y;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    unsigned s = lane < kSelectWarps ? sums[lane] : 0u, w = s;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, w, x);
        if (lane >= x) w += y;
    }
    *all = __shfl_sync(0xffffffffu, w, 31);
    const unsigned before = __shfl_sync(0xffffffffu, w - s, warp);
    __syncthreads();
    return before + upto - v;
}

// One CTA per (sequence, layer, head): which positions stay, in order, and their weights.  The weight that decides (the need-th largest) is found digit by
// digit, 11, 11 and 10 bits, with a count of every digit in shared memory: at most three passes over the weights, whatever they are, two where
// all weights that share the digits so far stay.  Up to kSelectCached weights are
// read from memory once.  Six sequences of up to 8192 positions, four layers, eight heads: 20 us, a chain of barriers and passes over shared memory (1024 threads
// instead of 512 take as long).
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
    const int h = blockIdx.x, layer = blockIdx.y, i = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait();
    const EvictRow r = evict_row(p, i);
    float *w = p.weights + (((size_t)r.track * p.n_layers + layer) * p.n_kv_heads + h) * p.track_tokens;
    int32_t *kept = p.kept + (((size_t)layer * p.n + i) * p.n_kv_heads + h) * p.kept_ld;
    for (int64_t j = r.keep + tid; j < p.kept_ld; j += kSelectThreads) kept[j] = -1;
    if (r.keep == r.len) {
        for (int j = tid; j < r.keep; j += kSelectThreads) kept[j] = j;
        return;
    }
    extern __shared__ uint32_t keys[];  // kSelectCached
    __shared__ unsigned bins[kBins], sums[kSelectWarps], digit_s, left_s, whole_s;
    const int old = r.len - r.recent;  // candidates
    const bool whole = r.len <= kSelectCached;
    for (int j = tid; j < kBins; j += kSelectThreads) bins[j] = 0;
    if (whole)
        for (int j = tid; j < r.len; j += kSelectThreads) keys[j] = weight_key(w[j]);
    __syncthreads();
    unsigned need = (unsigned)(r.keep - r.recent), key = 0;
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const unsigned mask = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u, digits = pass == 2 ? 1023u : 2047u;
        if (whole) {
            for (int j = tid; j < old; j += kSelectThreads) {
                const uint32_t u = keys[j];
                if ((u & mask) == key) atomicAdd(&bins[u >> shift & digits], 1u);
            }
        } else {
            for (int j = tid; j < old; j += kSelectThreads) {
                const uint32_t u = weight_key(w[j]);
                if ((u & mask) == key) atomicAdd(&bins[u >> shift & digits], 1u);
            }
        }
        __syncthreads();
        // from the largest digit down: the one in which the need-th weight lies
        constexpr int EACH = kBins / kSelectThreads;
        unsigned mine = 0, count[EACH], all;
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            mine += count[k] = bins[kBins - 1 - EACH * tid - k];
            bins[kBins - 1 - EACH * tid - k] = 0;  // for the next pass
        }
        unsigned before = block_before(mine, sums, &all);
        if (before < need && need <= before + mine) {
#pragma unroll
            for (int k = 0; k < EACH; k++) {
                if (before < need && need <= before + count[k]) {
                    digit_s = kBins - 1 - EACH * tid - k;
                    left_s = need - before;
                    whole_s = left_s == count[k];
                }
                before += count[k];
            }
        }
        __syncthreads();
        if (need > 0) {
            key |= digit_s << shift;
            need = left_s;
            if (whole_s && key > 0) {  // all that begin with these digits stay
                key--;
                need = 0;
                break;
            }
        } else {
            key = 0xffffffffu;  // no weight has this key
            break;
        }
    }
    // positions above `key` stay, and the first `need` of those that equal it.  A warp has a run of the positions; those of one stretch are all read before any
    // weight moves, and weights move to the front.
    unsigned done = 0, equal = 0;
    for (int base = 0; base < r.len; base += kSelectCached) {
        const int n = min(kSelectCached, r.len - base), run = (n + kSelectWarps * 32 - 1) / (kSelectWarps * 32) * 32, from = min(n, warp * run), to = min(n, from + run);
        if (!whole) {
            __syncthreads();
            for (int j = tid; j < n; j += kSelectThreads) keys[j] = weight_key(w[base + j]);
            __syncthreads();
        }
        unsigned same = 0, above = 0;  // of this warp
        for (int j = from + lane; j - lane < to; j += 32) {
            const uint32_t u = j < to ? keys[j] : 0u;
            same += __popc(__ballot_sync(0xffffffffu, u == key && j < to && base + j < old));
            above += __popc(__ballot_sync(0xffffffffu, j < to && (u > key || base + j >= old)));
        }
        unsigned all;
        unsigned rank = equal + __shfl_sync(0xffffffffu, block_before(lane == 0 ? same : 0u, sums, &all), 0);
        equal += all;
        const unsigned taken = rank < need ? min(same, need - rank) : 0u;
        unsigned out = done + __shfl_sync(0xffffffffu, block_before(lane == 0 ? above + taken : 0u, sums, &all), 0);
        done += all;
        for (int j = from + lane; j - lane < to; j += 32) {
            const int at = base + j;
            const uint32_t u = j < to ? keys[j] : 0u;
            const bool eq = u == key && j < to && at < old;
            const unsigned eqs = __ballot_sync(0xffffffffu, eq);
            const bool stays = j < to && (u > key || at >= old || (eq && rank + __popc(eqs & ((1u << lane) - 1u)) < need));
            const unsigned st = __ballot_sync(0xffffffffu, stays);
            if (stays) {
                const unsigned to_j = out + __popc(st & ((1u << lane) - 1u));
                kept[to_j] = at;
                w[to_j] = key_weight(u);
            }
            rank += __popc(eqs);
            out += __popc(st);
        }
    }
}

// A row in pieces, one to a lane of sixteen: the numbers of keys and values in 16 bytes, steps and offsets of both in 2 NG.  Where piece i of position pp
// lies: at + pp * stride, but for the values' numbers, whose pieces are permuted.
template <int HD>
struct Q4Piece {
    static constexpr int NG = HD / kQ4Group, CODES = HD / 32, PIECES = 2 * CODES + 4;
    int kind, at, stride, group;  // 0: 16 bytes, 1: values' 16 bytes, 2: NG half words, 3: none
    __device__ __forceinline__ explicit Q4Piece(int i) : kind(3), at(0), stride(0), group(0) {
        if (i < CODES) {
            kind = 0, at = q4_k_code(HD, 0, 0, 0) + 16 * i, stride = HD / 2;
        } else if (i < 2 * CODES) {
            kind = 1, at = 10 * HD, stride = HD / 2, group = i - CODES;
        } else if (i < PIECES) {
            const int k = i - 2 * CODES;
            kind = 2, at = k == 0 ? q4_k_step(HD, 0, 0) : k == 1 ? q4_k_offset(HD, 0, 0) : k == 2 ? q4_v_step(HD, 0, 0) : q4_v_offset(HD, 0, 0), stride = 2 * NG;
        }
    }
    __device__ __forceinline__ int place(int pp) const { return at + pp * stride + (kind == 1 ? 16 * q4_v_piece(HD, pp, group) : 0); }
    static __device__ __forceinline__ void flip(uint4 &v, int pp) {
        const uint32_t f = q4_v_flip(pp);
        v = make_uint4(v.x ^ f, v.y ^ f, v.z ^ f, v.w ^ f);
    }
    __device__ __forceinline__ uint4 load(const uint8_t *block, int pp) const {
        const uint8_t *b = block + place(pp);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (kind <= 1) {
            v = *reinterpret_cast<const uint4 *>(b);
            if (kind == 1) flip(v, pp);
        } else if (kind == 2 && NG == 4) {
            const uint2 y = *reinterpret_cast<const uint2 *>(b);
            v.x = y.x;
            v.y = y.y;
        } else if (kind == 2)
            v.x = *reinterpret_cast<const uint32_t *>(b);
        return v;
    }
    __device__ __forceinline__ void store(uint8_t *block, int pp, uint4 v) const {
        uint8_t *b = block + place(pp);
        if (kind == 1) flip(v, pp);
        if (kind <= 1)
            *reinterpret_cast<uint4 *>(b) = v;
        else if (kind == 2 && NG == 4)
            *reinterpret_cast<uint2 *>(b) = make_uint2(v.x, v.y);
        else if (kind == 2)
            *reinterpret_cast<uint32_t *>(b) = v.x;
    }
};

// The rows that stay, into fresh pages: a warp has one page of one head, two rows a step, all eight loads of a lane under way together.  24 sequences and layers times
// 1001 rows of eight heads: 31 MB read and written in 26 us; DRAM hands out 80 MB for it, as the four pieces of 8 bytes that a row has beside its numbers lie in
// four places.
template <int HD>
__global__ void __launch_bounds__(256) evict_gather_kernel(const __grid_constant__ EvictParams p) {
    static_assert(Q4Piece<HD>::PIECES <= 16, "a piece to a lane");
    const int i = blockIdx.z, layer = blockIdx.y, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();
    const EvictRow r = evict_row(p, i);
    if (r.keep == r.len) return;
    const int unit = blockIdx.x * 8 + (threadIdx.x >> 5), h = unit % p.n_kv_heads, base = unit / p.n_kv_heads * kPageTokens, n = min(kPageTokens, r.keep - base);
    if (n <= 0) return;
    const int32_t *kept = p.kept + (((size_t)layer * p.n + i) * p.n_kv_heads + h) * p.kept_ld + base;
    const int src = kept[min(lane, n - 1)], src_page = old_page(p, r, src);
    const size_t page_bytes = (size_t)p.n_kv_heads * q4_block_bytes(HD);
    uint8_t *plane = p.pool + (size_t)layer * p.n_pages * page_bytes + h * q4_block_bytes(HD);
    uint8_t *to = plane + new_page(p, r, base) * page_bytes;
    const Q4Piece<HD> piece(lane & 15);
    uint4 v[kPageTokens / 2];
#pragma unroll
    for (int k = 0; k < kPageTokens / 2; k++) {  // rows behind the last one: that one again
        const int j = min(2 * k + (lane >> 4), n - 1), at = __shfl_sync(0xffffffffu, src, j), page = __shfl_sync(0xffffffffu, src_page, j);
        v[k] = piece.load(plane + page * page_bytes, at & 15);
    }
#pragma unroll
    for (int k = 0; k < kPageTokens / 2; k++)
        if (2 * k + (lane >> 4) < n) piece.store(to, 2 * k + (lane >> 4), v[k]);
}

// The same in place, for a pool without enough free pages: one CTA per (sequence, layer, head) takes kMoveRows rows a step, in order.  A row moves to the
// front or stays, so that what a step overwrites has been read by it or by an earlier one.
constexpr int kMoveThreads = 512, kMoveRows = kMoveThreads / 16 * 2;
template <int HD>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
    const int h = blockIdx.x, layer = blockIdx.y, i = blockIdx.z, sub = threadIdx.x >> 4;
    pdl_launch_dependents();
    pdl_wait();
    const EvictRow r = evict_row(p, i);
    if (r.keep == r.len) return;
    const int32_t *kept = p.kept + (((size_t)layer * p.n + i) * p.n_kv_heads + h) * p.kept_ld;
    const size_t page_bytes = (size_t)p.n_kv_heads * q4_block_bytes(HD);
    uint8_t *plane = p.pool + (size_t)layer * p.n_pages * page_bytes + h * q4_block_bytes(HD);
    const Q4Piece<HD> piece(threadIdx.x & 15);
    for (int base = 0; base < r.keep; base += kMoveRows) {
        uint4 v[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int j = base + sub + k * (kMoveThreads / 16), src = j < r.keep ? kept[j] : 0;
            if (j < r.keep) v[k] = piece.load(plane + old_page(p, r, src) * page_bytes, src & 15);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int j = base + sub + k * (kMoveThreads / 16);
            if (j < r.keep) piece.store(plane + new_page(p, r, j) * page_bytes, j & 15, v[k]);
        }
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

int cache_call_distinct(const juno_kvpool *p, int n, juno_seq *const *seqs, bool weights_only) {
    std::vector<char> seen((size_t)p->max_slots, 0);
    for (int i = 0; i < n; i++) {
        if (weights_only && seqs[i]->track < 0) continue;
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
        rows->push_back({seqs[i]->slot, positions[i], (int)sum, seqs[i]->track, 0});
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
        std::vector<int32_t> table;
        int rc = JUNO_OK;
        for (int i = 0; rc == JUNO_OK && i < n; i++)
            if (counts[i]) rc = seq_reserve(seqs[i], positions[i], positions[i] + counts[i], s.st, &table);
        JUNO_TRY(table_store_pairs(p, table, s.st));  // of those that have their pages, too, when others do not
        JUNO_TRY(rc);
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
            rows.push_back({seqs[i]->slot, counts[i], i, seqs[i]->track, 0});
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
            JUNO_CUDA_TRY(launch_pdl(weights_kernel<true>, grid, dim3(256), 0, s.st, r, p->weights, layer, p->n_layers, p->n_kv_heads, p->track_tokens, w_dev, ld));
        else
            JUNO_CUDA_TRY(launch_pdl(weights_kernel<false>, grid, dim3(256), 0, s.st, r, p->weights, layer, p->n_layers, p->n_kv_heads, p->track_tokens, w_dev, ld));
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
        int most = 1;
        for (int i = 0; i < n; i++) most = std::max(most, seqs[i]->len);
        const int kept_ld = keep;
        keep = std::min(keep, most);  // where no sequence is longer nothing is cut
        recent = std::min(recent, keep);
        // The rows go to fresh pages where the pool has enough of them, which all warps can fill side by side; else they move within their pages, but for pages
        // that another sequence holds too: those are left to it, and their rows go to fresh ones.  Fresh pages and rows moved in place, four layers of eight heads, a call
        // and its wait: one sequence from 2600 to 2048 positions 39 and 96 us, from 8192 to 4000 55 and 199, six from 8192 to 1001 75 and 93.
        const int np = (keep + kPageTokens - 1) / kPageTokens;
        size_t shared = 0, cut = 0;
        for (int i = 0; i < n; i++) {
            const juno_seq *s = seqs[i];
            if (s->len <= keep) continue;
            cut++;
            for (int j = 0; j < np; j++) shared += p->page_refs[(size_t)s->pages[(size_t)j]] > 1;
        }
        if (shared > p->free_pages.size()) {
            set_error("KV pool exhausted: %zu pages free, %zu needed for rows of shared pages", p->free_pages.size(), shared);
            return JUNO_ERR_OOM;
        }
        const bool fresh = cut * np <= p->free_pages.size();
        std::vector<EvictRow> rows;
        std::vector<int32_t> pages;
        size_t next = p->free_pages.size();
        for (int i = 0; i < n; i++) {
            const juno_seq *s = seqs[i];
            EvictRow r{s->len, std::min(s->len, keep), std::min(s->len, recent), s->track, s->slot, (int)pages.size()};
            if (s->len > keep)
                for (int j = 0; j < np; j++) {
                    const int pg = s->pages[(size_t)j];
                    pages.push_back(fresh || p->page_refs[(size_t)pg] > 1 ? p->free_pages[--next] : pg);
                }
            rows.push_back(r);
        }
        std::vector<int32_t> table;
        table.reserve(2 * pages.size());
        CacheStream st(c, stream);
        JUNO_TRY(st.status);
        const size_t row_words = rows.size() * kRowWords, words = row_words + pages.size();
        const size_t word_bytes = words <= kEvictWords ? 0 : (words * sizeof(int32_t) + 255) & ~(size_t)255;
        const size_t kept_bytes = kept_dev ? 0 : (size_t)p->n_layers * n * p->n_kv_heads * keep * sizeof(int32_t);
        uint8_t *scratch = nullptr;
        if (word_bytes + kept_bytes) JUNO_TRY(cache_scratch(c, word_bytes + kept_bytes, &scratch));
        EvictParams a;
        a.far = nullptr;
        if (word_bytes) {
            std::vector<int32_t> all(words);
            memcpy(all.data(), rows.data(), row_words * sizeof(int32_t));
            memcpy(all.data() + row_words, pages.data(), pages.size() * sizeof(int32_t));
            JUNO_TRY(cache_words(c, all.data(), words, reinterpret_cast<int32_t *>(scratch), st.st));
            a.far = reinterpret_cast<const int32_t *>(scratch);
        } else {
            memcpy(a.in, rows.data(), row_words * sizeof(int32_t));
            if (!pages.empty()) memcpy(a.in + row_words, pages.data(), pages.size() * sizeof(int32_t));
        }
        a.table = p->d_table;
        a.max_pages_per_seq = p->max_pages_per_seq;
        a.pool = static_cast<uint8_t *>(p->k);
        a.n = n;
        a.n_pages = p->n_pages;
        a.n_kv_heads = p->n_kv_heads;
        a.n_layers = p->n_layers;
        a.track_tokens = p->track_tokens;
        a.weights = p->weights;
        a.kept = kept_dev ? kept_dev : reinterpret_cast<int32_t *>(scratch + word_bytes);
        a.kept_ld = kept_dev ? kept_ld : keep;
        const dim3 heads((unsigned)p->n_kv_heads, (unsigned)p->n_layers, (unsigned)n), units((unsigned)((np * p->n_kv_heads + 7) / 8), (unsigned)p->n_layers, (unsigned)n);
        const size_t cached = kSelectCached * sizeof(float);
        static bool set[64] = {false};  // per device
        if (!set[c->device & 63]) {
            JUNO_CUDA_TRY(cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cached));
            set[c->device & 63] = true;
        }
        {
            ProfScope prof(c, st.st, PROF_OTHER, 0);
            JUNO_CUDA_TRY(launch_pdl(evict_select_kernel, heads, dim3(kSelectThreads), cached, st.st, a));
            if (fresh)
                JUNO_CUDA_TRY(launch_pdl(p->head_dim == 128 ? evict_gather_kernel<128> : evict_gather_kernel<64>, units, dim3(256), 0, st.st, a));
            else
                JUNO_CUDA_TRY(launch_pdl(p->head_dim == 128 ? evict_move_kernel<128> : evict_move_kernel<64>, heads, dim3(kMoveThreads), 0, st.st, a));
        }
        c->kernel_launches += 2;
        p->free_pages.resize(next);
        for (int i = 0; i < n; i++) {
            juno_seq *s = seqs[i];
            if (s->len <= keep) continue;
            int32_t *row = p->h_table + (size_t)s->slot * p->max_pages_per_seq;
            for (int j = 0; j < (int)s->pages.size(); j++) {
                const int old = s->pages[(size_t)j], now = j < np ? pages[(size_t)rows[(size_t)i].new_pages + j] : -1;
                if (now == old) continue;
                if (--p->page_refs[(size_t)old] == 0) p->free_pages.push_back(old);
                if (now < 0) continue;
                p->page_refs[(size_t)now] = 1;
                s->pages[(size_t)j] = row[j] = now;
                table.push_back(s->slot * p->max_pages_per_seq + j);
                table.push_back(now);
            }
            s->pages.resize((size_t)np);
            s->len = keep;
        }
        return table_store_pairs(p, table, st.st);
    });
}

}  // extern "C"
