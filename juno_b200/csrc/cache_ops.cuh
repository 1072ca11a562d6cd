// Calls on cache pages that take device pointers and a stream: what append, read, attention, weights and eviction share.
#pragma once
#include <new>
#include <vector>

#include "attn.cuh"

namespace juno {

// One sequence of a call as its kernels see it.  The rows of a call travel with the launch up to kInlineRows of them, so that a call of a few sequences
// copies nothing; more lie in the context's working memory.
struct CacheRow {
    int slot;   // row of the page table
    int upto;   // append, read: first position; attention: positions to attend
    int first;  // the row's first unit of work among those of all rows (cached position of the call, context split): ascending
    int track;  // weight plane, -1 = none
    int share;  // attention: the share of the work that has the row's first page
};
constexpr int kInlineRows = 64;
struct CacheRows {
    const CacheRow *far;  // null: `in`
    int n;
    CacheRow in[kInlineRows];
};
#if defined(__CUDACC__)
__device__ __forceinline__ CacheRow cache_row(const CacheRows &r, int i) { return r.far ? r.far[i] : r.in[i]; }
// The row that unit `id` of the call's work belongs to: the last one with first <= id.
__device__ __forceinline__ int cache_find(const CacheRows &r, int id) {
    int lo = 0, hi = r.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((r.far ? r.far[mid].first : r.in[mid].first) <= id)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}
#endif

// The order of calls on several streams: all of a context's work on its pools is one sequence.  A call on a stream of the caller's begins after what the
// context's stream has so far, and the context's stream goes on after it; on the context's own stream nothing has to be done.  Streams that are being
// captured, and those of other devices, are refused: a graph would hold page tables and working memory of the moment.
class CacheStream {
public:
    CacheStream(juno_ctx *c, void *stream);
    ~CacheStream();
    int status = JUNO_OK;
    cudaStream_t st;

private:
    int join();
    juno_ctx *c_;
    bool joined_ = false;
};

// JUNO_ERR_INVALID_ARG while the context's stream is being captured: changes of the page table would be part of the graph, and be missing where they are due.
int cache_call_outside_graph(const juno_ctx *c);
// What every such call requires of its handles; a call that writes to a sequence has each one once.
int cache_call_check(juno_ctx *c, juno_kvpool *p, int layer, int n, juno_seq *const *seqs);
// weights_only: sequences that keep no weights may be there several times
int cache_call_distinct(const juno_kvpool *p, int n, juno_seq *const *seqs, bool weights_only = false);
// JUNO_ERR_INVALID_ARG unless p is memory that this context's device can use (device or managed memory of its own).
int device_memory(const juno_ctx *c, const void *p, const char *name);
// The context's working memory, at least `bytes`; what an earlier call left there is gone.
int cache_scratch(juno_ctx *c, size_t bytes, uint8_t **out);
// Grows a piece of working memory to `bytes` or more.
int cache_room(void **ptr, size_t *cur, size_t bytes);
// Fills `out` for `n` rows; `far`: room for them in the working memory when they are more than kInlineRows.
int cache_rows(juno_ctx *c, const CacheRow *rows, int n, CacheRow *far, CacheRows *out, cudaStream_t st);
inline size_t cache_rows_bytes(int n) { return n > kInlineRows ? ((size_t)n * sizeof(CacheRow) + 255) & ~(size_t)255 : 0; }
// Whole numbers that travel with a launch: neither the caller's memory nor a staging buffer has to outlive the call.
struct WordsByValue {
    int32_t v[2000];  // 8 KB of parameters
};
// Whole numbers to device memory.
int cache_words(juno_ctx *c, const int32_t *words, size_t n, int32_t *dst, cudaStream_t st);

// Rows [n_tokens][ld] of keys and values into the pages: row j belongs to the sequence of `rows` that holds unit j.  The pages exist and are writable.
int launch_kv_append(juno_ctx *c, const juno_kvpool *p, int layer, const CacheRow *rows, int n, int n_tokens, const float *k, const float *v, int64_t ld,
                     cudaStream_t st);
// Decode attention over 4-bit pages, lens[i] (null: all cached) positions of each sequence; adds to the weights of sequences that keep them.
// `word`: where its kernel reports a wait that it gave up.
int q4_attend(juno_ctx *c, juno_kvpool *p, int layer, int n, juno_seq *const *seqs, const int32_t *lens, int n_heads, const float *q, int64_t ldq, float *out,
              int64_t ldo, WaitWord word, cudaStream_t st);

// No C++ exception crosses the C ABI.
template <class F>
int guarded(F &&f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        set_error("out of host memory");
        return JUNO_ERR_OOM;
    } catch (...) {
        set_error("unexpected failure on the host");
        return JUNO_ERR_CUDA;
    }
}

}  // namespace juno
