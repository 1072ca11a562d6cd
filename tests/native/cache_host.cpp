// Test-only host program: calls on pools and sequences that are put together by hand, without a GPU.  `cache_host NAME` runs one check and exits 0 if it holds.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>

#include "../../include/juno_b200.h"
#include "../../juno_b200/csrc/attn.cuh"

using namespace juno;

// The program's own allocation, which the library uses too: the one after `g_left` others fails.
static long g_left = -1;
void *operator new(size_t n) {
    if (g_left == 0) throw std::bad_alloc();
    if (g_left > 0) g_left--;
    if (void *p = malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
void operator delete(void *p) noexcept { free(p); }
void operator delete(void *p, size_t) noexcept { free(p); }

#define WANT(x)                                                        \
    do {                                                               \
        if (!(x)) {                                                    \
            printf("line %d: %s (%s)\n", __LINE__, #x, juno_last_error()); \
            return 1;                                                  \
        }                                                              \
    } while (0)

// A pool of 64 pages and 8 slots whose device memory does not exist.
struct Pool {
    juno_ctx ctx;
    juno_kvpool pool;
    int32_t table[8 * 64];
    explicit Pool(int dtype) {
        ctx.magic = kMagicCtx;
        ctx.device = 0;
        ctx.sm_count = 148;
        ctx.stream = nullptr;
        pool.magic = kMagicPool;
        pool.ctx = &ctx;
        pool.n_layers = 2;
        pool.n_kv_heads = 2;
        pool.head_dim = 64;
        pool.n_pages = 64;
        pool.dtype = dtype;
        pool.page_tokens = 16;
        pool.elem_bytes = dtype == 0 ? 2 : dtype == 1 ? 4 : 0;
        pool.max_slots = 8;
        pool.max_pages_per_seq = 64;
        pool.k = pool.v = nullptr;
        pool.d_table = nullptr;
        pool.h_table = table;
        pool.owned_by_model = 0;
        memset(table, 0, sizeof table);
        for (int i = 63; i >= 0; i--) pool.free_pages.push_back(i);
        pool.page_refs.assign(64, 0);
        for (int i = 7; i >= 0; i--) pool.free_slots.push_back(i);
    }
    // a sequence of `len` positions, with their pages; track: its weight plane
    juno_seq *seq(int len, int track = -1) {
        juno_seq *s = nullptr;
        if (juno_kvseq_create(&pool, 512, &s) != JUNO_OK) return nullptr;
        for (int i = 0; i < (len + 15) / 16; i++) {
            const int pg = pool.free_pages.back();
            pool.free_pages.pop_back();
            pool.page_refs[pg] = 1;
            s->pages.push_back(pg);
            table[s->slot * 64 + i] = pg;
        }
        s->len = len;
        s->track = track;
        return s;
    }
};

// Rows of one sequence would add to the same weights: refused, as for device memory.
static int twice() {
    Pool p(3);
    juno_seq *a = p.seq(20, 0), *b = p.seq(20), *two[2] = {a, a}, *mixed[3] = {b, a, a};
    float x[3 * 256] = {0};
    WANT(juno_attn_decode(&p.ctx, &p.pool, 0, 2, two, 4, x, x) == JUNO_ERR_INVALID_ARG && strstr(juno_last_error(), "there twice"));
    WANT(juno_attn_decode(&p.ctx, &p.pool, 0, 3, mixed, 4, x, x) == JUNO_ERR_INVALID_ARG && strstr(juno_last_error(), "there twice"));
    return 0;
}

// A sequence without weights may be there several times beside one that has some: what stops such a call here comes after its checks.
static int beside() {
    Pool p(3);
    juno_seq *a = p.seq(20, 0), *b = p.seq(20), *mixed[3] = {b, a, b};
    float x[3 * 256] = {0};
    const int rc = juno_attn_decode(&p.ctx, &p.pool, 0, 3, mixed, 4, x, x);
    WANT(rc != JUNO_OK && !strstr(juno_last_error(), "there twice"));
    return 0;
}

// What reaches a pool's memory through a sequence is refused once the pool, or its context, is closed; a handle of an open pool can be freed then.
static int closed() {
    for (int which = 0; which < 2; which++) {
        Pool p(3);
        juno_seq *a = p.seq(20), *b = nullptr;
        float x[2 * 128] = {0}, w = 0;
        (which ? p.ctx.magic : p.pool.magic) = kMagicDead;
        WANT(juno_seq_append_kv(a, 0, 3, 1, x, x) == JUNO_ERR_CLOSED);
        WANT(juno_seq_append_kv(a, 0, 20, 2, x, x) == JUNO_ERR_CLOSED);
        WANT(juno_seq_fork(a, 0, &b) == JUNO_ERR_CLOSED && !b);
        WANT(juno_seq_fork(a, 20, &b) == JUNO_ERR_CLOSED && !b);
        WANT(juno_kvpool_track(&p.pool, 1, 16) == JUNO_ERR_CLOSED);
        WANT(juno_kvseq_create(&p.pool, 16, &b) == JUNO_ERR_CLOSED && !b);
        p.pool.weights = &w;
        WANT(juno_seq_track(a) == JUNO_ERR_CLOSED);
        WANT(a->len == 20 && a->pages.size() == 2);
        WANT(which == 0 || (juno_seq_free(a) == JUNO_OK && juno_seq_free(a) == JUNO_ERR_CLOSED));
    }
    return 0;
}

// Positions whose end passes 32 bits are beyond the limit, whatever the sum wraps to.
static int far() {
    for (int dtype : {0, 1, 3}) {
        Pool p(dtype);
        juno_seq *a = p.seq(20);
        float x[2 * 128] = {0};
        WANT(juno_seq_append_kv(a, 0, 2147483647, 1, x, x) == JUNO_ERR_INVALID_ARG && strstr(juno_last_error(), "limit of 512"));
        WANT(juno_seq_append_kv(a, 0, 2147483640, 2147483647, x, x) == JUNO_ERR_INVALID_ARG);
        WANT(juno_seq_append_kv(a, 0, 5, 2147483647, x, x) == JUNO_ERR_INVALID_ARG);
        WANT(juno_seq_append_kv(a, 0, 512, 1, x, x) == JUNO_ERR_INVALID_ARG);
        WANT(a->len == 20 && a->pages.size() == 2);
    }
    return 0;
}

// A call that runs out of host memory says so, and leaves pages, slots and the list of changes as they were.
static int memory() {
    for (long n = 0;; n++) {
        Pool p(3);
        juno_seq *a = p.seq(20), *b = nullptr;
        std::vector<int32_t> later(3, 7);
        const size_t pages = p.pool.free_pages.size();
        bool thrown = false;
        int rc = JUNO_OK;
        g_left = n;
        try {
            rc = seq_reserve(a, 20, 300, nullptr, &later);
        } catch (const std::bad_alloc &) {
            thrown = true;
        }
        g_left = -1;
        if (!thrown) {
            WANT(rc == JUNO_OK && a->pages.size() == 19 && later.size() == 3 + 2 * 17 && p.pool.free_pages.size() == pages - 17);
            WANT(n > 0);
            break;
        }
        WANT(a->pages.size() == 2 && later.size() == 3 && p.pool.free_pages.size() == pages);
    }
    for (long n = 0;; n++) {
        Pool p(3);
        juno_seq *a = p.seq(20), *b = nullptr;
        const size_t slots = p.pool.free_slots.size();
        g_left = n;
        const int rc = juno_seq_fork(a, 20, &b);  // without a GPU the page table does not reach it: an error, too
        g_left = -1;
        WANT(rc != JUNO_OK && !b && p.pool.free_slots.size() == slots && p.pool.page_refs[a->pages[0]] == 1 && p.pool.page_refs[a->pages[1]] == 1);
        if (rc != JUNO_ERR_OOM) {
            WANT(n > 0);
            break;
        }
    }
    for (long n = 0;; n++) {
        Pool p(0);
        juno_seq *b = nullptr;
        g_left = n;
        const int rc = juno_kvseq_create(&p.pool, 16, &b);
        g_left = -1;
        WANT((rc == JUNO_OK) == (b != nullptr) && p.pool.free_slots.size() == (b ? 7 : 8));
        if (b) break;
        WANT(rc == JUNO_ERR_OOM);
    }
    for (long n = 0; n < 2; n++) {
        Pool p(n ? 0 : 3);
        juno_seq *a = p.seq(20);
        float x[256] = {0};
        g_left = 0;
        const int decode = juno_attn_decode(&p.ctx, &p.pool, 0, 1, &a, 4, x, x), append = juno_seq_append_kv(a, 0, 20, 100, x, x);
        juno_kvpool *q = nullptr;
        const int create = juno_kvpool_create(&p.ctx, 1, 1, 64, 4, 0, &q);
        g_left = -1;
        WANT(decode == JUNO_ERR_OOM && append == JUNO_ERR_OOM && create == JUNO_ERR_OOM && !q && a->pages.size() == 2);
    }
    return 0;
}

// A freed sequence keeps its handle, and nothing that grows with its length.
static int freed() {
    Pool p(3);
    juno_seq *a = p.seq(300);
    WANT(a->pages.capacity() >= 19);
    WANT(juno_seq_free(a) == JUNO_OK && a->pages.capacity() == 0);
    WANT(p.pool.free_pages.size() == 64 && p.pool.free_slots.size() == 8);
    return 0;
}

// The lists of a pool are as long as it: they are made once the device has room for its pages, so that a pool that is far too large costs the host nothing.
static int huge() {
    Pool p(0);
    juno_kvpool *q = nullptr;
    g_left = 1;  // the pool itself
    const int rc = juno_kvpool_create(&p.ctx, 1, 1, 64, 2000000000, 0, &q);
    g_left = -1;
    WANT(rc != JUNO_OK && !q && strstr(juno_last_error(), "cudaMalloc of the KV pool"));
    return 0;
}

int main(int argc, char **argv) {
    setenv("CUDA_VISIBLE_DEVICES", "", 1);  // the pools' device memory does not exist: nothing may be launched, on a machine with a GPU neither
    const struct {
        const char *name;
        int (*run)();
    } checks[] = {{"twice", twice}, {"beside", beside}, {"closed", closed}, {"far", far}, {"memory", memory}, {"freed", freed}, {"huge", huge}};
    for (const auto &c : checks)
        if (argc == 2 && !strcmp(argv[1], c.name)) return c.run();
    printf("no such check\n");
    return 2;
}
