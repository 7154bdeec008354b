// What the kernels over the paged 4-bit cache share: the cache and batch as a
// kernel sees them, the search for a token's sequence and its rows' places,
// and the argument checks of the entry points.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "dm_device.cuh"
#include "dm_internal.h"

namespace dm {

constexpr int kKvErrRange = 1;  // a position that the page table, the pages or the rotary tables do not cover
constexpr int kKvErrWait = 2;   // a bounded wait gave up

struct KvView {
    uint8_t *codes;
    uint16_t *scales;
    const int32_t *table, *q_start, *kv_len;
    int64_t tstride, pages;
    int32_t cols, seqs, tokens, nkv, ps, pshift;
    int *err;
};

inline KvView kv_view(const dm_kv4_cache *c, const dm_kv4_batch *b) {
    KvView v;
    v.codes = (uint8_t *)c->codes;
    v.scales = (uint16_t *)c->scales;
    v.table = b->page_table;
    v.q_start = b->q_start;
    v.kv_len = b->kv_len;
    v.tstride = b->table_stride;
    v.pages = c->pages;
    v.cols = b->table_cols;
    v.seqs = b->seqs;
    v.tokens = b->tokens;
    v.nkv = c->kv_heads;
    v.ps = c->page_size;
    v.pshift = 0;
    while ((1 << v.pshift) < c->page_size) ++v.pshift;
    v.err = (int *)b->error;
    return v;
}

// The sequence of token t: the number of sequences that end at or before it,
// 32 at a time (the whole warp calls this).
__device__ __forceinline__ int kv_sequence(const KvView &v, int t, int lane) {
    int b = 0;
    for (int j0 = 0; j0 < v.seqs; j0 += 32) {
        const int j = j0 + lane;
        const bool before = j < v.seqs && v.q_start[j + 1] <= t;
        b += __popc(__ballot_sync(0xffffffffu, before));
    }
    return b;
}

// The page of position p (>= 0) of sequence b, or -1 when the table or the pages
// do not cover it (recorded if p >= seen: a page that nobody looks into need not be there).
__device__ __forceinline__ int64_t kv_page(const KvView &v, int b, int64_t p, int64_t seen = 0) {
    const int64_t col = p >> v.pshift;
    const int64_t page = col < v.cols ? v.table[(int64_t)b * v.tstride + col] : -1;
    if (page >= 0 && page < v.pages) return page;
    if (p >= seen) atomicExch(v.err, kKvErrRange);
    return -1;
}

// Refuses with a message, without an allocation that could throw.
inline int kv_refuse(char *err, size_t len, const char *fmt, ...) {
    if (err && len) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(err, len, fmt, ap);
        va_end(ap);
    }
    return DM_EINVAL;
}

inline int kv_launched(const char *what, cudaError_t e, char *err, size_t len) {
    if (e == cudaSuccess) e = cudaGetLastError();
    else cudaGetLastError();  // the error is reported here, not by a later call
    if (e == cudaSuccess) return DM_OK;
    kv_refuse(err, len, "%s: %s", what, cudaGetErrorString(e));
    return DM_ECUDA;
}

inline bool kv_aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The cache and batch of an entry point: DM_OK, or the refusal.
inline int kv_check_args(const char *who, const dm_kv4_cache *c, const dm_kv4_batch *b, char *err, size_t len) {
    if (!c || !b) return kv_refuse(err, len, "%s: null cache or batch", who);
    if (!c->codes || !c->scales || c->pages < 1 || c->pages > INT32_MAX || c->kv_heads < 1 || c->kv_heads > 4096)
        return kv_refuse(err, len, "%s: bad cache (null buffer, no pages or kv heads)", who);
    if (c->head_dim != 64 && c->head_dim != 128)
        return kv_refuse(err, len, "%s: head_dim must be 64 or 128, not %d", who, c->head_dim);
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return kv_refuse(err, len, "%s: page_size must be 16, 32, 64, 128 or 256, not %d", who, c->page_size);
    if (!kv_aligned(c->codes, 16) || !kv_aligned(c->scales, 16))
        return kv_refuse(err, len, "%s: the cache's buffers must be 16-byte aligned", who);
    if (!b->page_table || !b->q_start || !b->kv_len || !b->error || b->seqs < 1 || b->tokens < 0 || b->max_q < 1 ||
        b->table_cols < 1 || b->table_stride < b->table_cols)
        return kv_refuse(err, len, "%s: bad batch (null array, no sequences, or a negative size)", who);
    if (!kv_aligned(b->error, 4)) return kv_refuse(err, len, "%s: the error word is not aligned", who);
    return DM_OK;
}

}  // namespace dm
