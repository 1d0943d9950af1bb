// kv_cache.cuh -- the paged K/V cache object (zilla_kv_create) and the batch
// description that its append and its attention share.
//
// K and V are [pages][kv_heads][page][head_dim], bf16 or fp16: one head's keys of one page are
// contiguous, so a TMA box fetches them and a page's rows fill whole 128-byte lines.
#pragma once

#include "half_types.cuh"
#include "tc_common.cuh"

namespace zb {

struct KvCache {
    int pages = 0, page = 0, page_log2 = 0, kv_heads = 0, head_dim = 0, type = kBf16;
    int k_id = 0, v_id = 0;
    unsigned long long k_made = 0, v_made = 0;   // their allocations: a freed buffer's handle may come back as another's
    void *k = nullptr, *v = nullptr;
    CUtensorMap k_map, v_map;   // [pages * kv_heads * page][head_dim], box {min(head_dim, 64), box_rows}
    int box_rows = 0;           // rows of one TMA box: a page, 64 at most
    size_t floats = 0;          // registry floats of K, and of V
};

// The cache of an id; nullptr when unknown, or when one of its buffers was freed.
const KvCache *kv_get(int id);

// Error codes of the device error word.
enum KvErr : int {
    kErrKvLength = 0x4b560001,   // a sequence's rows or length do not fit the call's sizes
    kErrKvPage = 0x4b560002,     // a page number outside the cache, or a token behind the page table's end
    kErrDraft = 0x4b560003,      // a drafted token outside the vocabulary, or rows that do not fit
};

// The batch's packed rows: sequence b has the new rows start[b] .. start[b + 1] - 1 and len[b] tokens
// of its own in the cache, those included.
struct KvBatch {
    const int *start, *len, *pages;   // pages: [batch][max_pages]
    int batch, rows, max_pages, prefix_len;
};

__device__ __forceinline__ bool kv_rows_fit(const KvBatch &batch, int first, int next) {
    return 0 <= first && first <= next && next <= batch.rows;
}

// The sequences [first, last) that can own one of the rows row0 .. row0 + n - 1: all of a small batch; of a large one what
// lies between two of 256 evenly spaced starts, so that a block looks at a few hundred sequences and not at all of them.
// range: two ints of shared memory.  Ends with the block synchronised.
__device__ __forceinline__ int2 kv_range(int *range, const int *__restrict__ start, int batch, int row0, int n, int tid, int threads) {
    constexpr int kAll = 1024, kMarks = 256;
    if (batch <= kAll) return make_int2(0, batch);
    const int step = (batch + kMarks - 1) / kMarks;
    if (tid == 0) {
        range[0] = 0;
        range[1] = batch;
    }
    __syncthreads();
    for (int i = tid; i < kMarks; i += threads) {
        const int b = i * step;
        if (b >= batch) continue;
        const int s = start[b];
        if (s <= row0) atomicMax(range, b);
        if (s >= row0 + n) atomicMin(range + 1, b);
    }
    __syncthreads();
    return make_int2(range[0], range[1]);
}

// The sequences of the block's rows row0 .. row0 + n - 1 into owner[] (shared memory; -1 behind the last sequence, and for one
// whose rows do not fit the call's).  Every thread looks at some of the sequences, so there is no chain of dependent loads
// as in a search.  Ends with the block synchronised.
__device__ __forceinline__ void kv_owners(int *owner, int *range, const KvBatch &batch, int row0, int n, int tid, int threads) {
    for (int i = tid; i < n; i += threads) owner[i] = -1;
    const int2 some = kv_range(range, batch.start, batch.batch, row0, n, tid, threads);
    __syncthreads();
    for (int b = some.x + tid; b < some.y; b += threads) {
        const int first = batch.start[b], next = batch.start[b + 1];
        const int lo = max(first, row0), hi = kv_rows_fit(batch, first, next) ? min(next, row0 + n) : lo;
        for (int t = lo; t < hi; ++t) owner[t - row0] = b;
    }
    __syncthreads();
}

}  // namespace zb
