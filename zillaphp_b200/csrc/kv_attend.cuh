// kv_attend.cuh -- attention of a batch's new tokens over a prefix that all
// sequences share and over each sequence's own cached keys: the parameters
// and the parts that its kernels share.
//
// For row j of sequence b (n new rows, len own cached tokens) and one query head:
//   o = sum_i softmax_i(scale q.k_i) v_i over the prefix's keys and the own keys i < len - n + j + 1.
// The keys are cut into slots (prefix_splits of the prefix, own_splits of the own keys); a slot's kernel
// leaves the row's maximum m (in units of log2), its sum l = sum 2^(s - m) and o = sum 2^(s - m) v in
// fp32, and the join takes sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c in slot order.
#pragma once

#include "kv_cache.cuh"

namespace zb {
namespace kv {

struct AttendParams {
    CUtensorMap k_map, v_map;
    const void *q;
    void *out;
    float *part_o;      // [slots][rows * q_heads][head_dim]
    float2 *part_ml;    // [slots][rows * q_heads]
    int *item_slots;    // the tcgen05 kernel's items: how many slots each took
    KvBatch batch;
    const int *prefix_pages;
    int q_heads, kv_heads, group, page_log2, pages, box_rows;
    FastDiv by_group;   // rows are token-major, then the group's heads
    int max_new, max_len;
    int prefix_splits, prefix_chunk, own_splits, own_chunk;   // slots, and keys of a slot
    int prefix_tiles, own_tiles;                              // row tiles of this launch
    int prefix_items;                                         // blocks [0, prefix_items) take the prefix
    int tc_blocks;      // > 0: the prefix is cut evenly over this many blocks of the tcgen05 kernel
    int behind_tc;      // the split kernel runs beside the tcgen05 kernel in front of it
    int direct;         // one slot in all: its kernel writes out itself
    int front_steps;    // and this many steps over the prefix come in front of it
    float scale_log2;
    int *err;
};

// The tcgen05 kernel's cut of the prefix.  Its work is items (kv head, pair of row tiles) x key tiles of 128, item after
// item; block c of n takes units [c U / n, (c + 1) U / n), so that no block has more than a tile over another, whatever the
// counts.  An item's slots are the blocks that touch it, in order.
struct PrefixCut {
    int units, tiles, blocks;   // units * blocks may pass 31 bits
    __host__ __device__ int begin(int c) const { return (int)((long long)c * units / blocks); }
    __host__ __device__ int first_block(int item) const { return (int)((((long long)item * tiles + 1) * blocks - 1) / units); }
};
__host__ __device__ __forceinline__ PrefixCut prefix_cut(int prefix_len, int items, int blocks) {
    PrefixCut c;
    c.tiles = (prefix_len + 127) / 128;
    c.units = items * c.tiles;
    c.blocks = blocks;
    return c;
}

// The slots of an item as the tcgen05 kernel noted them.  Where one of its waits has run out the note is missing and the word
// is whatever the workspace held; the join never reads more than the prefix's slots.
__host__ __device__ __forceinline__ int noted_slots(int note, int prefix_splits) { return (unsigned)note <= (unsigned)prefix_splits ? note : prefix_splits; }

// Slots of `chunk` keys that `keys` keys take, and the end of the slot that starts at `begin`, `len` at most.  keys + chunk
// and begin + chunk may pass 31 bits.
__host__ __device__ __forceinline__ int slots_of(int keys, int chunk) { return keys > 0 ? (keys - 1) / chunk + 1 : 0; }
__host__ __device__ __forceinline__ int slot_end(int begin, int chunk, int len) {
    return begin < len && chunk < len - begin ? begin + chunk : len;
}

// Keys that row j of a sequence sees of its own: clamped to 0 .. len.
__device__ __forceinline__ int own_limit(int len, int n, int j) { return max(0, len - n + j + 1); }

__device__ __forceinline__ bool sequence_fits(const AttendParams &p, int first, int n, int len) {
    return first >= 0 && n >= 0 && n <= p.max_new && (long long)first + n <= p.batch.rows && len >= 0 && len <= p.max_len;
}

// A sequence's new rows and length; one that does not fit the call's sizes is recorded and has no rows.
__device__ __forceinline__ void load_sequence(const AttendParams &p, int b, int &first, int &n, int &len) {
    first = __ldcg(p.batch.start + b);
    n = __ldcg(p.batch.start + b + 1) - first;
    len = __ldcg(p.batch.len + b);
    if (!sequence_fits(p, first, n, len)) {
        atomicCAS(p.err, 0, kErrKvLength);
        n = 0;
        len = 0;
    }
}

// The TMA row coordinate of the box at `key` in page `id`: the cache's end (a box of zeros) for a page number outside the
// cache, which is recorded.
__device__ __forceinline__ int box_row_of(const AttendParams &p, int id, int kv_head, int key) {
    if (id < 0 || id >= p.pages) {
        atomicCAS(p.err, 0, kErrKvPage);
        return p.pages * p.kv_heads << p.page_log2;
    }
    return ((id * p.kv_heads + kv_head) << p.page_log2) + (key & ((1 << p.page_log2) - 1));
}
// The same with the page number looked up; behind `end` the cache's end too.
__device__ __forceinline__ int box_row(const AttendParams &p, const int *pages, int kv_head, int key, int end) {
    if (key >= end) return p.pages * p.kv_heads << p.page_log2;
    return box_row_of(p, __ldcg(pages + (key >> p.page_log2)), kv_head, key);
}

// tc::mbar_wait with the clock read only after 64 failed tries: short waits do without it.
__device__ __forceinline__ bool wait_phase(uint64_t *bar, uint32_t parity, volatile int *abort, int *err, int code) {
    uint64_t t0 = 0;
    for (uint32_t i = 1;; ++i) {
        if (tc::mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 0u) {
            if (*abort) return false;
            const uint64_t t = tc::global_ns();
            if (t0 == 0) t0 = t;
            else if (t - t0 > tc::kWaitLimitNs) break;
        }
    }
    *abort = 1;
    if (err) atomicCAS(err, 0, code);
    return false;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// D += A B, one warp's 16 x 8 tile with K = 16, fp32 accumulation.
template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte offset of the 16-byte chunk of a key row in a tile that TMA wrote: 128-byte rows whose chunks are
// XORed with the row's low three bits (64-byte rows, head_dim 32: with bits 1 and 2), one such block of
// 64 rows for each 64 elements of the head.
template <int D>
__device__ __forceinline__ uint32_t tile_chunk(int row, int chunk, int rows) {
    if constexpr (D == 32) return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    else return (chunk >> 3) * rows * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

}  // namespace kv
}  // namespace zb
