// kv_attend.cu -- attention over a shared prefix and each sequence's own cached keys (zilla_kv_attend).
#include <math.h>

#include <algorithm>

#include "kv_attend.cuh"
#include "kv_attend_tc.cuh"

namespace zb {
namespace kv {
namespace {

using namespace tc;

constexpr int kTile = 64;                                 // keys of a stage
constexpr int kSplitThreads = 128;   // four warps: a fifth that only loads would cost a quarter of an SM partition's registers
// What one block of the two kernels below takes: a tile of rows (token-major, then the group's query heads, which share
// the keys) and one slot of keys, of the prefix or of one sequence.
struct SplitItem {
    bool shared;
    int head, row0, rows;    // kv head; first row of the tile, rows of the whole sequence (prefix: batch)
    int first, n, len;
    int begin, end, slot;
    int front;               // steps over the prefix in front of the own keys (one block takes all keys of its rows)
    const int *pages;
    bool empty;              // no rows, or no keys (and not to write zeros either)
};

__device__ __forceinline__ SplitItem split_item(const AttendParams &p, int item, int tile_rows) {
    SplitItem x;
    x.shared = item < p.prefix_items;
    if (!x.shared) item -= p.prefix_items;
    x.head = item % p.kv_heads;
    item /= p.kv_heads;
    const int tiles = x.shared ? p.prefix_tiles : p.own_tiles;
    x.row0 = item % tiles * tile_rows;
    item /= tiles;
    x.first = 0;
    x.n = p.batch.rows;
    x.len = p.batch.prefix_len;
    x.slot = item;
    x.pages = p.prefix_pages;
    int chunk = p.prefix_chunk;
    if (!x.shared) {
        x.slot = item % p.own_splits;
        const int b = item / p.own_splits;
        load_sequence(p, b, x.first, x.n, x.len);
        x.pages = p.batch.pages + (size_t)b * p.batch.max_pages;
        chunk = p.own_chunk;
    }
    x.rows = x.n * p.group;
    x.begin = x.slot * chunk;
    const int last_j = p.by_group.div(max(0, min(x.rows - 1, x.row0 + tile_rows - 1)));
    x.end = slot_end(x.begin, chunk, x.shared ? x.len : own_limit(x.len, x.n, last_j));
    x.front = x.shared ? 0 : p.front_steps;
    x.empty = x.row0 >= x.rows || (x.begin >= x.end && !(p.direct && x.slot == 0));
    if (!x.shared) x.slot += p.prefix_splits;
    return x;
}

// K and V of 64-key steps by TMA, one box a lane, into a ring of ST stages.  The four warps take turns in loading the stage
// of the step before, whose page numbers they have looked up a step ahead: a fifth warp that only loads would cost a quarter
// of an SM partition's registers, and one of the four that loads always would hold the others up.
template <int D, int ST>
struct SplitRing {
    static constexpr int kTileBytes = kTile * D * 2, kHalves = D == 128 ? 2 : 1, kRowBytes = D < 64 ? D * 2 : 128;
    static constexpr int kBytes = ST * 2 * kTileBytes;
    uint8_t *base;         // stage st: K at 2 st tiles, V at 2 st + 1
    uint64_t *full, *empty;
    volatile int *abort_flag;
    int all, r0, half, is_v, steps, warp, lane, next_page;
    __device__ __forceinline__ SplitRing(uint8_t *smem, int boxes) : base(smem), warp(threadIdx.x >> 5), lane(threadIdx.x & 31), next_page(0) {
        full = reinterpret_cast<uint64_t *>(smem + kBytes);
        empty = full + ST;
        abort_flag = reinterpret_cast<volatile int *>(empty + ST);
        all = boxes * kHalves * 2;   // 2 .. 16
        r0 = lane % boxes * (kTile / boxes);
        half = lane / boxes % kHalves;
        is_v = lane / (boxes * kHalves);
        if (threadIdx.x == 0) {
            for (int i = 0; i < ST; ++i) {
                mbar_init(full + i, 1);
                mbar_init(empty + i, 4);
            }
            *abort_flag = 0;
            fence_barrier_init();
        }
    }
    __device__ __forceinline__ void load(const AttendParams &p, int step, int at) const {
        const int st = step % ST;
        if (lane == 0) mbar_arrive_expect_tx(full + st, 2 * kTileBytes);
        __syncwarp();
        if (lane < all)
            tma_load_2d(base + (2 * st + is_v) * kTileBytes + half * kTile * 128 + r0 * kRowBytes, is_v ? &p.v_map : &p.k_map, full + st,
                        half * 64, at);
    }
    // a step's first key, in the prefix or among the item's own, and the end of its keys
    static __device__ __forceinline__ int first_key(const SplitItem &x, int step) {
        return step < x.front ? step * kTile : x.begin + (step - x.front) * kTile;
    }
    static __device__ __forceinline__ int end_of(const AttendParams &p, const SplitItem &x, int step) {
        return step < x.front ? p.batch.prefix_len : x.end;
    }
    // the first ST steps, by the first warp
    __device__ __forceinline__ void start(const AttendParams &p, const SplitItem &x) {
        steps = x.front + (x.begin < x.end ? (x.end - x.begin + kTile - 1) / kTile : 0);
        if (warp != 0) return;
        int at[ST];
#pragma unroll
        for (int i = 0; i < ST; ++i) {
            const int key = first_key(x, i) + r0;
            at[i] = i < steps && lane < all ? box_row(p, i < x.front ? p.prefix_pages : x.pages, x.head, key, end_of(p, x, i)) : 0;
        }
#pragma unroll
        for (int i = 0; i < ST; ++i)
            if (i < steps) load(p, i, at[i]);
    }
    // At the start of step `it`, by all warps: the warp whose turn it is loads step it - 1 + ST over step it - 1; the next
    // one looks its page numbers up.  False: given up.
    __device__ __forceinline__ bool refill(const AttendParams &p, const SplitItem &x, int it) {
        const int step = it - 1 + ST;
        if (it > 0 && step < steps && (it & 3) == warp) {
            const int key = first_key(x, step) + r0;
            const int at = key < end_of(p, x, step) ? box_row_of(p, next_page, x.head, key) : p.pages * p.kv_heads << p.page_log2;
            if (!__all_sync(0xffffffffu, wait_phase(empty + step % ST, (step / ST - 1) & 1, abort_flag, p.err, kErrEmptyWait))) return false;
            load(p, step, lane < all ? at : 0);
        }
        if (((it + 1) & 3) == warp && lane < all && step + 1 < steps) {
            const int key = first_key(x, step + 1) + r0;
            if (key < end_of(p, x, step + 1)) next_page = __ldcg((step + 1 < x.front ? p.prefix_pages : x.pages) + (key >> p.page_log2));
        }
        return true;
    }
    __device__ __forceinline__ bool wait(const AttendParams &p, int it) const {
        return __all_sync(0xffffffffu, wait_phase(full + it % ST, (it / ST) & 1, abort_flag, p.err, kErrFullWait)) != 0;
    }
    // This warp has read the step's stage.  The fence orders its shared-memory reads before the copy (another proxy) that
    // the arrival allows: without it a copy overtook reads still on their way, a handful of 16-wide columns in a run.
    __device__ __forceinline__ void done(int it) const {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + it % ST);
    }
    // A warp that gives up at step `it`: the copies in flight (steps up to it - 1 + ST) end before the block's shared memory goes.
    __device__ __forceinline__ void drain(const AttendParams &p, int it) const {
        if (lane == 0)
            for (int i = max(0, it - 1); i < min(steps, it + ST); ++i)
                if (!mbar_wait_drain(full + i % ST, (i / ST) & 1)) atomicCAS(p.err, 0, kErrDrain);
        __syncwarp();
    }
};

// The wait at the start.  Behind the tcgen05 kernel nothing here depends on that kernel's results, and it has been started
// only after all blocks of it found the work before them done (they wait, then allow this one): the two run side by side.
// What the host's earlier kernels wrote is read past L1 (__ldcg, TMA).  The last block only waits for the tcgen05 kernel,
// so that this grid does not end before it: the join behind waits for this grid alone.  False: the block is done.
__device__ __forceinline__ bool split_start(const AttendParams &p) {
    griddep_launch();
    if (!p.behind_tc) {
        griddep_wait();
    } else if (blockIdx.x == gridDim.x - 1) {
        griddep_wait();
        return false;
    }
    return true;
}

__device__ __forceinline__ void movmatrix_trans(uint32_t &d, uint32_t a) {
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
}

// Few rows (up to 8 R8 = 8 .. 24 that share the keys): the products are taken with the keys as the long side, so that
// rows are padded to 8 and not to 16, and all four warps lie along the keys (16 of each 64):
//   S^T = K Q^T        16 keys x 8 rows an MMA, K from shared memory, Q^T in registers
//   O^T += V^T P^T     16 of head_dim x 8 rows, V read transposed, P^T by a transposition of S^T's registers
// A row's reference maximum follows the scores only when they pass it by 2^8, so most steps need no maximum across lanes
// at all.  P is rounded to the cache's type (half a step of 2^-8 or 2^-11 on weights that average out), everything else is
// fp32; the warps are joined at the end through shared memory.
// Bound by HBM: K and V come once, by TMA through the page list, several stages ahead.
constexpr int few_blocks(int D, int R8) { return D == 128 && R8 == 3 ? 2 : D == 32 ? 4 : 3; }
constexpr int few_stages(int D, int R8) { return D == 128 ? (R8 == 3 ? 3 : 2) : D == 64 ? 4 : 6; }
constexpr int few_smem(int D, int R8) { return few_stages(D, R8) * 2 * kTile * D * 2 + 1024 + 256; }

template <typename T, int D, int R8>
__global__ void __launch_bounds__(kSplitThreads, few_blocks(D, R8)) attend_few_kernel(const __grid_constant__ AttendParams p) {
    constexpr int ST = few_stages(D, R8), kTileBytes = kTile * D * 2, kRows = 8 * R8, kPitch = D + 4;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    SplitRing<D, ST> ring(base, kTile / p.box_rows);
    if (!split_start(p)) return;
    const SplitItem x = split_item(p, blockIdx.x, kRows);
    if (x.empty) return;
    __syncthreads();
    ring.start(p, x);
    const int steps = ring.steps;
    // this warp's 16 keys of a step: the thread holds keys g, g + 8 and rows 8 i + c2, 8 i + c2 + 1 of S^T, and row 8 i + g of Q
    const int g = lane >> 2, c2 = 2 * (lane & 3);
    uint32_t qf[D / 16][R8][2];
#pragma unroll
    for (int i = 0; i < R8; ++i) {
        const int row = x.row0 + 8 * i + g;
        const bool real = row < x.rows;
        const int j = real ? p.by_group.div(row) : 0, hq = x.head * p.group + (real ? row - j * p.group : 0);
        const uint32_t *src = reinterpret_cast<const uint32_t *>(static_cast<const T *>(p.q) + ((size_t)(x.first + j) * p.q_heads + hq) * D + c2);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            qf[k][i][0] = real ? __ldcg(src + 8 * k) : 0u;
            qf[k][i][1] = real ? __ldcg(src + 8 * k + 4) : 0u;
        }
    }
    auto limit = [&](int i, int e) {   // keys that a row of S^T's columns sees end here
        const int row = x.row0 + 8 * i + c2 + e;
        return x.shared || row >= x.rows ? x.end : min(x.end, own_limit(x.len, x.n, p.by_group.div(row)));
    };
    const int low = x.shared ? x.end : min(x.end, own_limit(x.len, x.n, p.by_group.div(x.row0)));   // the first row sees the fewest keys
    float o[D / 16][R8][4] = {}, m[R8][2], l[R8][2];   // m: the rows' references in units of log2, 0 before the first key
#pragma unroll
    for (int i = 0; i < R8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            m[i][e] = -INFINITY;
            l[i][e] = 0.0f;
        }
    const float sl = p.scale_log2;
    int it = 0;
    bool ok = true, open = true;   // open: some row that sees keys has no finite reference yet
    for (; it < steps; ++it) {
        const int st = it % ST, key0 = ring.first_key(x, it) + warp * 16, end = ring.end_of(p, x, it);
        const bool all_see = it < x.front;   // every row sees the prefix
        ok = ring.refill(p, x, it) && ring.wait(p, it);
        if (!ok) break;
        const uint32_t sk = smem_u32(base) + 2 * st * kTileBytes, sv = sk + kTileBytes;
        float s[R8][4];
#pragma unroll
        for (int i = 0; i < R8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            uint32_t a[4];
            ldmatrix_x4(a, sk + tile_chunk<D>(warp * 16 + (lane & 15), 2 * k + (lane >> 4), kTile));
#pragma unroll
            for (int i = 0; i < R8; ++i) mma_16816<T>(s[i], a, qf[k][i][0], qf[k][i][1]);
        }
#pragma unroll
        for (int i = 0; i < R8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] *= sl;
        if (key0 + 16 > (all_see ? end : low)) {   // keys behind some row's last
#pragma unroll
            for (int i = 0; i < R8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int last = all_see ? end : limit(i, e);
                    if (key0 + g >= last) s[i][e] = -INFINITY;
                    if (key0 + g + 8 >= last) s[i][e + 2] = -INFINITY;
                }
        }
        bool over = open;
#pragma unroll
        for (int i = 0; i < R8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) over |= s[i][e] > m[i][e & 1] + 8.0f;
        if (__any_sync(0xffffffffu, over)) {
            bool still = false;
#pragma unroll
            for (int i = 0; i < R8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(s[i][e], s[i][e + 2]);
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                    const float now = fmaxf(m[i][e], top), f = now == -INFINITY ? 1.0f : ex2(m[i][e] - now);
                    m[i][e] = now;
                    l[i][e] *= f;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        o[d][i][e] *= f;
                        o[d][i][e + 2] *= f;
                    }
                    if (now == -INFINITY) still |= key0 < (all_see ? end : limit(i, e));
                }
            open = __any_sync(0xffffffffu, still);
        }
        uint32_t pt[R8][2];
#pragma unroll
        for (int i = 0; i < R8; ++i) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = ex2(s[i][e] - (m[i][e & 1] == -INFINITY ? 0.0f : m[i][e & 1]));
                l[i][e & 1] += w[e];
            }
            movmatrix_trans(pt[i][0], pack2<T>(w[0], w[1]));   // keys 0-7 x rows, then keys 8-15
            movmatrix_trans(pt[i][1], pack2<T>(w[2], w[3]));
        }
        if (key0 + 16 > end) {   // the keys behind the last: whatever their page holds, V counts as zero
            const int from = max(0, end - key0);
            for (int i = lane; i < (16 - from) * (D / 8); i += 32)
                *reinterpret_cast<uint4 *>(base + (2 * st + 1) * kTileBytes + tile_chunk<D>(warp * 16 + from + i / (D / 8), i % (D / 8), kTile)) =
                    make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();   // before a later copy into this stage
            __syncwarp();
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            uint32_t a[4];
            ldmatrix_x4_trans(a, sv + tile_chunk<D>(warp * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * d + ((lane >> 3) & 1), kTile));
#pragma unroll
            for (int i = 0; i < R8; ++i) mma_16816<T>(o[d][i], a, pt[i][0], pt[i][1]);
        }
        ring.done(it);
    }
    if (!ok) ring.drain(p, it);
    // join the warps over the stages, which all of them have read
    float *red = reinterpret_cast<float *>(base);                              // [4][kRows][kPitch]
    float2 *ml = reinterpret_cast<float2 *>(red + 4 * kRows * kPitch);         // [4][kRows]
    static_assert(4 * kRows * (kPitch + 2) * 4 <= ST * 2 * kTileBytes, "the join fits the stages");
    named_bar_sync(1, 128);
#pragma unroll
    for (int i = 0; i < R8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = warp * kRows + 8 * i + c2 + e;
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], w);
            if (g == 0) ml[r] = make_float2(m[i][e], l[i][e]);
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                red[r * kPitch + 16 * d + g] = o[d][i][e];
                red[r * kPitch + 16 * d + g + 8] = o[d][i][e + 2];
            }
        }
    named_bar_sync(1, 128);
    if (*ring.abort_flag) return;
    for (int i = threadIdx.x; i < min(kRows, x.rows - x.row0) * (D / 4); i += 128) {
        const int r = i / (D / 4), c = i % (D / 4), row = x.row0 + r, j = p.by_group.div(row), hq = x.head * p.group + row - j * p.group;
        float2 y[4];
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            y[w] = ml[w * kRows + r];
            top = fmaxf(top, y[w].x);
        }
        const float use = top == -INFINITY ? 0.0f : top;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = ex2(y[w].x - use);
            const float4 z = *reinterpret_cast<const float4 *>(red + (w * kRows + r) * kPitch + 4 * c);
            sum += f * y[w].y;
            acc.x += f * z.x;
            acc.y += f * z.y;
            acc.z += f * z.z;
            acc.w += f * z.w;
        }
        const size_t at = (size_t)(x.first + j) * p.q_heads + hq;
        if (p.direct) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + at * D + 4 * c) =
                make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        } else {
            const size_t to = (size_t)x.slot * p.batch.rows * p.q_heads + at;
            *reinterpret_cast<float4 *>(p.part_o + to * D + 4 * c) = acc;
            if (c == 0) p.part_ml[to] = make_float2(top, sum);
        }
    }
}

// Many rows (64 a tile): four warps along the rows, each with all keys of a step.  S = Q K^T and O += P V by warp-level
// MMA, one pass with the running maximum and sum in registers, the same roundings and lazy rescale as above.
// Compute bound: K and V are read from shared memory by each of the four warps.
constexpr int kManyRows = 64, kManyBlocks = 3;
constexpr int many_stages(int D) { return D == 128 ? 2 : D == 64 ? 4 : 6; }
constexpr int many_smem(int D) { return many_stages(D) * 2 * kTile * D * 2 + 1024 + 256; }

template <typename T, int D>
__global__ void __launch_bounds__(kSplitThreads, kManyBlocks) attend_many_kernel(const __grid_constant__ AttendParams p) {
    constexpr int NT = kTile / 8, ST = many_stages(D), kTileBytes = kTile * D * 2;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    SplitRing<D, ST> ring(base, kTile / p.box_rows);
    if (!split_start(p)) return;
    const SplitItem x = split_item(p, blockIdx.x, kManyRows);
    if (x.empty) return;
    __syncthreads();
    ring.start(p, x);
    const int steps = ring.steps;
    // this warp's 16 rows; the thread holds rows g and g + 8 of them, columns c2, c2 + 1 of each 8
    const int g = lane >> 2, c2 = 2 * (lane & 3);
    const int row[2] = {x.row0 + warp * 16 + g, x.row0 + warp * 16 + g + 8};
    int limit[2];
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool real = row[i] < x.rows;
        const int j = real ? p.by_group.div(row[i]) : 0, hq = x.head * p.group + (real ? row[i] - j * p.group : 0);
        limit[i] = x.shared || !real ? x.end : min(x.end, own_limit(x.len, x.n, j));
        const uint32_t *src = reinterpret_cast<const uint32_t *>(static_cast<const T *>(p.q) + ((size_t)(x.first + j) * p.q_heads + hq) * D + c2);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            qf[k][i] = real ? __ldcg(src + 8 * k) : 0u;
            qf[k][i + 2] = real ? __ldcg(src + 8 * k + 4) : 0u;
        }
    }
    float o[D / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const int low = x.shared ? x.end : min(x.end, own_limit(x.len, x.n, p.by_group.div(min(x.rows - 1, x.row0 + warp * 16))));
    int it = 0;
    bool ok = true;
    for (; it < steps; ++it) {
        const int st = it % ST, key0 = ring.first_key(x, it), end = ring.end_of(p, x, it);
        const bool all_see = it < x.front;   // every row sees the prefix
        ok = ring.refill(p, x, it) && ring.wait(p, it);
        if (!ok) break;
        const uint32_t sk = smem_u32(base) + 2 * st * kTileBytes, sv = sk + kTileBytes;
        float s[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int i = 0; i < NT / 2; ++i) {
                uint32_t b[4];
                ldmatrix_x4(b, sk + tile_chunk<D>(16 * i + ((lane >> 4) << 3) + (lane & 7), 2 * k + ((lane >> 3) & 1), kTile));
                mma_16816<T>(s[2 * i], qf[k], b[0], b[1]);
                mma_16816<T>(s[2 * i + 1], qf[k], b[2], b[3]);
            }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] *= p.scale_log2;
        if (key0 + kTile > (all_see ? end : low)) {   // keys behind some row's last
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (key0 + 8 * i + c2 + (e & 1) >= (all_see ? end : limit[e >> 1])) s[i][e] = -INFINITY;
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[i][e]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] + 8.0f || top[1] > m[1] + 8.0f)) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float now = fmaxf(m[i], top[i]), f = now == -INFINITY ? 1.0f : ex2(m[i] - now);
                m[i] = now;
                l[i] *= f;
#pragma unroll
                for (int d = 0; d < D / 8; ++d) {
                    o[d][2 * i] *= f;
                    o[d][2 * i + 1] *= f;
                }
            }
        }
        const float use[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};   // a row without keys so far
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[i][e] = ex2(s[i][e] - use[e >> 1]);
                l[e >> 1] += s[i][e];
            }
        if (key0 + kTile > end) {   // the keys behind the last: whatever their page holds, V counts as zero
            const int from = end - key0;   // each warp writes the same zeros before it reads them
            for (int i = lane; i < (kTile - from) * (D / 8); i += 32)
                *reinterpret_cast<uint4 *>(base + (2 * st + 1) * kTileBytes + tile_chunk<D>(from + i / (D / 8), i % (D / 8), kTile)) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();   // before a later copy into this stage
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) {
            const uint32_t a[4] = {pack2<T>(s[2 * i][0], s[2 * i][1]), pack2<T>(s[2 * i][2], s[2 * i][3]),
                                   pack2<T>(s[2 * i + 1][0], s[2 * i + 1][1]), pack2<T>(s[2 * i + 1][2], s[2 * i + 1][3])};
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                uint32_t b[4];
                ldmatrix_x4_trans(b, sv + tile_chunk<D>(16 * i + (lane & 15), 2 * d + (lane >> 4), kTile));
                mma_16816<T>(o[2 * d], a, b[0], b[1]);
                mma_16816<T>(o[2 * d + 1], a, b[2], b[3]);
            }
        }
        ring.done(it);
    }
    if (!ok) ring.drain(p, it);
    if (!ok) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (row[i] >= x.rows) continue;
        const int j = p.by_group.div(row[i]), hq = x.head * p.group + row[i] - j * p.group;
        const size_t at = (size_t)(x.first + j) * p.q_heads + hq;
        if (p.direct) {
            const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
            uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<T *>(p.out) + at * D + c2);
#pragma unroll
            for (int d = 0; d < D / 8; ++d) dst[4 * d] = pack2<T>(o[d][2 * i] * inv, o[d][2 * i + 1] * inv);
        } else {
            const size_t to = (size_t)x.slot * p.batch.rows * p.q_heads + at;
            float *dst = p.part_o + to * D + c2;
#pragma unroll
            for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2 *>(dst + 8 * d) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
            if ((lane & 3) == 0) p.part_ml[to] = make_float2(m[i], l[i]);
        }
    }
}

// The join: one warp a (row, query head), each lane D / 32 columns.  Reads the slots' parts once, mostly from L2, BATCH
// slots at a time (their addresses do not depend on their maxima, so the loads of a batch are on the way together): eight
// where few blocks wait for the latency of many slots, four (and twice the blocks an SM) where the rows are many.  A row
// of no sequence is left as it is, a row without keys becomes zero.
template <typename T, int D, int BATCH>
__global__ void __launch_bounds__(256, BATCH == 4 ? 5 : 2) attend_join_kernel(const __grid_constant__ AttendParams p) {
    constexpr int C = D / 32, kBatch = BATCH;
    __shared__ int owner[8], own_slots[8], range[2];   // of the block's tokens, eight at most
    griddep_launch();
    const int tid = threadIdx.x, lane = tid & 31;
    const long long unit0 = (long long)blockIdx.x * 8, units = (long long)p.batch.rows * p.q_heads, unit = unit0 + (tid >> 5);
    const int t0 = (int)(unit0 / p.q_heads), n = (int)(min(unit0 + 8, units) - 1) / p.q_heads - t0 + 1;
    const int t = (int)(unit / p.q_heads), hq = (int)(unit - (long long)t * p.q_heads);
    if (tid < 8) owner[tid] = -1;
    griddep_wait();
    int front = p.prefix_splits;   // the prefix's slots come first
    if (p.tc_blocks && unit < units) {
        const int head = p.by_group.div(hq), row = t * p.group + hq - head * p.group;
        front = noted_slots(p.item_slots[row / (2 * kTcTile) * p.kv_heads + head], p.prefix_splits);
    }
    const int2 some = kv_range(range, p.batch.start, p.batch.batch, t0, n, tid, 256);
    __syncthreads();
    for (int b = some.x + tid; b < some.y; b += 256) {
        const int first = p.batch.start[b], next = p.batch.start[b + 1], len = p.batch.len[b];
        const int lo = max(first, t0), hi = min(next, t0 + n);
        if (lo < hi && sequence_fits(p, first, next - first, len))
            for (int x = lo; x < hi; ++x) {
                owner[x - t0] = b;
                own_slots[x - t0] = slots_of(min(len, own_limit(len, next - first, x - first)), p.own_chunk);
            }
    }
    __syncthreads();
    if (unit >= units || owner[t - t0] < 0) return;
    const int slots = front + own_slots[t - t0], skip = p.prefix_splits - front;   // the own ones lie behind the most that the prefix can have
    float m = -INFINITY, acc[C] = {}, l = 0.0f;
    for (int s0 = 0; s0 < slots; s0 += kBatch) {
        float2 ml[kBatch];
        float v[kBatch][C];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int s = s0 + i;
            ml[i] = make_float2(-INFINITY, 0.0f);
            if (s >= slots) continue;
            const long long at = (s < front ? s : s + skip) * units + unit;
            ml[i] = p.part_ml[at];
            load_vec<float, C>(p.part_o + at * D + lane * C, v[i]);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) top = fmaxf(top, ml[i].x);
        const float use = top == -INFINITY ? 0.0f : top, f = ex2(m - use);
        m = top;
        l *= f;
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] *= f;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (s0 + i >= slots) continue;
            const float w = ex2(ml[i].x - use);
            l += w * ml[i].y;
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] += w * v[i][c];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] *= inv;
    store_vec<T, C>(static_cast<T *>(p.out) + unit * D + lane * C, acc);
}

// ---------------------------------------------------------------- plan
struct Plan {
    int tc_blocks;             // > 0: the prefix on tcgen05, by this many blocks
    int own_form, prefix_form; // 8-row tiles of the few-rows kernel, 0: the many-rows kernel
    int own_tiles, prefix_tiles, own_chunk, own_splits, prefix_chunk, prefix_splits;
    int front_steps;           // > 0: no shared work, every block runs over the prefix in front of its own keys
    bool direct;
    size_t units, part_floats;   // rows * q_heads; floats of the parts
};

// The few-rows kernel takes up to 24 rows; with 40 (eight heads, five tokens, head_dim 64) its accumulators fill the
// register file and the many-rows kernel is faster (18.6 us against 24.9 for 64 sequences of 513 keys).
int row_form(long long rows) {
    return rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 ? 3 : 0;
}
int form_rows(int form) { return form ? 8 * form : kManyRows; }
int form_blocks(int head_dim, int form) { return form ? few_blocks(head_dim, form) : kManyBlocks; }

// The shared prefix goes to tcgen05 where more than kTcRows rows share its keys, although 17 leave a 256-row tile mostly empty:
// 8 sequences of four query heads a key head behind 2029 keys 18.5 us against 20.4 of the mma.sync kernels, behind 16000 keys
// 31 against 46.  And where it is enough work for that kernel's longer start, counted in 64 x 64 tiles x head_dim: one key
// head, 128 rows, head_dim 128 behind 1000 keys (4096) 12.6 us against 10.6, behind 2029 (8192) 13.5 against 13.8; eight key
// heads, 24 rows behind 1000 keys (16384) 11.7 against 12.2; head_dim 64, 72 rows behind 1000 keys (16384) 9.9 against 9.4.
constexpr int kTcRows = 16, kTcWork = 12288;

// Blocks of the tcgen05 kernel.  It takes whole SMs (one block each) and is bound by the tensor cores and the softmax, the own
// keys' kernel behind it by HBM, and runs on the SMs that are left; so with n blocks the call takes about
//   t = units / n * tile + start,  plus what the other SMs - n have not moved by then at the whole machine's rate,
// and the n that minimises it is taken, among the multiples of the row tiles where they are few.  A tile of 256 rows and 128
// keys takes 2.2 us with head_dim 128 in a loop of such calls, which runs into the power limit (1.7 at full clock: 88% of the
// measured matrix rate), 1.8 with 64; 12 us stands for the start, the queries and the parts (a fit, not measured apart); an SM draws about 45 GB/s, all
// together 5.6 TB/s.  Lengths are on the device: half of their bound is assumed.
// Where the rule lands, in graphs of calls: 128 sequences of up to 2048 keys behind 16384 take 96 blocks, 209 to 231 us with the
// clock under the power limit (80 blocks 238, 112 230, 148 237); 64 drafts of head_dim 64 behind 4001 take 133, 35.6 us (96
// blocks 35.0, 64 40.8); 64 sequences behind 1000 take 44, 28.8 to 32.6 us (32 blocks 29.2, 64 30.1, 148 33.7); 32 sequences of
// up to 700 behind 2029 take 85, 24.4 us, where 32 would take 20.3 and 64 23.4: every count from 64 to 85 has the same longest
// block, and of equals the largest is taken.
int choose_tc_blocks(const KvCache &c, int row_tiles, long long units, double own_bytes) {
    const int sms = sm_count();
    const double tile = c.head_dim == 128 ? 2.2e-6 : 1.8e-6, start = 12e-6, one = 45e9, all = 5.6e12;
    int best = 1;
    double least = 1e30;
    const int step = row_tiles <= sms / 8 ? row_tiles : 1;
    const int most = (int)std::min<long long>(units, sms) / step * step;
    for (int n = most; n >= 1 && n >= std::min(most, sms / 8); n -= step) {
        const double t = (double)((units + n - 1) / n) * tile + start, left = std::max(0.0, own_bytes - (sms - n) * one * t);
        if (t + left / all < least) {
            least = t + left / all;
            best = n;
        }
    }
    return best;
}

// Row tiles by the rows that share the keys, and slots of whole 64-key steps: as many blocks as fit the machine at least,
// of four steps if there are enough, and about `kWaves` rounds of them where there are many (longer ones leave SMs idle
// at the end, shorter ones add starts, parts to write and to join).
Plan make_plan(const KvCache &c, int batch, int rows, int q_heads, int prefix_len, int max_new, int max_len) {
    constexpr int kWaves = 3;
    Plan p;
    const int group = q_heads / c.kv_heads;
    max_new = std::min(max_new, std::max(rows, 1));   // a loose bound: no sequence has more rows than the call
    const long long own_rows = (long long)max_new * group, prefix_rows = (long long)rows * group;
    const long long own_steps = (max_len + kTile - 1) / kTile, prefix_steps = (prefix_len + kTile - 1) / kTile;
    p.own_form = row_form(own_rows);
    p.own_tiles = (int)((own_rows + form_rows(p.own_form) - 1) / form_rows(p.own_form));
    // Few keys in all, or a short prefix in front of enough blocks: reading the prefix for every sequence (from L2) is
    // cheaper than parts and a join behind them.
    const long long own_blocks = (long long)batch * p.own_tiles * c.kv_heads;
    p.front_steps = 0;
    if (prefix_steps + own_steps <= 4 ||
        (prefix_steps <= 4 && own_steps <= 16 && own_blocks >= (long long)form_blocks(c.head_dim, p.own_form) * sm_count())) {
        p.front_steps = (int)prefix_steps;
        p.tc_blocks = p.prefix_splits = p.prefix_tiles = 0;
        p.prefix_form = p.own_form;
        p.prefix_chunk = kTile;
        p.own_splits = 1;
        p.own_chunk = (int)std::max(1LL, own_steps) * kTile;
        p.direct = true;
        p.units = (size_t)rows * q_heads;
        p.part_floats = 0;
        return p;
    }
    const bool tc = prefix_rows > kTcRows &&
                    (prefix_rows + kManyRows - 1) / kManyRows * prefix_steps * c.kv_heads * c.head_dim > kTcWork;
    p.prefix_form = row_form(prefix_rows);
    // one launch where the own keys are few (8 MB), in the prefix's form
    if (!tc && 4.0 * batch * max_len * c.kv_heads * c.head_dim < (double)(8 << 20)) p.own_form = p.prefix_form;
    p.own_tiles = (int)((own_rows + form_rows(p.own_form) - 1) / form_rows(p.own_form));
    const int tile_rows = tc ? 2 * kTcTile : form_rows(p.prefix_form);
    p.prefix_tiles = (int)((prefix_rows + tile_rows - 1) / tile_rows);
    // (as doubles: loose bounds of many sequences pass 63 bits)
    const double total = c.kv_heads * ((double)own_steps * batch * p.own_tiles + (tc ? 0.0 : (double)prefix_steps * p.prefix_tiles));
    const double fit = (double)form_blocks(c.head_dim, p.own_form) * sm_count();
    const double per = std::max(std::min(4.0, std::max(1.0, floor(total / fit))), floor(total / (kWaves * fit)));
    p.own_chunk = (int)std::min(per, (double)std::max(1LL, own_steps)) * kTile;
    p.own_splits = std::max(1, slots_of(max_len, p.own_chunk));   // one without own keys too: its blocks look at every sequence's sizes
    p.prefix_chunk = (int)std::min(per, (double)std::max(1LL, prefix_steps)) * kTile;
    p.prefix_splits = slots_of(prefix_len, p.prefix_chunk);
    p.tc_blocks = 0;
    if (tc) {
        const long long tiles = (prefix_len + kTcTile - 1) / kTcTile, units = tiles * c.kv_heads * p.prefix_tiles;
        p.tc_blocks = choose_tc_blocks(c, p.prefix_tiles, units, 0.5 * 4.0 * batch * max_len * c.kv_heads * c.head_dim);
        const long long each = units / p.tc_blocks;   // a block's units at least
        p.prefix_splits = (int)std::min<long long>((tiles + each - 2) / each + 1, p.tc_blocks);
    }
    p.direct = p.own_splits == 1 && p.prefix_splits == 0;
    p.units = (size_t)rows * q_heads;
    p.part_floats = p.direct ? 0 : p.units * (p.own_splits + p.prefix_splits) * (c.head_dim + 2);
    if (p.tc_blocks) p.part_floats += (size_t)c.kv_heads * p.prefix_tiles;   // the items' slots
    return p;
}

// Shared memory above 48 KB is asked for once a device.
template <typename K>
int allow_smem(K kernel, int bytes, bool (&set)[64], const char *name) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && set[dev]) return kOk;
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (int rc = check_cuda(name)) return rc;
    if (dev >= 0 && dev < 64) set[dev] = true;
    return kOk;
}

template <typename K>
int launch_blocks(K kernel, const AttendParams &p, long long blocks, int smem, bool (&set)[64], const char *name) {
    if (blocks >= 0x7fffffffLL) return fail(kBadArg, "%s: %lld blocks are too many", name, blocks);
    if (int rc = allow_smem(kernel, smem, set, name)) return rc;
    launch_pdl(kernel, dim3((unsigned)(blocks + (p.behind_tc ? 1 : 0))), dim3(kSplitThreads), smem, p);
    ZB_LAUNCH_CHECK(name);
    return kOk;
}

template <typename T, int D, int R8>
int launch_few(const AttendParams &p, long long blocks, const char *name) {
    static bool set[64] = {};
    return launch_blocks(attend_few_kernel<T, D, R8>, p, blocks, few_smem(D, R8), set, name);
}

template <typename T, int D>
int run_split(const AttendParams &p, int form, long long blocks, const char *name) {
    if (blocks == 0) return kOk;
    if (form == 1) return launch_few<T, D, 1>(p, blocks, name);
    if (form == 2) return launch_few<T, D, 2>(p, blocks, name);
    if (form == 3) return launch_few<T, D, 3>(p, blocks, name);
    static bool set[64] = {};
    return launch_blocks(attend_many_kernel<T, D>, p, blocks, many_smem(D), set, name);
}

template <typename T, int D>
int run(AttendParams p, const Plan &plan, const char *name) {
    const long long own = (long long)p.batch.batch * p.own_splits * p.own_tiles * p.kv_heads;
    const long long prefix = (long long)p.prefix_splits * p.prefix_tiles * p.kv_heads;
    if (prefix > 0x7fffffffLL) return fail(kBadArg, "%s: %lld blocks are too many", name, prefix);
    if (plan.tc_blocks) {
        static bool set[64] = {};
        if (int rc = allow_smem(attend_tc_kernel<T, D>, tc_smem<D>(), set, name)) return rc;
        launch_pdl(attend_tc_kernel<T, D>, dim3(plan.tc_blocks), dim3(kTcThreads), tc_smem<D>(), p);
        ZB_LAUNCH_CHECK(name);
        p.behind_tc = 1;
        if (int rc = run_split<T, D>(p, plan.own_form, own, name)) return rc;
    } else if (plan.own_form == plan.prefix_form) {
        p.prefix_items = (int)prefix;
        if (int rc = run_split<T, D>(p, plan.own_form, prefix + own, name)) return rc;
    } else {
        p.prefix_items = (int)prefix;
        if (int rc = run_split<T, D>(p, plan.prefix_form, prefix, name)) return rc;
        p.prefix_items = 0;
        if (int rc = run_split<T, D>(p, plan.own_form, own, name)) return rc;
    }
    if (p.direct) return kOk;
    const dim3 grid((unsigned)((plan.units + 7) / 8));
    if (grid.x <= 2u * sm_count()) launch_pdl(attend_join_kernel<T, D, 8>, grid, dim3(256), 0, p);
    else launch_pdl(attend_join_kernel<T, D, 4>, grid, dim3(256), 0, p);
    ZB_LAUNCH_CHECK(name);
    return kOk;
}

// Refuses sizes; shared by the call and by the size of its workspace.
int check_sizes(const char *name, const KvCache *c, int kv, int batch, int rows, int q_heads, int prefix_len, int max_new,
                int max_len) {
    if (!c) return fail(kBadHandle, "%s: unknown cache %d", name, kv);
    if (batch < 0 || rows < 0 || prefix_len < 0 || max_new < 1 || max_len < 0)
        return fail(kBadArg, "%s: bad sizes batch=%d rows=%d prefix_len=%d max_new=%d max_len=%d", name, batch, rows, prefix_len,
                    max_new, max_len);
    if (q_heads < 1 || q_heads > 65536 || q_heads % c->kv_heads)
        return fail(kBadArg, "%s: %d query heads are not a multiple of the cache's %d", name, q_heads, c->kv_heads);
    if ((long long)prefix_len + max_len > 0x7fffffffLL - 4096 || (long long)rows * q_heads > 0x7fffffffLL)
        return fail(kBadArg, "%s: sizes pass 31 bits", name);
    return kOk;
}

}  // namespace
}  // namespace kv
}  // namespace zb

using namespace zb;
using namespace zb::kv;

extern "C" {

long zilla_kv_attend_work(int kv, int batch, int rows, int q_heads, int prefix_len, int max_new, int max_len) {
    const char *name = "zilla_kv_attend_work";
    const KvCache *c = kv_get(kv);
    if (int rc = check_sizes(name, c, kv, batch, rows, q_heads, prefix_len, max_new, max_len)) return rc;
    return (long)make_plan(*c, batch, rows, q_heads, prefix_len, max_new, max_len).part_floats;
}

int zilla_kv_attend(int kv, int q_id, int out_id, int start_id, int len_id, int pages_id, int prefix_pages_id, int batch,
                    int rows, int q_heads, int max_pages, int prefix_len, int max_new, int max_len, float scale, int work_id) {
    const char *name = "zilla_kv_attend";
    const KvCache *c = kv_get(kv);
    if (int rc = check_sizes(name, c, kv, batch, rows, q_heads, prefix_len, max_new, max_len)) return rc;
    if (max_pages < 1 || (long long)max_pages * c->page < max_len)
        return fail(kBadArg, "%s: max_len %d does not fit %d pages of %d", name, max_len, max_pages, c->page);
    if (!(fabsf(scale) < INFINITY)) return fail(kBadArg, "%s: scale is not finite", name);
    const Plan plan = make_plan(*c, batch, rows, q_heads, prefix_len, max_new, max_len);
    for (int from : {q_id, start_id, len_id, pages_id, prefix_len ? prefix_pages_id : 0, c->k_id, c->v_id})
        if (from && (from == out_id || (plan.part_floats && from == work_id)))
            return fail(kBadArg, "%s: buffer %d is read and written", name, from);
    if (plan.part_floats && work_id == out_id) return fail(kBadArg, "%s: out is the workspace", name);
    const size_t q_floats = elem_floats(plan.units * c->head_dim, c->type);
    if (int rc = check_buffers(name, {{q_id, q_floats, "q"},
                                      {out_id, q_floats, "out"},
                                      {c->k_id, c->floats, "the cache"},
                                      {c->v_id, c->floats, "the cache"},
                                      {start_id, (size_t)batch + 1, "start"},
                                      {len_id, (size_t)batch, "len"},
                                      {pages_id, (size_t)batch * max_pages, "pages"}}))
        return rc;
    if (prefix_len)
        if (int rc = check_buffers(name, {{prefix_pages_id, (size_t)(prefix_len + c->page - 1) / c->page, "prefix_pages"}}))
            return rc;
    if (plan.part_floats)
        if (int rc = check_buffers(name, {{work_id, plan.part_floats, "work"}})) return rc;
    if ((long long)plan.prefix_tiles * c->kv_heads * (prefix_len / kTcTile + 1) > 0x7fffffffLL)
        return fail(kBadArg, "%s: prefix of %d tokens for %d rows is too large", name, prefix_len, rows);
    if (!batch || !rows) return kOk;
    AttendParams p;
    p.k_map = c->k_map;
    p.v_map = c->v_map;
    p.q = ptr(q_id);
    p.out = ptr(out_id);
    p.part_o = plan.part_floats ? ptr(work_id) : nullptr;
    const size_t slots = (size_t)plan.own_splits + plan.prefix_splits;
    p.part_ml = plan.part_floats ? reinterpret_cast<float2 *>(ptr(work_id) + plan.units * slots * c->head_dim) : nullptr;
    p.item_slots = plan.part_floats ? reinterpret_cast<int *>(ptr(work_id) + plan.units * slots * (c->head_dim + 2)) : nullptr;
    p.batch = {reinterpret_cast<const int *>(ptr(start_id)), reinterpret_cast<const int *>(ptr(len_id)),
               reinterpret_cast<const int *>(ptr(pages_id)), batch, rows, max_pages, prefix_len};
    p.prefix_pages = prefix_len ? reinterpret_cast<const int *>(ptr(prefix_pages_id)) : nullptr;
    p.q_heads = q_heads;
    p.kv_heads = c->kv_heads;
    p.group = q_heads / c->kv_heads;
    p.by_group = FastDiv(p.group);
    p.page_log2 = c->page_log2;
    p.pages = c->pages;
    p.box_rows = c->box_rows;
    p.max_new = max_new;
    p.max_len = max_len;
    p.prefix_splits = plan.prefix_splits;
    p.prefix_chunk = plan.prefix_chunk;
    p.own_splits = plan.own_splits;
    p.own_chunk = plan.own_chunk;
    p.prefix_tiles = plan.prefix_tiles;
    p.own_tiles = plan.own_tiles;
    p.prefix_items = 0;
    p.tc_blocks = plan.tc_blocks;
    p.behind_tc = 0;
    p.direct = plan.direct;
    p.front_steps = plan.front_steps;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.err = device_error_word();
    if (!p.err) return fail(kBadHandle, "%s: no device error word", name);
    const int D = c->head_dim;
    if (c->type == kBf16)
        return D == 128 ? run<__nv_bfloat16, 128>(p, plan, name)
                        : D == 64 ? run<__nv_bfloat16, 64>(p, plan, name) : run<__nv_bfloat16, 32>(p, plan, name);
    return D == 128 ? run<__half, 128>(p, plan, name)
                    : D == 64 ? run<__half, 64>(p, plan, name) : run<__half, 32>(p, plan, name);
}

}  // extern "C"
