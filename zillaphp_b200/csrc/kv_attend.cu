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
constexpr int kSplitThreads = 160;                        // four warps that compute, one that loads
template <int D>
constexpr int split_stages() { return D == 128 ? 3 : D == 64 ? 4 : 6; }
template <int D>
constexpr int split_smem() { return split_stages<D>() * 2 * kTile * D * 2 + 1024 + 256; }

// One block takes a tile of 16 WM rows (rows of several tokens and of the group's query heads, which share
// the keys) and one slot of keys.  WM warps lie along the rows; the others take their part of each 64 keys
// and are joined at the end through shared memory.  One pass with the running maximum and sum in registers:
// S = Q K^T and O += P V by warp-level MMA, P rounded to the cache's type (half a step of 2^-8 or 2^-11 on
// weights that average out), everything else fp32.
// Bound by HBM where the rows are few: K and V come once, by TMA through the page list, three to six
// stages ahead.
template <typename T, int D, int WM>
__global__ void __launch_bounds__(kSplitThreads) attend_split_kernel(const __grid_constant__ AttendParams p) {
    constexpr int WN = 4 / WM, KW = kTile / WN, NT = KW / 8, ST = split_stages<D>();
    constexpr int kTileBytes = kTile * D * 2, kHalves = D == 128 ? 2 : 1, kRowBytes = D < 64 ? D * 2 : 128;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint64_t *full = reinterpret_cast<uint64_t *>(base + ST * 2 * kTileBytes), *empty = full + ST;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(empty + ST);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 4);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    // Behind the tcgen05 kernel nothing here depends on that kernel's results, and it has been started only after all blocks of
    // it found the work before them done (they wait, then allow this one): the two run side by side.  What the host's
    // earlier kernels wrote is read past L1 (__ldcg, TMA).  The last block only waits for
    // the tcgen05 kernel, so that this grid does not end before it: the join behind waits for this grid alone.
    griddep_launch();
    if (!p.behind_tc) {
        griddep_wait();
    } else if (blockIdx.x == gridDim.x - 1) {
        griddep_wait();
        return;
    }

    // the block's item: (slot, row tile, kv head) of the prefix or of one sequence
    int item = blockIdx.x;
    const bool shared = item < p.prefix_items;
    if (!shared) item -= p.prefix_items;
    const int head = item % p.kv_heads;
    item /= p.kv_heads;
    const int tiles = shared ? p.prefix_tiles : p.own_tiles;
    const int tile = item % tiles;
    item /= tiles;
    int first = 0, n = p.batch.rows, len = p.batch.prefix_len, slot = item, chunk = p.prefix_chunk;
    const int *pages = p.prefix_pages;
    if (!shared) {
        slot = item % p.own_splits;
        const int b = item / p.own_splits;
        load_sequence(p, b, first, n, len);
        pages = p.batch.pages + (size_t)b * p.batch.max_pages;
        chunk = p.own_chunk;
    }
    const int row0 = tile * 16 * WM, rows = n * p.group;   // rows of the item: token-major, then the group's heads
    if (row0 >= rows) return;
    const int last_j = min(rows - 1, row0 + 16 * WM - 1) / p.group;
    const int begin = slot * chunk, end = min(min(begin + chunk, len), shared ? len : own_limit(len, n, last_j));
    if (begin >= end && !(p.direct && slot == 0)) return;
    const int steps = begin < end ? (end - begin + kTile - 1) / kTile : 0;
    if (!shared) slot += p.prefix_splits;
    __syncthreads();

    if (warp == 4) {
        const int boxes = kTile / p.box_rows, all = boxes * kHalves * 2;
        const int r0 = lane % boxes * p.box_rows, half = lane / boxes % kHalves, is_v = lane / (boxes * kHalves);
        bool ok = true;
        int it = 0;
        for (; it < steps; ++it) {
            const int st = it % ST, at = lane < all ? box_row(p, pages, head, begin + it * kTile + r0, end) : 0;
            ok = it < ST || wait_phase(empty + st, (it / ST - 1) & 1, abort_flag, p.err, kErrEmptyWait);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(full + st, 2 * kTileBytes);
            __syncwarp();
            if (lane < all)
                tma_load_2d(base + (2 * st + is_v) * kTileBytes + half * kTile * 128 + r0 * kRowBytes, is_v ? &p.v_map : &p.k_map,
                            full + st, half * 64, at);
        }
        if (!ok && lane == 0)   // the copies in flight end before the block's shared memory goes
            for (int i = max(0, it - ST); i < it; ++i)
                if (!mbar_wait_drain(full + i % ST, (i / ST) & 1)) atomicCAS(p.err, 0, kErrDrain);
        return;
    }

    // this warp's 16 rows; the thread holds rows g and g + 8 of them, columns 2c, 2c + 1 of each 8
    const int wm = warp % WM, wn = warp / WM, g = lane >> 2, c2 = 2 * (lane & 3);
    const int row[2] = {row0 + wm * 16 + g, row0 + wm * 16 + g + 8};
    int limit[2];
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool real = row[i] < rows;
        const int j = real ? row[i] / p.group : 0, hq = head * p.group + row[i] - j * p.group;
        limit[i] = shared ? end : min(end, own_limit(len, n, j));
        const uint32_t *src = reinterpret_cast<const uint32_t *>(static_cast<const T *>(p.q) +
                                                                 ((size_t)(first + j) * p.q_heads + (real ? hq : 0)) * D + c2);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            qf[k][i] = real ? __ldcg(src + 8 * k) : 0u;
            qf[k][i + 2] = real ? __ldcg(src + 8 * k + 4) : 0u;
        }
    }
    float o[D / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const int low = min(limit[0], limit[1]);
    bool ok = true;
    for (int it = 0; it < steps; ++it) {
        const int st = it % ST, key0 = begin + it * kTile + wn * KW;
        ok = wait_phase(full + st, (it / ST) & 1, abort_flag, p.err, kErrFullWait);
        if (!__all_sync(0xffffffffu, ok)) break;
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
                ldmatrix_x4(b, sk + tile_chunk<D>(wn * KW + 16 * i + ((lane >> 4) << 3) + (lane & 7), 2 * k + ((lane >> 3) & 1), kTile));
                mma_16816<T>(s[2 * i], qf[k], b[0], b[1]);
                mma_16816<T>(s[2 * i + 1], qf[k], b[2], b[3]);
            }
        float top[2] = {m[0], m[1]};
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[i][e] *= p.scale_log2;
                if (key0 + KW > low && key0 + 8 * i + c2 + (e & 1) >= limit[e >> 1]) s[i][e] = -INFINITY;
                top[e >> 1] = fmaxf(top[e >> 1], s[i][e]);
            }
        float use[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
            use[i] = top[i] == -INFINITY ? 0.0f : top[i];   // a row without keys so far
            const float f = ex2(m[i] - use[i]);
            m[i] = top[i];
            l[i] *= f;
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
                o[d][2 * i] *= f;
                o[d][2 * i + 1] *= f;
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[i][e] = ex2(s[i][e] - use[e >> 1]);
                l[e >> 1] += s[i][e];
            }
        if (key0 + KW > end) {   // the rows behind the last key: whatever their page holds, V counts as zero
            const int from = max(0, end - key0);
            for (int x = lane; x < (KW - from) * (D / 8); x += 32) {
                const int r = wn * KW + from + x / (D / 8);
                *reinterpret_cast<uint4 *>(base + (2 * st + 1) * kTileBytes + tile_chunk<D>(r, x % (D / 8), kTile)) = make_uint4(0, 0, 0, 0);
            }
            if constexpr (WM > 1) named_bar_sync(2 + wn, 32 * WM);   // the warps that share these keys write the same zeros
            else __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) {
            const uint32_t a[4] = {pack2<T>(s[2 * i][0], s[2 * i][1]), pack2<T>(s[2 * i][2], s[2 * i][3]),
                                   pack2<T>(s[2 * i + 1][0], s[2 * i + 1][1]), pack2<T>(s[2 * i + 1][2], s[2 * i + 1][3])};
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                uint32_t b[4];
                ldmatrix_x4_trans(b, sv + tile_chunk<D>(wn * KW + 16 * i + (lane & 15), 2 * d + (lane >> 4), kTile));
                mma_16816<T>(o[2 * d], a, b[0], b[1]);
                mma_16816<T>(o[2 * d + 1], a, b[2], b[3]);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + st);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    if constexpr (WN > 1) {   // join the warps that took the same rows: over the stages, which all warps have read
        constexpr int kPitch = D + 4;
        float *red = reinterpret_cast<float *>(base);                      // [WN - 1][16 WM][kPitch]
        float2 *ml = reinterpret_cast<float2 *>(red + (WN - 1) * 16 * WM * kPitch);
        static_assert(((WN - 1) * 16 * WM * (kPitch + 2)) * 4 <= split_stages<D>() * 2 * kTileBytes, "the join fits the stages");
        named_bar_sync(1, 128);
        if (wn > 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = ((wn - 1) * WM + wm) * 16 + g + 8 * i;
                if ((lane & 3) == 0) ml[r] = make_float2(m[i], l[i]);
#pragma unroll
                for (int d = 0; d < D / 8; ++d)
                    *reinterpret_cast<float2 *>(red + r * kPitch + 8 * d + c2) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
            }
        }
        named_bar_sync(1, 128);
        if (wn > 0) return;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float top = m[i];
#pragma unroll
            for (int w = 0; w < WN - 1; ++w) top = fmaxf(top, ml[(w * WM + wm) * 16 + g + 8 * i].x);
            const float use = top == -INFINITY ? 0.0f : top, f = ex2(m[i] - use);
            m[i] = top;
            l[i] *= f;
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
                o[d][2 * i] *= f;
                o[d][2 * i + 1] *= f;
            }
#pragma unroll
            for (int w = 0; w < WN - 1; ++w) {
                const int r = (w * WM + wm) * 16 + g + 8 * i;
                const float2 x = ml[r];
                const float fw = ex2(x.x - use);
                l[i] += fw * x.y;
#pragma unroll
                for (int d = 0; d < D / 8; ++d) {
                    const float2 y = *reinterpret_cast<const float2 *>(red + r * kPitch + 8 * d + c2);
                    o[d][2 * i] += fw * y.x;
                    o[d][2 * i + 1] += fw * y.y;
                }
            }
        }
    }
    if (*abort_flag) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (row[i] >= rows) continue;
        const int j = row[i] / p.group, hq = head * p.group + row[i] - j * p.group;
        const size_t at = (size_t)(first + j) * p.q_heads + hq;
        if (p.direct) {
            const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
            uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<T *>(p.out) + at * D + c2);
#pragma unroll
            for (int d = 0; d < D / 8; ++d) dst[4 * d] = pack2<T>(o[d][2 * i] * inv, o[d][2 * i + 1] * inv);
        } else {
            const size_t to = (size_t)slot * p.batch.rows * p.q_heads + at;
            float *dst = p.part_o + to * D + c2;
#pragma unroll
            for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2 *>(dst + 8 * d) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
            if ((lane & 3) == 0) p.part_ml[to] = make_float2(m[i], l[i]);
        }
    }
}

// The join: one warp a (row, query head), each lane D / 32 columns.  Reads the slots' parts once, mostly from L2, eight
// slots at a time (their addresses do not depend on their maxima, so all loads of a row are on the way together); a row
// of no sequence is left as it is, a row without keys becomes zero.
template <typename T, int D>
__global__ void __launch_bounds__(256) attend_join_kernel(const __grid_constant__ AttendParams p) {
    constexpr int C = D / 32, kBatch = 8;
    __shared__ int owner[8], own_slots[8];   // of the block's tokens, eight at most
    griddep_launch();
    const int tid = threadIdx.x, lane = tid & 31;
    const long long unit0 = (long long)blockIdx.x * 8, units = (long long)p.batch.rows * p.q_heads, unit = unit0 + (tid >> 5);
    const int t0 = (int)(unit0 / p.q_heads), n = (int)(min(unit0 + 8, units) - 1) / p.q_heads - t0 + 1;
    const int t = (int)(unit / p.q_heads), hq = (int)(unit - (long long)t * p.q_heads);
    if (tid < 8) owner[tid] = -1;
    griddep_wait();
    int front = p.prefix_splits;   // the prefix's slots come first
    if (p.tc_blocks && unit < units) {
        const int head = hq / p.group, row = t * p.group + hq - head * p.group;
        front = p.item_slots[head * p.prefix_tiles + row / (2 * kTcTile)];
    }
    __syncthreads();
    for (int b = tid; b < p.batch.batch; b += 256) {   // every sequence looked at by one thread: no chain of dependent loads
        const int first = p.batch.start[b], next = p.batch.start[b + 1], len = p.batch.len[b];
        const int lo = max(first, t0), hi = min(next, t0 + n);
        if (lo < hi && sequence_fits(p, first, next - first, len))
            for (int x = lo; x < hi; ++x) {
                owner[x - t0] = b;
                own_slots[x - t0] = (min(len, own_limit(len, next - first, x - first)) + p.own_chunk - 1) / p.own_chunk;
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
    int tc_blocks;          // > 0: the prefix on tcgen05, by this many blocks
    int own_wm, prefix_wm;
    int own_tiles, prefix_tiles, own_chunk, own_splits, prefix_chunk, prefix_splits;
    bool direct;
    size_t units, part_floats;   // rows * q_heads; floats of the parts
};

int row_warps(long long rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

// Rows that share the prefix's keys from which it goes to tcgen05.
constexpr int kTcRows = 64;

// Blocks of the tcgen05 kernel.  It takes whole SMs (one block each) and is bound by the tensor cores and the softmax, the own
// keys' kernel behind it by HBM, and runs on the SMs that are left; so with n blocks the call takes about
//   t = units / n * tile + start,  plus what the other SMs - n have not moved by then at the whole machine's rate,
// and n minimises that.  Measured: a tile of 256 rows and 128 keys 2.4 us with head_dim 128, 2.1 below; an SM alone draws about
// 85 GB/s, all together 5.8 TB/s.  Lengths are on the device: half of their bound is assumed.
int choose_tc_blocks(const KvCache &c, long long units, double own_bytes) {
    const int sms = sm_count();
    const double tile = c.head_dim == 128 ? 2.4e-6 : 2.1e-6, start = 6e-6, one = 85e9, all = 5.8e12;
    int best = 1;
    double least = 1e30;
    for (int n = (int)std::min<long long>(units, sms); n >= 1 && n >= sms / 8; --n) {
        const double t = (double)((units + n - 1) / n) * tile + start, left = std::max(0.0, own_bytes - (sms - n) * one * t);
        if (t + left / all < least) {
            least = t + left / all;
            best = n;
        }
    }
    return best;
}

// Row tiles of 16, 32 or 64 rows by the rows that share the keys, and slots of whole 64-key stages such
// that all blocks together are about `kWaves` rounds of two blocks an SM: fewer would leave SMs idle, more would
// add parts to write and join.
Plan make_plan(const KvCache &c, int batch, int rows, int q_heads, int prefix_len, int max_new, int max_len) {
    constexpr int kWaves = 2;
    Plan p;
    const int group = q_heads / c.kv_heads;
    const long long own_rows = (long long)max_new * group, prefix_rows = (long long)rows * group;
    const bool tc = prefix_rows > kTcRows && prefix_len > 0;
    p.own_wm = row_warps(own_rows);
    p.prefix_wm = row_warps(prefix_rows);
    p.own_tiles = (int)((own_rows + 16 * p.own_wm - 1) / (16 * p.own_wm));
    const int tile_rows = tc ? 2 * kTcTile : 16 * p.prefix_wm;
    p.prefix_tiles = (int)((prefix_rows + tile_rows - 1) / tile_rows);
    const long long own_steps = (max_len + kTile - 1) / kTile, prefix_steps = (prefix_len + kTile - 1) / kTile;
    const long long total = c.kv_heads * (own_steps * batch * p.own_tiles + (tc ? 0 : prefix_steps * p.prefix_tiles));
    const long long per = std::max<long long>(1, total / (2LL * kWaves * sm_count()));
    p.own_chunk = (int)std::min(per, std::max(1LL, own_steps)) * kTile;
    p.own_splits = (int)((max_len + p.own_chunk - 1) / p.own_chunk);
    p.prefix_chunk = (int)std::min(per, std::max(1LL, prefix_steps)) * kTile;
    p.prefix_splits = (int)(((long long)prefix_len + p.prefix_chunk - 1) / p.prefix_chunk);
    p.tc_blocks = 0;
    if (tc) {
        const long long tiles = (prefix_len + kTcTile - 1) / kTcTile, units = tiles * c.kv_heads * p.prefix_tiles;
        p.tc_blocks = choose_tc_blocks(c, units, 0.5 * 4.0 * batch * max_len * c.kv_heads * c.head_dim);
        const long long each = units / p.tc_blocks;   // a block's units at least
        p.prefix_splits = (int)std::min<long long>((tiles + each - 2) / each + 1, p.tc_blocks);
    }
    if (p.own_splits + p.prefix_splits == 0) p.own_splits = 1;   // no keys at all: the rows are still written
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

template <typename T, int D, int WM>
int launch_split(const AttendParams &p, long long blocks, const char *name) {
    static bool set[64] = {};
    if (int rc = allow_smem(attend_split_kernel<T, D, WM>, split_smem<D>(), set, name)) return rc;
    if (blocks > 0x7fffffffLL) return fail(kBadArg, "%s: %lld blocks are too many", name, blocks);
    launch_pdl(attend_split_kernel<T, D, WM>, dim3((unsigned)blocks), dim3(kSplitThreads), split_smem<D>(), p);
    ZB_LAUNCH_CHECK(name);
    return kOk;
}

template <typename T, int D>
int run_split(const AttendParams &p, int wm, long long blocks, const char *name) {
    if (blocks == 0) return kOk;
    return wm == 1 ? launch_split<T, D, 1>(p, blocks, name)
                   : wm == 2 ? launch_split<T, D, 2>(p, blocks, name) : launch_split<T, D, 4>(p, blocks, name);
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
        if (int rc = run_split<T, D>(p, plan.own_wm, own ? own + 1 : 0, name)) return rc;
    } else if (plan.own_wm == plan.prefix_wm) {
        p.prefix_items = (int)prefix;
        if (int rc = run_split<T, D>(p, plan.own_wm, prefix + own, name)) return rc;
    } else {
        p.prefix_items = (int)prefix;
        if (int rc = run_split<T, D>(p, plan.prefix_wm, prefix, name)) return rc;
        p.prefix_items = 0;
        if (int rc = run_split<T, D>(p, plan.own_wm, own, name)) return rc;
    }
    if (p.direct) return kOk;
    launch_pdl(attend_join_kernel<T, D>, dim3((unsigned)((plan.units + 7) / 8)), dim3(256), 0, p);
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
                                      {c->k_id, 0, "the cache"},
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
