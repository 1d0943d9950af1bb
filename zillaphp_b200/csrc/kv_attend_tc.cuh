// kv_attend_tc.cuh -- the shared prefix's part of zilla_kv_attend on tcgen05, for batches with enough rows
// (tokens x query heads of a kv head) and keys.
//
// An item is two 128-row tiles ("streams") of one kv head; both streams use each K and V tile of 128 keys, so a
// tile crosses L2 once for 256 rows.  Items run over the heads first, then over the rows, and a block takes an even share of
// all items' key tiles (PrefixCut): parts of one to a few items ("segments"), one after the other.  With a block count that
// the row tiles divide, the blocks of all row tiles stand at the same keys at the same time and read them from HBM once
// (128 sequences of 2 to 5 tokens, head_dim 128, 16384 shared keys and up to 2048 own, in a loop: 217 to 225 us, 235 to 246 with
// the rows first; 32768 shared keys 359 to 368, 382 to 392).  Per tile and stream, in two steps of 64 keys:
//   S = Q K^T          M = 128 rows, N = 64 keys, K = head_dim, fp32 in TMEM
//   P = 2^(S - ref)    one thread a row; P (16 bits) replaces S in TMEM, two keys a column
//   O += P V           A = P from TMEM, B = V [key][d] (N-major), N = head_dim, K = 64 keys, fp32 in TMEM
// A stream has two S buffers of 64 columns, so that S of the next step is there when P of this one is done: the softmax
// never waits for an MMA of its own stream.  One buffer of 128 keys makes softmax, P V and Q K^T a chain: 206 us against 199
// at full clock for the large batch above, with each row's softmax shared by two warps and the streams issued in turn (260 if
// both streams' MMAs are issued side by side, which keeps them in step).  That sharing alone changes nothing (200), nor does
// a delay between the streams.  A further tile takes 1.7 us with head_dim 128 at full clock (from 16384 to 32768 shared keys),
// 88% of what the measured matrix rate would give; the whole kernel of the large batch, with its start, its parts, 1804 rows in
// 2048 and 96 blocks, has the tensor pipe active for 48% of their SMs' time.
// ref is the row's maximum as of its last change: it follows the true maximum only when that has passed it
// by 2^8 (then O and l are rescaled), so that O rarely has to travel through registers; weights stay
// below 2^8 and l and O carry the same factor, so the quotient does not change.  Before the first finite score (a key may
// be infinite) it is the lowest number: weights of zero, and the first finite score sets it, however low.
// Warps 0-3 and 4-7 are the streams' softmax, warp 8 loads (TMA through the page list), warps 9 and 10 issue the streams'
// MMAs, so that a wait for one stream's softmax does not hold up the other's step.
//
// Order of a stream's MMAs: P V of step h, then Q K^T of step h + 2 over the same TMEM columns; one thread
// issues both and the tensor pipe takes them in order.
#pragma once

#include <float.h>

#include "kv_attend.cuh"

namespace zb {
namespace kv {

using namespace tc;

constexpr int kTcTile = 128;      // rows of a stream, keys of a tile
constexpr int kTcStep = 64;       // keys of a step
constexpr int kTcThreads = 352;

template <int D>
constexpr int tc_stages() { return D == 128 ? 5 : 8; }
template <int D>
constexpr int tc_smem() { return (2 + tc_stages<D>()) * kTcTile * D * 2 + 1024 + 256; }

template <typename T>
constexpr uint32_t attend_idesc(int n, bool b_mn) {
    return __is_same(T, __half) ? (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24)
                                : idesc_bf16(128, n, false, b_mn);
}

// D += A B with A in TMEM (16-bit elements, two a column).
__device__ __forceinline__ void mma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// 32 lanes x 32 columns, without the wait.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// Waits for the thread's TMEM loads; the registers pass through, so nothing that reads them moves ahead.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 unpack_f32x2(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 1) attend_tc_kernel(const __grid_constant__ AttendParams p) {
    constexpr int ST = tc_stages<D>(), kTileBytes = kTcTile * D * 2, kHalves = D == 128 ? 2 : 1, kRowBytes = D < 64 ? D * 2 : 128;
    constexpr int kHalfBytes = kTcTile * 128;                       // one 64-column block of a tile (D >= 64)
    constexpr Swizzle kSw = D == 32 ? kSw64 : kSw128;
    constexpr uint32_t kAtom = D == 32 ? 512 : 1024;                // eight rows
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *base = smem_raw + (((raw + 1023u) & ~1023u) - raw);    // Q of both streams, then the ring
    uint8_t *ring = base + 2 * kTileBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(ring + ST * kTileBytes);
    uint64_t *full = bars, *empty = bars + ST, *q_full = bars + 2 * ST, *s_full = q_full + 1, *p_full = s_full + 4, *o_done = p_full + 4, *drain = o_done + 4;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int rows = p.batch.rows * p.group;
    const PrefixCut cut = prefix_cut(p.batch.prefix_len, p.kv_heads * p.prefix_tiles, p.tc_blocks);
    const int unit0 = cut.begin(blockIdx.x), unit1 = cut.begin(blockIdx.x + 1);
    // the block's segments in order, the same in every role: fn(item, first row, streams, first tile, tiles) until it returns false
    auto segments = [&](auto fn) {
        for (int unit = unit0; unit < unit1;) {
            const int item = unit / cut.tiles, tile0 = unit - item * cut.tiles, tiles = min(cut.tiles - tile0, unit1 - unit);
            const int row0 = item / p.kv_heads * 2 * kTcTile;
            if (!fn(item, row0, rows - row0 > kTcTile ? 2 : 1, tile0, tiles)) return;
            unit += tiles;
        }
    };

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 2);        // both streams
        }
        mbar_init(q_full, 8);
        for (int i = 0; i < 4; ++i) {   // [stream][step & 1]: a waiter is at most one phase behind
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);       // one arrival a warp: 128 on one barrier queue up behind each other
            mbar_init(o_done + i, 1);
        }
        mbar_init(drain, 1);
        mbar_init(drain + 1, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    griddep_wait();
    griddep_launch();   // behind the wait: a kernel started by it finds everything before this one done

    if (warp == 8) {
        // ---- loads: K and V tiles alternate through the ring
        const int boxes = kTcTile / p.box_rows, all = boxes * kHalves;   // 2 .. 16
        const int r0 = lane % boxes * p.box_rows, half = lane / boxes;
        bool ok = true;
        int i = 0;   // loads so far: K of a tile, then V
        segments([&](int item, int, int, int tile0, int tiles) {
            const int head = item % p.kv_heads;
            for (int x = 0; x < 2 * tiles; ++x, ++i) {
                const int st = i % ST;
                const int at = lane < all ? box_row(p, p.prefix_pages, head, (tile0 + (x >> 1)) * kTcTile + r0, p.batch.prefix_len) : 0;
                ok = i < ST || wait_phase(empty + st, (i / ST - 1) & 1, abort_flag, p.err, kErrEmptyWait);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return false;
                if (lane == 0) mbar_arrive_expect_tx(full + st, kTileBytes);
                __syncwarp();
                if (lane < all)
                    tma_load_2d(ring + st * kTileBytes + half * kHalfBytes + r0 * kRowBytes, x & 1 ? &p.v_map : &p.k_map, full + st, half * 64, at);
            }
            return true;
        });
        if (!ok && lane == 0)   // the copies in flight end before the block's shared memory goes
            for (int x = max(0, i - ST); x < i; ++x)
                if (!mbar_wait_drain(full + x % ST, (x / ST) & 1)) atomicCAS(p.err, 0, kErrDrain);
    } else if (warp > 8) {
        // ---- MMAs of one stream.  The whole warp runs the loop, one elected lane issues: addresses stay in uniform
        // registers, and a step's twelve MMAs follow each other without work between them.
        const int s = warp - 9;
        constexpr uint32_t kIdS = attend_idesc<T>(kTcStep, false), kIdO = attend_idesc<T>(D, true);
        constexpr uint32_t kStep16 = kTcStep * kRowBytes / 16, kTile16 = kTileBytes / 16;   // in the descriptors' units of 16 bytes
        const uint64_t q_desc = smem_desc(smem_u32(base), 16, kAtom, kSw), k_desc = smem_desc(smem_u32(ring), 16, kAtom, kSw),
                       v_desc = smem_desc(smem_u32(ring), kHalfBytes, kAtom, kSw);
        struct Place {   // a load's place in the ring
            int st = 0, turn = 0;
            __device__ __forceinline__ void next() {
                if (++st == ST) {
                    st = 0;
                    turn ^= 1;
                }
            }
        };
        auto wait_load = [&](const Place &x) { return wait_phase(full + x.st, x.turn, abort_flag, p.err, kErrFullWait); };
        const uint32_t s_at = tmem + s * 128, o_at = tmem + 256 + s * D;
        auto qk = [&](int h, int st) {   // step h of a tile, whose K is in stage st
            const uint64_t a = q_desc + s * kTile16, b = k_desc + st * kTile16 + h * kStep16;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t at = ((k >> 2) * kHalfBytes + (k & 3) * 32) / 16;
                    mma_bf16(s_at + h * kTcStep, a + at, b + at, kIdS, k != 0);
                }
                mma_commit(s_full + 2 * s + h);
            }
            __syncwarp();
        };
        auto pv = [&](int h, int st, bool more, bool last) {
            const uint64_t b = v_desc + st * kTile16 + h * kStep16;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kTcStep / 16; ++k)
                    mma_f16_ta(o_at, s_at + h * kTcStep + 8 * k, b + k * (2 * kAtom / 16), kIdO, more || k != 0);
                if (last) mma_commit(o_done + 2 * s + h);
            }
            __syncwarp();
        };
        auto release = [&](int st) {
            if (elect_one()) mma_commit(empty + st);
            __syncwarp();
        };
        bool ok = true;
        int done = 0, segment = 0;   // tiles of this stream, segments
        Place k_at, v_at;            // the tile's K and V
        v_at.next();
        segments([&](int, int, int streams, int, int tiles) {
            if (s >= streams) {      // no rows: the tiles are handed back
                ok = wait_phase(q_full, segment++ & 1, abort_flag, p.err, kErrFullWait);   // not to be two phases ahead of it later
                if (!ok) return false;
                for (int x = 0; x < 2 * tiles; ++x) {
                    Place &at = x & 1 ? v_at : k_at;
                    ok = wait_load(at);
                    if (!ok) return false;
                    if (lane == 0) mbar_arrive(empty + at.st);
                    at.next();
                    at.next();
                }
                return true;
            }
            ok = wait_phase(q_full, segment++ & 1, abort_flag, p.err, kErrFullWait) && wait_load(k_at);
            if (!ok) return false;
            tc_fence_after();
            qk(0, k_at.st);
            qk(1, k_at.st);
            release(k_at.st);
            for (int j = 0; j < tiles; ++j, ++done) {
                const bool more = j + 1 < tiles;
                k_at.next();
                k_at.next();
                ok = wait_load(v_at) && (!more || wait_load(k_at)) && wait_phase(p_full + 2 * s, done & 1, abort_flag, p.err, kErrAccWait);
                if (!ok) return false;
                tc_fence_after();
                pv(0, v_at.st, j > 0, !more);
                if (more) qk(0, k_at.st);
                ok = wait_phase(p_full + 2 * s + 1, done & 1, abort_flag, p.err, kErrAccWait);
                if (!ok) return false;
                tc_fence_after();
                pv(1, v_at.st, true, !more);
                release(v_at.st);
                if (more) {
                    qk(1, k_at.st);
                    release(k_at.st);
                }
                v_at.next();
                v_at.next();
            }
            return true;
        });
        if (!ok) {   // MMAs in flight end before TMEM goes
            if (elect_one()) {
                mma_commit(drain + s);
                if (!mbar_wait_drain(drain + s, 0)) atomicCAS(p.err, 0, kErrDrain);
            }
            __syncwarp();
        }
    } else {
        // ---- softmax: thread = row of the stream
        const int s = warp >> 2, r = threadIdx.x & (kTcTile - 1);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + lanes + s * 128, to = tmem + lanes + 256 + s * D;
        const float sl = fmaxf(fabsf(p.scale_log2), 1e-30f);   // above zero: a masked -inf stays one
        const uint64_t sl2 = pack_f32x2(sl, sl);
        int done = 0, loads = 0, segment = 0, mine = 0;   // steps of this stream, loads of the ring, segments, this stream's segments
        segments([&](int item, int row0, int streams, int tile0, int tiles) {
            if (s >= streams) {   // no rows here; not to arrive for the next segment before this one's queries are there
                if (lane == 0) mbar_arrive(q_full);
                loads += 2 * tiles;
                return __all_sync(0xffffffffu, wait_phase(q_full, segment++ & 1, abort_flag, p.err, kErrAccWait)) != 0;
            }
            ++segment;
            // this warp's 32 rows; row = (token, query head of the kv head), unit its place in q and in the parts
            const int head = item % p.kv_heads, warp_row = row0 + s * kTcTile + (warp & 3) * 32, row = warp_row + lane;
            const int t = row < rows ? p.by_group.div(row) : 0, unit = t * p.q_heads + head * p.group + (row < rows ? row - t * p.group : 0);
            {
                // Q, 16 bytes a lane along the rows.  With a negative scale the queries change their sign, so that the largest
                // product has the largest score.
                const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
                uint4 x[D / 8];
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const int rr = (i * 32 + lane) / (D / 8), c = (i * 32 + lane) % (D / 8), u = __shfl_sync(0xffffffffu, unit, rr);
                    x[i] = warp_row + rr < rows ? reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q) + (size_t)u * D)[c] : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const int rr = (i * 32 + lane) / (D / 8), c = (i * 32 + lane) % (D / 8);
                    x[i].x ^= flip; x[i].y ^= flip; x[i].z ^= flip; x[i].w ^= flip;
                    *reinterpret_cast<uint4 *>(base + s * kTileBytes + tile_chunk<D>((warp & 3) * 32 + rr, c, kTcTile)) = x[i];
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            const int slot = (int)blockIdx.x - cut.first_block(item);
            if (threadIdx.x == 0 && tile0 + tiles == cut.tiles) p.item_slots[item] = slot + 1;
            float ref = 0.0f, l = 0.0f;   // ref in units of log2
            for (int h = 0; h < 2 * tiles; ++h, ++done) {
                const int buf = h & 1;
                bool ok = wait_phase(s_full + 2 * s + buf, (done >> 1) & 1, abort_flag, p.err, kErrAccWait);
                if (!__all_sync(0xffffffffu, ok)) return false;
                tc_fence_after();
                uint32_t v[2][32];
                tmem_ld32_async(ts + buf * kTcStep, v[0]);
                tmem_ld32_async(ts + buf * kTcStep + 32, v[1]);
                tmem_ld_wait(v[0]);
                tmem_ld_wait(v[1]);
                const int left = p.batch.prefix_len - tile0 * kTcTile - h * kTcStep;   // keys from this step's first on
                if (left < kTcTile) {
                    if (left < kTcStep) {   // the missing keys
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (32 * c + i >= left) v[c][i] = 0xff800000u;
                    }
                    if (!buf) {   // V behind the last key counts as zero, whatever its page holds
                        const int load = loads + h + 1, st = load % ST;
                        ok = wait_phase(full + st, (load / ST) & 1, abort_flag, p.err, kErrFullWait);
                        if (!__all_sync(0xffffffffu, ok)) return false;
                        for (int x = r; x < (kTcTile - left) * (D / 8); x += kTcTile)
                            *reinterpret_cast<uint4 *>(ring + st * kTileBytes + tile_chunk<D>(left + x / (D / 8), x % (D / 8), kTcTile)) =
                                make_uint4(0, 0, 0, 0);
                        fence_proxy_async_smem();
                    }
                }
                float top[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top[c] = __uint_as_float(v[c >> 1][(c & 1) * 16]);
#pragma unroll
                    for (int i = 1; i < 16; ++i) top[c] = fmaxf(top[c], __uint_as_float(v[c >> 1][(c & 1) * 16 + i]));
                }
                const float m = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * sl, -FLT_MAX);
                if (h == 0) ref = m;
                else if (__any_sync(0xffffffffu, m > ref + 8.0f)) {
                    // O with the step before in it: S of the next step is committed behind that, or the segment's last steps themselves
                    ok = h + 1 < 2 * tiles ? wait_phase(s_full + 2 * s + (buf ^ 1), ((done + 1) >> 1) & 1, abort_flag, p.err, kErrAccWait)
                                           : wait_phase(o_done + 2 * s + (buf ^ 1), mine & 1, abort_flag, p.err, kErrAccWait);
                    if (!__all_sync(0xffffffffu, ok)) return false;
                    tc_fence_after();
                    const float f = m > ref ? ex2(ref - m) : 1.0f;
                    ref = fmaxf(ref, m);
                    l *= f;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32_async(to + 32 * c, o);
                        tmem_ld_wait(o);
                        uint32_t w[2][16];
#pragma unroll
                        for (int i = 0; i < 32; ++i) w[i >> 4][i & 15] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st16(to + 32 * c, w[0]);
                        tmem_st16(to + 32 * c + 16, w[1]);
                    }
                }
                const uint64_t nref = pack_f32x2(-ref, -ref);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 x = unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[c][2 * i]), __uint_as_float(v[c][2 * i + 1])), sl2, nref));
                        const float a = ex2(x.x), b = ex2(x.y);
                        sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(a, b));
                        w[i] = pack2<T>(a, b);
                    }
                    tmem_st16(ts + buf * kTcStep + 16 * c, w);
                }
                const float2 add = unpack_f32x2(add_f32x2(sum[0], sum[1]));
                l += add.x + add.y;
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 2 * s + buf);
            }
            loads += 2 * tiles;
            bool ok = wait_phase(o_done + 2 * s + 1, mine++ & 1, abort_flag, p.err, kErrAccWait);
            if (!__all_sync(0xffffffffu, ok)) return false;
            tc_fence_after();
            // O through shared memory (over this warp's rows of Q, whose MMAs are done), so that whole lines are written
            constexpr int kCols = D >= 64 ? 32 : 16, kChunks = kCols / 4;
            uint32_t high[16];   // head_dim 32: two halves of 16 columns, as its Q leaves no more room
            uint8_t *stage = base + s * kTileBytes + (warp & 3) * 32 * kRowBytes;   // its rows of the first block: no other warp writes there
            const size_t at = (size_t)slot * p.batch.rows * p.q_heads;
#pragma unroll
            for (int c = 0; c < D / kCols; ++c) {
                uint32_t o[32];
                if constexpr (kCols == 32) {
                    tmem_ld32_async(to + 32 * c, o);
                    tmem_ld_wait(o);
                } else if (c == 0) {
                    tmem_ld32_async(to, o);
                    tmem_ld_wait(o);
#pragma unroll
                    for (int i = 0; i < 16; ++i) high[i] = o[16 + i];
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = high[i];
                }
#pragma unroll
                for (int i = 0; i < kChunks; ++i)
                    *reinterpret_cast<uint4 *>(stage + lane * kCols * 4 + ((i ^ (lane & (kChunks - 1))) << 4)) =
                        make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    const int rr = (i * 32 + lane) / kChunks, x = (i * 32 + lane) % kChunks, u = __shfl_sync(0xffffffffu, unit, rr);
                    const uint4 y = *reinterpret_cast<const uint4 *>(stage + rr * kCols * 4 + ((x ^ (rr & (kChunks - 1))) << 4));
                    if (warp_row + rr < rows) reinterpret_cast<uint4 *>(p.part_o + (at + u) * D + c * kCols)[x] = y;
                }
                __syncwarp();
            }
            if (row < rows) p.part_ml[at + unit] = make_float2(ref, l);
            tc_fence_before();
            return true;
        });
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace kv
}  // namespace zb
