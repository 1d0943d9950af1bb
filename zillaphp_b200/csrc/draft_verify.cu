// draft_verify.cu -- drafted tokens against the target's probabilities, from
// given random numbers (draft_verify_dev).
//
// Sequence b's rows are start[b] .. start[b] + k, k drafts and the row behind the last one.  With
// p_j, q_j the target's and the drafter's probabilities of row j, d_j the draft and u_j its number:
//   accept d_j while u_j q_j(d_j) < p_j(d_j); a = the number accepted;
//   w = max(p_a - q_a, 0) where a draft failed, p_a behind the last one;
//   the token drawn is the lowest t with w_0 + ... + w_t > r (w_0 + ... + w_{V-1}), r = u_k.
// fp32 sums over a large vocabulary are off by more than the distance between neighbouring borders, and would make
// the token depend on how a row is split: weights are differences in fp64 and summed in fp64, a thread's four together, so
// that its chain of additions is short (192 rows of 100,003 in a graph of calls 28.6 us; one after the other 29.9).  A sum
// is off by at most 2^-53 of itself for each addition behind each other: V / 4096 a thread and some 50 to join them.
#include <cooperative_groups.h>
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.cuh"

namespace cg = cooperative_groups;

namespace zb {
namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxCluster = 8;

struct VerifyParams {
    const float *p, *q;    // q nullptr: the drafts are certain (q is one at the draft)
    long long p_ld, q_ld;
    const int *draft, *start;
    const float *u;
    int *tokens, *accepted;
    int rows, vocab, seg;   // seg: elements of one warp's segment, a multiple of 128
    int *err;
};

// w_t of one element in fp64; NaN counts as 0, an infinity as the largest finite number.
__device__ __forceinline__ double residual(float p, float q) {
    return p > q ? (double)fminf(p, FLT_MAX) - (double)fmaxf(q, -FLT_MAX) : 0.0;
}

// Bound by HBM: one row of p, and one of q where a draft failed, read once by the sequence's cluster.
// Each warp sums one segment of the row; the segments' sums meet in the cluster's shared memory, and the
// block that owns the crossing segment reads it again (it is in L2) to find the token.
// Six blocks an SM (40 registers a thread), so that blocks that look for their row or for their token leave enough others
// that stream: 28.6 us against 31.2 with four.  ALONE: so few blocks that no SM has a second one; then a thread's own loads
// have to cover the latency, and four times as many are in flight (one row of 131,072: 7.2 against 8.5 us).
template <bool VEC, bool ALONE>
__global__ void __launch_bounds__(kVerifyThreads, ALONE ? 1 : 6) draft_verify_kernel(const VerifyParams a) {
    __shared__ double sums[kVerifyWarps];                      // read by the whole cluster
    __shared__ double all[kVerifyMaxCluster * kVerifyWarps];
    __shared__ double part[kVerifyWarps], s_base, s_target;
    __shared__ int s_taken, s_seg, s_found, s_last;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int b = blockIdx.x / ranks;
    griddep_launch();
    griddep_wait();
    const int first = a.start[b], n = a.start[b + 1] - first;
    if (first < 0 || n <= 0 || (long long)first + n > a.rows) {   // the same in every block of the cluster
        if (rank == 0 && tid == 0) {
            if (n != 0) atomicCAS(a.err, 0, kErrDraft);
            a.accepted[b] = 0;
        }
        return;
    }
    const int k = n - 1, V = a.vocab;
    if (warp == 0) {
        int taken = k;
        for (int j0 = 0; j0 < k && taken == k; j0 += 32) {
            const int j = j0 + lane;
            bool fails = false;
            if (j < k) {
                const int row = first + j, d = a.draft[row];
                if (d < 0 || d >= V) {
                    atomicCAS(a.err, 0, kErrDraft);
                    fails = true;
                } else {
                    const float pd = a.p[(size_t)row * a.p_ld + d], qd = a.q ? a.q[(size_t)row * a.q_ld + d] : 1.0f;
                    fails = !((double)a.u[row] * (double)qd < (double)pd);
                }
            }
            const unsigned no = __ballot_sync(0xffffffffu, fails);
            if (no) taken = j0 + __ffs(no) - 1;
        }
        if (lane == 0) s_taken = taken;
        if (rank == 0) {
            for (int j = lane; j < n; j += 32)
                if (j != taken) a.tokens[first + j] = j < taken ? a.draft[first + j] : -1;
            if (lane == 0) a.accepted[b] = taken;
        }
    }
    __syncthreads();
    const int taken = s_taken, row = first + taken;
    const double r = (double)a.u[first + k];
    const float *p = a.p + (size_t)row * a.p_ld;
    const float *q = taken < k && a.q ? a.q + (size_t)row * a.q_ld : nullptr;
    int skip = taken < k && !a.q ? a.draft[row] : -1;   // a certain draft that failed is not drawn again
    // two passes only where no residual is left (every p_t <= q_t, as rounded rows can have it): the
    // second draws from p itself
    for (int pass = 0; pass < 2; ++pass) {
        auto w = [&](int i) { return i == skip ? 0.0 : residual(p[i], q ? q[i] : 0.0f); };
        const long long lo = (long long)(rank * kVerifyWarps + warp) * a.seg;
        const int begin = (int)min(lo, (long long)V), end = (int)min(lo + a.seg, (long long)V);
        double s = 0.0;
        auto weigh = [&](int i, float x, float y) { return i == skip ? 0.0 : residual(x, y); };
        // a batch of loads in front of its sums: 64 bytes a thread in flight, or 256
        auto stream = [&](auto with_q) {
            constexpr bool kQ = decltype(with_q)::value;
            if constexpr (VEC) {
                constexpr int kBatch = (kQ ? 2 : 4) * (ALONE ? 4 : 1);
                auto take4 = [&](int i, const float4 &x, const float4 &y) {
                    s += (weigh(i, x.x, y.x) + weigh(i + 1, x.y, y.y)) + (weigh(i + 2, x.z, y.z) + weigh(i + 3, x.w, y.w));
                };
                int i = begin + 4 * lane;
                const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (; i + 3 + 128 * (kBatch - 1) < end; i += 128 * kBatch) {
                    float4 x[kBatch], y[kBatch];
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) {
                        x[e] = *reinterpret_cast<const float4 *>(p + i + 128 * e);
                        y[e] = kQ ? *reinterpret_cast<const float4 *>(q + i + 128 * e) : zero;
                    }
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) take4(i + 128 * e, x[e], y[e]);
                }
                for (; i + 3 < end; i += 128)
                    take4(i, *reinterpret_cast<const float4 *>(p + i), kQ ? *reinterpret_cast<const float4 *>(q + i) : zero);
                for (; i < end; ++i) s += weigh(i, p[i], kQ ? q[i] : 0.0f);   // the row's last one to three elements, one lane's
            } else {
                constexpr int kBatch = (kQ ? 4 : 8) * (ALONE ? 4 : 1);
                int i = begin + lane;
                for (; i + 32 * (kBatch - 1) < end; i += 32 * kBatch) {
                    float x[kBatch], y[kBatch];
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) {
                        x[e] = p[i + 32 * e];
                        y[e] = kQ ? q[i + 32 * e] : 0.0f;
                    }
#pragma unroll
                    for (int e = 0; e < kBatch; e += 2) s += weigh(i + 32 * e, x[e], y[e]) + weigh(i + 32 * (e + 1), x[e + 1], y[e + 1]);
                }
                for (; i < end; i += 32) s += weigh(i, p[i], kQ ? q[i] : 0.0f);
            }
        };
        if (q) stream(std::true_type());
        else stream(std::false_type());
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) sums[warp] = s;
        cluster.sync();
        for (int i = tid; i < kVerifyMaxCluster * kVerifyWarps; i += kVerifyThreads)
            all[i] = i < ranks * kVerifyWarps ? cluster.map_shared_rank(sums, i / kVerifyWarps)[i % kVerifyWarps] : 0.0;
        cluster.barrier_arrive();   // waited for below: no block leaves, or sums again, while another still reads
        __syncthreads();
        if (warp == 0) {  // every block works out the same
            constexpr int kEach = kVerifyMaxCluster * kVerifyWarps / 32;   // segments a lane
            const double *v = all + kEach * lane;
            double incl = 0.0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) incl += v[e];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            double run = __shfl_up_sync(0xffffffffu, incl, 1);
            if (lane == 0) run = 0.0;
            const double total = __shfl_sync(0xffffffffu, incl, 31), target = r * total;
            int hit = -1, last = -1;
            double hit_base = 0.0, last_base = 0.0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (v[e] > 0.0) {
                    last = kEach * lane + e;
                    last_base = run;
                    if (hit < 0 && run + v[e] > target) {
                        hit = last;
                        hit_base = run;
                    }
                }
                run += v[e];
            }
            const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), lasts = __ballot_sync(0xffffffffu, last >= 0);
            // no border lies above the number (one that is 1 or more): the last segment with a weight
            const int who = hits ? __ffs(hits) - 1 : 31 - __clz(lasts | 1u);
            if (lane == who) {
                s_seg = hits ? hit : last;   // -1: nothing to draw from
                s_base = hits ? hit_base : last_base;
                s_target = target;
            }
        }
        if (tid == 0) {
            s_found = 0x7fffffff;
            s_last = -1;
        }
        __syncthreads();
        const int seg = s_seg;
        if (seg < 0 && pass == 1) {
            if (rank == 0 && tid == 0) a.tokens[row] = 0;
        } else if (seg >= 0 && seg / kVerifyWarps == rank) {
            // the whole block reads the crossing segment again: a few neighbours a thread
            const long long from = (long long)seg * a.seg;
            const int stop = (int)min(from + a.seg, (long long)V), per = (a.seg + kVerifyThreads - 1) / kVerifyThreads;
            const int i0 = min((int)from + tid * per, stop), i1 = min(i0 + per, stop);
            double mine = 0.0;
#pragma unroll 8
            for (int i = i0; i < i1; ++i) mine += w(i);
            double incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            if (lane == 31) part[warp] = incl;
            __syncthreads();
            double run = s_base;
            for (int i = 0; i < warp; ++i) run += part[i];
            run += incl - mine;
            int found = 0x7fffffff, last = -1;
            for (int i = i0; i < i1; ++i) {
                const double e = w(i);
                run += e;
                if (e > 0.0) {
                    last = i;
                    if (run > s_target && found == 0x7fffffff) found = i;
                }
            }
            if (found != 0x7fffffff) atomicMin(&s_found, found);
            if (last >= 0) atomicMax(&s_last, last);
            __syncthreads();
            if (tid == 0) a.tokens[row] = s_found != 0x7fffffff ? s_found : s_last;
        }
        cluster.barrier_wait();
        if (seg >= 0) return;
        q = nullptr;
        skip = -1;
        __syncthreads();   // s_seg is read by all before it is written again
    }
}

cudaLaunchConfig_t verify_launch(cudaLaunchAttribute *attr, int blocks, int ranks) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kVerifyThreads);
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

// Clusters of `ranks` blocks that the machine holds at once (worked out once a size).
int clusters_at_once(void (*kernel)(VerifyParams), bool vec, int ranks) {
    static int found[2][kVerifyMaxCluster + 1] = {};
    int &n = found[vec][ranks];
    if (!n) {
        cudaLaunchAttribute attr[1];
        const cudaLaunchConfig_t cfg = verify_launch(attr, ranks, ranks);
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = std::max(1, 5 * sm_count() / ranks);
        }
    }
    return n;
}

// Blocks to a sequence: the most with which all sequences run at once, and in a second round, a third, ... only where a block
// would have more than 24576 elements otherwise (its start and its search at the end then count for little).  Measured against
// eight blocks to a sequence: 192 rows of 32,000 11.4 us against 13.8, 384 rows 21.0 (two blocks) against 27.1; 192 rows of
// 100,003 take eight, 28.6 against 29.6 with four.  A block has 512 elements at least.
int choose_ranks(void (*kernel)(VerifyParams), bool vec, int batch, int vocab) {
    const int most = std::max(1, std::min(kVerifyMaxCluster, vocab / 512)), least = std::min(most, (vocab + 24575) / 24576);
    const int fit = clusters_at_once(kernel, vec, least);
    const long long rounds = ((long long)batch + fit - 1) / fit;
    int ranks = most;
    while (ranks > least && batch > rounds * clusters_at_once(kernel, vec, ranks)) --ranks;
    return ranks;
}

}  // namespace
}  // namespace zb

using namespace zb;

extern "C" int draft_verify_dev(int p_id, int p_ld, int q_id, int q_ld, int draft_id, int u_id, int start_id,
                                int tokens_id, int accepted_id, int batch, int rows, int vocab) {
    const char *name = "draft_verify_dev";
    if (batch < 0 || rows < 0 || vocab < 1 || vocab > (1 << 28))
        return fail(kBadArg, "%s: bad sizes batch=%d rows=%d vocab=%d", name, batch, rows, vocab);
    if (p_ld < vocab || (q_id && q_ld < vocab)) return fail(kBadArg, "%s: a row stride is smaller than vocab", name);
    for (int to : {tokens_id, accepted_id})
        for (int from : {p_id, q_id, draft_id, u_id, start_id})
            if (to && to == from) return fail(kBadArg, "%s: buffer %d is read and written", name, to);
    if (tokens_id && tokens_id == accepted_id) return fail(kBadArg, "%s: tokens and accepted are one buffer", name);
    const size_t n = rows;
    if (int rc = check_buffers(name, {{p_id, rows ? (n - 1) * p_ld + vocab : 0, "p"},
                                      {draft_id, n, "draft"},
                                      {u_id, n, "u"},
                                      {start_id, (size_t)batch + 1, "start"},
                                      {tokens_id, n, "tokens"},
                                      {accepted_id, (size_t)batch, "accepted"}}))
        return rc;
    if (q_id)
        if (int rc = check_buffers(name, {{q_id, rows ? (n - 1) * q_ld + vocab : 0, "q"}})) return rc;
    if (!batch) return kOk;
    VerifyParams a;
    a.p = ptr(p_id);
    a.q = q_id ? ptr(q_id) : nullptr;
    a.p_ld = p_ld;
    a.q_ld = q_ld;
    a.draft = reinterpret_cast<const int *>(ptr(draft_id));
    a.start = reinterpret_cast<const int *>(ptr(start_id));
    a.u = ptr(u_id);
    a.tokens = reinterpret_cast<int *>(ptr(tokens_id));
    a.accepted = reinterpret_cast<int *>(ptr(accepted_id));
    a.rows = rows;
    a.vocab = vocab;
    a.err = device_error_word();
    if (!a.err) return fail(kBadHandle, "%s: no device error word", name);
    const bool vec = p_ld % 4 == 0 && (!q_id || q_ld % 4 == 0);   // rows start on 16 bytes
    const int ranks = choose_ranks(vec ? draft_verify_kernel<true, false> : draft_verify_kernel<false, false>, vec, batch, vocab);
    const int warps = ranks * kVerifyWarps;
    a.seg = ((vocab + warps - 1) / warps + 127) / 128 * 128;
    if ((long long)batch * ranks > 0x7fffffffLL) return fail(kBadArg, "%s: batch %d is too large", name, batch);
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = verify_launch(attr, batch * ranks, ranks);
    cfg.stream = stream();
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
    if (batch * ranks <= sm_count()) cudaLaunchKernelEx(&cfg, vec ? draft_verify_kernel<true, true> : draft_verify_kernel<false, true>, a);
    else cudaLaunchKernelEx(&cfg, vec ? draft_verify_kernel<true, false> : draft_verify_kernel<false, false>, a);
    ZB_LAUNCH_CHECK(name);
    return kOk;
}
