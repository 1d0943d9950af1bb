// kv_cache.cu -- the paged K/V cache: creation, and appending a batch's new
// keys and values with the rotary rotation applied on the way.
#include <map>

#include "kv_cache.cuh"
#include "rope.cuh"

namespace zb {
namespace {

std::map<int, KvCache *> g_caches;
int g_next_cache = 1;

constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 8;

struct AppendParams {
    const void *q, *k, *v;
    void *q_out, *k_cache, *v_cache;
    long long q_ld, k_ld, v_ld;
    const double *table;   // nullptr: no rotation
    KvBatch batch;
    int q_heads, kv_heads, page_log2, pages, tokens;
    RopeShape shape;
    FastDiv per_row, per_head;   // units of a row over all q, k and v heads; units of a head
    int *err;
};

// Bound by HBM for prompts (each element read and written once) and by latency for single tokens: one
// block finds its rows' sequences, slots and angles together, then moves all heads.
template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const AppendParams p) {
    __shared__ int owner[kAppendTokens], pos[kAppendTokens], page_of[kAppendTokens], slot[kAppendTokens];
    __shared__ float2 cs[kAppendTokens * kRopeMaxDim / 2];
    griddep_launch();
    griddep_wait();
    const int tid = threadIdx.x, row0 = blockIdx.x * p.tokens, n = min(p.tokens, p.batch.rows - row0);
    const int half_rot = p.shape.rot >> 1;
    kv_owners(owner, p.batch.start, p.batch.batch, row0, n, tid, kAppendThreads);
    if (tid < n) {
        const int b = owner[tid];
        int at_pos = 0, id = -1, s = 0;
        if (b >= 0) {
            const int first = p.batch.start[b], count = p.batch.start[b + 1] - first, held = p.batch.len[b];
            const int i = held - count + (row0 + tid - first), at = i >> p.page_log2;
            if (i < 0) {
                atomicCAS(p.err, 0, kErrKvLength);
            } else if (at >= p.batch.max_pages) {
                atomicCAS(p.err, 0, kErrKvPage);
            } else {
                id = p.batch.pages[(size_t)b * p.batch.max_pages + at];
                if (id < 0 || id >= p.pages) {
                    atomicCAS(p.err, 0, kErrKvPage);
                    id = -1;
                }
                at_pos = p.batch.prefix_len + i;
                s = i & ((1 << p.page_log2) - 1);
            }
        }
        page_of[tid] = id;   // -1: the row is left alone
        slot[tid] = s;
        pos[tid] = at_pos;
    }
    __syncthreads();
    if (half_rot) {
        rope_angles(cs, pos, n, half_rot, p.table, 1.0f, tid, kAppendThreads);
        __syncthreads();
    }
    const int D = p.shape.head_dim;
    const RopeShape turn = p.shape;
    RopeShape copy = p.shape;   // the values: the same units, none turned; a pair unit then copies two vectors
    const int total = n * (int)p.per_row.d;
#pragma unroll 2
    for (int idx = tid; idx < total; idx += kAppendThreads) {
        const int t = p.per_row.div(idx), in_row = idx - t * (int)p.per_row.d;
        int h = p.per_head.div(in_row);
        const int u = in_row - h * (int)p.per_head.d;
        const int id = page_of[t];
        if (id < 0) continue;
        const float2 *c = cs + t * half_rot;
        if (h < p.q_heads) {
            rope_unit<TI, TO, V>(static_cast<const TI *>(p.q) + (size_t)(row0 + t) * p.q_ld + h * D,
                                 static_cast<TO *>(p.q_out) + ((size_t)(row0 + t) * p.q_heads + h) * D, c, u, turn);
            continue;
        }
        h -= p.q_heads;
        const bool is_k = h < p.kv_heads;
        if (!is_k) h -= p.kv_heads;
        const size_t to = ((((size_t)id * p.kv_heads + h) << p.page_log2) + slot[t]) * D;
        if (is_k) {
            rope_unit<TI, TO, V>(static_cast<const TI *>(p.k) + (size_t)(row0 + t) * p.k_ld + h * D,
                                 static_cast<TO *>(p.k_cache) + to, c, u, turn);
        } else {
            const TI *src = static_cast<const TI *>(p.v) + (size_t)(row0 + t) * p.v_ld + h * D;
            TO *dst = static_cast<TO *>(p.v_cache) + to;
            float a[V];
            if (u < copy.pair_units) {
                const int a_at = copy.interleaved ? 2 * u * V : u * V;
                const int b_at = copy.interleaved ? a_at + V : half_rot + u * V;
                float b[V];
                load_vec<TI, V>(src + a_at, a);
                load_vec<TI, V>(src + b_at, b);
                store_vec<TO, V>(dst + a_at, a);
                store_vec<TO, V>(dst + b_at, b);
            } else {
                const int at = copy.rot + (u - copy.pair_units) * V;
                load_vec<TI, V>(src + at, a);
                store_vec<TO, V>(dst + at, a);
            }
        }
    }
}

template <typename TI, typename TO>
void launch_append(const AppendParams &p, int vec) {
    const dim3 grid((p.batch.rows + p.tokens - 1) / p.tokens), block(kAppendThreads);
    if (vec == 8) launch_pdl(kv_append_kernel<TI, TO, 8>, grid, block, 0, p);
    else if (vec == 4) launch_pdl(kv_append_kernel<TI, TO, 4>, grid, block, 0, p);
    else if (vec == 2) launch_pdl(kv_append_kernel<TI, TO, 2>, grid, block, 0, p);
    else launch_pdl(kv_append_kernel<TI, TO, 1>, grid, block, 0, p);
}

}  // namespace

const KvCache *kv_get(int id) {
    auto it = g_caches.find(id);
    if (it == g_caches.end()) return nullptr;
    const KvCache *c = it->second;
    return ptr(c->k_id) == c->k && ptr(c->v_id) == c->v ? c : nullptr;
}

}  // namespace zb

using namespace zb;

extern "C" {

int zilla_kv_create(int pages, int page, int kv_heads, int head_dim, int type) {
    const char *name = "zilla_kv_create";
    if (type != kBf16 && type != kF16) return fail(kBadArg, "%s: the cache is bf16 (1) or fp16 (2), not type %d", name, type);
    if (page != 16 && page != 32 && page != 64 && page != 128)
        return fail(kBadArg, "%s: a page holds 16, 32, 64 or 128 tokens, not %d", name, page);
    if (head_dim != 32 && head_dim != 64 && head_dim != 128)
        return fail(kBadArg, "%s: head_dim is 32, 64 or 128, not %d", name, head_dim);
    if (pages < 1 || kv_heads < 1 || kv_heads > 1024) return fail(kBadArg, "%s: bad sizes pages=%d kv_heads=%d", name, pages, kv_heads);
    const long long rows = (long long)pages * kv_heads * page;
    if (rows > 0x7fffffffLL - 128) return fail(kBadArg, "%s: %lld rows of keys are too many", name, rows);
    KvCache *c = new KvCache();
    c->pages = pages;
    c->page = page;
    while ((1 << c->page_log2) < page) ++c->page_log2;
    c->kv_heads = kv_heads;
    c->head_dim = head_dim;
    c->type = type;
    c->box_rows = page < 64 ? page : 64;
    const size_t floats = (size_t)rows * head_dim / 2;
    c->k_id = zilla_buffer_alloc(floats);
    if (c->k_id > 0) c->v_id = zilla_buffer_alloc(floats);
    int rc = c->k_id > 0 && c->v_id > 0 ? kOk : kBadHandle;
    if (!rc) {
        c->k = ptr(c->k_id);
        c->v = ptr(c->v_id);
        cudaMemsetAsync(c->k, 0, floats * sizeof(float), stream());
        cudaMemsetAsync(c->v, 0, floats * sizeof(float), stream());
        rc = check_cuda(name);
    }
    const uint64_t dims[2] = {(uint64_t)head_dim, (uint64_t)rows}, strides[1] = {(uint64_t)head_dim * 2};
    const uint32_t box[2] = {(uint32_t)(head_dim < 64 ? head_dim : 64), (uint32_t)c->box_rows};
    const auto dtype = type == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const tc::Swizzle sw = head_dim < 64 ? tc::kSw64 : tc::kSw128;
    if (!rc) rc = tc::make_tmap_typed(&c->k_map, dtype, c->k, 2, dims, strides, box, sw);
    if (!rc) rc = tc::make_tmap_typed(&c->v_map, dtype, c->v, 2, dims, strides, box, sw);
    if (rc) {
        if (c->k_id > 0) zilla_buffer_free(c->k_id);
        if (c->v_id > 0) zilla_buffer_free(c->v_id);
        delete c;
        return rc;
    }
    g_caches[g_next_cache] = c;
    return g_next_cache++;
}

int zilla_kv_destroy(int kv) {
    auto it = g_caches.find(kv);
    if (it == g_caches.end()) return fail(kBadHandle, "zilla_kv_destroy: unknown cache %d", kv);
    KvCache *c = it->second;
    if (ptr(c->k_id) == c->k) zilla_buffer_free(c->k_id);
    if (ptr(c->v_id) == c->v) zilla_buffer_free(c->v_id);
    g_caches.erase(it);
    delete c;
    return kOk;
}

int zilla_kv_k_id(int kv) {
    const KvCache *c = kv_get(kv);
    return c ? c->k_id : fail(kBadHandle, "zilla_kv_k_id: unknown cache %d", kv);
}

int zilla_kv_v_id(int kv) {
    const KvCache *c = kv_get(kv);
    return c ? c->v_id : fail(kBadHandle, "zilla_kv_v_id: unknown cache %d", kv);
}

int zilla_kv_append(int kv, int x_type, int q_id, int q_off, int q_ld, int k_id, int k_off, int k_ld, int v_id,
                    int v_off, int v_ld, int qout_id, int start_id, int len_id, int pages_id, int batch, int rows,
                    int q_heads, int max_pages, int prefix_len, int table_id, int rot_dim, int interleaved) {
    const char *name = "zilla_kv_append";
    const KvCache *c = kv_get(kv);
    if (!c) return fail(kBadHandle, "%s: unknown cache %d", name, kv);
    if (x_type != kF32 && x_type != c->type)
        return fail(kBadArg, "%s: the rows are fp32 (0) or the cache's type (%d), not type %d", name, c->type, x_type);
    if (batch < 0 || rows < 0 || q_heads < 0 || q_heads > 65536 || max_pages < 1 || prefix_len < 0)
        return fail(kBadArg, "%s: bad sizes batch=%d rows=%d q_heads=%d max_pages=%d prefix_len=%d", name, batch, rows,
                    q_heads, max_pages, prefix_len);
    const int D = c->head_dim;
    if ((long long)prefix_len + (long long)max_pages * c->page > 0x7fffffffLL)
        return fail(kBadArg, "%s: positions pass 31 bits", name);
    if (rot_dim < 0 || (rot_dim & 1) || rot_dim > D)
        return fail(kBadArg, "%s: rot_dim %d is not an even number up to head_dim", name, rot_dim);
    const long long wq = (long long)q_heads * D, wk = (long long)c->kv_heads * D;
    if (q_off < 0 || k_off < 0 || v_off < 0 || (q_heads && q_off + wq > q_ld) || k_off + wk > k_ld || v_off + wk > v_ld)
        return fail(kBadArg, "%s: the heads do not fit the row strides", name);
    if (q_heads && qout_id == q_id && (q_off || q_ld != wq || x_type != c->type))
        return fail(kBadArg, "%s: q is rotated in place only where its rows have the output's layout and type", name);
    for (int to : {q_heads ? qout_id : 0, c->k_id, c->v_id})
        for (int from : {to == qout_id ? 0 : q_heads ? q_id : 0, k_id, v_id, start_id, len_id, pages_id, rot_dim ? table_id : 0})
            if (to && to == from) return fail(kBadArg, "%s: buffer %d is read and written", name, to);
    if (q_heads && (qout_id == c->k_id || qout_id == c->v_id)) return fail(kBadArg, "%s: q's output is the cache", name);
    const size_t n = rows;
    auto span = [&](long long off, long long ld, long long wide) {
        return rows ? elem_floats((n - 1) * ld + off + wide, x_type) : 0;
    };
    if (int rc = check_buffers(name, {{k_id, span(k_off, k_ld, wk), "k"},
                                      {v_id, span(v_off, v_ld, wk), "v"},
                                      {c->k_id, 0, "the cache"},
                                      {start_id, (size_t)batch + 1, "start"},
                                      {len_id, (size_t)batch, "len"},
                                      {pages_id, (size_t)batch * max_pages, "pages"}}))
        return rc;
    if (q_heads)
        if (int rc = check_buffers(name, {{q_id, span(q_off, q_ld, wq), "q"}, {qout_id, elem_floats(n * wq, c->type), "q_out"}}))
            return rc;
    if (rot_dim)
        if (int rc = check_buffers(name, {{table_id, (size_t)rot_dim + 2, "table"}})) return rc;
    if (!rows || !batch) return kOk;
    const int vec = rope_vector(D, rot_dim, {q_heads ? q_off : 0, q_heads ? q_ld : 0, k_off, k_ld, v_off, v_ld});
    const size_t es = elem_size(x_type);
    AppendParams p;
    p.q = q_heads ? reinterpret_cast<const char *>(ptr(q_id)) + q_off * es : nullptr;
    p.k = reinterpret_cast<const char *>(ptr(k_id)) + k_off * es;
    p.v = reinterpret_cast<const char *>(ptr(v_id)) + v_off * es;
    p.q_out = q_heads ? ptr(qout_id) : nullptr;
    p.k_cache = c->k;
    p.v_cache = c->v;
    p.q_ld = q_ld;
    p.k_ld = k_ld;
    p.v_ld = v_ld;
    p.table = rot_dim ? reinterpret_cast<const double *>(ptr(table_id)) : nullptr;
    p.batch = {reinterpret_cast<const int *>(ptr(start_id)), reinterpret_cast<const int *>(ptr(len_id)),
               reinterpret_cast<const int *>(ptr(pages_id)), batch, rows, max_pages, prefix_len};
    p.q_heads = q_heads;
    p.kv_heads = c->kv_heads;
    p.page_log2 = c->page_log2;
    p.pages = c->pages;
    p.shape = rope_shape(D, rot_dim, interleaved != 0, vec);
    p.err = device_error_word();
    if (!p.err) return fail(kBadHandle, "%s: no device error word", name);
    const int per_row = (q_heads + 2 * c->kv_heads) * p.shape.units;
    // as rope_dev: four units a thread where every SM still gets two blocks
    int tokens = 1;
    while (tokens < kAppendTokens && tokens * per_row < 4 * kAppendThreads && rows / (2 * tokens) >= 2 * sm_count()) tokens *= 2;
    p.tokens = tokens;
    p.per_row = FastDiv(per_row);
    p.per_head = FastDiv(p.shape.units);
    if (c->type == kBf16) {
        if (x_type == kF32) launch_append<float, __nv_bfloat16>(p, vec);
        else launch_append<__nv_bfloat16, __nv_bfloat16>(p, vec);
    } else {
        if (x_type == kF32) launch_append<float, __half>(p, vec);
        else launch_append<__half, __half>(p, vec);
    }
    ZB_LAUNCH_CHECK(name);
    return kOk;
}

}  // extern "C"
