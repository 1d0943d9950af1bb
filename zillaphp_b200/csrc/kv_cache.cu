// kv_cache.cu -- the paged K/V cache: creation, and appending a batch's new
// keys and values with the rotary rotation applied on the way.
#include <map>
#include <new>

#include "kv_cache.cuh"
#include "rope.cuh"

namespace zb {
namespace {

std::map<int, KvCache *> g_caches;
int g_next_cache = 1;

constexpr int kCheckBatch = 1024;

struct AppendParams {
    const void *q, *k, *v;
    void *q_out, *k_cache, *v_cache;
    long long q_ld, k_ld, v_ld;
    const double *table;   // nullptr: no rotation
    KvBatch batch;
    int q_heads, kv_heads, page_log2, pages;
    RopeShape shape;
    RopeGrid grid;   // over the q, k and v heads together
    unsigned row_blocks;   // blocks along x that take rows; the ones behind them check kCheckBatch sequences each
    int *err;
};

// Bound by HBM for prompts (each element read and written once) and by latency for single tokens.  Where a
// row comes from does not depend on its sequence, so a thread's first loads are under way while the block finds its
// rows' sequences (a look at every start) and slots.
template <typename TI, typename TO, int V, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kRopeBlocks) kv_append_kernel(const AppendParams p) {
    __shared__ int owner[kRopeThreads], range[2];
    griddep_launch();
    griddep_wait();
    // Blocks that only check: a sequence outside the call's rows may be seen by none that takes rows.  Checked by those, in
    // their look at the starts, it costs 2% of a prompt's time; so, one more block, 0.1 us of a call.
    if (blockIdx.x >= p.row_blocks) {
        const int b0 = (blockIdx.x - p.row_blocks) * kCheckBatch, b1 = b0 + min(kCheckBatch, p.batch.batch - b0);
        for (int b = b0 + threadIdx.x; b < b1 && blockIdx.y == 0; b += blockDim.x)
            if (!kv_rows_fit(p.batch, p.batch.start[b], p.batch.start[b + 1])) atomicCAS(p.err, 0, kErrKvLength);
        return;
    }
    const int u = threadIdx.x % p.shape.units, rest = threadIdx.x / p.shape.units, lane = rest % p.grid.lanes;
    const int in_block = rest / p.grid.lanes, row0 = blockIdx.x * p.grid.rows, n = min(p.grid.rows, p.batch.rows - row0);
    const bool works = in_block < n;
    const size_t row = row0 + (works ? in_block : 0);
    const int step = p.grid.lanes * p.grid.splits, D = p.shape.head_dim, heads = works ? p.q_heads + 2 * p.kv_heads : 0;
    using Form = RopeForm<V, INTER>;
    RopeLane<V, INTER> lane_of;
    lane_of.place(u, p.shape);
    RopeUnit<TI, V, Form::kTwo> unit[Form::kBatch];
    const TI *q = static_cast<const TI *>(p.q) + row * p.q_ld, *k = static_cast<const TI *>(p.k) + row * p.k_ld - p.q_heads * D,
             *v = static_cast<const TI *>(p.v) + row * p.v_ld - (p.q_heads + p.kv_heads) * D;
    auto load = [&](int h0) {
#pragma unroll
        for (int i = 0; i < Form::kBatch; ++i) {
            const int h = h0 + i * step;
            if (h < heads) unit[i].load((h < p.q_heads ? q : h < p.q_heads + p.kv_heads ? k : v) + h * D, lane_of.at);
        }
    };
    int h0 = blockIdx.y * p.grid.lanes + lane;
    load(h0);
    kv_owners(owner, range, p.batch, row0, n, threadIdx.x, blockDim.x);
    const int b = works ? owner[in_block] : -1;
    if (b < 0) return;
    const int first = p.batch.start[b], own = p.batch.len[b] - (p.batch.start[b + 1] - first) + ((int)row - first), at = own >> p.page_log2;
    if (own < 0 || at >= p.batch.max_pages) {
        atomicCAS(p.err, 0, own < 0 ? kErrKvLength : kErrKvPage);
        return;
    }
    const int id = p.batch.pages[(size_t)b * p.batch.max_pages + at];
    if (p.shape.rot) lane_of.angles(u, p.batch.prefix_len + own, p.shape, p.table, 1.0f);
    if (id < 0 || id >= p.pages) {
        atomicCAS(p.err, 0, kErrKvPage);
        return;
    }
    TO *q_out = static_cast<TO *>(p.q_out) + row * p.q_heads * D;
    const size_t slot = (((size_t)id * p.kv_heads) << p.page_log2) + (own & ((1 << p.page_log2) - 1));
    while (h0 < heads) {
#pragma unroll
        for (int i = 0; i < Form::kBatch; ++i) {
            int h = h0 + i * step;
            if (h >= heads) continue;
            TO *dst = q_out + h * D;
            h -= p.q_heads;
            const bool is_v = h >= p.kv_heads;   // values are copied
            if (h >= 0) dst = static_cast<TO *>(is_v ? p.v_cache : p.k_cache) + (slot + ((size_t)(is_v ? h - p.kv_heads : h) << p.page_log2)) * D;
            lane_of.finish(unit[i], dst, !is_v);
        }
        h0 += Form::kBatch * step;
        load(h0);
    }
}

template <typename TI, typename TO, bool INTER>
void launch_append(const AppendParams &p, int vec) {
    const dim3 grid(p.row_blocks + (p.batch.batch - 1) / kCheckBatch + 1, p.grid.splits), block(p.grid.threads);
    if constexpr (sizeof(TI) == 2)
        if (vec == 8) {
            launch_pdl(kv_append_kernel<TI, TO, 8, INTER>, grid, block, 0, p);
            return;
        }
    if (vec == 4) launch_pdl(kv_append_kernel<TI, TO, 4, INTER>, grid, block, 0, p);
    else if (vec == 2) launch_pdl(kv_append_kernel<TI, TO, 2, INTER>, grid, block, 0, p);
    else launch_pdl(kv_append_kernel<TI, TO, 1, INTER>, grid, block, 0, p);
}

}  // namespace

const KvCache *kv_get(int id) {
    auto it = g_caches.find(id);
    if (it == g_caches.end()) return nullptr;
    const KvCache *c = it->second;
    return allocation(c->k_id) == c->k_made && allocation(c->v_id) == c->v_made ? c : nullptr;
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
    KvCache *c = new (std::nothrow) KvCache();
    if (!c) return fail(kBadHandle, "%s: out of host memory", name);
    c->pages = pages;
    c->page = page;
    while ((1 << c->page_log2) < page) ++c->page_log2;
    c->kv_heads = kv_heads;
    c->head_dim = head_dim;
    c->type = type;
    c->box_rows = page < 64 ? page : 64;
    const size_t floats = c->floats = (size_t)rows * head_dim / 2;
    c->k_id = zilla_buffer_alloc(floats);
    if (c->k_id > 0) c->v_id = zilla_buffer_alloc(floats);
    int rc = c->k_id > 0 && c->v_id > 0 ? kOk : kBadHandle;
    if (!rc) {
        c->k = ptr(c->k_id);
        c->v = ptr(c->v_id);
        c->k_made = allocation(c->k_id);
        c->v_made = allocation(c->v_id);
        cudaMemsetAsync(c->k, 0, floats * sizeof(float), stream());
        cudaMemsetAsync(c->v, 0, floats * sizeof(float), stream());
        cudaStreamSynchronize(stream());   // zero before work on any other stream
        rc = check_cuda(name);
    }
    const uint64_t dims[2] = {(uint64_t)head_dim, (uint64_t)rows}, strides[1] = {(uint64_t)head_dim * 2};
    const uint32_t box[2] = {(uint32_t)(head_dim < 64 ? head_dim : 64), (uint32_t)c->box_rows};
    const auto dtype = type == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const tc::Swizzle sw = head_dim < 64 ? tc::kSw64 : tc::kSw128;
    if (!rc) rc = tc::make_tmap_typed(&c->k_map, dtype, c->k, 2, dims, strides, box, sw);
    if (!rc) rc = tc::make_tmap_typed(&c->v_map, dtype, c->v, 2, dims, strides, box, sw);
    if (!rc) {
        try {
            g_caches[g_next_cache] = c;
            return g_next_cache++;
        } catch (...) {   // nothing is thrown through the C entry
            rc = fail(kBadHandle, "%s: out of host memory", name);
        }
    }
    if (c->k_id > 0) zilla_buffer_free(c->k_id);
    if (c->v_id > 0) zilla_buffer_free(c->v_id);
    delete c;
    return rc;
}

int zilla_kv_destroy(int kv) {
    auto it = g_caches.find(kv);
    if (it == g_caches.end()) return fail(kBadHandle, "zilla_kv_destroy: unknown cache %d", kv);
    KvCache *c = it->second;
    if (allocation(c->k_id) == c->k_made) zilla_buffer_free(c->k_id);
    if (allocation(c->v_id) == c->v_made) zilla_buffer_free(c->v_id);
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
    if (interleaved != 0 && interleaved != 1) return fail(kBadArg, "%s: interleaved is 0 or 1", name);
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
                                      {c->k_id, c->floats, "the cache"},
                                      {c->v_id, c->floats, "the cache"},
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
    const int vec = rope_vector(x_type == kF32 ? 4 : 8, D, rot_dim, interleaved, {q_heads ? q_off : 0, q_heads ? q_ld : 0, k_off, k_ld, v_off, v_ld});
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
    p.grid = rope_grid(rows, q_heads + 2 * c->kv_heads, p.shape.units);
    p.row_blocks = (unsigned)((rows + (long long)p.grid.rows - 1) / p.grid.rows);
    auto launch = [&](auto in, auto out) {
        if (interleaved) launch_append<decltype(in), decltype(out), true>(p, vec);
        else launch_append<decltype(in), decltype(out), false>(p, vec);
    };
    if (c->type == kBf16) {
        if (x_type == kF32) launch(float(), __nv_bfloat16());
        else launch(__nv_bfloat16(), __nv_bfloat16());
    } else {
        if (x_type == kF32) launch(float(), __half());
        else launch(__half(), __half());
    }
    ZB_LAUNCH_CHECK(name);
    return kOk;
}

}  // extern "C"
