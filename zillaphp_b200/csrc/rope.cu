// rope.cu -- rotary positions: the table of frequencies and the rotation of
// rows of heads, forward and backward (rope_table_dev, rope_dev).
#include <math.h>

#include "rope.cuh"

namespace zb {
namespace {

// One thread a pair.  Scaling:
//   0  f_i = base^(-2i/rot) / 2 pi
//   1  positions divided by factor (linear interpolation)
//   2  base * factor^(rot / (rot - 2)): the slowest pair is stretched by factor, the fastest kept
//   3  by parts (Peng et al., "YaRN: Efficient Context Window Extension of Large Language Models",
//      section 3.2): a pair that turns more than `fast` times in the original length keeps f_i, one
//      that turns less than `slow` times takes f_i / factor, linear between; m = 0.1 ln factor + 1.
__global__ void rope_table_kernel(double *table, int half_rot, double base, int scaling, double factor,
                                  double original, double slow, double fast) {
    griddep_launch();
    griddep_wait();
    const int i = threadIdx.x, rot = 2 * half_rot;
    if (scaling == 2 && rot > 2) base *= pow(factor, (double)rot / (rot - 2));
    if (i < half_rot) {
        double f = pow(base, -2.0 * i / rot) / 6.283185307179586476925286766559;
        if (scaling == 1) f /= factor;
        if (scaling == 3) {
            const double keep = fmin(1.0, fmax(0.0, (f * original - slow) / (fast - slow)));
            f = f * keep + f / factor * (1.0 - keep);
        }
        table[i] = f;
    }
    if (i == 0) table[half_rot] = scaling == 3 ? 0.1 * log(factor) + 1.0 : 1.0;
}

struct RopeParams {
    const void *x;
    void *y;
    const int *pos;
    const double *table;
    long long x_ld, y_ld;
    int rows, heads;
    RopeShape shape;
    RopeGrid grid;
    float sign;
};

// Bound by HBM: each element is read and written once, by whole warps along a head.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kRopeBlocks) rope_kernel(const RopeParams p) {
    griddep_launch();
    griddep_wait();
    const int u = threadIdx.x % p.shape.units, rest = threadIdx.x / p.shape.units, lane = rest % p.grid.lanes;
    const long long row = (long long)blockIdx.x * p.grid.rows + rest / p.grid.lanes;
    if (rest >= p.grid.rows * p.grid.lanes || row >= p.rows) return;
    const int step = p.grid.lanes * p.grid.splits, D = p.shape.head_dim;
    using Form = RopeForm<V, INTER>;
    RopeLane<V, INTER> lane_of;
    lane_of.place(u, p.shape);
    const T *x = static_cast<const T *>(p.x) + row * p.x_ld;
    T *y = static_cast<T *>(p.y) + row * p.y_ld;
    const int pos = p.pos[row];
    RopeUnit<T, V, Form::kTwo> unit[Form::kBatch];
    auto load = [&](int h0) {
#pragma unroll
        for (int i = 0; i < Form::kBatch; ++i)
            if (h0 + i * step < p.heads) unit[i].load(x + (h0 + i * step) * D, lane_of.at);
    };
    int h0 = blockIdx.y * p.grid.lanes + lane;
    load(h0);   // under way while the angles are worked out
    lane_of.angles(u, pos, p.shape, p.table, p.sign);
    while (h0 < p.heads) {
#pragma unroll
        for (int i = 0; i < Form::kBatch; ++i)
            if (h0 + i * step < p.heads) lane_of.finish(unit[i], y + (h0 + i * step) * D, true);
        h0 += Form::kBatch * step;
        load(h0);
    }
}

template <typename T, bool INTER>
void launch_rope(const RopeParams &p, int vec) {
    const dim3 grid((unsigned)((p.rows + (long long)p.grid.rows - 1) / p.grid.rows), p.grid.splits), block(p.grid.threads);
    if constexpr (sizeof(T) == 2)
        if (vec == 8) {
            launch_pdl(rope_kernel<T, 8, INTER>, grid, block, 0, p);
            return;
        }
    if (vec == 4) launch_pdl(rope_kernel<T, 4, INTER>, grid, block, 0, p);
    else if (vec == 2) launch_pdl(rope_kernel<T, 2, INTER>, grid, block, 0, p);
    else launch_pdl(rope_kernel<T, 1, INTER>, grid, block, 0, p);
}

}  // namespace
}  // namespace zb

using namespace zb;

extern "C" {

int rope_table_dev(int table_id, int rot_dim, float base, int scaling, float factor, int original, float slow,
                   float fast) {
    const char *name = "rope_table_dev";
    if (rot_dim < 2 || rot_dim > kRopeMaxDim || (rot_dim & 1))
        return fail(kBadArg, "%s: rot_dim %d is not an even number from 2 to %d", name, rot_dim, kRopeMaxDim);
    if (!(base > 0.0f) || isinf(base)) return fail(kBadArg, "%s: base must be positive", name);
    if (scaling < 0 || scaling > 3) return fail(kBadArg, "%s: unknown scaling %d", name, scaling);
    if (scaling && (!(factor > 0.0f) || isinf(factor))) return fail(kBadArg, "%s: factor must be positive", name);
    if (scaling == 3 && (original < 1 || !(fast > slow) || isinf(fast) || isinf(slow)))
        return fail(kBadArg, "%s: scaling by parts needs original >= 1 and fast > slow", name);
    if (int rc = check_buffers(name, {{table_id, (size_t)rot_dim + 2, "table"}})) return rc;
    launch_pdl(rope_table_kernel, dim3(1), dim3(kRopeMaxDim / 2), 0, reinterpret_cast<double *>(ptr(table_id)),
               rot_dim / 2, (double)base, scaling, (double)factor, (double)original, (double)slow, (double)fast);
    ZB_LAUNCH_CHECK(name);
    return kOk;
}

int rope_dev(int x_id, int x_off, int x_ld, int y_id, int y_off, int y_ld, int pos_id, int table_id, int type,
             int rows, int heads, int head_dim, int rot_dim, int interleaved, int inverse) {
    const char *name = "rope_dev";
    if (type < kF32 || type > kF16) return fail(kBadArg, "%s: unknown element type %d", name, type);
    if (rows < 0 || heads < 1 || head_dim < 2 || head_dim > kRopeMaxDim)
        return fail(kBadArg, "%s: bad sizes rows=%d heads=%d head_dim=%d (at most %d)", name, rows, heads, head_dim,
                    kRopeMaxDim);
    if (rot_dim < 2 || (rot_dim & 1) || rot_dim > head_dim)
        return fail(kBadArg, "%s: rot_dim %d is not an even number from 2 to head_dim", name, rot_dim);
    if ((interleaved != 0 && interleaved != 1) || (inverse != 0 && inverse != 1))
        return fail(kBadArg, "%s: interleaved and inverse are 0 or 1", name);
    const long long wide = (long long)heads * head_dim;
    if (wide > (1 << 24)) return fail(kBadArg, "%s: rows of %lld elements are too wide", name, wide);
    if (x_off < 0 || y_off < 0 || x_off + wide > x_ld || y_off + wide > y_ld)
        return fail(kBadArg, "%s: heads * head_dim = %lld elements do not fit the row strides", name, wide);
    if (x_id == y_id && (x_off != y_off || x_ld != y_ld) &&
        (x_ld != y_ld || (x_off < y_off + wide && y_off < x_off + wide)))
        return fail(kBadArg, "%s: x and y overlap in one buffer without being the same rows", name);
    if (table_id == y_id || pos_id == y_id) return fail(kBadArg, "%s: y is also the table or the positions", name);
    const size_t n = rows;
    if (int rc = check_buffers(name, {{x_id, rows ? elem_floats((n - 1) * x_ld + x_off + wide, type) : 0, "x"},
                                      {y_id, rows ? elem_floats((n - 1) * y_ld + y_off + wide, type) : 0, "y"},
                                      {pos_id, n, "positions"},
                                      {table_id, (size_t)rot_dim + 2, "table"}}))
        return rc;
    if (!rows) return kOk;
    const int vec = rope_vector(type == kF32 ? 4 : 8, head_dim, rot_dim, interleaved, {x_off, y_off, x_ld, y_ld});
    RopeParams p;
    p.x = reinterpret_cast<const char *>(ptr(x_id)) + (size_t)x_off * elem_size(type);
    p.y = reinterpret_cast<char *>(ptr(y_id)) + (size_t)y_off * elem_size(type);
    p.pos = reinterpret_cast<const int *>(ptr(pos_id));
    p.table = reinterpret_cast<const double *>(ptr(table_id));
    p.x_ld = x_ld;
    p.y_ld = y_ld;
    p.rows = rows;
    p.shape = rope_shape(head_dim, rot_dim, interleaved != 0, vec);
    p.heads = heads;
    p.grid = rope_grid(rows, heads, p.shape.units);
    p.sign = inverse ? -1.0f : 1.0f;
    auto launch = [&](auto kind) {
        using T = decltype(kind);
        if (interleaved) launch_rope<T, true>(p, vec);
        else launch_rope<T, false>(p, vec);
    };
    if (type == kF32) launch(float());
    else if (type == kBf16) launch(__nv_bfloat16());
    else launch(__half());
    ZB_LAUNCH_CHECK(name);
    return kOk;
}

}  // extern "C"
