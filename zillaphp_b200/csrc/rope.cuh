// rope.cuh -- rotary positions: the parts that rope_dev and the cache append share.
//
// Pair i of a head at position pos is turned by the angle 2 pi pos f_i and scaled by m:
//   (a, b) -> m (a cos - b sin, a sin + b cos).
// The table holds f_i in turns a position, as fp64, then m: pos * f_i is then one fp64 product
// whose integer part drops out exactly, so an angle is as good at position 2^30 as at 0 (fp32
// angles are off by 6e-8 * pos radians).  The turn's fraction, in [-1/2, 1/2], is rounded to fp32
// (at most 2^-26 turns off) and goes to sincospif.
#pragma once

#include "half_types.cuh"

namespace zb {

struct RopeShape {
    int head_dim, rot, interleaved;
    int pair_units, units;   // rotated units and all units of a head
};

// A head's row is cut into units.  A rotated unit is two vectors with V pairs between them (half layout, and single
// elements) or one vector that holds V / 2 pairs (interleaved), so that a warp's accesses stay contiguous; the
// rest of the head is units of one vector that are copied.
template <int V, bool INTER>
struct RopeForm {
    static constexpr bool kTwo = !INTER || V == 1;
    static constexpr int kPairs = kTwo ? V : V / 2;
    // Units that a thread loads before it finishes one: 128 bytes of 16-byte vectors, which with three blocks of
    // 256 threads keeps 96 KB an SM on the way (HBM's 44 bytes a nanosecond and SM times two microseconds).  A copied unit of
    // the half layout is one vector, so that its thread has 64 bytes on the way: 335 MB of bf16 heads, half of each rotated,
    // take 83 us there and 54 interleaved.
    static constexpr int kBatch = kTwo ? 4 : 8;
};

// Where unit u's vectors lie in a head; y -1: one vector only.
template <int V, bool INTER>
__device__ __forceinline__ int2 rope_places(int u, const RopeShape &r) {
    if (u >= r.pair_units) return make_int2(r.rot + (u - r.pair_units) * V, -1);
    if (INTER) return V > 1 ? make_int2(u * V, -1) : make_int2(2 * u, 2 * u + 1);
    return make_int2(u * V, (r.rot >> 1) + u * V);
}

// One unit's vectors as loaded.  A thread loads several units before it finishes one; a unit is stored after its
// own loads, so dst may be src.
template <typename TI, int V, bool TWO>
struct RopeUnit {
    RawVec<TI, V> a, b;
    __device__ __forceinline__ void load(const TI *src, int2 at) {
        a = load_raw<TI, V>(src + at.x);
        if (TWO && at.y >= 0) b = load_raw<TI, V>(src + at.y);
    }
};

// A thread's unit of every head that it takes: where it lies and its pairs' cosines and sines, which are the same for
// all heads of a row, so they stay in registers.
template <int V, bool INTER>
struct RopeLane {
    using Form = RopeForm<V, INTER>;
    int2 at;
    bool turns;        // a rotated unit (copied otherwise)
    float co[Form::kPairs], si[Form::kPairs];
    __device__ __forceinline__ void place(int u, const RopeShape &r) {
        at = rope_places<V, INTER>(u, r);
        turns = u < r.pair_units;
    }
    __device__ __forceinline__ void angles(int u, int pos, const RopeShape &r, const double *__restrict__ table, float sign) {
        if (!turns) return;
        const float m = (float)table[r.rot >> 1];
#pragma unroll
        for (int e = 0; e < Form::kPairs; ++e) {
            const double t = (double)pos * table[u * Form::kPairs + e];
            float s, c;
            sincospif(2.0f * (float)(t - rint(t)), &s, &c);
            co[e] = m * c;
            si[e] = m * sign * s;
        }
    }
    static __device__ __forceinline__ void turn(float &x, float &y, float c, float s) {
        const float t = x;
        x = t * c - y * s;
        y = t * s + y * c;
    }
    template <typename TI, typename TO>
    __device__ __forceinline__ void finish(const RopeUnit<TI, V, Form::kTwo> &unit, TO *dst, bool rotate) const {
        float x[V], y[V];
        widen<TI, V>(unit.a, x);
        if (Form::kTwo && at.y >= 0) widen<TI, V>(unit.b, y);
        if (rotate && turns) {
#pragma unroll
            for (int e = 0; e < Form::kPairs; ++e) {
                if (Form::kTwo) turn(x[e], y[e], co[e], si[e]);
                else turn(x[2 * e], x[(2 * e + 1) % V], co[e], si[e]);
            }
        }
        store_vec<TO, V>(dst + at.x, x);
        if (Form::kTwo && at.y >= 0) store_vec<TO, V>(dst + at.y, y);
    }
};

// The widest vector (`widest`: 16 bytes of the input's type; or less: 4, 2, 1 elements) that divides a head's halves
// (interleaved: its rotated part), its copied rest and every offset and row stride of the call.
inline int rope_vector(int widest, int head_dim, int rot, int interleaved, std::initializer_list<long long> also) {
    long long all = (long long)head_dim | (interleaved ? rot : rot / 2);
    for (long long a : also) all |= a;
    for (int v = widest; v > 1; v /= 2)
        if (all % v == 0) return v;
    return 1;
}

inline RopeShape rope_shape(int head_dim, int rot, int interleaved, int vec) {
    RopeShape r;
    r.head_dim = head_dim;
    r.rot = rot;
    r.interleaved = interleaved;
    r.pair_units = rot / 2 / (interleaved && vec > 1 ? vec / 2 : vec);
    r.units = r.pair_units + (head_dim - rot) / vec;
    return r;
}

constexpr int kRopeMaxDim = 256;
constexpr int kRopeThreads = 256;
constexpr int kRopeBlocks = 3;       // blocks an SM at least (80 registers a thread)

// How threads share the work: a thread takes one unit of a row for heads h, h + lanes * splits, ...  A block is
// rows x lanes x units (units fastest, so a warp reads along a head).  Heads are spread over as many threads as it
// takes to fill the machine twice (two times 1024 threads an SM), and no more: each thread works out its pairs' angles.
struct RopeGrid {
    int rows, lanes, splits, threads;
};
inline RopeGrid rope_grid(long long rows, int heads, int units) {
    RopeGrid g;
    const long long want = 2048LL * sm_count(), have = rows * units;
    long long spread = (want + have - 1) / have;
    if (spread > heads) spread = heads;
    const int room = kRopeThreads / units;   // units are 256 at most
    g.lanes = (int)(spread < room ? spread : room);
    g.splits = (int)((spread + g.lanes - 1) / g.lanes);
    g.rows = room / g.lanes;
    if (g.rows > rows) g.rows = (int)rows;
    g.threads = (g.rows * g.lanes * units + 31) / 32 * 32;
    return g;
}

}  // namespace zb
