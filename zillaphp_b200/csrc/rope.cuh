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
    int pair_units, units;   // rotated units and all units of a head: a rotated one is two vectors, a copied one is one
};

// Shared-memory (cos, sin) of `tokens` tokens' pairs: cs[token * rot/2 + pair].  pos[token] comes from
// shared memory; sign -1 turns back.
__device__ __forceinline__ void rope_angles(float2 *cs, const int *pos, int tokens, int half_rot,
                                            const double *__restrict__ table, float sign, int tid, int threads) {
    const float m = (float)table[half_rot];
    for (int k = tid; k < tokens * half_rot; k += threads) {
        const int t = k / half_rot, i = k - t * half_rot;
        const double turns = (double)pos[t] * table[i];
        const float f = (float)(turns - rint(turns));
        float s, c;
        sincospif(2.0f * f, &s, &c);
        cs[k] = make_float2(m * c, m * sign * s);
    }
}

// One unit of a head: u < pair_units turns V pairs, the rest copy V elements.  Everything is loaded
// before anything is stored, so dst may be src.
template <typename TI, typename TO, int V>
__device__ __forceinline__ void rope_unit(const TI *src, TO *dst, const float2 *cs, int u, const RopeShape &r) {
    if (u < r.pair_units) {
        const int a_at = r.interleaved ? 2 * u * V : u * V, b_at = r.interleaved ? a_at + V : (r.rot >> 1) + u * V;
        float a[V], b[V], x[V], y[V];
        load_vec<TI, V>(src + a_at, a);
        load_vec<TI, V>(src + b_at, b);
        const float2 *c = cs + u * V;   // the unit's pairs are u V .. u V + V - 1 in both layouts
        if (r.interleaved && V > 1) {
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                const float2 p = c[e], q = c[V / 2 + e];
                x[2 * e] = a[2 * e] * p.x - a[2 * e + 1] * p.y;
                x[2 * e + 1] = a[2 * e] * p.y + a[2 * e + 1] * p.x;
                y[2 * e] = b[2 * e] * q.x - b[2 * e + 1] * q.y;
                y[2 * e + 1] = b[2 * e] * q.y + b[2 * e + 1] * q.x;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 p = c[e];
                x[e] = a[e] * p.x - b[e] * p.y;
                y[e] = a[e] * p.y + b[e] * p.x;
            }
        }
        store_vec<TO, V>(dst + a_at, x);
        store_vec<TO, V>(dst + b_at, y);
    } else {
        const int at = r.rot + (u - r.pair_units) * V;
        float a[V];
        load_vec<TI, V>(src + at, a);
        store_vec<TO, V>(dst + at, a);
    }
}

// The widest vector (8, 4, 2 or 1 elements) that divides a head's halves, its copied rest and every
// offset and row stride of the call: 8 moves 16 bytes of a 16-bit type in one access.
inline int rope_vector(int head_dim, int rot, std::initializer_list<long long> also) {
    long long all = (long long)head_dim | (rot / 2);
    for (long long a : also) all |= a;
    return all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
}

inline RopeShape rope_shape(int head_dim, int rot, int interleaved, int vec) {
    RopeShape r;
    r.head_dim = head_dim;
    r.rot = rot;
    r.interleaved = interleaved;
    r.pair_units = rot / 2 / vec;
    r.units = r.pair_units + (head_dim - rot) / vec;
    return r;
}

constexpr int kRopeMaxDim = 256;

}  // namespace zb
