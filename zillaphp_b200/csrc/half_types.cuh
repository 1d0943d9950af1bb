// half_types.cuh -- element types of the generation operators (fp32, bf16,
// fp16) and vector loads and stores that widen to and round from fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace zb {

// Type codes of the C-ABI.
enum ElemType : int { kF32 = 0, kBf16 = 1, kF16 = 2 };

inline size_t elem_size(int type) { return type == kF32 ? 4 : 2; }
// Registry floats that hold n elements of the type.
inline size_t elem_floats(size_t n, int type) { return type == kF32 ? n : (n + 1) / 2; }

// Two fp32 values rounded to the nearest 16-bit value and packed, a in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (__is_same(T, __half)) return __half2float(v);
    else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (__is_same(T, __half)) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

// V elements of T as they lie in memory, loaded in accesses of 16 bytes at most (p aligned to V elements, 16
// bytes suffice): kept like this while more loads are in flight, a 16-bit vector takes half of fp32's registers.
template <typename T, int V>
struct RawVec {
    static constexpr int kWords = V * (int)sizeof(T) / 4;   // 0: one 16-bit element
    uint32_t w[kWords > 0 ? kWords : 1];
};

template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> load_raw(const T *p) {
    RawVec<T, V> r;
    constexpr int N = RawVec<T, V>::kWords;
    if constexpr (N == 0) {
        r.w[0] = *reinterpret_cast<const uint16_t *>(p);
    } else if constexpr (N == 1) {
        r.w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else if constexpr (N == 2) {
        const uint2 a = *reinterpret_cast<const uint2 *>(p);
        r.w[0] = a.x; r.w[1] = a.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 a = reinterpret_cast<const uint4 *>(p)[i];
            r.w[4 * i] = a.x; r.w[4 * i + 1] = a.y; r.w[4 * i + 2] = a.z; r.w[4 * i + 3] = a.w;
        }
    }
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void widen(const RawVec<T, V> &r, float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = __uint_as_float(r.w[i]);
    } else if constexpr (V == 1) {
        v[0] = unpack2<T>(r.w[0]).x;
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 f = unpack2<T>(r.w[i]);
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
}

// V elements of T at p as fp32.
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T *p, float (&v)[V]) {
    widen<T, V>(load_raw<T, V>(p), v);
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[V]) {
    if constexpr (V == 1) {
        *p = from_f32<T>(v[0]);
    } else if constexpr (sizeof(T) == 4) {
        if constexpr (V == 2) {
            *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
        } else {
#pragma unroll
            for (int i = 0; i < V / 4; ++i)
                reinterpret_cast<float4 *>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
    } else {
        uint32_t w[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
        if constexpr (V == 2) *reinterpret_cast<uint32_t *>(p) = w[0];
        else if constexpr (V == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

}  // namespace zb
