// cafe_dense.h -- what the dense-side kernels (cafe_linear.hip, cafe_interact.hip, cafe_adamw.hip) share: element
// types, 16-byte accesses at any element alignment, the 16 x 16 product, the order of tiles over the XCDs.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cafe_internal.h"

namespace cafe {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// A row of an odd number of 16-bit elements starts at any even address.  Global memory takes 16-byte accesses at any
// address; the type only tells the compiler not to assume more.
template <int A> struct __attribute__((packed, aligned(A))) Chunk { u32x4 v; };

template <class T> struct Elem {
    static constexpr int per_chunk = 16 / (int)sizeof(T);
};

template <class T> __device__ __forceinline__ u32x4 load16(const T *p) { return ((const Chunk<sizeof(T)> *)p)->v; }
template <class T> __device__ __forceinline__ void store16(T *p, u32x4 v) { ((Chunk<sizeof(T)> *)p)->v = v; }

// chunk moved down by `n` elements, zeros behind (n up to the chunk's length: all zeros); selects, no branches
template <class T> __device__ __forceinline__ u32x4 shift_down(u32x4 v, int n) {
    const int bits = n * 8 * (int)sizeof(T), s = bits & 63;
    const uint64_t lo = (uint64_t)v.x | ((uint64_t)v.y << 32), hi = (uint64_t)v.z | ((uint64_t)v.w << 32);
    uint64_t a = bits & 64 ? hi : lo, b = bits & 64 ? 0 : hi;
    a = bits & 128 ? 0 : a;
    b = bits & 128 ? 0 : b;
    a = (a >> s) | ((b << 1) << (63 - s));
    b >>= s;
    return u32x4{(uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32)};
}

// the first `n` elements at p (n may be <= 0 or exceed the chunk), zeros behind; nothing past them is read
template <class T> __device__ __forceinline__ u32x4 load_some(const T *p, int n) {
    union { u32x4 v; T e[Elem<T>::per_chunk]; } u;
    u.v = u32x4{0, 0, 0, 0};
    if (n >= Elem<T>::per_chunk) return load16(p);
#pragma unroll
    for (int i = 0; i < Elem<T>::per_chunk; i++)
        if (i < n) u.e[i] = p[i];
    return u.v;
}
template <class T> __device__ __forceinline__ void store_some(T *p, u32x4 v, int n) {
    if (n >= Elem<T>::per_chunk) { store16(p, v); return; }
    union { u32x4 v; T e[Elem<T>::per_chunk]; } u;
    u.v = v;
#pragma unroll
    for (int i = 0; i < Elem<T>::per_chunk; i++)
        if (i < n) p[i] = u.e[i];
}

// a chunk as floats and back (round to nearest even)
template <class T> __device__ __forceinline__ void unpack(u32x4 v, float *f) {
    union { u32x4 v; T e[Elem<T>::per_chunk]; } u;
    u.v = v;
#pragma unroll
    for (int i = 0; i < Elem<T>::per_chunk; i++) f[i] = (float)u.e[i];
}
template <class T> __device__ __forceinline__ u32x4 pack(const float *f) {
    union { u32x4 v; T e[Elem<T>::per_chunk]; } u;
#pragma unroll
    for (int i = 0; i < Elem<T>::per_chunk; i++) u.e[i] = (T)f[i];
    return u.v;
}

// 16 x 16 product of one 16-byte chunk per lane on either side: lane l holds row l % 16, chunk l / 16 of four.
// Accumulator element e of lane l: row 4 (l / 16) + e of the first, row l % 16 of the second operand.
template <class T> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma16<__bf16>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<_Float16>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<float>(u32x4 a, u32x4 b, f32x4 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int q = 0; q < 4; q++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[q], y[q], c, 0, 0, 0);
    return c;
}

// Workgroups are handed to the eight XCDs in turn; each XCD has its own L2.  Renumbered so that one XCD works on a
// contiguous run of tiles (neighbours share operand rows).  A permutation of 0 .. n-1 for every n.
__device__ __forceinline__ int xcd_tile(int id, int n) {
    const int x = id & 7, q = n >> 3, r = n & 7;
    return x * q + (x < r ? x : r) + (id >> 3);
}

constexpr int kF32 = 0, kBF16 = 1, kF16 = 2;

}  // namespace cafe
