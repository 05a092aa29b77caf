// Device-side pieces shared by the layer operators: element types, vector
// loads at element alignment, reductions over the lanes of a wave.
#pragma once

#include "hx_device.hpp"

namespace hx {

typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int32_t i32x4v __attribute__((ext_vector_type(4)));

// 16 bytes at the alignment of the elements: global memory takes a dwordx4
// at any byte address, so rows of odd width keep whole vectors.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> struct Pack16;
template <> struct Pack16<float> { static constexpr int N = 4; };
template <> struct Pack16<bf16> { static constexpr int N = 8; };

__device__ __forceinline__ u32x4 load_raw(const float *p) { return *(const u32x4_a4 *)p; }
__device__ __forceinline__ u32x4 load_raw(const bf16 *p) { return *(const u32x4_a2 *)p; }
// 16 bytes of a row of `width` elements from element c on, zeros past its end, in
// two steps, so that nothing waits for them before all loads are under way: the
// last, partial vector is loaded as the sixteen bytes that end the row, and
// shifted when it is used.  Element by element it would cost a wait each.
template <typename T> __device__ __forceinline__ u32x4 load_part(const T *row, uint32_t c, uint32_t width) {
    constexpr uint32_t N = Pack16<T>::N;
    u32x4 v = {0, 0, 0, 0};
    if (width >= N) {
        if (c < width) v = load_raw(row + min(c, width - N));
    } else if (c == 0) {
        T part[N];
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) part[i] = i < width ? row[i] : (T)0.0f;
        __builtin_memcpy(&v, part, 16);
    }
    return v;
}
template <typename T> __device__ __forceinline__ u32x4 place_part(u32x4 v, uint32_t c, uint32_t width) {
    constexpr uint32_t N = Pack16<T>::N;
    if (width < N || c >= width || c + N <= width) return v;
    return __builtin_bit_cast(u32x4, __builtin_bit_cast(unsigned __int128, v) >> (8 * sizeof(T) * (c + N - width)));
}
// f32 values of 16 bytes of elements.
template <typename T, int N> __device__ __forceinline__ void unpack(u32x4 v, float (&x)[N]) {
    static_assert(N == Pack16<T>::N);
    if constexpr (sizeof(T) == 4) {
        const f32x4 f = __builtin_bit_cast(f32x4, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = f[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t two = v[i];
            x[2 * i] = __builtin_bit_cast(float, two << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, two & 0xFFFF0000u);
        }
    }
}
__device__ __forceinline__ void store_pack(float *p, const float (&x)[4]) {
    *(f32x4_a4 *)p = f32x4{x[0], x[1], x[2], x[3]};
}
// Rounded to bf16, halfway cases to even.
__device__ __forceinline__ void store_pack(bf16 *p, const float (&x)[8]) {
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (bf16)x[i];
    *(u32x4_a2 *)p = __builtin_bit_cast(u32x4, r);
}

} // namespace hx
