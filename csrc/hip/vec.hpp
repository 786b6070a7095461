// Element types and vector access shared by the transformer kernels.
//
// A kernel holds f32 values; ld8/st8 move eight elements of a row at once
// (16 B for the 16-bit types, 2 x 16 B for f32) and round to nearest even
// on the way out.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace kfv {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr int WAVE = 64;

template <typename T>
struct vec8;
template <>
struct vec8<__bf16> {
    typedef bf16x8 type;
};
template <>
struct vec8<_Float16> {
    typedef f16x8 type;
};
template <>
struct vec8<float> {  // loaded as two pieces of 16 bytes
    typedef __attribute__((ext_vector_type(8), aligned(16))) float type;
};

template <typename T>
__device__ inline void ld8(float *f, const T *p)
{
    const typename vec8<T>::type v = *(const typename vec8<T>::type *)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
}
template <>
__device__ inline void ld8<float>(float *f, const float *p)
{
    const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = a[i];
        f[4 + i] = b[i];
    }
}

template <typename T>
__device__ inline void st8(T *p, const float *f)
{
    typename vec8<T>::type v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)f[i];
    *(typename vec8<T>::type *)p = v;
}
template <>
__device__ inline void st8<float>(float *p, const float *f)
{
    f32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = f[i];
        b[i] = f[4 + i];
    }
    *(f32x4 *)p = a;
    *(f32x4 *)(p + 4) = b;
}

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace kfv
