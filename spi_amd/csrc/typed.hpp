// Typed values and 16-byte chunks of rows, shared by the row operators (norm.hip, linear.hip).
#pragma once
#include "common.hpp"

#ifdef __HIPCC__
typedef _Float16 half_t;
typedef __bf16 bf16_t;
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_acc __attribute__((ext_vector_type(16)));
typedef int i32x16_acc __attribute__((ext_vector_type(16)));

template <typename T> struct Chunk {                            // 16 bytes of a row: 4 floats, 8 halves, 16 bytes
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};

// `n` valid values at p (any alignment of T), the others 0.  A whole chunk is one 16-byte load: gfx950 takes it at the alignment of T.
template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* __restrict__ p, int n) {
    Chunk<T> c;
    if (n >= Chunk<T>::N) { __builtin_memcpy(&c, p, 16); return c; }
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; ++i) c.v[i] = i < n ? p[i] : (T)0;
    return c;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* __restrict__ p, const Chunk<T>& c, int n) {
    if (n >= Chunk<T>::N) { __builtin_memcpy(p, &c, 16); return; }
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; ++i) if (i < n) p[i] = c.v[i];
}
// N values of a row vector whose type is known at run time only (a wave-uniform branch), widened to fp32
template <int N>
__device__ __forceinline__ void load_f32(const void* base, int dtype, int64_t at, int n, float (&out)[N]) {
    if (dtype == SPI_DTYPE_F32) {
        const float* p = (const float*)base + at;
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const Chunk<float> c = load_chunk(p + i, n - i);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[i + j] = c.v[j];
        }
        return;
    }
    const uint16_t* p = (const uint16_t*)base + at;
    uint16_t v[N];
    if (n >= N) __builtin_memcpy(v, p, 2 * N);
    else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? p[i] : (uint16_t)0;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = dtype == SPI_DTYPE_F16 ? (float)__builtin_bit_cast(half_t, v[i]) : __builtin_bit_cast(float, (uint32_t)v[i] << 16);
}
__device__ __forceinline__ void store_f32(void* base, int dtype, int64_t at, float v) {          // one rounding, to nearest even
    if (dtype == SPI_DTYPE_F32) ((float*)base)[at] = v;
    else if (dtype == SPI_DTYPE_F16) ((half_t*)base)[at] = (half_t)v;
    else ((bf16_t*)base)[at] = (bf16_t)v;
}
// four neighbours of a row (the first n of them), rounded once
template <typename T>
__device__ __forceinline__ void store_row4(T* p, const float (&v)[4], int n) {
    T o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (T)v[i];
    if (n >= 4) { __builtin_memcpy(p, o, sizeof(o)); return; }
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i < n) p[i] = o[i];
}
__device__ __forceinline__ void store_f32x4(void* base, int dtype, int64_t at, const float (&v)[4], int n) {
    if (dtype == SPI_DTYPE_F32) store_row4((float*)base + at, v, n);
    else if (dtype == SPI_DTYPE_F16) store_row4((half_t*)base + at, v, n);
    else store_row4((bf16_t*)base + at, v, n);
}
__device__ __forceinline__ int dtype_bytes(int dtype) { return dtype == SPI_DTYPE_F32 ? 4 : dtype == SPI_DTYPE_I8 ? 1 : 2; }

// ---- rows in 8 bits: t = max|v| / 127, q = rint(v / t).  The quotients are IEEE divisions: a row gives the same integers wherever it is quantised.
// A row with an infinity or NaN has no scale: t = NaN (its products are NaN) and q = 0.
__device__ __forceinline__ float abs_or_inf(float v) { const float a = fabsf(v); return a <= 3.402823466e38f ? a : __builtin_inff(); }
__device__ __forceinline__ float row_scale(float amax) { return amax == __builtin_inff() ? __builtin_nanf("") : amax / 127.f; }
__device__ __forceinline__ int quantize_value(float v, float scale) {          // scale 0 (an all-zero row) and NaN: 0
    const float q = scale > 0.f ? rintf(v / scale) : 0.f;
    return (int)fminf(fmaxf(q, -127.f), 127.f);
}
#endif
