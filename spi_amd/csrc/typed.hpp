// Typed values and 16-byte chunks of rows, shared by the row operators (norm.hip, linear.hip).
#pragma once
#include "common.hpp"

#ifdef __HIPCC__
typedef _Float16 half_t;
typedef __bf16 bf16_t;
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_acc __attribute__((ext_vector_type(16)));
typedef int i32x16_acc __attribute__((ext_vector_type(16)));

// N neighbours of a row; `n` of them valid at p (any alignment of T), the others 0.  All of them are one load of up to 16 bytes: gfx950 takes it at the alignment of T.
template <typename T, int N_ = 16 / (int)sizeof(T)>
struct Chunk {
    static constexpr int N = N_;
    T v[N];
};
template <typename T, int N = 16 / (int)sizeof(T)>
__device__ __forceinline__ Chunk<T, N> load_chunk(const T* __restrict__ p, int n) {
    Chunk<T, N> c;
    if (n >= N) { __builtin_memcpy(&c, p, sizeof(c)); return c; }
#pragma unroll
    for (int i = 0; i < N; ++i) c.v[i] = i < n ? p[i] : (T)0;
    return c;
}
template <typename T, int N>
__device__ __forceinline__ void store_chunk(T* __restrict__ p, const Chunk<T, N>& c, int n) {
    if (n >= N) { __builtin_memcpy(p, &c, sizeof(c)); return; }
#pragma unroll
    for (int i = 0; i < N; ++i) if (i < n) p[i] = c.v[i];
}
// A thread's N columns of a row, for loads that ask nothing: N neighbours from `start` on, of which those before `first` are not this thread's (they belong to the chunk before
// it, or -- first >= N -- all of them to others).  A load under a condition would be closed by a wait for it; these stay under way until their values are used.
struct Columns { int start, first; };
template <int N>
__device__ __forceinline__ Columns columns(int chunk, int width) {             // width >= N
    const int c0 = chunk * N, start = min(c0, width - N);
    return Columns{start, c0 - start};
}
template <typename T, int N>
__device__ __forceinline__ Chunk<T, N> load_all(const T* __restrict__ p) {
    Chunk<T, N> c;
    __builtin_memcpy(&c, p, sizeof(c));
    return c;
}
template <int N, typename V>
__device__ __forceinline__ void mask_first(float (&v)[N], int first, V other) {
    if (first > 0)
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < first ? other : v[j];
}
template <typename T, int N>
__device__ __forceinline__ void widen(const Chunk<T, N>& c, int first, float (&out)[N]) {       // 0 where the column is not this thread's
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = (float)c.v[j];
    mask_first(out, first, 0.f);
}
// values of a type known at run time only (a wave-uniform branch): as they lie in memory, and widened to fp32
template <int N> struct Raw { uint32_t v[N]; };
template <int N>
__device__ __forceinline__ Raw<N> load_raw(const void* base, int dtype, int64_t at) {
    Raw<N> r;
    if (dtype == SPI_DTYPE_F32) __builtin_memcpy(&r, (const uint32_t*)base + at, 4 * N);
    else if constexpr (N > 1) __builtin_memcpy(&r, (const uint16_t*)base + at, 2 * N);
    else r.v[0] = ((const uint16_t*)base)[at];
    return r;
}
template <int N>
__device__ __forceinline__ void widen(const Raw<N>& r, int dtype, float (&out)[N]) {
    if (dtype == SPI_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = __builtin_bit_cast(float, r.v[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint16_t h = (uint16_t)(r.v[i / 2] >> (i % 2 * 16));
        out[i] = dtype == SPI_DTYPE_F16 ? (float)__builtin_bit_cast(half_t, h) : __builtin_bit_cast(float, (uint32_t)h << 16);
    }
}
template <int N>
__device__ __forceinline__ void load_f32(const void* base, int dtype, int64_t at, float (&out)[N]) { widen<N>(load_raw<N>(base, dtype, at), dtype, out); }
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
// a thread's columns, rounded once: all of them, or those from `first` on
template <typename T, int N>
__device__ __forceinline__ void store_columns(T* p, const float (&v)[N], int first) {
    Chunk<T, N> c;
#pragma unroll
    for (int j = 0; j < N; ++j) c.v[j] = (T)v[j];
    if (first <= 0) { __builtin_memcpy(p, &c, sizeof(c)); return; }
#pragma unroll
    for (int j = 0; j < N; ++j) if (j >= first) p[j] = c.v[j];
}
template <int N>
__device__ __forceinline__ void store_columns(void* base, int dtype, int64_t at, const float (&v)[N], int first) {
    if (dtype == SPI_DTYPE_F32) store_columns((float*)base + at, v, first);
    else if (dtype == SPI_DTYPE_F16) store_columns((half_t*)base + at, v, first);
    else store_columns((bf16_t*)base + at, v, first);
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
// N values of a row by its scale.  The IEEE quotient only where it could round to another integer than the product with 1 / scale does: the two are within
// 127 * (2^-23 + 2^-24) < 2.3e-5 of each other.  (8192 x 4096 bf16 with a division for each value: 29 us, of which 20 are memory's.)
template <int N>
__device__ __forceinline__ Chunk<int8_t, N> quantize_values(const float (&v)[N], float scale, float inverse) {
    Chunk<int8_t, N> q;
    if (!(scale >= 0x1p-100f)) {                                               // zeros, NaN, and scales whose inverse is far from exact
#pragma unroll
        for (int j = 0; j < N; ++j) q.v[j] = (int8_t)quantize_value(v[j], scale);
        return q;
    }
    float r[N], off = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float x = v[j] * inverse;
        r[j] = rintf(x);
        off = fmaxf(off, fabsf(x - r[j]));
    }
    if (off > 0.5f - 1e-4f)
#pragma unroll
        for (int j = 0; j < N; ++j) r[j] = rintf(v[j] / scale);
#pragma unroll
    for (int j = 0; j < N; ++j) q.v[j] = (int8_t)(int)r[j];
    return q;
}
// n blocks as a grid of two axes, for kernels whose blocks take rows or tiles: along one axis a launch has less than 2^32 threads (here: 2^31 in blocks of 1024).
// The blocks behind n have no work.
inline dim3 row_grid(int64_t n) {
    const int64_t x = n < (1 << 21) ? n : 1 << 21;
    return dim3((unsigned)x, (unsigned)ceil_div64(n, x));
}
__device__ __forceinline__ int64_t row_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
#endif
