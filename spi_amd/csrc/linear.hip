// Products of rows with weights: 8-bit integers with scales for each row and each output (spi_linear_int8) and ragged groups of rows with a weight each
// (spi_grouped_linear_*).  Matrix-core tiles: every operand enters v_mfma_*_32x32x* as 16-byte chunks along the summed axis, whatever its type.
#include "typed.hpp"
#include <algorithm>

namespace {

// ---- 32x32 tile steps: lane l holds 16 bytes of row (l & 31), chunk half (l >> 5); result register r of lane l is row 8 (r >> 2) + 4 (l >> 5) + (r & 3) of A,
// row (l & 31) of B ------------------------------------------------------------------------------------------------------------------------
template <typename T> struct Mma;
template <> struct Mma<half_t> {
    typedef f32x16_acc Acc;
    typedef half_t V __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ Acc step(i32x4_t a, i32x4_t b, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <> struct Mma<bf16_t> {
    typedef f32x16_acc Acc;
    typedef bf16_t V __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ Acc step(i32x4_t a, i32x4_t b, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <> struct Mma<float> {                                 // four steps of two: values j of both halves' chunks are summed together
    typedef f32x16_acc Acc;
    typedef float V __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ Acc step(i32x4_t a, i32x4_t b, Acc c) {
        const V x = __builtin_bit_cast(V, a), y = __builtin_bit_cast(V, b);          // (whole vectors: a bit cast of one element reads element 0)
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
};
template <> struct Mma<int8_t> {
    typedef i32x16_acc Acc;
    static __device__ __forceinline__ Acc step(i32x4_t a, i32x4_t b, Acc c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
};

// ---- groups ------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int wave_scan_max(int v) {                         // inclusive running maximum over the lanes of a wave
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_up(v, s);
        if ((int)(threadIdx.x & 63) >= s) v = max(v, o);
    }
    return v;
}

// A tile of rows: group e, or e = -1 for rows of no group.
struct RowTile { int e, row, end; };

// The `tile`-th tile of BM rows, counted over [rows before the first group | group 0 | .. | group E-1 | rows behind the last]: every wave scans the offsets, 64 at
// a time.  The offsets count as their running maximum clamped to 0 .. T, so that ranges never overlap or leave the tensor whatever is in memory.
// row >= end: there is no such tile.
__device__ RowTile find_tile(const int32_t* __restrict__ offsets, int E, int T, int BM, int tile) {
    const int lane = threadIdx.x & 63;
    int carry = 0, before = 0;                                                 // end of the range before this batch; tiles before this batch
    for (int b = 0; b <= E + 1; b += 64) {                                     // range i ends at offsets[i], i = 0 .. E; range E + 1 ends at T
        const int i = b + lane;
        int end = i <= E ? min(max(offsets[i], 0), T) : T;
        end = max(wave_scan_max(end), carry);
        int start = __shfl_up(end, 1);
        if (lane == 0) start = carry;
        const int n = i <= E + 1 ? (end - start + BM - 1) / BM : 0;
        const int upto = before + wave_scan_add(n);
        const uint64_t hit = __ballot(tile < upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const int first = __shfl(upto - n, l), s = __shfl(start, l), e = __shfl(end, l);
            const int range = b + l;
            return RowTile{range == 0 || range == E + 1 ? -1 : range - 1, s + (tile - first) * BM, e};
        }
        carry = __shfl(end, 63);
        before = __shfl(upto, 63);
    }
    return RowTile{-1, 0, 0};
}
// rows of group e, by the same reading of the offsets
__device__ RowTile group_rows(const int32_t* __restrict__ offsets, int T, int e) {
    const int lane = threadIdx.x & 63;
    int start = 0;
    for (int i = lane; i <= e; i += 64) start = max(start, min(max(offsets[i], 0), T));
    start = __shfl(wave_scan_max(start), 63);
    return RowTile{e, start, max(start, min(max(offsets[e + 1], 0), T))};
}
// tiles that T rows in E groups can need
int64_t most_tiles(int64_t T, int E, int BM) { return T / BM + E + 2; }

// ---- one 64 x 64 tile, any strides --------------------------------------------------------------------------------------------------------
// An operand: value (i, k) at p[i * si + k * sk], i < ni, k < nk; one of the strides is 1.
template <typename T> struct Operand { const T* p; int64_t si, sk; int ni, nk; };
constexpr int PITCH = 144;                                                     // bytes of an LDS row: 128 and a chunk that spreads the banks

template <typename T>
__device__ __forceinline__ void stage_operand(const Operand<T>& o, int k0, char* lds) {
    constexpr int N = Chunk<T>::N, KT = 128 / (int)sizeof(T);
    if (o.sk == 1) {
#pragma unroll
        for (int it = 0; it < 2; ++it) {
            const int id = threadIdx.x + it * 256, i = id >> 3, c = id & 7, k = k0 + c * N;
            const Chunk<T> v = load_chunk(o.p + (i < o.ni ? i : 0) * o.si + k, i < o.ni ? o.nk - k : 0);
            *reinterpret_cast<i32x4_t*>(lds + i * PITCH + c * 16) = __builtin_bit_cast(i32x4_t, v);
        }
    } else {
#pragma unroll
        for (int it = 0; it < 2; ++it) {
            const int id = threadIdx.x + it * 256, k = id % KT, i = (id / KT) * N;      // KT * 64 / N = 512 chunks
            const Chunk<T> v = load_chunk(o.p + (int64_t)(k0 + k < o.nk ? k0 + k : 0) * o.sk + i, k0 + k < o.nk ? o.ni - i : 0);
#pragma unroll
            for (int j = 0; j < N; ++j) *reinterpret_cast<T*>(lds + (i + j) * PITCH + k * (int)sizeof(T)) = v.v[j];
        }
    }
}

template <typename T>
__device__ __forceinline__ void tile64(const Operand<T>& A, const Operand<T>& B, char* lds, typename Mma<T>::Acc& acc) {
    constexpr int KT = 128 / (int)sizeof(T);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
    const char* pa = lds + (wm * 32 + (lane & 31)) * PITCH + (lane >> 5) * 16;
    const char* pb = lds + 64 * PITCH + (wn * 32 + (lane & 31)) * PITCH + (lane >> 5) * 16;
    for (int k0 = 0; k0 < A.nk; k0 += KT) {
        __syncthreads();
        stage_operand(A, k0, lds);
        stage_operand(B, k0, lds + 64 * PITCH);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; ++c)
            acc = Mma<T>::step(*reinterpret_cast<const i32x4_t*>(pa + c * 32), *reinterpret_cast<const i32x4_t*>(pb + c * 32), acc);
    }
}
// f(i, j, value) for the values of this thread's part of the tile
template <typename Acc, typename F>
__device__ __forceinline__ void tile64_out(const Acc& acc, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
#pragma unroll
    for (int r = 0; r < 16; ++r) f(wm * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3), wn * 32 + (lane & 31), acc[r]);
}

// ---- 8-bit integers ----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float linear_act(int act, float alpha, float x) {
    switch (act) {
    case SPI_ACT_RELU: return x < 0.f ? 0.f : x;
    case SPI_ACT_LRELU: return x > 0.f ? x : x * alpha;
    case SPI_ACT_TANH: return tanhf(x);
    case SPI_ACT_SIGMOID: return 1.f / (1.f + expf(-x));
    case SPI_ACT_ELU: return x >= 0.f ? x : expm1f(x);
    case SPI_ACT_SELU: return 1.0507009873554805f * (x >= 0.f ? x : 1.6732632423543772f * expm1f(x));
    case SPI_ACT_SOFTPLUS: return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x)));
    case SPI_ACT_SWISH: return x / (1.f + expf(-x));
    default: return x;
    }
}

struct Int8Args {
    const int8_t* q; const float* q_scale; const int8_t* w; const float* w_scale; const float* bias; void* y;
    int64_t q_stride, w_stride;
    int M, N, K, y_dtype, act;
    float alpha, gain, clamp;
};

__device__ __forceinline__ float int8_epilogue(const Int8Args& a, int acc, float scale, float w_scale, float bias) {
    float v = linear_act(a.act, a.alpha, (float)acc * (scale * w_scale) + bias) * a.gain;
    if (a.clamp >= 0.f) v = v > a.clamp ? a.clamp : (v < -a.clamp ? -a.clamp : v);           // (NaN stays)
    return v;
}

__global__ void __launch_bounds__(256) int8_tile64_kernel(const Int8Args a) {
    __shared__ __attribute__((aligned(16))) char lds[2 * 64 * PITCH];
    const int m0 = blockIdx.x * 64, n0 = blockIdx.y * 64;
    i32x16_acc acc = {};
    tile64<int8_t>({a.q + (int64_t)m0 * a.q_stride, a.q_stride, 1, a.M - m0, a.K}, {a.w + (int64_t)n0 * a.w_stride, a.w_stride, 1, a.N - n0, a.K}, lds, acc);
    tile64_out(acc, [&](int i, int j, int v) {
        const int m = m0 + i, n = n0 + j;
        if (m < a.M && n < a.N) store_f32(a.y, a.y_dtype, (int64_t)m * a.N + n, int8_epilogue(a, v, a.q_scale[m], a.w_scale[n], a.bias ? a.bias[n] : 0.f));
    });
}

// One row in TPR threads, NV chunks each held in registers (NV = 0: a row of any length, read twice)
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int width, int64_t x_stride, int8_t* __restrict__ q, int64_t q_stride,
                                                            int q_room, float* __restrict__ scales) {
    constexpr int VEC = Chunk<T>::N, G = 256 / TPR;
    __shared__ float red[4];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / TPR;
    const bool live = row < rows;
    const T* p = x + (live ? row : 0) * x_stride;
    const int w = live ? width : 0, room = live ? q_room : 0;
    Chunk<T> v[NV ? NV : 1];
    float amax = 0.f;
    auto add = [&](const Chunk<T>& c) {                                        // (values behind the row are 0)
#pragma unroll
        for (int j = 0; j < VEC; ++j) amax = fmaxf(amax, abs_or_inf((float)c.v[j]));
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = load_chunk(p + (t + i * TPR) * VEC, w - (t + i * TPR) * VEC);
#pragma unroll
        for (int i = 0; i < NV; ++i) add(v[i]);
    } else
        for (int c = t * VEC; c < w; c += TPR * VEC) add(load_chunk(p + c, w - c));
    amax = wave_max(amax);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }
    const float scale = row_scale(amax);
    if (live && t == 0) scales[row] = scale;
    auto put = [&](const Chunk<T>& c, int c0) {
        int8_t o[VEC], *out = q + (live ? row : 0) * q_stride + c0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = (int8_t)quantize_value((float)c.v[j], scale);
        if (room - c0 >= VEC) __builtin_memcpy(out, o, VEC);
        else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) if (j < room - c0) out[j] = o[j];
        }
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) put(v[i], (t + i * TPR) * VEC);
    } else
        for (int c = t * VEC; c < room; c += TPR * VEC) put(load_chunk(p + c, w - c), c);
}

template <typename T, int TPR, int NV>
void launch_quantize(const void* x, int64_t rows, int width, int64_t x_stride, int8_t* q, int64_t q_stride, int room, float* scale, hipStream_t st) {
    hipLaunchKernelGGL((quantize_rows_kernel<T, TPR, NV>), dim3((unsigned)ceil_div64(rows, 256 / TPR)), dim3(256), 0, st, (const T*)x, rows, width, x_stride, q, q_stride, room,
                       scale);
}
template <typename T>
void quantize(const void* x, int64_t rows, int width, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, hipStream_t st) {
    const int room = (int)std::min<int64_t>(q_stride, ceil_div64(width, 16) * 16), chunks = (int)ceil_div64(width, Chunk<T>::N);
    auto go = [&](auto f) { f(x, rows, width, x_stride, q, q_stride, room, scale, st); };
    if (chunks <= 64) go(launch_quantize<T, 64, 1>);
    else if (chunks <= 128) go(launch_quantize<T, 64, 2>);
    else if (chunks <= 256) go(launch_quantize<T, 64, 4>);
    else if (chunks <= 512) go(launch_quantize<T, 256, 2>);
    else if (chunks <= 1024) go(launch_quantize<T, 256, 4>);
    else go(launch_quantize<T, 256, 0>);
}
bool float_rows(int dtype) { return dtype == SPI_DTYPE_F32 || dtype == SPI_DTYPE_F16 || dtype == SPI_DTYPE_BF16; }
void quantize_any(const void* x, int64_t rows, int width, int64_t x_stride, int dtype, int8_t* q, int64_t q_stride, float* scale, hipStream_t st) {
    if (dtype == SPI_DTYPE_F32) quantize<float>(x, rows, width, x_stride, q, q_stride, scale, st);
    else if (dtype == SPI_DTYPE_F16) quantize<half_t>(x, rows, width, x_stride, q, q_stride, scale, st);
    else quantize<bf16_t>(x, rows, width, x_stride, q, q_stride, scale, st);
}

int check_int8(const spi_linear_int8_desc* d, const char* who) {
    SPI_REQUIRE(d, "%s: no descriptor", who);
    SPI_REQUIRE(d->M >= 0 && d->M < (1ll << 31) - 64 && d->N >= 1 && d->N <= 65535 * 64 && d->K >= 1 && d->K <= SPI_LINEAR_INT8_MAX_K, "%s: M %lld, N %d, K %d", who,
                (long long)d->M, d->N, d->K);
    SPI_REQUIRE(d->x_dtype == SPI_DTYPE_I8 || float_rows(d->x_dtype), "%s: x_dtype %d", who, d->x_dtype);
    SPI_REQUIRE(float_rows(d->y_dtype), "%s: y_dtype %d", who, d->y_dtype);
    SPI_REQUIRE(d->M == 0 || (d->x && d->y), "%s: null rows", who);
    SPI_REQUIRE(d->w && d->w_scale && (d->x_dtype != SPI_DTYPE_I8 || d->x_scale || d->M == 0), "%s: null weights or scales", who);
    SPI_REQUIRE(d->x_stride >= d->K && d->w_stride >= d->K && d->w_bytes >= (int64_t)(d->N - 1) * d->w_stride + d->K, "%s: strides %lld, %lld", who, (long long)d->x_stride,
                (long long)d->w_stride);
    SPI_REQUIRE(d->act >= SPI_ACT_LINEAR && d->act <= SPI_ACT_SWISH, "%s: act %d", who, d->act);
    return SPI_OK;
}
int64_t q_pitch(int K) { return ceil_div64(K, 16) * 16; }

// ---- ragged groups -----------------------------------------------------------------------------------------------------------------------
struct GroupArgs {
    const void *x, *w, *bias, *dy;
    void *y, *dx, *dw, *db;
    const int32_t* offsets;
    int T, E, N, K;
    float gain;
};

template <typename T>
__global__ void __launch_bounds__(256) grouped_fwd64_kernel(const GroupArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[2 * 64 * PITCH];
    const RowTile t = find_tile(a.offsets, a.E, a.T, 64, blockIdx.x);
    if (t.row >= t.end) return;
    const int n0 = blockIdx.y * 64;
    f32x16_acc acc = {};
    if (t.e >= 0)
        tile64<T>({(const T*)a.x + (int64_t)t.row * a.K, a.K, 1, t.end - t.row, a.K}, {(const T*)a.w + ((int64_t)t.e * a.N + n0) * a.K, a.K, 1, a.N - n0, a.K}, lds, acc);
    tile64_out(acc, [&](int i, int j, float v) {
        const int row = t.row + i, n = n0 + j;
        if (row < t.end && n < a.N)
            ((T*)a.y)[(int64_t)row * a.N + n] = (T)(t.e < 0 ? 0.f : v * a.gain + (a.bias ? (float)((const T*)a.bias)[(int64_t)t.e * a.N + n] : 0.f));
    });
}
template <typename T>
__global__ void __launch_bounds__(256) grouped_dgrad64_kernel(const GroupArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[2 * 64 * PITCH];
    const RowTile t = find_tile(a.offsets, a.E, a.T, 64, blockIdx.x);
    if (t.row >= t.end) return;
    const int k0 = blockIdx.y * 64;
    f32x16_acc acc = {};
    if (t.e >= 0)
        tile64<T>({(const T*)a.dy + (int64_t)t.row * a.N, a.N, 1, t.end - t.row, a.N}, {(const T*)a.w + (int64_t)t.e * a.N * a.K + k0, 1, a.K, a.K - k0, a.N}, lds, acc);
    tile64_out(acc, [&](int i, int j, float v) {
        const int row = t.row + i, k = k0 + j;
        if (row < t.end && k < a.K) ((T*)a.dx)[(int64_t)row * a.K + k] = (T)(v * a.gain);
    });
}
template <typename T>
__global__ void __launch_bounds__(256) grouped_wgrad64_kernel(const GroupArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[2 * 64 * PITCH];
    const int n0 = blockIdx.x * 64, k0 = blockIdx.y * 64, e = blockIdx.z;
    const RowTile t = group_rows(a.offsets, a.T, e);
    f32x16_acc acc = {};
    tile64<T>({(const T*)a.dy + (int64_t)t.row * a.N + n0, 1, a.N, a.N - n0, t.end - t.row}, {(const T*)a.x + (int64_t)t.row * a.K + k0, 1, a.K, a.K - k0, t.end - t.row}, lds, acc);
    tile64_out(acc, [&](int i, int j, float v) {
        const int n = n0 + i, k = k0 + j;
        if (n < a.N && k < a.K) ((T*)a.dw)[((int64_t)e * a.N + n) * a.K + k] = (T)(v * a.gain);
    });
}
// db[e][n] = sum of dy over the group's rows: 64 columns per block, four rows at a time, in a fixed order
template <typename T>
__global__ void __launch_bounds__(256) grouped_bias_grad_kernel(const GroupArgs a) {
    __shared__ float s[4][64];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6, n = blockIdx.x * 64 + c, e = blockIdx.y;
    const RowTile t = group_rows(a.offsets, a.T, e);
    float v = 0.f;
    if (n < a.N)
        for (int row = t.row + r; row < t.end; row += 4) v += (float)((const T*)a.dy)[(int64_t)row * a.N + n];
    s[r][c] = v;
    __syncthreads();
    if (r == 0 && n < a.N) ((T*)a.db)[(int64_t)e * a.N + n] = (T)((s[0][c] + s[1][c]) + (s[2][c] + s[3][c]));
}

int check_grouped(const spi_grouped_linear_desc* d, const char* who) {
    SPI_REQUIRE(d, "%s: no descriptor", who);
    SPI_REQUIRE(d->T >= 0 && d->T < (1ll << 31) - 64 && d->E >= 1 && d->E <= 65535 && d->N >= 1 && d->N <= 65535 * 64 && d->K >= 1 && d->K <= 65535 * 64,
                "%s: T %lld, E %d, N %d, K %d", who, (long long)d->T, d->E, d->N, d->K);
    SPI_REQUIRE(float_rows(d->dtype), "%s: dtype %d", who, d->dtype);
    SPI_REQUIRE(d->offsets, "%s: null offsets", who);
    return SPI_OK;
}
GroupArgs group_args(const spi_grouped_linear_desc& d) {
    return GroupArgs{d.x, d.w, d.bias, d.dy, d.y, d.dx, d.dw, d.db, d.offsets, (int)d.T, d.E, d.N, d.K, d.gain};
}

}  // namespace

extern "C" int spi_quantize_rows(const void* x, int64_t rows, int width, int64_t x_stride, int dtype, int8_t* q, int64_t q_stride, float* scale, spi_stream_t stream) {
    SPI_REQUIRE(rows >= 0 && rows < (1ll << 31) && width >= 1 && width <= SPI_LINEAR_INT8_MAX_K, "spi_quantize_rows: %lld rows of %d", (long long)rows, width);
    SPI_REQUIRE(float_rows(dtype), "spi_quantize_rows: dtype %d", dtype);
    SPI_REQUIRE(x_stride >= width && q_stride >= width, "spi_quantize_rows: strides %lld, %lld", (long long)x_stride, (long long)q_stride);
    if (rows == 0) return SPI_OK;
    SPI_REQUIRE(x && q && scale, "spi_quantize_rows: null pointer");
    quantize_any(x, rows, width, x_stride, dtype, q, q_stride, scale, as_stream(stream));
    SPI_LAUNCH_CHECK("spi_quantize_rows");
    return SPI_OK;
}

extern "C" int spi_sizeof_linear_int8_desc(void) { return (int)sizeof(spi_linear_int8_desc); }
extern "C" int64_t spi_linear_int8_workspace(const spi_linear_int8_desc* d) {
    if (check_int8(d, "spi_linear_int8_workspace") || d->x_dtype == SPI_DTYPE_I8) return 0;
    return d->M * (q_pitch(d->K) + (int64_t)sizeof(float));
}
extern "C" int spi_linear_int8(const spi_linear_int8_desc* d, spi_stream_t stream) {
    if (int rc = check_int8(d, "spi_linear_int8")) return rc;
    if (d->M == 0) return SPI_OK;
    SPI_REQUIRE(d->workspace_bytes >= spi_linear_int8_workspace(d) && (d->workspace || d->workspace_bytes == 0), "spi_linear_int8: workspace too small");
    hipStream_t st = as_stream(stream);
    Int8Args a{(const int8_t*)d->x, d->x_scale, d->w, d->w_scale, d->bias, d->y, d->x_stride, d->w_stride, (int)d->M, d->N, d->K, d->y_dtype, d->act, d->alpha, d->gain, d->clamp};
    if (d->x_dtype != SPI_DTYPE_I8) {
        a.q = (int8_t*)d->workspace;
        a.q_stride = q_pitch(d->K);
        a.q_scale = (float*)((char*)d->workspace + d->M * a.q_stride);
        quantize_any(d->x, d->M, d->K, d->x_stride, d->x_dtype, (int8_t*)a.q, a.q_stride, (float*)a.q_scale, st);
        SPI_LAUNCH_CHECK("spi_linear_int8 (quantize)");
    }
    hipLaunchKernelGGL(int8_tile64_kernel, dim3((unsigned)ceil_div64(d->M, 64), (unsigned)ceil_div64(d->N, 64)), dim3(256), 0, st, a);
    SPI_LAUNCH_CHECK("spi_linear_int8");
    return SPI_OK;
}

extern "C" int spi_sizeof_grouped_linear_desc(void) { return (int)sizeof(spi_grouped_linear_desc); }
extern "C" int64_t spi_grouped_linear_workspace(const spi_grouped_linear_desc* d, int pass) {
    (void)pass;
    return check_grouped(d, "spi_grouped_linear_workspace") ? 0 : 0;
}
#define SPI_BY_TYPE(kernel, grid, args)                                                                                   \
    do {                                                                                                                  \
        if (d->dtype == SPI_DTYPE_F32) hipLaunchKernelGGL(kernel<float>, grid, dim3(256), 0, as_stream(stream), args);        \
        else if (d->dtype == SPI_DTYPE_F16) hipLaunchKernelGGL(kernel<half_t>, grid, dim3(256), 0, as_stream(stream), args);  \
        else hipLaunchKernelGGL(kernel<bf16_t>, grid, dim3(256), 0, as_stream(stream), args);                                 \
    } while (0)

extern "C" int spi_grouped_linear_fwd(const spi_grouped_linear_desc* d, spi_stream_t stream) {
    if (int rc = check_grouped(d, "spi_grouped_linear_fwd")) return rc;
    if (d->T == 0) return SPI_OK;
    SPI_REQUIRE(d->x && d->w && d->y, "spi_grouped_linear_fwd: null pointer");
    const GroupArgs a = group_args(*d);
    SPI_BY_TYPE(grouped_fwd64_kernel, dim3((unsigned)most_tiles(d->T, d->E, 64), (unsigned)ceil_div64(d->N, 64)), a);
    SPI_LAUNCH_CHECK("spi_grouped_linear_fwd");
    return SPI_OK;
}
extern "C" int spi_grouped_linear_dgrad(const spi_grouped_linear_desc* d, spi_stream_t stream) {
    if (int rc = check_grouped(d, "spi_grouped_linear_dgrad")) return rc;
    if (d->T == 0) return SPI_OK;
    SPI_REQUIRE(d->dy && d->w && d->dx, "spi_grouped_linear_dgrad: null pointer");
    const GroupArgs a = group_args(*d);
    SPI_BY_TYPE(grouped_dgrad64_kernel, dim3((unsigned)most_tiles(d->T, d->E, 64), (unsigned)ceil_div64(d->K, 64)), a);
    SPI_LAUNCH_CHECK("spi_grouped_linear_dgrad");
    return SPI_OK;
}
extern "C" int spi_grouped_linear_wgrad(const spi_grouped_linear_desc* d, spi_stream_t stream) {
    if (int rc = check_grouped(d, "spi_grouped_linear_wgrad")) return rc;
    SPI_REQUIRE(d->T == 0 || d->dy, "spi_grouped_linear_wgrad: null dy");
    SPI_REQUIRE(d->T == 0 || !d->dw || d->x, "spi_grouped_linear_wgrad: null x");
    const GroupArgs a = group_args(*d);
    if (d->dw) {
        SPI_BY_TYPE(grouped_wgrad64_kernel, dim3((unsigned)ceil_div64(d->N, 64), (unsigned)ceil_div64(d->K, 64), (unsigned)d->E), a);
        SPI_LAUNCH_CHECK("spi_grouped_linear_wgrad");
    }
    if (d->db) {
        SPI_BY_TYPE(grouped_bias_grad_kernel, dim3((unsigned)ceil_div64(d->N, 64), (unsigned)d->E), a);
        SPI_LAUNCH_CHECK("spi_grouped_linear_wgrad (bias)");
    }
    return SPI_OK;
}
