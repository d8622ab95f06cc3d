// Products of rows with weights: 8-bit integers with scales for each row and each output (spi_linear_int8) and ragged groups of rows with a weight each
// (spi_grouped_linear_*).
#include "tile.hpp"
#include <algorithm>

namespace {

// ---- groups ------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int wave_scan_max(int v) {                         // inclusive running maximum over the lanes of a wave
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_up(v, s);
        if ((int)(threadIdx.x & 63) >= s) v = max(v, o);
    }
    return v;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }      // the same in all lanes: into a scalar register

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
            return RowTile{uniform(range == 0 || range == E + 1 ? -1 : range - 1), uniform(s + (tile - first) * BM), uniform(e)};
        }
        carry = __shfl(end, 63);
        before = __shfl(upto, 63);
    }
    return RowTile{-1, 0, 0};
}
// number of tiles that find_tile knows
__device__ int count_tiles(const int32_t* __restrict__ offsets, int E, int T, int BM) {
    const int lane = threadIdx.x & 63;
    int carry = 0, tiles = 0;
    for (int b = 0; b <= E + 1; b += 64) {
        const int i = b + lane;
        int end = i <= E ? min(max(offsets[i], 0), T) : T;
        end = max(wave_scan_max(end), carry);
        int start = __shfl_up(end, 1);
        if (lane == 0) start = carry;
        tiles += __shfl(wave_scan_add(i <= E + 1 ? (end - start + BM - 1) / BM : 0), 63);
        carry = __shfl(end, 63);
    }
    return uniform(tiles);
}
// rows of group e, by the same reading of the offsets
__device__ RowTile group_rows(const int32_t* __restrict__ offsets, int T, int e) {
    const int lane = threadIdx.x & 63;
    int start = 0;
    for (int i = lane; i <= e; i += 64) start = max(start, min(max(offsets[i], 0), T));
    start = __shfl(wave_scan_max(start), 63);
    return RowTile{e, uniform(start), uniform(max(start, min(max(offsets[e + 1], 0), T)))};
}
// tiles that T rows in E groups can need
int64_t most_tiles(int64_t T, int E, int BM) { return T / BM + E + 2; }

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

// Tiles of 256 x 256 (8 waves), 128 x 128 and 64 x 64 (4 waves).
template <typename T, int SIZE, bool COLA, bool COLB, int LOAD>
using Engine = TileEngine<T, SIZE, SIZE, 2, SIZE == 256 ? 4 : 2, COLA, COLB, LOAD>;

template <int SIZE, int LOAD>
__global__ void __launch_bounds__(SIZE == 256 ? 512 : 256) int8_tile_kernel(const Int8Args a, int rows, int cols) {
    typedef Engine<int8_t, SIZE, false, false, LOAD> E;
    __shared__ __attribute__((aligned(1024))) char s0[E::STAGE], s1[E::STAGE];
    const int64_t block = row_block();
    if (block >= rows * cols) return;                                          // (rows * cols < 2^31, see check_int8)
    int row, col;
    band_order(xcd_run((int)block, rows * cols), rows, cols, row, col);
    const int m0 = row * SIZE, n0 = col * SIZE, m = min(SIZE, a.M - m0), n = min(SIZE, a.N - n0);
    typename E::Accs acc = {};
    const int64_t k = LOAD == LOAD_DMA ? (a.K + 15) / 16 * 16 : a.K;           // (LOAD_DMA: the padding of the quantised rows is 0, so that of the weights does not count)
    const TileOperand A{(const char*)a.q + m0 * a.q_stride, a.q_stride, m * a.q_stride, k, m, (int64_t)(a.M - 1 - m0) * a.q_stride + a.K},
        B{(const char*)a.w + n0 * a.w_stride, a.w_stride, n * a.w_stride, k, n, (int64_t)(a.N - 1 - n0) * a.w_stride + a.K};
    E::run(A, B, s0, s1, acc);
    E::each(acc, s0, s1, [&](int i, int j, i32x4_t v) {
        if (i >= m || j >= n) return;
        const float scale = a.q_scale[m0 + i];
        const int c0 = n0 + j;
        float y[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = j + c < n ? int8_epilogue(a, v[c], scale, a.w_scale[c0 + c], a.bias ? a.bias[c0 + c] : 0.f) : 0.f;
        store_f32x4(a.y, a.y_dtype, (int64_t)(m0 + i) * a.N + c0, y, n - j);
    });
}

// Up to 16 rows: 16 outputs a block, the summed axis over its four waves, whose weights go straight from memory to the matrix cores (v_mfma_i32_16x16x64_i8) -- all of a wave's
// loads under way at once.  The rows wait in LDS: int8 rows as they are; up to four rows of floats are quantised by every block, each for itself (one launch fewer).
// Bound by latency: 1 x 512 x 512 4.3 us (as a tile of 64 x 64 behind a launch that quantises: 5.2 + 2.1), 14 x 2048 x 4096 (8 MB of weights) 6.4 us (9.1).
constexpr int FEW = 16, FEW_FLOATS = 4, FEW_LDS = 60000;
__host__ __device__ inline int few_pitch(int K) { return (K + 63) / 64 * 64 + 16; }

template <typename T>
__global__ void __launch_bounds__(256) int8_few_rows_kernel(const Int8Args a, const T* __restrict__ x, int64_t x_stride, int64_t w_bytes) {
    extern __shared__ __attribute__((aligned(16))) char rows[];               // [M][few_pitch(K)]
    __shared__ float scales[FEW], red[2][4];
    __shared__ int part[4][FEW][FEW + 1];
    constexpr int N = Chunk<T>::N;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pitch = few_pitch(a.K);
    const int64_t block = row_block();
    if (block * FEW >= a.N) return;
    const int n0 = (int)block * FEW;
    if constexpr (sizeof(T) == 1) {
        const int whole = a.K / 16, rest = pitch / 16 - whole;
#pragma unroll 4
        for (int c = tid; c < a.M * whole; c += 256) {
            const int m = c / whole, k = c % whole * 16;
            *reinterpret_cast<i32x4_t*>(rows + m * pitch + k) = __builtin_bit_cast(i32x4_t, load_all<int8_t, 16>((const int8_t*)x + m * x_stride + k));
        }
        for (int c = tid; c < a.M * rest; c += 256) {
            const int m = c / rest, k = (whole + c % rest) * 16;
            *reinterpret_cast<i32x4_t*>(rows + m * pitch + k) = __builtin_bit_cast(i32x4_t, load_chunk((const int8_t*)x + m * x_stride + (k < a.K ? k : 0), a.K - k));
        }
        if (tid < a.M) scales[tid] = a.q_scale[tid];
    } else {
        for (int m = 0; m < a.M; ++m) {                                        // the row is read twice, the second time from the cache
            const T* p = x + m * x_stride;
            float amax = 0.f;
            for (int k = tid * N; k < a.K; k += 256 * N) {
                const Chunk<T> c = load_chunk(p + k, a.K - k);
#pragma unroll
                for (int j = 0; j < N; ++j) amax = fmaxf(amax, abs_or_inf((float)c.v[j]));
            }
            amax = wave_max(amax);
            if (lane == 0) red[m & 1][wave] = amax;
            __syncthreads();
            const float scale = row_scale(fmaxf(fmaxf(red[m & 1][0], red[m & 1][1]), fmaxf(red[m & 1][2], red[m & 1][3])));
            const float inverse = 1.f / scale;
            if (tid == 0) scales[m] = scale;
            for (int k = tid * N; k < pitch; k += 256 * N) {
                const Chunk<T> c = load_chunk(p + (k < a.K ? k : 0), a.K - k);
                float f[N];
                widen(c, 0, f);
                const Chunk<int8_t, N> q = quantize_values(f, scale, inverse);
                __builtin_memcpy(rows + m * pitch + k, &q, N);
            }
        }
    }
    __syncthreads();
    const int steps = (a.K + 63) / 64, from = steps * wave / 4, to = steps * (wave + 1) / 4, n = min(n0 + (lane & 15), a.N - 1), kg = (lane >> 4) * 16;
    const int8_t* w = a.w + n * a.w_stride;
    const int64_t room = w_bytes - n * a.w_stride;                             // a chunk that runs on behind the row reads what lies there, against zeros in the rows
    const char* q = rows + min(lane & 15, a.M - 1) * pitch + kg;
    typedef int i32x4_acc __attribute__((ext_vector_type(4)));
    i32x4_acc acc = {0, 0, 0, 0};
    int k = from;
    const bool whole = to * 64 <= w_bytes - min(n0 + FEW - 1, a.N - 1) * a.w_stride;           // for the whole wave: a matrix instruction wants all its lanes
    for (; whole && k + 8 <= to; k += 8) {
        i32x4_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = __builtin_bit_cast(i32x4_t, load_all<int8_t, 16>(w + (k + i) * 64 + kg));
#pragma unroll
        for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4_t*>(q + (k + i) * 64), b[i], acc, 0, 0, 0);
    }
    for (; k < to; ++k) {
        const int64_t left = room - (k * 64 + kg);
        const i32x4_t b = __builtin_bit_cast(i32x4_t, load_chunk(w + (left > 0 ? k * 64 + kg : 0), (int)(left < 16 ? left : 16)));
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4_t*>(q + k * 64), b, acc, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][(lane >> 4) * 4 + r][lane & 15] = acc[r];
    __syncthreads();
    const int m = tid >> 4, c = tid & 15;
    if (m >= a.M || n0 + c >= a.N) return;
    const int sum = part[0][m][c] + part[1][m][c] + part[2][m][c] + part[3][m][c];
    store_f32(a.y, a.y_dtype, (int64_t)m * a.N + n0 + c, int8_epilogue(a, sum, scales[m], a.w_scale[n0 + c], a.bias ? a.bias[n0 + c] : 0.f));
}

// One row in TPR threads, NV chunks each held in registers; NV = 0: a row of any length, read twice.
// Bound by HBM: 8192 x 4096 bf16 21 us = 4.8 TB/s (29 us with a division for each value).
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int width, int64_t x_stride, int8_t* __restrict__ q, int64_t q_stride,
                                                            int q_room, float* __restrict__ scales) {
    constexpr int VEC = Chunk<T>::N, G = 256 / TPR;
    __shared__ float red[4];
    const int t = threadIdx.x % TPR;
    const int64_t row_at = row_block() * G + threadIdx.x / TPR;
    const bool live = row_at < rows;
    const int64_t row = live ? row_at : rows - 1;
    const T* p = x + row * x_stride;
    int8_t* out = q + row * q_stride;
    Chunk<T> v[NV ? NV : 1];
    Columns at[NV ? NV : 1];
    float amax = 0.f;
    auto add = [&](const Chunk<T>& c) {                                        // (values read twice, or 0 behind the row, change no maximum)
#pragma unroll
        for (int j = 0; j < VEC; ++j) amax = fmaxf(amax, abs_or_inf((float)c.v[j]));
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            at[i] = columns<VEC>(t + i * TPR, width);
            v[i] = load_all<T, VEC>(p + at[i].start);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) add(v[i]);
    } else
        for (int c = t * VEC; c < width; c += TPR * VEC) add(load_chunk(p + c, width - c));
    amax = wave_max(amax);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }
    if (!live) return;
    const float scale = row_scale(amax);
    if (t == 0) scales[row] = scale;
    if (t < q_room - width) out[width + t] = 0;                                // the padding (less than 16 bytes)
    const float inverse = 1.f / scale;
    auto quantized = [&](const Chunk<T>& c) {
        float f[VEC];
        widen(c, 0, f);
        return quantize_values(f, scale, inverse);
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Chunk<int8_t, VEC> o = quantized(v[i]);
            if (at[i].first <= 0) __builtin_memcpy(out + at[i].start, &o, VEC);
            else if (at[i].first < VEC)
#pragma unroll
                for (int j = 0; j < VEC; ++j) if (j >= at[i].first) out[at[i].start + j] = o.v[j];
        }
    } else
        for (int c = t * VEC; c < width; c += TPR * VEC) store_chunk(out + c, quantized(load_chunk(p + c, width - c)), width - c);
}

template <typename T, int TPR, int NV>
void launch_quantize(const void* x, int64_t rows, int width, int64_t x_stride, int8_t* q, int64_t q_stride, int room, float* scale, hipStream_t st) {
    hipLaunchKernelGGL((quantize_rows_kernel<T, TPR, NV>), row_grid(ceil_div64(rows, 256 / TPR)), dim3(256), 0, st, (const T*)x, rows, width, x_stride, q, q_stride, room,
                       scale);
}
template <typename T>
void quantize(const void* x, int64_t rows, int width, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, hipStream_t st) {
    const int room = (int)std::min<int64_t>(q_stride, ceil_div64(width, 16) * 16), chunks = (int)ceil_div64(width, Chunk<T>::N);
    auto go = [&](auto f) { f(x, rows, width, x_stride, q, q_stride, room, scale, st); };
    if (width < Chunk<T>::N) go(launch_quantize<T, 64, 0>);
    else if (chunks <= 64) go(launch_quantize<T, 64, 1>);
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
    SPI_REQUIRE(d->M >= 0 && d->M <= (1ll << 30) && d->N >= 1 && d->K >= 1 && d->K <= SPI_LINEAR_INT8_MAX_K && ceil_div64(d->M, 64) * ceil_div64(d->N, 64) < (1ll << 31),
                "%s: M %lld, N %d, K %d", who, (long long)d->M, d->N, d->K);
    SPI_REQUIRE(d->x_dtype == SPI_DTYPE_I8 || float_rows(d->x_dtype), "%s: x_dtype %d", who, d->x_dtype);
    SPI_REQUIRE(float_rows(d->y_dtype), "%s: y_dtype %d", who, d->y_dtype);
    SPI_REQUIRE(d->M == 0 || (d->x && d->y), "%s: null rows", who);
    SPI_REQUIRE(d->w && d->w_scale && (d->x_dtype != SPI_DTYPE_I8 || d->x_scale || d->M == 0), "%s: null weights or scales", who);
    SPI_REQUIRE(d->x_stride >= d->K && d->w_stride >= d->K && d->w_bytes >= (int64_t)(d->N - 1) * d->w_stride + d->K, "%s: strides %lld, %lld", who, (long long)d->x_stride,
                (long long)d->w_stride);
    SPI_REQUIRE(d->w_stride <= (1 << 22) && (d->x_dtype != SPI_DTYPE_I8 || d->x_stride <= (1 << 22)), "%s: 8-bit rows %lld, %lld bytes apart (at most 2^22)", who,
                (long long)d->x_stride, (long long)d->w_stride);
    SPI_REQUIRE(d->act >= SPI_ACT_LINEAR && d->act <= SPI_ACT_SWISH, "%s: act %d", who, d->act);
    return SPI_OK;
}
int64_t q_pitch(int K) { return ceil_div64(K, 16) * 16; }
bool few_rows(const spi_linear_int8_desc& d) { return d.M <= FEW && d.M * few_pitch(d.K) <= FEW_LDS; }
bool few_floats(const spi_linear_int8_desc& d) { return few_rows(d) && d.M <= FEW_FLOATS && d.x_dtype != SPI_DTYPE_I8; }
// rows of floats: as they lie in the workspace once they are quantised, the scales behind them
Int8Args int8_args(const spi_linear_int8_desc& d) {
    Int8Args a{(const int8_t*)d.x, d.x_scale, d.w, d.w_scale, d.bias, d.y, d.x_stride, d.w_stride, (int)d.M, d.N, d.K, d.y_dtype, d.act, d.alpha, d.gain, d.clamp};
    if (d.x_dtype != SPI_DTYPE_I8) {
        a.q = (const int8_t*)d.workspace;
        a.q_stride = q_pitch(d.K);
        a.q_scale = (const float*)(a.q + d.M * a.q_stride);
    }
    return a;
}
template <typename T>
void launch_few(const spi_linear_int8_desc& d, const Int8Args& a, const void* x, int64_t x_stride, hipStream_t st) {
    hipLaunchKernelGGL(int8_few_rows_kernel<T>, row_grid(ceil_div64(d.N, FEW)), dim3(256), (size_t)d.M * few_pitch(d.K), st, a, (const T*)x, x_stride, d.w_bytes);
}

// ---- ragged groups -----------------------------------------------------------------------------------------------------------------------
struct GroupArgs {
    const void *x, *w, *bias, *dy;
    void *y, *dx, *dw, *db;
    const int32_t* offsets;
    int T, E, N, K;
    float gain;
};

enum { PASS_FWD = 0, PASS_DGRAD = 1, PASS_WGRAD = 2 };
template <typename T, int PASS, int SIZE, int LOAD>
using PassEngine = Engine<T, SIZE, PASS == PASS_WGRAD, PASS != PASS_FWD, LOAD>;

// the tile of engine E at rows t.row .. (at most t.end), columns c0 ..; of dw: at (r0, c0) of group t.e
template <typename E, typename T, int PASS>
__device__ __forceinline__ void grouped_tile(const GroupArgs& a, const RowTile& t, int r0, int c0, char* s0, char* s1) {
    constexpr int ES = (int)sizeof(T);
    const int64_t pn = (int64_t)a.N * ES, pk = (int64_t)a.K * ES;
    const int width = PASS == PASS_FWD ? a.N : a.K, cols = min(E::BN, width - c0);
    typename E::Accs acc = {};
    auto run = [&](const TileOperand& A, const TileOperand& B) { E::run(A, B, s0, s1, acc); };
    if constexpr (PASS == PASS_WGRAD) {
        const int rows = min(E::BM, a.N - r0);
        const int64_t len = t.end - t.row;
        run({(const char*)a.dy + t.row * pn + r0 * ES, pn, len * pn - r0 * ES, len, rows, (a.T - t.row) * pn - r0 * ES},
            {(const char*)a.x + t.row * pk + c0 * ES, pk, len * pk - c0 * ES, len, cols, (a.T - t.row) * pk - c0 * ES});
        E::each(acc, s0, s1, [&](int i, int j, f32x4_t v) {
            if (i >= rows || j >= cols) return;
            const float y[4] = {v[0] * a.gain, v[1] * a.gain, v[2] * a.gain, v[3] * a.gain};
            store_row4((T*)a.dw + ((int64_t)t.e * a.N + r0 + i) * a.K + c0 + j, y, cols - j);
        });
    } else {
        const int rows = min(E::BM, t.end - t.row), inner = PASS == PASS_FWD ? a.K : a.N;
        if (t.e >= 0) {
            const int64_t pi = PASS == PASS_FWD ? pk : pn;
            const char* w = (const char*)a.w + (int64_t)t.e * a.N * pk;
            const TileOperand A{(const char*)(PASS == PASS_FWD ? a.x : a.dy) + t.row * pi, pi, rows * pi, inner, rows, (a.T - t.row) * pi};
            const int64_t end = (int64_t)(a.E - t.e) * a.N * pk;
            if constexpr (PASS == PASS_FWD) run(A, {w + c0 * pk, pk, cols * pk, inner, cols, end - c0 * pk});
            else run(A, {w + c0 * ES, pk, inner * pk - c0 * ES, inner, cols, end - c0 * ES});
        }
        const T* bias = PASS == PASS_FWD && a.bias && t.e >= 0 ? (const T*)a.bias + (int64_t)t.e * a.N + c0 : nullptr;
        T* out = (T*)(PASS == PASS_FWD ? a.y : a.dx) + (int64_t)t.row * width + c0;
        E::each(acc, s0, s1, [&](int i, int j, f32x4_t v) {
            if (i >= rows || j >= cols) return;
            float y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) y[q] = v[q] * a.gain + (bias && j + q < cols ? (float)bias[j + q] : 0.f);
            store_row4(out + (int64_t)i * width + j, y, cols - j);
        });
    }
}

// One tile a block.  Tiles of 256 x 256 come in rounds of one for each CU; where the last round would leave more than half of the chip idle, its tiles are cut into four.
constexpr int CUS = 256;
__device__ __forceinline__ int whole_tiles(int tiles) { const int last = tiles % CUS; return last <= CUS / 2 ? tiles - last : tiles; }
int64_t most_blocks(int64_t tiles) { return tiles + 3 * (CUS / 2); }

template <typename T, int PASS, int SIZE, int LOAD>
__global__ void __launch_bounds__(SIZE == 256 ? 512 : 256) grouped_tile_kernel(const GroupArgs a) {
    typedef PassEngine<T, PASS, SIZE, LOAD> E;
    __shared__ __attribute__((aligned(1024))) char s0[E::STAGE], s1[E::STAGE];
    const int width = PASS == PASS_FWD ? a.N : a.K, cols = (width + SIZE - 1) / SIZE;
    const int rows = PASS == PASS_WGRAD ? (a.N + SIZE - 1) / SIZE : count_tiles(a.offsets, a.E, a.T, SIZE), tiles = rows * cols * (PASS == PASS_WGRAD ? a.E : 1);
    const int64_t block = row_block();
    const int whole = SIZE == 256 ? whole_tiles(tiles) : tiles;
    if (block >= (SIZE == 256 ? whole + (int64_t)(tiles - whole) * 4 : tiles)) return;
    const int cut = (int)(block - whole), tile = cut < 0 ? (int)block : whole + cut / 4;
    int row, col, r0 = 0;
    RowTile t;
    if constexpr (PASS == PASS_WGRAD) {
        const int of = rows * cols;                            // each group's tiles over all XCDs: groups differ in length
        band_order(xcd_run(tile % of, of), rows, cols, row, col);
        t = group_rows(a.offsets, a.T, tile / of);
        r0 = row * SIZE;
    } else {
        band_order(cut < 0 ? xcd_run(tile, whole) : tile, rows, cols, row, col);
        t = find_tile(a.offsets, a.E, a.T, SIZE, row);
    }
    int c0 = col * SIZE;
    if constexpr (SIZE == 256) {
        if (cut >= 0) {
            typedef TileEngine<T, 128, 128, 2, 4, PASS == PASS_WGRAD, PASS != PASS_FWD, LOAD> Q;
            const int down = cut % 4 / 2 * 128, right = cut % 2 * 128;
            c0 += right;
            if (PASS == PASS_WGRAD) r0 += down;
            else t.row += down;
            if (c0 < width && (PASS == PASS_WGRAD ? r0 < a.N : t.row < t.end)) grouped_tile<Q, T, PASS>(a, t, r0, c0, s0, s1);
            return;
        }
    }
    grouped_tile<E, T, PASS>(a, t, r0, c0, s0, s1);
}
// db[e][n] = sum of dy over the group's rows, in two steps of a fixed order: part s of S of the group's rows into part [E][S][N] (S = 1: straight into db), then the
// parts.  A block takes 64 chunks of VEC columns by four rows at a time.  Bound by HBM: 16384 x 2048 bf16 12.8 us = 5.2 TB/s, and 5.2 us for the parts.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) grouped_bias_grad_kernel(const GroupArgs a, float* __restrict__ part, int S) {
    __shared__ float sum[4][64][VEC + 1];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6, s = blockIdx.y, e = blockIdx.z;
    const Columns at = columns<VEC>(blockIdx.x * 64 + c, a.N);
    const RowTile t = group_rows(a.offsets, a.T, e);
    const int64_t len = t.end - t.row, from = t.row + len * s / S, to = t.row + len * (s + 1) / S;
    float v[VEC] = {};
    const T* p = (const T*)a.dy + at.start;
#pragma unroll 8
    for (int64_t row = from + r; row < to; row += 4) {
        const Chunk<T, VEC> x = load_all<T, VEC>(p + row * a.N);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] += (float)x.v[j];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[r][c][j] = v[j];
    __syncthreads();
    if (r) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (sum[0][c][j] + sum[1][c][j]) + (sum[2][c][j] + sum[3][c][j]);
    if (at.first >= VEC) return;
    if (S > 1) store_columns(part + ((int64_t)e * S + s) * a.N + at.start, v, at.first);
    else store_columns((T*)a.db + (int64_t)e * a.N + at.start, v, at.first);
}
template <typename T>
__global__ void __launch_bounds__(256) grouped_bias_join_kernel(const GroupArgs a, const float* __restrict__ part, int S) {
    const int64_t i = row_block() * 256 + threadIdx.x;
    if (i >= (int64_t)a.E * a.N) return;
    const float* p = part + i / a.N * S * a.N + i % a.N;
    float v = 0.f;
#pragma unroll 16
    for (int s = 0; s < S; ++s) v += p[(int64_t)s * a.N];
    ((T*)a.db)[i] = (T)v;
}
// parts of a group's rows: enough blocks for the chip (four for each CU), no part under 64 rows of an average group
int bias_parts(const spi_grouped_linear_desc& d) {
    const int64_t blocks = ceil_div64(d.N, 64 * (d.dtype == SPI_DTYPE_F32 ? 4 : 8)) * d.E;
    return (int)std::max<int64_t>(1, std::min<int64_t>({ceil_div64(1024, blocks), d.T / d.E / 64, 32}));
}
template <typename T, int VEC>
void bias_grad(const spi_grouped_linear_desc& d, const GroupArgs& a, hipStream_t st) {
    const int S = bias_parts(d);
    hipLaunchKernelGGL((grouped_bias_grad_kernel<T, VEC>), dim3((unsigned)ceil_div64(d.N, 64 * VEC), (unsigned)S, (unsigned)d.E), dim3(256), 0, st, a, (float*)d.workspace, S);
    if (S > 1) hipLaunchKernelGGL(grouped_bias_join_kernel<T>, row_grid(ceil_div64((int64_t)d.E * d.N, 256)), dim3(256), 0, st, a, (const float*)d.workspace, S);
}
template <typename T>
void bias_grad(const spi_grouped_linear_desc& d, const GroupArgs& a, hipStream_t st) {
    if (d.N >= Chunk<T>::N) bias_grad<T, Chunk<T>::N>(d, a, st);
    else bias_grad<T, 1>(d, a, st);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// Edge of the tiles, from the number of tiles that there would be (`rows`(edge) tile rows).  A tile of 256 reads a fourth of what sixteen of 64 do, but a chip half idle costs
// more.  Measured, edges 64 / 128 / 256, us: bf16 forward 2048 x 1024 -> 1024 in 4 groups (144 tiles of 128) 11.5 / 15.6 / 17.0, 8192 x 1024 -> 1024 in 8 (544, 128 of 256)
// 33 / 25 / 34, 16384 x 2048 -> 2048 in 8 (512 of 256) 212 / 147 / 130; int8 4096 x 4096 -> 4096 (256 of 256) 127 / 105 / 95.  Rows that pass through registers pay for 128 later:
// fp32 4099 x 515 -> 771 in 5, weight gradient (175 tiles of 128) 74 / 134, row gradient (170) 58 / 74; bf16 8192 x 1003 -> 501 in 8, forward (272) 29 / 31, weights (256) 31 / 29,
// rows (544) 32 / 25.
// The rule counts tiles, not how full they are: 8192 x 1024 -> 2048 in 24 ragged groups, whose tiles of 256 are a fourth padding, takes 82 us from memory where tiles of 128 take 75
// (from the cache 59 and 62).
struct Tile { int edge, load; };
// rows(edge): tile rows at that edge; smallest: bytes of the smaller operand, from its first value to its tensor's end.  Rows that cannot be copied to LDS as they lie are read 16
// bytes at a time, which takes operands of 16 bytes at least -- whatever the edge, and for a sum over nothing, too: the first step's loads come before the count of steps.
template <typename F>
Tile choose_tile(F rows, int64_t width, bool dma, int64_t smallest) {
    if (!dma && smallest < 16) return Tile{64, LOAD_EACH};
    if (dma && rows(256) * ceil_div64(width, 256) >= CUS) return Tile{256, LOAD_DMA};
    return Tile{rows(128) * ceil_div64(width, 128) >= (dma ? CUS : CUS * 3 / 2) ? 128 : 64, dma ? LOAD_DMA : LOAD_WIDE};
}
Tile choose_int8(const spi_linear_int8_desc& d, const Int8Args& a) {
    // 16-byte rows; where they do not end on 16 bytes, the rows' own padding has to be 0 and the weights' readable
    const bool dma = aligned16(a.q) && aligned16(a.w) && a.q_stride % 16 == 0 && a.w_stride % 16 == 0 &&
                     (d.K % 16 == 0 || (d.x_dtype != SPI_DTYPE_I8 && d.w_bytes >= (d.N - 1) * d.w_stride + q_pitch(d.K)));
    return choose_tile([&](int edge) { return ceil_div64(d.M, edge); }, d.N, dma, std::min((d.M - 1) * a.q_stride, (d.N - 1) * a.w_stride) + d.K);
}
Tile choose_grouped(const spi_grouped_linear_desc& d, int pass) {
    const int64_t es = d.dtype == SPI_DTYPE_F32 ? 4 : 2, xs = d.T * d.K, ws = (int64_t)d.E * d.N * d.K, ds = d.T * d.N;
    const bool dma = d.N * es % 16 == 0 && d.K * es % 16 == 0 && aligned16(d.x) && aligned16(d.w) && aligned16(d.dy);
    const int64_t smallest = (pass == PASS_FWD ? std::min(xs, ws) : pass == PASS_DGRAD ? std::min(ds, ws) : std::min(ds, xs)) * es;
    auto rows = [&](int edge) { return pass == PASS_WGRAD ? ceil_div64(d.N, edge) * d.E : d.T / edge + std::min<int64_t>(d.T, d.E) / 2; };      // (of ragged groups half a tile each is empty)
    return choose_tile(rows, pass == PASS_FWD ? d.N : d.K, dma, smallest);
}
template <typename T, int PASS, int SIZE, int LOAD>
void launch_tiles(const GroupArgs& a, hipStream_t st) {
    const int64_t tiles = PASS == PASS_WGRAD ? ceil_div64(a.N, SIZE) * ceil_div64(a.K, SIZE) * a.E : most_tiles(a.T, a.E, SIZE) * ceil_div64(PASS == PASS_FWD ? a.N : a.K, SIZE);
    hipLaunchKernelGGL((grouped_tile_kernel<T, PASS, SIZE, LOAD>), row_grid(SIZE == 256 ? most_blocks(tiles) : tiles), dim3(SIZE == 256 ? 512 : 256), 0, st, a);
}
template <typename T, int PASS>
void grouped_pass(const GroupArgs& a, Tile t, hipStream_t st) {
    if (t.edge == 256) launch_tiles<T, PASS, 256, LOAD_DMA>(a, st);
    else if (t.edge == 128 && t.load == LOAD_DMA) launch_tiles<T, PASS, 128, LOAD_DMA>(a, st);
    else if (t.edge == 128) launch_tiles<T, PASS, 128, LOAD_WIDE>(a, st);
    else if (t.load == LOAD_DMA) launch_tiles<T, PASS, 64, LOAD_DMA>(a, st);
    else if (t.load == LOAD_WIDE) launch_tiles<T, PASS, 64, LOAD_WIDE>(a, st);
    else launch_tiles<T, PASS, 64, LOAD_EACH>(a, st);
}
template <int PASS>
void grouped_pass(const spi_grouped_linear_desc& d, const GroupArgs& a, hipStream_t st) {
    const Tile t = choose_grouped(d, PASS);
    if (d.dtype == SPI_DTYPE_F32) grouped_pass<float, PASS>(a, t, st);
    else if (d.dtype == SPI_DTYPE_F16) grouped_pass<half_t, PASS>(a, t, st);
    else grouped_pass<bf16_t, PASS>(a, t, st);
}
int check_grouped(const spi_grouped_linear_desc* d, const char* who) {
    SPI_REQUIRE(d, "%s: no descriptor", who);
    SPI_REQUIRE(d->T >= 0 && d->T <= (1ll << 30) && d->E >= 1 && d->E <= 65535 && d->N >= 1 && d->N <= (1 << 20) && d->K >= 1 && d->K <= (1 << 20),
                "%s: T %lld, E %d, N %d, K %d", who, (long long)d->T, d->E, d->N, d->K);
    SPI_REQUIRE((most_tiles(d->T, d->E, 64) * (int64_t)ceil_div64(std::max(d->N, d->K), 64) < (1ll << 31) - 1024) && ceil_div64(d->N, 64) * ceil_div64(d->K, 64) * d->E < (1ll << 31) - 1024,
                "%s: T %lld, E %d, N %d, K %d are more tiles than a launch has blocks", who, (long long)d->T, d->E, d->N, d->K);
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
    if (check_int8(d, "spi_linear_int8_workspace") || d->x_dtype == SPI_DTYPE_I8 || few_floats(*d)) return 0;
    return d->M * (q_pitch(d->K) + (int64_t)sizeof(float));
}
extern "C" int spi_linear_int8_tile(const spi_linear_int8_desc* d) {
    if (int rc = check_int8(d, "spi_linear_int8_tile")) return rc;
    if (d->M == 0 || few_rows(*d)) return 0;
    const Tile t = choose_int8(*d, int8_args(*d));
    return t.edge | t.load << 16;
}
extern "C" int spi_linear_int8(const spi_linear_int8_desc* d, spi_stream_t stream) {
    if (int rc = check_int8(d, "spi_linear_int8")) return rc;
    if (d->M == 0) return SPI_OK;
    SPI_REQUIRE(d->workspace_bytes >= spi_linear_int8_workspace(d) && (d->workspace || d->workspace_bytes == 0), "spi_linear_int8: workspace too small");
    hipStream_t st = as_stream(stream);
    const Int8Args a = int8_args(*d);
    if (few_floats(*d)) {
        if (d->x_dtype == SPI_DTYPE_F32) launch_few<float>(*d, a, d->x, d->x_stride, st);
        else if (d->x_dtype == SPI_DTYPE_F16) launch_few<half_t>(*d, a, d->x, d->x_stride, st);
        else launch_few<bf16_t>(*d, a, d->x, d->x_stride, st);
        SPI_LAUNCH_CHECK("spi_linear_int8");
        return SPI_OK;
    }
    if (d->x_dtype != SPI_DTYPE_I8) {
        quantize_any(d->x, d->M, d->K, d->x_stride, d->x_dtype, (int8_t*)a.q, a.q_stride, (float*)a.q_scale, st);
        SPI_LAUNCH_CHECK("spi_linear_int8 (quantize)");
    }
    if (few_rows(*d)) {
        launch_few<int8_t>(*d, a, a.q, a.q_stride, st);
        SPI_LAUNCH_CHECK("spi_linear_int8");
        return SPI_OK;
    }
    const Tile t = choose_int8(*d, a);
    const int rows = (int)ceil_div64(d->M, t.edge), cols = (int)ceil_div64(d->N, t.edge);
    const dim3 grid = row_grid((int64_t)rows * cols);
    if (t.edge == 256) hipLaunchKernelGGL((int8_tile_kernel<256, LOAD_DMA>), grid, dim3(512), 0, st, a, rows, cols);
    else if (t.edge == 128 && t.load == LOAD_DMA) hipLaunchKernelGGL((int8_tile_kernel<128, LOAD_DMA>), grid, dim3(256), 0, st, a, rows, cols);
    else if (t.edge == 128) hipLaunchKernelGGL((int8_tile_kernel<128, LOAD_WIDE>), grid, dim3(256), 0, st, a, rows, cols);
    else if (t.load == LOAD_DMA) hipLaunchKernelGGL((int8_tile_kernel<64, LOAD_DMA>), grid, dim3(256), 0, st, a, rows, cols);
    else if (t.load == LOAD_WIDE) hipLaunchKernelGGL((int8_tile_kernel<64, LOAD_WIDE>), grid, dim3(256), 0, st, a, rows, cols);
    else hipLaunchKernelGGL((int8_tile_kernel<64, LOAD_EACH>), grid, dim3(256), 0, st, a, rows, cols);
    SPI_LAUNCH_CHECK("spi_linear_int8");
    return SPI_OK;
}

extern "C" int spi_sizeof_grouped_linear_desc(void) { return (int)sizeof(spi_grouped_linear_desc); }
extern "C" int64_t spi_grouped_linear_workspace(const spi_grouped_linear_desc* d, int pass) {
    if (check_grouped(d, "spi_grouped_linear_workspace") || pass != PASS_WGRAD || !d->db) return 0;
    const int S = bias_parts(*d);
    return S > 1 ? (int64_t)d->E * S * d->N * (int64_t)sizeof(float) : 0;
}
extern "C" int spi_grouped_linear_tile(const spi_grouped_linear_desc* d, int pass) {
    if (int rc = check_grouped(d, "spi_grouped_linear_tile")) return rc;
    SPI_REQUIRE(pass >= PASS_FWD && pass <= PASS_WGRAD, "spi_grouped_linear_tile: pass %d", pass);
    if (d->T == 0 && pass != PASS_WGRAD) return 0;
    const Tile t = choose_grouped(*d, pass);
    return t.edge | t.load << 16;
}
extern "C" int spi_grouped_linear_fwd(const spi_grouped_linear_desc* d, spi_stream_t stream) {
    if (int rc = check_grouped(d, "spi_grouped_linear_fwd")) return rc;
    if (d->T == 0) return SPI_OK;
    SPI_REQUIRE(d->x && d->w && d->y, "spi_grouped_linear_fwd: null pointer");
    const GroupArgs a = group_args(*d);
    grouped_pass<PASS_FWD>(*d, a, as_stream(stream));
    SPI_LAUNCH_CHECK("spi_grouped_linear_fwd");
    return SPI_OK;
}
extern "C" int spi_grouped_linear_dgrad(const spi_grouped_linear_desc* d, spi_stream_t stream) {
    if (int rc = check_grouped(d, "spi_grouped_linear_dgrad")) return rc;
    if (d->T == 0) return SPI_OK;
    SPI_REQUIRE(d->dy && d->w && d->dx, "spi_grouped_linear_dgrad: null pointer");
    const GroupArgs a = group_args(*d);
    grouped_pass<PASS_DGRAD>(*d, a, as_stream(stream));
    SPI_LAUNCH_CHECK("spi_grouped_linear_dgrad");
    return SPI_OK;
}
extern "C" int spi_grouped_linear_wgrad(const spi_grouped_linear_desc* d, spi_stream_t stream) {
    if (int rc = check_grouped(d, "spi_grouped_linear_wgrad")) return rc;
    SPI_REQUIRE(d->T == 0 || d->dy, "spi_grouped_linear_wgrad: null dy");
    SPI_REQUIRE(d->T == 0 || !d->dw || d->x, "spi_grouped_linear_wgrad: null x");
    const GroupArgs a = group_args(*d);
    if (d->dw) {
        grouped_pass<PASS_WGRAD>(*d, a, as_stream(stream));
        SPI_LAUNCH_CHECK("spi_grouped_linear_wgrad");
    }
    if (d->db) {
        SPI_REQUIRE(d->workspace_bytes >= spi_grouped_linear_workspace(d, PASS_WGRAD) && (d->workspace || d->workspace_bytes == 0), "spi_grouped_linear_wgrad: workspace too small");
        if (d->dtype == SPI_DTYPE_F32) bias_grad<float>(*d, a, as_stream(stream));
        else if (d->dtype == SPI_DTYPE_F16) bias_grad<half_t>(*d, a, as_stream(stream));
        else bias_grad<bf16_t>(*d, a, as_stream(stream));
        SPI_LAUNCH_CHECK("spi_grouped_linear_wgrad (bias)");
    }
    return SPI_OK;
}
