// Norms before and after a residual block, fused with its gate and residual scale -- forward and backward.
//
//   z = Norm(h) * post_weight + post_bias   (or h: no norm behind the block)
//   s = residual + scale * a(gate) * z      (the residual stream, rounded once to the row type)
//   y = Norm(s) * pre_weight + pre_bias     (for the next block; from the UNROUNDED s), or its rows in 8 bits
//
// Bound by HBM: h and residual in, s and y out, once each.  A row stays in the registers of the threads that loaded it, so both norms' sums run over
// registers; sums are fp32.
#include "typed.hpp"
#include <algorithm>

namespace {

struct NormArgs {
    spi_norm_residual_desc d;
    float inv_width;
};

enum { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_SAMPLE = 2, GATE_FULL = 3 };

// sum over the TPR threads of a row.  `red`: one float per wave of the block, double-buffered by the caller's `phase` so that one barrier suffices.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red, int& phase) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x >> 6, first = wave / W * W;
        float* r = red + (phase & 1) * 16;
        ++phase;
        if ((threadIdx.x & 63) == 0) r[wave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) v += r[first + i];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ float row_max(float v, float* red, int& phase) {
    v = wave_max(v);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x >> 6, first = wave / W * W;
        float* r = red + (phase & 1) * 16;
        ++phase;
        if ((threadIdx.x & 63) == 0) r[wave] = v;
        __syncthreads();
        v = r[first];
#pragma unroll
        for (int i = 1; i < W; ++i) v = fmaxf(v, r[first + i]);
    }
    return v;
}

__device__ __forceinline__ float gate_value(int act, float g) {
    return act == SPI_ACT_TANH ? tanhf(g) : act == SPI_ACT_SIGMOID ? 1.f / (1.f + expf(-g)) : g;
}
__device__ __forceinline__ float gate_slope(int act, float a) {               // through the activation's value
    return act == SPI_ACT_TANH ? 1.f - a * a : act == SPI_ACT_SIGMOID ? a * (1.f - a) : 1.f;
}

__device__ __forceinline__ int64_t gate_at(const spi_norm_residual_desc& d, int64_t row) {
    return d.gate_mode == GATE_FULL ? row * d.width : d.gate_mode == GATE_SAMPLE ? (int64_t)((unsigned)row / (unsigned)d.rows_per_sample) * d.width : 0;     // (rows < 2^31)
}

// mean and 1 / sqrt(mean square + eps) of the row held as x[NV][VEC]; columns outside the row are 0 in x and stay out of the centred sum
template <int TPR, int NV, int VEC>
__device__ __forceinline__ void row_stats(const float (&x)[NV][VEC], const int (&left)[NV], int layer, float inv_width, float eps, float* red, int& phase, float& mean,
                                          float& rstd) {
    mean = 0.f;
    if (layer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += x[i][j];
        mean = row_sum<TPR>(s, red, phase) * inv_width;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float c = j < left[i] ? x[i][j] - mean : 0.f;
            q = fmaf(c, c, q);
        }
    rstd = 1.f / sqrtf(row_sum<TPR>(q, red, phase) * inv_width + eps);
}

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_fwd_kernel(const NormArgs a) {
    constexpr int VEC = Chunk<T>::N, THREADS = TPR > 256 ? TPR : 256, G = THREADS / TPR;
    __shared__ float red[32];
    const spi_norm_residual_desc& d = a.d;
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / TPR;
    const bool live = row < d.rows;                                            // (a dead row still meets every barrier of its block)
    const int64_t base = (live ? row : 0) * d.width;
    int phase = 0, left[NV];
    float s[NV][VEC], r[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c0 = (t + i * TPR) * VEC;
        left[i] = live ? d.width - c0 : 0;
        const Chunk<T> hc = load_chunk((const T*)d.h + base + c0, left[i]);
        const Chunk<T> rc = load_chunk((const T*)d.residual + base + c0, left[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) { s[i][j] = (float)hc.v[j]; r[i][j] = (float)rc.v[j]; }
    }
    float m1 = 0.f, r1 = 1.f;
    if (d.after) row_stats<TPR, NV, VEC>(s, left, d.layer, a.inv_width, d.eps, red, phase, m1, r1);
    const int64_t gbase = d.gate_mode ? gate_at(d, live ? row : 0) : 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c0 = (t + i * TPR) * VEC;
        float w[VEC];
        if (d.after) {
            load_f32(d.post_weight, d.weight_dtype, c0, left[i], w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[i][j] = (s[i][j] - m1) * r1 * w[j];
            if (d.post_bias) {
                load_f32(d.post_bias, d.weight_dtype, c0, left[i], w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[i][j] += w[j];
            }
        }
        if (d.gate_mode) {
            load_f32(d.gate, d.gate_dtype, gbase + c0, left[i], w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[i][j] *= gate_value(d.gate_act, w[j]);
        }
        Chunk<T> out;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            s[i][j] = j < left[i] ? r[i][j] + d.scale * s[i][j] : 0.f;
            out.v[j] = (T)s[i][j];
        }
        store_chunk((T*)d.stream_out + base + c0, out, left[i]);
    }
    float m2 = 0.f, r2 = 1.f;
    if (d.before) {
        row_stats<TPR, NV, VEC>(s, left, d.layer, a.inv_width, d.eps, red, phase, m2, r2);
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c0 = (t + i * TPR) * VEC;
            float w[VEC];
            load_f32(d.pre_weight, d.weight_dtype, c0, left[i], w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[i][j] = (s[i][j] - m2) * r2 * w[j];
            if (d.pre_bias) {
                load_f32(d.pre_bias, d.weight_dtype, c0, left[i], w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[i][j] += w[j];
            }
            if (d.q) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) amax = fmaxf(amax, j < left[i] ? abs_or_inf(s[i][j]) : 0.f);
            } else {
                Chunk<T> out;
#pragma unroll
                for (int j = 0; j < VEC; ++j) out.v[j] = (T)s[i][j];
                store_chunk((T*)d.normed + base + c0, out, left[i]);
            }
        }
        if (d.q) {
            const float scale = row_scale(row_max<TPR>(amax, red, phase));
            if (live && t == 0) d.q_scale[row] = scale;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c0 = (t + i * TPR) * VEC;
                int8_t* p = d.q + (live ? row : 0) * d.q_stride + c0;          // (the padding behind the row is written as 0)
                int8_t v[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = j < left[i] ? (int8_t)quantize_value(s[i][j], scale) : (int8_t)0;
                const int room = live ? (int)d.q_stride - c0 : 0;
                if (room >= VEC) __builtin_memcpy(p, v, VEC);
                else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) if (j < room) p[j] = v[j];
                }
            }
        }
    }
    if (d.stats && live && t == 0) {
        float* p = d.stats + row * 4;
        p[0] = m1; p[1] = r1; p[2] = m2; p[3] = r2;
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------------
// With u = dy * pre_weight, s^ the normalised stream and z, h^ as in the forward:
//   t  = ds + r2 (u - s^ mean(u s^) - mean(u));   d_residual = t;   dz = scale a(gate) t;   d_gate = a'(gate) scale z t
//   v  = dz * post_weight;   d_h = r1 (v - h^ mean(v h^) - mean(v))              (the means of u and v: layer norm only)
// and the column sums  d_pre_weight = sum dy s^,  d_pre_bias = sum dy,  d_post_weight = sum dz h^,  d_post_bias = sum dz,  d_gate of a shared gate.
// A block walks segments of rows (a segment never crosses a sample) and keeps the column sums of its rows in registers; they leave as ONE row of partial
// sums per block, which norm_bwd_reduce_kernel adds in a fixed order: no atomics, the same bits on every run.
constexpr int BT = 512;
enum { SUM_POST_W = 0, SUM_POST_B, SUM_PRE_W, SUM_PRE_B, N_SUMS, SUM_GATE = N_SUMS };

struct NormBwdArgs {
    spi_norm_residual_desc d;
    float inv_width;
    int64_t nseg, seg_rows, segs_per_sample;           // rows of a segment; segments of one sample (the whole batch is one sample unless the gate is per sample)
    int64_t sample_rows;
    float* part;                                       // [grid][sums in use][width], then the gate's [nseg][width]
    float* gate_part;                                  // NULL: segments write d_gate themselves
    int slot[N_SUMS], slots;
};

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(BT) norm_bwd_kernel(const NormBwdArgs a) {
    constexpr int VEC = Chunk<T>::N, G = BT / TPR;
    __shared__ float red[64];
    __shared__ float stage[G > 1 ? G * TPR * NV * VEC : 1];
    const spi_norm_residual_desc& d = a.d;
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    int phase = 0;
    float acc[N_SUMS + 1][NV][VEC];
#pragma unroll
    for (int k = 0; k <= N_SUMS; ++k)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[k][i][j] = 0.f;
    // sum of acc[k] over the block's row groups, in every thread of group 0
    auto over_groups = [&](float (&v)[NV][VEC]) {
        if constexpr (G > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) stage[((g * NV + i) * VEC + j) * TPR + t] = v[i][j];
            __syncthreads();
            if (g == 0)
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        for (int q = 1; q < G; ++q) v[i][j] += stage[((q * NV + i) * VEC + j) * TPR + t];
        }
    };
    for (int64_t seg = blockIdx.x; seg < a.nseg; seg += gridDim.x) {
        const int64_t sample = seg / a.segs_per_sample, row0 = sample * a.sample_rows + (seg % a.segs_per_sample) * a.seg_rows;
        const int64_t row1 = min(min(row0 + a.seg_rows, (sample + 1) * a.sample_rows), d.rows);
        for (int64_t rb = row0; rb < row1; rb += G) {
            const int64_t row = rb + g;
            const bool live = row < row1;
            const int64_t base = (live ? row : row0) * d.width;
            const float* st = d.stats + (live ? row : row0) * 4;
            const float m1 = st[0], r1 = st[1], m2 = st[2], r2 = st[3];
            const int64_t gbase = d.gate_mode ? gate_at(d, live ? row : row0) : 0;
            float hh[NV][VEC], z[NV][VEC], ga[NV][VEC], tt[NV][VEC], sh[NV][VEC], u[NV][VEC];
            int left[NV];
            float sum_us = 0.f, sum_u = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c0 = (t + i * TPR) * VEC;
                left[i] = live ? d.width - c0 : 0;
                const Chunk<T> hc = load_chunk((const T*)d.h + base + c0, left[i]);
                Chunk<T> rc, dsc, dyc;
                if (d.before) rc = load_chunk((const T*)d.residual + base + c0, left[i]);
                if (d.d_stream) dsc = load_chunk((const T*)d.d_stream + base + c0, left[i]);
                if (d.before) dyc = load_chunk((const T*)d.d_normed + base + c0, left[i]);
                float w[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) { hh[i][j] = ((float)hc.v[j] - m1) * r1; z[i][j] = hh[i][j]; ga[i][j] = 1.f; }
                if (d.after) {
                    load_f32(d.post_weight, d.weight_dtype, c0, left[i], w);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) z[i][j] *= w[j];
                    if (d.post_bias) {
                        load_f32(d.post_bias, d.weight_dtype, c0, left[i], w);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) z[i][j] += w[j];
                    }
                }
                if (d.gate_mode) {
                    load_f32(d.gate, d.gate_dtype, gbase + c0, left[i], w);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ga[i][j] = gate_value(d.gate_act, w[j]);
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) tt[i][j] = d.d_stream && j < left[i] ? (float)dsc.v[j] : 0.f;
                if (d.before) {
                    load_f32(d.pre_weight, d.weight_dtype, c0, left[i], w);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float dy = j < left[i] ? (float)dyc.v[j] : 0.f;
                        sh[i][j] = j < left[i] ? ((float)rc.v[j] + d.scale * ga[i][j] * z[i][j] - m2) * r2 : 0.f;
                        acc[SUM_PRE_W][i][j] = fmaf(dy, sh[i][j], acc[SUM_PRE_W][i][j]);
                        acc[SUM_PRE_B][i][j] += dy;
                        u[i][j] = dy * w[j];
                        sum_us = fmaf(u[i][j], sh[i][j], sum_us);
                        sum_u += u[i][j];
                    }
                }
            }
            if (d.before) {
                sum_us = row_sum<TPR>(sum_us, red, phase) * a.inv_width;
                sum_u = d.layer ? row_sum<TPR>(sum_u, red, phase) * a.inv_width : 0.f;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) tt[i][j] += j < left[i] ? r2 * (u[i][j] - sh[i][j] * sum_us - sum_u) : 0.f;
            }
            float sum_vh = 0.f, sum_v = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c0 = (t + i * TPR) * VEC;
                Chunk<T> out;
#pragma unroll
                for (int j = 0; j < VEC; ++j) out.v[j] = (T)tt[i][j];
                if (d.d_residual) store_chunk((T*)d.d_residual + base + c0, out, left[i]);
                float w[VEC];
                if (d.after) load_f32(d.post_weight, d.weight_dtype, c0, left[i], w);
                float dg[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    dg[j] = j < left[i] ? gate_slope(d.gate_act, ga[i][j]) * d.scale * z[i][j] * tt[i][j] : 0.f;
                    const float dz = d.scale * ga[i][j] * tt[i][j];
                    u[i][j] = dz;
                    if (d.after) {
                        const float hv = j < left[i] ? hh[i][j] : 0.f;
                        acc[SUM_POST_W][i][j] = fmaf(dz, hv, acc[SUM_POST_W][i][j]);
                        acc[SUM_POST_B][i][j] += dz;
                        u[i][j] = dz * w[j];
                        sum_vh = fmaf(u[i][j], hv, sum_vh);
                        sum_v += u[i][j];
                    }
                }
                if (d.gate_mode == GATE_FULL) {
                    if (d.d_gate)
#pragma unroll
                        for (int j = 0; j < VEC; ++j) if (j < left[i]) store_f32(d.d_gate, d.gate_dtype, base + c0 + j, dg[j]);
                } else if (d.gate_mode) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[SUM_GATE][i][j] += dg[j];
                }
            }
            if (d.after) {
                sum_vh = row_sum<TPR>(sum_vh, red, phase) * a.inv_width;
                sum_v = d.layer ? row_sum<TPR>(sum_v, red, phase) * a.inv_width : 0.f;
            }
            if (d.d_h)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c0 = (t + i * TPR) * VEC;
                    Chunk<T> out;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) out.v[j] = (T)(d.after ? r1 * (u[i][j] - hh[i][j] * sum_vh - sum_v) : u[i][j]);
                    store_chunk((T*)d.d_h + base + c0, out, left[i]);
                }
        }
        if (d.d_gate && (d.gate_mode == GATE_CHANNEL || d.gate_mode == GATE_SAMPLE)) {
            over_groups(acc[SUM_GATE]);
            if (g == 0)
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int c = (t + i * TPR) * VEC + j;
                        if (c >= d.width) continue;
                        if (a.gate_part) a.gate_part[seg * d.width + c] = acc[SUM_GATE][i][j];
                        else store_f32(d.d_gate, d.gate_dtype, sample * d.width + c, acc[SUM_GATE][i][j]);
                    }
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[SUM_GATE][i][j] = 0.f;
        }
    }
#pragma unroll
    for (int k = 0; k < N_SUMS; ++k) {
        if (a.slot[k] < 0) continue;
        over_groups(acc[k]);
        if (g == 0)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int c = (t + i * TPR) * VEC + j;
                    if (c < d.width) a.part[((int64_t)blockIdx.x * a.slots + a.slot[k]) * d.width + c] = acc[k][i][j];
                }
    }
}

// out[v][c] = sum_p part[v * v_stride + p * p_stride + c], four rows of partial sums per column in flight, added in a fixed order
struct ReduceJob { const float* part; void* out; int dtype; int64_t v_stride, p_stride, parts, vectors; };
struct ReduceArgs { ReduceJob job[N_SUMS + 1]; int64_t first[N_SUMS + 2]; int jobs, width, cols; };
__global__ void __launch_bounds__(256) norm_bwd_reduce_kernel(const ReduceArgs a) {
    __shared__ float s[4][64];
    int j = 0;
    while (j + 1 < a.jobs && (int64_t)blockIdx.x >= a.first[j + 1]) ++j;
    const ReduceJob& q = a.job[j];
    const int64_t b = blockIdx.x - a.first[j], v = b / a.cols;
    const int c = (int)(b % a.cols) * 64 + (threadIdx.x & 63), r = threadIdx.x >> 6;
    float x = 0.f;
    if (c < a.width)
        for (int64_t p = r; p < q.parts; p += 4) x += q.part[v * q.v_stride + p * q.p_stride + c];
    s[r][threadIdx.x & 63] = x;
    __syncthreads();
    if (r == 0 && c < a.width) store_f32(q.out, q.dtype, v * a.width + c, (s[0][threadIdx.x] + s[1][threadIdx.x]) + (s[2][threadIdx.x] + s[3][threadIdx.x]));
}

struct BwdPlan { int64_t nseg, seg_rows, segs_per_sample, sample_rows, samples; int grid, tpr; bool gate_reduce; };

// threads of a row in the backward: eight values each, sixteen over 4096 (so that five column sums of a thread's columns stay in its registers)
int bwd_tpr(int width) { return width <= 512 ? 64 : width <= 2048 ? 256 : 512; }

BwdPlan bwd_plan(const spi_norm_residual_desc& d) {
    BwdPlan p;
    p.tpr = bwd_tpr(d.width);
    const int G = BT / p.tpr;
    p.sample_rows = d.gate_mode == GATE_SAMPLE ? d.rows_per_sample : d.rows;
    p.samples = p.sample_rows ? d.rows / p.sample_rows : 0;
    const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(1, p.samples));              // segments of a sample: two blocks for every CU
    p.segs_per_sample = std::max<int64_t>(1, std::min(want, ceil_div64(p.sample_rows, G)));
    p.seg_rows = ceil_div64(ceil_div64(p.sample_rows, p.segs_per_sample), G) * G;
    p.segs_per_sample = std::max<int64_t>(1, ceil_div64(p.sample_rows, p.seg_rows ? p.seg_rows : 1));
    p.nseg = p.samples * p.segs_per_sample;
    p.grid = (int)std::min<int64_t>(p.nseg, 512);
    p.gate_reduce = d.d_gate && (d.gate_mode == GATE_CHANNEL || d.gate_mode == GATE_SAMPLE) && p.segs_per_sample > 1;
    return p;
}

int sums_in_use(const spi_norm_residual_desc& d, int (&slot)[N_SUMS]) {
    int n = 0;
    slot[SUM_POST_W] = d.d_post_weight ? n++ : -1;
    slot[SUM_POST_B] = d.d_post_bias ? n++ : -1;
    slot[SUM_PRE_W] = d.d_pre_weight ? n++ : -1;
    slot[SUM_PRE_B] = d.d_pre_bias ? n++ : -1;
    return n;
}

int check_desc(const spi_norm_residual_desc* d, const char* who) {
    SPI_REQUIRE(d, "%s: no descriptor", who);
    SPI_REQUIRE(d->rows >= 0 && d->width >= 1 && d->width <= SPI_NORM_MAX_WIDTH, "%s: rows %lld, width %d (1 .. %d)", who, (long long)d->rows, d->width, SPI_NORM_MAX_WIDTH);
    SPI_REQUIRE(d->rows < (1ll << 31), "%s: %lld rows", who, (long long)d->rows);
    SPI_REQUIRE(d->dtype == SPI_DTYPE_F32 || d->dtype == SPI_DTYPE_F16 || d->dtype == SPI_DTYPE_BF16, "%s: dtype %d", who, d->dtype);
    auto param_ok = [&](int t) { return t == SPI_DTYPE_F32 || t == d->dtype; };
    SPI_REQUIRE(param_ok(d->weight_dtype) && param_ok(d->gate_dtype), "%s: weights / gate are fp32 or of the rows' type", who);
    SPI_REQUIRE(d->h && d->residual, "%s: null rows", who);
    SPI_REQUIRE(d->after || d->before, "%s: no norm", who);
    SPI_REQUIRE(d->gate_mode >= GATE_NONE && d->gate_mode <= GATE_FULL && (d->gate_mode == GATE_NONE) == (d->gate == nullptr), "%s: gate and gate_mode disagree", who);
    SPI_REQUIRE(d->gate_mode != GATE_SAMPLE || (d->rows_per_sample >= 1 && d->rows % d->rows_per_sample == 0), "%s: rows_per_sample %lld", who, (long long)d->rows_per_sample);
    SPI_REQUIRE(d->gate_act == SPI_ACT_LINEAR || d->gate_act == SPI_ACT_TANH || d->gate_act == SPI_ACT_SIGMOID, "%s: gate_act %d", who, d->gate_act);
    SPI_REQUIRE(!d->after || d->post_weight, "%s: null post_weight", who);
    SPI_REQUIRE(!d->before || d->pre_weight, "%s: null pre_weight", who);
    SPI_REQUIRE(d->eps > 0.f, "%s: eps %g", who, (double)d->eps);
    return SPI_OK;
}

template <typename T, int TPR, int NV>
void launch_fwd(const NormArgs& a, hipStream_t st) {
    constexpr int THREADS = TPR > 256 ? TPR : 256;
    hipLaunchKernelGGL((norm_fwd_kernel<T, TPR, NV>), dim3((unsigned)ceil_div64(a.d.rows, THREADS / TPR)), dim3(THREADS), 0, st, a);
}
template <typename T>
void dispatch_fwd(const NormArgs& a, hipStream_t st) {
    const int chunks = (int)ceil_div64(a.d.width, Chunk<T>::N);
    if (chunks <= 64) launch_fwd<T, 64, 1>(a, st);
    else if (chunks <= 128) launch_fwd<T, 64, 2>(a, st);
    else if (chunks <= 256) launch_fwd<T, 256, 1>(a, st);
    else if (chunks <= 512) launch_fwd<T, 256, 2>(a, st);
    else if (chunks <= 1024) launch_fwd<T, 256, 4>(a, st);
    else if (chunks <= 2048) launch_fwd<T, 1024, 2>(a, st);
    else if (sizeof(T) < 4 || chunks <= 4096) launch_fwd<T, 1024, 4>(a, st);       // (SPI_NORM_MAX_WIDTH is 4096 chunks of eight)
    else if constexpr (sizeof(T) == 4) launch_fwd<T, 1024, 8>(a, st);
}
template <typename T>
void dispatch_bwd(const NormBwdArgs& a, const BwdPlan& p, hipStream_t st) {
    constexpr int NV = 8 / Chunk<T>::N;
    if (p.tpr == 64) hipLaunchKernelGGL((norm_bwd_kernel<T, 64, NV>), dim3(p.grid), dim3(BT), 0, st, a);
    else if (p.tpr == 256) hipLaunchKernelGGL((norm_bwd_kernel<T, 256, NV>), dim3(p.grid), dim3(BT), 0, st, a);
    else if (a.d.width <= 4096) hipLaunchKernelGGL((norm_bwd_kernel<T, 512, NV>), dim3(p.grid), dim3(BT), 0, st, a);
    else hipLaunchKernelGGL((norm_bwd_kernel<T, 512, 2 * NV>), dim3(p.grid), dim3(BT), 0, st, a);
}

}  // namespace

extern "C" int spi_norm_residual_fwd(const spi_norm_residual_desc* d, spi_stream_t stream) {
    if (int rc = check_desc(d, "spi_norm_residual_fwd")) return rc;
    SPI_REQUIRE(d->stream_out, "spi_norm_residual_fwd: null stream_out");
    SPI_REQUIRE(!d->before || (d->q ? (d->q_scale && d->q_stride >= d->width) : d->normed != nullptr), "spi_norm_residual_fwd: no place for the normed rows");
    // (a row's threads cover at least its chunks: the padding that they write as 0 ends with the last chunk, at most 15 bytes behind the row)
    SPI_REQUIRE(!d->q || d->q_stride <= ceil_div64(d->width, 16) * 16, "spi_norm_residual_fwd: q_stride %lld", (long long)d->q_stride);
    if (d->rows == 0) return SPI_OK;
    const NormArgs a{*d, 1.f / (float)d->width};
    if (d->dtype == SPI_DTYPE_F32) dispatch_fwd<float>(a, as_stream(stream));
    else if (d->dtype == SPI_DTYPE_F16) dispatch_fwd<half_t>(a, as_stream(stream));
    else dispatch_fwd<bf16_t>(a, as_stream(stream));
    SPI_LAUNCH_CHECK("spi_norm_residual_fwd");
    return SPI_OK;
}

extern "C" int64_t spi_norm_residual_bwd_workspace(const spi_norm_residual_desc* d) {
    if (check_desc(d, "spi_norm_residual_bwd_workspace") || d->rows == 0) return 0;
    const BwdPlan p = bwd_plan(*d);
    int slot[N_SUMS];
    return ((int64_t)p.grid * sums_in_use(*d, slot) + (p.gate_reduce ? p.nseg : 0)) * d->width * (int64_t)sizeof(float);
}

extern "C" int spi_norm_residual_bwd(const spi_norm_residual_desc* d, spi_stream_t stream) {
    if (int rc = check_desc(d, "spi_norm_residual_bwd")) return rc;
    SPI_REQUIRE(d->width <= SPI_NORM_MAX_WIDTH_BWD, "spi_norm_residual_bwd: width %d (1 .. %d)", d->width, SPI_NORM_MAX_WIDTH_BWD);
    SPI_REQUIRE(d->stats, "spi_norm_residual_bwd: null stats");
    SPI_REQUIRE(!d->before || d->d_normed, "spi_norm_residual_bwd: null d_normed");
    SPI_REQUIRE(d->after || !(d->d_post_weight || d->d_post_bias), "spi_norm_residual_bwd: gradients of a norm that is not there");
    SPI_REQUIRE(d->before || !(d->d_pre_weight || d->d_pre_bias), "spi_norm_residual_bwd: gradients of a norm that is not there");
    SPI_REQUIRE(d->workspace_bytes >= spi_norm_residual_bwd_workspace(d) && (d->workspace || d->workspace_bytes == 0), "spi_norm_residual_bwd: workspace too small");
    SPI_REQUIRE(d->rows > 0, "spi_norm_residual_bwd: no rows");
    const BwdPlan p = bwd_plan(*d);
    NormBwdArgs a;
    a.d = *d;
    a.inv_width = 1.f / (float)d->width;
    a.nseg = p.nseg; a.seg_rows = p.seg_rows; a.segs_per_sample = p.segs_per_sample; a.sample_rows = p.sample_rows;
    a.slots = sums_in_use(*d, a.slot);
    a.part = (float*)d->workspace;
    a.gate_part = p.gate_reduce ? a.part + (int64_t)p.grid * a.slots * d->width : nullptr;
    hipStream_t st = as_stream(stream);
    if (d->dtype == SPI_DTYPE_F32) dispatch_bwd<float>(a, p, st);
    else if (d->dtype == SPI_DTYPE_F16) dispatch_bwd<half_t>(a, p, st);
    else dispatch_bwd<bf16_t>(a, p, st);
    SPI_LAUNCH_CHECK("spi_norm_residual_bwd");
    ReduceArgs r;
    r.jobs = 0; r.width = d->width; r.cols = (int)ceil_div64(d->width, 64); r.first[0] = 0;
    auto add = [&](const float* part, void* out, int dtype, int64_t v_stride, int64_t p_stride, int64_t parts, int64_t vectors) {
        r.job[r.jobs] = ReduceJob{part, out, dtype, v_stride, p_stride, parts, vectors};
        r.first[r.jobs + 1] = r.first[r.jobs] + vectors * r.cols;
        ++r.jobs;
    };
    void* outs[N_SUMS] = {d->d_post_weight, d->d_post_bias, d->d_pre_weight, d->d_pre_bias};
    for (int k = 0; k < N_SUMS; ++k)
        if (outs[k]) add(a.part + (int64_t)a.slot[k] * d->width, outs[k], d->weight_dtype, 0, (int64_t)a.slots * d->width, p.grid, 1);
    if (p.gate_reduce) add(a.gate_part, d->d_gate, d->gate_dtype, p.segs_per_sample * d->width, d->width, p.segs_per_sample, p.samples);
    if (r.jobs) {
        hipLaunchKernelGGL(norm_bwd_reduce_kernel, dim3((unsigned)r.first[r.jobs]), dim3(256), 0, st, r);
        SPI_LAUNCH_CHECK("spi_norm_residual_bwd (sums)");
    }
    return SPI_OK;
}

extern "C" int spi_sizeof_norm_residual_desc(void) { return (int)sizeof(spi_norm_residual_desc); }
