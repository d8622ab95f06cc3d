// Norms before and after a residual block, fused with its gate and residual scale -- forward and backward.
//
//   z = Norm(h) * post_weight + post_bias   (or h: no norm behind the block)
//   s = residual + scale * a(gate) * z      (the residual stream, rounded once to the row type)
//   y = Norm(s) * pre_weight + pre_bias     (for the next block; from the UNROUNDED s), or its rows in 8 bits
//
// Bound by HBM: h and residual in, s and y out, once each (4 x 4096 x 2048 bf16: 74 us = 3.6 TB/s, where a copy of 1 GiB reaches 5.2).  A row stays in the
// registers of the threads that loaded it, so both norms' sums run over registers; sums are fp32 (a row whose squares pass the fp32 range has a deviation of
// infinity, and is normalised to 0).
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

// mean and 1 / sqrt(mean square + eps) of the row held as x[NV][VEC]; columns that are not this thread's are 0 in x and stay out of the centred sum
template <int TPR, int NV, int VEC, bool LAYER>
__device__ __forceinline__ void row_stats(const float (&x)[NV][VEC], const int (&first)[NV], float inv_width, float eps, float* red, int& phase, float& mean, float& rstd) {
    mean = 0.f;
    if (LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += x[i][j];
        mean = row_sum<TPR>(s, red, phase) * inv_width;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float c[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) c[j] = x[i][j] - mean;
        if (LAYER) mask_first(c, first[i], 0.f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) q = fmaf(c[j], c[j], q);
    }
    rstd = 1.f / sqrtf(row_sum<TPR>(q, red, phase) * inv_width + eps);
}

// One row in TPR threads, NV chunks of VEC values each.
template <typename T, int VEC, int TPR, int NV, bool LAYER>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_fwd_kernel(const NormArgs a) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, G = THREADS / TPR;
    __shared__ float red[32];
    const spi_norm_residual_desc& d = a.d;
    const int t = threadIdx.x % TPR;
    const int64_t row_at = row_block() * G + threadIdx.x / TPR;
    const bool live = row_at < d.rows;                                         // (a dead row meets every barrier of its block, with another row's values)
    const int64_t row = live ? row_at : d.rows - 1, base = row * d.width, gbase = d.gate_mode ? gate_at(d, row) : 0;
    int phase = 0, at[NV], first[NV];
    // (the gate and the weights are read where they are used.  4 x 4096 x 2048 bf16: 72 us; read ahead with the rows, 80: the registers cost rows under way.  Held in registers
    //  while a block walks several rows, 69 -- but 8 x 600 x 1024 fp16 15.6 instead of 13.4, and fp32 3 x 667 x 1003 13.7 instead of 12.8.)
    Chunk<T, VEC> hc[NV], rc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const Columns c = columns<VEC>(t + i * TPR, d.width);
        at[i] = c.start;
        first[i] = c.first;
        hc[i] = load_all<T, VEC>((const T*)d.h + base + c.start);
        rc[i] = load_all<T, VEC>((const T*)d.residual + base + c.start);
    }
    float s[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) widen(hc[i], first[i], s[i]);
    float m1 = 0.f, r1 = 1.f;
    if (d.after) row_stats<TPR, NV, VEC, LAYER>(s, first, a.inv_width, d.eps, red, phase, m1, r1);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float w[VEC], r[VEC];
        if (d.after) {
            load_f32(d.post_weight, d.weight_dtype, at[i], w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[i][j] = (s[i][j] - (LAYER ? m1 : 0.f)) * r1 * w[j];
            if (d.post_bias) {
                load_f32(d.post_bias, d.weight_dtype, at[i], w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[i][j] += w[j];
            }
        }
        if (d.gate_mode) {
            load_f32(d.gate, d.gate_dtype, gbase + at[i], w);
            if (d.gate_act != SPI_ACT_LINEAR)
#pragma unroll
                for (int j = 0; j < VEC; ++j) w[j] = gate_value(d.gate_act, w[j]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[i][j] *= w[j];
        }
        widen(rc[i], 0, r);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[i][j] = fmaf(d.scale, s[i][j], r[j]);
        mask_first(s[i], first[i], 0.f);
        if (live && first[i] < VEC) store_columns((T*)d.stream_out + base + at[i], s[i], first[i]);
    }
    float m2 = 0.f, r2 = 1.f;
    if (d.before) {
        row_stats<TPR, NV, VEC, LAYER>(s, first, a.inv_width, d.eps, red, phase, m2, r2);
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float w[VEC];
            load_f32(d.pre_weight, d.weight_dtype, at[i], w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[i][j] = (s[i][j] - (LAYER ? m2 : 0.f)) * r2 * w[j];
            if (d.pre_bias) {
                load_f32(d.pre_bias, d.weight_dtype, at[i], w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[i][j] += w[j];
            }
            if (d.q) {
                mask_first(s[i], first[i], 0.f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) amax = fmaxf(amax, abs_or_inf(s[i][j]));
            } else if (live && first[i] < VEC) store_columns((T*)d.normed + base + at[i], s[i], first[i]);
        }
        if (d.q) {
            const float scale = row_scale(row_max<TPR>(amax, red, phase));
            const float inverse = 1.f / scale;
            int8_t* q = d.q + row * d.q_stride;
            if (live) {
                if (t == 0) d.q_scale[row] = scale;
                if (t < d.q_stride - d.width) q[d.width + t] = 0;              // the padding (less than 16 bytes)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const Chunk<int8_t, VEC> v = quantize_values(s[i], scale, inverse);
                    if (first[i] <= 0) __builtin_memcpy(q + at[i], &v, VEC);
                    else if (first[i] < VEC)
#pragma unroll
                        for (int j = 0; j < VEC; ++j) if (j >= first[i]) q[at[i] + j] = v.v[j];
                }
            }
        }
    }
    if (d.stats && live && t == 0) {
        const f32x4_t v = {m1, r1, m2, r2};
        *reinterpret_cast<f32x4_t*>(d.stats + row * 4) = v;
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
    int64_t nseg, segs_per_sample;                     // segments of one sample (the whole batch is one sample unless the gate is per sample)
    int64_t sample_rows;
    float* part;                                       // [grid][sums in use][width], then the gate's [nseg][width]
    float* gate_part;                                  // NULL: segments write d_gate themselves
    int slot[N_SUMS], slots;
};

// two sums over a row's threads behind one barrier
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red, int& phase) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x >> 6, first = wave / W * W;
        float* r = red + (phase & 1) * 32;
        ++phase;
        if ((threadIdx.x & 63) == 0) { r[wave] = a; r[16 + wave] = b; }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) { a += r[first + i]; b += r[16 + first + i]; }
    }
}

// Bound by HBM (h, residual, ds, dy in; d_h, d_residual out) as far as enough of it is under way: a block holds few rows, so the next row's values are on their way while a
// row is worked on, in loads without a condition (a load under one is waited for at once).  4 x 4096 x 2048 bf16: 109 us = 3.7 TB/s.  (When it was
// chosen, on one card: 105; 139 with conditional loads, with or without the sums between the threads; 184 without the next row.)
template <typename T, int VEC, int TPR, int NV, bool LAYER>
__global__ void __launch_bounds__(TPR > BT ? TPR : BT, TPR > BT ? 4 : sizeof(T) == 4 && NV == 1 ? 3 : 2) norm_bwd_kernel(const NormBwdArgs a) {
    constexpr int G = TPR > BT ? 1 : BT / TPR;
    constexpr bool AHEAD = NV == 1;                    // the next row is on its way (wide rows leave no registers for it)
    typedef Chunk<T, VEC> Values;
    __shared__ float red[64];
    __shared__ float stage[G > 1 ? G * TPR * NV * VEC : 1];
    const spi_norm_residual_desc& d = a.d;
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const bool full = d.gate_mode == GATE_FULL, bent = d.gate_act != SPI_ACT_LINEAR;
    int phase = 0;
    float acc[N_SUMS + 1][NV][VEC], pw[NV][VEC], qw[NV][VEC], ga[NV][VEC];
    int at[NV], first[NV];                             // this thread's columns
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const Columns c = columns<VEC>(t + i * TPR, d.width);
        at[i] = c.start;
        first[i] = c.first;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
#pragma unroll
            for (int k = 0; k <= N_SUMS; ++k) acc[k][i][j] = 0.f;
            pw[i][j] = qw[i][j] = ga[i][j] = 1.f;
        }
        if (d.after) load_f32(d.post_weight, d.weight_dtype, at[i], pw[i]);
        if (d.before) load_f32(d.pre_weight, d.weight_dtype, at[i], qw[i]);
    }
    // the sum of v over the block's row groups, in every thread of group 0
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
        // G rows at a time, all segments of a sample side by side, so that the blocks together read one run of memory (blocks that each kept to rows of their own, 128 KB
        // apart: 4 % slower)
        const int64_t sample = seg / a.segs_per_sample, row0 = sample * a.sample_rows + seg % a.segs_per_sample * G, row1 = (sample + 1) * a.sample_rows;
        const int64_t stride = a.segs_per_sample * G;
        if (d.gate_mode && !full) {
            const int64_t gbase = gate_at(d, row0);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                load_f32(d.gate, d.gate_dtype, gbase + at[i], ga[i]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) ga[i][j] = bent ? gate_value(d.gate_act, ga[i][j]) : ga[i][j];
            }
        }
        struct Row { Values h[NV], r[NV], s[NV], y[NV]; Raw<VEC> g[NV]; f32x4_t st; } in;
        auto fetch = [&](int64_t row) {
            const int64_t from = row < row1 ? row : row0, base = from * d.width;
            in.st = *reinterpret_cast<const f32x4_t*>(d.stats + from * 4);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                in.h[i] = load_all<T, VEC>((const T*)d.h + base + at[i]);
                if (d.before) {
                    in.r[i] = load_all<T, VEC>((const T*)d.residual + base + at[i]);
                    in.y[i] = load_all<T, VEC>((const T*)d.d_normed + base + at[i]);
                }
                if (d.d_stream) in.s[i] = load_all<T, VEC>((const T*)d.d_stream + base + at[i]);
                if (full) in.g[i] = load_raw<VEC>(d.gate, d.gate_dtype, base + at[i]);
            }
        };
        if (AHEAD) fetch(row0 + g);
        for (int64_t rb = row0; rb < row1; rb += stride) {
            const int64_t row = rb + g, base = row * d.width;
            const bool live = row < row1;
            if (!AHEAD) fetch(row);
            // Columns of others, and all of a dead row, are taken as 0 (a dead row's statistics, too): their u, t and dz are 0 and add nothing to any sum; only the layer
            // norm's means reach them.
            const float m1 = live ? in.st[0] : 0.f, r1 = live ? in.st[1] : 0.f, m2 = live ? in.st[2] : 0.f, r2 = live ? in.st[3] : 0.f;
            float hh[NV][VEC], z[NV][VEC], tt[NV][VEC], sh[NV][VEC], u[NV][VEC];
            int skip[NV];
            float sum_us = 0.f, sum_u = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                skip[i] = live ? first[i] : VEC;
                float x[VEC];
                widen(in.h[i], skip[i], x);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { hh[i][j] = (x[j] - (LAYER ? m1 : 0.f)) * r1; z[i][j] = hh[i][j] * pw[i][j]; }
                if (d.post_bias) {
                    float w[VEC];
                    load_f32(d.post_bias, d.weight_dtype, at[i], w);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) z[i][j] += w[j];
                }
                if (full) {
                    widen<VEC>(in.g[i], d.gate_dtype, ga[i]);
                    if (bent)
#pragma unroll
                        for (int j = 0; j < VEC; ++j) ga[i][j] = gate_value(d.gate_act, ga[i][j]);
                }
                if (d.d_stream) widen(in.s[i], skip[i], tt[i]);
                else
#pragma unroll
                    for (int j = 0; j < VEC; ++j) tt[i][j] = 0.f;
                if (d.before) {
                    float dy[VEC];
                    widen(in.r[i], skip[i], x);
                    widen(in.y[i], skip[i], dy);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        sh[i][j] = (fmaf(d.scale * ga[i][j], z[i][j], x[j]) - (LAYER ? m2 : 0.f)) * r2;
                        acc[SUM_PRE_W][i][j] = fmaf(dy[j], sh[i][j], acc[SUM_PRE_W][i][j]);
                        u[i][j] = dy[j] * qw[i][j];
                        sum_us = fmaf(u[i][j], sh[i][j], sum_us);
                        if (LAYER) sum_u += u[i][j];
                    }
                    if (d.d_pre_bias)
#pragma unroll
                        for (int j = 0; j < VEC; ++j) acc[SUM_PRE_B][i][j] += dy[j];
                }
            }
            if (AHEAD && rb + stride < row1) fetch(row + stride);      // (the same for the whole block)
            if (d.before) {
                if (LAYER) row_sum2<TPR>(sum_us, sum_u, red, phase);
                else sum_us = row_sum<TPR>(sum_us, red, phase);
                sum_us *= a.inv_width;
                sum_u *= a.inv_width;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        if (LAYER) tt[i][j] += j >= skip[i] ? r2 * (fmaf(-sh[i][j], sum_us, u[i][j]) - sum_u) : 0.f;
                        else tt[i][j] = fmaf(r2, fmaf(-sh[i][j], sum_us, u[i][j]), tt[i][j]);
                    }
            }
            float sum_vh = 0.f, sum_v = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (d.d_residual && skip[i] < VEC) store_columns((T*)d.d_residual + base + at[i], tt[i], skip[i]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    tt[i][j] *= d.scale;
                    const float dz = ga[i][j] * tt[i][j];
                    u[i][j] = dz;
                    if (d.after) {
                        acc[SUM_POST_W][i][j] = fmaf(dz, hh[i][j], acc[SUM_POST_W][i][j]);
                        u[i][j] = dz * pw[i][j];
                        sum_vh = fmaf(u[i][j], hh[i][j], sum_vh);
                        if (LAYER) sum_v += u[i][j];
                    }
                }
                if (d.d_post_bias)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[SUM_POST_B][i][j] = fmaf(ga[i][j], tt[i][j], acc[SUM_POST_B][i][j]);
                if (d.d_gate) {
                    float dg[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) dg[j] = z[i][j] * tt[i][j];
                    if (bent)
#pragma unroll
                        for (int j = 0; j < VEC; ++j) dg[j] *= gate_slope(d.gate_act, ga[i][j]);
                    if (full) {
                        if (skip[i] < VEC) store_columns<VEC>(d.d_gate, d.gate_dtype, base + at[i], dg, skip[i]);
                    } else
#pragma unroll
                        for (int j = 0; j < VEC; ++j) acc[SUM_GATE][i][j] += dg[j];
                }
            }
            if (d.after) {
                if (LAYER) row_sum2<TPR>(sum_vh, sum_v, red, phase);
                else sum_vh = row_sum<TPR>(sum_vh, red, phase);
                sum_vh *= a.inv_width;
                sum_v *= a.inv_width;
            }
            if (d.d_h)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (d.after)
#pragma unroll
                        for (int j = 0; j < VEC; ++j) u[i][j] = r1 * (fmaf(-hh[i][j], sum_vh, u[i][j]) - sum_v);
                    if (skip[i] < VEC) store_columns((T*)d.d_h + base + at[i], u[i], skip[i]);
                }
        }
        if (d.d_gate && (d.gate_mode == GATE_CHANNEL || d.gate_mode == GATE_SAMPLE)) {
            over_groups(acc[SUM_GATE]);
            if (g == 0)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (first[i] >= VEC) continue;
                    if (a.gate_part) store_columns(a.gate_part + seg * d.width + at[i], acc[SUM_GATE][i], first[i]);
                    else store_columns<VEC>(d.d_gate, d.gate_dtype, sample * d.width + at[i], acc[SUM_GATE][i], first[i]);
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
                if (first[i] < VEC) store_columns(a.part + ((int64_t)blockIdx.x * a.slots + a.slot[k]) * d.width + at[i], acc[k][i], first[i]);
    }
}

// out[v][c] = sum_p part[v * v_stride + p * p_stride + c]: 16 chains of partial sums for each column, eight loads of each in flight, joined in a fixed order
struct ReduceJob { const float* part; void* out; int dtype; int64_t v_stride, p_stride, parts, vectors; };
struct ReduceArgs { ReduceJob job[N_SUMS + 1]; int64_t first[N_SUMS + 2]; int jobs, width, cols; };
__global__ void __launch_bounds__(1024) norm_bwd_reduce_kernel(const ReduceArgs a) {
    __shared__ float s[16][64];
    int j = 0;
    while (j + 1 < a.jobs && (int64_t)blockIdx.x >= a.first[j + 1]) ++j;
    const ReduceJob& q = a.job[j];
    const int64_t b = blockIdx.x - a.first[j], v = b / a.cols;
    const int c = (int)(b % a.cols) * 64 + (threadIdx.x & 63), r = threadIdx.x >> 6;
    float x = 0.f;
    if (c < a.width) {
        const float* p = q.part + v * q.v_stride + c;
#pragma unroll 8
        for (int64_t i = r; i < q.parts; i += 16) x += p[i * q.p_stride];
    }
    s[r][threadIdx.x & 63] = x;
    __syncthreads();
    if (r || c >= a.width) return;
    for (int i = 1; i < 16; ++i) x += s[i][threadIdx.x];
    store_f32(q.out, q.dtype, v * a.width + c, x);
}

struct BwdPlan { int64_t nseg, segs_per_sample, sample_rows, samples; int grid, tpr; bool wide, gate_reduce; };

// threads of a row in the backward
int bwd_tpr(int chunks, bool wide) { return chunks <= 64 ? 64 : chunks <= 256 ? 256 : chunks <= 512 || wide ? 512 : 1024; }

BwdPlan bwd_plan(const spi_norm_residual_desc& d) {
    BwdPlan p;
    const int chunks = (int)ceil_div64(d.width, d.dtype == SPI_DTYPE_F32 ? 4 : 8);
    p.wide = d.width > 4096;                           // sixteen values a thread
    p.tpr = bwd_tpr(chunks, p.wide);
    const int G = std::max(1, BT / p.tpr);
    p.sample_rows = d.gate_mode == GATE_SAMPLE ? d.rows_per_sample : d.rows;
    p.samples = p.sample_rows ? d.rows / p.sample_rows : 0;
    const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(1, p.samples));              // segments of a sample: two blocks for every CU
    p.segs_per_sample = std::max<int64_t>(1, std::min(want, ceil_div64(p.sample_rows, G)));
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
    SPI_REQUIRE(d->gate_mode >= GATE_NONE && d->gate_mode <= GATE_FULL && (d->gate_mode == GATE_NONE) == (d->gate == nullptr), "%s: gate and gate_mode disagree", who);
    SPI_REQUIRE(d->gate_mode != GATE_SAMPLE || (d->rows_per_sample >= 1 && d->rows % d->rows_per_sample == 0), "%s: rows_per_sample %lld", who, (long long)d->rows_per_sample);
    SPI_REQUIRE(d->gate_act == SPI_ACT_LINEAR || d->gate_act == SPI_ACT_TANH || d->gate_act == SPI_ACT_SIGMOID, "%s: gate_act %d", who, d->gate_act);
    SPI_REQUIRE(!d->after || d->post_weight, "%s: null post_weight", who);
    SPI_REQUIRE(!d->before || d->pre_weight, "%s: null pre_weight", who);
    SPI_REQUIRE(d->eps > 0.f, "%s: eps %g", who, (double)d->eps);
    SPI_REQUIRE(((uintptr_t)d->stats & 15) == 0, "%s: stats do not begin on 16 bytes", who);
    return SPI_OK;
}

template <typename T, int VEC, int TPR, int NV>
void launch_fwd(const NormArgs& a, hipStream_t st) {
    constexpr int THREADS = TPR > 256 ? TPR : 256;
    const dim3 grid = row_grid(ceil_div64(a.d.rows, THREADS / TPR));
    if (a.d.layer) hipLaunchKernelGGL((norm_fwd_kernel<T, VEC, TPR, NV, true>), grid, dim3(THREADS), 0, st, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, VEC, TPR, NV, false>), grid, dim3(THREADS), 0, st, a);
}
// One chunk a thread as far as a block goes: the latency of a row is what few rows cost, and many rows hide it either way.  One chunk / two in half the threads:
// 1 x 512 fp32 3.1 / 3.8 us, 8 x 600 x 1024 fp16 13.7 / 14.3, 2 x 4096 bf16 4.1 / 4.8, 4000 x 4096 bf16 35.8 / 36.1; two / four: 1 x 8000 fp16 6.5 / 9.2,
// 2000 x 8000 40.3 / 40.4.
template <typename T>
void dispatch_fwd(const NormArgs& a, hipStream_t st) {
    constexpr int N = Chunk<T>::N;
    const int chunks = (int)ceil_div64(a.d.width, N);
    if (a.d.width < N) launch_fwd<T, 1, 64, 1>(a, st);
    else if (chunks <= 64) launch_fwd<T, N, 64, 1>(a, st);
    else if (chunks <= 128) launch_fwd<T, N, 128, 1>(a, st);
    else if (chunks <= 256) launch_fwd<T, N, 256, 1>(a, st);
    else if (chunks <= 512) launch_fwd<T, N, 512, 1>(a, st);
    else if (chunks <= 1024) launch_fwd<T, N, 512, 2>(a, st);
    else if (chunks <= 2048) launch_fwd<T, N, 1024, 2>(a, st);
    else if (sizeof(T) < 4 || chunks <= 4096) launch_fwd<T, N, 1024, 4>(a, st);       // (SPI_NORM_MAX_WIDTH is 4096 chunks of eight)
    else if constexpr (sizeof(T) == 4) launch_fwd<T, N, 1024, 8>(a, st);
}
template <typename T, int VEC, int TPR, int NV>
void launch_bwd(const NormBwdArgs& a, int grid, hipStream_t st) {
    const dim3 block(TPR > BT ? TPR : BT);
    if (a.d.layer) hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, TPR, NV, true>), dim3(grid), block, 0, st, a);
    else hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, TPR, NV, false>), dim3(grid), block, 0, st, a);
}
template <typename T>
void dispatch_bwd(const NormBwdArgs& a, const BwdPlan& p, hipStream_t st) {
    constexpr int N = Chunk<T>::N;
    if (a.d.width < N) launch_bwd<T, 1, 64, 1>(a, p.grid, st);
    else if (p.wide) launch_bwd<T, N, 512, 16 / N>(a, p.grid, st);
    else if (p.tpr == 64) launch_bwd<T, N, 64, 1>(a, p.grid, st);
    else if (p.tpr == 256) launch_bwd<T, N, 256, 1>(a, p.grid, st);
    else if (p.tpr == 512) launch_bwd<T, N, 512, 1>(a, p.grid, st);
    else if constexpr (sizeof(T) == 4) launch_bwd<T, N, 1024, 1>(a, p.grid, st);
}

}  // namespace

extern "C" int spi_norm_residual_fwd(const spi_norm_residual_desc* d, spi_stream_t stream) {
    if (int rc = check_desc(d, "spi_norm_residual_fwd")) return rc;
    SPI_REQUIRE(d->after || d->before, "spi_norm_residual_fwd: no norm");
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
    a.nseg = p.nseg; a.segs_per_sample = p.segs_per_sample; a.sample_rows = p.sample_rows;
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
        hipLaunchKernelGGL(norm_bwd_reduce_kernel, dim3((unsigned)r.first[r.jobs]), dim3(1024), 0, st, r);
        SPI_LAUNCH_CHECK("spi_norm_residual_bwd (sums)");
    }
    return SPI_OK;
}

extern "C" int spi_sizeof_norm_residual_desc(void) { return (int)sizeof(spi_norm_residual_desc); }
