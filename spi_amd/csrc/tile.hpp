// Matrix-core tiles for products of rows (linear.hip): C[i, j] = sum_k A(i, k) B(j, k) over BM x BN values, GM x GN waves, for int8, fp16, bf16 and fp32.
//
// Both operands enter v_mfma_*_32x32x* as 16-byte chunks along the summed axis, so one engine serves every type: a step takes 128 bytes of that axis (128
// int8, 64 halves, 32 floats).  An operand lies in memory with the summed axis adjacent (`row`: x W^T) or with the tile's own axis adjacent (`col`: the gradients); both are
// copied memory -> LDS as they lie, and `col` tiles are transposed on the way from LDS to registers (ds_read_b64_tr_b16, or one float at a time).
#pragma once
#include "typed.hpp"

#ifdef __HIPCC__
// lane l holds 16 bytes of row (l & 31), half (l >> 5) of a 32-byte step; result register r of lane l: row 8 (r >> 2) + 4 (l >> 5) + (r & 3) of A, row (l & 31) of B
template <typename T> struct Mma;
template <> struct Mma<half_t> {
    typedef f32x16_acc Acc;
    typedef half_t V __attribute__((ext_vector_type(8)));
    static constexpr int N = 1;
    static __device__ __forceinline__ Acc step(i32x4_t a, i32x4_t b, Acc c, int) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <> struct Mma<bf16_t> {
    typedef f32x16_acc Acc;
    typedef bf16_t V __attribute__((ext_vector_type(8)));
    static constexpr int N = 1;
    static __device__ __forceinline__ Acc step(i32x4_t a, i32x4_t b, Acc c, int) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <> struct Mma<float> {                                 // N = 4 steps of two: value q of both halves' chunks
    typedef f32x16_acc Acc;
    typedef float V __attribute__((ext_vector_type(4)));
    static constexpr int N = 4;
    static __device__ __forceinline__ Acc step(i32x4_t a, i32x4_t b, Acc c, int q) {
        return __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(V, a)[q], __builtin_bit_cast(V, b)[q], c, 0, 0, 0);      // (whole vectors: a bit cast of a[q] reads a[0])
    }
};
template <> struct Mma<int8_t> {
    typedef i32x16_acc Acc;
    static constexpr int N = 1;
    static __device__ __forceinline__ Acc step(i32x4_t a, i32x4_t b, Acc c, int) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ unsigned lds_offset(char* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)p; }
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// One operand of a tile.  p: its first value; pitch: bytes between neighbours on the axis that is not adjacent; k: values of the summed axis; n: valid values of the
// tile's own axis; bytes: what may be read from p on (row: n * pitch; col: k * pitch less the bytes of a row before p).  256 * pitch < 2^31.
// Summed values behind k are 0 in the tile.  Rows (`row`) or columns (`col`) behind n may hold what follows in memory, or 0: they only reach results that lie outside, too.
// end: bytes from p to the end of the tensor that the operand is part of.
struct TileOperand { const char* p; int64_t pitch, bytes, k; int n; int64_t end; };

// row: which chunk a tile row's chunks are XORed with, so that 16 rows' chunks c fall on all of the 64 banks (and eight rows' on 32)
__device__ __forceinline__ int row_swizzle(int r) { return (r & 7) ^ ((r >> 3) & 1); }

// How a stage is filled.
//   LOAD_DMA   memory -> LDS without registers: rows that begin on 16 bytes and (row) hold a whole number of 16-byte chunks; reads outside are answered with 0 by the buffer's
//              bounds check
//   LOAD_WIDE  through registers (`fetch` before a step's products, `put` behind them), 16 bytes at a time at any alignment, without a condition -- a load under a condition
//              would be waited for at once.  A chunk that would pass the tensor's end is read from its last 16 bytes and moved into place by `put`, which also clears what lies
//              behind the summed axis
//              behind the summed axis.  The tensor has 16 bytes at least
//   LOAD_EACH  value by value where a tensor has less than 16 bytes, or none
enum { LOAD_DMA = SPI_TILE_COPY, LOAD_WIDE = SPI_TILE_WIDE, LOAD_EACH = SPI_TILE_EACH };
template <typename T, int R, int NW, bool COL, int LOAD>
struct TileLoader {
    static constexpr int ES = (int)sizeof(T), KT = 128 / ES, PER = R / 8 / NW, ROW = COL ? R * ES : 128, RPI = 1024 / ROW, CHUNKS = ROW / 16;
    static_assert(R % (8 * NW) == 0 && NW % 2 == 0 && ROW <= 1024, "a wave copies 1024 bytes at a time");
    const char* base;
    int64_t pitch, left, k;                   // left: bytes from `base` to the operand's (LOAD_WIDE: the tensor's) end; k: values of the summed axis still to come
    int n;
    unsigned voff[PER];
    i32x4_t hold[LOAD == LOAD_DMA ? 1 : PER];
    int moved[LOAD == LOAD_WIDE ? PER : 1];   // bytes by which a held chunk was read too early

    // col: where the chunks of summed row kr lie; keeps the 8 rows x 64 bytes of a transposing read (16-bit) and the two 128-byte halves of a float read apart
    static __device__ __forceinline__ int swizzle(int kr) {
        if constexpr (ES == 4) return ((kr >> 2) & 1) * 8 % CHUNKS;
        else return (((kr & 3) | ((kr >> 3) & 1) << 2) * 4) % CHUNKS;
    }
    // copy i of this thread: chunk c of row r of the stage (row: r a tile row; col: r a summed row)
    static __device__ __forceinline__ void place(int i, int& r, int& c) {
        const int lane = threadIdx.x & 63, at = (threadIdx.x >> 6) + i * NW;
        r = at * RPI + lane / CHUNKS;
        c = (lane % CHUNKS) ^ (COL ? swizzle(r) : row_swizzle(r));
    }
    __device__ __forceinline__ void init(const TileOperand& o) {
        base = o.p; pitch = o.pitch; k = o.k; n = o.n; left = LOAD == LOAD_WIDE ? o.end : o.bytes;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int r, c;
            place(i, r, c);
            voff[i] = (unsigned)(r * (int)pitch + c * 16);
        }
    }
    // starts the copies of the next step (DMA: into `stage`, R * 128 bytes)
    __device__ __forceinline__ void fetch(char* stage) {
        if constexpr (LOAD == LOAD_DMA) {
            const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
            const int64_t most = (int64_t)(COL ? KT : R) * pitch;
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(base, left > 0 ? (left < most ? left : most) : 0);
            int r, c;
            place(0, r, c);                                       // (row: every copy of a thread has the same chunk, an even number of copies apart)
            const bool whole = COL || k >= KT || c * 16 < (int)k * ES;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(stage + (wave + i * NW) * 1024), 16, whole ? voff[i] : BUF_OOB, 0, 0, 0);
        } else if constexpr (LOAD == LOAD_WIDE) {
            const int last = (int)max(min(left - 16, (int64_t)0x7fffffff), -(int64_t)0x7fffffff);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int at = min((int)voff[i], last);
                moved[i] = (int)voff[i] - at;
                hold[i] = __builtin_bit_cast(i32x4_t, load_all<char, 16>(base + at));
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                int r, c;
                place(i, r, c);
                const int64_t valid = COL ? (r < k ? n - c * (16 / ES) : 0) : (r < n ? k - c * (16 / ES) : 0);
                hold[i] = __builtin_bit_cast(i32x4_t, load_chunk((const T*)(base + (valid > 0 ? voff[i] : 0u)), valid > 0 ? (int)(valid < 16 ? valid : 16) : 0));
            }
        }
        const int64_t step = COL ? KT * pitch : 128;
        base += step;
        left -= step;
        k -= KT;
    }
    __device__ __forceinline__ void put(char* stage) {
        if constexpr (LOAD != LOAD_DMA)
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if constexpr (LOAD == LOAD_WIDE) {
                    int r, c;
                    place(i, r, c);
                    const int64_t before = k + KT, valid = COL ? (r < before ? 16 : 0) : (before - c * (16 / ES)) * ES;      // bytes of the chunk on the summed axis
                    if (moved[i] | (valid < 16)) {
                        typedef unsigned __int128 u128;
                        u128 v = __builtin_bit_cast(u128, hold[i]);
                        v = moved[i] < 16 ? v >> (moved[i] * 8) : (u128)0;
                        if (valid < 16) v &= valid > 0 ? ((u128)1 << (int)(valid * 8)) - 1 : (u128)0;
                        hold[i] = __builtin_bit_cast(i32x4_t, v);
                    }
                }
                *reinterpret_cast<i32x4_t*>(stage + ((threadIdx.x >> 6) + i * NW) * 1024 + (threadIdx.x & 63) * 16) = hold[i];
            }
    }
};

// fragments of 32 tile rows from a stage
template <typename T, int R, bool COL, int F>
struct TileReader {
    int at[F];                                // row: at[0] (the step's chunk is XORed in), col: one per fragment
    int key;
    __device__ __forceinline__ void init(int first) {
        const int l = threadIdx.x & 63;
        if constexpr (!COL) {
            at[0] = (first + (l & 31)) * 128;
            key = row_swizzle(l) << 4;
        } else if constexpr (sizeof(T) == 2) {
            constexpr int CHUNKS = R * 2 / 16;
            const int q = l >> 4, j = l & 15, row = (q >> 1) * 8 + (j >> 2), swz = (((j >> 2) | (q >> 1) << 2) * 4) % CHUNKS;
#pragma unroll
            for (int f = 0; f < F; ++f) at[f] = row * R * 2 + ((((first + f * 32) / 8 + (q & 1) * 2 + ((j & 3) >> 1)) ^ swz) << 4) + (j & 1) * 8;
        } else {
            const int h = l >> 5, c = l & 31, swz = h * 8 % (R * 4 / 16);
#pragma unroll
            for (int f = 0; f < F; ++f) at[f] = h * 4 * R * 4 + ((((first + f * 32 + c) / 4) ^ swz) << 4) + (c & 3) * 4;
        }
    }
    __device__ __forceinline__ i32x4_t read(const char* stage, int f, int kk) const {
        if constexpr (!COL) {
            const int half = (threadIdx.x & 63) >> 5;
            return *reinterpret_cast<const i32x4_t*>(stage + at[0] + f * 4096 + ((((kk * 2 + half) << 4)) ^ key));
        } else if constexpr (sizeof(T) == 2) {
            const char* p = stage + at[f] + kk * 16 * R * 2;
            const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p));
            const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p + 4 * R * 2));
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(i32x4_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            typedef float f32x4 __attribute__((ext_vector_type(4)));
            const char* p = stage + at[f] + kk * 8 * R * 4;
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float*>(p + j * R * 4);
            return __builtin_bit_cast(i32x4_t, v);
        }
    }
};

// Two stages of LDS: the copies of step k + 1 are under way while step k is multiplied, one barrier a step.  (16384 x 2048 x 2048 bf16 at 256 x 256, both sides on one card: 132 us; four
// stages of 64 bytes of the summed axis, 143: half cache lines, and the latency is already covered.)
template <typename T, int BM_, int BN_, int GM_, int GN_, bool COLA, bool COLB, int LOAD>
struct TileEngine {
    static constexpr int BM = BM_, BN = BN_, GM = GM_, GN = GN_, NW = GM * GN, WM = BM / GM, WN = BN / GN, FM = WM / 32, FN = WN / 32, KT = 128 / (int)sizeof(T),
                         STAGE = (BM + BN) * 128;
    typedef typename Mma<T>::Acc Acc;
    typedef Acc Accs[FM][FN];

    // s0, s1: LDS arrays of their own (the compiler then knows that the copies into one do not touch the reads of the other)
    static __device__ __forceinline__ void run(const TileOperand& a, const TileOperand& b, char* s0, char* s1, Accs& acc) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        TileLoader<T, BM, NW, COLA, LOAD> la;
        TileLoader<T, BN, NW, COLB, LOAD> lb;
        TileReader<T, BM, COLA, FM> ra;
        TileReader<T, BN, COLB, FN> rb;
        la.init(a);
        lb.init(b);
        ra.init(wave / GN * WM);
        rb.init(wave % GN * WN);
        const int steps = (int)((a.k + KT - 1) / KT);
        auto fetch = [&](char* to) { la.fetch(to); lb.fetch(to + BM * 128); };
        auto put = [&](char* to) { la.put(to); lb.put(to + BM * 128); };
        // the fragments of part kk + 1 are read while part kk is multiplied; the copies of the next step start behind the first fragments' reads
        auto multiply = [&](const char* from, char* next) {
            i32x4_t fa[2][FM], fb[2][FN];
            auto read = [&](int kk) {
#pragma unroll
                for (int i = 0; i < FM; ++i) fa[kk & 1][i] = ra.read(from, i, kk);
#pragma unroll
                for (int j = 0; j < FN; ++j) fb[kk & 1][j] = rb.read(from + BM * 128, j, kk);
            };
            read(0);
            __builtin_amdgcn_sched_barrier(0);
            fetch(next);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                if (kk < 3) read(kk + 1);
                __builtin_amdgcn_sched_barrier(0);               // (the compiler would put these reads behind the products, and then wait for them)
#pragma unroll
                for (int q = 0; q < Mma<T>::N; ++q)              // (the steps of one accumulator apart: each waits for the one before it)
#pragma unroll
                    for (int i = 0; i < FM; ++i)
#pragma unroll
                        for (int j = 0; j < FN; ++j) acc[i][j] = Mma<T>::step(fa[kk & 1][i], fb[kk & 1][j], acc[i][j], q);
                __builtin_amdgcn_sched_barrier(0);               // (else the compiler reads all parts first, and spills)
            }
        };
        // behind the barrier a stage is whole (it waits for this wave's copies, too) and nobody reads the other one any more; copies behind the last step read nothing
        auto step = [&](char* now, char* next) {
            __syncthreads();
            multiply(now, next);
            put(next);
        };
        fetch(s0);
        put(s0);
        int k = 0;
        for (; k + 2 <= steps; k += 2) {
            step(s0, s1);
            step(s1, s0);
        }
        if (k < steps) step(s0, s1);
        __syncthreads();                                         // every copy has landed and every stage has been read: the caller may use the LDS
    }
    // f(i, j, v): four values (i, j .. j + 3) at a time, for all of the tile.  Each wave turns its accumulators around in LDS (half of the waves in each stage), 32
    // rows at a time, so that a row's values leave in one piece; the loop stays rolled, whatever f does.
    template <typename F>
    static __device__ __forceinline__ void each(const Accs& acc, char* s0, char* s1, F f) {
        typedef decltype(Acc{}[0] + Acc{}[0]) V;
        typedef V V4 __attribute__((ext_vector_type(4)));
        constexpr int PITCH = WN + 4;                            // (16-byte rows; the rows of the two halves of a wave fall on different banks)
        static_assert(NW / 2 * 32 * PITCH * 4 <= STAGE, "half of the waves' slabs fit a stage");
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m0 = wave / GN * WM, n0 = wave % GN * WN;
        // (chosen as LDS offsets: a choice of generic pointers would turn the accesses into flat ones)
        const unsigned room = wave < NW / 2 ? lds_offset(s0) : lds_offset(s1);
        typedef __attribute__((address_space(3))) V lds_V;
        typedef __attribute__((address_space(3))) V4 lds_V4;
        lds_V* slab = (lds_V*)(uintptr_t)(room + wave % (NW / 2) * 32 * PITCH * 4);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) slab[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * PITCH + j * 32 + (lane & 31)] = acc[i][j][r];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int q = lane; q < 32 * WN / 4; q += 64) {
                const int row = q / (WN / 4), col = q % (WN / 4) * 4;
                f(m0 + i * 32 + row, n0 + col, *(const lds_V4*)(slab + row * PITCH + col));
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
};

// Block b of `total` blocks -> its place in an order in which each of the eight XCDs (blocks go to them in turn) works on one run of neighbours, whose operands
// then meet in that XCD's L2
__device__ __forceinline__ int xcd_run(int b, int total) {
    const int per = total / 8, more = total % 8, x = b % 8;
    return x * per + min(x, more) + b / 8;
}
// place t of rows x cols tiles -> (row, col): bands of 8 rows, a band column by column
__device__ __forceinline__ void band_order(int t, int rows, int cols, int& row, int& col) {
    const int band = t / (8 * cols), in = t - band * 8 * cols, high = min(8, rows - band * 8);
    row = band * 8 + in % high;
    col = in / high;
}
#endif
