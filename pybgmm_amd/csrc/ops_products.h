// Products of rows with the matrix of their own component (include/bgmm_ops.h): shared by the four element types.
//
//   rows      out[p] = in[src(p)] W_e (+ b_e) for the rows p of component e           forward, and the rows' gradient
//   weight    dW_e = sum over the rows of e of g_p in[src(p)] (x) d[dst(p)], db_e      the weights' gradient
//   combine   sums over a row's k components and over split contractions
//   gates     dg_p = in[src(p)] . (W_e d[p]) + b_e . d[p]: the first part falls off the rows' gradient, whose tiles hold W_e d[p]
//
// Tiles.  A workgroup of four waves owns a tile of one component's rows (found in the grouping's prefix sums) times a tile of
// the other axis and walks the contraction in steps of 128 bytes per row: 64 half, 32 single or 16 double precision elements,
// so that all four types share one tile geometry.  A 16-byte LDS read is a lane's operand for one 16x16x32 (half), four
// 16x16x4 (single) or two 16x16x4 (double) matrix instructions: where an instruction takes fewer elements than a lane has
// read, its k-th element is not the k-th of the row but the same permutation holds for both operands, which a sum does
// not see.  The weights are the instruction's row operand and the data rows its columns: a lane then holds four consecutive
// elements of one output row (two pairs in double precision), which go to LDS as one vector and from there to memory by rows.
//
// LDS layouts (both without bank conflicts on the operand reads, by XOR on the 16-byte granule):
//   KTile: rows along the contraction, [row][8 granules], granule ^ (row & 7); read 16 bytes per lane.
//   MTile: contraction outermost, [k][width], for an operand whose contiguous axis is not the contraction; half precision
//   goes through the transposing LDS read (16 lanes read 4 x 16 elements, each gets a column of 4), the wider types are read
//   element by element (their matrix instructions take 32 and 64 cycles, the reads hide behind them).
#pragma once
#include "ops_common.h"

typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

union Granule {                 // 16 bytes of any element type
    v4i raw;
    v4s half[2];
    double d[2];
    float f[4];
    f16_t h[8];
    bf16_t b[8];
    v8h vh;
    v8b vb;
};
template <class T> struct Elems;
template <> struct Elems<double> { static __device__ double *of(Granule &g) { return g.d; } };
template <> struct Elems<float> { static __device__ float *of(Granule &g) { return g.f; } };
template <> struct Elems<f16_t> { static __device__ f16_t *of(Granule &g) { return g.h; } };
template <> struct Elems<bf16_t> { static __device__ bf16_t *of(Granule &g) { return g.b; } };

// The matrix instructions of one granule of each operand: kParts of them, each on a part of the granules.  A kernel runs part
// s of all its accumulators before part s + 1 of any, so that no instruction waits for the one in front of it.
template <class T> constexpr int kParts = sizeof(T) == 8 ? 2 : sizeof(T) == 4 ? 4 : 1;
template <class T> __device__ __forceinline__ void mma(typename Acc<T>::v4 &c, const Granule &a, const Granule &b, int s);
template <> __device__ __forceinline__ void mma<double>(v4d &c, const Granule &a, const Granule &b, int s) {
    c = __builtin_amdgcn_mfma_f64_16x16x4f64(a.d[s], b.d[s], c, 0, 0, 0);
}
template <> __device__ __forceinline__ void mma<float>(v4f &c, const Granule &a, const Granule &b, int s) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.f[s], b.f[s], c, 0, 0, 0);
}
template <> __device__ __forceinline__ void mma<f16_t>(v4f &c, const Granule &a, const Granule &b, int) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.vh, b.vh, c, 0, 0, 0);
}
template <> __device__ __forceinline__ void mma<bf16_t>(v4f &c, const Granule &a, const Granule &b, int) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.vb, b.vb, c, 0, 0, 0);
}

constexpr int kStepBytes = 128;                                  // of the contraction per step and row
template <class T> constexpr int kStep = kStepBytes / (int)sizeof(T);
template <class T> constexpr int kGran = 16 / (int)sizeof(T);    // elements per granule

// Column (or row) of a 16-wide block that the matrix instruction's index r stands for, so that what a lane stores at once is
// 16 consecutive bytes and the four lanes of a row 64: the double-precision instruction gives lane l rows l / 16 + 4 i, the
// others rows 4 (l / 16) + i.  result_col: the block's column of a lane's result i.
template <class T> __device__ __forceinline__ int result_row(int r) { return r; }
template <> __device__ __forceinline__ int result_row<double>(int r) { return (r >> 3) * 8 + (r & 3) * 2 + ((r >> 2) & 1); }
template <class T> __device__ __forceinline__ int result_col(int q, int i) { return q * 4 + i; }
template <> __device__ __forceinline__ int result_col<double>(int q, int i) { return (i >> 1) * 8 + q * 2 + (i & 1); }

template <class T> struct KTile {
    static __device__ __forceinline__ int at(int row, int granule) { return row * kStepBytes + ((granule ^ (row & 7)) << 4); }
    // rows block .. block + 15, half-step ks of the contraction
    template <bool RESULT> static __device__ __forceinline__ Granule read(const char *tile, int block, int ks) {
        const int l = wave_lane(), r = RESULT ? result_row<T>(l & 15) : (l & 15);
        Granule g;
        g.raw = *(const v4i *)(tile + at(block + r, ks * 4 + (l >> 4)));
        return g;
    }
};

template <class T, int WIDTH> struct MTile {
    static constexpr int kPitch = WIDTH * (int)sizeof(T), kPerRow = kPitch / 16;
    static __device__ __forceinline__ int spread(int k) {
        if (sizeof(T) == 2) return (((k & 3) | ((k >> 1) & 4)) << 1) & (kPerRow - 1);
        if (sizeof(T) == 4) return (((k >> 2) & 3) << 2) & (kPerRow - 1);
        return (((k >> 1) & 1) << 3) & (kPerRow - 1);
    }
    static __device__ __forceinline__ int at(int k, int granule) { return k * kPitch + ((granule ^ spread(k)) << 4); }
    template <bool RESULT> static __device__ __forceinline__ Granule read(const char *tile, int block, int ks) {
        const int l = wave_lane(), r = RESULT ? result_row<T>(l & 15) : (l & 15), q = l >> 4;
        Granule g;
        if constexpr (sizeof(T) == 2) {
            const int col = block + (r & 3) * 4;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = ks * 32 + q * 8 + h * 4 + (r >> 2);
                g.half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) v4s *)(tile + at(k, col >> 3) + (col & 7) * 2));
            }
        } else if constexpr (sizeof(T) == 4) {
            const int col = block + r;
#pragma unroll
            for (int s = 0; s < 4; ++s) g.f[s] = *(const float *)(tile + at(ks * 16 + q * 4 + s, col >> 2) + (col & 3) * 4);
        } else {
            const int col = block + r;
#pragma unroll
            for (int s = 0; s < 2; ++s) g.d[s] = *(const double *)(tile + at(ks * 8 + q * 2 + s, col >> 1) + (col & 1) * 8);
        }
        return g;
    }
};

// 16 bytes at p, at whatever alignment its elements have
template <class T> __device__ __forceinline__ Granule load_whole(const T *p) {
    Granule g;
    g.raw = load_any<v4i>(p);
    return g;
}
// 16 bytes at p of which the first `avail` elements exist; the rest become zero
template <class T> __device__ __forceinline__ Granule load_part(const T *p, int avail) {
    Granule g;
    g.raw = (v4i){0, 0, 0, 0};
    if (avail >= kGran<T>) {
        g = load_whole(p);
    } else {
        T *e = Elems<T>::of(g);
#pragma unroll
        for (int j = 0; j < kGran<T>; ++j)
            if (j < avail) e[j] = p[j];
    }
    return g;
}

// elements `avail` and behind zeroed
template <class T> __device__ __forceinline__ void keep(Granule &g, int avail) {
    T *e = Elems<T>::of(g);
#pragma unroll
    for (int j = 0; j < kGran<T>; ++j) e[j] = j < avail ? e[j] : (T)0.0f;
}

// n / d for n < 2^31 by one multiplication: (n m) >> s with m = floor(2^s / d) + 1, s = 31 + ceil(log2 d).  The error
// n (m - 2^s / d) / 2^s is below n / 2^s <= 1 / d, so the quotient is exact.
struct Divisor {
    unsigned m;
    int s;
};
__device__ __forceinline__ int divide(int n, Divisor d) { return (int)(((unsigned long long)(unsigned)n * d.m) >> d.s); }

// Workgroups go round the eight dies in turn: number them so that a die gets runs of consecutive work, whose operands its own L2
// then holds.  A permutation of 0 .. blocks - 1 (a multiple of 8 * run) that needs no load; first: of a launch's part of them, such a
// multiple too.
__device__ __forceinline__ int die_order(int run, int first) {
    const int b = first + blockIdx.x, die = b & 7, at = b >> 3;
    return (at / run * 8 + die) * run + at % run;
}

struct RowsArgs {
    const int4 *tiles;              // the grouping's
    const int *order;
    int K, tile_blocks, run;        // blocks of eight tiles, consecutive workgroups on a die
    int first;                      // of a launch's workgroups
    const void *in;                 // row src = p / in_div of `in`
    i64 in_stride;
    Divisor in_div;
    const void *w;                  // W_e[k][n] at e * w_component + k * w_row + n, or [n][k] at ... + n * w_row + k
    i64 w_component, w_row;
    const void *bias;               // [K][n], row stride bias_row, or null
    i64 bias_row;
    const void *gates;              // accumulator type, [P], or null
    void *out;                      // element type, row p at p * out_stride
    i64 out_stride;
    void *ws;                       // or, instead of out: accumulator type, [splits][P][n], neither gated nor rounded
    const void *dot_in;             // with dots: row p / dot_div, ndim elements
    i64 dot_stride;
    Divisor dot_div;
    void *dots;                     // accumulator type, [P][n_dots]: the parts of dot_in . u_p, ungated; or null
    int n_dots;
    i64 P;
    int kdim, ndim, splits, n_tiles;
    int in_safe;                    // rows of `in` in front of this have 16 bytes from any of their elements on
    int w_safe;                     // rows of a component's matrix likewise (along w_row)
};

struct WeightArgs {
    const int *bucket_first;        // prefix sums for chunks of `chunk` rows
    const int *offsets, *order;
    int K, level, run, first;       // (run, first: as above)
    const void *in;                 // row p / in_div
    i64 in_stride;
    Divisor in_div;
    const void *d;                  // row p / d_div
    i64 d_stride;
    Divisor d_div;
    int in_safe, d_safe;            // rows in front of this have 16 bytes from any of their elements on
    const void *gates;
    void *dw, *db;                  // element type, [K][idim][odim] and [K][odim] (db may be null; dw too)
    void *ws;                       // accumulator type: a slot of idim * odim + odim per chunk of a component with several
    int idim, odim, i_tiles, o_tiles;
};

struct CombineArgs {
    const int *bucket;              // [rows * k]
    int K, k, splits;
    i64 rows, P;
    i64 first;                      // (of a launch's rows)
    const void *ws;                 // [splits][P][dim]
    const void *gates;              // [rows * k] or null
    void *out;                      // [rows], stride out_stride
    i64 out_stride;
    int dim;
    // the gates' gradient (null: none): in . u + bias . d
    void *dgates;
    const void *in;
    i64 in_stride;
    const void *bias;
    i64 bias_row;
    const void *d;
    i64 d_stride;
    int d_div, ddim;
};

struct GatesArgs {
    const int *bucket;              // [P]
    int K, n_dots;
    i64 P;
    const void *dots;               // accumulator type, [P][n_dots]
    const void *bias;               // [K], row stride bias_row, or null
    i64 bias_row;
    const void *d;                  // with bias: row p / d_div, ddim elements
    i64 d_stride;
    Divisor d_div;
    int ddim;
    void *dgates;                   // accumulator type, [P]
};

// One product with rows; bm x bn: its tiles (16 x 128, 128 x 16, 32, 64 or 128).  `kcontig`: the weights' contiguous axis is the
// contraction.  The weights' gradient by tiles of bi x bo (16, 64 or 128 each, but not 16 x 64 nor 64 x 16).
template <class T> int launch_rows(const RowsArgs &a, bool kcontig, int bm, int bn, i64 blocks, hipStream_t st);
template <class T> int launch_weight(const WeightArgs &a, int bi, int bo, i64 blocks, hipStream_t st);
template <class T> int launch_combine(const CombineArgs &a, hipStream_t st);
template <class T> int launch_gates(const GatesArgs &a, hipStream_t st);
