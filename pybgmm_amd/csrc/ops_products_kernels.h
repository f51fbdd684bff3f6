// The kernels behind ops_products.h, instantiated once per element type (ops_products_{f64,f32,f16,bf16}.hip).
#pragma once
#include "ops_products.h"

// Consecutive elements of an output row from accumulators, as one store where all of them exist (at any alignment).
template <int N, class T, class V> __device__ __forceinline__ void store_run(T *p, const V &v, int from, int avail) {
    struct Run { T e[N]; } o;
#pragma unroll
    for (int i = 0; i < N; ++i) o.e[i] = (T)v[from + i];
    if (avail >= N) {
        store_any(p, o);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < avail) p[i] = o.e[i];
    }
}

// N elements of a row as accumulators, at any alignment; behind the row's end zeros.
template <int N, class S, class A> __device__ __forceinline__ void load_few(const S *p, int avail, A (&v)[N]) {
    if (avail >= N) {
        struct Few { S e[N]; };
        const Few f = load_any<Few>(p);
#pragma unroll
        for (int x = 0; x < N; ++x) v[x] = (A)f.e[x];
    } else {
#pragma unroll
        for (int x = 0; x < N; ++x) v[x] = x < avail ? (A)p[x] : (A)0;
    }
}
template <class S, class A> __device__ __forceinline__ void load4(const S *p, int avail, A (&v)[4]) { load_few<4>(p, avail, v); }

// Waves per SIMD.  The loads of the next step fly in registers while the LDS buffer is in use, one buffer and two barriers a
// step instead of two and one: that a third workgroup fits a compute unit covers more latency (and the other two's
// beginnings and ends) than a second buffer or a second step in flight (N = 1e6, D = 64 double: 316 -> 295 us; 64 experts of
// 1024 x 2048, bfloat16: 197 -> 174 and 163 -> 134 us).
template <class T, int TILE> constexpr int kWavesPerSimd = TILE >= 128 * 128 ? (sizeof(T) == 8 ? 2 : 3) : sizeof(T) == 8 && TILE >= 128 * 64 ? 3 : 4;

// A tile's results leave through LDS, so that a row's are one stretch of memory per store instruction: straight from the
// accumulators a lane has 8 or 16 bytes of a row, an instruction sixteen pieces of it, and the address unit takes them one by
// one (64 experts' gradients of 1024 x 2048, bfloat16: 237 -> 188 us; 1e6 rows of 64 doubles: 272 -> 264 us).  As many rows at
// a time as the buffer of BYTES holds; a granule of a row goes to place ^ (row & 15).  A 128 x 128 tile of doubles would take
// four rounds, which cost more than they save (2e6 rows: 1344 -> 1389 us): those leave directly, 64 bytes of a row together.
// S: what is stored.  part(m, i, j): the four results of row m in block i of 16 columns, of the lane's own in block j of rows;
// row(m): where row m begins (m below n_rows), of which `width` columns exist.
template <class T, class S, int BYTES, int BM, int BN, int FA, int FB, class Part, class Row>
__device__ __forceinline__ void store_tile(char *lds, int wn, int wm, int n_rows, int width, Part part, Row row) {
    constexpr int kFit = BYTES / (BN * (int)sizeof(S));
    constexpr int R = kFit >= BM ? BM : kFit >= 64 ? 64 : kFit >= 32 ? 32 : 16;
    constexpr int G = BN * (int)sizeof(S) / 16, E = 16 / (int)sizeof(S), kMask = G < 16 ? G - 1 : 15;
    static_assert(R * BN * (int)sizeof(S) <= BYTES && BM % R == 0, "a tile's results by whole rounds");
    const int lane = wave_lane(), q = lane >> 4;
    if constexpr (sizeof(S) == 8 && BM * BN >= 128 * 128) {
#pragma unroll
        for (int j = 0; j < FB; ++j) {
            const int m = (wm * FB + j) * 16 + (lane & 15);
            if (m >= n_rows) continue;
            S *line = row(m);
#pragma unroll
            for (int i = 0; i < FA; ++i) {
                const auto v = part(m, i, j);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = (wn * FA + i) * 16 + result_col<T>(q, 2 * h);
                    store_run<2>(line + col, v, 2 * h, width - col);
                }
            }
        }
        return;
    }
#pragma unroll
    for (int r0 = 0; r0 < BM; r0 += R) {
        if (r0 >= n_rows) break;
        __syncthreads();                                        // (the buffer is free: of operands, or of the round before)
#pragma unroll
        for (int j = 0; j < FB; ++j) {
            const int block = (wm * FB + j) * 16;
            if (block < r0 || block >= r0 + R) continue;
            const int m = block + (lane & 15) - r0;
            char *line = lds + m * (G * 16);
#pragma unroll
            for (int i = 0; i < FA; ++i) {
                const auto v = part(m + r0, i, j);
                const int c = (wn * FA + i) * 16;
                if constexpr (sizeof(T) == 8) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int col = c + result_col<T>(q, 2 * h);
                        struct alignas(16) Run { S e[2]; } o = {{(S)v[2 * h], (S)v[2 * h + 1]}};
                        *(Run *)(line + (((col / E) ^ (m & kMask)) << 4)) = o;
                    }
                } else {
                    const int col = c + q * 4;
                    struct alignas(sizeof(S) == 2 ? 8 : 16) Run { S e[4]; } o = {{(S)v[0], (S)v[1], (S)v[2], (S)v[3]}};
                    *(Run *)(line + (((col / E) ^ (m & kMask)) << 4) + col % E * (int)sizeof(S)) = o;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int x0 = 0; x0 < R * G; x0 += 256) {
            const int x = x0 + threadIdx.x, m = x / G, g = x % G;
            if ((R * G) % 256 != 0 && x >= R * G) continue;
            if (m + r0 >= n_rows) continue;
            struct alignas(16) Run { S e[E]; };
            const Run o = *(const Run *)(lds + m * (G * 16) + ((g ^ (m & kMask)) << 4));
            S *p = row(m + r0) + g * E;
            const int avail = width - g * E;
            if (avail >= E) {
                store_any(p, o);
            } else {
#pragma unroll
                for (int c = 0; c < E; ++c)
                    if (c < avail) p[c] = o.e[c];
            }
        }
    }
}

// What bounds it.  1e6 rows of 64 doubles: memory, 240 us for 1.04 GB.  2e6 of 128 doubles: 1.32 ms, 49 TFLOP/s, the matrix pipe 64 %
// busy; the rest is the beginnings and ends of tiles of eight steps (without the results' stores 1.19 of 1.44 ms when that was
// measured, without loads 1.37).  16384 rows, 64 experts of 1024 x 2048, bfloat16: 130 - 150 us, 500 TFLOP/s; every byte of a tile
// comes from L2 (1.3 GB for both operands, 9 TB/s), ragged ends are a fifth of the tiles.  A tile of 256 columns halves
// the rows' share of that and takes two workgroups a compute unit instead of three: 182 against 146 us.
template <class T, bool KCONTIG, int BM, int BN, int WN, int WM>
__global__ __launch_bounds__(256, (kWavesPerSimd<T, BM * BN>)) void rows_kernel(RowsArgs a) {
    typedef typename Acc<T>::type A;
    typedef typename Acc<T>::v4 A4;
    constexpr int FA = BN / WN / 16, FB = BM / WM / 16;
    constexpr int XP = (BM + 31) / 32, WP = (BN + 31) / 32;        // granules a thread moves per step
    // Steps at a time: two beside 16 rows, where the weights stream through and bytes in flight are what counts (64 experts of
    // 1024 x 1024, 16 rows each, bfloat16: 28.6 -> 26.0 us; 8 rows of 2 experts, 2048 -> 1024: 17.7 -> 16.5 us).
    constexpr int U = BM == 16 ? 2 : 1, kBuf = (BM + BN) * kStepBytes;
    __shared__ __attribute__((aligned(128))) char lds[U * kBuf];
    __shared__ int row_of[BM];      // what the results need is here before the products are done: rows, gates, bias
    __shared__ A gate_of[BM];
    __shared__ __attribute__((aligned(16))) A bias_of[BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % WN, wm = wave / WN;

    // ---- which tile: blocks of eight row tiles, within a block every column tile (of every split) in turn
    constexpr int kBlock = 8;
    const int per_block = kBlock * a.n_tiles * a.splits;
    const int id = die_order(a.run, a.first), blk = id / per_block, local = id - blk * per_block;
    if (blk >= a.tile_blocks) return;
    const int t = blk * kBlock + local % kBlock, rest = local / kBlock, nt = rest % a.n_tiles, split = rest / a.n_tiles;
    const int4 tile = a.tiles[t];
    const int e = tile.x, n_rows = tile.z;
    if (e < 0 || (e == a.K && !a.out)) return;
    const int *list = a.order + tile.y;
    const int n0 = nt * BN;

    if (e == a.K) {                 // rows of no component: zeros
        T *out = (T *)a.out;
        const int n = a.ndim - n0 < BN ? a.ndim - n0 : BN;
        for (int j = tid; j < n_rows * n; j += 256) out[(i64)list[j / n] * a.out_stride + n0 + j % n] = (T)0.0f;
        return;
    }

    // ---- contraction range of this split, in whole steps
    const int steps_all = (a.kdim + kStep<T> - 1) / kStep<T>;
    const int s_lo = steps_all * split / a.splits, s_hi = steps_all * (split + 1) / a.splits;
    const int k_end = s_hi * kStep<T> < a.kdim ? s_hi * kStep<T> : a.kdim;

    // What a thread moves: granule column tid % 8 of the rows tid / 8 + 32 p of a KTile, granules tid + 256 p of an MTile.  16-byte
    // loads at any alignment; places outside (rows behind the last, columns behind ndim) read a neighbour that exists, whose
    // results are not stored, so that the loop has loads and additions only.  The last step of a contraction that is not whole
    // steps reads over its end, too, and zeroes what is behind it in both operands.  Only a wave with a granule that could be
    // across the end of the whole tensor takes its elements one by one (1e6 rows, 7 -> 7 double: 59 -> 51 us; 301 -> 301
    // bfloat16, 16384 rows: 24.5 -> 20.2 us).
    typedef MTile<T, BN> WTile;
    const int kcol = (tid & 7) * kGran<T>;
    const T *xp[XP], *wp[WP];
    int pair[XP];
#pragma unroll
    for (int p = 0; p < XP; ++p) {
        const int r = (tid >> 3) + p * 32;
        pair[p] = list[r < n_rows ? r : n_rows - 1];
    }
    const T *w = (const T *)a.w + (i64)e * a.w_component;
    const int w_safe = (a.K - 1 - e) * a.w_component >= kGran<T> - 1 ? 0x7fffffff : a.w_safe;      // (a component behind this one)
    bool x_careful = false, w_careful = false;
    const i64 w_step = KCONTIG ? kStep<T> : kStep<T> * a.w_row;
#pragma unroll
    for (int p = 0; p < WP; ++p) {
        if (KCONTIG) {
            const int n = n0 + (tid >> 3) + p * 32;
            w_careful = w_careful || (n < a.ndim ? n : a.ndim - 1) >= w_safe;
            wp[p] = w + (i64)(n < a.ndim ? n : a.ndim - 1) * a.w_row + s_lo * kStep<T> + kcol;
        } else {
            const int g = tid + p * 256, n = n0 + (g % WTile::kPerRow) * kGran<T>;
            wp[p] = w + (i64)(s_lo * kStep<T> + g / WTile::kPerRow) * a.w_row + (n < a.ndim ? n : n0);
        }
    }
    A my_bias = 0;
    if (tid < BN && a.bias && split == 0 && n0 + tid < a.ndim) my_bias = (A)((const T *)a.bias)[(i64)e * a.bias_row + n0 + tid];
#pragma unroll
    for (int p = 0; p < XP; ++p) {
        xp[p] = (const T *)a.in + (i64)divide(pair[p], a.in_div) * a.in_stride + s_lo * kStep<T> + kcol;
        const int r = (tid >> 3) + p * 32;
        x_careful = x_careful || divide(pair[p], a.in_div) >= a.in_safe;
        if ((tid & 7) == 0 && r < BM) {
            row_of[r] = pair[p];
            gate_of[r] = a.gates ? ((const A *)a.gates)[pair[p]] : (A)1;
        }
    }
    Granule gx[U * XP], gw[U * WP];
    const int last = s_hi - 1;
    const bool ragged = s_hi * kStep<T> > k_end;
    const bool edge = !KCONTIG && a.ndim - n0 < BN && a.ndim % kGran<T> != 0;
    x_careful = __any(x_careful);
    w_careful = __any(w_careful);
    const auto fetch_rows = [&](int s, int u) {      // (step after step: the pointers move along)
        if (!(ragged && s == last)) {
#pragma unroll
            for (int p = 0; p < XP; ++p)
                if (BM >= 32 || tid < BM * 8) gx[u * XP + p] = load_whole(xp[p]);
        } else {
            const int left_k = k_end - s * kStep<T> - kcol;
            if (!x_careful) {
#pragma unroll
                for (int p = 0; p < XP; ++p)
                    if (BM >= 32 || tid < BM * 8) gx[u * XP + p] = load_whole(left_k > 0 ? xp[p] : xp[p] - kcol);
#pragma unroll
                for (int p = 0; p < XP; ++p) keep<T>(gx[u * XP + p], left_k);
            } else {
#pragma unroll
                for (int p = 0; p < XP; ++p)
                    if (BM >= 32 || tid < BM * 8) gx[u * XP + p] = load_part(xp[p], left_k);
            }
        }
#pragma unroll
        for (int p = 0; p < XP; ++p) xp[p] += kStep<T>;
    };
    const auto fetch_weights = [&](int s, int u) {
        const bool careful = KCONTIG ? w_careful && ragged && s == last : edge && (s + 1) * kStep<T> > w_safe;
        if (!(ragged && s == last) && !careful) {
#pragma unroll
            for (int p = 0; p < WP; ++p)
                if (BN >= 32 || tid < BN * 8) gw[u * WP + p] = load_whole(wp[p]);
        } else if (!careful) {
#pragma unroll
            for (int p = 0; p < WP; ++p) {
                // (KCONTIG: a granule behind the end reads the step's first; else a row behind the end reads the last one)
                const int left = KCONTIG ? k_end - s * kStep<T> - kcol : k_end - s * kStep<T> - (tid + p * 256) / WTile::kPerRow;
                const T *from = left > 0 ? wp[p] : KCONTIG ? wp[p] - kcol : wp[p] + (left - 1) * a.w_row;
                if (BN >= 32 || tid < BN * 8) gw[u * WP + p] = load_whole(from);
            }
#pragma unroll
            for (int p = 0; p < WP; ++p) {
                const int left = KCONTIG ? k_end - s * kStep<T> - kcol : k_end - s * kStep<T> - (tid + p * 256) / WTile::kPerRow;
                if (KCONTIG) keep<T>(gw[u * WP + p], left);
                else if (left <= 0) gw[u * WP + p].raw = (v4i){0, 0, 0, 0};
            }
        } else {
#pragma unroll
            for (int p = 0; p < WP; ++p) {
                if (BN < 32 && tid >= BN * 8) continue;
                if (KCONTIG) {
                    gw[u * WP + p] = load_part(wp[p], k_end - s * kStep<T> - kcol);
                } else {
                    const int g = tid + p * 256, n = n0 + (g % WTile::kPerRow) * kGran<T>;
                    gw[u * WP + p] = load_part(wp[p], s * kStep<T> + g / WTile::kPerRow < k_end ? a.ndim - (n < a.ndim ? n : n0) : 0);
                }
            }
        }
#pragma unroll
        for (int p = 0; p < WP; ++p) wp[p] += w_step;
    };
    const auto fetch = [&](int s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u > 0 && s + u > last) continue;
            fetch_weights(s + u, u);
            fetch_rows(s + u, u);
        }
    };
    const auto put_one = [&](int u) {
#pragma unroll
        for (int p = 0; p < XP; ++p)
            if (BM >= 32 || tid < BM * 8) *(v4i *)(lds + u * kBuf + KTile<T>::at((tid >> 3) + p * 32, tid & 7)) = gx[u * XP + p].raw;
        char *wb = lds + u * kBuf + BM * kStepBytes;
#pragma unroll
        for (int p = 0; p < WP; ++p) {
            if (BN < 32 && tid >= BN * 8) continue;
            const int x = tid + p * 256;
            *(v4i *)(wb + (KCONTIG ? KTile<T>::at((tid >> 3) + p * 32, tid & 7) : WTile::at(x / WTile::kPerRow, x % WTile::kPerRow))) = gw[u * WP + p].raw;
        }
    };

    const auto put = [&](int s) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u == 0 || s + u <= last) put_one(u);
    };

    A4 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = (A4){0, 0, 0, 0};
    // a wave whose part of the tile lies behind the last column or row multiplies nothing
    const bool busy = n0 + wn * FA * 16 < a.ndim && wm * FB * 16 < n_rows;
    const auto compute = [&](int at) {
        const char *wb = lds + at + BM * kStepBytes;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            Granule fa[FA], fb[FB];
#pragma unroll
            for (int i = 0; i < FA; ++i) {
                const int block = wn * FA * 16 + i * 16;
                fa[i] = KCONTIG ? KTile<T>::template read<true>(wb, block, ks) : WTile::template read<true>(wb, block, ks);
            }
#pragma unroll
            for (int j = 0; j < FB; ++j) fb[j] = KTile<T>::template read<false>(lds + at, wm * FB * 16 + j * 16, ks);
#pragma unroll
            for (int part = 0; part < kParts<T>; ++part)
#pragma unroll
                for (int i = 0; i < FA; ++i)
#pragma unroll
                    for (int j = 0; j < FB; ++j) mma<T>(acc[i][j], fa[i], fb[j], part);
        }
    };

    fetch(s_lo);                                                // (a split has at least one step)
    if (tid < BN) bias_of[tid] = my_bias;
    put(s_lo);
    __syncthreads();
    for (int s = s_lo; s <= last; s += U) {
        if (s + U <= last) fetch(s + U);
        if (busy) {
            compute(0);
            if (U > 1 && s + 1 <= last) compute(kBuf);
        }
        __syncthreads();
        if (s + U <= last) put(s + U);
        __syncthreads();
    }

    // ---- results
    constexpr int kBytes = U * kBuf;
    const auto biased = [&](int i, int j) {
        A4 v = acc[i][j];
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] += bias_of[(wn * FA + i) * 16 + result_col<T>(lane >> 4, x)];
        return v;
    };
    if (a.dots) {
        // the gates' gradient wants in . u: each wave's columns of a row, added up by gates_kernel
#pragma unroll
        for (int j = 0; j < FB; ++j) {
            const int m = (wm * FB + j) * 16 + (lane & 15);
            A s = 0;
            if (m < n_rows) {
                const T *x = (const T *)a.dot_in + (i64)divide(row_of[m], a.dot_div) * a.dot_stride + n0;
#pragma unroll
                for (int i = 0; i < FA; ++i) {
                    constexpr int kRun = sizeof(T) == 8 ? 2 : 4;        // consecutive columns among a lane's four results
#pragma unroll
                    for (int h = 0; h < 4; h += kRun) {
                        const int col = (wn * FA + i) * 16 + result_col<T>(lane >> 4, h), avail = a.ndim - n0 - col;
                        A v[kRun];
                        load_few<kRun>(x + col, avail, v);
#pragma unroll
                        for (int y = 0; y < kRun; ++y) s += y < avail ? acc[i][j][h + y] * v[y] : (A)0;
                    }
                }
            }
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            if (m < n_rows && lane < 16) ((A *)a.dots)[(i64)row_of[m] * a.n_dots + (split * a.n_tiles + nt) * WN + wn] = s;
        }
    }
    if (a.ws) {
        A *ws = (A *)a.ws + (i64)split * a.P * a.ndim + n0;
        store_tile<T, A, kBytes, BM, BN, FA, FB>(lds, wn, wm, n_rows, a.ndim - n0, [&](int, int i, int j) { return biased(i, j); },
                                                 [&](int m) { return ws + (i64)row_of[m] * a.ndim; });
    } else if (a.out) {
        T *out = (T *)a.out + n0;
        store_tile<T, T, kBytes, BM, BN, FA, FB>(lds, wn, wm, n_rows, a.ndim - n0, [&](int m, int i, int j) { return biased(i, j) * gate_of[m]; },
                                                 [&](int m) { return out + (i64)row_of[m] * a.out_stride; });
    }
}

// A number as two of bfloat16, which has its range: the upper half of its bits, and the rest rounded to 8 bits (2^-15 of the number
// at most is lost).  The second is NaN beside infinity.
__device__ __forceinline__ void two_pieces(float v, bf16_t &high, bf16_t &low) {
    const float h = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
    high = (bf16_t)h;
    low = (bf16_t)(v - h);
}

// dW: the rows of a chunk are the contraction, both operands have it outermost (MTile).
// PIECES, the gates of 16-bit types: g d in 16 bits would be a rounding more than the operands have, and in half precision it leaves
// the range (a gate of 1e-4 times a gradient of 1e-4 is zero there).  It goes into the product as two of bfloat16, the rows in half
// precision too (11 bits are whole in two): two or four products of pieces in one accumulator, 2^-15 of a term lost.  Forward and this,
// 16384 rows of 64 experts, 1024 x 2048: bfloat16 330 us with g d rounded, 375 in pieces (25 the second product, 25 to make them),
// half precision 334 and 490.
// 64 experts of 1024 x 2048 from 16384 rows, bfloat16: 190 us, 360 TFLOP/s, without pieces.  A component's 256 rows are four steps, so the time is
// what four steps do not hide: finding the chunk, its rows and the first loads (a quarter, alone), and the results' stores (4 MB
// for 1.5 MB of operands; a third).
template <class T, int BI, int BO, int WO, int WI, bool PIECES>
__global__ __launch_bounds__(256, (kWavesPerSimd<T, BI * BO>)) void weight_kernel(WeightArgs a) {
    static_assert(!PIECES || sizeof(T) == 2, "pieces of 16 bits");
    typedef typename Acc<T>::type A;
    typedef typename Acc<T>::v4 A4;
    constexpr int FA = BO / WO / 16, FB = BI / WI / 16;
    constexpr int NI = (BI + 31) / 32, NO = (BO + 31) / 32;     // granules of either operand a thread moves per step
    constexpr bool kAllI = BI >= 32, kAllO = BO >= 32, kSame = BI == BO;        // every thread moves some; the same rows of both
    typedef MTile<T, BI> ITile;
    typedef MTile<T, BO> OTile;
    constexpr bool kHalves = PIECES && std::is_same_v<T, f16_t>;       // the rows in pieces, too
    typedef std::conditional_t<PIECES, bf16_t, T> M;                    // what is multiplied
    constexpr int kBytes = (BI + BO + (PIECES ? BO : 0) + (kHalves ? BI : 0)) * kStepBytes;
    __shared__ __attribute__((aligned(128))) char lds[kBytes];
    char *const lds_o = lds + BI * kStepBytes, *const low_o = lds_o + BO * kStepBytes, *const low_i = low_o + BO * kStepBytes;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wo = wave % WO, wi = wave / WO;
    const int out_tiles = a.i_tiles * a.o_tiles;
    const int id = die_order(a.run, a.first), chunk = id / out_tiles, tile = id % out_tiles;
    const Bucket at_b = find_bucket(a.bucket_first, a.offsets, a.K, chunk);
    if (at_b.b < 0) return;
    const int e = at_b.b, c = chunk - at_b.first, chunks = at_b.next_first - at_b.first;
    const int rows_per = 256 << a.level;
    const int row0 = at_b.offset + c * rows_per, left = at_b.next_offset - row0, n_rows = left < rows_per ? left : rows_per;
    const int *list = a.order + row0;
    const int i0 = (tile % a.i_tiles) * BI, o0 = (tile / a.i_tiles) * BO;
    const A *gates = (const A *)a.gates;
    const bool want_db = a.db && i0 == 0;

    // a thread moves the same granule column of rows r, r + kRows, ...; an operand's rows go by indices read one step
    // before its rows are asked for (the same ones for both in square tiles).  As in rows_kernel, places outside read a neighbour; rows behind the last are
    // zero in both operands, and a granule across the end of a row is read with care where no row is behind it.
    constexpr int kRowsI = 256 / ITile::kPerRow < kStep<T> ? 256 / ITile::kPerRow : kStep<T>;
    constexpr int kRowsO = 256 / OTile::kPerRow < kStep<T> ? 256 / OTile::kPerRow : kStep<T>;
    const int i_row = tid / ITile::kPerRow, i_at = tid % ITile::kPerRow, o_row = tid / OTile::kPerRow, o_at = tid % OTile::kPerRow;
    const int i_col = i0 + i_at * kGran<T> < a.idim ? i0 + i_at * kGran<T> : i0, o_col = o0 + o_at * kGran<T> < a.odim ? o0 + o_at * kGran<T> : o0;
    const T *in = (const T *)a.in + i_col, *dd = (const T *)a.d + o_col;
    const int i_safe = a.idim - i_col < kGran<T> ? a.in_safe : 0x7fffffff, o_safe = a.odim - o_col < kGran<T> ? a.d_safe : 0x7fffffff;
    struct Held { Granule i[NI], o[NO]; A gate[NO]; } held;
    int at_i[NI], at_o[NO];
    const auto look = [&](int s) {
        if (!kSame) {
#pragma unroll
            for (int p = 0; p < NI; ++p) {
                const int r = s * kStep<T> + i_row + p * kRowsI;
                at_i[p] = list[r < n_rows ? r : n_rows - 1];
            }
        }
#pragma unroll
        for (int p = 0; p < NO; ++p) {
            const int r = s * kStep<T> + o_row + p * kRowsO;
            at_o[p] = list[r < n_rows ? r : n_rows - 1];
        }
    };
    const bool edge = (a.idim - i0 < BI && a.idim % kGran<T> != 0) || (a.odim - o0 < BO && a.odim % kGran<T> != 0);
    const auto fetch = [&](Held &h, int s) {        // (at_i, at_o: the indices of step s; leaves those of s + 1)
        int ri[NI], ro[NO];
#pragma unroll
        for (int p = 0; p < NI; ++p) ri[p] = divide(kSame ? at_o[p] : at_i[p], a.in_div);
#pragma unroll
        for (int p = 0; p < NO; ++p) ro[p] = divide(at_o[p], a.d_div);
        bool careful = false;
        if (edge) {
#pragma unroll
            for (int p = 0; p < NI; ++p) careful = careful || ri[p] >= i_safe;
#pragma unroll
            for (int p = 0; p < NO; ++p) careful = careful || ro[p] >= o_safe;
            careful = __any(careful);
        }
        if (!careful) {
            if (kAllI || tid < BI * 8) {
#pragma unroll
                for (int p = 0; p < NI; ++p) h.i[p] = load_whole(in + (i64)ri[p] * a.in_stride);
            }
            if (kAllO || tid < BO * 8) {
#pragma unroll
                for (int p = 0; p < NO; ++p) h.o[p] = load_whole(dd + (i64)ro[p] * a.d_stride);
            }
        } else {
            if (kAllI || tid < BI * 8) {
#pragma unroll
                for (int p = 0; p < NI; ++p) {
                    const T *pi = in + (i64)ri[p] * a.in_stride;
                    if (ri[p] < i_safe) h.i[p] = load_whole(pi);
                    else h.i[p] = load_part(pi, a.idim - i_col);
                }
            }
            if (kAllO || tid < BO * 8) {
#pragma unroll
                for (int p = 0; p < NO; ++p) {
                    const T *po = dd + (i64)ro[p] * a.d_stride;
                    if (ro[p] < o_safe) h.o[p] = load_whole(po);
                    else h.o[p] = load_part(po, a.odim - o_col);
                }
            }
        }
        if (gates && (kAllO || tid < BO * 8)) {
#pragma unroll
            for (int p = 0; p < NO; ++p) h.gate[p] = gates[at_o[p]];
        }
        look(s + 1);
    };
    A dsum[kGran<T>];
#pragma unroll
    for (int j = 0; j < kGran<T>; ++j) dsum[j] = 0;
    const int n_steps = (n_rows + kStep<T> - 1) / kStep<T>;     // (at least one: a chunk has rows)
    const auto put = [&](Held &h, int s) {
        if (s == n_steps - 1) {                                 // rows behind the last
#pragma unroll
            for (int p = 0; p < NI; ++p)
                if (s * kStep<T> + i_row + p * kRowsI >= n_rows) h.i[p].raw = (v4i){0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < NO; ++p)
                if (s * kStep<T> + o_row + p * kRowsO >= n_rows) {
                    h.o[p].raw = (v4i){0, 0, 0, 0};
                    h.gate[p] = 0;
                }
        }
        if (kAllO || tid < BO * 8) {
#pragma unroll
            for (int p = 0; p < NO; ++p) {
                T *el = Elems<T>::of(h.o[p]);
                if constexpr (PIECES) {
                    Granule low;
#pragma unroll
                    for (int j = 0; j < kGran<T>; ++j) {
                        const A v = (A)el[j] * h.gate[p];
                        if (want_db) dsum[j] += v;
                        two_pieces(v, h.o[p].b[j], low.b[j]);
                    }
                    *(v4i *)(low_o + OTile::at(o_row + p * kRowsO, o_at)) = low.raw;
                } else if (gates) {
#pragma unroll
                    for (int j = 0; j < kGran<T>; ++j) {
                        const A v = (A)el[j] * h.gate[p];
                        if (want_db) dsum[j] += v;
                        el[j] = (T)v;
                    }
                } else if (want_db) {
#pragma unroll
                    for (int j = 0; j < kGran<T>; ++j) dsum[j] += (A)el[j];
                }
                *(v4i *)(lds_o + OTile::at(o_row + p * kRowsO, o_at)) = h.o[p].raw;
            }
        }
        if (kAllI || tid < BI * 8) {
#pragma unroll
            for (int p = 0; p < NI; ++p) {
                if constexpr (kHalves) {
                    Granule low;
#pragma unroll
                    for (int j = 0; j < kGran<T>; ++j) two_pieces((float)h.i[p].h[j], h.i[p].b[j], low.b[j]);
                    *(v4i *)(low_i + ITile::at(i_row + p * kRowsI, i_at)) = low.raw;
                }
                *(v4i *)(lds + ITile::at(i_row + p * kRowsI, i_at)) = h.i[p].raw;
            }
        }
    };

    A4 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = (A4){0, 0, 0, 0};
    const auto compute = [&]() {
        if (WO * WI < 4 && wave >= WO * WI) return;             // (a tile too small for four waves: the others only move data)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            Granule fa[FA], fb[FB];
#pragma unroll
            for (int turn = (PIECES ? 2 : 1) * (kHalves ? 2 : 1) - 1; turn >= 0; --turn) {          // (the small products first)
                const bool low = turn & 1, rows_low = turn >> 1;
                if (turn == (kHalves ? 3 : PIECES ? 1 : 0) || (kHalves && turn == 1)) {
#pragma unroll
                    for (int j = 0; j < FB; ++j) fb[j] = ITile::template read<false>(rows_low ? low_i : lds, (wi * FB + j) * 16, ks);
                }
#pragma unroll
                for (int i = 0; i < FA; ++i) fa[i] = OTile::template read<true>(low ? low_o : lds_o, (wo * FA + i) * 16, ks);
#pragma unroll
                for (int part = 0; part < kParts<T>; ++part)
#pragma unroll
                    for (int i = 0; i < FA; ++i)
#pragma unroll
                        for (int j = 0; j < FB; ++j) mma<M>(acc[i][j], fa[i], fb[j], part);
                // (the next turn's operands in these ones' registers: 123 spilled with all at once)
                if (PIECES) __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    look(0);
    fetch(held, 0);
    put(held, 0);
    __syncthreads();
    for (int s = 0; s < n_steps; ++s) {
        if (s + 1 < n_steps) fetch(held, s + 1);
        compute();
        __syncthreads();
        if (s + 1 < n_steps) put(held, s + 1);
        __syncthreads();
    }
    if constexpr (PIECES) {
        // An infinite number makes NaN in pieces, by its own second one or another's that is zero.  A wave that has a NaN adds up its
        // results once more, whole numbers one by one (forward and this where every result is NaN: 0.41 -> 1.9 ms, 16384 rows as above).
        bool undefined = false;
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) undefined = undefined || acc[i][j][x] != acc[i][j][x];
        if (__any(undefined)) {
#pragma unroll
            for (int i = 0; i < FA; ++i)
#pragma unroll
                for (int j = 0; j < FB; ++j) acc[i][j] = (A4){0, 0, 0, 0};
            for (int r = 0; r < n_rows; ++r) {
                const int p = list[r];
                const T *pi = (const T *)a.in + (i64)divide(p, a.in_div) * a.in_stride, *po = (const T *)a.d + (i64)divide(p, a.d_div) * a.d_stride;
                A row[FB];
#pragma unroll
                for (int j = 0; j < FB; ++j) {
                    const int m = i0 + (wi * FB + j) * 16 + (lane & 15);
                    row[j] = (A)pi[m < a.idim ? m : i0];
                }
#pragma unroll
                for (int i = 0; i < FA; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int n = o0 + (wo * FA + i) * 16 + result_col<T>(lane >> 4, x);
                        const A v = (A)po[n < a.odim ? n : o0] * gates[p];
#pragma unroll
                        for (int j = 0; j < FB; ++j) acc[i][j][x] = __builtin_fmaf(v, row[j], acc[i][j][x]);
                    }
            }
        }
    }

    // a component with one chunk is finished here; several leave partial sums, added in the chunks' order by weight_reduce
    A *slot = nullptr;
    if (chunks > 1) slot = (A *)a.ws + ((((i64)at_b.offset * 2) >> (8 + a.level)) + c) * ((i64)a.idim * a.odim + a.odim);
    if (a.dw) {
        const int n_i = a.idim - i0 < BI ? a.idim - i0 : BI, w_o = WO * WI < 4 && wave >= WO * WI ? 0 : wo, w_i = WO * WI < 4 && wave >= WO * WI ? BI : wi;
        const auto part = [&](int, int i, int j) { return acc[i][j]; };         // (waves without a part of the tile: none of its rows)
        if (slot) {
            A *to = slot + (i64)i0 * a.odim + o0;
            store_tile<T, A, kBytes, BI, BO, FA, FB>(lds, w_o, w_i, n_i, a.odim - o0, part, [&](int m) { return to + (i64)m * a.odim; });
        } else {
            T *to = (T *)a.dw + ((i64)e * a.idim + i0) * a.odim + o0;
            store_tile<T, T, kBytes, BI, BO, FA, FB>(lds, w_o, w_i, n_i, a.odim - o0, part, [&](int m) { return to + (i64)m * a.odim; });
        }
    }
    if (!want_db) return;
    // column sums: a thread has those of its granule's columns over its own rows; the threads of a column add up in order
    A *sums = (A *)lds;                       // [kRowsO][BO]
    __syncthreads();
    if (kAllO || tid < BO * 8) {
#pragma unroll
        for (int j = 0; j < kGran<T>; ++j) sums[o_row * BO + o_at * kGran<T> + j] = dsum[j];
    }
    __syncthreads();
    for (int n = tid; n < BO && o0 + n < a.odim; n += 256) {
        A v = 0;
        for (int r = 0; r < kRowsO; ++r) v += sums[r * BO + n];
        if (slot) slot[(i64)a.idim * a.odim + o0 + n] = v;
        else ((T *)a.db)[(i64)e * a.odim + o0 + n] = (T)v;
    }
}

// Components with several chunks: their partial sums in order.  Components without rows: zeros.
template <class T> __global__ __launch_bounds__(256) void weight_reduce(WeightArgs a) {
    typedef typename Acc<T>::type A;
    const int e = blockIdx.y;
    const int chunks = a.bucket_first[e + 1] - a.bucket_first[e];
    if (chunks == 1) return;
    const i64 n_w = (i64)a.idim * a.odim, size = n_w + a.odim;
    if (chunks == 0 && a.dw) {
        struct Run { T e[kGran<T>]; } zeros;
#pragma unroll
        for (int q = 0; q < kGran<T>; ++q) zeros.e[q] = (T)0.0f;
        T *dw = (T *)a.dw + (i64)e * n_w;
        const i64 whole = n_w / kGran<T>;
        for (i64 g = (i64)blockIdx.x * 256 + threadIdx.x; g < whole; g += (i64)gridDim.x * 256) store_any(dw + g * kGran<T>, zeros);
        if (blockIdx.x == 0 && threadIdx.x < n_w - whole * kGran<T>) dw[whole * kGran<T> + threadIdx.x] = (T)0.0f;
    }
    const A *slot = (const A *)a.ws + (((i64)a.offsets[e] * 2) >> (8 + a.level)) * size;
    for (i64 j = (chunks == 0 ? n_w : 0) + (i64)blockIdx.x * 256 + threadIdx.x; j < size; j += (i64)gridDim.x * 256) {
        const bool is_w = j < n_w;
        if (is_w ? !a.dw : !a.db) continue;
        A v = 0;
        int c = 0;
        for (; c + 8 <= chunks; c += 8) {           // (eight loads in flight)
            A t[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) t[q] = slot[(c + q) * size + j];
#pragma unroll
            for (int q = 0; q < 8; ++q) v += t[q];
        }
        for (; c < chunks; ++c) v += slot[c * size + j];
        if (is_w) ((T *)a.dw)[(i64)e * n_w + j] = (T)v;
        else ((T *)a.db)[(i64)e * a.odim + (j - n_w)] = (T)v;
    }
}

// u_p, the sum of its parts
template <class A> __device__ __forceinline__ void parts4(const A *src, i64 part, int splits, int avail, A (&u)[4]) {
    load4(src, avail, u);
    for (int s = 1; s < splits; ++s) {
        A t[4];
        load4(src + s * part, avail, t);
#pragma unroll
        for (int x = 0; x < 4; ++x) u[x] += t[x];
    }
}

// out[i] = sum over j of g_ij u_ij, u_ij the sum of its splits: one thread per four elements.  Memory-bound: 8192 x 2 x 2048, 35 us
// for 168 MB.
template <class T> __global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
    typedef typename Acc<T>::type A;
    const int quads = (a.dim + 3) >> 2;
    for (i64 t = (i64)blockIdx.x * 256 + threadIdx.x; t < a.rows * quads; t += (i64)gridDim.x * 256) {
        const i64 i = t / quads;
        const int c = (int)(t - i * quads) * 4, avail = a.dim - c;
        typename Acc<T>::v4 v = {0, 0, 0, 0};
        for (int j = 0; j < a.k; ++j) {
            const i64 p = i * a.k + j;
            if (a.bucket[p] >= a.K) continue;
            A u[4];
            parts4<A>((const A *)a.ws + p * a.dim + c, a.P * a.dim, a.splits, avail, u);
            const A g = a.gates ? ((const A *)a.gates)[p] : (A)1;
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] += g * u[x];
        }
        store_run<4>((T *)a.out + i * a.out_stride + c, v, 0, avail);
    }
}

// The same for few results of many parts: sixteen lanes share the k x splits terms of four elements, so that they are all in
// flight at once (product and sum, one row of 4 experts, 2048 -> 1024 bfloat16: 16.7 -> 8.8 us, 600 rows, 4096 -> 128 single: 22.6
// -> 19.1 us; but 300 rows, 2048 -> 1024 bfloat16: 17.8 -> 18.3 us).
template <class T> __global__ __launch_bounds__(256) void combine_parts_kernel(CombineArgs a) {
    typedef typename Acc<T>::type A;
    const int quads = (a.dim + 3) >> 2, lane = threadIdx.x & 15;
    const i64 t = (i64)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool on = t < a.rows * quads;
    const i64 i = on ? t / quads : 0;
    const int c = on ? (int)(t - i * quads) * 4 : 0, avail = a.dim - c;
    typename Acc<T>::v4 v = {0, 0, 0, 0};
    for (int x = lane; x < a.k * a.splits; x += 16) {
        const i64 p = i * a.k + x % a.k;
        if (a.bucket[p] >= a.K) continue;
        A u[4];
        load4((const A *)a.ws + ((i64)(x / a.k) * a.P + p) * a.dim + c, avail, u);
        const A g = a.gates ? ((const A *)a.gates)[p] : (A)1;
#pragma unroll
        for (int y = 0; y < 4; ++y) v[y] += g * u[y];
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) v[y] = group_sum<16>((A)v[y]);
    if (on && lane == 0) store_run<4>((T *)a.out + i * a.out_stride + c, v, 0, avail);
}

// With the gates' gradient in . u_ij + b . d_i: one wave per row.  KJ >= k.
template <class T, int KJ> __global__ __launch_bounds__(256) void combine_gates_kernel(CombineArgs a) {
    typedef typename Acc<T>::type A;
    const int lane = wave_lane();
    const i64 i = a.first + (i64)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= a.rows) return;
    A dot[KJ], g[KJ];
    int e[KJ];
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
        dot[j] = 0;
        e[j] = j < a.k ? a.bucket[i * a.k + j] : a.K;
        g[j] = e[j] < a.K ? ((const A *)a.gates)[i * a.k + j] : (A)0;
    }
    const T *in = (const T *)a.in + i * a.in_stride;
    for (int c = lane * 4; c < a.dim; c += 256) {
        const int avail = a.dim - c;
        typename Acc<T>::v4 v = {0, 0, 0, 0};
        A x[4];
        load4(in + c, avail, x);
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
            if (e[j] >= a.K) continue;
            A u[4];
            parts4<A>((const A *)a.ws + (i * a.k + j) * a.dim + c, a.P * a.dim, a.splits, avail, u);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                dot[j] += x[q] * u[q];
                v[q] += g[j] * u[q];
            }
        }
        if (a.out) store_run<4>((T *)a.out + i * a.out_stride + c, v, 0, avail);
    }
    if (a.bias) {
        for (int c = lane * 4; c < a.ddim; c += 256) {
#pragma unroll
            for (int j = 0; j < KJ; ++j)
                if (e[j] < a.K) {
                    A b[4], d[4];
                    load4((const T *)a.bias + (i64)e[j] * a.bias_row + c, a.ddim - c, b);
                    load4((const T *)a.d + ((i * a.k + j) / a.d_div) * a.d_stride + c, a.ddim - c, d);
#pragma unroll
                    for (int q = 0; q < 4; ++q) dot[j] += b[q] * d[q];
                }
        }
    }
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
        if (j >= a.k) break;
        const A v = group_sum<64>(dot[j]);
        if (lane == 0) ((A *)a.dgates)[i * a.k + j] = v;
    }
}

// The gates' gradient where a row has one product: the parts of in . u_p that the product left, and b_e . d: sixteen lanes per row.
template <class T> __global__ __launch_bounds__(256) void gates_kernel(GatesArgs a) {
    typedef typename Acc<T>::type A;
    const int lane = threadIdx.x & 15;
    for (i64 p0 = (i64)blockIdx.x * 16; p0 < a.P; p0 += (i64)gridDim.x * 16) {
        const i64 p = p0 + (threadIdx.x >> 4);
        const int e = p < a.P ? a.bucket[p] : a.K;
        A s = 0;
        if (e < a.K) {
            for (int c = lane; c < a.n_dots; c += 16) s += ((const A *)a.dots)[p * a.n_dots + c];
            if (a.bias) {
                const T *b = (const T *)a.bias + (i64)e * a.bias_row, *d = (const T *)a.d + divide((int)p, a.d_div) * a.d_stride;
                for (int c = lane * 4; c < a.ddim; c += 64) {
                    A x[4], y[4];
                    load4(b + c, a.ddim - c, x);
                    load4(d + c, a.ddim - c, y);
#pragma unroll
                    for (int q = 0; q < 4; ++q) s += x[q] * y[q];
                }
            }
        }
        s = group_sum<16>(s);
        if (p < a.P && lane == 0) ((A *)a.dgates)[p] = s;
    }
}

// Workgroups of 256 in as many launches as they take.
template <class Args, class F> static void in_parts(Args a, i64 blocks, F launch) {
    constexpr i64 kEach = kThreadsAtOnce / 256;
    for (i64 b = 0; b < blocks; b += kEach) {
        a.first = (int)b;
        launch(a, blocks - b < kEach ? blocks - b : kEach);
    }
}

template <class T, bool KCONTIG> static void rows_by_tile(const RowsArgs &a, int bm, int bn, i64 blocks, hipStream_t st) {
    const dim3 g((unsigned)blocks);
    if (bm == 16) rows_kernel<T, KCONTIG, 16, 128, 4, 1><<<g, 256, 0, st>>>(a);
    else if (bn == 16) rows_kernel<T, KCONTIG, 128, 16, 1, 4><<<g, 256, 0, st>>>(a);
    else if (bn == 32) rows_kernel<T, KCONTIG, 128, 32, 1, 4><<<g, 256, 0, st>>>(a);
    else if (bn == 64) rows_kernel<T, KCONTIG, 128, 64, 2, 2><<<g, 256, 0, st>>>(a);
    else rows_kernel<T, KCONTIG, 128, 128, 2, 2><<<g, 256, 0, st>>>(a);
}

template <class T> int launch_rows(const RowsArgs &a, bool kcontig, int bm, int bn, i64 blocks, hipStream_t st) {
    in_parts(a, blocks, [&](const RowsArgs &part, i64 n) {
        kcontig ? rows_by_tile<T, true>(part, bm, bn, n, st) : rows_by_tile<T, false>(part, bm, bn, n, st);
    });
    return ops_launched("rows_product");
}

template <class T, bool PIECES> static void weight_by_tile(const WeightArgs &a, int bi, int bo, i64 blocks, hipStream_t st) {
    const dim3 g((unsigned)blocks);
    if (bi == 16 && bo == 16) weight_kernel<T, 16, 16, 1, 1, PIECES><<<g, 256, 0, st>>>(a);
    else if (bi == 16) weight_kernel<T, 16, 128, 4, 1, PIECES><<<g, 256, 0, st>>>(a);
    else if (bo == 16) weight_kernel<T, 128, 16, 1, 4, PIECES><<<g, 256, 0, st>>>(a);
    else if (bi == 64 && bo == 64) weight_kernel<T, 64, 64, 2, 2, PIECES><<<g, 256, 0, st>>>(a);
    else if (bi == 64) weight_kernel<T, 64, 128, 2, 2, PIECES><<<g, 256, 0, st>>>(a);
    else if (bo == 64) weight_kernel<T, 128, 64, 2, 2, PIECES><<<g, 256, 0, st>>>(a);
    else weight_kernel<T, 128, 128, 2, 2, PIECES><<<g, 256, 0, st>>>(a);
}

template <class T> int launch_weight(const WeightArgs &a, int bi, int bo, i64 blocks, hipStream_t st) {
    in_parts(a, blocks, [&](const WeightArgs &part, i64 n) {
        a.gates && sizeof(T) == 2 ? weight_by_tile<T, sizeof(T) == 2>(part, bi, bo, n, st) : weight_by_tile<T, false>(part, bi, bo, n, st);
    });
    // (most components have one chunk and nothing to add up: about 4096 workgroups in all)
    const i64 size = (i64)a.idim * a.odim + a.odim, most = 4096 / a.K > 4 ? 4096 / a.K : 4;
    const i64 bx = (size + 255) / 256 < most ? (size + 255) / 256 : most;
    weight_reduce<T><<<dim3((unsigned)bx, (unsigned)a.K), 256, 0, st>>>(a);
    return ops_launched("weight_product");
}

template <class T> int launch_combine(const CombineArgs &a, hipStream_t st) {
    if (a.rows == 0) return BGMM_OPS_OK;
    if (a.dgates) {
        // (a launch's threads are counted in 32 bits; a loop over rows in the kernel instead: 8192 rows of 2 x 1024 51 us, 37)
        constexpr i64 kAtOnce = (i64)1 << 25;
        CombineArgs b = a;
        for (b.first = 0; b.first < a.rows; b.first += kAtOnce) {
            const i64 n = a.rows - b.first < kAtOnce ? a.rows - b.first : kAtOnce;
            const dim3 g((unsigned)((n + 3) / 4));
            if (a.k == 1) combine_gates_kernel<T, 1><<<g, 256, 0, st>>>(b);
            else if (a.k == 2) combine_gates_kernel<T, 2><<<g, 256, 0, st>>>(b);
            else if (a.k <= 4) combine_gates_kernel<T, 4><<<g, 256, 0, st>>>(b);
            else if (a.k <= 8) combine_gates_kernel<T, 8><<<g, 256, 0, st>>>(b);
            else combine_gates_kernel<T, 32><<<g, 256, 0, st>>>(b);
        }
    } else {
        const i64 threads = a.rows * ((a.dim + 3) / 4);
        if (a.splits > 1 && threads < 32768) {
            combine_parts_kernel<T><<<dim3((unsigned)((threads + 15) / 16)), 256, 0, st>>>(a);
        } else {
            const i64 b = (threads + 255) / 256 < 65536 ? (threads + 255) / 256 : 65536;
            combine_kernel<T><<<dim3((unsigned)b), 256, 0, st>>>(a);
        }
    }
    return ops_launched("combine");
}

template <class T> int launch_gates(const GatesArgs &a, hipStream_t st) {
    const i64 b = (a.P + 15) / 16 < 65536 ? (a.P + 15) / 16 : 65536;
    gates_kernel<T><<<dim3((unsigned)b), 256, 0, st>>>(a);
    return ops_launched("gate_gradient");
}
