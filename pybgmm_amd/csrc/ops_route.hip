// The k most probable components of every row of log weights, and their weights (include/bgmm_ops.h: bgmm_route).
//
//   chosen: the first k of the components ordered by (log weight descending, index ascending); -inf and NaN never
//   w_j = exp(l_j - m) / total,  m = the row's maximum,  total = the sum over the chosen ones, or over all
//   gradient, g the weights':    renormalised   dl_j = w_j (g_j - sum_c w_c g_c) on the chosen, 0 elsewhere
//                                over all       dl_i = [i chosen] w_i g_i - p_i sum_c w_c g_c
//
// Bound by reading the row once (forward: 1e6 x 200 doubles, k = 4, shares of all, 442 us, 3.75 TB/s, the arithmetic of the double
// exponentials close behind) and writing its gradient once (backward).
#include "ops_common.h"

namespace {

struct RouteArgs {
    const void *l;              // [n][K], row stride
    i64 stride;
    i64 n;
    int K, k;
    bool renormalise;
    int64_t *labels;            // [n][k]
    void *weights;              // [n][k], accumulator type
    void *stats;                // [n][2]: maximum and total, or null
    const void *dweights;       // backward
    void *dl;                   // [n][K] dense
};

template <class A> __device__ __forceinline__ A neg_inf();
template <> __device__ __forceinline__ float neg_inf<float>() { return -__builtin_inff(); }
template <> __device__ __forceinline__ double neg_inf<double>() { return -__builtin_inf(); }

// Of two values the larger or smaller, the other one for a quiet NaN: one instruction each (the builtins put another in front of
// every operand that quiets signalling NaNs; here that is done once, where the values are read).
__device__ __forceinline__ double larger(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double smaller(double a, double b) {
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float smaller(float a, float b) {
    float r;
    asm("v_min_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// y[q] = exp(x[q]) for x <= 0, N at once so that they share the constants' registers.  Double: 2^k exp(r), |r| <= ln 2 / 2, k ln 2
// taken off in two parts; the Taylor series to r^13 / 13! leaves 4e-18.  About twenty instructions each where the library's
// takes twice as many.  Arguments below -800, -inf among them, give zero by underflow.
template <int N> __device__ __forceinline__ void exps(const double *x, double *y) {
    constexpr double c[14] = {1.0, 1.0, 0.5, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800,
                              1.0 / 39916800, 1.0 / 479001600, 1.0 / 6227020800};
    double k[N], r[N];
#pragma unroll
    for (int q = 0; q < N; ++q) {
        const double v = larger(x[q], -800.0);
        k[q] = __builtin_rint(v * 1.4426950408889634074);
        r[q] = __builtin_fma(k[q], -0x1.62e42fefa39efp-1, v);           // ln 2 rounded to 53 bits ...
        r[q] = __builtin_fma(k[q], -0x1.abc9e3b39803fp-56, r[q]);       // ... and what it is short by
        y[q] = c[13];
    }
#pragma unroll
    for (int t = 12; t >= 0; --t)
#pragma unroll
        for (int q = 0; q < N; ++q) y[q] = __builtin_fma(y[q], r[q], c[t]);
#pragma unroll
    for (int q = 0; q < N; ++q) y[q] = __builtin_ldexp(y[q], (int)k[q]);
}
// Single: 2^(x log2 e) on the hardware's exponential, the rounding of the product made good to first order (its error alone is |x|
// half steps).  The hardware's results end at the smallest normal number, 2^-126; below, -inf among them, they are zero.  (Subnormal ones
// by taking the exponent's whole part apart: 500000 x 200, k = 4, 128 -> 140 us.)
template <int N> __device__ __forceinline__ void exps(const float *x, float *y) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
        const float v = larger(x[q], -100.0f);
        const float t = v * 1.44269504f;
        const float low = __builtin_fmaf(v, 1.44269504f, -t) + v * 1.92596303e-8f;
        const float e = __builtin_amdgcn_exp2f(t);
        y[q] = __builtin_fmaf(e, low * 0.693147181f, e);
    }
}

// exp(v - m) for v <= m, exactly 1 where they are equal: also where both are infinite, whose difference is NaN and the smaller of that
// and 0 is 0.  m = +inf: 0 for the others.  (m = -inf: 1 everywhere, for callers that ask for no such row.)
template <int N, class A> __device__ __forceinline__ void ratios(const A *v, A m, A *y) {
    A x[N];
#pragma unroll
    for (int q = 0; q < N; ++q) x[q] = smaller(v[q] - m, (A)0);
    exps<N>(x, y);
}
template <class A> __device__ __forceinline__ A ratio(A v, A m) {
    A y;
    ratios<1>(&v, m, &y);
    return y;
}

// Granule c / E of a row (E elements, E = 1 or 16 bytes' worth), -inf behind the end and for NaN.
template <class T, int E, class A> __device__ __forceinline__ void load_logs(const T *row, int c, bool on, A *v) {
    struct alignas(E == 1 ? sizeof(T) : 16) Pack { T e[E]; } p;
    if (on) p = *(const Pack *)(row + c);
#pragma unroll
    for (int q = 0; q < E; ++q) {
        const A x = (A)p.e[q];
        v[q] = on ? larger(neg_inf<A>(), larger(x, x)) : neg_inf<A>();
    }
}

// G lanes per row hold it in registers, NG granules of E elements each: read once.  A round takes the maximum, then the lowest
// index that has it, then takes that element out: six instructions per element and round.  Lane r of the group keeps
// round r's result (k <= G).
template <class T, int G, int NG, int E> __global__ __launch_bounds__(256) void route_rows_kernel(RouteArgs a) {
    typedef typename Acc<T>::type A;
    const int lane = threadIdx.x & (G - 1);
    const i64 i = (i64)blockIdx.x * (256 / G) + threadIdx.x / G;
    const bool on = i < a.n;                                    // (rows behind the last: their lanes reduce along)
    const T *row = (const T *)a.l + (on ? i : 0) * a.stride;
    constexpr int kBatch = NG * E % 7 == 0 ? 7 : NG * E % 8 == 0 ? 8 : NG * E % 4 == 0 ? 4 : 2;      // exponentials at once
    A v[NG * E];
#pragma unroll
    for (int g = 0; g < NG; ++g) {                              // (K is whole granules)
        const int c = (g * G + lane) * E;
        if ((g + 1) * G * E <= a.K) load_logs<T, E>(row, c, true, v + g * E);
        else load_logs<T, E>(row, c, c < a.K, v + g * E);
    }
    A m;
    int at;
    const auto find = [&]() {
        m = v[0];
#pragma unroll
        for (int q = 1; q < NG * E; ++q) m = larger(m, v[q]);
        m = group_reduce<G>(m, [](A x, A y) { return larger(x, y); });
        at = 0x7fffffff;
#pragma unroll
        for (int q = NG * E - 1; q >= 0; --q) at = v[q] == m ? (q / E) * G * E + q % E : at;
        at = at == 0x7fffffff ? at : at + lane * E;
        at = group_reduce<G>(at, [](int x, int y) { return x < y ? x : y; });
    };
    find();
    const A top = m;
    A mine = m, total = 0;                                      // (every lane starts with the first; lane r takes round r's)
    int mine_at = m > neg_inf<A>() ? at : -1;
    if (!a.renormalise) {
#pragma unroll
        for (int b = 0; b < NG * E; b += kBatch) {
            A y[kBatch];
            ratios<kBatch>(v + b, top, y);
#pragma unroll
            for (int q = 0; q < kBatch; ++q) total += y[q];
        }
        total = group_sum<G>(total);
    }
    for (int r = 1; r < a.k; ++r) {
        const int g = at / E, slot = g % G == lane ? (g / G) * E + at % E : -1;
#pragma unroll
        for (int q = 0; q < NG * E; ++q) v[q] = q == slot ? neg_inf<A>() : v[q];
        find();
        if (lane == r) {
            mine = m;
            mine_at = m > neg_inf<A>() ? at : -1;
        }
    }
    const A e = mine_at >= 0 && lane < a.k ? ratio(mine, top) : (A)0;
    if (a.renormalise) total = group_sum<G>(e);
    if (!on) return;
    if (lane < a.k) {
        a.labels[i * a.k + lane] = mine_at;
        ((A *)a.weights)[i * a.k + lane] = mine_at >= 0 ? e / total : (A)0;
    }
    if (a.stats && lane == 0) {
        ((A *)a.stats)[2 * i] = top;
        ((A *)a.stats)[2 * i + 1] = total;
    }
}

// Longer rows: a workgroup of W waves per row.  HELD: its threads have the row in registers as above, 16 elements each (up to 4096
// and 16384 components); else it is read again for every chosen component, the next one being the largest behind the last
// in the order.  A round's W maxima meet in LDS, in one of two places in turn, so that it takes one barrier.  (single precision,
// 10000 rows of 8000, k = 4: 250 us, one row 8 us, 1000 rows of 100000, k = 2: 294 us; a wave per row took 417, 86 and 2232.)
template <class T, int W, bool HELD, int E> __global__ __launch_bounds__(64 * W) void route_wide_kernel(RouteArgs a) {
    typedef typename Acc<T>::type A;
    constexpr int NG = 16 / E, N = 64 * W;
    __shared__ A top_of[2][W], sum_of[W];
    __shared__ int at_of[2][W];
    const int lane = wave_lane(), w = threadIdx.x >> 6;
    int turn = 0;
    for (i64 i = blockIdx.x; i < a.n; i += gridDim.x) {
        const T *row = (const T *)a.l + i * a.stride;
        A v[HELD ? 16 : 1];
        if constexpr (HELD) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {                      // (K is whole granules)
                const int c = (g * N + threadIdx.x) * E;
                load_logs<T, E>(row, c, c < a.K, v + g * E);
            }
        }
        A m = neg_inf<A>(), last = 0;
        int at = -1;
        const auto find = [&](bool first) {
            A best = neg_inf<A>();
            int mine = 0x7fffffff;
            if constexpr (HELD) {
#pragma unroll
                for (int q = 0; q < 16; ++q) best = larger(best, v[q]);
                best = group_reduce<64>(best, [](A x, A y) { return larger(x, y); });
#pragma unroll
                for (int q = 15; q >= 0; --q) mine = v[q] == best ? ((q / E) * N + (int)threadIdx.x) * E + q % E : mine;
            } else {
#pragma unroll 4
                for (int c = threadIdx.x; c < a.K; c += N) {
                    A x;
                    load_logs<T, 1>(row, c, true, &x);
                    const bool after = first || x < last || (x == last && c > at);
                    mine = after && x > best ? c : mine;
                    best = after && x > best ? x : best;
                }
                const A own = best;
                best = group_reduce<64>(best, [](A x, A y) { return larger(x, y); });
                mine = own == best ? mine : 0x7fffffff;
            }
            mine = group_reduce<64>(mine, [](int x, int y) { return x < y ? x : y; });
            if (lane == 0) {
                top_of[turn][w] = best;
                at_of[turn][w] = mine;
            }
            __syncthreads();
            const A t = top_of[turn][lane % W];
            m = group_reduce<16>(t, [](A x, A y) { return larger(x, y); });
            at = group_reduce<16>(t == m ? at_of[turn][lane % W] : 0x7fffffff, [](int x, int y) { return x < y ? x : y; });
            last = m;
            turn ^= 1;
        };
        find(true);
        const A top = m;
        A chosen = neg_inf<A>(), total = 0;
        int chosen_at = -1;
        if (top > neg_inf<A>()) {
            if (!a.renormalise) {
                if constexpr (HELD) {
#pragma unroll
                    for (int b = 0; b < 16; b += 4) {
                        A y[4];
                        ratios<4>(v + b, top, y);
#pragma unroll
                        for (int q = 0; q < 4; ++q) total += y[q];
                    }
                } else {
                    for (int c = threadIdx.x; c < a.K; c += N) {
                        A x;
                        load_logs<T, 1>(row, c, true, &x);
                        total += ratio(x, top);
                    }
                }
                total = group_sum<64>(total);
                if (lane == 0) sum_of[w] = total;
                __syncthreads();
                total = 0;
#pragma unroll
                for (int j = 0; j < W; ++j) total += sum_of[j];
            }
            for (int r = 0;;) {
                if (lane == r) {
                    chosen = m;
                    chosen_at = at;
                }
                if (++r == a.k) break;
                if constexpr (HELD) {
                    const int g = at / E, slot = g % N == (int)threadIdx.x ? (g / N) * E + at % E : -1;
#pragma unroll
                    for (int q = 0; q < 16; ++q) v[q] = q == slot ? neg_inf<A>() : v[q];
                }
                find(false);
                if (!(m > neg_inf<A>())) break;                 // (no other; the same for every wave)
            }
        }
        const A e = chosen_at >= 0 ? ratio(chosen, top) : (A)0;
        if (a.renormalise) total = group_sum<64>(e);
        if (w != 0) continue;
        if (lane < a.k) {
            a.labels[i * a.k + lane] = chosen_at;
            ((A *)a.weights)[i * a.k + lane] = chosen_at >= 0 ? e / total : (A)0;
        }
        if (a.stats && lane == 0) {
            ((A *)a.stats)[2 * i] = top;
            ((A *)a.stats)[2 * i + 1] = total;
        }
    }
}

// A workgroup owns `rows` whole rows of the gradient, a contiguous stretch: it writes them once, coalesced (zeros, or what the
// softmax over all gives), and behind a barrier the chosen elements again with their full value.
constexpr int kBackRows = 64;
template <class T> __global__ __launch_bounds__(256) void route_backward_kernel(RouteArgs a, int rows) {
    typedef typename Acc<T>::type A;
    __shared__ A sums[kBackRows], tops[kBackRows], scales[kBackRows];
    const i64 i0 = (i64)blockIdx.x * rows;
    const int n = a.n - i0 < rows ? (int)(a.n - i0) : rows;
    for (int r = threadIdx.x; r < n; r += 256) {
        A s = 0;
        for (int j = 0; j < a.k; ++j) {
            const i64 at = (i0 + r) * a.k + j;
            if (a.labels[at] >= 0) s += ((const A *)a.weights)[at] * ((const A *)a.dweights)[at];
        }
        sums[r] = s;
        if (!a.renormalise) {
            tops[r] = ((const A *)a.stats)[2 * (i0 + r)];
            scales[r] = tops[r] > neg_inf<A>() ? s / ((const A *)a.stats)[2 * (i0 + r) + 1] : (A)0;
        }
    }
    __syncthreads();
    const auto spread = [&](int r, i64 c) {                     // the softmax over all
        const A l = (A)((const T *)a.l)[(i0 + r) * a.stride + c];
        return l > neg_inf<A>() && tops[r] > neg_inf<A>() ? -scales[r] * ratio(l, tops[r]) : (A)0;
    };
    T *out = (T *)a.dl + i0 * a.K;
    const i64 size = (i64)n * a.K;
    if (a.renormalise) {
        constexpr int E = 16 / (int)sizeof(T);
        struct alignas(16) Zeros { T e[E]; };
        Zeros z;
#pragma unroll
        for (int q = 0; q < E; ++q) z.e[q] = (T)0.0f;
        const i64 whole = ((uintptr_t)out & 15) == 0 ? size / E : 0;
        for (i64 g = threadIdx.x; g < whole; g += 256) ((Zeros *)out)[g] = z;
        for (i64 x = whole * E + threadIdx.x; x < size; x += 256) out[x] = (T)0.0f;
    } else {
        for (i64 x = threadIdx.x; x < size; x += 256) out[x] = (T)spread((int)(x / a.K), x % a.K);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < n * a.k; x += 256) {
        const int r = x / a.k;
        const i64 at = i0 * a.k + x;
        const i64 c = a.labels[at];
        if (c < 0) continue;
        const A w = ((const A *)a.weights)[at], g = ((const A *)a.dweights)[at];
        out[(i64)r * a.K + c] = (T)(a.renormalise ? w * (g - sums[r]) : spread(r, c) + w * g);
    }
}

// The form for this K and k: 8 lanes up to 16 elements each, then 16, 32, 64 -- at least k --, then workgroups.  A lane has 16 elements or
// the least of 4, 8 and 14 that hold the row: every element costs six instructions a round (k = 4, shares of all, 14 and 16: 1e6 x 200
// double 478 and 520 us, 1e6 x 400 952 and 1046, 1e6 x 201 single 305 and 316, 1e6 x 101 bfloat16 122 and 130; 12 in 14's place serve
// 1e6 x 180 double, 420 and 457, but not 193 to 224).
template <class T, int G, int E> void route_by_size(const RouteArgs &a, hipStream_t st) {
    const int need = (a.K + G * E - 1) / (G * E);
    constexpr int kMost = 16 / E;
    const dim3 g((unsigned)((a.n + 256 / G - 1) / (256 / G)));
    if (need <= (kMost + 3) / 4) route_rows_kernel<T, G, (kMost + 3) / 4, E><<<g, 256, 0, st>>>(a);
    else if (need <= kMost / 2) route_rows_kernel<T, G, (kMost + 1) / 2, E><<<g, 256, 0, st>>>(a);
    else if (need <= (kMost * 7 + 7) / 8 && kMost > 4) route_rows_kernel<T, G, (kMost * 7 + 7) / 8, E><<<g, 256, 0, st>>>(a);
    else route_rows_kernel<T, G, kMost, E><<<g, 256, 0, st>>>(a);
}
template <class T, int E> void route_by_width(const RouteArgs &a, hipStream_t st) {
    const dim3 g((unsigned)(a.n < (1 << 20) ? a.n : 1 << 20));
    if (a.K <= 8 * 16 && a.k <= 8) route_by_size<T, 8, E>(a, st);
    else if (a.K <= 16 * 16 && a.k <= 16) route_by_size<T, 16, E>(a, st);
    else if (a.K <= 32 * 16) route_by_size<T, 32, E>(a, st);
    else if (a.K <= 64 * 16) route_by_size<T, 64, E>(a, st);
    else if (a.K <= 4096) route_wide_kernel<T, 4, true, E><<<g, 256, 0, st>>>(a);
    else if (a.K <= 16384) route_wide_kernel<T, 16, true, E><<<g, 1024, 0, st>>>(a);
    else route_wide_kernel<T, 16, false, 1><<<g, 1024, 0, st>>>(a);
}

// Rows of a launch: a launch's threads are counted in 32 bits.
constexpr i64 kRowsAtOnce = (i64)1 << 25;

int check(const char *what, int dtype, i64 n, int K, int k, i64 stride) {
    if (dtype < BGMM_F64 || dtype > BGMM_BF16) return ops_fail(BGMM_OPS_EINVAL, "%s: element type %d", what, dtype);
    if (n < 0 || K < 1 || k < 1 || k > K || stride < 0)
        return ops_fail(BGMM_OPS_EINVAL, "%s: n = %lld, K = %d, k = %d, stride %lld", what, (long long)n, K, k, (long long)stride);
    if (k > BGMM_OPS_MAX_CHOSEN) return ops_fail(BGMM_OPS_EUNSUPPORTED, "%s: k = %d (at most %d)", what, k, BGMM_OPS_MAX_CHOSEN);
    if (n > ((i64)1 << 32)) return ops_fail(BGMM_OPS_EUNSUPPORTED, "%s: n = %lld rows (at most 2^32)", what, (long long)n);
    return BGMM_OPS_OK;
}

}  // namespace

extern "C" int bgmm_route(int32_t dtype, const void *log_weights, int64_t stride, int64_t n, int32_t K, int32_t k, int32_t renormalise,
                          int64_t *labels, void *weights, void *stats, void *stream) {
    const int rc = check("route", dtype, n, K, k, stride);
    if (rc || n == 0) return rc;
    if (!log_weights || !labels || !weights) return ops_fail(BGMM_OPS_EINVAL, "route: a null pointer");
    const hipStream_t st = (hipStream_t)stream;
    return by_type(dtype, [&](auto *t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        constexpr int E = 16 / (int)sizeof(T);
        // 16 bytes a load where rows begin on them, else an element (n = 1e6, K = 200, double: 299 and 411 us; 1e5 x 64 bfloat16: 10.3, 11.4)
        const bool vec = ((uintptr_t)log_weights & 15) == 0 && stride % E == 0 && K % E == 0;
        typedef typename Acc<T>::type A;
        for (i64 i = 0; i < n; i += kRowsAtOnce) {
            const RouteArgs a = {(const T *)log_weights + i * stride, stride, n - i < kRowsAtOnce ? n - i : kRowsAtOnce, K, k, renormalise != 0, labels + i * k,
                                 (A *)weights + i * k, stats ? (A *)stats + 2 * i : nullptr, nullptr, nullptr};
            vec ? route_by_width<T, E>(a, st) : route_by_width<T, 1>(a, st);
        }
        return ops_launched("route");
    });
}

extern "C" int bgmm_route_backward(int32_t dtype, const void *log_weights, int64_t stride, int64_t n, int32_t K, int32_t k, int32_t renormalise,
                                   const int64_t *labels, const void *weights, const void *stats, const void *dweights, void *dlog_weights,
                                   void *stream) {
    const int rc = check("route_backward", dtype, n, K, k, stride);
    if (rc || n == 0) return rc;
    if (!labels || !weights || !dweights || !dlog_weights || (!renormalise && (!log_weights || !stats)))
        return ops_fail(BGMM_OPS_EINVAL, "route_backward: a null pointer");
    // rows of a workgroup: about 8192 elements, a multiple of eight (so that stretches of any K start on 16 bytes)
    int rows = 8;
    while (rows < kBackRows && (i64)rows * K < 8192) rows *= 2;
    return by_type(dtype, [&](auto *t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        typedef typename Acc<T>::type A;
        for (i64 i = 0; i < n; i += kRowsAtOnce) {
            const i64 m = n - i < kRowsAtOnce ? n - i : kRowsAtOnce;
            const RouteArgs a = {log_weights ? (const T *)log_weights + i * stride : nullptr, stride, m, K, k, renormalise != 0, (int64_t *)labels + i * k,
                                 (A *)weights + i * k, stats ? (A *)stats + 2 * i : nullptr, (const A *)dweights + i * k, (T *)dlog_weights + i * K};
            route_backward_kernel<T><<<dim3((unsigned)((m + rows - 1) / rows)), 256, 0, (hipStream_t)stream>>>(a, rows);
        }
        return ops_launched("route_backward");
    });
}
