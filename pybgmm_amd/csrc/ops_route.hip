// The k most probable components of every row of log weights, and their weights (include/bgmm_ops.h: bgmm_route).
//
//   chosen: the first k of the components ordered by (log weight descending, index ascending); -inf and NaN never
//   w_j = exp(l_j - m) / total,  m = the row's maximum,  total = the sum over the chosen ones, or over all
//   gradient, g the weights':    renormalised   dl_j = w_j (g_j - sum_c w_c g_c) on the chosen, 0 elsewhere
//                                over all       dl_i = [i chosen] w_i g_i - p_i sum_c w_c g_c
//
// The order makes marking unnecessary: the next one chosen is the largest that comes strictly after the last.  Bound by reading
// the row once (forward) and writing its gradient once (backward).
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

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// exp(v - m) with v == m exactly 1, infinities included
template <class A> __device__ __forceinline__ A ratio(A v, A m) { return v == m ? (A)1 : exp_of(v - m); }

// One wave per row; the row is read again for every chosen component (from the caches).
template <class T> __global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
    typedef typename Acc<T>::type A;
    const int lane = wave_lane();
    const i64 i = (i64)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= a.n) return;
    const T *row = (const T *)a.l + i * a.stride;
    A top = neg_inf<A>(), last = 0, mine = neg_inf<A>();
    int last_at = -1, mine_at = -1;
    for (int j = 0; j < a.k; ++j) {
        A best = neg_inf<A>();
        int at = 0x7fffffff;
        for (int c = lane; c < a.K; c += 64) {
            const A v = (A)row[c];
            const bool after = j == 0 || v < last || (v == last && c > last_at);
            if (after && v > best) { best = v; at = c; }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const A ov = __shfl_xor(best, o);
            const int oa = __shfl_xor(at, o);
            if (ov > best || (ov == best && oa < at)) { best = ov; at = oa; }
        }
        if (best == neg_inf<A>()) break;
        if (j == 0) top = best;
        if (lane == j) { mine = best; mine_at = at; }
        last = best;
        last_at = at;
    }
    A total = 0;
    if (a.renormalise) {
        total = mine_at >= 0 ? ratio(mine, top) : (A)0;
    } else if (top > neg_inf<A>()) {
        for (int c = lane; c < a.K; c += 64) {
            const A v = (A)row[c];
            if (v > neg_inf<A>()) total += ratio(v, top);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    if (lane < a.k) {
        a.labels[i * a.k + lane] = mine_at;
        ((A *)a.weights)[i * a.k + lane] = mine_at >= 0 ? ratio(mine, top) / total : (A)0;
    }
    if (a.stats && lane == 0) {
        ((A *)a.stats)[2 * i] = top;
        ((A *)a.stats)[2 * i + 1] = total;
    }
}

template <class T> __global__ __launch_bounds__(256) void route_backward_kernel(RouteArgs a) {
    typedef typename Acc<T>::type A;
    const int lane = wave_lane();
    const i64 i = (i64)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= a.n) return;
    A w = 0, g = 0;
    int at = -1;
    if (lane < a.k) {
        at = (int)a.labels[i * a.k + lane];
        if (at >= 0) {
            w = ((const A *)a.weights)[i * a.k + lane];
            g = ((const A *)a.dweights)[i * a.k + lane];
        }
    }
    const A wg = w * g;
    A s = wg;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    const A d = a.renormalise ? w * (g - s) : wg;
    A top = 0, scale = 0;
    if (!a.renormalise) {
        top = ((const A *)a.stats)[2 * i];
        const A total = ((const A *)a.stats)[2 * i + 1];
        scale = top > neg_inf<A>() ? s / total : (A)0;
    }
    const T *row = (const T *)a.l + i * a.stride;
    T *out = (T *)a.dl + i * a.K;
    for (int c0 = 0; c0 < a.K; c0 += 64) {
        const int c = c0 + lane;
        A v = 0;
        if (!a.renormalise && c < a.K) {
            const A l = (A)row[c];
            if (l > neg_inf<A>() && top > neg_inf<A>()) v = -scale * ratio(l, top);
        }
        for (int j = 0; j < a.k; ++j) {
            const A dj = __shfl(d, j);
            if (__shfl(at, j) == c) v += dj;
        }
        if (c < a.K) out[c] = (T)v;
    }
}

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
    RouteArgs a = {log_weights, stride, n, K, k, renormalise != 0, labels, weights, stats, nullptr, nullptr};
    const dim3 g((unsigned)((n + 3) / 4));
    return by_type(dtype, [&](auto *t) {
        route_kernel<std::remove_pointer_t<decltype(t)>><<<g, 256, 0, (hipStream_t)stream>>>(a);
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
    RouteArgs a = {log_weights, stride, n, K, k, renormalise != 0, (int64_t *)labels, (void *)weights, (void *)stats, dweights, dlog_weights};
    const dim3 g((unsigned)((n + 3) / 4));
    return by_type(dtype, [&](auto *t) {
        route_backward_kernel<std::remove_pointer_t<decltype(t)>><<<g, 256, 0, (hipStream_t)stream>>>(a);
        return ops_launched("route_backward");
    });
}
