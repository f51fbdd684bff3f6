// Drafted labels verified against the target's probabilities from given uniforms (include/bgmm_ops.h: bgmm_verify_drafts).
//
//   draft t is accepted iff u_t q_t(z_t) < p_t(z_t); a = the drafts in front of the first rejection
//   a < length:  the label behind them from max(0, p_a - q_a), or from p_a where that is zero everywhere
//   a = length:  from p_a
//   a draw from weights w with the uniform v: the first label whose cumulative sum exceeds v * sum(w), the samplers' rule
//   (utils/utils.py:13-20 of the reference) without normalising first
//
// The labels that come out are distributed as if every one had been drawn from the target: min(p, q) of each label's
// probability is kept and the remainder is what max(0, p - q) holds.  All comparisons and sums are in 64 bits: probabilities of
// fewer bits are exact there, so that a draw depends on the order of the sum in the last bits of the total only.
//
// Bound by reading one row of the target (and of the draft) per sequence.  The sum over V labels is hierarchical: sixteen regions,
// one wave each, then sixteen parts of the region that holds the draw, then a scan of 64 labels at a time: V (1 + 1/16 + 1/256)
// reads and no table whose size would bound V.
#include "ops_common.h"

namespace {

struct VerifyArgs {
    const void *target, *draft;             // [B][T + 1][V], [B][T][V]: strides in elements, the last axis contiguous
    i64 target_b, target_t, draft_b, draft_t;
    const int64_t *labels;                  // [B][T]
    const double *u_accept, *u_draw;        // [B][T], [B]
    const int64_t *lengths;                 // [B], or null: T
    int B, T;
    i64 V;
    int64_t *out, *accepted;                // [B][T + 1], [B]
};

// what is not a positive finite number counts as zero
template <class T> __device__ __forceinline__ double clean(T v) {
    const double d = (double)v;
    return d > 0 && d < __builtin_inf() ? d : 0.0;
}

template <class T> __device__ __forceinline__ double weight(const T *p, const T *q, i64 j) {
    const double w = clean(p[j]);
    if (!q) return w;
    const double r = w - clean(q[j]);
    return r > 0 ? r : 0.0;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

constexpr int kParts = 16;

// Sums of the sixteen parts of [lo, hi), one wave each; every thread returns with the same part that holds `target` (relative
// to the sum before lo; target < 0: none wanted) and *before = the sum in front of it.  -1: nothing positive.
template <class T>
__device__ __forceinline__ int find_part(const T *p, const T *q, i64 lo, i64 hi, double *sums, double *total, double u, double *target, double *before) {
    const int w = threadIdx.x >> 6;
    const i64 len = (hi - lo + kParts - 1) / kParts;
    const i64 a = lo + w * len < hi ? lo + w * len : hi, b = a + len < hi ? a + len : hi;
    double s = 0;
    for (i64 j = a + wave_lane(); j < b; j += 64) s += weight(p, q, j);
    s = wave_sum64(s);
    __syncthreads();
    if (wave_lane() == 0) sums[w] = s;
    __syncthreads();
    double at = *before;
    if (total) {                // the whole row: its sum gives the target
        double t = 0;
        for (int j = 0; j < kParts; ++j) t += sums[j];
        *total = t;
        *target = u * t;
    }
    int last = -1;
    double last_before = at;
    for (int j = 0; j < kParts; ++j) {
        if (sums[j] > 0) {
            last = j;
            last_before = at;
            if (at + sums[j] > *target) break;
        }
        at += sums[j];
    }
    *before = last_before;
    return last;
}

template <class T> __global__ __launch_bounds__(64 * kParts) void verify_kernel(VerifyArgs a) {
    __shared__ double sums[kParts];
    const int b = blockIdx.x, lane = wave_lane();
    // ---- acceptance: every wave finds the same
    i64 len = a.lengths ? a.lengths[b] : a.T;
    len = len < 0 ? 0 : len > a.T ? a.T : len;
    const T *tgt = (const T *)a.target + b * a.target_b, *dft = (const T *)a.draft + b * a.draft_b;
    int acc = 0;
    for (int t0 = 0; t0 < len; t0 += 64) {
        const int t = t0 + lane;
        bool ok = false;
        if (t < len) {
            const i64 z = a.labels[(i64)b * a.T + t];
            if (z >= 0 && z < a.V) ok = a.u_accept[(i64)b * a.T + t] * clean(dft[t * a.draft_t + z]) < clean(tgt[t * a.target_t + z]);
        }
        const unsigned long long bad = __ballot(!ok);       // (lanes behind the length end the run)
        const int run = bad ? __ffsll(bad) - 1 : 64;
        acc += run;
        if (run < 64) break;
    }
    const bool rejected = acc < len;
    const T *p = tgt + acc * a.target_t, *q = rejected ? dft + acc * a.draft_t : nullptr;
    // ---- the draw
    const double u = a.u_draw[b];
    double total = 0, target = 0, before = 0;
    int part = find_part(p, q, 0, a.V, sums, &total, u, &target, &before);
    if (part < 0 && q) {
        q = nullptr;
        before = 0;
        part = find_part(p, q, 0, a.V, sums, &total, u, &target, &before);
    }
    i64 drawn = -1;
    if (part >= 0) {
        i64 len1 = (a.V + kParts - 1) / kParts, lo = part * len1, hi = lo + len1 < a.V ? lo + len1 : a.V;
        part = find_part(p, q, lo, hi, sums, (double *)nullptr, u, &target, &before);
        const i64 len2 = (hi - lo + kParts - 1) / kParts;
        lo += part * len2;
        hi = lo + len2 < hi ? lo + len2 : hi;
        if (threadIdx.x < 64) {
            for (i64 j0 = lo; j0 < hi; j0 += 64) {
                const i64 j = j0 + lane;
                const double w = j < hi ? weight(p, q, j) : 0.0;
                double s = w;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const double t = __shfl_up(s, o);
                    if (lane >= o) s += t;
                }
                const unsigned long long pos = __ballot(w > 0), hit = __ballot(w > 0 && before + s > target);
                if (hit) {
                    drawn = j0 + __ffsll(hit) - 1;
                    break;
                }
                if (pos) drawn = j0 + 63 - __clzll(pos);    // (rounding: the last one with any weight)
                before += __shfl(s, 63);
            }
        }
    }
    if (threadIdx.x < 64) {
        for (int t = lane; t <= a.T; t += 64)
            a.out[(i64)b * (a.T + 1) + t] = t < acc ? a.labels[(i64)b * a.T + t] : t == acc ? drawn : -1;
        if (lane == 0) a.accepted[b] = acc;
    }
}

}  // namespace

extern "C" int bgmm_verify_drafts(int32_t dtype, const void *target, int64_t target_b, int64_t target_t, const void *draft, int64_t draft_b,
                                  int64_t draft_t, const int64_t *labels, const double *u_accept, const double *u_draw, const int64_t *lengths,
                                  int64_t B, int32_t T, int64_t V, int64_t *out, int64_t *accepted, void *stream) {
    if (dtype < BGMM_F64 || dtype > BGMM_BF16) return ops_fail(BGMM_OPS_EINVAL, "verify_drafts: element type %d", dtype);
    if (B < 0 || T < 0 || T > (1 << 20) || V < 1 || target_b < 0 || target_t < 0 || draft_b < 0 || draft_t < 0)
        return ops_fail(BGMM_OPS_EINVAL, "verify_drafts: B = %lld, T = %d, V = %lld", (long long)B, T, (long long)V);
    if (B > 0x7fffffff || V > 0x7fffffff) return ops_fail(BGMM_OPS_EUNSUPPORTED, "verify_drafts: B = %lld, V = %lld", (long long)B, (long long)V);
    if (B == 0) return BGMM_OPS_OK;
    if (!target || !u_draw || !out || !accepted || (T > 0 && (!draft || !labels || !u_accept)))
        return ops_fail(BGMM_OPS_EINVAL, "verify_drafts: a null pointer");
    VerifyArgs a = {target, draft, target_b, target_t, draft_b, draft_t, labels, u_accept, u_draw, lengths, (int)B, T, V, out, accepted};
    return by_type(dtype, [&](auto *t) {
        verify_kernel<std::remove_pointer_t<decltype(t)>><<<dim3((unsigned)B), 64 * kParts, 0, (hipStream_t)stream>>>(a);
        return ops_launched("verify_drafts");
    });
}
