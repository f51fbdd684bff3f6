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
// Bound by reading one row of the target (and of the draft) per sequence, and for a few sequences by the latency of the chain
// label -> its probabilities -> the row.  Up to 2048 labels a wave has a sequence and its row in registers, one launch.  Beyond,
// a workgroup sums a chunk of a row (16-byte loads, however the row is aligned), so that one sequence already fills many
// compute units, and a second launch finds the chunk that holds the draw and reads only that again.  20000 sequences of 200 doubles:
// 16.2 us, 3.5 TB/s; 256 of 131072 bfloat16: 33 us, 3.7 TB/s; one of 50000 singles: 9 us, the chain of loads twice.
#include "ops_common.h"

namespace {

struct VerifyArgs {
    const void *target, *draft;             // [B][T + 1][V], [B][T][V]: strides in elements, the last axis contiguous
    i64 target_b, target_t, draft_b, draft_t;
    const int64_t *labels;                  // [B][T]
    const double *u_accept, *u_draw;        // [B][T], [B]
    const int64_t *lengths;                 // [B], or null: T
    int B, T;
    int first;                              // of a launch's sequences
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

// The drafts accepted: the same for every lane of every wave that asks.  Everything about the first 64 drafts is asked for at
// once, the length too; *z0: the label that was drafted at this lane's place.
template <class T> __device__ __forceinline__ int accepted_drafts(const VerifyArgs &a, i64 b, int *length, i64 *z0) {
    const int lane = wave_lane();
    i64 len = a.lengths ? a.lengths[b] : a.T;
    const T *tgt = (const T *)a.target + b * a.target_b, *dft = (const T *)a.draft + b * a.draft_b;
    int acc = 0;
    *z0 = -1;
    for (int t0 = 0; t0 < a.T; t0 += 64) {
        const int t = t0 + lane;
        bool ok = false;
        if (t < a.T) {
            const i64 z = a.labels[b * a.T + t];
            const double u = a.u_accept[b * a.T + t];
            if (t0 == 0) *z0 = z;
            if (z >= 0 && z < a.V) ok = u * clean(dft[t * a.draft_t + z]) < clean(tgt[t * a.target_t + z]);
        }
        const unsigned long long bad = __ballot(!ok || t >= len);       // (the length ends the run)
        const int run = bad ? __ffsll(bad) - 1 : 64;
        acc += run;
        if (run < 64) break;
    }
    len = len < 0 ? 0 : len > a.T ? a.T : len;
    *length = (int)len;
    return acc;
}

// One wave writes a sequence's results.
__device__ __forceinline__ void write_labels(const VerifyArgs &a, i64 b, int acc, i64 drawn, i64 z0) {
    const int lane = wave_lane();
    if (lane <= a.T) a.out[b * (a.T + 1) + lane] = lane < acc ? z0 : lane == acc ? drawn : -1;
    for (int t = lane + 64; t <= a.T; t += 64) a.out[b * (a.T + 1) + t] = t < acc ? a.labels[b * a.T + t] : t == acc ? drawn : -1;
    if (lane == 0) a.accepted[b] = acc;
}

// 16 bytes of a row at any alignment its elements have
template <class T> constexpr int kPack = 16 / (int)sizeof(T);
template <class T, int E = kPack<T>> __device__ __forceinline__ void load_pack(const T *p, T *v) {
    if constexpr (E == 1) {
        *v = *p;
    } else {
        struct Pack { T e[E]; };
        const Pack k = load_any<Pack>(p);
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = k.e[j];
    }
}

// The row's packs of this lane, NG x 64 of them in all (V >= E).  One that reaches over the row's end is read where it ends with the
// row, so that no load has a branch around it ...
template <class T, int NG, int E> __device__ __forceinline__ void load_row(const T *p, int V, T *v) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const int c = (g * 64 + wave_lane()) * E;
        load_pack<T, E>(p + (c + E <= V ? c : V - E), v + g * E);
    }
}
// ... and shifted to its place here, zeros behind it (apart, so that a second row is asked for before the first one is waited for).
template <class T, int NG, int E> __device__ __forceinline__ void end_row(int V, T *v) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        if ((g + 1) * 64 * E <= V) continue;
        const int behind = (g * 64 + wave_lane()) * E + E - V;
        if constexpr (E == 1) {
            if (behind > 0) v[g] = (T)0.0f;
        } else {
            struct Pack { T e[E]; } k;
#pragma unroll
            for (int j = 0; j < E; ++j) k.e[j] = v[g * E + j];
            unsigned __int128 bits = __builtin_bit_cast(unsigned __int128, k);
            if (behind > 0) bits = behind < E ? bits >> (behind * 8 * (int)sizeof(T)) : 0;
            k = __builtin_bit_cast(Pack, bits);
#pragma unroll
            for (int j = 0; j < E; ++j) v[g * E + j] = k.e[j];
        }
    }
}

// ---- few labels: a wave per sequence has its row in registers, NG packs a lane.  The sums run over a lane's pack, then over the lanes.
template <class T, int NG, int E> __global__ __launch_bounds__(256) void verify_rows_kernel(VerifyArgs a) {
    const i64 b = (i64)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= a.B) return;
    const int lane = wave_lane(), V = (int)a.V;
    const double u = a.u_draw[b];
    int len;
    i64 z0;
    const int acc = accepted_drafts<T>(a, b, &len, &z0);
    const bool has_q = acc < len;
    T p[NG * E], q[NG * E];
    load_row<T, NG, E>((const T *)a.target + b * a.target_b + acc * a.target_t, V, p);
    if (has_q) load_row<T, NG, E>((const T *)a.draft + b * a.draft_b + acc * a.draft_t, V, q);
    end_row<T, NG, E>(V, p);
    if (has_q) end_row<T, NG, E>(V, q);
    double res[NG * E], total = 0;
#pragma unroll
    for (int j = 0; j < NG * E; ++j) {
        const double r = has_q ? clean(p[j]) - clean(q[j]) : clean(p[j]);
        res[j] = r > 0 ? r : 0.0;
        total += res[j];
    }
    total = group_sum<64>(total);
    if (has_q && !(total > 0)) {
        total = 0;
#pragma unroll
        for (int j = 0; j < NG * E; ++j) {
            res[j] = clean(p[j]);
            total += res[j];
        }
        total = group_sum<64>(total);
    }
    const double goal = u * total;
    double before = 0;
    int drawn = -1;
    bool found = false;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        if (found || g * 64 * E >= V) continue;
        double x = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) x += res[g * E + j];
        const double s = wave_scan_sum(x);
        const unsigned long long pos = __ballot(x > 0), hit = __ballot(x > 0 && before + s > goal);
        if (hit | pos) {
            // in the lane that has it: the first of its pack beyond the goal (else, by rounding, the last one with any weight)
            double at = before + (s - x);
            int mine = -1;
            bool over = false;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                at += res[g * E + j];
                if (!over && res[g * E + j] > 0) {
                    mine = j;
                    over = at > goal;
                }
            }
            const int l = hit ? __ffsll(hit) - 1 : 63 - __clzll(pos);
            drawn = (g * 64 + l) * E + __builtin_amdgcn_readlane(mine, l);
            found = hit != 0;
        }
        before += lane_read(s, 63);
    }
    write_labels(a, b, acc, drawn, z0);
}

// ---- many labels: chunks of a row
// Sums of max(0, p - q) (p where q is null) and of p over [lo, hi) by `n` threads, this one the `me`-th.
template <class T> __device__ __forceinline__ void sum_span(const T *p, const T *q, i64 lo, i64 hi, int me, int n, double *res, double *all) {
    constexpr int E = kPack<T>;
    double r = 0, s = 0;
    i64 j = lo + (i64)me * E;
    for (; j + E <= hi; j += (i64)n * E) {
        T x[E], y[E];
        load_pack(p + j, x);
        if (q) load_pack(q + j, y);
#pragma unroll
        for (int c = 0; c < E; ++c) {
            const double w = clean(x[c]);
            s += w;
            if (q) {
                const double d = w - clean(y[c]);
                r += d > 0 ? d : 0.0;
            }
        }
    }
    for (; j < hi && j < lo + (hi - lo + E - 1) / E * E; ++j) {          // (the last, shorter pack: one thread's)
        const double w = clean(p[j]);
        s += w;
        if (q) {
            const double d = w - clean(q[j]);
            r += d > 0 ? d : 0.0;
        }
    }
    *all = s;
    *res = q ? r : s;
}

// ws: [B][chunks][2] sums, [B] accepted, [B] lengths
struct VerifyWs {
    double *sums;
    int *acc, *len;
    int chunks;
    i64 chunk;
};

template <class T> __global__ __launch_bounds__(256) void verify_sums_kernel(VerifyArgs a, VerifyWs w) {
    __shared__ double part[4][2];
    const i64 b = a.first + blockIdx.x / w.chunks;
    const int c = (int)(blockIdx.x % w.chunks);
    int len;
    i64 z0;
    const int acc = accepted_drafts<T>(a, b, &len, &z0);
    const T *p = (const T *)a.target + b * a.target_b + acc * a.target_t;
    const T *q = acc < len ? (const T *)a.draft + b * a.draft_b + acc * a.draft_t : nullptr;
    const i64 lo = c * w.chunk, hi = lo + w.chunk < a.V ? lo + w.chunk : a.V;
    double res, all;
    sum_span(p, q, lo, hi, threadIdx.x, 256, &res, &all);
    res = group_sum<64>(res);
    all = group_sum<64>(all);
    if (wave_lane() == 0) {
        part[threadIdx.x >> 6][0] = res;
        part[threadIdx.x >> 6][1] = all;
    }
    __syncthreads();
    if (threadIdx.x < 2) w.sums[((i64)b * w.chunks + c) * 2 + threadIdx.x] = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
    if (c == 0 && threadIdx.x == 0) {
        w.acc[b] = acc;
        w.len[b] = len;
    }
}

// The part that holds the goal, from n sums in memory: the first whose running sum exceeds it (else, by rounding, the last with
// any weight; -1: none has).  *before becomes the sum in front of it.  One wave.
template <class F> __device__ __forceinline__ int pick(int n, F sum_of, double goal, double *before) {
    int last = -1;
    double at = *before;
    for (int c0 = 0; c0 < n; c0 += 64) {
        const int c = c0 + wave_lane();
        const double x = c < n ? sum_of(c) : 0.0;
        const double s = wave_scan_sum(x);
        const unsigned long long pos = __ballot(x > 0), hit = __ballot(x > 0 && at + s > goal);
        const int l = hit ? __ffsll(hit) - 1 : pos ? 63 - __clzll(pos) : -1;
        if (l >= 0) {
            last = c0 + l;
            *before = at + lane_read(s - x, l);
        }
        if (hit) break;
        at += lane_read(s, 63);
    }
    return last;
}

template <class T, int W> __global__ __launch_bounds__(64 * W) void verify_draw_kernel(VerifyArgs a, VerifyWs w) {
    __shared__ double part[W];
    const i64 b = a.first + blockIdx.x;
    const int acc = w.acc[b], len = w.len[b], wave = threadIdx.x >> 6;
    const T *p = (const T *)a.target + b * a.target_b + acc * a.target_t;
    const T *q = acc < len ? (const T *)a.draft + b * a.draft_b + acc * a.draft_t : nullptr;
    const double *sums = w.sums + b * w.chunks * 2;
    // every wave picks the chunk for itself
    double total[2] = {0, 0};
    for (int c = wave_lane(); c < w.chunks; c += 64) {
        total[0] += sums[2 * c];
        total[1] += sums[2 * c + 1];
    }
    const double res = group_sum<64>(total[0]), all = group_sum<64>(total[1]);
    const int which = res > 0 ? 0 : 1;
    if (which) q = nullptr;
    const double goal = a.u_draw[b] * (which ? all : res);
    double before = 0;
    const int c = pick(w.chunks, [&](int j) { return sums[2 * j + which]; }, goal, &before);
    i64 drawn = -1;
    if (c >= 0) {
        // a part of the chunk per wave; then 64 labels at a time
        const i64 lo = c * w.chunk, hi = lo + w.chunk < a.V ? lo + w.chunk : a.V;
        const i64 len1 = ((hi - lo + W - 1) / W + 63) & ~(i64)63;
        const i64 lo1 = lo + wave * len1 < hi ? lo + wave * len1 : hi, hi1 = lo1 + len1 < hi ? lo1 + len1 : hi;
        double r, s;
        sum_span(p, q, lo1, hi1, wave_lane(), 64, &r, &s);
        r = group_sum<64>(r);
        if (wave_lane() == 0) part[wave] = r;
        __syncthreads();
        if (wave == 0) {
            const int k = pick(W, [&](int j) { return part[j]; }, goal, &before);
            if (k >= 0) {
                const i64 lo2 = lo + k * len1, hi2 = lo2 + len1 < hi ? lo2 + len1 : hi;
                const int j = pick((int)(hi2 - lo2), [&](int x) { return weight(p, q, lo2 + x); }, goal, &before);
                if (j >= 0) drawn = lo2 + j;
            }
        }
    }
    if (wave == 0) write_labels(a, b, acc, drawn, wave_lane() < a.T ? a.labels[b * a.T + wave_lane()] : -1);
}

// Labels per chunk: enough workgroups for the chip (two thousand), at least 4096.
i64 chunk_of(i64 B, i64 V) {
    i64 chunk = 4096;
    while (chunk < 32768 && B * ((V + chunk - 1) / chunk) > 4096) chunk *= 2;
    return chunk;
}
// A wave has the row in registers, by packs of 16 bytes beyond 256 labels (20000 sequences of 200 bfloat16: 21.5 us by packs, 18.3
// one by one; of 1000 singles: 30 by packs, 59 one by one, 207 by chunks; 5000 of 2000 singles: 23, 38 by chunks; one: 6.6 and 8.5).
bool few_labels(i64 V) { return V <= 2048; }
template <class T> void verify_few(const VerifyArgs &a, hipStream_t st) {
    constexpr int E = kPack<T>;
    const dim3 g((unsigned)((a.B + 3) / 4));
    if (a.V <= 64) verify_rows_kernel<T, 1, 1><<<g, 256, 0, st>>>(a);
    else if (a.V <= 256) verify_rows_kernel<T, 4, 1><<<g, 256, 0, st>>>(a);
    else if (a.V <= 512) verify_rows_kernel<T, 8 / E, E><<<g, 256, 0, st>>>(a);
    else if (a.V <= 1024) verify_rows_kernel<T, 16 / E, E><<<g, 256, 0, st>>>(a);
    else verify_rows_kernel<T, 32 / E, E><<<g, 256, 0, st>>>(a);
}

}  // namespace

extern "C" int64_t bgmm_verify_drafts_ws(int64_t B, int64_t V) {
    if (B < 1 || V < 1 || few_labels(V)) return 0;
    const i64 chunk = chunk_of(B, V);
    return B * ((V + chunk - 1) / chunk) * 16 + B * 8;
}

extern "C" int bgmm_verify_drafts(int32_t dtype, const void *target, int64_t target_b, int64_t target_t, const void *draft, int64_t draft_b,
                                  int64_t draft_t, const int64_t *labels, const double *u_accept, const double *u_draw, const int64_t *lengths,
                                  int64_t B, int32_t T, int64_t V, int64_t *out, int64_t *accepted, void *ws, int64_t ws_bytes, void *stream) {
    if (dtype < BGMM_F64 || dtype > BGMM_BF16) return ops_fail(BGMM_OPS_EINVAL, "verify_drafts: element type %d", dtype);
    if (B < 0 || T < 0 || T > (1 << 20) || V < 1 || target_b < 0 || target_t < 0 || draft_b < 0 || draft_t < 0)
        return ops_fail(BGMM_OPS_EINVAL, "verify_drafts: B = %lld, T = %d, V = %lld", (long long)B, T, (long long)V);
    if (B > (1 << 24) || V > 0x7fffffff - 65536) return ops_fail(BGMM_OPS_EUNSUPPORTED, "verify_drafts: B = %lld (at most 2^24), V = %lld (at most 2^31 - 65537)", (long long)B, (long long)V);
    if (B == 0) return BGMM_OPS_OK;
    if (!target || !u_draw || !out || !accepted || (T > 0 && (!draft || !labels || !u_accept)))
        return ops_fail(BGMM_OPS_EINVAL, "verify_drafts: a null pointer");
    const i64 need = bgmm_verify_drafts_ws(B, V);
    if (ws_bytes < need || (need > 0 && (!ws || ((uintptr_t)ws & 7)))) return ops_fail(BGMM_OPS_EINVAL, "verify_drafts: workspace of %lld bytes", (long long)ws_bytes);
    VerifyArgs a = {target, draft, target_b, target_t, draft_b, draft_t, labels, u_accept, u_draw, lengths, (int)B, T, 0, V, out, accepted};
    const hipStream_t st = (hipStream_t)stream;
    VerifyWs w = {};
    if (need > 0) {
        w.chunk = chunk_of(B, V);
        w.chunks = (int)((V + w.chunk - 1) / w.chunk);
        w.sums = (double *)ws;
        w.acc = (int *)(w.sums + B * w.chunks * 2);
        w.len = w.acc + B;
    }
    return by_type(dtype, [&](auto *t) {
        typedef std::remove_pointer_t<decltype(t)> E;
        if (few_labels(V)) {
            verify_few<E>(a, st);
        } else {
            // (a sequence has at most 2^19 chunks)
            const auto parts = [&](i64 each, auto launch) {
                for (i64 b = 0; b < B; b += each) {
                    a.first = (int)b;
                    launch((unsigned)(B - b < each ? B - b : each));
                }
            };
            parts(kThreadsAtOnce / 256 / w.chunks, [&](unsigned n) { verify_sums_kernel<E><<<dim3(n * (unsigned)w.chunks), 256, 0, st>>>(a, w); });
            // few sequences: more waves for the latency of each (5000 sequences of 2000 singles: 38 us with 4, 68 with 16)
            if (B > 512) parts(kThreadsAtOnce / 256, [&](unsigned n) { verify_draw_kernel<E, 4><<<dim3(n), 256, 0, st>>>(a, w); });
            else parts(B, [&](unsigned n) { verify_draw_kernel<E, 16><<<dim3(n), 1024, 0, st>>>(a, w); });
        }
        return ops_launched("verify_drafts");
    });
}
