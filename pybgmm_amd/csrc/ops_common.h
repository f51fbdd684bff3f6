// Shared by the operators of libbgmm_ops.so (include/bgmm_ops.h): element types, wave helpers, error reporting.
#pragma once
#include "../../include/bgmm_ops.h"

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

typedef long long i64;
typedef _Float16 f16_t;
typedef __bf16 bf16_t;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef double v4d __attribute__((ext_vector_type(4)));

// What an element type accumulates in.
template <class T> struct Acc { typedef float type; typedef v4f v4; };
template <> struct Acc<double> { typedef double type; typedef v4d v4; };

// The tiles of a grouping's products: 16 rows where components have up to 16 on average, 128 beyond (1000 components, 64 x 64 double,
// 16 rows each: 18 us against 24 with 128; 64 experts, 1024 x 1024 bfloat16, bound by their weights' 134 MB: 16 rows each 26 and
// 25 us, 64 rows each 45 and 27 us).  At most this many, those of the rows of no component included, in whole blocks of eight.
inline bool small_tiles(i64 P, int K) { return P <= 16 * (i64)K; }
inline int tile_log2(i64 P, int K) { return small_tiles(P, K) ? 4 : 7; }
inline i64 tiles_at_most(i64 P, int K) { return ((P >> tile_log2(P, K)) + (K < P ? K : P) + 8) & ~(i64)7; }

// f(a null pointer of the element type's own): the dispatch of the C entry points, whose checks know the four types
template <class F> int by_type(int dtype, F f) {
    switch (dtype) {
    case BGMM_F64: return f((double *)nullptr);
    case BGMM_F32: return f((float *)nullptr);
    case BGMM_F16: return f((f16_t *)nullptr);
    default: return f((bf16_t *)nullptr);
    }
}

int ops_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int ops_launched(const char *what);         // the status of the launch just made

// Threads of a launch: they are counted in 32 bits.  What needs more is launched in parts.
constexpr i64 kThreadsAtOnce = (i64)1 << 31;

__device__ __forceinline__ int wave_lane() { return threadIdx.x & 63; }

// N bytes (4, 8, 16 or 32) from or to memory as one access per 16, at whatever alignment p has.  (Through a vector of words: element
// by element the compiler would put the pieces together again as it likes.)
typedef unsigned words1 __attribute__((ext_vector_type(1)));
typedef unsigned words2 __attribute__((ext_vector_type(2)));
typedef unsigned words4 __attribute__((ext_vector_type(4)));
template <int N> struct WordsOf { typedef words4 type; };
template <> struct WordsOf<4> { typedef words1 type; };
template <> struct WordsOf<8> { typedef words2 type; };
template <class R> __device__ __forceinline__ R load_any(const void *p) {
    constexpr int kEach = sizeof(R) < 16 ? (int)sizeof(R) : 16, kNum = (int)sizeof(R) / kEach;
    typedef typename WordsOf<kEach>::type W;
    struct __attribute__((packed, may_alias)) Loose { W w; };
    struct All { W w[kNum]; } all;
#pragma unroll
    for (int i = 0; i < kNum; ++i) all.w[i] = ((const Loose *)p)[i].w;
    return __builtin_bit_cast(R, all);
}
template <class R> __device__ __forceinline__ void store_any(void *p, const R &r) {
    constexpr int kEach = sizeof(R) < 16 ? (int)sizeof(R) : 16, kNum = (int)sizeof(R) / kEach;
    typedef typename WordsOf<kEach>::type W;
    struct __attribute__((packed, may_alias)) Loose { W w; };
    struct All { W w[kNum]; };
    const All all = __builtin_bit_cast(All, r);
#pragma unroll
    for (int i = 0; i < kNum; ++i) ((Loose *)p)[i].w = all.w[i];
}

// Lanes of the wave whose `key` (bits 0 .. nbits-1) equals this lane's; inactive lanes are in no group.
__device__ __forceinline__ unsigned long long wave_match(int key, int nbits, bool active) {
    unsigned long long m = __ballot(active);
    for (int b = 0; b < nbits; ++b) {
        const unsigned long long set = __ballot((key >> b) & 1);
        m &= ((key >> b) & 1) ? set : ~set;
    }
    return m;
}

// Exchange within a row of 16 lanes without the LDS crossbar; all-reduce of groups of G lanes (8, 16, 32, 64).
template <int CTRL> __device__ __forceinline__ int lane_move(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false); }
template <int CTRL> __device__ __forceinline__ float lane_move(float v) { return __int_as_float(lane_move<CTRL>(__float_as_int(v))); }
template <int CTRL> __device__ __forceinline__ double lane_move(double v) {
    return __hiloint2double(lane_move<CTRL>(__double2hiint(v)), lane_move<CTRL>(__double2loint(v)));
}
template <int G, class V, class F> __device__ __forceinline__ V group_reduce(V v, F f) {
    v = f(v, lane_move<0xB1>(v));                   // quad_perm [1,0,3,2]
    v = f(v, lane_move<0x4E>(v));                   // quad_perm [2,3,0,1]
    v = f(v, lane_move<0x141>(v));                  // row_half_mirror
    if (G >= 16) v = f(v, lane_move<0x140>(v));     // row_mirror
    if (G >= 32) v = f(v, __shfl_xor(v, 16));
    if (G >= 64) v = f(v, __shfl_xor(v, 32));
    return v;
}
template <int G, class V> __device__ __forceinline__ V group_sum(V v) {
    return group_reduce<G>(v, [](V a, V b) { return a + b; });
}

// Inclusive sum over the wave's lanes: inside a row of 16 by row shifts, the rows' totals through readlane.
__device__ __forceinline__ double lane_read(double v, int l) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
}
__device__ __forceinline__ double wave_scan_sum(double v) {
    v += lane_move<0x111>(v);
    v += lane_move<0x112>(v);
    v += lane_move<0x114>(v);
    v += lane_move<0x118>(v);
    const double t0 = lane_read(v, 15), t1 = t0 + lane_read(v, 31), t2 = t1 + lane_read(v, 47);
    const int row = wave_lane() >> 4;
    return v + (row == 0 ? 0.0 : row == 1 ? t0 : row == 2 ? t1 : t2);
}

// Which bucket chunk t belongs to: the last b in 0 .. n-1 with first[b] <= t (first is non-decreasing, first[0] = 0, first[n] what is
// behind the last), with the bucket's and the next one's entries of `first` and `offsets`.  64 candidates per probe: one up
// to 63 buckets, two up to 4032, three beyond; the last probe brings the entries with it, so that nothing waits for another
// load.  Every wave of a workgroup finds the same answer by itself.  b < 0: t is behind the last.
struct Bucket {
    int b, first, next_first, offset, next_offset;
};
__device__ __forceinline__ Bucket find_bucket(const int *first, const int *offsets, int n, int t) {
    const int lane = wave_lane();
    int lo = 0, span = n + 1;                               // (entries 0 .. n)
    while (span > 64) {
        const int step = (span + 62) / 63;                  // (so that 64 probes overlap by one and the next entry is among them)
        const int at = lo + lane * step;
        const int v = lane * step < span ? first[at <= n ? at : n] : 0x7fffffff;
        const int below = __popcll(__ballot(v <= t && at <= n));
        lo += (below - 1) * step;
        span = step + 1 < n + 1 - lo ? step + 1 : n + 1 - lo;
    }
    const int at = lo + lane < n ? lo + lane : n;
    const int v = first[at], o = offsets[at];
    const int below = __popcll(__ballot(lane < span && v <= t));
    Bucket r;
    r.b = lo + below - 1;
    if (r.b >= n) {
        r.b = -1;
        return r;
    }
    r.first = __builtin_amdgcn_readlane(v, below - 1);
    r.offset = __builtin_amdgcn_readlane(o, below - 1);
    r.next_first = __builtin_amdgcn_readlane(v, below);
    r.next_offset = __builtin_amdgcn_readlane(o, below);
    return r;
}
