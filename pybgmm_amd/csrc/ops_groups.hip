// Rows grouped by component: a stable counting sort of P labels into K + 1 buckets (bucket K: unassigned rows).
//
//   order = argsort(bucket, stable), offsets = exclusive sum of the bucket sizes,
//   first[l][b] = sum over b' < b of ceil(size(b') / (256 << l)), and the table of tiles that the products work by
//
// Stable and without atomics across workgroups, so that a grouping is the same every time: the gradients that sum over a
// group's rows in this order are too.  A wave owns a segment of consecutive rows and a histogram of its own in LDS; the 64
// rows it looks at together find their equals with one ballot per label bit.
//
// Up to kSmall rows one workgroup does everything in one launch (a single served row pays one launch, not three).  Beyond:
// histograms per segment and workgroup, an exclusive sum over the workgroups per bucket, the scatter -- bound by the
// latency of the segments' dependent LDS steps, not by the 20 P bytes that move.
#include "ops_common.h"

namespace {

constexpr int kSmall = 8192;            // rows of the one-workgroup form
constexpr int kWaves = 16;              // its waves
constexpr int kSmallBuckets = 890;      // its buckets (K + 1): 16 histograms, the sizes and the sums fit 64 KB of LDS

__device__ __forceinline__ int bucket_of(const int64_t *labels, i64 i, int K) {
    const int64_t z = labels[i];
    return z >= 0 && z < K ? (int)z : K;
}

__device__ __forceinline__ int wave_incl_scan(int v) {         // rows of 16 lanes by row shifts, their totals by readlane
    v += lane_move<0x111>(v);
    v += lane_move<0x112>(v);
    v += lane_move<0x114>(v);
    v += lane_move<0x118>(v);
    const int t0 = __builtin_amdgcn_readlane(v, 15), t1 = t0 + __builtin_amdgcn_readlane(v, 31), t2 = t1 + __builtin_amdgcn_readlane(v, 47);
    const int row = wave_lane() >> 4;
    return v + (row == 0 ? 0 : row == 1 ? t0 : row == 2 ? t1 : t2);
}

// Exclusive sum of f(0 .. n-1) over the whole workgroup, handed to g(b, sum before b); returns the total.  `part` holds one
// int per wave plus one; ends behind a barrier.
template <class F, class G>
__device__ __forceinline__ int block_scan(int n, int *part, F f, G g) {
    const int nw = blockDim.x >> 6, w = threadIdx.x >> 6;
    int carry = 0;
    for (int base = 0; base < n; base += blockDim.x) {
        const int b = base + threadIdx.x;
        const int v = b < n ? f(b) : 0;
        const int incl = wave_incl_scan(v);
        if (wave_lane() == 63) part[w] = incl;
        __syncthreads();
        int before = carry, total = 0;
        for (int j = 0; j < nw; ++j) {
            if (j < w) before += part[j];
            total += part[j];
        }
        if (b < n) g(b, before + incl - v);
        carry += total;
        __syncthreads();
    }
    return carry;
}

// All the prefix sums over buckets at once: offsets, every level's chunks, the tiles of 1 << tile_lg rows; place(b, start, tiles
// before b) sees every bucket and b = K + 1, what is behind the last.  `part`: kSums * waves ints.
constexpr int kSums = BGMM_OPS_LEVELS + 2;
template <class P> __device__ __forceinline__ void write_sums(int K, int P_rows, const int *size_of, int *offsets, int *first, int tile_lg, int *part, P place) {
    const int nw = blockDim.x >> 6, w = threadIdx.x >> 6, B = K + 1;
    int carry[kSums];
#pragma unroll
    for (int l = 0; l < kSums; ++l) carry[l] = 0;
    for (int base = 0; base < B; base += blockDim.x) {
        const int b = base + threadIdx.x, size = b < B ? size_of[b] : 0;
        int incl[kSums];
#pragma unroll
        for (int l = 0; l < kSums; ++l) {
            const int lg = l == 0 ? 0 : l == 1 ? tile_lg : 6 + l;
            const int v = (int)(((i64)size + (1 << lg) - 1) >> lg);
            const int t = wave_incl_scan(v);
            if (wave_lane() == 63) part[l * nw + w] = t;
            incl[l] = t - v;
        }
        __syncthreads();
        int sum[kSums];
#pragma unroll
        for (int l = 0; l < kSums; ++l) {
            sum[l] = carry[l] + incl[l];
            for (int j = 0; j < nw; ++j) {
                const int t = part[l * nw + j];
                if (j < w) sum[l] += t;
                carry[l] += t;
            }
        }
        if (b < B) {
            offsets[b] = sum[0];
#pragma unroll
            for (int l = 2; l < kSums; ++l) first[(i64)(l - 2) * (K + 2) + b] = sum[l];
            place(b, sum[0], sum[1]);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        offsets[B] = P_rows;
#pragma unroll
        for (int l = 2; l < kSums; ++l) first[(i64)(l - 2) * (K + 2) + B] = carry[l];
        place(B, P_rows, carry[1]);
    }
}

struct Tiles { int4 *at; int n, lg; };

// The table of tiles from a grouping's sums in LDS (starts and tile_starts: [K + 2]): a wave per bucket.
__device__ __forceinline__ void write_tiles(int K, const int *starts, const int *tile_starts, Tiles t) {
    const int lg = t.lg, nw = blockDim.x >> 6;
    for (int b = threadIdx.x >> 6; b <= K; b += nw) {
        const int start = starts[b], n = starts[b + 1] - start, t0 = tile_starts[b];
        for (int i = wave_lane(); i << lg < n; i += 64) t.at[t0 + i] = make_int4(b, start + (i << lg), n - (i << lg) < 1 << lg ? n - (i << lg) : 1 << lg, 0);
    }
    for (int i = tile_starts[K + 1] + threadIdx.x; i < t.n; i += blockDim.x) t.at[i] = make_int4(-1, 0, 0, 0);
}

// A wave walks rows [lo, hi): cursor[b] moves by the rows of bucket b = bucket_at(i), write(i, b, place) sees every row's place.
template <class L, class W>
__device__ __forceinline__ void walk(i64 lo, i64 hi, int nbits, int *cursor, L bucket_at, W write) {
    constexpr int kRound = 4;                   // rows of a lane per round; the next round's load flies meanwhile
    const int lane = wave_lane();
    int next[kRound];
    const auto load = [&](i64 i0) {
#pragma unroll
        for (int r = 0; r < kRound; ++r) {
            const i64 i = i0 + r * 64 + lane;
            next[r] = i < hi ? bucket_at(i) : 0;
        }
    };
    if (lo < hi) load(lo);
    for (i64 i0 = lo; i0 < hi; i0 += 64 * kRound) {
        int bs[kRound];
#pragma unroll
        for (int r = 0; r < kRound; ++r) bs[r] = next[r];
        if (i0 + 64 * kRound < hi) load(i0 + 64 * kRound);
#pragma unroll
        for (int r = 0; r < kRound; ++r) {
            const i64 i = i0 + r * 64 + lane;
            const bool on = i < hi;
            const int b = bs[r];
            const unsigned long long same = wave_match(b, nbits, on);
            const int leader = on ? __ffsll((unsigned long long)same) - 1 : lane;
            int at = 0;
            if (on && leader == lane) at = atomicAdd(&cursor[b], __popcll(same));   // (LDS, this wave's own counters)
            at = __shfl(at, leader);
            if (on) write(i, b, at + __popcll(same & ((1ull << lane) - 1)));
        }
    }
}

__global__ __launch_bounds__(64 * kWaves) void group_small(const int64_t *labels, int P, int K, int nbits, int *bucket, int *order,
                                                           int *offsets, int *first, Tiles tiles) {
    extern __shared__ int lds[];
    const int B = K + 1, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    int *hist = lds;                          // [waves][K + 1]
    int *sizes = hist + nw * B;               // [K + 1], later the starts [K + 2]
    int *tile_starts = sizes + B + 1;         // [K + 2]
    int *part = tile_starts + B + 1;          // [kSums * waves]
    for (int j = threadIdx.x; j < nw * B; j += blockDim.x) hist[j] = 0;
    // a wave's rows: at most kHeld rounds of 64; their buckets and places among the wave's own stay in registers
    constexpr int kHeld = kSmall / (64 * kWaves);
    const int per = ((P + nw - 1) / nw + 63) & ~63, lane = wave_lane();
    const int lo = w * per < P ? w * per : P, hi = lo + per < P ? lo + per : P;
    int held_b[kHeld], held_at[kHeld];
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
        const int i = lo + r * 64 + lane;
        held_b[r] = i < hi ? bucket_of(labels, i, K) : -1;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
        if (lo + r * 64 >= hi) break;
        const int b = held_b[r];
        const bool on = b >= 0;
        const unsigned long long same = wave_match(b, nbits, on);
        const int leader = on ? __ffsll((unsigned long long)same) - 1 : lane;
        int at = 0;
        if (on && leader == lane) at = atomicAdd(&hist[w * B + b], __popcll(same));
        held_at[r] = __shfl(at, leader) + __popcll(same & ((1ull << lane) - 1));
        if (on) bucket[lo + r * 64 + lane] = b;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        int s = 0;
        for (int j = 0; j < nw; ++j) {
            const int n = hist[j * B + b];
            hist[j * B + b] = s;
            s += n;
        }
        sizes[b] = s;
    }
    __syncthreads();
    write_sums(K, P, sizes, offsets, first, tiles.lg, part, [&](int b, int start, int tile) {
        if (b < B)
            for (int j = 0; j < nw; ++j) hist[j * B + b] += start;
        sizes[b] = start;                     // (its own size has been read)
        tile_starts[b] = tile;
    });
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
        if (lo + r * 64 + lane < hi) order[hist[w * B + held_b[r]] + held_at[r]] = lo + r * 64 + lane;
    write_tiles(K, sizes, tile_starts, tiles);
}

// within[segment][b]: the workgroup's earlier segments' rows of bucket b;  counts[workgroup][b]: all of its.
__global__ void group_count(const int64_t *labels, i64 P, int K, int seg, int nseg, int *bucket, int *within, int *counts) {
    extern __shared__ int lds[];
    const int B = K + 1, w = threadIdx.x >> 6, nw = blockDim.x >> 6, s = blockIdx.x * nw + w;
    int *hist = lds + w * B;
    for (int b = wave_lane(); b < B; b += 64) hist[b] = 0;
    __syncthreads();
    const i64 lo = (i64)s * seg < P ? (i64)s * seg : P, hi = lo + seg < P ? lo + seg : P;
#pragma unroll 4
    for (i64 i = lo + wave_lane(); i < hi; i += 64) {           // (counts need no order)
        const int b = bucket_of(labels, i, K);
        atomicAdd(&hist[b], 1);
        bucket[i] = b;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        int sum = 0;
        for (int j = 0; j < nw; ++j) {
            if (blockIdx.x * nw + j < nseg) within[(i64)(blockIdx.x * nw + j) * B + b] = sum;
            sum += lds[j * B + b];
        }
        counts[(i64)blockIdx.x * B + b] = sum;
    }
}

// One wave per bucket: counts[.][b] becomes the exclusive sum over the workgroups, sizes[b] the total.  A lane has kRun
// consecutive ones, so that a round has kRun loads in flight instead of one.
constexpr int kRun = 4;
__global__ void group_columns(int *counts, int nseg, int B, int *sizes) {
    const int b = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    if (b >= B) return;
    int carry = 0;
    for (int s0 = 0; s0 < nseg; s0 += 64 * kRun) {
        const int s = s0 + wave_lane() * kRun;
        int v[kRun], sum = 0;
#pragma unroll
        for (int r = 0; r < kRun; ++r) v[r] = s + r < nseg ? counts[(i64)(s + r) * B + b] : 0;
#pragma unroll
        for (int r = 0; r < kRun; ++r) sum += v[r];
        const int incl = wave_incl_scan(sum);
        int before = carry + incl - sum;
#pragma unroll
        for (int r = 0; r < kRun; ++r) {
            if (s + r < nseg) counts[(i64)(s + r) * B + b] = before;
            before += v[r];
        }
        carry += __shfl(incl, 63);
    }
    if (wave_lane() == 0) sizes[b] = carry;
}

// The last workgroup writes the prefix sums and the tiles instead.
__global__ void group_scatter(const int *bucket, i64 P, int K, int nbits, int seg, int nseg, const int *within, const int *counts, const int *sizes,
                              int *order, int *offsets, int *first, Tiles tiles) {
    extern __shared__ int lds[];
    const int nw = blockDim.x >> 6;
    const int B = K + 1, w = threadIdx.x >> 6, s = blockIdx.x * nw + w;
    int *start = lds + nw * B, *part = start + B;
    if (blockIdx.x == gridDim.x - 1) {
        int *starts = lds, *tile_starts = starts + B + 1;       // (the sums' parts behind them)
        write_sums(K, (int)P, sizes, offsets, first, tiles.lg, tile_starts + B + 1, [&](int b, int at, int tile) {
            starts[b] = at;
            tile_starts[b] = tile;
        });
        __syncthreads();
        write_tiles(K, starts, tile_starts, tiles);
        return;
    }
    block_scan(B, part, [&](int b) { return sizes[b]; }, [&](int b, int v) { start[b] = v + counts[(i64)blockIdx.x * B + b]; });
    int *cursor = lds + w * B;
    if (s < nseg)
        for (int b = wave_lane(); b < B; b += 64) cursor[b] = start[b] + within[(i64)s * B + b];
    __syncthreads();
    const i64 lo = (i64)s * seg < P ? (i64)s * seg : P, hi = lo + seg < P ? lo + seg : P;
    walk(lo, hi, nbits, cursor, [&](i64 i) { return bucket[i]; }, [&](i64 i, int, int at) { order[at] = (int)i; });
}

struct Split { int seg, nseg, waves, groups; };

// Rows of a segment (a wave's): 512, 256 where that would leave most of the chip idle.  Segments per workgroup: eight while their histograms, the buckets' starts and the sums fit 64 KB of LDS.
Split split_of(i64 P, int K) {
    Split s;
    s.seg = P <= 131072 ? 256 : 512;
    s.nseg = (int)((P + s.seg - 1) / s.seg);
    s.waves = K + 1 <= 1780 ? 8 : K + 1 <= 3200 ? 4 : 1;
    s.groups = (s.nseg + s.waves - 1) / s.waves;
    return s;
}

bool small_form(i64 P, int K) { return P <= kSmall && K + 1 <= kSmallBuckets; }

}  // namespace

extern "C" int64_t bgmm_group_rows_ws(int64_t P, int32_t K) {
    if (P < 0 || K < 1 || small_form(P, K)) return 0;
    const Split s = split_of(P, K);
    return 4 * ((int64_t)s.nseg + s.groups + 1) * (K + 1);
}

extern "C" int64_t bgmm_group_rows_tiles(int64_t P, int32_t K) { return P < 0 || K < 1 ? 0 : tiles_at_most(P, K); }

extern "C" int bgmm_group_rows(const int64_t *labels, int64_t P, int32_t K, int32_t *bucket, int32_t *order, int32_t *offsets,
                               int32_t *first, int32_t *tiles, void *ws, int64_t ws_bytes, void *stream) {
    if (P < 0 || P > 0x7fffffff - 65536) return ops_fail(BGMM_OPS_EINVAL, "group_rows: P = %lld rows (0 .. 2^31 - 65537)", (long long)P);
    if (K < 1) return ops_fail(BGMM_OPS_EINVAL, "group_rows: K = %d components", K);
    if (K > BGMM_OPS_MAX_COMPONENTS) return ops_fail(BGMM_OPS_EUNSUPPORTED, "group_rows: K = %d components (at most %d)", K, BGMM_OPS_MAX_COMPONENTS);
    if (!offsets || !first || !tiles || ((uintptr_t)tiles & 15) || (P > 0 && (!labels || !bucket || !order))) return ops_fail(BGMM_OPS_EINVAL, "group_rows: a null pointer");
    if (ws_bytes < bgmm_group_rows_ws(P, K) || (bgmm_group_rows_ws(P, K) > 0 && !ws)) return ops_fail(BGMM_OPS_EINVAL, "group_rows: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const int B = K + 1;
    const Tiles table = {(int4 *)tiles, (int)tiles_at_most(P, K), tile_log2(P, K)};
    int nbits = 1;
    while ((1 << nbits) < B) ++nbits;
    if (small_form(P, K)) {
        const int waves = P <= 2048 ? 4 : kWaves;
        const size_t lds = sizeof(int) * ((size_t)(waves + 2) * B + 2 + kSums * waves);
        group_small<<<1, 64 * waves, lds, st>>>(labels, (int)P, K, nbits, bucket, order, offsets, first, table);
        return ops_launched("group_rows");
    }
    const Split s = split_of(P, K);
    int *within = (int *)ws, *counts = within + (size_t)s.nseg * B, *sizes = counts + (size_t)s.groups * B;
    // (P = 0 with many components: no segment, but the sums over nothing and the empty offsets are still written)
    if (s.groups > 0) group_count<<<s.groups, 64 * s.waves, sizeof(int) * (size_t)s.waves * B, st>>>(labels, P, K, s.seg, s.nseg, bucket, within, counts);
    group_columns<<<(B + 3) / 4, 256, 0, st>>>(counts, s.groups, B, sizes);
    group_scatter<<<s.groups + 1, 64 * s.waves, sizeof(int) * ((size_t)(s.waves + 1) * B + 2 + kSums * s.waves), st>>>(bucket, P, K, nbits, s.seg, s.nseg, within, counts,
                                                                                                                  sizes, order, offsets, first, table);
    return ops_launched("group_rows");
}
