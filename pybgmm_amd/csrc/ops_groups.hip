// Rows grouped by component: a stable counting sort of P labels into K + 1 buckets (bucket K: unassigned rows).
//
//   order = argsort(bucket, stable), offsets = exclusive sum of the bucket sizes,
//   first[l][b] = sum over b' < b of ceil(size(b') / (256 << l)), and the table of tiles that the products work by
//
// Stable and without atomics across workgroups, so that a grouping is the same every time: the gradients that sum over a
// group's rows in this order are too.  A wave owns a segment of consecutive rows and a histogram of its own in LDS; the 64
// rows it looks at together find their equals with one ballot per label bit.
//
// Up to 4096 rows one workgroup does everything in one launch (64 components, one row 4 us, 2048 rows 6.5, 4096 rows 9.4 us; in several
// launches 9, 8.5 and 8.7; 4096 rows of 1400 components 17 and 23).  Beyond: histograms per segment and workgroup, an exclusive
// sum over the workgroups per bucket -- by the scatter itself where they are few --, the scatter (20000 rows 9 us, 1e6 rows
// of 100 components 17 us): bound by the latency of the launches and of the segments' dependent LDS steps, not by the 20 P
// bytes that move (4 us).
#include "ops_common.h"

namespace {

constexpr int kSums = BGMM_OPS_LEVELS + 2;      // sums over buckets: offsets, tiles, chunks of every level
// The one-workgroup form: up to 512 rows for each of its 8 waves with rows, 4 of them where 8 histograms, the sizes and the sums
// would not fit 64 KB of LDS; the sums over buckets have a wave each.
constexpr int kWaves = 8, kHeld = 8;    // (rounds of 64 rows)
int small_waves(int K) { return K + 1 <= 1480 ? kWaves : K + 1 <= 2300 ? 4 : 0; }
bool small_form(i64 P, int K) { return P <= small_waves(K) * 64 * kHeld && small_waves(K) > 0; }
constexpr int kManyWaves = 8;           // waves of a workgroup of the other form

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

// All the prefix sums over buckets: offsets (sum 0), the tiles of 1 << tile_lg rows (1), every level's chunks.  Each sum is one
// wave's, 64 buckets at a time without a barrier (four rows, 2000 components: 12 us, 68 with a barrier per round over all sums
// and a wave per bucket in write_tiles).  start(b, ...) and tile(b, ...) see sums 0 and 1 of every bucket and of b = K + 1, what is
// behind the last.
template <class S, class T> __device__ __forceinline__ void write_sums(int K, const int *size_of, int *offsets, int *first, int tile_lg, S start, T tile) {
    constexpr int kRounds = 4;                  // loads in flight
    const int nw = blockDim.x >> 6, lane = wave_lane(), B = K + 1;
    for (int l = threadIdx.x >> 6; l < kSums; l += nw) {
        const int lg = l == 0 ? 0 : l == 1 ? tile_lg : 6 + l;
        const auto emit = [&](int b, int sum) {
            if (l == 0) {
                offsets[b] = sum;
                start(b, sum);
            } else if (l == 1) {
                tile(b, sum);
            } else {
                first[(i64)(l - 2) * (K + 2) + b] = sum;
            }
        };
        int carry = 0;
        for (int b0 = 0; b0 < B; b0 += 64 * kRounds) {
            int v[kRounds];
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int b = b0 + r * 64 + lane;
                v[r] = b < B ? size_of[b] : 0;
            }
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int b = b0 + r * 64 + lane, n = (int)(((i64)v[r] + (1 << lg) - 1) >> lg), incl = wave_incl_scan(n);
                if (b < B) emit(b, carry + incl - n);
                carry += __builtin_amdgcn_readlane(incl, 63);
            }
        }
        if (lane == 0) emit(B, carry);
    }
}

struct Tiles { int4 *at; int n, lg; };

// The table of tiles from a grouping's sums in LDS (starts and tile_starts: [K + 2]): a lane per bucket, the wave together for a
// bucket of more than four tiles.
__device__ __forceinline__ void write_tiles(int K, const int *starts, const int *tile_starts, Tiles t) {
    const int lg = t.lg, nw = blockDim.x >> 6, w = threadIdx.x >> 6, lane = wave_lane();
    const auto write = [&](int b, int start, int n, int t0, int i) { t.at[t0 + i] = make_int4(b, start + (i << lg), n - (i << lg) < 1 << lg ? n - (i << lg) : 1 << lg, 0); };
    for (int b0 = w; b0 <= K; b0 += 64 * nw) {
        const int b = b0 + lane * nw;
        const bool on = b <= K;
        const int start = on ? starts[b] : 0, n = on ? starts[b + 1] - start : 0, t0 = on ? tile_starts[b] : 0;
        const bool many = n > 4 << lg;
        if (!many)
            for (int i = 0; i << lg < n; ++i) write(b, start, n, t0, i);
        for (unsigned long long left = __ballot(many); left; left &= left - 1) {
            const int l = __ffsll(left) - 1;
            const int lb = b0 + l * nw, ls = __builtin_amdgcn_readlane(start, l), ln = __builtin_amdgcn_readlane(n, l), lt = __builtin_amdgcn_readlane(t0, l);
            for (int i = lane; i << lg < ln; i += 64) write(lb, ls, ln, lt, i);
        }
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

__global__ __launch_bounds__(64 * kSums) void group_small(const int64_t *labels, int P, int K, int nbits, int waves, int *bucket, int *order,
                                                           int *offsets, int *first, Tiles tiles) {
    extern __shared__ int lds[];
    const int B = K + 1, w = threadIdx.x >> 6;
    int *hist = lds;                          // [waves][K + 1]
    int *sizes = hist + waves * B;            // [K + 1]
    int *starts = sizes + B;                  // [K + 2]
    int *tile_starts = starts + B + 1;        // [K + 2]
    for (int j = threadIdx.x; j < waves * B; j += blockDim.x) hist[j] = 0;
    // a wave's rows: at most kHeld rounds of 64; their buckets and places among the wave's own stay in registers
    const int per = ((P + waves - 1) / waves + 63) & ~63, lane = wave_lane();
    const int lo = w * per < P ? w * per : P, hi = lo + per < P ? lo + per : P;       // (none for the waves behind them: waves * per >= P)
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
        int n[kWaves], s = 0;
#pragma unroll
        for (int j = 0; j < kWaves; ++j) n[j] = j < waves ? hist[j * B + b] : 0;
#pragma unroll
        for (int j = 0; j < kWaves; ++j) {
            if (j < waves) hist[j * B + b] = s;
            s += n[j];
        }
        sizes[b] = s;
    }
    __syncthreads();
    write_sums(K, sizes, offsets, first, tiles.lg, [&](int b, int sum) { starts[b] = sum; }, [&](int b, int sum) { tile_starts[b] = sum; });
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
        if (lo + r * 64 + lane < hi) order[starts[held_b[r]] + hist[w * B + held_b[r]] + held_at[r]] = lo + r * 64 + lane;
    write_tiles(K, starts, tile_starts, tiles);
}

// `waves` segments per workgroup (1, 4 or 8), of as many waves each as its kManyWaves allow.
// within[segment][b]: the workgroup's earlier segments' rows of bucket b (null: a workgroup has one);  counts[workgroup][b]: all of its.
__global__ void group_count(const int64_t *labels, i64 P, int K, int seg, int nseg, int waves, int *bucket, int *within, int *counts) {
    extern __shared__ int lds[];
    const int B = K + 1, w = threadIdx.x >> 6, parts = kManyWaves / waves, s0 = blockIdx.x * waves, s = s0 + w % waves;
    int *hist = lds + w % waves * B;
    for (int b = threadIdx.x; b < waves * B; b += blockDim.x) lds[b] = 0;
    __syncthreads();
    const i64 lo = (i64)s * seg < P ? (i64)s * seg : P, hi = lo + seg < P ? lo + seg : P;
#pragma unroll 4
    for (i64 i = lo + w / waves * 64 + wave_lane(); i < hi; i += 64 * parts) {          // (counts need no order)
        const int b = bucket_of(labels, i, K);
        atomicAdd(&hist[b], 1);
        bucket[i] = b;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        int sum = 0;
        for (int j = 0; j < waves; ++j) {
            if (within && s0 + j < nseg) within[(i64)(s0 + j) * B + b] = sum;
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

// The first `waves` waves of a workgroup have a segment each; the last workgroup writes the prefix sums and the tiles instead.
// sizes null: counts holds the workgroups' own counts, `groups` of them, which every workgroup adds up for itself.
__global__ void group_scatter(const int *bucket, i64 P, int K, int nbits, int seg, int nseg, int waves, int groups, const int *within, const int *counts,
                              const int *sizes, int *order, int *offsets, int *first, Tiles tiles) {
    extern __shared__ int lds[];
    const int B = K + 1, w = threadIdx.x >> 6, s = blockIdx.x * waves + w, me = blockIdx.x;
    int before = 0;
    const auto total = [&](int b) {             // (before: of the workgroups in front of this one)
        int sum = 0;
        before = 0;
#pragma unroll 8
        for (int g = 0; g < groups; ++g) {
            const int n = counts[(i64)g * B + b];
            before += g < me ? n : 0;
            sum += n;
        }
        return sum;
    };
    if (blockIdx.x == gridDim.x - 1) {
        int *starts = lds, *tile_starts = starts + B + 1;
        if (!sizes) {
            int *own = tile_starts + B + 1;
            for (int b = threadIdx.x; b < B; b += blockDim.x) own[b] = total(b);
            __syncthreads();
            sizes = own;
        }
        write_sums(K, sizes, offsets, first, tiles.lg, [&](int b, int sum) { starts[b] = sum; }, [&](int b, int sum) { tile_starts[b] = sum; });
        __syncthreads();
        write_tiles(K, starts, tile_starts, tiles);
        return;
    }
    int *start = lds + waves * B, *part = start + B;
    block_scan(B, part, [&](int b) { return sizes ? sizes[b] : total(b); }, [&](int b, int v) { start[b] = v + (sizes ? counts[(i64)me * B + b] : before); });
    const int v = w % waves, parts = kManyWaves / waves;
    if (blockIdx.x * waves + v < nseg) {
#pragma unroll 4
        for (int b = w / waves * 64 + wave_lane(); b < B; b += 64 * parts) lds[v * B + b] = start[b] + (within ? within[(i64)(blockIdx.x * waves + v) * B + b] : 0);
    }
    __syncthreads();
    if (w >= waves) return;
    int *cursor = lds + w * B;
    const i64 lo = (i64)s * seg < P ? (i64)s * seg : P, hi = lo + seg < P ? lo + seg : P;
    walk(lo, hi, nbits, cursor, [&](i64 i) { return bucket[i]; }, [&](i64 i, int, int at) { order[at] = (int)i; });
}

// Up to so many workgroups each of the scatter's adds up the counts itself (20011 rows 10.5 -> 8.7 us, 65536 rows 11.0 -> 9.5; 131072
// rows, 64 workgroups, 1000 components: 18.1 with the sums in a launch of their own, 19.2; 1e6 rows, 245: 16.5 and 23.7).
constexpr int kFewGroups = 32;
struct Split { int seg, nseg, waves, groups; };
i64 within_of(const Split &s) { return s.waves > 1 ? s.nseg : 0; }          // histograms in `within`

// Rows of a segment (a wave's): 512, 256 where that would leave most of the chip idle; more, up to the number of buckets, where the
// histograms in memory would be 8 MB and more (4 MB of few rows), so that they are no larger than that and the rows' indices (1e6 rows
// of 8000 components: 395 us and 125 MB with 512, 128 us with 4096, 140 us with 8192; of 3500: 169, 74 us with 2048, 77 with 4096; 4e6 of
// 8000: 1740, 325 us with 4096, 207 with 8192; 1e5 of 8000: 128, 87 us with 1024, 125 with 8192; but 8192 rows of 8000: 78, 92 with 2048).
// Segments per workgroup: eight while their histograms, the buckets' starts and the sums fit 64 KB of LDS.
Split split_of(i64 P, int K) {
    Split s;
    s.seg = P <= 131072 ? 256 : 512;
    while (s.seg <= K && (P + s.seg - 1) / s.seg * (K + 1) > (P <= 131072 ? 1 << 20 : 1 << 21)) s.seg *= 2;
    s.nseg = (int)((P + s.seg - 1) / s.seg);
    s.waves = K + 1 <= 1780 ? 8 : K + 1 <= 3200 ? 4 : 1;
    s.groups = (s.nseg + s.waves - 1) / s.waves;
    return s;
}

}  // namespace

extern "C" int64_t bgmm_group_rows_ws(int64_t P, int32_t K) {
    if (P < 0 || K < 1 || small_form(P, K)) return 0;
    const Split s = split_of(P, K);
    return 4 * (within_of(s) + s.groups + 1) * (K + 1);
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
        const int waves = small_waves(K);
        group_small<<<1, 64 * kSums, sizeof(int) * ((size_t)(waves + 3) * B + 2), st>>>(labels, (int)P, K, nbits, waves, bucket, order, offsets, first, table);
        return ops_launched("group_rows");
    }
    const Split s = split_of(P, K);
    int *within = s.waves > 1 ? (int *)ws : nullptr, *counts = (int *)ws + (size_t)within_of(s) * B, *sizes = counts + (size_t)s.groups * B;
    // (P = 0 with many components: no segment, but the sums over nothing and the empty offsets are still written)
    if (s.groups > 0) group_count<<<s.groups, 64 * kManyWaves, sizeof(int) * (size_t)s.waves * B, st>>>(labels, P, K, s.seg, s.nseg, s.waves, bucket, within, counts);
    const bool columns = s.groups > kFewGroups || s.waves < 8;
    if (columns) group_columns<<<(B + 3) / 4, 256, 0, st>>>(counts, s.groups, B, sizes);
    group_scatter<<<s.groups + 1, 64 * kManyWaves, sizeof(int) * ((size_t)(s.waves + 1) * B + 2 + kManyWaves), st>>>(
        bucket, P, K, nbits, s.seg, s.nseg, s.waves, s.groups, within, counts, columns ? sizes : nullptr, order, offsets, first, table);
    return ops_launched("group_rows");
}
