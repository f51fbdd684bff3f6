// C entry points of the products with a component's own matrix: checks, tile sizes, splits, the dispatch on the element type.
#include "ops_products.h"

namespace {

int size_of(int dtype) { return dtype == BGMM_F64 ? 8 : dtype == BGMM_F32 ? 4 : 2; }
int acc_size(int dtype) { return dtype == BGMM_F64 ? 8 : 4; }
Divisor divisor(int d) {
    int lg = 0;
    while ((1ll << lg) < d) ++lg;
    return {(unsigned)((1ull << (31 + lg)) / (unsigned)d + 1), 31 + lg};
}
i64 at_most(i64 a, i64 b) { return a < b ? a : b; }

// Of `rows` rows `stride` elements apart, the first how many have 16 bytes from their last element on: the rows behind them, up to
// the last row's last element, hold the rest.
int safe_rows(i64 rows, i64 stride, int size) {
    if (stride < 1) return 0;
    const i64 n = rows - (16 / size - 1 + stride - 1) / stride;
    return n < 0 ? 0 : (int)n;
}

// Columns of a tile of a product with rows: 128 beside 16 rows; else the next of 16, 32, 64, 128 (1e6 rows, 32 -> 32 double: 147 us
// with 64, 113 with 32), 64 instead of 128 where that would leave
// compute units without a workgroup (20011 rows, 33 components, 192 -> 77 single: 23.1 -> 21.5 us; 2000 rows, 4 components,
// 256 -> 512 bfloat16: 8.0 -> 6.3 us).
int cols_tile(i64 P, int K, int ndim) {
    if (small_tiles(P, K)) return 128;
    if (ndim <= 64) return ndim <= 16 ? 16 : ndim <= 32 ? 32 : 64;
    return tiles_at_most(P, K) * ((ndim + 127) / 128) < 512 ? 64 : 128;
}

// Workgroups for `useful` ones in runs per die (die_order): runs of up to 64, shorter where the dies would get less than eight.
struct Grid { int run; i64 blocks; };
Grid grid_of(i64 useful) {
    Grid g = {64, 0};
    while (g.run > 1 && useful < (i64)g.run * 64) g.run /= 2;
    g.blocks = (useful + 8 * g.run - 1) / (8 * g.run) * (8 * g.run);
    return g;
}

// Tile of the weights' gradient (bi x bo) and chunk of rows (a level of the grouping): chunks as long as about a thousand
// workgroups remain, 256 .. 32768 rows -- a chunk leaves a tile of partial sums, which 256 rows of both operands outweigh --
// (forward and this, 1e6 rows, 4 components of 64 x 64 single: 338 us with chunks of 256, 302 us), and tiles of 64 where 128
// would leave compute units idle even so (20011 rows, 33 components, 192 x 77: 61.5 -> 53.1 us).
// An axis of up to 16 or 64 gets a tile of that width (forward and this, 114804 rows, 905 x 16 double: 773 us with 128 x 128, 379;
// 1e6 rows, 128 x 10 single: 457 and 277 us).
struct WeightTiles { int bi, bo, level; };
WeightTiles weight_tiles(i64 P, int idim, int odim) {
    const auto tiles = [&](int ti, int to) { return (i64)((idim + ti - 1) / ti) * ((odim + to - 1) / to); };
    const auto width = [](int d) { return d <= 16 ? 16 : d <= 64 ? 64 : 128; };
    WeightTiles w = {width(idim), width(odim), 0};
    if (w.bi + w.bo == 80 || (w.bi + w.bo > 80 && (P / 256 + 1) * tiles(w.bi, w.bo) < 512)) w.bi = w.bo = 64;
    while (w.level < BGMM_OPS_LEVELS - 1 && P / (256 << (w.level + 1)) * tiles(w.bi, w.bo) >= 1024) ++w.level;
    return w;
}

int check(const char *what, int dtype, i64 P, int K, int a, int b) {
    if (dtype < BGMM_F64 || dtype > BGMM_BF16) return ops_fail(BGMM_OPS_EINVAL, "%s: element type %d", what, dtype);
    if (P < 0 || P > 0x7fffffff - 65536 || K < 1 || a < 1 || b < 1)
        return ops_fail(BGMM_OPS_EINVAL, "%s: P = %lld, K = %d, dimensions %d and %d", what, (long long)P, K, a, b);
    if (K > BGMM_OPS_MAX_COMPONENTS) return ops_fail(BGMM_OPS_EUNSUPPORTED, "%s: K = %d components (at most %d)", what, K, BGMM_OPS_MAX_COMPONENTS);
    if (a > BGMM_OPS_MAX_AXIS || b > BGMM_OPS_MAX_AXIS) return ops_fail(BGMM_OPS_EUNSUPPORTED, "%s: dimensions %d and %d (at most %d)", what, a, b, BGMM_OPS_MAX_AXIS);
    return BGMM_OPS_OK;
}

}  // namespace

extern "C" int bgmm_rows_product_splits(int32_t dtype, int64_t P, int32_t K, int32_t kdim, int32_t ndim) {
    if (check("rows_product_splits", dtype, P, K, kdim, ndim) != BGMM_OPS_OK || P == 0) return 1;
    const int bn = cols_tile(P, K, ndim);
    const i64 groups = ((P >> tile_log2(P, K)) + at_most(K, P)) * ((ndim + bn - 1) / bn);
    const int steps = (kdim * size_of(dtype) + kStepBytes - 1) / kStepBytes;
    // Few rows leave compute units idle while a few stream the weights: the contraction in parts, as many workgroups as the compute
    // units hold of either tile, but a part has four steps to do, and the steps saved outweigh adding the parts up.  (bfloat16,
    // one row of 4 experts of 64, 2048 -> 1024: 29.6 -> 8.6 us; one row, 4096 -> 4096: 57 -> 17 us, 33.5 MB of weights; 5000
    // rows, 8 components, 1024 -> 64, twelve steps saved: 12.7 -> 11.8 us; but 20000 rows, 32, 768 -> 64, six: 13.0 -> 16.6 us.)
    const i64 s = at_most(at_most((small_tiles(P, K) ? 1024 : 512) / groups, steps / 4), 16);
    return s > 1 && steps - steps / s >= 8 ? (int)s : 1;
}

extern "C" int bgmm_rows_product_dots(int32_t dtype, int64_t P, int32_t K, int32_t kdim, int32_t ndim, int32_t splits) {
    if (check("rows_product_dots", dtype, P, K, kdim, ndim) != BGMM_OPS_OK || splits < 1) return 0;
    const int bn = cols_tile(P, K, ndim);
    return splits * ((ndim + bn - 1) / bn) * (small_tiles(P, K) ? 4 : bn >= 64 ? 2 : 1);       // (waves side by side along a tile's columns)
}

extern "C" int bgmm_rows_product(int32_t dtype, const void *in, int64_t in_stride, int32_t in_div, const void *w, int64_t w_component,
                                 int64_t w_row, int32_t kcontig, const void *bias, int64_t bias_row, const void *gates, void *out,
                                 int64_t out_stride, void *ws, int32_t splits, const void *dot_in, int64_t dot_stride, int32_t dot_div, void *dots,
                                 int64_t P, int32_t K, int32_t kdim, int32_t ndim, const int32_t *order, const int32_t *tiles, void *stream) {
    const int rc = check("rows_product", dtype, P, K, kdim, ndim);
    if (rc) return rc;
    if (P == 0) return BGMM_OPS_OK;
    if (!in || !w || !order || !tiles || (out && ws) || (!out && !ws && !dots) || (dots && !dot_in))
        return ops_fail(BGMM_OPS_EINVAL, "rows_product: a null pointer (one of out and ws, or neither with dots)");
    if (dots && (dot_stride < 0 || dot_div < 1)) return ops_fail(BGMM_OPS_EINVAL, "rows_product: stride %lld, divisor %d of the rows of dots", (long long)dot_stride, dot_div);
    if (in_div < 1 || splits < 1 || (out && splits != 1) || in_stride < 0 || out_stride < 0 || w_component < 0 || w_row < 0)
        return ops_fail(BGMM_OPS_EINVAL, "rows_product: in_div %d, splits %d, strides %lld %lld", in_div, splits, (long long)in_stride, (long long)out_stride);
    const int bm = small_tiles(P, K) ? 16 : 128, bn = cols_tile(P, K, ndim);
    RowsArgs a;
    a.tiles = (const int4 *)tiles;
    a.tile_blocks = (int)(tiles_at_most(P, K) / 8);
    a.order = order;
    a.K = K;
    a.in = in;
    a.in_stride = in_stride;
    a.in_div = divisor(in_div);
    a.w = w;
    a.w_component = w_component;
    a.w_row = w_row;
    a.bias = bias;
    a.bias_row = bias_row;
    a.gates = gates;
    a.out = out;
    a.out_stride = out_stride;
    a.ws = ws;
    a.dot_in = dot_in;
    a.dot_stride = dot_stride;
    a.dot_div = divisor(dots ? dot_div : 1);
    a.dots = dots;
    a.n_dots = bgmm_rows_product_dots(dtype, P, K, kdim, ndim, splits);
    a.P = P;
    a.kdim = kdim;
    a.ndim = ndim;
    a.splits = splits;
    a.n_tiles = (ndim + bn - 1) / bn;
    a.in_safe = safe_rows(P / in_div, in_stride, size_of(dtype));
    a.w_safe = safe_rows(kcontig ? ndim : kdim, w_row, size_of(dtype));
    const Grid g = grid_of((i64)a.tile_blocks * 8 * a.n_tiles * splits);
    if (g.blocks > 0x7fffffff) return ops_fail(BGMM_OPS_EUNSUPPORTED, "rows_product: %lld tiles", (long long)g.blocks);
    a.run = g.run;
    return by_type(dtype, [&](auto *t) { return launch_rows<std::remove_pointer_t<decltype(t)>>(a, kcontig != 0, bm, bn, g.blocks, (hipStream_t)stream); });
}

extern "C" int64_t bgmm_weight_product_ws(int32_t dtype, int64_t P, int32_t K, int32_t idim, int32_t odim) {
    if (check("weight_product_ws", dtype, P, K, idim, odim) != BGMM_OPS_OK) return 0;
    const i64 rows = (i64)256 << weight_tiles(P, idim, odim).level;
    if (P <= rows) return 0;
    return (2 * P / rows + 2) * ((i64)idim * odim + odim) * acc_size(dtype);
}

extern "C" int bgmm_weight_product(int32_t dtype, const void *in, int64_t in_stride, int32_t in_div, const void *d, int64_t d_stride,
                                   int32_t d_div, const void *gates, void *dw, void *db, void *ws, int64_t ws_bytes, int64_t P, int32_t K,
                                   int32_t idim, int32_t odim, const int32_t *order, const int32_t *offsets, const int32_t *first, void *stream) {
    const int rc = check("weight_product", dtype, P, K, idim, odim);
    if (rc) return rc;
    if (!dw && !db) return BGMM_OPS_OK;
    if (!offsets || !first || (P > 0 && (!in || !d || !order))) return ops_fail(BGMM_OPS_EINVAL, "weight_product: a null pointer");
    if (in_div < 1 || d_div < 1 || in_stride < 0 || d_stride < 0) return ops_fail(BGMM_OPS_EINVAL, "weight_product: divisors %d %d, strides %lld %lld", in_div, d_div, (long long)in_stride, (long long)d_stride);
    if (ws_bytes < bgmm_weight_product_ws(dtype, P, K, idim, odim) || (ws_bytes > 0 && (!ws || ((uintptr_t)ws & 15))))
        return ops_fail(BGMM_OPS_EINVAL, "weight_product: workspace of %lld bytes", (long long)ws_bytes);
    const WeightTiles w = weight_tiles(P, idim, odim);
    WeightArgs a;
    a.level = w.level;
    a.bucket_first = first + (size_t)a.level * (K + 2);
    a.offsets = offsets;
    a.order = order;
    a.K = K;
    a.in = in;
    a.in_stride = in_stride;
    a.in_div = divisor(in_div);
    a.d = d;
    a.d_stride = d_stride;
    a.d_div = divisor(d_div);
    a.gates = gates;
    a.dw = dw;
    a.db = db;
    a.ws = ws;
    a.idim = idim;
    a.odim = odim;
    a.i_tiles = dw ? (idim + w.bi - 1) / w.bi : 1;        // (the bias's sums come with the first)
    a.o_tiles = (odim + w.bo - 1) / w.bo;
    a.in_safe = safe_rows(P / in_div, in_stride, size_of(dtype));
    a.d_safe = safe_rows(P / d_div, d_stride, size_of(dtype));
    const Grid g = grid_of(P == 0 ? 0 : (P / ((i64)256 << a.level) + at_most(K, P)) * a.i_tiles * a.o_tiles);
    if (g.blocks > 0x7fffffff) return ops_fail(BGMM_OPS_EUNSUPPORTED, "weight_product: %lld tiles", (long long)g.blocks);
    a.run = g.run;
    return by_type(dtype, [&](auto *t_) { return launch_weight<std::remove_pointer_t<decltype(t_)>>(a, w.bi, w.bo, g.blocks, (hipStream_t)stream); });
}

extern "C" int bgmm_combine(int32_t dtype, const void *ws, int32_t splits, int64_t rows, int32_t k, int32_t K, const int32_t *bucket,
                            const void *gates, void *out, int64_t out_stride, int32_t dim, void *dgates, const void *in, int64_t in_stride,
                            const void *bias, int64_t bias_row, const void *d, int64_t d_stride, int32_t d_div, int32_t ddim, void *stream) {
    const int rc = check("combine", dtype, rows, K, dim, 1);
    if (rc) return rc;
    if (k < 1 || k > BGMM_OPS_MAX_CHOSEN || splits < 1) return ops_fail(BGMM_OPS_EINVAL, "combine: k = %d (1 .. %d), splits %d", k, BGMM_OPS_MAX_CHOSEN, splits);
    if (rows == 0) return BGMM_OPS_OK;
    if (!ws || !bucket || (!out && !dgates) || (dgates && (!gates || !in)) || (dgates && bias && (!d || d_div < 1 || ddim < 1)))
        return ops_fail(BGMM_OPS_EINVAL, "combine: a null pointer");
    CombineArgs a;
    a.bucket = bucket;
    a.K = K;
    a.k = k;
    a.splits = splits;
    a.rows = rows;
    a.P = rows * k;
    a.first = 0;
    a.ws = ws;
    a.gates = gates;
    a.out = out;
    a.out_stride = out_stride;
    a.dim = dim;
    a.dgates = dgates;
    a.in = in;
    a.in_stride = in_stride;
    a.bias = bias;
    a.bias_row = bias_row;
    a.d = d;
    a.d_stride = d_stride;
    a.d_div = d_div < 1 ? 1 : d_div;
    a.ddim = ddim;
    return by_type(dtype, [&](auto *t) { return launch_combine<std::remove_pointer_t<decltype(t)>>(a, (hipStream_t)stream); });
}

extern "C" int bgmm_gate_gradient(int32_t dtype, const void *dots, int32_t n_dots, int64_t P, int32_t K, const int32_t *bucket, const void *bias,
                                  int64_t bias_row, const void *d, int64_t d_stride, int32_t d_div, int32_t ddim, void *dgates, void *stream) {
    const int rc = check("gate_gradient", dtype, P, K, n_dots, 1);
    if (rc) return rc;
    if (P == 0) return BGMM_OPS_OK;
    if (!dots || !bucket || !dgates || (bias && (!d || d_div < 1 || ddim < 1 || d_stride < 0 || bias_row < 0)))
        return ops_fail(BGMM_OPS_EINVAL, "gate_gradient: a null pointer, or a bias with a size or stride that is none");
    const GatesArgs a = {bucket, K, n_dots, P, dots, bias, bias_row, d, d_stride, divisor(bias ? d_div : 1), ddim, dgates};
    return by_type(dtype, [&](auto *t) { return launch_gates<std::remove_pointer_t<decltype(t)>>(a, (hipStream_t)stream); });
}
