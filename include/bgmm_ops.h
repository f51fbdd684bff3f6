/*
 * libbgmm_ops.so -- C-ABI of the mixture-of-experts operators: a fitted mixture (or a learned gate) routes rows to components,
 * rows are multiplied with their own component's matrix, drafted labels are verified against exact probabilities.
 *
 * Conventions
 *   - plain C, no exceptions; every call returns BGMM_OPS_OK or a negative code (the values of bgmm.h's BGMM_E*), with a
 *     message in bgmm_ops_last_error() (per thread).
 *   - every pointer is device memory of the CURRENT device, every call queues its kernels on `stream` (a hipStream_t) and
 *     returns without waiting; nothing is kept from one call to the next and nothing is allocated: the caller brings the
 *     workspaces, and two calls that may run at the same time bring different ones.  All calls may be captured into a graph.
 *   - strides and sizes are counted in elements; element (i, j) of a matrix is p[i * stride + j]: the last axis is contiguous.
 *   - the library does not link the HIP runtime: it binds to the one its process has loaded globally (a C host links
 *     -lamdhip64; pybgmm_amd.ops loads the copy that PyTorch uses, so that streams and pointers mean the same to both).
 */
#ifndef BGMM_OPS_H
#define BGMM_OPS_H

#include <stdint.h>

#define BGMM_OPS_API __attribute__((visibility("default")))

#ifdef __cplusplus
extern "C" {
#endif

enum {
    BGMM_OPS_OK = 0,
    BGMM_OPS_EINVAL = -1,      /* a size, stride, pointer or type that the call does not take */
    BGMM_OPS_EDEVICE = -2,     /* HIP runtime error (message holds hipGetErrorString)         */
    BGMM_OPS_EUNSUPPORTED = -5 /* a size beyond the call's documented limit                   */
};

/* element types */
enum { BGMM_F64 = 0, BGMM_F32 = 1, BGMM_F16 = 2, BGMM_BF16 = 3 };

/* limits */
enum {
    BGMM_OPS_MAX_COMPONENTS = 8000,  /* components of a grouping                               */
    BGMM_OPS_MAX_CHOSEN = 32,        /* components chosen per row by bgmm_route                */
    BGMM_OPS_MAX_AXIS = (1 << 27) - 1,  /* d_in and d_out of a product                           */
    BGMM_OPS_LEVELS = 8              /* chunk sizes of a grouping: 256, 512, ..., 32768 rows   */
};

BGMM_OPS_API const char *bgmm_ops_last_error(void);

/* Path of the HIP runtime this library is bound to. */
BGMM_OPS_API const char *bgmm_ops_runtime_path(void);

/*
 * Rows grouped by component: a stable counting sort of P labels.  A label outside 0 .. K-1 (the samplers' -1 = unassigned)
 * puts its row into bucket K.
 *   labels   int64[P]
 *   bucket   int32[P]      out: the label, or K
 *   order    int32[P]      out: row indices sorted by (bucket, row)
 *   offsets  int32[K + 2]  out: bucket b holds order[offsets[b] .. offsets[b + 1])
 *   first    int32[BGMM_OPS_LEVELS][K + 2]  out: in chunks of 256 << level rows, how many the buckets before b have
 *   tiles    int32[bgmm_group_rows_tiles(P, K)][4]  out, 16-byte aligned: the tiles the products work by, {bucket, first place
 *            in order, rows, 0}, bucket by bucket, {-1, ...} behind the last
 *   ws       bgmm_group_rows_ws(P, K) bytes
 */
BGMM_OPS_API int64_t bgmm_group_rows_ws(int64_t P, int32_t K);
BGMM_OPS_API int64_t bgmm_group_rows_tiles(int64_t P, int32_t K);
BGMM_OPS_API int bgmm_group_rows(const int64_t *labels, int64_t P, int32_t K, int32_t *bucket, int32_t *order, int32_t *offsets,
                                 int32_t *first, int32_t *tiles, void *ws, int64_t ws_bytes, void *stream);

/*
 * Rows times their own component's matrix: for every row p of component e (order / tiles: a grouping's)
 *     u_p = in[p / in_div] W_e + b_e
 * out != NULL: out[p] = g_p u_p, rounded once (rows of no component: zeros); splits must be 1.
 * ws != NULL: ws[s][p] = the part s of u_p, in the accumulator type (double for BGMM_F64, else float), not gated, bias in part
 *   0; rows of no component are left alone.  bgmm_combine adds the parts.
 *   dtype        of in, W, bias, out; products of half precision types accumulate in 32 bits
 *   W            element (k, n) of component e at e * w_component + k * w_row + n (kcontig 0) or + n * w_row + k (kcontig 1)
 *   bias         [K][ndim] with row stride bias_row, or NULL;  gates  accumulator type [P], or NULL
 *   dots         [P][bgmm_rows_product_dots(...)] in the accumulator type, or NULL: parts of dot_in[p / dot_div] . u_p (ungated, without
 *                bias), which bgmm_gate_gradient adds up; out and ws may then both be NULL
 * Operands' rows are read by 16 bytes: up to 15 bytes behind a row's end, where another row follows, whose values do not matter.
 * bgmm_rows_product_splits: how many parts serve a product well (1: write `out`).
 */
BGMM_OPS_API int bgmm_rows_product_splits(int32_t dtype, int64_t P, int32_t K, int32_t kdim, int32_t ndim);
BGMM_OPS_API int bgmm_rows_product(int32_t dtype, const void *in, int64_t in_stride, int32_t in_div, const void *w, int64_t w_component,
                                   int64_t w_row, int32_t kcontig, const void *bias, int64_t bias_row, const void *gates, void *out,
                                   int64_t out_stride, void *ws, int32_t splits, const void *dot_in, int64_t dot_stride, int32_t dot_div,
                                   void *dots, int64_t P, int32_t K, int32_t kdim, int32_t ndim, const int32_t *order, const int32_t *tiles,
                                   void *stream);
BGMM_OPS_API int bgmm_rows_product_dots(int32_t dtype, int64_t P, int32_t K, int32_t kdim, int32_t ndim, int32_t splits);

/*
 * The weights' gradient: dW_e = sum over the rows p of component e of g_p in[p / in_div] (x) d[p / d_div], db_e = sum of
 * g_p d[p / d_div]; components without rows get zeros.  dw [K][idim][odim] and db [K][odim] dense, either may be NULL.  Long
 * groups are split and their partial sums added in a fixed order.  ws: bgmm_weight_product_ws(...) bytes.
 */
BGMM_OPS_API int64_t bgmm_weight_product_ws(int32_t dtype, int64_t P, int32_t K, int32_t idim, int32_t odim);
BGMM_OPS_API int bgmm_weight_product(int32_t dtype, const void *in, int64_t in_stride, int32_t in_div, const void *d, int64_t d_stride,
                                     int32_t d_div, const void *gates, void *dw, void *db, void *ws, int64_t ws_bytes, int64_t P, int32_t K,
                                     int32_t idim, int32_t odim, const int32_t *order, const int32_t *offsets, const int32_t *first,
                                     void *stream);

/*
 * out[i] = sum over j < k of g_ij u_ij, u_ij = sum of the splits' parts ws[s][i k + j]; entries without a component add
 * nothing.  gates NULL: ones.  dgates != NULL (needs gates, in): dgates[i k + j] = in[i] . u_ij + bias_e . d[(i k + j) / d_div]
 * (bias NULL: without it), and out may be NULL.
 */
BGMM_OPS_API int bgmm_combine(int32_t dtype, const void *ws, int32_t splits, int64_t rows, int32_t k, int32_t K, const int32_t *bucket,
                              const void *gates, void *out, int64_t out_stride, int32_t dim, void *dgates, const void *in, int64_t in_stride,
                              const void *bias, int64_t bias_row, const void *d, int64_t d_stride, int32_t d_div, int32_t ddim, void *stream);

/*
 * The gates' gradient dgates[p] = sum of dots[p] + bias_e . d[p / d_div] (bias NULL: without it; rows of no component: zero), dots what
 * the product of d with the transposed weights left (dot_in: the rows that the forward pass multiplied).
 */
BGMM_OPS_API int bgmm_gate_gradient(int32_t dtype, const void *dots, int32_t n_dots, int64_t P, int32_t K, const int32_t *bucket, const void *bias,
                                    int64_t bias_row, const void *d, int64_t d_stride, int32_t d_div, int32_t ddim, void *dgates,
                                    void *stream);

/*
 * The k most probable components of every row of log weights [n][K] (row stride `stride`): ordered by (log weight descending,
 * index ascending); -inf and NaN are never chosen, a row with fewer than k others fills up with label -1 and weight 0.
 * weights: the softmax over the chosen ones (renormalise 1) or over all (0), in the accumulator type (double for BGMM_F64, else
 * float).  stats [n][2] (maximum and total; may be NULL): what the backward pass over all needs.
 * bgmm_route_backward: the log weights' gradient [n][K], dense, in their type; log_weights and stats only with renormalise 0.
 */
BGMM_OPS_API int bgmm_route(int32_t dtype, const void *log_weights, int64_t stride, int64_t n, int32_t K, int32_t k, int32_t renormalise,
                            int64_t *labels, void *weights, void *stats, void *stream);
BGMM_OPS_API int bgmm_route_backward(int32_t dtype, const void *log_weights, int64_t stride, int64_t n, int32_t K, int32_t k,
                                     int32_t renormalise, const int64_t *labels, const void *weights, const void *stats, const void *dweights,
                                     void *dlog_weights, void *stream);

/*
 * Drafted labels verified from given uniforms: draft t of sequence b is accepted iff u_accept q_t(z) < p_t(z); behind the
 * accepted ones a label is drawn with u_draw from max(0, p - q) at the rejected place (from p where that is zero), or from p
 * where all were accepted: the first label whose cumulative sum exceeds u_draw times the sum (64 bits).  What is not a
 * positive finite number counts as zero, a drafted label outside 0 .. V-1 is rejected, nothing to draw from gives -1.
 *   target [B][T + 1][V], draft [B][T][V]  strides _b, _t;  labels [B][T];  u_accept [B][T], u_draw [B] in [0, 1)
 *   lengths [B]: drafts of each sequence (0 .. T, clamped), or NULL: T
 *   out [B][T + 1]: the accepted labels, the drawn one, -1 behind;  accepted [B]
 *   ws: bgmm_verify_drafts_ws(B, V) bytes
 */
BGMM_OPS_API int64_t bgmm_verify_drafts_ws(int64_t B, int64_t V);
BGMM_OPS_API int bgmm_verify_drafts(int32_t dtype, const void *target, int64_t target_b, int64_t target_t, const void *draft, int64_t draft_b,
                                    int64_t draft_t, const int64_t *labels, const double *u_accept, const double *u_draw,
                                    const int64_t *lengths, int64_t B, int32_t T, int64_t V, int64_t *out, int64_t *accepted, void *ws,
                                    int64_t ws_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
