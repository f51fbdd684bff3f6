// pybgmm_amd.ops._binding: the operators of libbgmm_ops.so (include/bgmm_ops.h) on torch tensors -- argument checks, outputs and
// workspaces from torch's allocator, the caller's current stream, gradients.  Host code only, in C++ because a call's cost on the
// host (5 us here, twice that and more through ctypes and a Python autograd function) is what the small calls are made of.
#include <torch/extension.h>

#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <cstdarg>
#include <cstdio>
#include <stdexcept>
#include <string>
#include <unordered_set>

#include "../../include/bgmm_ops.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

namespace {

// ------------------------------------------------------------------------------------------ errors
struct Refusal : std::runtime_error {           // becomes pybgmm_amd._lib.BGMMError
    int code;
    Refusal(int c, const std::string &m) : std::runtime_error(m), code(c) {}
};

[[noreturn]] void refuse(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    throw Refusal(code, buf);
}

void check(int rc) {
    if (rc != BGMM_OPS_OK) refuse(rc, "%s", bgmm_ops_last_error());
}

std::string shape_of(const Tensor &t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

int type_of(at::ScalarType t) {
    return t == at::kDouble ? BGMM_F64 : t == at::kFloat ? BGMM_F32 : t == at::kHalf ? BGMM_F16 : t == at::kBFloat16 ? BGMM_BF16 : -1;
}

int type_of(const char *what, const char *name, const Tensor &t) {
    const int c = type_of(t.scalar_type());
    if (c < 0) refuse(BGMM_OPS_EINVAL, "%s: %s is %s", what, name, c10::toString(t.scalar_type()));
    return c;
}

at::ScalarType acc_of(at::ScalarType t) { return t == at::kDouble ? at::kDouble : at::kFloat; }

// All tensors of a call (undefined ones: absent) on one HIP device.
struct Device {
    const char *what;
    std::optional<c10::Device> at;
    void operator()(const char *name, const Tensor &t) {
        if (!t.defined()) return;
        if (!t.device().is_cuda()) refuse(BGMM_OPS_EDEVICE, "%s: %s is on %s; the operators run on HIP devices only", what, name, t.device().str().c_str());
        if (!at) at = t.device();
        else if (*at != t.device()) refuse(BGMM_OPS_EINVAL, "%s: %s is on %s, the others on %s", what, name, t.device().str().c_str(), at->str().c_str());
    }
};

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor given(const Maybe &t) { return t ? *t : Tensor(); }
// What the kernels read is the memory, so a view that torch negates on reading (the imaginary part of a conjugate) becomes values.
Tensor values(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor packed(const Tensor &t) { return values(t).contiguous(); }

// A (n, d) tensor as rows: the tensor itself if its last axis is contiguous, a copy otherwise.
struct Rows {
    Tensor t;
    int64_t stride = 0;
};
Rows rows_of(Tensor t) {
    if (!t.defined()) return {};
    t = values(t);
    if (t.dim() == 3) t = t.reshape({-1, t.size(2)});               // (a view where the strides allow it)
    if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < 0)) t = t.contiguous();
    return {t, t.size(0) > 1 ? t.stride(0) : t.size(1)};
}

void first_order_only(const char *what) {
    if (at::GradMode::is_enabled()) refuse(BGMM_OPS_EUNSUPPORTED, "%s: differentiable once (no create_graph)", what);
}

// Whether gradients are wanted of any of a call's tensors (undefined ones: absent), and whether the call can give them.
// Under capture, a node of the graph behind them that belongs to the default stream -- a leaf's too, while an eager graph that
// was made there lives -- would draw the default stream into the capture in backward, which ends the process there; refused here.
bool differentiable(const char *what, std::initializer_list<Tensor> inputs) {
    bool any = false;
    for (const Tensor &t : inputs) {
        if (!t.defined()) continue;
        if (t._fw_grad(0).defined()) refuse(BGMM_OPS_EUNSUPPORTED, "%s: no forward-mode derivatives", what);
        any = any || t.requires_grad();
    }
    if (!any || !at::GradMode::is_enabled()) return false;
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return true;
    std::vector<std::shared_ptr<torch::autograd::Node>> todo;
    std::unordered_set<const torch::autograd::Node *> seen;
    const auto visit = [&](const std::shared_ptr<torch::autograd::Node> &f) {
        if (f && seen.insert(f.get()).second) todo.push_back(f);
    };
    for (const Tensor &t : inputs)
        if (t.defined() && t.requires_grad()) visit(t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t));
    while (!todo.empty()) {
        const auto f = todo.back();
        todo.pop_back();
        const auto s = f->stream();
        if (s && s->id() == 0)
            refuse(BGMM_OPS_EUNSUPPORTED, "%s: captured with gradients, but %s belongs to an eager graph of the default stream (free that graph, detach, or capture under no_grad)", what, f->name().c_str());
        for (const auto &edge : f->next_edges()) visit(edge.function);
    }
    return true;
}

// ------------------------------------------------------------------------------------------ groupings
struct RowGroups {
    std::vector<int64_t> shape;             // the labels'
    int64_t n, k, P, K, n_tiles;
    Tensor store;                           // int32: tiles [n_tiles][4], bucket [P], order [P], offsets [K + 2], first [levels][K + 2]

    RowGroups(std::vector<int64_t> s, int64_t components, Tensor st) : shape(std::move(s)), K(components), store(std::move(st)) {
        n = shape.at(0);
        k = shape.size() == 2 ? shape[1] : 1;
        P = n * k;
        n_tiles = bgmm_group_rows_tiles(P, (int32_t)K);
        if (store.scalar_type() != at::kInt || store.dim() != 1 || store.numel() < size(P, K)) refuse(BGMM_OPS_EINVAL, "RowGroups: the store does not fit");
    }
    static int64_t size(int64_t P, int64_t K) {
        return 4 * bgmm_group_rows_tiles(P, (int32_t)K) + 2 * P + (BGMM_OPS_LEVELS + 1) * (K + 2);
    }
    int32_t *tiles() const { return store.numel() ? store.data_ptr<int32_t>() : nullptr; }
    int32_t *bucket() const { return tiles() + 4 * n_tiles; }
    int32_t *order() const { return bucket() + P; }
    int32_t *offsets() const { return order() + P; }
    int32_t *first() const { return offsets() + K + 2; }
    Tensor part(int64_t at, int64_t size) const { return store.narrow(0, at, size); }
};
typedef std::shared_ptr<RowGroups> Groups;

Groups group_rows(const Tensor &labels, int64_t components) {
    const char *what = "group_rows";
    if (labels.scalar_type() != at::kLong) refuse(BGMM_OPS_EINVAL, "%s: labels are %s, not int64", what, c10::toString(labels.scalar_type()));
    if (labels.dim() != 1 && labels.dim() != 2) refuse(BGMM_OPS_EINVAL, "%s: labels have %d axes, not 1 or 2", what, (int)labels.dim());
    if (labels.dim() == 2 && (labels.size(1) < 1 || labels.size(1) > BGMM_OPS_MAX_CHOSEN))
        refuse(BGMM_OPS_EINVAL, "%s: %lld labels per row (1 .. %d)", what, (long long)labels.size(1), BGMM_OPS_MAX_CHOSEN);
    if (components < 1) refuse(BGMM_OPS_EINVAL, "%s: %lld components", what, (long long)components);
    if (components > BGMM_OPS_MAX_COMPONENTS) refuse(BGMM_OPS_EUNSUPPORTED, "%s: %lld components (at most %d)", what, (long long)components, BGMM_OPS_MAX_COMPONENTS);
    if (labels.numel() > 0x7fffffff - 65536) refuse(BGMM_OPS_EUNSUPPORTED, "%s: %lld labels (at most 2^31 - 65537)", what, (long long)labels.numel());
    Device dev{what};
    dev("labels", labels);
    const Tensor flat = packed(labels);
    const c10::OptionalDeviceGuard guard(labels.device());
    auto g = std::make_shared<RowGroups>(labels.sizes().vec(), components, at::empty({RowGroups::size(labels.numel(), components)}, labels.options().dtype(at::kInt)));
    const int64_t bytes = bgmm_group_rows_ws(g->P, (int32_t)g->K);
    const Tensor ws = bytes ? at::empty({bytes}, labels.options().dtype(at::kByte)) : Tensor();
    check(bgmm_group_rows(g->P ? flat.data_ptr<int64_t>() : nullptr, g->P, (int32_t)g->K, g->bucket(), g->order(), g->offsets(), g->first(), g->tiles(), ptr(ws), bytes,
                          stream_of(labels)));
    return g;
}

// ------------------------------------------------------------------------------------------ route
struct Routed {
    Tensor labels, weights, stats;
};

Routed route_forward(const Tensor &lw, int64_t k, bool renormalise, bool want_stats) {
    const c10::OptionalDeviceGuard guard(lw.device());
    const Rows rows = rows_of(lw);
    const int64_t n = lw.size(0), K = lw.size(1);
    const auto acc = lw.options().dtype(acc_of(lw.scalar_type()));
    Routed r;
    r.labels = at::empty({n, k}, lw.options().dtype(at::kLong));
    r.weights = at::empty({n, k}, acc);
    if (want_stats) r.stats = at::empty({n, 2}, acc);
    check(bgmm_route(type_of(lw.scalar_type()), ptr(rows.t), rows.stride, n, (int32_t)K, (int32_t)k, renormalise, (int64_t *)ptr(r.labels), ptr(r.weights),
                     ptr(r.stats), stream_of(lw)));
    return r;
}

struct RouteFunction : torch::autograd::Function<RouteFunction> {
    static variable_list forward(AutogradContext *ctx, const Tensor &lw, int64_t k, bool renormalise) {
        const Routed r = route_forward(lw, k, renormalise, !renormalise);
        ctx->saved_data["k"] = k;
        ctx->saved_data["K"] = lw.size(1);
        ctx->saved_data["renormalise"] = renormalise;
        ctx->saved_data["dtype"] = (int64_t)lw.scalar_type();
        ctx->save_for_backward(renormalise ? variable_list{r.labels, r.weights} : variable_list{r.labels, r.weights, lw, r.stats});
        ctx->mark_non_differentiable({r.labels});
        ctx->set_materialize_grads(false);
        return {r.labels, r.weights};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        first_order_only("route");
        if (!grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &labels = saved[0], &weights = saved[1];
        const bool renormalise = ctx->saved_data["renormalise"].toBool();
        const int64_t k = ctx->saved_data["k"].toInt(), K = ctx->saved_data["K"].toInt();
        const at::ScalarType dtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
        const c10::OptionalDeviceGuard guard(labels.device());
        const Rows lw = renormalise ? Rows() : rows_of(saved[2]);
        const Tensor d = packed(grads[1]);
        Tensor out = at::empty({labels.size(0), K}, labels.options().dtype(dtype));
        check(bgmm_route_backward(type_of(dtype), ptr(lw.t), lw.stride, labels.size(0), (int32_t)K, (int32_t)k, renormalise, (int64_t *)ptr(labels), ptr(weights),
                                  renormalise ? nullptr : ptr(saved[3]), ptr(d), ptr(out), stream_of(labels)));
        return {out, Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> route(const Tensor &lw, int64_t k, bool renormalise) {
    const char *what = "route";
    if (lw.dim() != 2) refuse(BGMM_OPS_EINVAL, "%s: log_weights has %d axes, not 2", what, (int)lw.dim());
    type_of(what, "log_weights", lw);
    if (k < 1 || k > lw.size(1)) refuse(BGMM_OPS_EINVAL, "%s: k = %lld of %lld components", what, (long long)k, (long long)lw.size(1));
    if (k > BGMM_OPS_MAX_CHOSEN) refuse(BGMM_OPS_EUNSUPPORTED, "%s: k = %lld (at most %d)", what, (long long)k, BGMM_OPS_MAX_CHOSEN);
    if (lw.size(1) > 0x7fffffff) refuse(BGMM_OPS_EUNSUPPORTED, "%s: %lld components", what, (long long)lw.size(1));
    Device dev{what};
    dev("log_weights", lw);
    const c10::OptionalDeviceGuard guard(lw.device());
    if (differentiable(what, {lw})) {
        const variable_list r = RouteFunction::apply(lw, k, renormalise);
        return {r[0], r[1]};
    }
    const Routed r = route_forward(lw, k, renormalise, false);
    return {r.labels, r.weights};
}

// ------------------------------------------------------------------------------------------ grouped_matmul
// A (K, d_in, d_out) weight: strides of its components and rows, and whether d_in is the contiguous axis.
struct Matrices {
    Tensor t;
    int64_t component, row;
    bool in_contiguous;
};
Matrices matrices_of(const Tensor &stored) {
    const Tensor w = values(stored);
    const int64_t s0 = w.stride(0), s1 = w.stride(1), s2 = w.stride(2);
    if (s0 >= 0 && s1 >= 0 && (s2 == 1 || w.size(2) == 1)) return {w, s0, s1, false};
    if (s0 >= 0 && s2 >= 0 && (s1 == 1 || w.size(1) == 1)) return {w, s0, s2, true};
    return {w.contiguous(), w.size(1) * w.size(2), w.size(2), false};
}

// One product; `transposed` contracts over the weight's second axis instead of its first.
void product(const RowGroups &g, const Rows &x, int64_t x_div, const Matrices &w, bool transposed, const Rows &bias, const Tensor &gates, const Tensor &out,
             const Tensor &ws, int splits, const Rows &dot_in = {}, int64_t dot_div = 1, const Tensor &dots = {}) {
    const int64_t d_in = w.t.size(1), d_out = w.t.size(2), kdim = transposed ? d_out : d_in, ndim = transposed ? d_in : d_out;
    check(bgmm_rows_product(type_of(x.t.scalar_type()), ptr(x.t), x.stride, (int32_t)x_div, ptr(w.t), w.component, w.row, w.in_contiguous != transposed,
                            ptr(bias.t), bias.stride, ptr(gates), ptr(out), ndim, ptr(ws), splits, ptr(dot_in.t), dot_in.stride, (int32_t)dot_div, ptr(dots), g.P, (int32_t)g.K,
                            (int32_t)kdim, (int32_t)ndim, g.order(),
                            g.tiles(), stream_of(x.t)));
}

Tensor matmul_forward(const Tensor &x_in, const Tensor &weight, const RowGroups &g, const Tensor &bias_in, const Tensor &gates_in) {
    const c10::OptionalDeviceGuard guard(x_in.device());
    const int type = type_of(x_in.scalar_type());
    const int64_t d_in = weight.size(1), d_out = weight.size(2), x_div = x_in.dim() == 3 ? 1 : g.k;
    const bool gated = gates_in.defined();
    std::vector<int64_t> shape = gated ? std::vector<int64_t>{g.n} : g.shape;
    shape.push_back(d_out);
    Tensor y = at::empty(shape, x_in.options());
    if (g.P == 0) return y;
    const Rows x = rows_of(x_in), bias = rows_of(bias_in);
    const Tensor gates = gated ? packed(gates_in) : gates_in;
    const int splits = bgmm_rows_product_splits(type, g.P, (int32_t)g.K, (int32_t)d_in, (int32_t)d_out);
    if (splits == 1 && !(gated && g.k > 1)) {
        product(g, x, x_div, matrices_of(weight), false, bias, gates, y, Tensor(), 1);
    } else {
        const Tensor ws = at::empty({splits, g.P, d_out}, x_in.options().dtype(acc_of(x_in.scalar_type())));
        product(g, x, x_div, matrices_of(weight), false, bias, Tensor(), Tensor(), ws, splits);
        check(bgmm_combine(type, ptr(ws), splits, gated ? g.n : g.P, gated ? (int32_t)g.k : 1, (int32_t)g.K, g.bucket(), ptr(gates), ptr(y), d_out, (int32_t)d_out,
                           nullptr, nullptr, 0, nullptr, 0, nullptr, 0, 1, 1, stream_of(x_in)));
    }
    return y;
}

struct MatmulFunction : torch::autograd::Function<MatmulFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Maybe &bias, const Maybe &gates, const Groups &g) {
        ctx->saved_data["K"] = g->K;
        ctx->saved_data["shape"] = g->shape;
        ctx->save_for_backward({x, weight, given(bias), given(gates), g->store});
        ctx->set_materialize_grads(false);
        return matmul_forward(x, weight, *g, given(bias), given(gates));
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        first_order_only("grouped_matmul");
        variable_list out(5);
        if (!grads[0].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x_in = saved[0], &weight = saved[1], &bias_in = saved[2];
        const RowGroups g(ctx->saved_data["shape"].toIntVector(), ctx->saved_data["K"].toInt(), saved[4]);
        const c10::OptionalDeviceGuard guard(x_in.device());
        const auto opts = x_in.options(), acc = opts.dtype(acc_of(x_in.scalar_type()));
        const int type = type_of(x_in.scalar_type());
        const int64_t d_in = weight.size(1), d_out = weight.size(2), x_div = x_in.dim() == 3 ? 1 : g.k;
        const bool has_b = bias_in.defined(), has_g = saved[3].defined();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(2),
                   need_g = has_g && ctx->needs_input_grad(2 + has_b);
        const Tensor gates = has_g ? packed(saved[3]) : Tensor();
        const Rows x = rows_of(x_in), d = rows_of(grads[0]);
        const int64_t d_div = has_g ? g.k : 1;
        void *st = stream_of(x_in);
        if (need_x) out[0] = at::empty(x_in.sizes(), opts);
        if (need_g) out[3] = at::empty(gates.sizes(), acc);
        if ((need_x || need_g) && g.P > 0) {
            const int splits = bgmm_rows_product_splits(type, g.P, (int32_t)g.K, (int32_t)d_out, (int32_t)d_in);
            const Rows bias = need_g ? rows_of(bias_in) : Rows();
            // (which way does not depend on what else is asked for, so that a gradient is the same bits either way)
            if (splits == 1 && x_div == 1) {
                // The gates' gradient from dots beside the product, so that nothing else is written (114804 rows, 905 -> 16 double, all
                // gradients: 1166 us with a workspace, 890; the gates' alone 763 and 455).
                const int n_dots = need_g ? bgmm_rows_product_dots(type, g.P, (int32_t)g.K, (int32_t)d_out, (int32_t)d_in, splits) : 0;
                const Tensor dots = need_g ? at::empty({g.P, n_dots}, acc) : Tensor();
                product(g, d, d_div, matrices_of(weight), true, {}, gates, out[0], Tensor(), splits, need_g ? x : Rows(), x_div, dots);
                if (need_g)
                    check(bgmm_gate_gradient(type, ptr(dots), n_dots, g.P, (int32_t)g.K, g.bucket(), ptr(bias.t), bias.stride, ptr(d.t), d.stride, (int32_t)d_div,
                                             (int32_t)d_out, ptr(out[3]), st));
            } else {
                // several products of a row to add: their workspace is read anyway, by whole rows, and the dots come from it (8192 rows, 2
                // of 64 components, 1024 -> 2048 bfloat16: 474 us, 507 with dots beside the product)
                const Tensor ws = at::empty({splits, g.P, d_in}, acc);
                product(g, d, d_div, matrices_of(weight), true, {}, Tensor(), Tensor(), ws, splits);
                check(bgmm_combine(type, ptr(ws), splits, g.P / x_div, (int32_t)x_div, (int32_t)g.K, g.bucket(), ptr(gates), ptr(out[0]), d_in, (int32_t)d_in,
                                   ptr(out[3]), need_g ? ptr(x.t) : nullptr, x.stride, ptr(bias.t), bias.stride, ptr(d.t), d.stride, (int32_t)d_div, (int32_t)d_out, st));
            }
        }
        if (need_w || need_b) {
            if (need_w) out[1] = at::empty({g.K, d_in, d_out}, opts);
            if (need_b) out[2] = at::empty({g.K, d_out}, opts);
            const int64_t bytes = bgmm_weight_product_ws(type, g.P, (int32_t)g.K, (int32_t)d_in, (int32_t)d_out);
            const Tensor ws = bytes ? at::empty({bytes}, opts.dtype(at::kByte)) : Tensor();
            check(bgmm_weight_product(type, ptr(x.t), x.stride, (int32_t)x_div, ptr(d.t), d.stride, (int32_t)d_div, ptr(gates), ptr(out[1]), ptr(out[2]), ptr(ws), bytes,
                                      g.P, (int32_t)g.K, (int32_t)d_in, (int32_t)d_out, g.order(), g.offsets(), g.first(), st));
        }
        return out;
    }
};

Tensor grouped_matmul(const Tensor &x, const Tensor &weight, const Groups &g, const Maybe &bias, const Maybe &gates) {
    const char *what = "grouped_matmul";
    type_of(what, "x", x);
    const Tensor b = given(bias), gt = given(gates);
    if (weight.scalar_type() != x.scalar_type() || (b.defined() && b.scalar_type() != x.scalar_type()))
        refuse(BGMM_OPS_EINVAL, "%s: x, weight and bias have to be of one type", what);
    if (weight.dim() != 3 || weight.size(0) != g->K || weight.size(1) < 1 || weight.size(2) < 1 || weight.size(1) > BGMM_OPS_MAX_AXIS || weight.size(2) > BGMM_OPS_MAX_AXIS)
        refuse(BGMM_OPS_EINVAL, "%s: weight is %s, not (%lld, d_in, d_out)", what, shape_of(weight).c_str(), (long long)g->K);
    const int64_t d_in = weight.size(1), d_out = weight.size(2);
    const bool per_label = x.dim() == 3 && g->shape.size() == 2;
    if (per_label ? x.size(0) != g->n || x.size(1) != g->k || x.size(2) != d_in : x.dim() != 2 || x.size(0) != g->n || x.size(1) != d_in)
        refuse(BGMM_OPS_EINVAL, "%s: x is %s with a grouping of %lld rows, %lld labels each, and %lld inputs", what, shape_of(x).c_str(), (long long)g->n, (long long)g->k, (long long)d_in);
    if (b.defined() && (b.dim() != 2 || b.size(0) != g->K || b.size(1) != d_out))
        refuse(BGMM_OPS_EINVAL, "%s: bias is %s, not (%lld, %lld)", what, shape_of(b).c_str(), (long long)g->K, (long long)d_out);
    if (gt.defined()) {
        if (gt.sizes() != at::IntArrayRef(g->shape)) refuse(BGMM_OPS_EINVAL, "%s: gates are %s, not of the labels' shape", what, shape_of(gt).c_str());
        if (gt.scalar_type() != acc_of(x.scalar_type()))
            refuse(BGMM_OPS_EINVAL, "%s: gates are %s, not %s", what, c10::toString(gt.scalar_type()), c10::toString(acc_of(x.scalar_type())));
    }
    Device dev{what};
    dev("x", x);
    dev("weight", weight);
    dev("bias", b);
    dev("gates", gt);
    dev("the grouping", g->store);
    const c10::OptionalDeviceGuard guard(x.device());
    if (differentiable(what, {x, weight, b, gt}))
        return MatmulFunction::apply(x, weight, bias, gates, g);
    return matmul_forward(x, weight, *g, b, gt);
}

// ------------------------------------------------------------------------------------------ verify_drafts
Tensor last_contiguous(const Tensor &t) { return t.size(2) == 1 || t.stride(2) == 1 ? values(t) : packed(t); }

std::tuple<Tensor, Tensor> verify_drafts(const Tensor &target_in, const Tensor &draft_in, const Tensor &labels, const Tensor &u_accept, const Tensor &u_draw,
                                         const Maybe &lengths_in) {
    const char *what = "verify_drafts";
    if (target_in.dim() != 3 || draft_in.dim() != 3) refuse(BGMM_OPS_EINVAL, "%s: target and draft have %d and %d axes, not 3", what, (int)target_in.dim(), (int)draft_in.dim());
    const int64_t B = draft_in.size(0), T = draft_in.size(1), V = draft_in.size(2);
    if (target_in.size(0) != B || target_in.size(1) != T + 1 || target_in.size(2) != V)
        refuse(BGMM_OPS_EINVAL, "%s: target is %s, draft %s", what, shape_of(target_in).c_str(), shape_of(draft_in).c_str());
    if (V < 1) refuse(BGMM_OPS_EINVAL, "%s: no labels", what);
    if (T > (1 << 20)) refuse(BGMM_OPS_EUNSUPPORTED, "%s: %lld drafts (at most 2^20)", what, (long long)T);
    const int type = type_of(what, "target", target_in);
    if (draft_in.scalar_type() != target_in.scalar_type()) refuse(BGMM_OPS_EINVAL, "%s: target is %s, draft %s", what, c10::toString(target_in.scalar_type()), c10::toString(draft_in.scalar_type()));
    const auto wants = [&](const char *name, const Tensor &t, at::ScalarType type, at::IntArrayRef shape) {
        if (t.scalar_type() != type || t.sizes() != shape) refuse(BGMM_OPS_EINVAL, "%s: %s is %s %s", what, name, c10::toString(t.scalar_type()), shape_of(t).c_str());
    };
    wants("labels", labels, at::kLong, {B, T});
    wants("u_accept", u_accept, at::kDouble, {B, T});
    wants("u_draw", u_draw, at::kDouble, {B});
    const Tensor len_in = given(lengths_in);
    if (len_in.defined()) wants("lengths", len_in, at::kLong, {B});
    Device dev{what};
    dev("target", target_in);
    dev("draft", draft_in);
    dev("labels", labels);
    dev("u_accept", u_accept);
    dev("u_draw", u_draw);
    dev("lengths", len_in);
    const c10::OptionalDeviceGuard guard(target_in.device());
    const Tensor p = last_contiguous(target_in), q = last_contiguous(draft_in), z = packed(labels), ua = packed(u_accept), ud = packed(u_draw);
    const Tensor len = len_in.defined() ? packed(len_in) : len_in;
    Tensor out = at::empty({B, T + 1}, labels.options()), accepted = at::empty({B}, labels.options());
    const int64_t bytes = bgmm_verify_drafts_ws(B, V);
    const Tensor ws = bytes ? at::empty({bytes}, labels.options().dtype(at::kByte)) : Tensor();
    check(bgmm_verify_drafts(type, ptr(p), p.stride(0), p.stride(1), ptr(q), q.stride(0), q.stride(1), (const int64_t *)ptr(z), (const double *)ptr(ua),
                             (const double *)ptr(ud), (const int64_t *)ptr(len), B, (int32_t)T, V, (int64_t *)ptr(out), (int64_t *)ptr(accepted), ptr(ws), bytes,
                             stream_of(p)));
    return {out, accepted};
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refusal &r) {
            const py::object cls = py::module_::import("pybgmm_amd._lib").attr("BGMMError");
            PyErr_SetObject(cls.ptr(), cls(r.code, r.what()).ptr());
        }
    });
    py::class_<RowGroups, Groups>(m, "RowGroups")
        .def(py::init([](std::vector<int64_t> shape, int64_t components, Tensor store) {
                 // (what the kernels follow is group_rows' own work)
                 if (!store.device().is_cpu()) refuse(BGMM_OPS_EDEVICE, "RowGroups: a grouping on a device comes from group_rows");
                 return std::make_shared<RowGroups>(std::move(shape), components, store);
             }),
             py::arg("labels_shape"), py::arg("n_components"), py::arg("store"))
        .def_static("store_size", &RowGroups::size)
        .def("record_stream", [](const RowGroups &g, const py::object &stream) { py::cast(g.store).attr("record_stream")(stream); }, py::arg("stream"),
             "What Tensor.record_stream is for a tensor: this grouping's memory is not used again before the work queued on `stream` is done.")
        .def_property_readonly("labels_shape", [](const RowGroups &g) { return py::tuple(py::cast(g.shape)); })
        .def_readonly("n_components", &RowGroups::K)
        .def_readonly("n", &RowGroups::n)
        .def_readonly("k", &RowGroups::k)
        .def_property_readonly("tiles", [](const RowGroups &g) { return g.part(0, 4 * g.n_tiles); })
        .def_property_readonly("bucket", [](const RowGroups &g) { return g.part(4 * g.n_tiles, g.P); })
        .def_property_readonly("order", [](const RowGroups &g) { return g.part(4 * g.n_tiles + g.P, g.P); })
        .def_property_readonly("offsets", [](const RowGroups &g) { return g.part(4 * g.n_tiles + 2 * g.P, g.K + 2); })
        .def_property_readonly("first", [](const RowGroups &g) { return g.part(4 * g.n_tiles + 2 * g.P + g.K + 2, BGMM_OPS_LEVELS * (g.K + 2)); })
        .def_property_readonly("counts", [](const RowGroups &g) {
            const int64_t at = 4 * g.n_tiles + 2 * g.P;
            return g.part(at + 1, g.K) - g.part(at, g.K);
        });
    m.def("group_rows", &group_rows);
    m.def("route", &route);
    m.def("grouped_matmul", &grouped_matmul, py::arg("x"), py::arg("weight"), py::arg("groups").none(false), py::arg("bias"), py::arg("gates"));
    m.def("verify_drafts", &verify_drafts);
}
