"""Rows times the matrix of their own component, ragged groups (``grouped_matmul``)."""
import torch

from . import _native as nat
from .routing import RowGroups, _row_stride


def grouped_matmul(x, weight, groups, bias=None, gates=None):
    """
    Every row times its own component's matrix: ``y_i = x_i W_e + b_e`` for the component e of row i.

    x       (n, d_in); or (n, k, d_in) -- a row per label -- where the grouping has k labels per row
    weight  (K, d_in, d_out), x's type; a transposed view of (K, d_out, d_in) is taken as it is
    groups  ``group_rows(labels, K)``
    bias    (K, d_out), x's type, or None
    gates   the grouping's label shape, float64 for float64 rows and float32 otherwise (``route``'s weights), or None

    Returns, in x's type and in the rows' own order: with gates (n, d_out), the gated sum over a row's components; without, a
    row per label, (n, d_out) or (n, k, d_out).  Labels of no component contribute zeros, and whatever x holds in such rows is not
    read.  Products of 16-bit types accumulate in 32 bits, and so does the gated sum, which is rounded once.  Differentiable
    with respect to x, weight, bias and gates (once); the sums run in a fixed order.  float64 / 32 / 16, bfloat16.
    """
    what = "grouped_matmul"
    if not (isinstance(groups, RowGroups)):
        nat.refuse("%s: groups is no RowGroups", what)
    nat.require_tensors(what, x=x, weight=weight, bias=bias, gates=gates)
    n, k, K = groups.n, groups.k, groups.n_components
    if not (x.dtype in nat.DTYPES):
        nat.refuse("%s: x is %s", what, x.dtype)
    if not (weight.dtype == x.dtype and (bias is None or bias.dtype == x.dtype)):
        nat.refuse("%s: x, weight and bias have to be of one type", what)
    if not (weight.dim() == 3 and weight.shape[0] == K and min(weight.shape) >= 1):
        nat.refuse("%s: weight is %s, not (%d, d_in, d_out)", what, tuple(weight.shape), K)
    d_in, d_out = weight.shape[1:]
    per_label = x.dim() == 3
    if not (tuple(x.shape) == ((n, k, d_in) if per_label and len(groups.labels_shape) == 2 else (n, d_in))):
        nat.refuse("%s: x is %s with a grouping of %s labels and %d inputs", what, tuple(x.shape), groups.labels_shape, d_in)
    if not (bias is None or tuple(bias.shape) == (K, d_out)):
        nat.refuse("%s: bias is %s, not (%d, %d)", what, None if bias is None else tuple(bias.shape), K, d_out)
    if gates is not None:
        if not (tuple(gates.shape) == groups.labels_shape):
            nat.refuse("%s: gates are %s, the labels %s", what, tuple(gates.shape), groups.labels_shape)
        if not (gates.dtype == nat.acc_dtype(x.dtype)):
            nat.refuse("%s: gates are %s, not %s", what, gates.dtype, nat.acc_dtype(x.dtype))
    dev = nat.require_device(what, x=x, weight=weight, bias=bias, gates=gates)
    if not (dev == groups.device):
        nat.refuse("%s: the grouping is on %s, x on %s", what, groups.device, dev)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, gates)):
        return _GroupedMatmul.apply(x, weight, bias, gates, groups)
    return _forward(x, weight, bias, gates, groups)


def _rows(t):
    """A (n, d) or (n, k, d) tensor as rows: (tensor, row stride)."""
    if t.dim() == 3:
        t = t.reshape(-1, t.shape[2])        # (a view where the strides allow it)
    return _row_stride(t)


def _matrices(w):
    """(tensor, component stride, row stride, whether d_in is the contiguous axis) of a (K, d_in, d_out) weight."""
    _, d_in, d_out = w.shape
    s0, s1, s2 = w.stride()
    if s0 >= 0 and (s2 == 1 or d_out == 1) and s1 >= 0:
        return w, s0, s1, False
    if s0 >= 0 and (s1 == 1 or d_in == 1) and s2 >= 0:
        return w, s0, s2, True
    w = w.contiguous()
    return w, d_in * d_out, d_out, False


def _product(x, x_stride, x_div, w, transposed, bias, gates, out, ws, splits, groups, P):
    """One ``bgmm_rows_product``: ``transposed`` contracts over the weight's second axis instead of its first."""
    L = nat.load()
    w, w_comp, w_row, in_contiguous = _matrices(w)
    kdim, ndim = (w.shape[2], w.shape[1]) if transposed else (w.shape[1], w.shape[2])
    bias, bias_row = (None, 0) if bias is None else _row_stride(bias)
    nat.check(L.bgmm_rows_product(nat.DTYPES[x.dtype], nat.ptr(x), x_stride, x_div, nat.ptr(w), w_comp, w_row, int(in_contiguous != transposed),
                                  nat.ptr(bias), bias_row, nat.ptr(gates), nat.ptr(out), ndim, nat.ptr(ws), splits, P, groups.n_components,
                                  kdim, ndim, nat.ptr(groups.order), nat.ptr(groups.tiles), nat.stream(x.device)))


def _forward(x, weight, bias, gates, groups):
    L = nat.load()
    n, k, K = groups.n, groups.k, groups.n_components
    P, dev, dt = n * k, x.device, x.dtype
    d_in, d_out = weight.shape[1:]
    x_div = 1 if x.dim() == 3 else k
    x, x_stride = _rows(x)
    gates = None if gates is None else gates.contiguous()
    summed = gates is not None and k > 1
    y = torch.empty((n, d_out) if gates is not None else groups.labels_shape + (d_out,), dtype=dt, device=dev)
    with nat.on(dev):
        splits = L.bgmm_rows_product_splits(nat.DTYPES[dt], P, K, d_in, d_out)
        if splits == 1 and not summed:
            _product(x, x_stride, x_div, weight, False, bias, gates, y, None, 1, groups, P)
        else:
            ws = torch.empty((splits, P, d_out), dtype=nat.acc_dtype(dt), device=dev)
            _product(x, x_stride, x_div, weight, False, bias, None, None, ws, splits, groups, P)
            rows, per = (n, k) if gates is not None else (P, 1)
            nat.check(L.bgmm_combine(nat.DTYPES[dt], nat.ptr(ws), splits, rows, per, K, nat.ptr(groups.bucket), nat.ptr(gates), nat.ptr(y), d_out,
                                     d_out, None, None, 0, None, 0, None, 0, 1, 1, nat.stream(dev)))
    return y


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gates, groups):
        ctx.groups = groups
        ctx.save_for_backward(x, weight, bias, gates)
        return _forward(x, weight, bias, gates, groups)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        L = nat.load()
        x_in, weight, bias, gates_in = ctx.saved_tensors
        g = ctx.groups
        n, k, K = g.n, g.k, g.n_components
        P, dev, dt = n * k, x_in.device, x_in.dtype
        code, acc = nat.DTYPES[dt], nat.acc_dtype(dt)
        d_in, d_out = weight.shape[1:]
        need_x, need_w, need_b, need_g = ctx.needs_input_grad[:4]
        x_div = 1 if x_in.dim() == 3 else k
        x, x_stride = _rows(x_in)
        gates = None if gates_in is None else gates_in.contiguous()
        d, d_stride = _rows(dy)
        d_div = k if gates is not None else 1
        dx = dw = db = dg = None
        with nat.on(dev):
            st = nat.stream(dev)
            if need_x or need_g:
                splits = L.bgmm_rows_product_splits(code, P, K, d_out, d_in)
                if need_x:
                    dx = torch.empty(x_in.shape, dtype=dt, device=dev)
                if splits == 1 and x_div == 1 and not need_g:
                    _product(d, d_stride, d_div, weight, True, None, gates, dx, None, 1, g, P)
                else:
                    ws = torch.empty((splits, P, d_in), dtype=acc, device=dev)
                    _product(d, d_stride, d_div, weight, True, None, None, None, ws, splits, g, P)
                    if need_g:
                        dg = torch.empty(gates.shape, dtype=acc, device=dev)
                    b, b_row = (None, 0) if bias is None else _row_stride(bias)
                    nat.check(L.bgmm_combine(code, nat.ptr(ws), splits, P // x_div, x_div, K, nat.ptr(g.bucket), nat.ptr(gates), nat.ptr(dx), d_in,
                                             d_in, nat.ptr(dg), nat.ptr(x) if need_g else None, x_stride, nat.ptr(b) if need_g else None, b_row,
                                             nat.ptr(d), d_stride, d_div, d_out, st))
            if need_w or need_b:
                if need_w:
                    dw = torch.empty((K, d_in, d_out), dtype=dt, device=dev)
                if need_b:
                    db = torch.empty((K, d_out), dtype=dt, device=dev)
                ws_bytes = L.bgmm_weight_product_ws(code, P, K, d_in, d_out)
                ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
                nat.check(L.bgmm_weight_product(code, nat.ptr(x), x_stride, x_div, nat.ptr(d), d_stride, d_div, nat.ptr(gates), nat.ptr(dw),
                                                nat.ptr(db), nat.ptr(ws), ws_bytes, P, K, d_in, d_out, nat.ptr(g.order), nat.ptr(g.offsets),
                                                nat.ptr(g.first), st))
        return dx, dw, db, dg, None
