"""Rows routed to components: the most probable ones of every row (``route``), rows grouped by component (``group_rows``)."""
import torch

from . import _native as nat


def route(log_weights, k, renormalise=True):
    """
    The ``k`` most probable components of every row of ``log_weights`` (n, K) and their weights.

    Returns ``(labels, weights)``: int64 (n, k), ordered by (log weight descending, index ascending), and the softmax over
    the chosen components (``renormalise=True``) or over all of them (``False``: the posterior's own shares), float64 for float64
    input and float32 otherwise.  Components at -inf (no members, masked) or NaN are never chosen and have no weight; a row with
    fewer than ``k`` others fills up with label -1, weight 0 -- what ``group_rows`` takes for "no component".
    ``weights`` is differentiable with respect to ``log_weights``.  float64 / 32 / 16, bfloat16; k at most 32.
    """
    what = "route"
    nat.require_tensors(what, log_weights=log_weights)
    if not (log_weights.dim() == 2):
        nat.refuse("%s: log_weights has %d axes, not 2", what, log_weights.dim())
    if not (log_weights.dtype in nat.DTYPES):
        nat.refuse("%s: log_weights are %s", what, log_weights.dtype)
    K = log_weights.shape[1]
    if not (int(k) == k and 1 <= k <= K):
        nat.refuse("%s: k = %s of %d components", what, k, K)
    if k > nat.MAX_CHOSEN:
        nat.refuse("%s: k = %d (at most %d)", what, k, nat.MAX_CHOSEN, code=-5)
    nat.require_device(what, log_weights=log_weights)
    if torch.is_grad_enabled() and log_weights.requires_grad:
        return _Route.apply(log_weights, int(k), bool(renormalise))
    return _route(log_weights, int(k), bool(renormalise), False)[:2]


def _row_stride(t):
    """(tensor, stride of its rows): the tensor itself if its last axis is contiguous, a copy otherwise."""
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < 0):
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else t.shape[1])


def _route(lw, k, renormalise, want_stats):
    L = nat.load()
    lw, stride = _row_stride(lw)
    n, K = lw.shape
    acc = nat.acc_dtype(lw.dtype)
    labels = torch.empty((n, k), dtype=torch.int64, device=lw.device)
    weights = torch.empty((n, k), dtype=acc, device=lw.device)
    stats = torch.empty((n, 2), dtype=acc, device=lw.device) if want_stats else None
    with nat.on(lw.device):
        nat.check(L.bgmm_route(nat.DTYPES[lw.dtype], nat.ptr(lw), stride, n, K, k, int(renormalise), nat.ptr(labels), nat.ptr(weights),
                               nat.ptr(stats), nat.stream(lw.device)))
    return labels, weights, stats


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lw, k, renormalise):
        labels, weights, stats = _route(lw, k, renormalise, not renormalise)
        ctx.k, ctx.renormalise, ctx.K, ctx.dtype = k, renormalise, lw.shape[1], lw.dtype
        ctx.save_for_backward(labels, weights, *(() if renormalise else (lw, stats)))
        ctx.mark_non_differentiable(labels)
        return labels, weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, dweights):
        L = nat.load()
        labels, weights = ctx.saved_tensors[:2]
        lw, stats = (None, None) if ctx.renormalise else ctx.saved_tensors[2:]
        stride = 0
        if lw is not None:
            lw, stride = _row_stride(lw)
        n = labels.shape[0]
        dweights = dweights.contiguous()
        out = torch.empty((n, ctx.K), dtype=ctx.dtype, device=labels.device)
        with nat.on(out.device):
            nat.check(L.bgmm_route_backward(nat.DTYPES[ctx.dtype], nat.ptr(lw), stride, n, ctx.K, ctx.k, int(ctx.renormalise), nat.ptr(labels),
                                            nat.ptr(weights), nat.ptr(stats), nat.ptr(dweights), nat.ptr(out), nat.stream(out.device)))
        return out, None, None


class RowGroups(object):
    """
    Rows grouped by component (``group_rows``).

    ``labels_shape``: (n,) or (n, k); ``n_components``; ``order`` int32: flat label indices sorted by (component, index), those of
    no component last; ``offsets`` int32 (n_components + 2,): component e holds ``order[offsets[e]:offsets[e + 1]]``, the last
    bucket the rows of no component.  ``counts``: rows per component.  The tensors belong to the grouping: products read them.
    """

    def __init__(self, labels_shape, n_components, bucket, order, offsets, first, tiles):
        self.labels_shape, self.n_components = tuple(labels_shape), n_components
        self.bucket, self.order, self.offsets, self.first, self.tiles = bucket, order, offsets, first, tiles
        self.device = order.device
        self.n = self.labels_shape[0]
        self.k = self.labels_shape[1] if len(self.labels_shape) == 2 else 1

    @property
    def counts(self):
        return self.offsets[1:self.n_components + 1] - self.offsets[:self.n_components]


def group_rows(labels, n_components):
    """
    Group rows by their component: ``labels`` int64 (n,), one per row, or (n, k), k per row (``route``'s).  A label outside
    0 .. n_components - 1 -- the samplers' -1 -- is a row of no component: products give zeros for it.  The order within a
    component is the rows' own, so that a grouping, and every sum over one, is the same every time.  At most 8000 components.
    Returns a ``RowGroups`` for any number of ``grouped_matmul`` calls.
    """
    what = "group_rows"
    nat.require_tensors(what, labels=labels)
    if not (labels.dtype == torch.int64):
        nat.refuse("%s: labels are %s, not int64", what, labels.dtype)
    if not (labels.dim() in (1, 2)):
        nat.refuse("%s: labels have %d axes, not 1 or 2", what, labels.dim())
    if not (labels.dim() == 1 or 1 <= labels.shape[1] <= nat.MAX_CHOSEN):
        nat.refuse("%s: %d labels per row (1 .. %d)", what, labels.shape[-1] if labels.dim() == 2 else 1, nat.MAX_CHOSEN)
    if not (int(n_components) == n_components and n_components >= 1):
        nat.refuse("%s: %s components", what, n_components)
    if n_components > nat.MAX_COMPONENTS:
        nat.refuse("%s: %d components (at most %d)", what, n_components, nat.MAX_COMPONENTS, code=-5)
    nat.require_device(what, labels=labels)
    L = nat.load()
    K, P = int(n_components), labels.numel()
    dev = labels.device
    flat = labels.contiguous()
    n_first = nat.LEVELS * (K + 2)
    n_tiles, ws_bytes = L.bgmm_group_rows_tiles(P, K), L.bgmm_group_rows_ws(P, K)
    # one allocation
    tiles, bucket, order, offsets, first, ws = torch.empty(4 * n_tiles + 2 * P + K + 2 + n_first + ws_bytes // 4, dtype=torch.int32, device=dev).split(
        [4 * n_tiles, P, P, K + 2, n_first, ws_bytes // 4])
    with nat.on(dev):
        nat.check(L.bgmm_group_rows(nat.ptr(flat), P, K, nat.ptr(bucket), nat.ptr(order), nat.ptr(offsets), nat.ptr(first), nat.ptr(tiles), nat.ptr(ws),
                                    ws_bytes, nat.stream(dev)))
    return RowGroups(labels.shape, K, bucket, order, offsets, first, tiles)
