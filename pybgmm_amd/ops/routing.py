"""Rows routed to components: the most probable ones of every row (``route``), rows grouped by component (``group_rows``)."""
from ._native import binding

_b = binding()
RowGroups = _b.RowGroups


def route(log_weights, k, renormalise=True):
    """
    The ``k`` most probable components of every row of ``log_weights`` (n, K) and their weights.

    Returns ``(labels, weights)``: int64 (n, k), ordered by (log weight descending, index ascending), and the softmax over
    the chosen components (``renormalise=True``) or over all of them (``False``: the posterior's own shares), float64 for float64
    input and float32 otherwise.  Components at -inf (no members, masked) or NaN are never chosen and have no weight; a row with
    fewer than ``k`` others fills up with label -1, weight 0 -- what ``group_rows`` takes for "no component".
    Weights held in 32 bits that are below their smallest normal number, 2^-126 of the largest, are zero.
    ``weights`` is differentiable with respect to ``log_weights``.  float64 / 32 / 16, bfloat16; k at most 32.
    """
    return _b.route(log_weights, k, renormalise)


def group_rows(labels, n_components):
    """
    Group rows by their component: ``labels`` int64 (n,), one per row, or (n, k), k per row (``route``'s).  A label outside
    0 .. n_components - 1 -- the samplers' -1 -- is a row of no component: products give zeros for it.  The order within a
    component is the rows' own, so that a grouping, and every sum over one, is the same every time.  At most 8000 components.

    Returns a ``RowGroups`` for any number of ``grouped_matmul`` calls: ``labels_shape``, ``n_components``; ``order`` int32, flat
    label indices sorted by (component, index), those of no component last; ``offsets`` int32 (n_components + 2,), component e
    holds ``order[offsets[e]:offsets[e + 1]]``, the last bucket the rows of no component; ``counts``, rows per component.  The
    products read them: they are not for writing.  For products on another stream than the one it was made on, that stream has to
    wait for this one, and ``record_stream(stream)`` keeps the grouping's memory until they are done, as a tensor's does.
    """
    return _b.group_rows(labels, n_components)
