"""
Operators on torch tensors around a fitted mixture (or a learned gate): rows routed to components, rows times their own
component's matrix, drafted labels verified against exact probabilities.  Hand-written HIP kernels behind
include/bgmm_ops.h; every call runs on the caller's current stream of the tensors' device, waits for nothing and may be
captured into a graph -- with gradients only if no eager graph of the default stream is behind it (a leaf that one still refers
to, say): its backward pass would end the process, so the call refuses.

    labels, weights = route(log_weights, k)
    groups = group_rows(labels, n_components)
    y = grouped_matmul(x, weight, groups, bias, gates=weights)

    out, accepted = verify_drafts(target, draft, drafted_labels, u_accept, u_draw)
"""
from .drafts import verify_drafts
from .products import grouped_matmul
from .routing import RowGroups, group_rows, route

__all__ = ["route", "group_rows", "RowGroups", "grouped_matmul", "verify_drafts"]
