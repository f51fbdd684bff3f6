"""Drafted labels verified against exact probabilities from given uniforms (``verify_drafts``)."""
import torch

from . import _native as nat


def verify_drafts(target, draft, labels, u_accept, u_draw, lengths=None):
    """
    Accept or reject labels that were drawn from a cheaper model, so that the labels kept are distributed as if every one had
    been drawn from the target, and draw the label behind them.  Like the samplers' sweeps it takes its uniforms as inputs.

    target    (B, T + 1, V) probabilities of the model to follow, the last axis behind T drafts
    draft     (B, T, V) probabilities the drafted labels were drawn from, target's type (float64 / 32 / 16, bfloat16)
    labels    int64 (B, T);  u_accept float64 (B, T) and u_draw float64 (B,) in [0, 1);  lengths int64 (B,): drafts of each
              sequence, 0 .. T (clamped), None: T each

    Draft t is accepted iff ``u_accept * draft < target`` at its label; the first rejection ends the run.  The label behind
    the accepted ones is the first whose cumulative sum exceeds ``u_draw`` times the sum: of ``max(0, target - draft)`` at the
    rejected place (of the target there where that is zero everywhere), or of the target behind the last draft.  Sums and
    comparisons are in 64 bits; rows need not sum to one.  What is not a positive finite number counts as zero, a label
    outside 0 .. V - 1 is rejected, and a row with nothing to draw from gives -1.

    Returns ``(out, accepted)``: int64 (B, T + 1), the accepted labels, the drawn one, -1 behind; int64 (B,).
    """
    what = "verify_drafts"
    given = dict(target=target, draft=draft, labels=labels, u_accept=u_accept, u_draw=u_draw, lengths=lengths)
    nat.require_tensors(what, **given)
    if not (target.dim() == 3 and draft.dim() == 3):
        nat.refuse("%s: target and draft have %d and %d axes, not 3", what, target.dim(), draft.dim())
    B, T, V = draft.shape
    if not (tuple(target.shape) == (B, T + 1, V)):
        nat.refuse("%s: target is %s, draft %s", what, tuple(target.shape), tuple(draft.shape))
    if not (V >= 1):
        nat.refuse("%s: no labels", what)
    if not (target.dtype in nat.DTYPES and draft.dtype == target.dtype):
        nat.refuse("%s: target is %s, draft %s", what, target.dtype, draft.dtype)
    if not (labels.dtype == torch.int64 and tuple(labels.shape) == (B, T)):
        nat.refuse("%s: labels are %s %s", what, labels.dtype, tuple(labels.shape))
    if not (u_accept.dtype == torch.float64 and tuple(u_accept.shape) == (B, T)):
        nat.refuse("%s: u_accept is %s %s", what, u_accept.dtype, tuple(u_accept.shape))
    if not (u_draw.dtype == torch.float64 and tuple(u_draw.shape) == (B,)):
        nat.refuse("%s: u_draw is %s %s", what, u_draw.dtype, tuple(u_draw.shape))
    if not (lengths is None or (lengths.dtype == torch.int64 and tuple(lengths.shape) == (B,))):
        nat.refuse("%s: lengths have to be int64 (%d,)", what, B)
    dev = nat.require_device(what, **given)
    L = nat.load()
    target, draft = _last_contiguous(target), _last_contiguous(draft)
    labels, u_accept, u_draw = labels.contiguous(), u_accept.contiguous(), u_draw.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    out = torch.empty((B, T + 1), dtype=torch.int64, device=dev)
    accepted = torch.empty((B,), dtype=torch.int64, device=dev)
    ws_bytes = L.bgmm_verify_drafts_ws(B, V)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    with nat.on(dev):
        nat.check(L.bgmm_verify_drafts(nat.DTYPES[target.dtype], nat.ptr(target), target.stride(0), target.stride(1), nat.ptr(draft), draft.stride(0),
                                       draft.stride(1), nat.ptr(labels), nat.ptr(u_accept), nat.ptr(u_draw), nat.ptr(lengths), B, T, V,
                                       nat.ptr(out), nat.ptr(accepted), nat.ptr(ws), ws_bytes, nat.stream(dev)))
    return out, accepted


def _last_contiguous(t):
    return t if t.shape[2] == 1 or t.stride(2) == 1 else t.contiguous()
