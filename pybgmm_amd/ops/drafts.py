"""Drafted labels verified against exact probabilities from given uniforms (``verify_drafts``)."""
from ._native import binding

_b = binding()


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
    return _b.verify_drafts(target, draft, labels, u_accept, u_draw, lengths)
