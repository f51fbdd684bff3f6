"""Rows times the matrix of their own component, ragged groups (``grouped_matmul``)."""
from ._native import binding

_b = binding()


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
    return _b.grouped_matmul(x, weight, groups, bias, gates)
