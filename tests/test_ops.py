"""
The operators of pybgmm_amd.ops against plain implementations in 64 bits (include/bgmm_ops.h).

Tolerances.  A result rounded to a type of precision eps is off by eps / 2 of its value; a sum of m products held in a type
of precision acc is off by at most m acc / 2 (and a few more roundings) of the sum of the products' magnitudes, whatever
its order: `close` takes both, the second from the same sum over magnitudes.
"""
import ctypes
import math
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu
TYPES = [torch.float64, torch.float32, torch.float16, torch.bfloat16]


def acc_of(dt):
    return torch.float64 if dt == torch.float64 else torch.float32


def half_step(dt):
    return torch.finfo(dt).eps / 2


def close(got, want, magnitude, terms, operand=0.0):
    """got (its type's rounding) against want (64 bits); magnitude: the sum of the terms' magnitudes; operand: relative error
    of a single term (operands rounded before the product)."""
    want, magnitude = want.to(got.device), magnitude.to(got.device)
    acc = half_step(acc_of(got.dtype))
    tol = half_step(got.dtype) * want.abs() * (1 + 1e-3) + (acc * (terms + 8) + operand) * magnitude + torch.finfo(got.dtype).tiny
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), "%d of %d off, worst %g over its tolerance" % (
        int(bad.sum()), bad.numel(), float(((got.double() - want).abs() / tol)[bad].max()))


# ------------------------------------------------------------------------------------------ the C-ABI and refusals (CPU)
def test_header_symbols_are_exported_and_bound():
    from pybgmm_amd.ops import _native as nat
    hdr = open(os.path.join(ROOT, "include", "bgmm_ops.h")).read()
    declared = set(re.findall(r"\b(bgmm_[a-z_0-9]+)\s*\(", hdr)) - {"bgmm_create"}
    calls = set(n for n in declared if re.search(r"BGMM_OPS_API [^;]*\b%s\s*\(" % n, hdr))
    assert calls == set(nat.SIGNATURES), calls.symmetric_difference(nat.SIGNATURES)
    L = nat.load()
    for name in calls:
        assert hasattr(L, name)
    for name, value in (("MAX_COMPONENTS", nat.MAX_COMPONENTS), ("MAX_CHOSEN", nat.MAX_CHOSEN), ("LEVELS", nat.LEVELS)):
        assert int(re.search(r"BGMM_OPS_%s\s*=\s*(\d+)" % name, hdr).group(1)) == value


def test_the_operators_bind_to_the_runtime_of_torch():
    from pybgmm_amd import _lib
    from pybgmm_amd.ops import _native as nat
    _lib.load()                                     # (may bring another HIP runtime into the process)
    path = nat.load().bgmm_ops_runtime_path().decode()
    assert os.path.samefile(path, os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so"))


def cpu_groups(shape, K):
    from pybgmm_amd import ops
    P = shape[0] * (shape[1] if len(shape) == 2 else 1)
    return ops.RowGroups(shape, K, torch.zeros(ops.RowGroups.store_size(P, K), dtype=torch.int32))


def refused(code, call, *args, **kw):
    from pybgmm_amd._lib import BGMMError
    with pytest.raises(BGMMError) as ei:
        call(*args, **kw)
    assert ei.value.code == code, ei.value
    return str(ei.value)


def test_refusals_of_route_and_group_rows():
    from pybgmm_amd import ops
    lw = torch.zeros(3, 5)
    pytest.raises(TypeError, ops.route, [1.0], 1)
    refused(-1, ops.route, lw[0], 1)
    refused(-1, ops.route, lw.long(), 1)
    refused(-1, ops.route, lw, 0)
    refused(-1, ops.route, lw, 6)
    pytest.raises(TypeError, ops.route, lw, 1.5)
    refused(-5, ops.route, torch.zeros(2, 64), 33)
    assert "HIP" in refused(-2, ops.route, lw, 2)
    z = torch.zeros(4, dtype=torch.int64)
    refused(-1, ops.group_rows, z.int(), 3)
    refused(-1, ops.group_rows, z.view(1, 2, 2), 3)
    refused(-1, ops.group_rows, torch.zeros(2, 33, dtype=torch.int64), 3)
    refused(-1, ops.group_rows, torch.zeros(2, 0, dtype=torch.int64), 3)
    refused(-1, ops.group_rows, z, 0)
    refused(-5, ops.group_rows, z, 8001)
    refused(-2, ops.group_rows, z, 3)


def test_refusals_of_grouped_matmul():
    from pybgmm_amd import ops
    g1, g2 = cpu_groups((4,), 3), cpu_groups((4, 2), 3)
    x, w, b = torch.zeros(4, 6), torch.zeros(3, 6, 5), torch.zeros(3, 5)
    mm = ops.grouped_matmul
    pytest.raises(TypeError, mm, x, w, None)
    refused(-1, ops.RowGroups, (4,), 3, torch.zeros(3, dtype=torch.int32))
    refused(-1, mm, x.long(), w.long(), g1)
    refused(-1, mm, x, w.double(), g1)
    refused(-1, mm, x, w, g1, bias=b.double())
    refused(-1, mm, x, w[:2], g1)
    refused(-1, mm, x, w[0], g1)
    refused(-1, mm, x[:3], w, g1)
    refused(-1, mm, x[:, :5], w, g1)
    refused(-1, mm, torch.zeros(4, 2, 6), w, g1)                # a row per label needs a grouping of (n, k) labels
    refused(-1, mm, torch.zeros(4, 3, 6), w, g2)
    refused(-1, mm, x, w, g1, bias=b[:, :4])
    refused(-1, mm, x, w, g1, gates=torch.zeros(4, 1))
    refused(-1, mm, x, w, g2, gates=torch.zeros(4))
    refused(-1, mm, x, w, g1, gates=torch.zeros(4).double())
    refused(-1, mm, x.bfloat16(), w.bfloat16(), g1, gates=torch.zeros(4).bfloat16())
    refused(-1, mm, x, torch.zeros(3, 6, 0), g1)
    refused(-2, mm, x, w, g1, bias=b, gates=torch.zeros(4))


def test_refusals_of_verify_drafts():
    from pybgmm_amd import ops
    v = ops.verify_drafts
    p, q, z = torch.zeros(2, 4, 5), torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64)
    ua, ud = torch.zeros(2, 3, dtype=torch.float64), torch.zeros(2, dtype=torch.float64)
    refused(-1, v, p[0], q, z, ua, ud)
    refused(-1, v, p[:, :3], q, z, ua, ud)
    refused(-1, v, p[..., :4], q, z, ua, ud)
    refused(-1, v, p.double(), q, z, ua, ud)
    refused(-1, v, p.long(), q.long(), z, ua, ud)
    refused(-1, v, p, q, z.int(), ua, ud)
    refused(-1, v, p, q, z[:, :2], ua, ud)
    refused(-1, v, p, q, z, ua.float(), ud)
    refused(-1, v, p, q, z, ua, ud[:1])
    refused(-1, v, p, q, z, ua, ud, lengths=torch.zeros(2, dtype=torch.int32))
    refused(-1, v, p[..., :0], q[..., :0], z, ua, ud)
    refused(-2, v, p, q, z, ua, ud)


def test_c_entry_points_refuse_before_they_launch():
    """Sizes, types, null pointers: negative codes with a message, no launch (this runs without a device)."""
    from pybgmm_amd.ops import _native as nat
    L = nat.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)
    calls = [
        (-1, L.bgmm_group_rows(p, -1, 3, p, p, p, p, p, p, 0, None)),
        (-1, L.bgmm_group_rows(p, 1 << 31, 3, p, p, p, p, p, p, 0, None)),
        (-1, L.bgmm_group_rows(p, 5, 0, p, p, p, p, p, p, 0, None)),
        (-5, L.bgmm_group_rows(p, 5, 8001, p, p, p, p, p, p, 0, None)),
        (-1, L.bgmm_group_rows(None, 5, 3, p, p, p, p, p, p, 0, None)),
        (-1, L.bgmm_group_rows(p, 100000, 3, p, p, p, p, p, p, 8, None)),
        (-1, L.bgmm_route(9, p, 4, 2, 4, 1, 1, p, p, None, None)),
        (-1, L.bgmm_route(1, p, 4, 2, 4, 5, 1, p, p, None, None)),
        (-5, L.bgmm_route(1, p, 64, 2, 64, 33, 1, p, p, None, None)),
        (-1, L.bgmm_route(1, None, 4, 2, 4, 1, 1, p, p, None, None)),
        (-1, L.bgmm_route_backward(1, p, 4, 2, 4, 1, 0, p, p, None, p, p, None)),
        (-1, L.bgmm_verify_drafts(1, p, 4, 4, p, 4, 4, p, p, p, None, 1, -1, 4, p, p, None, 0, None)),
        (-1, L.bgmm_verify_drafts(1, p, 4, 4, None, 4, 4, p, p, p, None, 1, 1, 4, p, p, None, 0, None)),
        (-1, L.bgmm_verify_drafts(1, p, 4, 4, p, 4, 4, p, p, p, None, 1, 1, 0, p, p, None, 0, None)),
        (-1, L.bgmm_verify_drafts(1, p, 4, 4, p, 4, 4, p, p, p, None, 1, 1, 5000, p, p, p, 8, None)),                 # workspace
        (-1, L.bgmm_rows_product(1, p, 4, 1, p, 4, 4, 0, None, 0, None, p, 4, p, 1, None, 0, 1, None, 8, 2, 4, 4, p, p, None)),     # out and ws
        (-1, L.bgmm_rows_product(1, p, 4, 1, p, 4, 4, 0, None, 0, None, p, 4, None, 2, None, 0, 1, None, 8, 2, 4, 4, p, p, None)),  # splits without ws
        (-1, L.bgmm_rows_product(1, p, 4, 0, p, 4, 4, 0, None, 0, None, p, 4, None, 1, None, 0, 1, None, 8, 2, 4, 4, p, p, None)),
        (-1, L.bgmm_rows_product(4, p, 4, 1, p, 4, 4, 0, None, 0, None, p, 4, None, 1, None, 0, 1, None, 8, 2, 4, 4, p, p, None)),
        (-1, L.bgmm_weight_product(1, p, 4, 1, p, 4, 1, None, p, None, None, 0, 1 << 20, 2, 4, 4, p, p, p, None)),   # workspace
        (-1, L.bgmm_weight_product(1, None, 4, 1, p, 4, 1, None, p, None, None, 0, 8, 2, 4, 4, p, p, p, None)),
        (-1, L.bgmm_rows_product(1, p, 4, 1, p, 4, 4, 0, None, 0, None, None, 4, None, 1, None, 0, 1, None, 8, 2, 4, 4, p, p, None)),   # no result
        (-1, L.bgmm_rows_product(1, p, 4, 1, p, 4, 4, 0, None, 0, None, None, 4, None, 1, None, 4, 1, p, 8, 2, 4, 4, p, p, None)),      # dots without rows
        (-1, L.bgmm_rows_product(1, p, 4, 1, p, 4, 4, 0, None, 0, None, None, 4, None, 1, p, 4, 0, p, 8, 2, 4, 4, p, p, None)),
        (-1, L.bgmm_combine(1, p, 1, 4, 33, 2, p, None, p, 4, 4, None, None, 0, None, 0, None, 0, 1, 1, None)),
        (-1, L.bgmm_combine(1, p, 1, 4, 1, 2, p, None, p, 4, 4, p, p, 4, None, 0, None, 0, 1, 1, None)),             # dgates without gates
        (-1, L.bgmm_gate_gradient(1, p, 0, 4, 2, p, None, 0, None, 0, 1, 1, p, None)),
        (-1, L.bgmm_gate_gradient(1, p, 2, 4, 2, p, p, 4, None, 0, 1, 4, p, None)),                                   # a bias without d
        (-1, L.bgmm_gate_gradient(5, p, 2, 4, 2, p, None, 0, None, 0, 1, 1, p, None)),
    ]
    for i, (want, got) in enumerate(calls):
        assert got == want, (i, got)
    assert L.bgmm_ops_last_error()


# ------------------------------------------------------------------------------------------ route
def route_ref(lw, k, renormalise):
    """Labels and weights in 64 bits, one row at a time."""
    n, K = lw.shape
    labels, weights = torch.full((n, k), -1, dtype=torch.int64), torch.zeros(n, k, dtype=torch.float64)
    for i in range(n):
        row = lw[i].double().tolist()
        at = sorted((j for j in range(K) if row[j] > -math.inf), key=lambda j: (-row[j], j))
        if not at:
            continue
        top = row[at[0]]

        def ratio(v):
            return 1.0 if v == top else math.exp(v - top)
        total = math.fsum(ratio(row[j]) for j in (at[:k] if renormalise else at))
        for c, j in enumerate(at[:k]):
            labels[i, c], weights[i, c] = j, ratio(row[j]) / total
    return labels, weights


def route_grad_ref(lw, labels, weights, dw, renormalise):
    n, K = lw.shape
    d = torch.zeros(n, K, dtype=torch.float64)
    for i in range(n):
        on = [(c, int(j)) for c, j in enumerate(labels[i]) if j >= 0]
        s = math.fsum(float(weights[i, c] * dw[i, c]) for c, _ in on)
        if not renormalise and on:
            row = lw[i].double()
            row = torch.where(torch.isnan(row), torch.tensor(-math.inf, dtype=torch.float64), row)
            p = torch.where(row == row.max(), torch.ones(K, dtype=torch.float64), torch.exp(row - row.max()))
            d[i] = -s * p / p.sum()
        for c, j in on:
            d[i, j] += float(weights[i, c]) * (float(dw[i, c]) - (s if renormalise else 0.0))
    return d


def route_rows(n, K, dt, seed):
    g = torch.Generator().manual_seed(seed)
    lw = torch.randn(n, K, generator=g, dtype=torch.float64) * 4
    lw[torch.rand(n, K, generator=g) < 0.1] = -math.inf
    lw[torch.rand(n, K, generator=g) < 0.02] = math.nan
    lw[torch.rand(n, K, generator=g) < 0.2] = 0.5                     # ties
    if n > 4:
        lw[0] = -math.inf                                             # nothing to choose
        lw[1] = torch.finfo(dt).min                                   # a mask of the type's lowest value is a value like others
        lw[2, : max(1, K // 2)] = -math.inf
        lw[3] = math.nan
        lw[4, K - 1] = math.inf
    return lw.to(dt)


@gpu
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,K,k", [(1, 1, 1), (1, 200, 4), (7, 2, 2), (33, 64, 6), (65, 100, 1), (20, 129, 8), (9, 1000, 32), (5, 5000, 3), (300, 17, 17),
                                   (3, 1025, 32), (5, 4096, 8), (4, 4097, 3), (2, 16384, 32), (3, 16385, 5), (2, 40001, 2)])
@pytest.mark.parametrize("renormalise", [True, False])
def test_route_forward_and_backward(dt, n, K, k, renormalise):
    from pybgmm_amd import ops
    lw = route_rows(n, K, dt, 1000 * n + K)
    x = lw.cuda().requires_grad_()
    labels, w = ops.route(x, k, renormalise=renormalise)
    want_l, want_w = route_ref(lw, k, renormalise)
    assert torch.equal(labels.cpu(), want_l)
    # exp is off by about an ulp of its value, the difference in its argument by half a step of |l_j - m| <= 40 at most
    acc = half_step(acc_of(dt))
    tol = acc * (K + 100) * want_w + 1e-30
    assert w.dtype == acc_of(dt) and bool(((w.cpu().double() - want_w).abs() <= tol).all())
    with torch.no_grad():
        l2, w2 = ops.route(x, k, renormalise=renormalise)
    assert torch.equal(l2, labels) and torch.equal(w2, w)
    dw = torch.randn(n, k, generator=torch.Generator().manual_seed(n), dtype=acc_of(dt))
    got, = torch.autograd.grad(w, x, dw.cuda())
    want = route_grad_ref(lw, want_l, want_w, dw, renormalise)
    assert got.dtype == dt
    scale = (want_w * dw.double()).abs().sum(1, keepdim=True)
    tol = half_step(dt) * want.abs() * 1.001 + acc * (K + 200) * scale + torch.finfo(dt).tiny
    assert bool(((got.cpu().double() - want).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("dt,bits,i", [(torch.float64, 0x7FF0000000000001, torch.int64), (torch.float32, 0x7F800001, torch.int32),
                                       (torch.float16, 0x7C01, torch.int16), (torch.bfloat16, 0x7F81, torch.int16)], ids=str)
def test_route_never_chooses_a_signalling_nan(dt, bits, i):
    from pybgmm_amd import ops
    raw = torch.linspace(-3, 2, 40, device="cuda").to(dt).repeat(5, 1)
    raw.view(i)[:, 1::2] = bits
    assert torch.isnan(raw[:, 1::2]).all()
    labels, w = ops.route(raw, 3, renormalise=False)
    assert labels.tolist() == [[38, 36, 34]] * 5
    row = raw[0].cpu().double()
    soft = torch.softmax(torch.where(torch.isnan(row), -math.inf, row), 0)[[38, 36, 34]]
    assert torch.allclose(w.cpu().double(), soft.expand(5, 3), rtol=1e-5, atol=0)


@gpu
def test_route_rows_with_strides_and_no_rows():
    from pybgmm_amd import ops
    lw = route_rows(40, 96, torch.float32, 3).cuda()
    for view in (lw[::2], lw[:, :50], lw.t().contiguous().t(), lw[5:6], lw[:, 3:80][::3]):
        got, want = ops.route(view, 3), ops.route(view.contiguous(), 3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        x, y = view.detach().requires_grad_(), view.contiguous().requires_grad_()
        ga = torch.autograd.grad(ops.route(x, 3, renormalise=False)[1].sum(1).square().sum(), x)[0]
        gb = torch.autograd.grad(ops.route(y, 3, renormalise=False)[1].sum(1).square().sum(), y)[0]
        assert torch.equal(ga, gb)
    labels, w = ops.route(lw[:0], 2)
    assert labels.shape == (0, 2) and w.shape == (0, 2)


@gpu
def test_route_gradient_against_differences():
    from pybgmm_amd import ops
    x = torch.randn(6, 11, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).requires_grad_()
    for renormalise in (True, False):
        assert torch.autograd.gradcheck(lambda t: ops.route(t, 3, renormalise=renormalise)[1], (x,), eps=1e-6, atol=1e-8, rtol=1e-5)


# ------------------------------------------------------------------------------------------ group_rows
@gpu
@pytest.mark.parametrize("shape,K", [((0,), 3), ((0,), 2000), ((1,), 1), ((5,), 8000), ((64,), 7), ((1000, 4), 64), ((8192,), 889), ((8192,), 890), ((1024,), 50), ((1025,), 50),
                                     ((8193,), 3), ((40000,), 200), ((30011, 3), 1779), ((30011,), 1780), ((30011, 3), 3199), ((30011,), 3200), ((100003,), 8000), ((1000000,), 100),
                                     ((4096,), 64), ((4097,), 64), ((513, 7), 20), ((4096,), 1479), ((2048,), 1480), ((2049,), 1480), ((2048,), 2299), ((300, 2), 2300), ((6000,), 2)])
def test_group_rows(shape, K):
    from pybgmm_amd import ops
    g = torch.Generator().manual_seed(K + len(shape))
    z = torch.randint(-1, K, shape, generator=g)
    if z.numel() > 3:
        z.view(-1)[1], z.view(-1)[2] = K, -(1 << 40)              # outside: no component
        z.view(-1)[3] = 1 << 33
    grp = ops.group_rows(z.cuda(), K)
    flat = z.view(-1)
    bucket = torch.where((flat >= 0) & (flat < K), flat, torch.tensor(K))
    assert torch.equal(grp.bucket.cpu().long(), bucket)
    assert torch.equal(grp.order.cpu().long(), torch.argsort(bucket, stable=True))
    size = torch.bincount(bucket, minlength=K + 1)
    off = torch.cat([torch.zeros(1, dtype=torch.int64), size.cumsum(0)])
    assert torch.equal(grp.offsets.cpu().long(), off)
    assert torch.equal(grp.counts.cpu().long(), size[:K])
    assert grp.labels_shape == shape and grp.n_components == K
    first = grp.first.view(8, K + 2).cpu().long()
    for level in range(8):
        tiles = (size + (256 << level) - 1) // (256 << level)
        assert torch.equal(first[level], torch.cat([torch.zeros(1, dtype=torch.int64), tiles.cumsum(0)])), level
    rows = 16 if z.numel() <= 16 * K else 128
    want = [[b, int(off[b]) + r, min(rows, int(size[b]) - r), 0] for b in range(K + 1) for r in range(0, int(size[b]), rows)]
    got = grp.tiles.view(-1, 4).cpu()
    assert got[:len(want)].tolist() == want and bool((got[len(want):, 0] == -1).all())


@gpu
def test_group_rows_one_component_has_all_and_non_contiguous_labels():
    from pybgmm_amd import ops
    z = torch.full((50000,), 5, device="cuda")
    grp = ops.group_rows(z, 9)
    assert torch.equal(grp.order.long(), torch.arange(50000, device="cuda")) and grp.counts.tolist() == [0] * 5 + [50000] + [0] * 3
    z = torch.randint(0, 9, (100, 6), device="cuda")[:, ::2]
    assert torch.equal(ops.group_rows(z, 9).order, ops.group_rows(z.contiguous(), 9).order)


# ------------------------------------------------------------------------------------------ grouped_matmul
def products_ref(x, w, z, bias, gates, dy=None):
    """Everything in 64 bits on x's device, with the sums over magnitudes next to every result."""
    K, din, dout = w.shape
    n, k = z.shape
    per = x.dim() == 3
    X, W = x.double(), w.double()
    pair, mag = [torch.zeros(n, k, dout, dtype=torch.float64, device=x.device) for _ in range(2)]
    out = {}
    if dy is not None:
        dpair, dmag = [torch.zeros(n, k, din, dtype=torch.float64, device=x.device) for _ in range(2)]
        dw, dwm = torch.zeros_like(W), torch.zeros_like(W)
        db, dbm = [torch.zeros(K, dout, dtype=torch.float64, device=x.device) for _ in range(2)]
        dg, dgm = [torch.zeros(n, k, dtype=torch.float64, device=x.device) for _ in range(2)]
    for e in range(K):
        i, j = torch.nonzero(z == e, as_tuple=True)
        if i.numel() == 0:
            continue
        xe = X[i, j] if per else X[i]
        be = bias[e].double() if bias is not None else torch.zeros(dout, dtype=torch.float64, device=x.device)
        u, um = xe @ W[e] + be, xe.abs() @ W[e].abs() + be.abs()
        ge = gates.double().view(n, k)[i, j][:, None] if gates is not None else torch.ones(i.numel(), 1, dtype=torch.float64, device=x.device)
        pair[i, j], mag[i, j] = ge * u, ge.abs() * um
        if dy is not None:
            d = dy.double().view(n, k, dout)[i, j] if gates is None else dy.double()[i]
            wt = W[e].t().contiguous()
            v, vm = d @ wt, d.abs() @ wt.abs()
            dpair[i, j], dmag[i, j] = ge * v, ge.abs() * vm
            dw[e], dwm[e] = xe.t().contiguous() @ (ge * d), xe.abs().t().contiguous() @ (ge * d).abs()
            db[e], dbm[e] = (ge * d).sum(0), (ge * d).abs().sum(0)
            dg[i, j] = (xe * v).sum(1) + (d * be).sum(1)
            dgm[i, j] = (xe.abs() * vm).sum(1) + (d * be).abs().sum(1)
    summed = gates is not None
    out["y"] = (pair.sum(1), mag.sum(1)) if summed else (pair, mag)
    if dy is not None:
        out["x"] = (dpair, dmag) if per else (dpair.sum(1), dmag.sum(1))
        out["w"], out["b"], out["g"] = (dw, dwm), (db, dbm), (dg, dgm)
    return out


def product_case(n, k, K, din, dout, dt, seed, flat=False, per_label=False, bias=True, gates=True):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda", dtype=torch.float64).to(dt)
    share = torch.rand(K, generator=g, device="cuda") ** 3 + 1e-3
    z = torch.multinomial(share, max(n, 1) * k, replacement=True, generator=g).view(-1, k)[:n]
    z[torch.rand(n, k, generator=g, device="cuda") < 0.05] = -1
    if n > 2:
        z[1] = -1                                                    # a row of no component at all
    x = randn(n, k, din) if per_label else randn(n, din)
    if n > 2:
        x[1] = math.nan                                              # ... whose contents nobody reads
    w = randn(K, din, dout)
    b = randn(K, dout) if bias else None
    gt = None
    if gates:
        gt = torch.rand(n, k, generator=g, device="cuda", dtype=acc_of(dt)) + 0.1
        if n > 2:
            gt[1] = math.nan
        if flat:
            gt = gt[:, 0]
    return (z[:, 0] if flat else z).contiguous(), x, w, b, gt, g


CASES = [
    # n, k, K, din, dout
    (1, 1, 1, 1, 1), (1, 4, 64, 256, 128), (3, 2, 5, 64, 64), (1, 2, 3, 2048, 40), (17, 1, 40, 96, 200), (130, 1, 3, 64, 64),
    (257, 2, 4, 130, 66), (1000, 1, 7, 16, 16), (999, 3, 6, 33, 5), (700, 1, 2, 128, 300), (2050, 1, 20, 192, 77), (5000, 2, 9, 72, 136),
    (4000, 1, 1, 20, 16), (64, 8, 16, 513, 129), (300, 1, 2, 65, 1), (300, 1, 2, 1, 65), (2000, 1, 3, 129, 3),
    (3000, 1, 5, 8, 16), (2500, 2, 4, 16, 31), (900, 1, 60, 2, 2), (1500, 1, 3, 32, 9), (1, 1, 1, 16, 16),
    (1100, 1, 4, 17, 32), (1300, 2, 5, 32, 17), (800, 1, 3, 29, 23), (600, 1, 2, 300, 24), (900, 2, 4, 31, 1),
    (70000, 1, 30, 150, 12), (70000, 1, 30, 12, 150), (40000, 2, 9, 140, 40), (70000, 1, 30, 40, 140), (5000, 1, 4, 16, 60), (5000, 1, 4, 60, 16),
]


@gpu
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("form", ["plain", "gated", "per_label", "per_label_gated"])
def test_grouped_matmul_forward_and_backward(dt, case, form):
    from pybgmm_amd import ops
    n, k, K, din, dout = case
    gated, per_label = "gated" in form, "per_label" in form
    flat = k == 1 and not per_label
    z, x, w, b, gt, g = product_case(n, k, K, din, dout, dt, sum(case), flat=flat, per_label=per_label, bias=form != "per_label", gates=gated)
    groups = ops.group_rows(z, K)
    leaves = [t.requires_grad_() for t in (x, w, b, gt) if t is not None]
    y = ops.grouped_matmul(x, w, groups, bias=b, gates=gt)
    assert y.dtype == dt and tuple(y.shape) == ((n, dout) if gated or flat else (n, k, dout))
    with torch.no_grad():
        assert torch.equal(ops.grouped_matmul(x, w, groups, bias=b, gates=gt), y)
    dy = torch.randn(y.shape, generator=g, device="cuda", dtype=torch.float64).to(dt)
    grads = torch.autograd.grad(y, leaves, dy)
    again = torch.autograd.grad(ops.grouped_matmul(x, w, groups, bias=b, gates=gt), leaves, dy)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))
    names = ["x", "w"] + (["b"] if b is not None else []) + (["g"] if gated else [])
    ref = products_ref(x.detach(), w.detach(), z.view(n, k), None if b is None else b.detach(), None if gt is None else gt.detach(), dy)
    close(y.detach(), ref["y"][0].view(y.shape), ref["y"][1].view(y.shape), din + k + 16)
    rows = int((z.view(-1) >= 0).sum())
    for name, got in zip(names, grads):
        want, mag = (t.view(got.shape) for t in ref[name])
        terms = {"x": dout + k, "w": rows, "b": rows, "g": din + 2 * dout}[name] + 16
        # (16-bit types: a gated row of dy is rounded to the operands' type before the weights' gradient sums its products)
        close(got, want, mag, terms, operand=half_step(dt) * 1.001 if name == "w" and gated and dt.itemsize == 2 else 0.0)


@gpu
@pytest.mark.parametrize("dt", [torch.float64, torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,K,din,dout", [(40000, 2, 64, 64), (70000, 3, 16, 16), (35000, 1, 136, 40)])
def test_long_groups_are_split_and_joined(dt, rows, K, din, dout):
    from pybgmm_amd import ops
    z, x, w, b, _, g = product_case(rows, 1, K, din, dout, dt, rows, flat=True, gates=False)
    groups = ops.group_rows(z, K)
    for t in (x, w, b):
        t.requires_grad_()
    y = ops.grouped_matmul(x, w, groups, bias=b)
    dy = torch.randn(y.shape, generator=g, device="cuda", dtype=torch.float64).to(dt)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ref = products_ref(x.detach(), w.detach(), z.view(-1, 1), b.detach(), None, dy)
    close(y.detach(), ref["y"][0][:, 0], ref["y"][1][:, 0], din + 16)
    close(dx, ref["x"][0], ref["x"][1], dout + 16)
    close(dw, *ref["w"], rows)
    close(db, *ref["b"], rows)


@gpu
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,k,K,din,dout", [(40000, 1, 20, 2, 2), (35001, 1, 30, 8, 5), (33000, 1, 12, 7, 8), (20000, 2, 9, 3, 4), (40000, 1, 1, 1, 1)])
@pytest.mark.parametrize("gated", [False, True])
def test_many_thin_rows(dt, n, k, K, din, dout, gated):
    from pybgmm_amd import ops
    z, x, w, b, gt, g = product_case(n, k, K, din, dout, dt, n + din, flat=k == 1, gates=gated)
    groups = ops.group_rows(z, K)
    leaves = [t.requires_grad_() for t in (x, w, b, gt) if t is not None]
    y = ops.grouped_matmul(x, w, groups, bias=b, gates=gt)
    dy = torch.randn(y.shape, generator=g, device="cuda", dtype=torch.float64).to(dt)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = products_ref(x.detach(), w.detach(), z.view(n, k), b.detach(), None if gt is None else gt.detach(), dy)
    close(y.detach(), ref["y"][0].view(y.shape), ref["y"][1].view(y.shape), din + k + 16)
    for name, got in zip("xwbg", grads):
        want, mag = (t.view(got.shape) for t in ref[name])
        close(got, want, mag, {"x": dout + k, "w": n * k, "b": n * k, "g": din + 2 * dout}[name] + 16,
              operand=half_step(dt) * 1.001 if name == "w" and gated and dt.itemsize == 2 else 0.0)


@gpu
@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_strides_alignment_and_transposed_weights(dt):
    from pybgmm_amd import ops
    n, K, din, dout = 300, 4, 72, 56
    z, x, w, b, _, g = product_case(n, 1, K, din, dout, dt, 11, flat=True, gates=False)
    groups = ops.group_rows(z, K)
    want = ops.grouped_matmul(x, w, groups, bias=b)
    wide = torch.zeros(n, din + 5, device="cuda", dtype=dt)
    wide[:, 3:3 + din] = x
    odd = torch.zeros(K * din * dout + 1, device="cuda", dtype=dt)
    odd[1:] = w.reshape(-1)
    views = {
        "x inside wider rows": (wide[:, 3:3 + din], w, b),
        "x by columns": (x.t().contiguous().t(), w, b),
        "weights by output": (x, w.transpose(1, 2).contiguous().transpose(1, 2), b),
        "weights off alignment": (x, odd[1:].view(K, din, dout), b),
        "weights by component last": (x, w.permute(1, 2, 0).contiguous().permute(2, 0, 1), b),
        "bias broadcast from one row": (x, w, b[:1].expand(K, dout)),
    }
    for name, (xv, wv, bv) in views.items():
        ref = want if "bias" not in name else ops.grouped_matmul(x, w, groups, bias=bv.contiguous())
        got = ops.grouped_matmul(xv, wv, groups, bias=bv)
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(ref)), name
    # gradients of the views arrive in the leaves' own shape
    leaf = w.transpose(1, 2).contiguous().requires_grad_()
    wl = w.clone().requires_grad_()
    xs = x.clone().requires_grad_()
    dy = torch.randn(n, dout, generator=g, device="cuda", dtype=torch.float64).to(dt)
    ga = torch.autograd.grad(ops.grouped_matmul(xs, leaf.transpose(1, 2), groups), (xs, leaf), dy)
    gb = torch.autograd.grad(ops.grouped_matmul(xs, wl, groups), (xs, wl), dy)
    assert torch.equal(ga[0], gb[0]) and torch.equal(ga[1].transpose(1, 2), gb[1])
    one = torch.ones(1, device="cuda", dtype=dt).expand(n, dout)                 # a gradient broadcast from one number
    gc = torch.autograd.grad(ops.grouped_matmul(xs, wl, groups), (xs, wl), one)
    gd = torch.autograd.grad(ops.grouped_matmul(xs, wl, groups), (xs, wl), one.contiguous())
    assert all(torch.equal(a, c) for a, c in zip(gc, gd))


@gpu
def test_grouped_matmul_without_rows_and_components_without_rows():
    from pybgmm_amd import ops
    w, b = torch.randn(5, 8, 6, device="cuda", requires_grad=True), torch.randn(5, 6, device="cuda", requires_grad=True)
    x = torch.randn(0, 8, device="cuda", requires_grad=True)
    y = ops.grouped_matmul(x, w, ops.group_rows(torch.zeros(0, dtype=torch.int64, device="cuda"), 5), bias=b)
    assert y.shape == (0, 6)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert dx.shape == (0, 8) and not dw.any() and not db.any()
    x = torch.randn(7, 8, device="cuda", requires_grad=True)
    y = ops.grouped_matmul(x, w, ops.group_rows(torch.full((7,), -1, device="cuda"), 5), bias=b)
    assert not y.any()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.full_like(y, math.nan))
    assert not dx.any() and not dw.any() and not db.any()
    y = ops.grouped_matmul(x, w, ops.group_rows(torch.tensor([3] * 7, device="cuda"), 5), bias=b)
    dw, = torch.autograd.grad(y, (w,), torch.ones_like(y))
    assert dw[3].any() and not dw[[0, 1, 2, 4]].any()


@gpu
def test_grouped_matmul_gradients_against_differences():
    from pybgmm_amd import ops
    z, x, w, b, gt, _ = product_case(5, 2, 3, 4, 3, torch.float64, 2)
    x = torch.nan_to_num(x).requires_grad_()
    gt = torch.nan_to_num(gt).requires_grad_()
    w.requires_grad_()
    b.requires_grad_()
    groups = ops.group_rows(z, 3)
    assert torch.autograd.gradcheck(lambda x, w, b, g: ops.grouped_matmul(x, w, groups, bias=b, gates=g), (x, w, b, gt), eps=1e-6, atol=1e-7)
    assert torch.autograd.gradcheck(lambda x, w, b: ops.grouped_matmul(x, w, groups, bias=b), (x, w, b), eps=1e-6, atol=1e-7)


@gpu
def test_some_gradients_only():
    from pybgmm_amd import ops
    z, x, w, b, gt, g = product_case(200, 2, 5, 40, 24, torch.float32, 8)
    groups = ops.group_rows(z, 5)
    full = [t.clone().requires_grad_() for t in (x, w, b, gt)]
    dy = torch.randn(200, 24, device="cuda", generator=g)
    want = torch.autograd.grad(ops.grouped_matmul(full[0], full[1], groups, bias=full[2], gates=full[3]), full, dy)
    for i in range(4):
        leaf = (x, w, b, gt)[i].clone().requires_grad_()
        args = [leaf if j == i else (x, w, b, gt)[j] for j in range(4)]
        got, = torch.autograd.grad(ops.grouped_matmul(args[0], args[1], groups, bias=args[2], gates=args[3]), leaf, dy)
        assert torch.equal(got, want[i]), i


# ------------------------------------------------------------------------------------------ verify_drafts
def verify_ref(p, q, z, ua, ud, lengths):
    """One sequence at a time in exact rational arithmetic (the inputs are floats: every sum below is exact)."""
    from fractions import Fraction

    def clean(v):
        return Fraction(v) if v > 0 and v < math.inf else Fraction(0)
    B, T, V = q.shape
    out, acc = torch.full((B, T + 1), -1, dtype=torch.int64), torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        length, a = min(max(int(lengths[b]), 0), T), 0
        while a < length:
            j = int(z[b, a])
            # (the product of the comparison is rounded to 64 bits, as stated)
            if not (0 <= j < V and float(ua[b, a]) * float(clean(float(q[b, a, j]))) < float(clean(float(p[b, a, j])))):
                break
            out[b, a] = j
            a += 1
        acc[b] = a
        row = [clean(float(v)) for v in p[b, a].double()]
        w = row
        if a < length:
            w = [max(x - clean(float(y)), Fraction(0)) for x, y in zip(row, q[b, a].double())]
            if not any(w):
                w = row
        total, at = sum(w), Fraction(0)
        goal = Fraction(float(ud[b])) * total
        for j in range(V):
            at += w[j]
            if w[j] > 0 and at > goal:
                out[b, a] = j
                break
    return out, acc


def verify_case(B, T, V, dt, seed, spread=0.6):
    g = torch.Generator().manual_seed(seed)
    lp = torch.randn(B, T + 1, V, generator=g, dtype=torch.float64) * 2
    lq = lp[:, :T] + torch.randn(B, T, V, generator=g, dtype=torch.float64) * spread
    p, q = torch.softmax(lp, -1).to(dt), torch.softmax(lq, -1).to(dt)
    z = torch.multinomial(torch.softmax(lq, -1).view(B * T, V), 1, generator=g).view(B, T) if B * T else torch.zeros(B, T, dtype=torch.int64)
    ua, ud = torch.rand(B, T, generator=g, dtype=torch.float64), torch.rand(B, generator=g, dtype=torch.float64)
    lengths = torch.randint(-1, T + 2, (B,), generator=g)
    return p, q, z, ua, ud, lengths


def verify_on_gpu(*args):
    from pybgmm_amd import ops
    out, acc = ops.verify_drafts(*(t.cuda() for t in args[:5]), lengths=args[5].cuda())
    return out.cpu(), acc.cpu()


@gpu
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (1, 0, 7), (3, 4, 2), (50, 8, 20), (40, 3, 200), (5, 70, 33), (9, 2, 256), (7, 2, 999), (6, 2, 1025), (4, 5, 5003), (2, 3, 20000), (1, 1, 70001), (3, 2, 65536), (3, 2, 65537), (130, 1, 3001), (513, 1, 1100), (9, 3, 129), (9, 3, 257), (9, 2, 511), (9, 2, 513), (5, 2, 2048), (5, 2, 2049)])
def test_verify_drafts(dt, B, T, V):
    args = verify_case(B, T, V, dt, B * V + T)
    want = verify_ref(*args)
    got = verify_on_gpu(*args)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0], want[0])


@gpu
def test_verify_drafts_without_lengths_strides_and_no_sequences():
    from pybgmm_amd import ops
    p, q, z, ua, ud, _ = verify_case(12, 4, 50, torch.float32, 5)
    want = verify_ref(p, q, z, ua, ud, torch.full((12,), 4))
    dev = [t.cuda() for t in (p, q, z, ua, ud)]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(ops.verify_drafts(*dev), want))
    pv = torch.zeros(5, 12, 64, device="cuda")
    pv[..., 7:57] = dev[0].transpose(0, 1)
    qv = dev[1].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(ops.verify_drafts(pv.transpose(0, 1)[..., 7:57], qv, *dev[2:]), want))
    out, acc = ops.verify_drafts(*(t[:0] for t in dev))
    assert out.shape == (0, 5) and acc.shape == (0,)


@gpu
@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_verify_drafts_at_the_edges(dt):
    """Values next to a border, rows without weight, labels outside: everything here is exact in every type."""
    V = 8
    one = torch.zeros(V, dtype=dt)
    one[3] = 1
    half = torch.zeros(V, dtype=dt)
    half[2], half[5] = 0.5, 0.5
    none = torch.zeros(V, dtype=dt)
    bad = torch.tensor([math.nan, -1, math.inf, 0, 0.25, math.nan, 0.25, -math.inf], dtype=dt)
    rows = [
        # p at the draft, p behind, q, label, u_accept, u_draw
        (half, one, half, 2, 0.999, 0.0),        # p = q: always accepted; the draw from p behind
        (half, one, one, 3, 0.0, 0.0),           # p = 0 at the label, q > 0, u = 0: 0 < 0 is false
        (half, one, none, 2, 0.9, 0.3),          # q = 0 at the label: accepted
        (none, one, none, 2, 0.0, 0.5),          # p = q = 0: rejected, nothing to draw from
        (half, one, half, 9, 0.0, 0.49999),      # a label outside: rejected, p - q = 0 everywhere: the draw from p
        (half, one, half, -1, 0.0, 0.5),         # ... on the border: the cumulative sum has to EXCEED u * total
        (half, one, one, 3, 0.5, 0.0),           # u = 0: the first label with any weight
        (half, one, one, 3, 0.5, 1 - 2.0 ** -53),
        (bad, one, half, 4, 0.999, 0.0),         # q = 0 there
        (bad, one, half, 2, 0.1, 0.75),          # p infinite there: counts as zero; the draw from what is finite and positive
        (half, bad, half, 5, 0.2, 0.5),
        (half, none, half, 5, 0.2, 0.5),
    ]
    p = torch.stack([torch.stack([r[0], r[1]]) for r in rows])
    q = torch.stack([r[2][None] for r in rows])
    z = torch.tensor([[r[3]] for r in rows])
    ua, ud = torch.tensor([[r[4]] for r in rows], dtype=torch.float64), torch.tensor([r[5] for r in rows], dtype=torch.float64)
    args = (p, q, z, ua, ud, torch.ones(len(rows), dtype=torch.int64))
    want, got = verify_ref(*args), verify_on_gpu(*args)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0], want[0]), (got, want)
    assert want[1].tolist() == [1, 0, 1, 0, 0, 0, 0, 0, 1, 0, 1, 1]
    assert want[0][3].tolist() == [-1, -1] and want[0][5].tolist() == [5, -1] and want[0][4].tolist() == [2, -1]


@gpu
def test_verified_labels_follow_the_target():
    """The property the operator exists for: whatever the draft, the first label is distributed as the target says."""
    g = torch.Generator("cuda").manual_seed(9)
    from pybgmm_amd import ops
    B, V = 400000, 6
    p = torch.softmax(torch.randn(V, generator=g, device="cuda", dtype=torch.float64), 0)
    q = torch.softmax(torch.randn(V, generator=g, device="cuda", dtype=torch.float64) * 2, 0)
    z = torch.multinomial(q.float(), B, replacement=True, generator=g)[:, None]
    ua, ud = torch.rand(B, 1, generator=g, device="cuda", dtype=torch.float64), torch.rand(B, generator=g, device="cuda", dtype=torch.float64)
    out, acc = ops.verify_drafts(p.expand(B, 2, V), q.expand(B, 1, V), z, ua, ud)
    share = torch.bincount(out[:, 0], minlength=V).double() / B
    # (six standard deviations of a share of B draws; the draft's own float32 sampling is off by about 1e-7)
    assert bool(((share - p).abs() <= 6 * torch.sqrt(p * (1 - p) / B) + 1e-6).all())
    want = torch.minimum(p, q).sum()
    assert abs(float(acc.double().mean() - want)) <= 6 * math.sqrt(0.25 / B) + 1e-6


# ------------------------------------------------------------------------------------------ together
def layer(lw, x, w1, b1, w2, k, K):
    from pybgmm_amd import ops
    labels, weights = ops.route(lw, k)
    groups = ops.group_rows(labels, K)
    h = torch.tanh(ops.grouped_matmul(x, w1, groups, bias=b1))
    return ops.grouped_matmul(h, w2, groups, gates=weights)


def layer_inputs(n=150, K=6, k=2, din=24, hid=40, dout=12):
    g = torch.Generator("cuda").manual_seed(21)
    t = [torch.randn(*s, generator=g, device="cuda", dtype=torch.float64) * 0.5 for s in
         ((n, K), (n, din), (K, din, hid), (K, hid), (K, hid, dout))]
    return t, k, K


@gpu
def test_a_layer_of_experts_routed_and_trained():
    """route -> group_rows -> grouped_matmul twice, forward and backward, against the same layer written densely."""
    t, k, K = layer_inputs()
    leaves = [a.clone().requires_grad_() for a in t]
    y = layer(*leaves, k, K)
    dense = [a.clone().requires_grad_() for a in t]
    lw, x, w1, b1, w2 = dense
    top = torch.topk(lw, k, dim=1)
    wts = torch.softmax(top.values, 1)
    h = torch.tanh((x[:, None, None, :] @ w1[top.indices])[:, :, 0] + b1[top.indices])
    want = ((h[:, :, None, :] @ w2[top.indices])[:, :, 0] * wts[..., None]).sum(1)
    assert torch.allclose(y, want, rtol=0, atol=1e-12)
    dy = torch.randn_like(y)
    for a, b in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, dense, dy)):
        assert torch.allclose(a, b, rtol=0, atol=1e-11)


@gpu
def test_another_stream_and_two_calls_at_once():
    t, k, K = layer_inputs()
    with torch.no_grad():
        want = layer(*t, k, K)
        half = layer(*[a * 0.5 for a in t], k, K)
        torch.cuda.synchronize()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        other = [a * 0.5 for a in t]
        s1.wait_stream(torch.cuda.current_stream())
        s2.wait_stream(torch.cuda.current_stream())
        got = []
        for _ in range(5):
            with torch.cuda.stream(s1):
                a = layer(*t, k, K)
            with torch.cuda.stream(s2):
                b = layer(*other, k, K)
            got.append((a, b))
        s1.synchronize()
        s2.synchronize()
    for a, b in got:
        assert torch.equal(a, want) and torch.equal(b, half)


@gpu
def test_captured_and_replayed():
    """The layer and a verification in one graph: every replay on new inputs equals the eager result."""
    from pybgmm_amd import ops
    t, k, K = layer_inputs(n=700)
    draft = [a.cuda() for a in verify_case(9, 4, 300, torch.float32, 77)]
    static = [a.clone() for a in t]
    sdraft = [a.clone() for a in draft]

    def both(a, d):
        return (layer(*a, k, K),) + tuple(ops.verify_drafts(*d[:5], lengths=d[5]))
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            both(static, sdraft)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both(static, sdraft)
        for r in range(4):
            new = [a + 0.3 * r * torch.randn_like(a) for a in t]
            nd = [a.cuda() for a in verify_case(9, 4, 300, torch.float32, 100 + r)]
            for dst, src in zip(static + sdraft, new + nd):
                dst.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            want = both(new, nd)
            for a, b in zip(got, want):
                assert torch.equal(a, b), r


@gpu
def test_a_training_step_captured_and_replayed():
    t, k, K = layer_inputs(n=300)
    static = [a.clone().requires_grad_() for a in t]
    dy = torch.randn(300, 12, device="cuda", dtype=torch.float64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(layer(*static, k, K), static, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(layer(*static, k, K), static, dy)
    for r in range(3):
        new = [a + 0.2 * r * torch.randn_like(a) for a in t]
        with torch.no_grad():
            for dst, src in zip(static, new):
                dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        leaves = [a.clone().requires_grad_() for a in new]
        want = torch.autograd.grad(layer(*leaves, k, K), leaves, dy)
        for a, b in zip(got, want):
            assert torch.equal(a, b), r


@gpu
def test_rows_beyond_32_bits_of_elements():
    """A target whose rows start beyond 2^31 elements, and rows of x beyond 2^32 bytes."""
    from pybgmm_amd import ops
    V = 1 << 20
    p = torch.zeros(1100, 2, V, device="cuda", dtype=torch.float16)              # 2.3e9 elements
    q = torch.zeros(1, 1, V, device="cuda", dtype=torch.float16).expand(1100, 1, V)
    p[1099, 0, 12345] = 0.5
    p[1099, 1, V - 1] = 1
    z = torch.full((1100, 1), 12345, device="cuda")
    u = torch.full((1100, 1), 0.5, device="cuda", dtype=torch.float64)
    out, acc = ops.verify_drafts(p, q, z, u, u[:, 0].contiguous())
    assert out[1099].tolist() == [12345, V - 1] and int(acc.sum()) == 1 and bool((out[:1099] == -1).all())
    del p, q
    n, d = 2200000, 1024
    x = torch.zeros(n, d, device="cuda", dtype=torch.float16)                    # 2.25e9 elements
    x[n - 1] = 1
    w = torch.ones(2, d, 16, device="cuda", dtype=torch.float16)
    z = torch.zeros(n, dtype=torch.int64, device="cuda")
    z[n - 1] = 1
    y = ops.grouped_matmul(x, w, ops.group_rows(z, 2))
    assert bool((y[n - 1] == d).all()) and not bool(y[:n - 1].any())


# ------------------------------------------------------------------------------------------ the model classes' own calls
@gpu
def test_posterior_labels_and_standardised_points():
    import numpy as np
    from pybgmm_amd.igmm import CRPMM
    from pybgmm_amd.prior import NIW
    from pybgmm_amd.utils import gendata
    import random
    random.seed(3)
    np.random.seed(3)
    X, _ = gendata.synth_mixture(600, 5, 4, seed=2)
    mm = CRPMM(X, NIW(np.zeros(5), 0.05, 8, np.eye(5)), 1.0, None, assignments="rand", K=6)
    mm.collapsed_gibbs_sampler(5, np.zeros(600, dtype=int))
    comp, K = mm.components, mm.components.K
    # the densities are the sampler's own: log_post_pred of a training point, the prior's log predictive
    dens = comp.log_predictive(X[:40])
    for i in range(40):
        np.testing.assert_allclose(dens[i, :K], comp.log_post_pred(i), rtol=1e-9, atol=1e-9)
        np.testing.assert_allclose(dens[i, K], comp.log_prior(i), rtol=1e-9, atol=1e-9)
    # labels and weights: the visit's normalised weights
    lw = dens + np.log(np.append(comp.counts[:K].astype(float), mm.alpha))
    p = np.exp(lw - lw.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    labels, w = mm.posterior_labels(X[:40], k=min(3, K + 1))
    order = np.argsort(-lw, axis=1, kind="stable")[:, :labels.shape[1]]
    np.testing.assert_array_equal(labels, order)
    np.testing.assert_allclose(w, np.take_along_axis(p, order, 1), rtol=1e-9, atol=1e-13)
    t_labels, t_w = mm.posterior_labels(torch.from_numpy(X[:40]).cuda(), k=labels.shape[1])
    assert np.array_equal(t_labels.cpu().numpy(), labels) and np.array_equal(t_w.cpu().numpy(), w)
    # standardised points: mean and scale of the predictive taken out
    r = comp.standardise()
    z, counts = comp.assignments, comp.counts
    m, S = comp.m_N_numerators, comp.S_N_partials
    for i in range(0, 600, 37):
        k = z[i]
        kN, vN = 0.05 + counts[k], 8 + counts[k]
        mean = m[k] / kN
        cov = (kN + 1) / (kN * (vN - 5 + 1)) * (S[k] - kN * np.outer(mean, mean))
        want = np.linalg.solve(np.linalg.cholesky(cov), X[i] - mean)
        np.testing.assert_allclose(r[i], want, rtol=1e-9, atol=1e-9)
    assert not comp.standardise(X[:3], np.array([-1, 0, -1]))[[0, 2]].any()
    with pytest.raises(ValueError):
        comp.standardise(X[:3])
    with pytest.raises(ValueError):
        mm.posterior_labels(X[:, :4])


@gpu
def test_diagonal_components_have_no_factors():
    import numpy as np
    from pybgmm_amd.igmm import CRPMM
    from pybgmm_amd.prior import NIW
    X = np.random.RandomState(0).randn(30, 3)
    mm = CRPMM(X, NIW(np.zeros(3), 0.1, 5, np.ones(3)), 1.0, None, assignments="rand", K=2, covariance_type="diag")
    with pytest.raises(NotImplementedError):
        mm.posterior_labels(X)


# ------------------------------------------------------------------------------------------ what the documentation allows or refuses
@gpu
def test_weights_and_their_gradients_beyond_32_bits_of_elements():
    """Three matrices of 2^30 elements: the last begins at element 2^31.  Small integers, so every result is exact."""
    from pybgmm_amd import ops
    d = 1 << 15
    w = torch.zeros(3, d, d, device="cuda", dtype=torch.float16)
    w[2, d - 1, d - 1], w[2, 0, 5], w[1, 7, d - 1] = 3, 2, 1
    x = torch.zeros(5, d, device="cuda", dtype=torch.float16)
    x[:, d - 1], x[:, 0], x[:, 7] = 1, torch.arange(5, device="cuda", dtype=torch.float16), 4
    w.requires_grad_()
    z = torch.tensor([2, 0, 2, 1, 2], device="cuda")
    y = ops.grouped_matmul(x, w, ops.group_rows(z, 3))
    want = torch.zeros_like(y)
    want[[0, 2, 4], d - 1], want[3, d - 1] = 3, 4
    want[[0, 2, 4], 5] = 2 * torch.tensor([0, 2, 4], device="cuda", dtype=torch.float16)
    assert torch.equal(y, want)
    dy = torch.zeros_like(y)
    dy[:, d - 2] = 1
    dw, = torch.autograd.grad(y, w, dy)
    for e, rows in enumerate(([1], [3], [0, 2, 4])):
        assert torch.equal(dw[e, :, d - 2], x.detach()[rows].sum(0))
    assert int(torch.count_nonzero(dw)) == int(torch.count_nonzero(dw[:, :, d - 2]))


@gpu
def test_a_label_is_compared_in_64_bits():
    from pybgmm_amd import ops
    z = torch.tensor([1, (1 << 32) + 1, -(1 << 32), (1 << 62), 0], device="cuda")
    g = ops.group_rows(z, 2)
    assert g.counts.tolist() == [1, 1]
    x = torch.ones(5, 3, device="cuda")
    y = ops.grouped_matmul(x, torch.ones(2, 3, 2, device="cuda"), g)
    assert y[:, 0].tolist() == [3, 0, 0, 0, 3]
    p = torch.ones(2, 2, 2, device="cuda")
    out, acc = ops.verify_drafts(p, p[:, :1], torch.tensor([[(1 << 32) + 1], [1]], device="cuda"), torch.zeros(2, 1, device="cuda", dtype=torch.float64),
                                 torch.full((2,), 0.75, device="cuda", dtype=torch.float64))
    assert acc.tolist() == [0, 1] and out.tolist() == [[1, -1], [1, 1]]


@gpu
def test_views_that_are_negated_on_reading():
    """The imaginary part of a conjugate shares the memory of the number; the operators see its values."""
    from pybgmm_amd import ops
    g = torch.Generator("cuda").manual_seed(5)

    def neg(t):
        return torch.complex(torch.zeros_like(t), -t).conj().imag
    lw = torch.randn(40, 6, device="cuda", dtype=torch.float64, generator=g)
    x = torch.randn(40, 6, device="cuda", dtype=torch.float64, generator=g)
    w = torch.randn(6, 6, 5, device="cuda", dtype=torch.float64, generator=g)
    b = torch.randn(6, 5, device="cuda", dtype=torch.float64, generator=g)
    assert neg(lw).is_neg() and torch.equal(neg(lw), lw)
    labels, gates = ops.route(lw, 2)
    for a, c in zip((labels, gates), ops.route(neg(lw), 2)):
        assert torch.equal(a, c)
    groups = ops.group_rows(labels, 6)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, gates)]
    views = [t.clone().requires_grad_() for t in (x, w, b, gates)]
    y = ops.grouped_matmul(leaves[0], leaves[1], groups, bias=leaves[2], gates=leaves[3])
    y2 = ops.grouped_matmul(neg(views[0]), neg(views[1]), groups, bias=neg(views[2]), gates=neg(views[3]))
    assert torch.equal(y, y2)
    dy = torch.randn_like(y)
    for a, c in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(y2, views, neg(dy))):
        assert torch.equal(a, c)
    p = torch.rand(3, 3, 9, device="cuda", dtype=torch.float64, generator=g)
    u = torch.rand(3, 2, device="cuda", dtype=torch.float64, generator=g)
    z = torch.tensor([[1, 2], [3, 4], [8, 0]], device="cuda")
    want = ops.verify_drafts(p, p[:, 1:].contiguous(), z, u, u[:, 0].contiguous())
    got = ops.verify_drafts(neg(p), neg(p[:, 1:].contiguous()), z, neg(u), neg(u[:, 0].contiguous()))
    assert all(torch.equal(a, c) for a, c in zip(want, got))


@gpu
def test_derivatives_that_are_refused():
    from pybgmm_amd import ops
    from pybgmm_amd._lib import BGMMError
    lw = torch.randn(8, 4, device="cuda", requires_grad=True)
    x = torch.randn(8, 3, device="cuda", requires_grad=True)
    w = torch.randn(4, 3, 2, device="cuda", requires_grad=True)
    labels, gates = ops.route(lw, 2)
    y = ops.grouped_matmul(x, w, ops.group_rows(labels, 4), gates=gates)
    for out, leaf in ((gates, lw), (y, w)):
        with pytest.raises(RuntimeError, match="differentiable once"):          # (reported by torch's engine)
            torch.autograd.grad(out.sum(), leaf, create_graph=True, retain_graph=True)
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        dual = fw.make_dual(lw.detach(), torch.ones_like(lw))
        with pytest.raises(BGMMError) as e:
            ops.route(dual, 2)
        assert e.value.code == -5
        with pytest.raises(BGMMError) as e:
            ops.grouped_matmul(fw.make_dual(x.detach(), torch.ones_like(x)), w.detach(), ops.group_rows(labels, 4))
        assert e.value.code == -5


@gpu
def test_a_captured_step_is_refused_while_an_eager_graph_of_its_leaves_lives():
    """Made on the default stream, that graph's leaves would draw it into the capture in backward."""
    from pybgmm_amd import ops
    from pybgmm_amd._lib import BGMMError
    t, k, K = layer_inputs(n=120)
    leaves = [a.clone().requires_grad_() for a in t]
    dy = torch.randn(120, 12, device="cuda", dtype=torch.float64)
    y = layer(*leaves, k, K)                                        # lives
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    x, w = torch.randn(6, 3, device="cuda"), torch.randn(2, 3, 2, device="cuda", requires_grad=True)
    groups = ops.group_rows(torch.tensor([0, 1, 1, 0, -1, 1], device="cuda"), 2)
    kept = w * 2
    torch.cuda.synchronize()
    with pytest.raises(BGMMError) as e:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            dy.add(1.0)
            layer(*leaves, k, K)
    assert e.value.code == -5 and "default stream" in str(e.value)
    with pytest.raises(BGMMError) as e:                             # the leaf, and a product behind it
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            dy.add(1.0)
            ops.grouped_matmul(x, w, groups)
    assert e.value.code == -5
    with pytest.raises(BGMMError) as e:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            dy.add(1.0)
            ops.grouped_matmul(x, kept, groups)
    assert e.value.code == -5
    with torch.no_grad():                                           # without gradients it is an ordinary capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            again = layer(*leaves, k, K)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, y)
    del y, kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(layer(*leaves, k, K), leaves, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@gpu
def test_route_of_more_rows_than_a_launch_takes():
    from pybgmm_amd import ops
    n = (1 << 25) + 5
    lw = torch.randint(-8, 8, (n, 3), device="cuda", dtype=torch.int8).to(torch.bfloat16).requires_grad_()
    for renormalise in (True, False):
        labels, weights = ops.route(lw, 1, renormalise)
        # (the first of equal ones, exactly: small integers)
        key = lw.detach() * 4 - torch.arange(3, device="cuda", dtype=torch.bfloat16)
        assert torch.equal(labels[:, 0], key.argmax(1))
        grad, = torch.autograd.grad(weights.sum(), lw)
        if renormalise:
            assert bool((weights == 1).all()) and not bool(grad.any())
            continue
        p = torch.softmax(lw.detach().float(), 1)
        top = p.gather(1, labels)
        # (softmax in 32 bits on either side: a few units of 2^-24 each; the gradient is rounded to bfloat16, 2^-8 of at most 1/4)
        assert float((weights - top).abs().max()) < 2e-6
        want = top * (torch.nn.functional.one_hot(labels[:, 0], 3) - p)
        assert float((grad.float() - want).abs().max()) < 2.0 ** -8 / 4 + 2e-6


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
def test_a_large_batch_draws_as_its_parts_do(dt):
    """Batches of more than 512 sequences and smaller ones take the sums of a chunk in different parts."""
    from pybgmm_amd import ops
    args = [a.cuda() for a in verify_case(600, 2, 9001, dt, 11)]
    out, acc = ops.verify_drafts(*args[:5], lengths=args[5])
    for i in range(0, 600, 120):
        part = [a[i:i + 120] for a in args]
        o, c = ops.verify_drafts(*part[:5], lengths=part[5])
        assert torch.equal(o, out[i:i + 120]) and torch.equal(c, acc[i:i + 120])


@gpu
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,k,K,din,dout", [(300, 1, 5, 37, 21), (300, 2, 4, 64, 16), (5, 2, 3, 7, 9), (2000, 1, 6, 130, 67)])
def test_broadcast_operands(dt, n, k, K, din, dout):
    """Operands of stride zero give what their copies give, and the gradients of what was broadcast are sums."""
    from pybgmm_amd import ops
    z, x, w, b, gt, g = product_case(n, k, K, din, dout, dt, 3 * n + din)
    groups = ops.group_rows(z, K)
    gt = torch.nan_to_num(gt)
    one_row, one_matrix, one_line = torch.randn(1, din, generator=g, device="cuda").to(dt), w[:1].clone(), w[:1, :1].clone()
    cases = [(one_row.expand(n, din), w, b, gt), (x, one_matrix.expand(K, din, dout), b, gt), (x, one_line.expand(K, din, dout), b[:1].expand(K, dout), gt),
             (x, w, b[:, :1].expand(K, dout), gt[:1].expand(n, k)), (x, w[:, :1].expand(K, din, dout).transpose(1, 2).contiguous().transpose(1, 2), b, gt)]
    dy = torch.randn(n, 1, generator=g, device="cuda").to(dt).expand(n, dout)
    for case in cases:
        views = [t.detach().requires_grad_() for t in case]
        copies = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in case]
        if case is cases[4]:
            copies[1] = case[1].detach().clone(memory_format=torch.preserve_format).requires_grad_()
        y, y2 = (ops.grouped_matmul(t[0], t[1], groups, bias=t[2], gates=t[3]) for t in (views, copies))
        assert torch.equal(y, y2) or (torch.isnan(y) == torch.isnan(y2)).all() and torch.equal(torch.nan_to_num(y), torch.nan_to_num(y2))
        for a, c in zip(torch.autograd.grad(y, views, dy), torch.autograd.grad(y2, copies, dy.contiguous())):
            assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(c))
    leaf = one_row.clone().requires_grad_()
    y = ops.grouped_matmul(leaf.expand(n, din), w, groups, bias=b, gates=gt)
    full = one_row.expand(n, din).clone().requires_grad_()
    y2 = ops.grouped_matmul(full, w, groups, bias=b, gates=gt)
    got, = torch.autograd.grad(y, leaf, dy)
    rows, = torch.autograd.grad(y2, full, dy)
    assert torch.equal(got, rows.sum(0, keepdim=True))


@gpu
def test_the_same_label_in_every_place_and_one_grouping_for_two_products():
    from pybgmm_amd import ops
    g = torch.Generator("cuda").manual_seed(9)
    z = torch.full((130, 3), 2, device="cuda")
    groups = ops.group_rows(z, 4)
    x = torch.randn(130, 19, device="cuda", dtype=torch.float64, generator=g, requires_grad=True)
    w = torch.randn(4, 19, 6, device="cuda", dtype=torch.float64, generator=g, requires_grad=True)
    gates = torch.rand(130, 3, device="cuda", dtype=torch.float64, generator=g, requires_grad=True)
    y = ops.grouped_matmul(x, w, groups, gates=gates)
    want = (x @ w[2]) * gates.sum(1, keepdim=True)
    tol = dict(rtol=1e-12, atol=1e-12)                  # (19 products of about one, 3 of them added: a few hundred steps of 2^-53)
    assert torch.allclose(y, want, **tol)
    dy = torch.randn_like(y)
    for a, c in zip(torch.autograd.grad(y, (x, w, gates), dy), torch.autograd.grad(want, (x, w, gates), dy)):
        assert torch.allclose(a, c, rtol=1e-11, atol=1e-11)      # (dW: 390 terms)
    w2 = torch.randn(4, 6, 19, device="cuda", dtype=torch.float64, generator=g)
    with torch.no_grad():
        h = ops.grouped_matmul(x, w, groups)                     # a row per label, straight into the next product
        out = ops.grouped_matmul(h, w2, groups, gates=gates)
        assert tuple(h.shape) == (130, 3, 6)
        assert torch.allclose(out, ((x @ w[2]) @ w2[2]) * gates.sum(1, keepdim=True), rtol=1e-11, atol=1e-11)


@gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n,k,K,din,dout", [(700, 1, 3, 16, 16), (900, 2, 4, 130, 136), (2100, 1, 2, 24, 200), (1500, 2, 3, 200, 12), (800, 1, 3, 64, 60), (3000, 1, 2, 40, 70)])
@pytest.mark.parametrize("gate,d_size,x_size", [(1.0, 1.0, 1.0), (1e-4, 1e-4, 3e4), (1e-3, 1e-4, 3e4), (100.0, 1000.0, 1e-3), (1e30, 1e-3, 1.0)])
def test_gates_of_any_size_in_the_weights_gradient(dt, n, k, K, din, dout, gate, d_size, x_size):
    """
    Gates times gradients that 16 bits cannot hold (nothing of 1e-4 x 1e-4 is left in half precision, 100 x 1000 is infinite there), next
    to ordinary ones.  The product takes g d as two bfloat16 numbers, which lose at most 2^-15 of it (the first has 8 bits, the rest is
    rounded to 8: 2^-7 2^-8), in half precision x likewise (whose 11 bits are whole in two): 2^-14 of a term covers that with its
    second pieces' own roundings; 32-bit sums of a component's own rows (two to four products a term), and the result's own rounding.
    """
    from pybgmm_amd import ops
    if gate == 1e30 and dt == torch.float16:
        gate, x_size = 1e-30, 1e4                                           # (a result of zero: nothing may become infinite or NaN)
    g = torch.Generator("cuda").manual_seed(n + din)

    def rand(*s):
        sign = torch.randint(0, 2, s, generator=g, device="cuda") * 2 - 1
        return (torch.rand(*s, generator=g, device="cuda", dtype=torch.float64) + 0.5) * sign
    z = torch.randint(0, K, (n, k), generator=g, device="cuda")
    z[5] = -1
    x, dy = (rand(n, din) * x_size).to(dt), (rand(n, dout) * d_size).to(dt)
    w = rand(K, din, dout).to(dt).requires_grad_()
    gates = (rand(n, k) * gate).float()
    groups = ops.group_rows(z, K)
    got, = torch.autograd.grad(ops.grouped_matmul(x, w, groups, gates=gates), w, dy)
    bits, top = half_step(dt), torch.finfo(dt).max
    smallest = torch.finfo(dt).tiny * bits                                  # half of the type's smallest step
    for e in range(K):
        i, j = torch.nonzero(z == e, as_tuple=True)
        gd = gates[i, j].double()[:, None] * dy[i].double()
        want, mag = (a.t().contiguous() @ b for a, b in ((x[i].double(), gd), (x[i].double().abs(), gd.abs())))
        tol = (2.0 ** -14 + 2.0 ** -24 * (4 * i.numel() + 8)) * mag
        fits = want.abs() + tol < top
        off = (got[e].double() - want).abs()
        assert bool((off <= tol + bits * (want.abs() + tol) + smallest)[fits].all()), float((off / mag)[fits].max())
        assert fits.float().mean() > 0.9 and not torch.isnan(got[e]).any()


@gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=str)
def test_infinite_and_undefined_gates_and_gradients_stay_in_their_columns(dt):
    from pybgmm_amd import ops
    n, K, din, dout = 300, 2, 40, 33
    z = torch.arange(n, device="cuda") % K
    x, dy = torch.full((n, din), 1.5, device="cuda", dtype=dt), torch.ones(n, dout, device="cuda", dtype=dt)
    dy[4, 3], dy[7, 5], dy[6, 8] = math.inf, math.nan, -math.inf            # components 0, 1, 0
    x[12, 11] = math.inf
    w = torch.zeros(K, din, dout, device="cuda", dtype=dt, requires_grad=True)
    gates = torch.full((n,), 0.5, device="cuda")
    got, = torch.autograd.grad(ops.grouped_matmul(x, w, ops.group_rows(z, K), gates=gates), w, dy)
    want = torch.full((K, din, dout), 1.5 * 0.5 * n / K, device="cuda", dtype=torch.float64)
    want[0, :, 3], want[1, :, 5], want[0, :, 8] = math.inf, math.nan, -math.inf
    want[0, 11] = math.inf
    want[0, 11, 8] = math.nan
    ok = (got.double() == want) | (torch.isnan(got) & torch.isnan(want)) | ((got.double() - want).abs() <= 112.5 * half_step(dt))
    assert bool(ok.all())


@gpu
def test_more_sequences_than_a_launch_takes():
    """2^24 sequences, the most a call takes: with 256 threads each they are more threads than a launch counts."""
    from pybgmm_amd import ops
    B, V = 1 << 24, 2049
    p = torch.randint(0, 4, (V,), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    u = (torch.arange(B, device="cuda", dtype=torch.float64) * 48271 % B) / B
    none = torch.empty(B, 0, dtype=torch.int64, device="cuda")
    out, acc = ops.verify_drafts(p.to(torch.bfloat16).expand(B, 1, V), torch.empty(B, 0, V, device="cuda", dtype=torch.bfloat16), none, none.double(), u)
    total = p.double().cumsum(0)                                            # (whole numbers: the same in any order)
    assert not acc.any() and torch.equal(out[:, 0], torch.searchsorted(total, u * total[-1], right=True))


@gpu
def test_more_tiles_than_a_launch_takes():
    """8000 components times 2094 tiles of columns: more workgroups of 256 than a launch counts threads for, in every product."""
    from pybgmm_amd import ops
    K, dout = 8000, 268032
    g = torch.Generator("cuda").manual_seed(4)
    z = torch.randperm(K, device="cuda", generator=g)
    x = torch.randint(-8, 9, (K, 1), device="cuda", generator=g).to(torch.bfloat16).requires_grad_()
    w = torch.randint(-8, 9, (1, 1, dout), device="cuda", generator=g).to(torch.bfloat16).expand(K, 1, dout).requires_grad_()
    y = ops.grouped_matmul(x, w, ops.group_rows(z, K))
    assert torch.equal(y.detach(), x.detach() * w.detach()[0])              # (products of small integers: exact)
    dy = torch.randint(-1, 2, (K, 1), device="cuda", generator=g).to(torch.bfloat16)
    dx, dw = torch.autograd.grad(y, (x, w), dy.expand(K, dout))
    del y
    assert torch.equal(dw[z, 0], (x.detach() * dy).expand(K, dout))
    want = dy.double() * w.detach()[0].double().sum()
    assert bool(((dx.double() - want).abs() <= 2.0 ** -8 * want.abs()).all())           # (268000 terms of at most 8: exact in 32 bits)


@gpu
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,K", [(9, 7), (5, 64), (3, 1000), (2, 5000), (2, 20001)])
@pytest.mark.parametrize("renormalise", [True, False])
def test_the_largest_number_beside_infinity_has_no_weight(dt, n, K, renormalise):
    """exp(v - inf) is zero for every finite v, the type's largest among them; several infinite ones share the weight."""
    from pybgmm_amd import ops
    lw = torch.zeros(n, K, dtype=dt, device="cuda")
    lw[:, 1], lw[:, 3], lw[:, 5] = torch.finfo(dt).max, math.inf, torch.finfo(dt).min
    lw[0, 6] = math.inf
    lw.requires_grad_()
    labels, weights = ops.route(lw, 4, renormalise)
    want = torch.tensor([[1.0, 0, 0, 0]] * n, dtype=weights.dtype, device="cuda")
    want[0, :2] = 0.5
    assert torch.equal(weights.detach(), want)
    assert torch.equal(labels[1:, :3].cpu(), torch.tensor([[3, 1, 0]] * (n - 1))) and labels[0, :3].tolist() == [3, 6, 1]
    up = torch.arange(1.0, 5.0, dtype=weights.dtype, device="cuda").expand(n, 4).contiguous()
    grad, = torch.autograd.grad(weights, lw, up)
    want = torch.zeros(n, K, dtype=dt, device="cuda")
    want[0, 3], want[0, 6] = -0.25, 0.25                                  # 0.5 (1 - 1.5), 0.5 (2 - 1.5)
    assert torch.equal(grad, want)


@gpu
@pytest.mark.parametrize("cls,fit,powered", [("CRPMM", {}, False), ("PCRPMM", dict(n_power=1.4), True), ("PCRPMM", dict(n_power=1.4, flag_power=False), False),
                                             ("PCRPMM", dict(n_power=1.4, power_burnin=9), False), ("ADAPCRPMM", dict(r_up=1.6, adapcrp_perct=0.5, adapcrp_burnin=-1), True),
                                             ("ADAPCRPMM", dict(flag_adapcrp=False), False)])
def test_posterior_labels_weigh_as_the_last_sweep_did(cls, fit, powered):
    """The visit's weights, n_k ** power times the predictive and alpha times the prior's, normalised, for every sampler's own power."""
    import random
    import numpy as np
    from pybgmm_amd import igmm
    from pybgmm_amd.prior import NIW
    from pybgmm_amd.utils import gendata
    random.seed(4)
    np.random.seed(4)
    X, _ = gendata.synth_mixture(400, 3, 3, seed=5, mu_scale=1.5)
    seen = []

    class Watched(getattr(igmm, cls)):
        def _sweep(self, order=None, power=None):
            seen.append(power)
            super()._sweep(order=order, power=power)
    mm = Watched(X, NIW(np.zeros(3), 0.05, 6, np.eye(3)), 0.7, None, assignments="rand", K=5)
    comp = mm.components

    def weights(power):
        lw = np.append(np.log(comp.counts[:comp.K] ** power), np.log(mm.alpha)) + np.array([np.append(comp.log_post_pred(i), comp.log_prior(i)) for i in range(30)])
        p = np.exp(lw - lw.max(1, keepdims=True))
        return p / p.sum(1, keepdims=True)

    def check(expected, **kw):
        labels, w = mm.posterior_labels(X[:30], k=comp.K + 1, **kw)
        # (64-bit predictives of two routes, as in the comparison of the densities themselves: 1e-9 of each logarithm)
        np.testing.assert_allclose(np.take_along_axis(w, np.argsort(labels, axis=1), 1), weights(expected), rtol=1e-7, atol=1e-12)
    check(1.0)                                                      # no sweep yet
    mm.collapsed_gibbs_sampler(4, np.zeros(400, dtype=int), **fit)
    power = 1.0 if seen[-1] is None else seen[-1]
    assert (power > 1.1) == powered
    check(power)
    check(2.5, power=2.5)
    if powered:
        assert np.abs(weights(power) - weights(1.0)).max() > 1e-3           # (the power matters to these points)


def test_a_groupings_memory_is_its_rows_and_components():
    """The workspace does not grow with rows times components, and a grouping keeps none of it."""
    from pybgmm_amd import ops
    from pybgmm_amd.ops import _native as nat
    L = nat.load()
    for P in (0, 1, 4096, 4097, 131072, 131073, 1000000, 10**7, 10**9, 2**31 - 65537):
        for K in (1, 100, 511, 512, 900, 1779, 1780, 3199, 3200, 8000):
            # 4 bytes for each of at most 2^21 or P + K + 1 counts of segments, a quarter as many of workgroups, one per bucket and their remainders
            assert L.bgmm_group_rows_ws(P, K) <= 5 * max(1 << 21, P + K + 1) + 12 * (K + 1), (P, K)
            assert ops.RowGroups.store_size(P, K) == 4 * L.bgmm_group_rows_tiles(P, K) + 2 * P + 9 * (K + 2)


@gpu
@pytest.mark.parametrize("P,K", [(131072, 8000), (131073, 8000), (262144, 3199), (300001, 3200), (1200000, 8000), (270000, 7999), (4300000, 511), (2200000, 1023)])
def test_groupings_of_long_segments(P, K):
    from pybgmm_amd import ops
    g = torch.Generator("cuda").manual_seed(P)
    z = (torch.rand(P, device="cuda", generator=g) ** 3 * (K + 1)).long() - 1
    grp = ops.group_rows(z, K)
    bucket = torch.where(z >= 0, z, torch.full_like(z, K))
    assert torch.equal(grp.order.long(), torch.argsort(bucket, stable=True))
    size = torch.bincount(bucket, minlength=K + 1)
    assert torch.equal(grp.counts.long(), size[:K]) and torch.equal(grp.offsets[1:].long(), size.cumsum(0))
    again = ops.group_rows(z, K)
    assert all(torch.equal(getattr(grp, a), getattr(again, a)) for a in ("order", "offsets", "first", "tiles", "bucket"))


@gpu
def test_a_grouping_recorded_on_another_stream_keeps_its_memory():
    from pybgmm_amd import ops
    z = torch.randint(0, 7, (3000000,), device="cuda")
    x, w = torch.randn(3000000, 4, device="cuda"), torch.randn(7, 4, 4, device="cuda")
    want = ops.grouped_matmul(x, w, ops.group_rows(z, 7))
    groups = ops.group_rows(z, 7)
    at = groups.tiles.data_ptr()
    size = ops.RowGroups.store_size(3000000, 7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200000000)                                # (cycles: about 0.1 s)
        y = ops.grouped_matmul(x, w, groups)
    groups.record_stream(side)
    del groups
    others = [torch.full((size,), 1 << 20, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert not side.query()                                         # (the product still waits)
    assert at not in [t.data_ptr() for t in others]
    side.synchronize()
    assert torch.equal(y, want)
    with pytest.raises(RuntimeError):                                # (as Tensor.record_stream)
        ops.group_rows(z, 7).record_stream(3)


# components' rows around a tile's, a step's and a chunk's borders; and enough rows for longer chunks
BORDERS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 4095, 4097, 8193]
MANY = [600001, 300000, 131072, 65537, 32769, 32767, 16385, 8191, 2049, 1023, 513, 255, 20, 0, 3]


@gpu
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("din,dout,sizes", [(16, 16, BORDERS), (5, 100, BORDERS), (130, 7, BORDERS), (64, 64, BORDERS), (40, 128, BORDERS), (128, 33, BORDERS),
                                            (131, 140, BORDERS), (3, 4, MANY), (16, 70, MANY), (70, 9, MANY), (129, 130, MANY[1:])])
def test_sums_of_whole_numbers_are_exact(dt, gated, din, dout, sizes):
    """
    Small whole numbers and gates that are powers of two: every product and every partial sum is held exactly (in quarters below 2^24, which
    the magnitudes' sum shows), so that a row, a step or a chunk that is lost, doubled or misplaced cannot hide behind a tolerance;
    what is left is the result's one rounding.
    """
    from pybgmm_amd import ops
    K, n = len(sizes), sum(sizes)
    g = torch.Generator("cuda").manual_seed(din * dout)

    def whole(*s):
        return torch.randint(-2, 3, s, generator=g, device="cuda").to(dt)
    z = torch.repeat_interleave(torch.arange(K, device="cuda"), torch.tensor(sizes, device="cuda"))[torch.randperm(n, device="cuda", generator=g)]
    x, w, b, dy = whole(n, din), whole(K, din, dout), whole(K, dout), whole(n, dout)
    gates = 2.0 ** torch.randint(-2, 2, (n,), generator=g, device="cuda").to(acc_of(dt)) if gated else None
    leaves = [t.requires_grad_() for t in (x, w, b, gates) if t is not None]
    y = ops.grouped_matmul(x, w, ops.group_rows(z, K), bias=b, gates=gates)
    grads = torch.autograd.grad(y, leaves, dy)
    got = dict(zip(("x", "w", "b", "g"), grads), y=y.detach())
    want = {a: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for a, t in got.items()}
    largest = 0.0
    with torch.no_grad():
        for e in range(K):
            i = torch.nonzero(z == e)[:, 0]
            xe, de, we, be = x[i].double(), dy[i].double(), w[e].double(), b[e].double()
            ge = gates[i].double()[:, None] if gated else 1.0
            u, v = xe @ we + be, de @ we.t().contiguous()
            want["y"][i], want["x"][i], want["w"][e], want["b"][e] = ge * u, ge * v, xe.t().contiguous() @ (ge * de), (ge * de).sum(0)
            if gated:
                want["g"][i] = (de * u).sum(1)
            largest = max(largest, float((xe.abs().t().contiguous() @ (ge * de).abs()).max())) if i.numel() else largest
    assert largest * 4 < 2 ** 24
    for name, t in got.items():
        exact = want[name].float().to(t.dtype) if t.dtype != torch.float64 else want[name]
        off = t != exact
        assert not bool(off.any()), (name, int(off.sum()), torch.nonzero(off)[:4].tolist(), t[off][:4].tolist(), want[name][off][:4].tolist())


def test_c_entry_points_refuse_axes_whose_bytes_32_bits_do_not_count():
    from pybgmm_amd.ops import _native as nat
    L = nat.load()
    buf = ctypes.create_string_buffer(64)
    p, big = ctypes.addressof(buf), 1 << 27
    assert L.bgmm_rows_product_splits(0, 8, 2, 1 << 28, 4) == 1             # (2^31 bytes of doubles)
    assert L.bgmm_weight_product_ws(0, 1000, 2, big, 4) == 0
    for kdim, ndim in ((big, 4), (4, big)):
        assert L.bgmm_rows_product(0, p, 4, 1, p, 4, 4, 0, None, 0, None, p, 4, None, 1, None, 0, 1, None, 8, 2, kdim, ndim, p, p, None) == -5
        assert L.bgmm_weight_product(0, p, 4, 1, p, 4, 1, None, p, None, None, 0, 8, 2, kdim, ndim, p, p, p, None) == -5
    assert L.bgmm_combine(0, p, 1, 4, 1, 2, p, None, p, 4, big, None, None, 0, None, 0, None, 0, 1, 1, None) == -5


@gpu
@pytest.mark.parametrize("K", [5, 300, 3000, 20001])
def test_route_weights_down_to_the_smallest_normal_number(K):
    """
    Single precision.  The difference x from the maximum is rounded, |x| 2^-24, which is that much of the result; exp is off by at most
    2^-21 (the hardware's one step, the argument's correction, three roundings and the quotient's); below 2^-126 it is zero.
    """
    from pybgmm_amd import ops
    down = torch.arange(1, 401, dtype=torch.float64) * -0.2625                # to -105; e^-87.34 is 2^-126
    lw = torch.full((400, K), -math.inf)
    lw[:, 1], lw[:, 3] = 2.0, (2.0 + down).float()
    labels, w = ops.route(lw.cuda(), 3, False)
    x = lw[:, 3].double() - 2.0
    want = torch.exp(x) / (1 + torch.exp(x))
    assert bool((labels.cpu() == torch.tensor([1, 3, -1])).all())
    off = (w[:, 1].cpu().double() - want).abs()
    assert bool((off <= (2.0 ** -21 + 2.0 ** -24 * x.abs()) * want)[x > -87.3].all())
    assert bool((off <= want)[x <= -87.3].all()) and bool((w[-5:, 1].cpu() == 0).all()) and not w[:, 2].any()


@gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=str)
def test_a_large_grouping_and_gated_gradients_captured_and_replayed(dt):
    """A grouping in several launches, whose workspace is gone when it returns, and the product of 16-bit pieces."""
    from pybgmm_amd import ops
    n, K = 140000, 2500
    g = torch.Generator("cuda").manual_seed(8)

    def inputs():
        z = (torch.rand(n, device="cuda", generator=g) ** 2 * (K + 1)).long() - 1
        return [z] + [torch.randn(*s, device="cuda", generator=g).to(dt) for s in ((n, 20), (K, 20, 24), (n, 24))] + [torch.rand(n, device="cuda", generator=g)]

    def step(z, x, w, dy, gates):
        groups = ops.group_rows(z, K)
        y = ops.grouped_matmul(x, w, groups, gates=gates)
        return (groups.order, y.detach()) + torch.autograd.grad(y, (x, w, gates), dy)
    static = inputs()
    for i in (1, 2, 4):
        static[i].requires_grad_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*static)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*static)
    for r in range(4):
        new = inputs()
        with torch.no_grad():
            for dst, src in zip(static, new):
                dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        for i in (1, 2, 4):
            new[i].requires_grad_()
        for a, b in zip(got, step(*new)):
            assert torch.equal(a, b), r
