"""
Cases of the mixture-of-experts operators (``pybgmm_amd.ops``) and their plain forms.

Three operators and what they have to compute:

  route      the k most probable components of every row of log weights (ties to the lowest index), with their weights: the
             softmax over the chosen ones, or over all of them; its gradient
  products   rows grouped by their component and multiplied with that component's matrix, ragged groups, rows in the caller's
             order on both sides; optionally weighted by gates and summed over a row's k components; its gradients
  verify     drafted labels accepted or rejected against the target's probabilities from given uniforms, the label behind the
             last accepted one drawn from the target, or from what the target has in excess of the draft

``own = False``: elementary torch operations.  ``own = True``: the calls a user makes.  ``listed()`` holds the cases by name,
``draw(rng)`` one more of the same ranges, ``exact(case, seed)`` the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one new point routed over a fitted mixture's components: latency
        dict(name="route-one-point", op="route", n=1, K=200, k=4, dtype="f64", backward=False, renormalise=False),
        # the posterior labels of every point of the benchmark's data set (N = 1e6, K = 200)
        dict(name="route-every-point", op="route", n=1000000, K=200, k=4, dtype="f64", backward=False, renormalise=False),
        # a learned gate in training: 64 experts, six chosen, with the gradient of its log weights
        dict(name="route-train", op="route", n=32768, K=64, k=6, dtype="bf16", backward=True, renormalise=True),
        # every point standardised by its own component's factor: the benchmark's data set, D = 64
        dict(name="standardise-64", op="products", n=1000000, K=200, k=1, din=64, dout=64, dtype="f64", backward=False, gated=False, bias=True, skew=1.0),
        # the same at D = 128 and N = 2e6
        dict(name="standardise-128", op="products", n=2000000, K=200, k=1, din=128, dout=128, dtype="f64", backward=False, gated=False, bias=True, skew=1.0),
        # one linear map per component over many short rows, in half precision
        dict(name="map-16", op="products", n=1000000, K=100, k=1, din=16, dout=16, dtype="f16", backward=False, gated=False, bias=True, skew=0.0),
        # a layer of 64 experts in training, two per row, gated, all gradients
        dict(name="train-wide", op="products", n=8192, K=64, k=2, din=1024, dout=2048, dtype="bf16", backward=True, gated=True, bias=True, skew=0.3),
        # per-component regressions in training: odd sizes, uneven groups, single precision
        dict(name="train-odd", op="products", n=20011, K=33, k=1, din=192, dout=77, dtype="f32", backward=True, gated=False, bias=True, skew=1.0),
        # one row served: four of 64 experts, latency and the chosen experts' weights
        dict(name="serve-one", op="products", n=1, K=64, k=4, din=2048, dout=1024, dtype="bf16", backward=False, gated=True, bias=True, skew=0.0),
        # one sequence of four drafts over a large set of labels: latency
        dict(name="verify-one", op="verify", B=1, T=4, V=50000, dtype="f32", agree=0.8),
        # many chains' drafted labels over a mixture's components
        dict(name="verify-chains", op="verify", B=20000, T=8, V=200, dtype="f64", agree=0.9),
        # a batch of sequences with ragged draft lengths over a large set of labels
        dict(name="verify-batch", op="verify", B=256, T=5, V=131072, dtype="bf16", agree=0.7),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("route", "products", "products", "verify"))
    while True:
        if op == "route":
            K = _log_int(rng, 2, 1024)
            c = dict(op=op, n=_log_int(rng, 1, 1000000), K=K, k=rng.randint(1, min(8, K)), dtype=rng.choice(("f64", "f32", "f16", "bf16")),
                     backward=rng.random() < 0.4, renormalise=rng.random() < 0.5)
            if c["n"] * K * SIZE[c["dtype"]] * (2 if c["backward"] else 1) <= 1.6e9:
                return c
        elif op == "products":
            K = _log_int(rng, 1, 256)
            c = dict(op=op, n=_log_int(rng, 1, 1000000), K=K, k=rng.randint(1, min(4, K)), din=_log_int(rng, 2, 2048), dout=_log_int(rng, 1, 2048),
                     dtype=rng.choice(("f64", "f32", "f16", "bf16")), backward=rng.random() < 0.5, gated=rng.random() < 0.5,
                     bias=rng.random() < 0.7, skew=rng.choice((0.0, 0.5, 1.0)))
            w = work(c)
            P = c["n"] * c["k"]
            # (f64 and f32 products run at a fraction of the 16-bit ones' rate)
            if w["flops"] <= (3e10 if c["dtype"] in ("f64", "f32") else 1e11) and w["bytes"] <= 3e9 and P * (c["din"] + c["dout"]) <= 3e8:
                return c
        else:
            c = dict(op=op, B=_log_int(rng, 1, 20000), T=rng.randint(1, 8), V=_log_int(rng, 2, 131072), dtype=rng.choice(("f64", "f32", "f16", "bf16")),
                     agree=rng.uniform(0.3, 0.95))
            if c["B"] * (2 * c["T"] + 1) * c["V"] <= 3e8:
                return c


def work(case):
    s = SIZE[case["dtype"]]
    if case["op"] == "route":
        n, K, k = case["n"], case["K"], case["k"]
        ws = 8 if case["dtype"] == "f64" else 4
        b = n * K * s + n * k * (8 + ws)
        if case["backward"]:
            b += n * K * s + n * k * ws
        return {"bytes": b, "flops": n * K * (4 + (4 if case["backward"] else 0))}
    if case["op"] == "products":
        n, K, k, din, dout = case["n"], case["K"], case["k"], case["din"], case["dout"]
        P, gs = n * k, 8 if case["dtype"] == "f64" else 4
        used = min(K, P)
        ny = n if (case["gated"] or k == 1) else P
        par = din * dout + (dout if case["bias"] else 0)
        b = P * 8 + n * din * s + used * par * s + ny * dout * s + (P * gs if case["gated"] else 0)
        f = 2 * P * din * dout
        if case["backward"]:
            b += ny * dout * s + n * din * s + K * par * s + (P * gs if case["gated"] else 0)
            f *= 3
        return {"bytes": b, "flops": f}
    B, T, V = case["B"], case["T"], case["V"]
    rows = 1.0 + (1.0 - case["agree"] ** T)           # the target's row; the draft's too where a draft was rejected
    return {"bytes": int(B * (V * s * rows + T * (8 + 8 + 2 * s) + 16 + (T + 2) * 8)), "flops": int(B * V * 3)}


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) + 1)
    return g


def _labels(case, g):
    """(n,) or (n, k) labels, the k of a row distinct; shares fall off as (j + 1) ** -skew; about 1 in 500 rows unassigned."""
    n, K, k = case["n"], case["K"], case["k"]
    share = (torch.arange(K, device="cuda", dtype=torch.float32) + 1.0) ** -case["skew"]
    share = share[torch.randperm(K, generator=g, device="cuda")]
    if k == 1:
        edges = torch.cumsum(share.double(), 0)
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * edges[-1]
        z = torch.searchsorted(edges, u, right=True).clamp_(max=K - 1)
        if n > 1:
            z[torch.rand(n, generator=g, device="cuda") < 0.002] = -1
        return z
    out = torch.empty(n, k, dtype=torch.int64, device="cuda")
    step = max(1, 50000000 // K)
    for i in range(0, n, step):
        m = min(step, n - i)
        gumbel = -torch.log(-torch.log(torch.rand(m, K, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)))
        out[i:i + m] = torch.topk(gumbel + torch.log(share), k, dim=1).indices
    return out


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    st = dict(case=case)
    if case["op"] == "route":
        n, K, k = case["n"], case["K"], case["k"]
        lw = torch.empty(n, K, device="cuda", dtype=dt)
        step = max(1, 100000000 // K)
        for i in range(0, n, step):
            m = min(step, n - i)
            v = torch.randn(m, K, generator=g, device="cuda") * 3.0
            v[torch.rand(m, K, generator=g, device="cuda") < 0.02] = -math.inf          # components without members
            lw[i:i + m] = v.to(dt)
        if n > 8:
            lw[n // 3] = -math.inf                                                       # a row that nothing explains
        st["log_weights"] = lw.requires_grad_(case["backward"])
        if case["backward"]:
            st["dweights"] = torch.randn(n, k, generator=g, device="cuda", dtype=torch.float64 if dt == torch.float64 else torch.float32)
    elif case["op"] == "products":
        n, K, k, din, dout = case["n"], case["K"], case["k"], case["din"], case["dout"]
        gt = torch.float64 if dt == torch.float64 else torch.float32
        rg = case["backward"]

        def randn(*shape, scale=1.0):
            t = torch.empty(*shape, device="cuda", dtype=dt)
            flat = t.view(-1)
            for i in range(0, flat.numel(), 1 << 27):
                m = min(1 << 27, flat.numel() - i)
                flat[i:i + m] = (torch.randn(m, generator=g, device="cuda", dtype=gt) * scale).to(dt)
            return t
        st["labels"] = _labels(case, g)
        st["x"] = randn(n, din).requires_grad_(rg)
        st["weight"] = randn(K, din, dout, scale=din ** -0.5).requires_grad_(rg)
        st["bias"] = randn(K, dout).requires_grad_(rg) if case["bias"] else None
        st["gates"] = None
        if case["gated"]:
            gates = torch.rand(n, k, generator=g, device="cuda", dtype=gt) + 0.1
            gates = gates / gates.sum(1, keepdim=True)
            st["gates"] = (gates[:, 0].contiguous() if k == 1 else gates).requires_grad_(rg)
        if rg:
            st["dy"] = randn(n, dout) if (case["gated"] or k == 1) else randn(n, k, dout)
    else:
        B, T, V = case["B"], case["T"], case["V"]
        target = torch.empty(B, T + 1, V, device="cuda", dtype=dt)
        draft = torch.empty(B, T, V, device="cuda", dtype=dt)
        labels = torch.empty(B, T, device="cuda", dtype=torch.int64)
        ct = torch.float64 if dt == torch.float64 else torch.float32
        step = max(1, 30000000 // ((T + 1) * V))
        for i in range(0, B, step):
            m = min(step, B - i)
            lp = torch.randn(m, T + 1, V, generator=g, device="cuda", dtype=ct) * 2.0
            target[i:i + m] = torch.softmax(lp, -1).to(dt)
            lq = lp[:, :T] + torch.randn(m, T, V, generator=g, device="cuda", dtype=ct) * (2.0 * (1.0 - case["agree"]))
            draft[i:i + m] = torch.softmax(lq, -1).to(dt)
            expo = -torch.log(torch.rand(m, T, V, generator=g, device="cuda", dtype=ct).clamp_(min=1e-30))
            labels[i:i + m] = (lq - torch.log(expo)).argmax(-1)
        st.update(target=target, draft=draft, labels=labels,
                  u_accept=torch.rand(B, T, generator=g, device="cuda", dtype=torch.float64),
                  u_draw=torch.rand(B, generator=g, device="cuda", dtype=torch.float64),
                  lengths=torch.randint(0 if B > 1 else T, T + 1, (B,), generator=g, device="cuda"))
    return st


# ------------------------------------------------------------------------------------------ plain forms
def _plain_route(st):
    case, lw = st["case"], st["log_weights"].detach()
    K, k = case["K"], case["k"]
    v = lw if lw.dtype == torch.float64 else lw.float()
    v = torch.where(v > -math.inf, v, torch.full_like(v, -math.inf))           # (NaN never chosen)
    idx = torch.arange(K, device=v.device)
    left, labels, vals = v, [], []
    for _ in range(k):
        m = left.max(1, keepdim=True).values
        j = torch.where(left == m, idx, K).min(1, keepdim=True).values
        left = torch.where(idx == j, -math.inf, left)
        labels.append(torch.where(m > -math.inf, j, -1))
        vals.append(m)
    labels, vals = torch.cat(labels, 1), torch.cat(vals, 1)
    top = vals[:, :1]
    some = top > -math.inf
    top = torch.where(some, top, 0.0)
    e = torch.exp(torch.where(vals == top, 0.0, vals - top))
    all_e = None
    if case["renormalise"]:
        total = e.sum(1, keepdim=True)
    else:
        all_e = torch.exp(torch.where(v == top, 0.0, v - top))
        total = all_e.sum(1, keepdim=True)
    total = torch.where(some, total, 1.0)
    w = torch.where(labels >= 0, e / total, 0.0)
    if not case["backward"]:
        return labels, w
    dw = st["dweights"]
    inner = torch.where(labels >= 0, w * dw, 0.0)
    s = inner.sum(1, keepdim=True)
    if case["renormalise"]:
        d = torch.zeros_like(v)
        d.scatter_add_(1, labels.clamp(min=0), torch.where(labels >= 0, w * (dw - s), 0.0))
    else:
        d = torch.where(some, -s * all_e / total, 0.0)
        d.scatter_add_(1, labels.clamp(min=0), inner)
    return labels, w, d.to(lw.dtype)


def _plain_products(st):
    case = st["case"]
    n, K, k, din, dout = (case[a] for a in ("n", "K", "k", "din", "dout"))
    dt = st["x"].dtype
    ct = torch.float64 if dt == torch.float64 else torch.float32
    x, W = st["x"].detach(), st["weight"].detach()
    b = st["bias"].detach() if case["bias"] else None
    flat = st["labels"].reshape(-1)
    gates = st["gates"].detach().reshape(-1) if case["gated"] else None
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat + 1, minlength=K + 1).tolist()
    pair = torch.zeros(n * k, dout, dtype=ct, device=x.device)
    summed = case["gated"] or k == 1
    if case["backward"]:
        dy = st["dy"]
        dpair = torch.zeros(n * k, din, dtype=ct, device=x.device)
        dW, db = torch.zeros(K, din, dout, dtype=ct, device=x.device), torch.zeros(K, dout, dtype=ct, device=x.device)
        dg = torch.zeros(n * k, dtype=ct, device=x.device)
    at = counts[0]
    for e in range(K):
        rows = order[at:at + counts[e + 1]]
        at += counts[e + 1]
        if rows.numel() == 0:
            continue
        xe, We = x[rows // k].to(ct), W[e].to(ct)
        ye = xe @ We
        if b is not None:
            ye = ye + b[e].to(ct)
        pair[rows] = ye * gates[rows, None] if case["gated"] else ye
        if case["backward"]:
            de = (dy[rows // k] if summed else dy.reshape(-1, dout)[rows]).to(ct)
            if case["gated"]:
                dg[rows] = (de * ye).sum(1)
                de = de * gates[rows, None]
            dpair[rows] = de @ We.t()
            dW[e] = xe.t() @ de
            db[e] = de.sum(0)
    y = (pair.view(n, k, dout).sum(1) if summed else pair.view(n, k, dout)).to(dt)
    if not case["backward"]:
        return y
    out = [y, dpair.view(n, k, din).sum(1).to(dt), dW.to(dt)]
    if case["bias"]:
        out.append(db.to(dt))
    if case["gated"]:
        out.append(dg.view(st["gates"].shape))
    return out


def _plain_verify(st):
    p, q, z, ua, ud, ln = (st[a] for a in ("target", "draft", "labels", "u_accept", "u_draw", "lengths"))
    B, T, V = q.shape

    def clean(t):
        t = t.double()
        return torch.where((t > 0) & (t < math.inf), t, 0.0)
    zi = z.clamp(0, V - 1)[..., None]
    px, qx = clean(p[:, :T].gather(2, zi)[..., 0]), clean(q.gather(2, zi)[..., 0])
    t = torch.arange(T, device=z.device)
    ok = (ua * qx < px) & (z >= 0) & (z < V) & (t < ln[:, None])
    acc = torch.cumprod(ok.long(), 1).sum(1)
    rejected = acc < ln
    rows = torch.arange(B, device=z.device)
    pr = clean(p[rows, acc])
    w = torch.where(rejected[:, None], torch.clamp(pr - clean(q[rows, acc.clamp(max=T - 1)]), min=0), pr)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, pr)
    cum = torch.cumsum(w, 1)
    j = (cum <= ud[:, None] * cum[:, -1:]).sum(1)
    last = torch.where(w > 0, torch.arange(V, device=z.device), -1).max(1).values
    j = torch.minimum(j, last)
    t1 = torch.arange(T + 1, device=z.device)
    out = torch.where(t1 < acc[:, None], torch.cat([z, z.new_full((B, 1), -1)], 1), -1)
    out = torch.where(t1 == acc[:, None], j[:, None], out)
    return out, acc


def run(state):
    case = state["case"]
    if not own:
        return {"route": _plain_route, "products": _plain_products, "verify": _plain_verify}[case["op"]](state)
    from pybgmm_amd import ops
    if case["op"] == "route":
        labels, w = ops.route(state["log_weights"], case["k"], renormalise=case["renormalise"])
        if not case["backward"]:
            return labels, w
        return (labels, w.detach()) + torch.autograd.grad(w, state["log_weights"], state["dweights"])
    if case["op"] == "products":
        groups = ops.group_rows(state["labels"], case["K"])
        y = ops.grouped_matmul(state["x"], state["weight"], groups, bias=state["bias"], gates=state["gates"])
        if not case["backward"]:
            return y
        leaves = [t for t in (state["x"], state["weight"], state["bias"], state["gates"]) if t is not None]
        return [y.detach()] + list(torch.autograd.grad(y, leaves, state["dy"]))
    return ops.verify_drafts(state["target"], state["draft"], state["labels"], state["u_accept"], state["u_draw"], lengths=state["lengths"])


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_route(st):
    case = st["case"]
    lw = st["log_weights"].detach().double()
    lw = torch.where(torch.isnan(lw), -math.inf, lw)
    srt, at = torch.sort(lw, dim=1, descending=True, stable=True)
    k = case["k"]
    labels = torch.where(srt[:, :k] > -math.inf, at[:, :k], -1)
    del srt, at
    lw = torch.where((lw > -math.inf).any(1, keepdim=True), lw, 0.0)
    if case["renormalise"]:
        keep = torch.zeros_like(lw, dtype=torch.bool).scatter_(1, labels.clamp(min=0), True)
        soft = torch.softmax(torch.where(keep, lw, -math.inf), 1)
    else:
        soft = torch.softmax(lw, 1)
    w = torch.where(labels >= 0, soft.gather(1, labels.clamp(min=0)), 0.0)
    if not case["backward"]:
        return labels, w
    up = torch.zeros_like(soft).scatter_add_(1, labels.clamp(min=0), torch.where(labels >= 0, st["dweights"].double(), 0.0))
    up = soft * (up - (soft * up).sum(1, keepdim=True))
    return labels, w, torch.where((labels >= 0).any(1, keepdim=True), up, 0.0)


def _exact_products(st):
    """Component by component and choice by choice, each summed in 64 bits."""
    case = st["case"]
    n, K, k, din, dout = (case[a] for a in ("n", "K", "k", "din", "dout"))
    z = st["labels"].reshape(n, k)
    x, W = st["x"].detach(), st["weight"].detach()
    summed = case["gated"] or k == 1
    y = torch.zeros((n, dout) if summed else (n, k, dout), dtype=torch.float64, device=x.device)
    gates = st["gates"].detach().double().reshape(n, k) if case["gated"] else torch.ones(n, k, dtype=torch.float64, device=x.device)
    bw = case["backward"]
    if bw:
        dx, dg = torch.zeros(n, din, dtype=torch.float64, device=x.device), torch.zeros(n, k, dtype=torch.float64, device=x.device)
        dW, db = torch.zeros(K, din, dout, dtype=torch.float64, device=x.device), torch.zeros(K, dout, dtype=torch.float64, device=x.device)
    for e in range(K):
        We = W[e].double().contiguous()
        be = st["bias"].detach()[e].double() if case["bias"] else 0.0
        for j in range(k):
            i = torch.nonzero(z[:, j] == e)[:, 0]
            if i.numel() == 0:
                continue
            xe = x.index_select(0, i).double()
            out = torch.addmm(torch.zeros(1, dout, dtype=torch.float64, device=x.device), xe, We) + be
            gi = gates[i, j].unsqueeze(1)
            if summed:
                y.index_add_(0, i, gi * out)
            else:
                y[i, j] = out
            if bw:
                up = st["dy"].index_select(0, i).double() if summed else st["dy"][i, j].double()
                dg[i, j] = (up * out).sum(1)
                up = up * gi
                dx.index_add_(0, i, up @ We.t().contiguous())
                dW[e] += xe.t().contiguous() @ up
                db[e] += up.sum(0)
    if not bw:
        return y
    res = [y, dx, dW]
    if case["bias"]:
        res.append(db)
    if case["gated"]:
        res.append(dg.reshape(st["gates"].shape))
    return res


def _exact_verify(st):
    p, q, ln = st["target"], st["draft"], st["lengths"].tolist()
    z, ua, ud = st["labels"].cpu().numpy(), st["u_accept"].cpu().numpy(), st["u_draw"].cpu().numpy()
    B, T, V = q.shape
    at = st["labels"].clamp(0, V - 1).unsqueeze(2)
    px = p[:, :T].gather(2, at)[..., 0].double().cpu().numpy()
    qx = q.gather(2, at)[..., 0].double().cpu().numpy()
    out, acc = np.full((B, T + 1), -1, dtype=np.int64), np.zeros(B, dtype=np.int64)
    for b in range(B):
        a = 0
        while a < ln[b] and ua[b, a] * qx[b, a] < px[b, a]:
            out[b, a] = z[b, a]
            a += 1
        acc[b] = a
    rows, accd = torch.arange(B, device=p.device), torch.from_numpy(acc).to(p.device)
    pr = p[rows, accd].double().cpu().numpy()
    qr = q[rows, accd.clamp(max=T - 1)].double().cpu().numpy()
    for b in range(B):
        w = np.maximum(pr[b] - qr[b], 0.0) if acc[b] < ln[b] else pr[b]
        c = np.cumsum(w)
        if not c[-1] > 0:
            c = np.cumsum(pr[b])
        out[b, acc[b]] = min(int(np.searchsorted(c, ud[b] * c[-1], side="right")), int(np.searchsorted(c, c[-1], side="left")))
    return torch.from_numpy(out), torch.from_numpy(acc)


def exact(case, seed):
    st = prepare(case, seed)
    return {"route": _exact_route, "products": _exact_products, "verify": _exact_verify}[case["op"]](st)
