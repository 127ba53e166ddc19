"""Norm with its gradient, weighted routing, weighted experts: against plain implementations in 64 bits.

Tolerances count roundings: u = 2^-24 for every 32-bit step (times the number of steps that can add up, on
the sum of the magnitudes they act on) and one half step of the output's type, ``half`` relative to the value.
"""
import math

import pytest
import torch

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want))
    assert not bad.any(), (what, int(bad.sum()), (got - want).abs()[bad][:4], tol[bad][:4], want[bad][:4])


# -- norm ---------------------------------------------------------------------------------------
def norm_reference(x, w, b, eps, kind, offset, dy=None):
    """64-bit norm, its gradients, and the tolerances of a 32-bit evaluation of both."""
    xd, N, d = x.double(), x.shape[0], x.shape[1]
    mean = xd.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(xd[:, :1])
    rstd = 1.0 / torch.sqrt(((xd - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (xd - mean) * rstd
    wd = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double() + offset
    bd = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    y = xh * wd + bd
    # a row's sums: up to 32 values a thread, then ten steps of a tree; x - mean is off by the mean's share of that
    # (A, in units of the row's spread), xh by as much and by half the variance's
    A = xd.abs().amax(1, keepdim=True) * rstd
    e_xh = 64 * U * (xh.abs() + A)
    out = {"y": (y, half(x.dtype) * y.abs() + e_xh * wd.abs() + 4 * U * (y.abs() + bd.abs()))}
    out["stats"] = (mean[:, 0], rstd[:, 0], 64 * U * xd.abs().amax(1), 64 * U * rstd[:, 0] * (1 + A[:, 0] ** 2))
    if dy is None:
        return out
    gd = dy.double()
    g = gd * wd
    m0 = g.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(mean)
    m1 = (g * xh).mean(1, keepdim=True)
    dx = rstd * (g - m0 - xh * m1)
    G = g.abs().amax(1, keepdim=True)
    X = xh.abs().amax(1, keepdim=True)
    # (rstd itself is off by 64 U (1 + A^2) at most: x - mean may have lost that much)
    tol = half(x.dtype) * dx.abs() + 128 * U * rstd * (1 + A + A ** 2) * (G + G + X * X * G)
    out["dx"] = (dx, tol)
    pt = x.dtype if w is None else w.dtype
    dw, db = (gd * xh).sum(0), gd.sum(0)
    # column sums: rows of a thread, blocks and parts in turn, 128 steps at most at these sizes
    steps = 128 + N / 256
    out["dw"] = (dw, half(pt) * dw.abs() + steps * U * (gd * xh).abs().sum(0) + (gd.abs() * e_xh).sum(0) +
                 (gd.abs() * xh.abs() * 64 * U * (1 + A ** 2)).sum(0))
    out["db"] = (db, half(pt) * db.abs() + steps * U * gd.abs().sum(0))
    return out


NORM_CASES = [
    # N, d, dtype, params, kind, offset, row gap
    (1, 1, "fp32", "same", "layer", 0.0, 0), (1, 1, "bf16", "same", "rms", 1.0, 0),
    (3, 2, "fp32", "same", "rms", 0.0, 1), (5, 7, "bf16", "fp32", "layer", 0.0, 3),
    (257, 8, "bf16", "same", "layer", 0.0, 0), (1000, 33, "fp32", "same", "layer", 0.0, 0),
    (63, 64, "bf16", "fp32", "rms", 1.0, 64), (130, 96, "fp32", "same", "layer", 0.0, 4),
    (1, 768, "bf16", "same", "layer", 0.0, 0), (37, 768, "bf16", "fp32", "layer", 0.0, 0),
    (2500, 768, "bf16", "fp32", "layer", 0.0, 8), (700, 768, "fp32", "same", "rms", 0.0, 0),
    (9, 776, "bf16", "same", "layer", 0.0, 4), (300, 1000, "bf16", "same", "layer", 0.0, 1),
    (4099, 1023, "fp32", "same", "layer", 0.0, 9), (65, 2048, "bf16", "same", "rms", 1.0, 0),
    (601, 2048, "bf16", "fp32", "rms", 1.0, 0), (5, 4099, "bf16", "same", "layer", 0.0, 0),
    (17, 8192, "bf16", "same", "layer", 0.0, 0), (3, 8192, "fp32", "same", "rms", 0.0, 0),
    (2, 16384, "bf16", "fp32", "layer", 0.0, 0), (2, 16384, "fp32", "same", "layer", 0.0, 0),
    (3, 16381, "fp32", "same", "layer", 0.0, 0),
]


def norm_inputs(N, d, dtype, params, kind, gap, seed=0):
    g = gen(seed + 1000 * N + d)
    dt = DT[dtype]
    pt = dt if params == "same" else torch.float32
    wide = torch.full((N, d + gap), math.nan, dtype=dt, device="cuda")
    x = wide[:, :d]
    x.copy_(randn(g, N, d) * (0.5 + randn(g, d).abs()) + 0.5 * randn(g, N, 1))
    w = (1.0 + 0.3 * randn(g, d)).to(pt)
    b = (0.3 * randn(g, d)).to(pt) if kind == "layer" else None
    wide_g = torch.full((N, d + 2 * gap), math.nan, dtype=dt, device="cuda")
    dy = wide_g[:, :d]
    dy.copy_(randn(g, N, d))
    return x, w, b, dy


@pytest.mark.gpu
@pytest.mark.parametrize("case", NORM_CASES, ids=str)
def test_norm_and_its_gradients(case):
    import d2dmoe_b200 as D
    N, d, dtype, params, kind, offset, gap = case
    x, w, b, dy = norm_inputs(N, d, dtype, params, kind, gap)
    eps = 1e-5
    ref = norm_reference(x, w, b, eps, kind, offset, dy)
    y, mean, rstd = D.ops.layer_norm(x, w, b, eps, kind=kind, weight_offset=offset)
    within(y, *ref["y"], "y")
    m, r, tm, tr = ref["stats"]
    assert (mean is None) == (kind == "rms")
    if mean is not None:
        within(mean, m, tm, "mean")
    within(rstd, r, tr, "rstd")
    dx, dw, db = D.ops.layer_norm_backward(dy, x, w, mean, rstd, kind=kind, weight_offset=offset,
                                           bias=b is not None)
    within(dx, *ref["dx"], "dx")
    within(dw, *ref["dw"], "dw")
    assert (db is None) == (b is None) and dw.dtype == w.dtype and y.is_contiguous() and dx.is_contiguous()
    if db is not None:
        within(db, *ref["db"], "db")
    # the same bits again, and by autograd; outputs that are not wanted change nothing
    xg = x.detach().requires_grad_()
    leaves = [xg, w.requires_grad_()] + ([b.requires_grad_()] if b is not None else [])
    y2 = D.layer_norm(xg, w, b, eps, kind=kind, weight_offset=offset)
    assert torch.equal(y2, y)
    for a, c in zip(torch.autograd.grad(y2, leaves, dy), (dx, dw, db)):
        assert torch.equal(a, c)
    only, none, none2 = D.ops.layer_norm_backward(dy, x, w.detach(), mean, rstd, kind=kind, weight_offset=offset,
                                                  bias=False, dweight=False)
    assert torch.equal(only, dx) and none is None and none2 is None
    none, dw2, _ = D.ops.layer_norm_backward(dy, x, w.detach(), mean, rstd, kind=kind, weight_offset=offset,
                                             bias=False, dx=False)
    assert none is None and torch.equal(dw2, dw)


@pytest.mark.gpu
def test_norm_gradient_against_differences():
    """fp32 rows around points where central differences of the 64-bit forward pass are exact to about h^2."""
    import d2dmoe_b200 as D
    for kind in ("layer", "rms"):
        x, w, b, dy = norm_inputs(6, 24, "fp32", "same", kind, 0)
        y, mean, rstd = D.ops.layer_norm(x, w, b, 1e-5, kind=kind)
        dx, dw, _ = D.ops.layer_norm_backward(dy, x, w, mean, rstd, kind=kind, bias=False)
        h = 1e-4

        def loss(xx, ww):
            return (norm_reference(xx, ww, b, 1e-5, kind, 0.0)["y"][0] * dy.double()).sum()
        xd, wd = x.double(), w.double()
        for i in range(0, 6 * 24, 7):
            e = torch.zeros_like(xd).view(-1)
            e[i] = h
            e = e.view_as(xd)
            num = (loss(xd + e, wd) - loss(xd - e, wd)) / (2 * h)
            # h^2 times the third derivative (of order rstd^3 |g|), and the kernel's own rounding
            assert abs(num - dx.view(-1)[i].double()) <= 1e-4, (kind, i)
        for i in range(24):
            e = torch.zeros_like(wd)
            e[i] = h
            num = (loss(xd, wd + e) - loss(xd, wd - e)) / (2 * h)
            assert abs(num - dw[i].double()) <= 1e-4


@pytest.mark.gpu
def test_gradients_of_some_inputs_only():
    """What autograd does not ask for is left out; a second derivative is refused, not wrong."""
    import d2dmoe_b200 as D
    x, w, b, dy = norm_inputs(50, 96, "fp32", "same", "layer", 0)
    y, mean, rstd = D.ops.layer_norm(x, w, b)
    want = D.ops.layer_norm_backward(dy, x, w, mean, rstd)
    for mask in range(1, 8):
        ins = [t.detach().clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        D.layer_norm(*ins).backward(dy)
        for i, t in enumerate(ins):
            assert (t.grad is None) == (not mask >> i & 1)
            assert t.grad is None or torch.equal(t.grad, want[i])
    # a bias without a weight
    bb = b.detach().clone().requires_grad_()
    D.layer_norm(x, None, bb).backward(dy)
    within(bb.grad, dy.double().sum(0), 128 * U * dy.double().abs().sum(0), "bias alone")
    leaf = x.detach().clone().requires_grad_()
    g = torch.autograd.grad(D.layer_norm(leaf, w, b), leaf, dy.clone().requires_grad_(), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="first derivatives only"):
        g.sum().backward()
    leaf = x.detach().clone().requires_grad_()
    wt, e = D.route_tokens(leaf, 3)
    assert wt.requires_grad and not e.requires_grad
    g = torch.autograd.grad(wt, leaf, torch.ones_like(wt).requires_grad_(), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="first derivatives only"):
        g.sum().backward()
    with torch.no_grad():
        assert not D.layer_norm(leaf).requires_grad and not D.route_tokens(leaf, 3)[0].requires_grad
    for call in (lambda: D.layer_norm(leaf, eps=-1.0), lambda: D.route_tokens(leaf, 200),
                 lambda: D.route_tokens(leaf, 2, groups=5), lambda: D.route_tokens(leaf, 2, scale=-1.0)):
        with pytest.raises(D.ops._capi.D2DError):
            call()
    with pytest.raises(TypeError):
        D.layer_norm(leaf, w.bfloat16())
    with pytest.raises(ValueError):
        D.route_tokens(leaf, 2, bias=w[:3])


@pytest.mark.gpu
def test_norm_shapes_and_odd_values():
    import d2dmoe_b200 as D
    g = gen(3)
    # leading dimensions, a transposed (copied) input, an expanded row (stride 0), no parameters
    x = randn(g, 3, 5, 48)
    assert torch.equal(D.layer_norm(x), D.layer_norm(x.view(15, 48)).view(3, 5, 48))
    xt = randn(g, 48, 15).t()
    assert torch.equal(D.layer_norm(xt), D.layer_norm(xt.contiguous()))
    row = randn(g, 1, 48)
    assert torch.equal(D.layer_norm(row.expand(9, 48)), D.layer_norm(row.repeat(9, 1)))
    y, mean, rstd = D.ops.layer_norm(x)
    dx, dw, db = D.ops.layer_norm_backward(x, x, None, mean, rstd)
    ref = norm_reference(x.view(15, 48), None, None, 1e-5, "layer", 0.0, x.view(15, 48))
    within(dx.view(15, 48), *ref["dx"], "dx without a weight")
    within(dw, *ref["dw"], "dw without a weight")
    # a broadcast gradient (stride 0 everywhere)
    xs = x.view(15, 48).clone().requires_grad_()
    D.layer_norm(xs, torch.ones(48, device="cuda") * 2).sum().backward()
    ref = norm_reference(xs.detach(), torch.full((48,), 2.0, device="cuda"), None, 1e-5, "layer", 0.0,
                         torch.ones(15, 48, device="cuda"))
    within(xs.grad, *ref["dx"], "dx of a sum")
    # no rows: gradients of nothing are zero
    e = torch.empty(0, 48, device="cuda")
    y, mean, rstd = D.ops.layer_norm(e)
    dx, dw, db = D.ops.layer_norm_backward(e, e, torch.ones(48, device="cuda"), mean, rstd)
    assert y.shape == (0, 48) and dx.shape == (0, 48) and not dw.any() and not db.any()
    # constant rows have no spread; infinities and NaN stay in their rows
    x = randn(g, 6, 768)
    x[1] = 3.25
    x[3, 5] = math.inf
    x[4, 7] = math.nan
    w, b = randn(g, 768), randn(g, 768)
    y = D.layer_norm(x, w, b)
    assert torch.equal(y[1], b)
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all()
    ok = torch.tensor([0, 2, 5], device="cuda")
    within(y[ok], *[t[ok] for t in norm_reference(x, w, b, 1e-5, "layer", 0.0)["y"]], "rows beside them")
    # a large common offset: the spread is not lost (two passes over the row)
    x = randn(g, 8, 768) + 1000.0
    within(D.layer_norm(x), *norm_reference(x, None, None, 1e-5, "layer", 0.0)["y"], "offset")


# -- routing --------------------------------------------------------------------------------------
def route_reference(logits, k, scores="softmax", bias=None, groups=1, top_groups=None, renormalise=True, scale=1.0):
    """64-bit routing, row by row on the CPU: (weights, experts, scores)."""
    l = logits.double().cpu()
    N, E = l.shape
    b = torch.zeros(E, dtype=torch.float64) if bias is None else bias.double().cpu()
    top_groups = groups if top_groups is None else top_groups
    W, I = torch.zeros(N, k, dtype=torch.float64), torch.full((N, k), -1, dtype=torch.int32)
    S = torch.zeros(N, E, dtype=torch.float64)
    for t in range(N):
        row = l[t]
        if not (row <= 3.5e38).all() or not (b <= 3.5e38).all():
            W[t] = math.nan
            S[t] = math.nan
            continue
        s = torch.softmax(row, 0) if scores == "softmax" else torch.sigmoid(row)
        s = torch.nan_to_num(s, nan=0.0)
        S[t] = s
        free = row > -math.inf
        value = s if bias is None else s + b
        value = torch.where(free, value, torch.tensor(-math.inf, dtype=torch.float64))
        key = value if bias is not None else torch.where(free, row, value)
        if groups > 1:
            v = value.view(groups, -1).sort(dim=1, descending=True).values
            v = torch.where(v[:, 1] > -math.inf, v[:, 0] + v[:, 1], v[:, 0]) if v.shape[1] > 1 else v[:, 0]
            kept = v.sort(descending=True, stable=True).indices[:top_groups]
            drop = torch.ones(groups, dtype=torch.bool)
            drop[kept] = False
            key = key.view(groups, -1).masked_fill(drop[:, None], -math.inf).view(-1)
        order = key.sort(descending=True, stable=True).indices[:k]
        order = order[key[order] > -math.inf]
        n = order.numel()
        I[t, :n] = order.int()
        w = s[order]
        if renormalise and n:
            lw = row[order] if scores == "softmax" else torch.nn.functional.logsigmoid(row[order])
            w = torch.softmax(lw, 0)                     # the same, without underflow
        W[t, :n] = w * scale
    return W, I, S


def route_gradient(logits, dw, experts, scores, renormalise, scale):
    """64-bit gradient by autograd of the definition, the choice held fixed."""
    l = logits.double().cpu().requires_grad_()
    e = experts.cpu().long()
    there = e >= 0
    if renormalise:      # of the chosen logits alone: what the others add cancels, and would leave 64-bit rounding in its place
        c = l.gather(1, e.clamp(min=0)).masked_fill(~there, -math.inf)
        c = c if scores == "softmax" else torch.nn.functional.logsigmoid(c)
        w = torch.softmax(torch.where(there.any(1, keepdim=True), c, 0.0), 1) * there
    else:
        w = (torch.softmax(l, 1) if scores == "softmax" else torch.sigmoid(l)).gather(1, e.clamp(min=0)) * there
    (w * scale * dw.double().cpu()).sum().backward()
    return l.grad


def check_route(logits, k, dw=None, **how):
    import d2dmoe_b200 as D
    W, I, S = route_reference(logits, k, **how)
    scale = how.get("scale", 1.0)
    leaf = logits.detach().clone().requires_grad_(dw is not None)
    w, e = D.route_tokens(leaf, k, **how)
    assert e.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(e.cpu(), I)
    fin = torch.where(logits.float().isfinite(), logits.float(), torch.zeros_like(logits.float())).double().cpu()
    spread = (fin.amax(1) - fin.amin(1)).clamp(max=120.0)[:, None]
    # an exponential's argument is off by half an ulp (spread U), the exponentials, their sum (softmax over all: 64 steps
    # and the fast exponential's) and the quotients by 96 U more; below the normal numbers by their step
    rel = (96 + 4 * spread) * U
    within(w.detach().cpu(), W, rel * W.abs() + 2e-38 * scale, "weights")
    if dw is not None:
        how2 = {n: how[n] for n in ("scores", "renormalise", "scale") if n in how}
        how2 = dict(dict(scores="softmax", renormalise=True, scale=1.0), **how2)
        got = torch.autograd.grad(w, leaf, dw)[0].cpu()
        want = route_gradient(logits, dw, e, **how2)
        p = (W / scale).abs()
        g = dw.double().cpu().abs() * scale * (I >= 0)
        dot = (p * g).sum(1, keepdim=True)               # what cancels, per row
        size = torch.zeros_like(want).scatter_add_(1, I.clamp(min=0).long(), p * (g + dot))
        if how2["scores"] == "softmax" and not how2["renormalise"]:
            size = S * dot + size
        within(got, want, half(logits.dtype) * want.abs() + 4 * rel * size + 1e-37, "dlogits")
    return w.detach(), e


ROUTES = [
    # E, k, how
    (1, 1, dict()), (2, 2, dict(scores="sigmoid")), (7, 3, dict(renormalise=False)),
    (24, 4, dict()), (24, 9, dict(scores="sigmoid", bias=True)), (32, 8, dict(bias=True)),
    (33, 5, dict(scores="sigmoid", renormalise=False, scale=2.5)), (64, 6, dict(groups=8, top_groups=3)),
    (96, 4, dict(renormalise=False)), (96, 12, dict(groups=4, top_groups=2, bias=True, scores="sigmoid")),
    (128, 8, dict()), (128, 16, dict(bias=True, renormalise=False)), (130, 8, dict(groups=13, top_groups=4)),
    (256, 8, dict(scores="sigmoid", bias=True, groups=8, top_groups=4, scale=2.5)), (256, 8, dict()),
    (256, 16, dict(groups=32, top_groups=2, bias=True)), (500, 10, dict(scores="sigmoid")),
    (1024, 8, dict(bias=True)), (1023, 16, dict(renormalise=False)), (40, 32, dict(bias=True)),
    (1024, 32, dict(groups=32, top_groups=3, scores="sigmoid")), (6, 3, dict(groups=6, top_groups=3)),
    (24, 17, dict(scores="sigmoid", renormalise=False)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("route", ROUTES, ids=str)
def test_route_and_its_gradient(route, dtype):
    E, k, how = route
    how = dict(how)
    g = gen(E * 100 + k)
    bias = 0.1 * randn(g, E) if how.pop("bias", False) else None
    for N in (1, 37, 301):
        logits = (randn(g, N, E) * (1 + randn(g, N, 1).abs())).to(DT[dtype])
        check_route(logits, k, randn(g, N, k), bias=bias, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("how", [dict(), dict(bias=True), dict(scores="sigmoid", bias=True, groups=4, top_groups=2),
                                 dict(groups=4, top_groups=3, renormalise=False)], ids=str)
def test_route_near_and_exact_ties(how, dtype):
    """Equal logits, logits one step of their type apart, and scores + bias that 32 bits cannot tell apart."""
    how = dict(how)
    g = gen(11)
    E, k, N = 64, 8, 200
    bias = None
    base = torch.round(randn(g, N, E) * 2) / 2
    if how.pop("bias", False):
        bias = torch.round(randn(g, E) * 4) / 64
    logits = base.to(DT[dtype])
    logits[0] = 0.25                                     # all equal
    logits[1] = torch.finfo(DT[dtype]).min               # all the lowest: as equal as any
    check_route(logits, k, randn(g, N, k), bias=bias, **how)
    step = torch.nextafter(logits, torch.full_like(logits, 9.0))
    logits = torch.where(torch.rand(N, E, generator=g, device="cuda") < 0.5, logits, step)
    check_route(logits, k, bias=bias, **how)
    if bias is not None:                                 # biases that nearly level the scores
        row = randn(g, E)
        s = torch.softmax(row.double(), 0) if how.get("scores") != "sigmoid" else torch.sigmoid(row.double())
        check_route(row.to(DT[dtype]).expand(20, E).contiguous(), k, bias=(0.5 - s).float(), **how)
        check_route(logits, k, bias=bias + 1000.0, **how)
        far = bias.clone()
        far[::3] = -1e9
        check_route(logits, k, bias=far, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_route_rows_without_a_choice(dtype):
    g = gen(5)
    E, k, N = 48, 6, 40
    lo = torch.finfo(DT[dtype]).min
    logits = randn(g, N, E).to(DT[dtype])
    logits[0] = -math.inf                                # nothing left
    logits[1, 3:] = -math.inf                            # fewer than k
    logits[2, 1:] = lo                                   # masked by the lowest value: still there, with no weight
    logits[3, 4] = math.nan
    logits[4, 5] = math.inf
    logits[5, ::2] = -math.inf
    logits[6] = -1e4                                     # sigmoids underflow
    logits[7, :24] = -200.0
    logits[8, 8:] = -math.inf
    bias = 0.1 * randn(g, E)
    out = bias.clone()
    out[5:20] = -math.inf                                # experts that a bias takes out
    bad = bias.clone()
    bad[7] = math.nan
    for scores in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            for extra in (dict(), dict(bias=bias), dict(bias=out), dict(bias=bad), dict(groups=6, top_groups=2),
                          dict(bias=bias, groups=4, top_groups=3)):
                w, e = check_route(logits, k, scores=scores, renormalise=renormalise, **extra)
                if extra.get("bias") is not bad:
                    assert (e[0] == -1).all() and not w[0].any()
                    assert (e[3] == -1).all() and torch.isnan(w[3]).all() and torch.isnan(w[4]).all()
    import d2dmoe_b200 as D
    leaf = logits.clone().requires_grad_()
    for how in (dict(), dict(scores="sigmoid"), dict(renormalise=False)):
        w, e = D.route_tokens(leaf, k, **how)
        d = torch.autograd.grad(w, leaf, torch.ones_like(w))[0]
        assert not d[0].any() and not d[3].any() and torch.isfinite(d).all()


@pytest.mark.gpu
def test_route_bits_and_routing_tensor():
    """The optional outputs say the same as the lists, in the compaction's and the expert kernels' terms."""
    import d2dmoe_b200 as D
    for E, k, dtype, how in ((24, 4, "bf16", {}), (96, 12, "fp32", dict(groups=4, top_groups=2)), (128, 20, "bf16", {}),
                             (100, 8, "fp32", dict(scores="sigmoid", bias=True))):
        g = gen(E)
        how = dict(how)
        if how.pop("bias", False):
            how["bias"] = 0.1 * randn(g, E)
        N = 333
        logits = randn(g, N, E).to(DT[dtype])
        logits[4] = -math.inf
        logits[9, 1] = math.nan
        wsp = D.ops.Workspace.allocate(N, E, "cuda")
        w, e, rt = D.ops.route(logits, k, wsp=wsp, routing_tensor=True, **how)
        want = torch.zeros(N, E, device="cuda").to(DT[dtype])
        on = e >= 0
        t = torch.arange(N, device="cuda")[:, None].expand_as(e)
        want[t[on], e[on].long()] = w[on].to(DT[dtype])
        assert torch.equal(rt, want)
        kept = torch.zeros(N, E, device="cuda")
        kept[t[on], e[on].long()] = 1.0
        assert torch.equal(D.ops.expand_mask(wsp, N, E, torch.float32), kept)
        assert rt.dtype == DT[dtype] and (e[9] == -1).all()


# -- weighted experts ---------------------------------------------------------------------------------
ACTS = {"relu": torch.relu, "gelu": torch.nn.functional.gelu, "tanh": torch.tanh,
        "leaky_relu": torch.nn.functional.leaky_relu,
        "gelu_tanh": lambda h: torch.nn.functional.gelu(h, approximate="tanh")}


def experts_reference(x, e, w, w1, b1, w2, act, w_up=None, last_bias=None, residual=False):
    """64-bit weighted sum and the tolerance of the kernels' roundings."""
    E, d, H = w1.shape
    xd, out = x.double(), torch.zeros_like(x, dtype=torch.float64)
    rounded, size = torch.zeros_like(out), torch.zeros_like(out)
    for i in range(E):
        t, j = (e == i).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        xe, wt = xd[t], w[t, j].double()[:, None]
        pre, pre_abs = xe @ w1[i].double(), xe.abs() @ w1[i].double().abs()
        if b1 is not None:
            pre, pre_abs = pre + b1[i].double(), pre_abs + b1[i].double().abs()
        h, h_abs = ACTS[act](pre), 1.2 * pre_abs
        if w_up is not None:
            up = xe @ w_up[i].double()
            h, h_abs = h * up, h_abs * (xe.abs() @ w_up[i].double().abs())
        y = h @ w2[i].double()
        out.index_add_(0, t, y * wt)
        # half a step on every hidden value; 2^-14 of the largest of eight neighbours on every expert's output
        top = y.abs().view(-1, d // 8, 8).amax(2, keepdim=True).expand(-1, -1, 8).reshape(-1, d) if d % 8 == 0 else 0 * y
        rounded.index_add_(0, t, (h.abs() @ w2[i].double().abs() + 2.0 ** -6 * top) * wt.abs())
        size.index_add_(0, t, (h_abs @ w2[i].double().abs()) * wt.abs())
    for a in ([last_bias] if last_bias is not None else []) + ([xd] if residual else []):
        out, size = out + a.double(), size + a.double().abs()
    u = half(x.dtype) if x.dtype == torch.bfloat16 else 0.0
    # 32-bit sums of d, H and k terms (a gated product has two of d)
    return out, half(x.dtype) * out.abs() + u * rounded + (2 * d + H + e.shape[1] + 16) * U * size


def experts_case(N, d, E, H, k, dtype, glu, bias, seed=0):
    g = gen(seed + N + d)
    dt = DT[dtype]
    x = randn(g, N, d).to(dt)
    w1, w2 = (randn(g, E, d, H) / math.sqrt(d)).to(dt), (randn(g, E, H, d) / math.sqrt(H)).to(dt)
    up = (randn(g, E, d, H) / math.sqrt(d)).to(dt) if glu else None
    b1 = (0.3 * randn(g, E, H)).to(dt) if bias else None
    lb = (0.3 * randn(g, d)).to(dt) if bias else None
    top, e = (randn(g, N, E) + 0.7 * randn(g, E)).topk(k, dim=1)
    return x, e.int().contiguous(), torch.softmax(top, 1), w1, b1, w2, up, lb


EXPERTS = [
    # N, d, E, H, k, dtype, gated, biases, activation
    (1, 1, 1, 1, 1, "fp32", False, True, "relu"), (1, 768, 24, 128, 4, "bf16", False, True, "relu"),
    (1, 2048, 16, 128, 8, "bf16", True, False, "gelu"), (3, 130, 7, 20, 3, "bf16", False, True, "gelu"),
    (2, 100, 5, 33, 5, "fp32", True, False, "tanh"), (8, 768, 12, 32, 8, "bf16", False, True, "gelu_tanh"),
    (16, 768, 24, 128, 4, "bf16", False, True, "relu"), (17, 768, 24, 128, 4, "bf16", False, True, "relu"),
    (40, 768, 24, 128, 2, "fp32", False, True, "gelu"), (65, 130, 7, 20, 7, "bf16", False, True, "gelu"),
    (33, 2048, 16, 128, 8, "bf16", True, False, "gelu"), (129, 64, 3, 16, 3, "bf16", False, True, "leaky_relu"),
    (300, 256, 33, 48, 5, "bf16", False, False, "tanh"), (1000, 768, 96, 32, 4, "bf16", False, True, "relu"),
    (513, 768, 24, 128, 1, "bf16", False, True, "gelu"), (700, 200, 9, 40, 4, "fp32", True, False, "gelu"),
    (1100, 768, 12, 32, 12, "bf16", False, True, "gelu"), (1500, 512, 128, 128, 8, "bf16", True, False, "gelu_tanh"),
    (1400, 101, 200, 7, 32, "fp32", False, True, "relu"), (5000, 128, 24, 64, 4, "bf16", False, True, "relu"),
    # either side of the line between the two forms (2048 pairs, or the experts' bytes), lists of one chunk and of several
    (682, 64, 3, 16, 3, "bf16", False, True, "leaky_relu"), (683, 64, 3, 16, 3, "bf16", False, True, "leaky_relu"),
    (900, 130, 7, 20, 3, "bf16", False, True, "gelu"), (2049, 200, 2, 50, 1, "fp32", True, False, "tanh"),
    (36, 2048, 128, 128, 8, "bf16", True, False, "gelu"), (38, 2048, 128, 128, 8, "bf16", True, False, "gelu"),
    (66, 768, 24, 128, 4, "bf16", False, True, "relu"), (70, 768, 24, 128, 4, "bf16", False, True, "relu"),
    (700, 3008, 4, 300, 3, "bf16", False, True, "gelu"), (33000, 64, 120, 16, 8, "bf16", False, True, "relu"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", EXPERTS, ids=str)
def test_weighted_experts(case):
    import d2dmoe_b200 as D
    N, d, E, H, k, dtype, glu, biases, act = case
    x, e, w, w1, b1, w2, up, lb = experts_case(N, d, E, H, k, dtype, glu, biases)
    packed = D.ops.prepack_experts(w1, b1, w2, up)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for residual in (False, True):
        want, tol = experts_reference(x, e, w, w1, b1, w2, act, up, lb, residual)
        args = dict(w_up=up, last_bias=lb, add_residual=residual, status=status)
        got = D.ops.experts_weighted(x, e, w, w1, b1, w2, act, packed=packed, **args)
        within(got, want, tol, "packed")
        assert torch.equal(got, D.ops.experts_weighted(x, e, w, w1, b1, w2, act, packed=packed, **args))
        if packed is not None:
            within(D.ops.experts_weighted(x, e, w, w1, b1, w2, act, **args), want, tol, "unpacked")
    assert int(status.item()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 400])             # 30 pairs, 2400 pairs
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_weighted_experts_odd_choices(N, dtype):
    """Slots without an expert, tokens without any, the same expert in several slots, weights of zero, negative and NaN,
    experts that nobody wants and that do not exist, all tokens for one expert."""
    import d2dmoe_b200 as D
    x, e, w, w1, b1, w2, up, lb = experts_case(N, 128, 12, 32, 6, dtype, False, True, seed=9)
    packed = D.ops.prepack_experts(w1, b1, w2)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    e[0] = -1
    e[1, 2:] = -1
    e[2] = 3
    e[3, ::2] = e[3, 1::2]
    w[4] = torch.tensor([0.0, -2.0, 1e-3, 0.5, 7.0, 0.0], device="cuda")

    def run():
        return D.ops.experts_weighted(x, e, w, w1, b1, w2, "gelu", packed=packed, last_bias=lb, status=status)
    within(run(), *experts_reference(x, e, w, w1, b1, w2, "gelu", None, lb), "holes and doubles")
    assert torch.equal(run()[0], lb)                     # no expert: the bias alone, whatever the weights say
    w[0] = math.nan
    assert torch.equal(run()[0], lb)
    w[1, 0] = math.nan
    out = run()
    assert torch.isnan(out[1]).all() and not torch.isnan(out[2:]).any()
    w[0], w[1] = 0.2, 0.2
    w1[7] = math.nan                                     # weights of an expert that nobody wants
    if packed is not None:
        packed = D.ops.prepack_experts(w1, b1, w2)
    e[e == 7] = -1
    assert not torch.isnan(run()).any()
    e[:] = 5
    within(run(), *experts_reference(x, e, w, w1, b1, w2, "gelu", None, lb), "one expert")
    e[:] = -1
    assert torch.equal(run(), lb.expand_as(x))
    assert int(status.item()) == 0
    e[:, 0], e[:, 1] = 2, 12                             # one that does not exist: skipped and reported
    want = experts_reference(x, torch.where(e == 12, -1, e), w, w1, b1, w2, "gelu", None, lb)
    within(run(), *want, "out of range")
    assert int(status.item()) == 5                       # INDEX_RANGE
    status.zero_()
    e[:, 1] = -7
    within(run(), *want, "out of range")
    assert int(status.item()) == 5
    none = D.ops.experts_weighted(x[:0], e[:0], w[:0], w1, b1, w2, "gelu", packed=packed)
    assert none.shape == (0, 128)


@pytest.mark.gpu
def test_weighted_experts_sizes_and_infinities():
    """Outputs of very different sizes beside each other, tiny, huge and zero rows; infinities and NaN stay what they are
    in their own columns."""
    import d2dmoe_b200 as D
    x, e, w, w1, b1, w2, up, lb = experts_case(900, 128, 12, 32, 3, "bf16", False, True, seed=4)
    e[:, 0], e[:, 1], e[:, 2] = 0, 1, 2
    w2[0] *= torch.logspace(-30, 30, 128, device="cuda").to(w2.dtype)
    w2[1] *= 1e-36
    w2[2] = 0.0
    packed = D.ops.prepack_experts(w1, b1, w2)
    for k in (3, 1):
        got = D.ops.experts_weighted(x, e[:, :k].contiguous(), w[:, :k].contiguous(), w1, b1, w2, "relu", packed=packed)
        want, tol = experts_reference(x, e[:, :k], w[:, :k], w1, b1, w2, "relu")
        within(got, want, tol + 2e-38, "sizes")
    w2[3] = w2[4]
    w2[3, :, 5] = 3e38                                   # one column overflows
    packed = D.ops.prepack_experts(w1, b1, w2)
    e[:, 0], e[:, 1] = 3, 4
    x.abs_()
    w1[3].abs_().mul_(30)                                # sums of 32 terms of about 3e38 times 10
    packed = D.ops.prepack_experts(w1, b1, w2)
    got = D.ops.experts_weighted(x, e, w, w1, b1, w2, "relu", packed=packed)
    want, tol = experts_reference(x, e, w, w1, b1, w2, "relu")
    assert torch.isinf(got[:, 5]).all()
    keep = torch.arange(128, device="cuda") != 5
    # (beside it the eight columns are bf16 without their lowest bit: 2^-7)
    within(got[:, keep], want[:, keep], tol[:, keep] + 2.0 ** -7 * want[:, keep].abs().amax(), "beside an infinity")
    assert torch.isfinite(got[:, keep]).all()
    x[7, 3] = math.nan
    got2 = D.ops.experts_weighted(x, e, w, w1, b1, w2, "gelu", packed=packed)
    assert torch.isnan(got2[7]).all() and torch.isfinite(got2[8:, keep]).all()


@pytest.mark.gpu
def test_weighted_experts_strided_and_misaligned():
    import d2dmoe_b200 as D
    x, e, w, w1, b1, w2, up, lb = experts_case(600, 128, 12, 32, 4, "bf16", False, True, seed=2)
    packed = D.ops.prepack_experts(w1, b1, w2)
    want, tol = experts_reference(x, e, w, w1, b1, w2, "relu", None, lb)
    wide = torch.zeros(600, 140, dtype=x.dtype, device="cuda")
    wide[:, 3:131] = x
    off = torch.zeros(600 * 128 + 1, dtype=x.dtype, device="cuda")[1:].view(600, 128)
    off.copy_(x)
    ew = torch.full((600, 9), -1, dtype=torch.int32, device="cuda")
    ew[:, 2:6] = e
    lbo = torch.zeros(129, dtype=x.dtype, device="cuda")[1:]
    lbo.copy_(lb)
    for n in (600, 9):
        for xx, bias in ((wide[:, 3:131], lb), (off, lb), (x, lbo)):
            got = D.ops.experts_weighted(xx[:n], ew[:n, 2:6], w.t().contiguous().t()[:n], w1, b1, w2, "relu",
                                         packed=packed, last_bias=bias)
            within(got, want[:n], tol[:n], "strides")
    batch = D.ops.experts_weighted(x.view(4, 150, 128), e.view(4, 150, 4), w.view(4, 150, 4), w1, b1, w2, "relu",
                                   packed=packed, last_bias=lb)
    assert torch.equal(batch.view(600, 128), D.ops.experts_weighted(x, e, w, w1, b1, w2, "relu", packed=packed,
                                                                     last_bias=lb))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Buffers of more than 2^31 elements: rows at their ends against the references of those rows."""
    import d2dmoe_b200 as D
    g = gen(1)
    d, N = 2048, 1_100_000
    x = torch.empty(N, d, dtype=torch.bfloat16, device="cuda")
    for part in x.split(1 << 17):
        part.copy_(randn(g, *part.shape))
    w = 1 + 0.1 * randn(g, d)
    rows = torch.tensor([0, 1, 1_048_575, 1_048_576, N - 2, N - 1], device="cuda")
    ref = norm_reference(x[rows], w, None, 1e-5, "layer", 0.0, x[rows])
    y, mean, rstd = D.ops.layer_norm(x, w)
    within(y[rows], *ref["y"], "y")
    dx, dw, db = D.ops.layer_norm_backward(x, x, w, mean, rstd)
    within(dx[rows], *ref["dx"], "dx")
    # sum of x xh = sum of x^2 rstd - x mean rstd over the columns; N terms in blocks of a few thousand steps each
    total = torch.zeros(d, dtype=torch.float64, device="cuda")
    for i, part in enumerate(x.split(1 << 17)):
        at = slice(i << 17, (i << 17) + part.shape[0])
        total += (part.double() * (part.double() - mean[at, None]) * rstd[at, None]).sum(0)
    assert ((dw - total).abs() <= 1e-4 * total.abs() + 1.0).all()
    del x, y, dx
    N, E, k = 131_072, 128, 8
    x, e, wt, w1, b1, w2, up, lb = experts_case(N, 2048, E, 16, k, "bf16", False, False)
    packed = D.ops.prepack_experts(w1, b1, w2)
    out = D.ops.experts_weighted(x, e, wt, w1, b1, w2, "relu", packed=packed)
    rows = torch.tensor([0, 1, 65_535, 131_000, N - 1], device="cuda")
    within(out[rows], *experts_reference(x[rows], e[rows], wt[rows], w1, b1, w2, "relu"), "experts")
    del out, x
    N = 17_000_000
    logits = torch.empty(N, E, dtype=torch.bfloat16, device="cuda")
    for part in logits.split(1 << 20):
        part.copy_(randn(g, *part.shape))
    w, e, rt = D.ops.route(logits, 2, routing_tensor=True)
    dl = D.ops.route_backward(torch.ones_like(w), logits, e, w, scores="sigmoid")
    rows = torch.tensor([0, 16_777_215, 16_777_216, N - 1], device="cuda")
    W, I, _ = route_reference(logits[rows], 2)
    assert torch.equal(e[rows].cpu(), I)
    within(w[rows].cpu(), W, 1e-5 * W, "weights")
    assert torch.equal((rt[rows] > 0).nonzero()[:, 1].view(-1, 2).sort(1).values.cpu(), I.long().sort(1).values)
    want = route_gradient(logits[rows], torch.ones(4, 2), e[rows], "sigmoid", True, 1.0)
    # (the weights are softmax's here, any will do for the addresses: only where the gradient is not zero is compared)
    assert torch.equal((dl[rows] != 0).cpu() | (want == 0), torch.ones(4, E, dtype=torch.bool))


# -- together, as a layer runs them -----------------------------------------------------------------------
def weighted_layer(dtype="bf16", glu=False, d=256, E=24, H=64, k=4, residual=False, seed=1, **routing):
    import d2dmoe_b200 as D
    torch.manual_seed(seed)
    moe = D.MoeficationMoE("ffn", d, E, not glu, H, torch.nn.GELU, add_residual_connection=residual,
                           add_intermediate_gating=glu)
    moe.router = D.MoeficationRouter(d, E, width=64, depth=2, bias=False, activation="relu",
                                     output_activation="identity")
    moe = moe.to(DT[dtype]).cuda().eval()
    with torch.no_grad():
        for p in moe.parameters():
            p.copy_(torch.randn(p.shape, device="cuda") / math.sqrt(max(p.shape[-2:]) if p.dim() > 1 else 4))
    moe.forward_mode, moe.k, moe.routing = "weighted", k, D.Routing(**routing)
    return moe


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,glu,residual,shape,routing", [
    ("bf16", False, True, (3, 100), dict()), ("bf16", True, False, (1, 1), dict(scores="sigmoid")),
    ("fp32", False, False, (5, 7), dict(groups=4, top_groups=2, scale=2.0)),
    ("bf16", True, True, (2, 400), dict(bias=True, renormalise=False))], ids=str)
def test_layer_in_weighted_mode(dtype, glu, residual, shape, routing):
    """Norm, router, routing and weighted experts as one layer call: every stage from the one before it."""
    import d2dmoe_b200 as D
    routing = dict(routing)
    if routing.pop("bias", False):
        routing["bias"] = 0.1 * randn(gen(8), 24)
    moe = weighted_layer(dtype, glu, residual=residual, **routing)
    h = randn(gen(4), *shape, 256).to(DT[dtype])
    norm = torch.nn.LayerNorm(256).to(h)
    with torch.no_grad():
        norm.weight.uniform_(0.5, 1.5)
    x = D.layer_norm(h, norm.weight.detach(), norm.bias.detach(), norm.eps)
    out, gating = moe(x)
    rt = gating["ffn"][0]
    x2 = x.view(-1, 256)
    with torch.no_grad():
        logits = moe.router(x2)
    W, I, _ = route_reference(logits, 4, **routing)
    p = moe.experts.kernel_params()
    w, e = D.route_tokens(logits, 4, **routing)
    assert torch.equal(e.cpu(), I) and torch.equal(moe.gate(x), rt) and rt.shape == (*shape, 24)
    lb = moe.last_bias.detach().view(-1) if moe.bias else None
    want = experts_reference(x2, e, w, p["w1"].detach(), None if p["b1"] is None else p["b1"].detach(),
                             p["w2"].detach(), "gelu", None if p["w_up"] is None else p["w_up"].detach(), lb, residual)
    within(out.view(-1, 256).detach(), *want, "layer")
    dense = torch.zeros(x2.shape[0], 24, device="cuda").scatter(1, e.long(), w).to(rt.dtype)
    assert torch.equal(rt.view(-1, 24), dense) and not out.requires_grad
    block, _ = moe.forward_block(x, norm)
    with torch.no_grad():
        assert torch.equal(block, x + moe(norm(x))[0])
    host = moe.forward_host(x.cpu().pin_memory())
    # (slices of the batch: other sizes, so the few-pairs form may take them; the same bounds hold)
    within(host.view(-1, 256).cuda(), *want, "host buffers")
    moe.experts.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("glu", [False, True])
def test_weighted_call_follows_its_module(glu):
    """What a call keeps of its module is checked by the next one: new values, new storage, another activation, dropped
    packed weights, a copy of the module, another stream; and it refuses what it cannot serve."""
    import copy
    import d2dmoe_b200 as D
    ex = weighted_layer(glu=glu).experts
    for N in (6, 900):
        g = gen(N)
        x = randn(g, N, 256).bfloat16()
        w, e = D.route_tokens(randn(g, N, 24), 4)

        def check(what):
            p = {n: t.detach() if torch.is_tensor(t) else t for n, t in ex.kernel_params().items()}
            want = experts_reference(x, e, w, p["w1"], p["b1"], p["w2"], p["act"], p["w_up"])
            within(ex.forward_weighted(x, e, w), *want, what)
        check("first")
        first = ex.kernel_params()["w1"]
        with torch.no_grad():
            first.mul_(-1.0)
        check("values")
        if glu:
            ex.layers[1].w = torch.nn.Parameter(ex.layers[1].w.detach().flip(0).contiguous())
        else:
            ex.w2 = torch.nn.Parameter(ex.w2.detach().flip(0).contiguous())
        check("storage")
        ex.activation_str = "relu"
        check("activation")
        ex.activation_str = "gelu"
        first.data.mul_(2.0)
        ex.invalidate_packed()
        check("written past the version counter")
        other = copy.deepcopy(ex)
        assert torch.equal(other.forward_weighted(x, e, w), ex.forward_weighted(x, e, w))
        s = torch.cuda.Stream()
        with torch.no_grad():
            first.mul_(0.5)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            check("stream")
        torch.cuda.synchronize()
        with pytest.raises(TypeError):
            ex.forward_weighted(x.float(), e, w)
        with pytest.raises(ValueError):
            ex.forward_weighted(x[:, :128], e, w)
        with pytest.raises(RuntimeError, match="CUDA"):
            ex.forward_weighted(x.cpu(), e, w)
        with pytest.raises(RuntimeError, match="CUDA"):
            ex.forward_weighted(x, e.cpu(), w)
        assert not ex.forward_weighted(x.clone().requires_grad_(), e, w).requires_grad
    ex.capture_norms("output")
    with pytest.raises(NotImplementedError):
        ex.forward_weighted(x, e, w)


@pytest.mark.gpu
def test_routing_gradient_trains_a_router_of_dense_experts():
    """The weights' gradient through a mixture that torch computes: experts frozen, router and norm learn."""
    import d2dmoe_b200 as D
    g = gen(6)
    d, E, k, N = 48, 12, 3, 64
    h = randn(g, N, d)
    wr, gamma, beta = randn(g, E, d) / 7, 1 + 0.1 * randn(g, d), 0.1 * randn(g, d)
    we, target = randn(g, E, d, d) / 7, randn(g, N, d)

    def loss(norm, route, leaves):
        x = norm(h.to(leaves[0].dtype), leaves[1], leaves[2])
        logits = x @ leaves[0].t()
        w, e = route(logits)
        y = torch.einsum("nd,edf->nef", x.detach(), we.to(x.dtype))
        out = (y.gather(1, e.long()[:, :, None].expand(-1, -1, d)) * w[:, :, None]).sum(1)
        return (out - target.to(x.dtype)).square().mean(), e

    ours = [t.clone().requires_grad_() for t in (wr, gamma, beta)]
    a, e = loss(lambda x, w, b: D.layer_norm(x, w, b), lambda l: D.route_tokens(l, k), ours)
    ga = torch.autograd.grad(a, ours)
    ref = [t.double().requires_grad_() for t in (wr, gamma, beta)]
    b, _ = loss(lambda x, w, b: torch.nn.functional.layer_norm(x, (d,), w, b),
                lambda l: (torch.softmax(l.gather(1, e.long()), 1), e), ref)
    gb = torch.autograd.grad(b, ref)
    assert abs(a.double() - b) <= 1e-4 * b
    for u, v in zip(ga, gb):         # sums of about N E terms of 32-bit products: 2^-24 sqrt(N E d) of their size
        assert (u.double() - v).norm() <= 1e-4 * v.norm()


# -- streams, devices, graphs ----------------------------------------------------------------------------------
def step(x, w, b, dy, logits, dw, ex, xe):
    import d2dmoe_b200 as D
    y, mean, rstd = D.ops.layer_norm(x, w, b)
    g = D.ops.layer_norm_backward(dy, x, w, mean, rstd)
    wt, e, rt = D.ops.route(logits, 4, routing_tensor=True)
    dl = D.ops.route_backward(dw, logits, e, wt)
    out = ex.forward_weighted(xe, e, wt)
    return (y, *g, wt, e, rt, dl, out)


def step_inputs(N, seed):
    g = gen(seed)
    x, w, b, dy = norm_inputs(N, 256, "bf16", "fp32", "layer", 0, seed)
    return x, w, b, dy, randn(g, N, 24), randn(g, N, 4), randn(g, N, 256).bfloat16()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [8, 1500])
def test_operators_in_graphs_and_on_streams(N):
    """Two graphs of the same operators replayed in turn and beside each other, on new inputs; another stream beside
    both: workspaces are the calls' own."""
    ex = weighted_layer().experts
    ex.packed()
    ex._status_words()[torch.device("cuda", 0)]
    graphs = []
    for seed in (1, 2):
        *ins, xe = step_inputs(N, seed)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(*ins, ex, xe)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step(*ins, ex, xe)
        graphs.append((gr, (*ins, xe), outs))
    for turn in range(3):
        for i, (gr, ins, _) in enumerate(graphs):
            for a, c in zip(ins, step_inputs(N, 10 + 2 * turn + i)):
                a.copy_(c)
        side = [torch.cuda.Stream() for _ in range(3)]
        for s in side:
            s.wait_stream(torch.cuda.current_stream())
        for (gr, _, _), s in zip(graphs, side):
            with torch.cuda.stream(s):
                gr.replay()
        *mine, xe = step_inputs(N, 99)
        side[2].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side[2]):
            third = step(*mine, ex, xe)
        torch.cuda.synchronize()
        for _, ins, outs in graphs:
            for a, c in zip(outs, step(*ins[:-1], ex, ins[-1])):
                assert torch.equal(a, c)
        for a, c in zip(third, step(*mine, ex, xe)):
            assert torch.equal(a, c)
    ex.check_status()


@pytest.mark.gpu
def test_training_step_in_a_graph():
    """Forward and backward pass captured and replayed on new inputs.  (No eager graph of the same leaves is alive during
    the capture: torch ends any capture of a backward pass beside one, whatever operators it is made of.)"""
    import d2dmoe_b200 as D
    x, w, b, dy = norm_inputs(300, 256, "bf16", "fp32", "layer", 0)
    logits, dw = randn(gen(1), 300, 24), randn(gen(2), 300, 4)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, logits)]

    def grads():
        return torch.autograd.grad((D.layer_norm(*leaves[:3]), D.route_tokens(leaves[3], 4)[0]), leaves, (dy, dw))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        grads()
    torch.cuda.current_stream().wait_stream(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = grads()
    for seed in (1, 2):
        with torch.no_grad():
            for t, n in zip(leaves[:3], norm_inputs(300, 256, "bf16", "fp32", "layer", 0, seed)):
                t.copy_(n)
            leaves[3].copy_(randn(gen(10 + seed), 300, 24))
        gr.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, grads()):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_operators_do_not_synchronise():
    ex = weighted_layer().experts
    for N in (4, 1500):
        *ins, xe = step_inputs(N, 5)
        step(*ins, ex, xe)
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            step(*ins, ex, xe)
        finally:
            torch.cuda.set_sync_debug_mode("default")


@pytest.mark.gpu
def test_weighted_experts_give_up_on_a_withheld_tile():
    """A weight tile that never comes: the bounded wait runs out, the status says so, and the next call is whole."""
    import d2dmoe_b200 as D
    from d2dmoe_b200 import _capi
    x, e, w, w1, b1, w2, up, lb = experts_case(700, 128, 12, 32, 4, "bf16", False, True)
    packed = D.ops.prepack_experts(w1, b1, w2)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _capi.lib.d2d_debug_configure(10, 1)
    try:
        D.ops.experts_weighted(x, e, w, w1, b1, w2, "relu", packed=packed, status=status)
        torch.cuda.synchronize()
    finally:
        _capi.lib.d2d_debug_configure(0, 0)
    assert int(status.item()) == 6
    status.zero_()
    got = D.ops.experts_weighted(x, e, w, w1, b1, w2, "relu", packed=packed, last_bias=lb, status=status)
    within(got, *experts_reference(x, e, w, w1, b1, w2, "relu", None, lb), "after it")
    assert int(status.item()) == 0


# -- refusals ---------------------------------------------------------------------------------------------------
def test_refusals_at_the_c_abi():
    """Bad arguments are refused on the host before any launch (no pointer is dereferenced)."""
    import ctypes as C
    from d2dmoe_b200 import _capi
    lib, a, n = _capi.lib, C.c_void_p(0x7f0000000000), C.c_size_t(0)
    odd = C.c_void_p(0x7f0000000001)
    OKAY, BAD, UNS, WS = 0, 1, 2, 4

    def norm(x=a, xs=8, eps=1e-5, kind=0, y=a, N=4, d=8, dt=1, pt=1):
        return lib.d2d_layer_norm(x, xs, None, None, eps, kind, 0.0, y, None, None, N, d, dt, pt, None)
    assert norm(N=0) == OKAY
    for kw in (dict(x=None), dict(y=None), dict(N=-1), dict(d=0), dict(xs=-1), dict(eps=-1.0), dict(eps=math.nan),
               dict(kind=2), dict(kind=-1)):
        assert norm(**kw) == BAD, kw
    for kw in (dict(dt=2), dict(dt=0, pt=1), dict(pt=3), dict(d=16385)):
        assert norm(**kw) == UNS, kw
    assert lib.d2d_layer_norm_workspace_bytes(1000, 768, C.byref(n)) == OKAY and n.value >= 296 * 2 * 768 * 4
    need = n.value
    assert lib.d2d_layer_norm_workspace_bytes(-1, 768, C.byref(n)) == BAD
    assert lib.d2d_layer_norm_workspace_bytes(1, 0, C.byref(n)) == BAD

    def back(dy=a, x=a, kind=0, mean=a, rstd=a, dx=a, dg=a, db=a, N=1000, d=768, dt=1, pt=0, ws=a, nb=need, st=768):
        return lib.d2d_layer_norm_backward(dy, st, x, st, None, kind, 0.0, mean, rstd, dx, dg, db, N, d, dt, pt, ws, nb, None)
    assert back(dx=None, dg=None, db=None) == OKAY
    for kw in (dict(dy=None), dict(x=None), dict(rstd=None), dict(mean=None), dict(kind=5), dict(N=-1), dict(ws=None),
               dict(ws=odd), dict(st=-768)):
        assert back(**kw) == BAD, kw
    assert back(nb=256) == WS and back(d=16385) == UNS and back(dt=0, pt=1) == UNS

    def route(l=a, scores=0, k=4, g=1, tg=1, scale=1.0, e=a, w=a, N=4, E=24, dt=1):
        return lib.d2d_route(l, None, scores, k, g, tg, 1, scale, e, w, None, None, N, E, dt, None)
    assert route(N=0) == OKAY
    for kw in (dict(l=None), dict(e=None), dict(w=None), dict(scores=2), dict(k=0), dict(k=25), dict(g=0), dict(g=5),
               dict(g=4, tg=0), dict(g=4, tg=5), dict(g=8, tg=1, k=4), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=math.nan), dict(scale=math.inf), dict(N=-1), dict(E=0)):
        assert route(**kw) == BAD, kw
    for kw in (dict(dt=7), dict(E=1025), dict(E=64, k=33), dict(E=66, g=33, tg=33)):
        assert route(**kw) == UNS, kw

    def rback(l=a, d=a, scores=0, k=4, scale=1.0, N=4, E=24, dt=1):
        return lib.d2d_route_backward(l, a, a, a, scores, 1, scale, d, N, E, k, dt, None)
    assert rback(N=0) == OKAY
    for kw in (dict(l=None), dict(d=None), dict(scores=3), dict(k=0), dict(k=25), dict(scale=0.0), dict(N=-1)):
        assert rback(**kw) == BAD, kw
    assert rback(E=1025) == UNS and rback(E=64, k=33) == UNS and rback(dt=2) == UNS

    def ws_bytes(N=4000, d=128, E=12, H=32, k=4, glu=0, packed=0, dt=1):
        rc = lib.d2d_experts_weighted_workspace_bytes(N, d, E, H, k, glu, packed, dt, C.byref(n))
        return rc if rc else n.value
    need = ws_bytes()
    assert need >= 4000 * 4 * 128 * 4 > ws_bytes(packed=1) >= 4000 * 4 * 128 * 2 and ws_bytes(N=0) >= 0
    assert ws_bytes(N=-1) == BAD and ws_bytes(k=13) == BAD and ws_bytes(dt=9) == UNS

    def experts(x=a, e=a, w=a, w1=a, w2=a, out=a, res=0, N=4000, d=128, E=12, H=32, k=4, act=0, dt=1, ws=a, nb=None):
        return lib.d2d_experts_weighted(x, e, w, w1, None, None, w2, None, None, res, out, N, d, E, H, k, act, dt, ws,
                                        need if nb is None else nb, None, None)
    assert experts(N=0) == OKAY
    for kw in (dict(x=None), dict(e=None), dict(w=None), dict(w1=None), dict(w2=None), dict(out=None), dict(res=2),
               dict(N=-1), dict(d=0), dict(H=0), dict(k=0), dict(k=13), dict(ws=None), dict(ws=odd), dict(x=odd),
               dict(e=odd), dict(out=odd)):
        assert experts(**kw) == BAD, kw
    for kw in (dict(act=9), dict(act=-1), dict(dt=2), dict(E=300, k=4), dict(E=64, k=33), dict(H=4000),
               dict(N=1 << 30, k=4)):
        assert experts(**kw) == UNS, kw
    assert experts(nb=need - 256) == WS


def test_cpu_tensors_are_refused():
    import d2dmoe_b200 as D
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.layer_norm(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.route_tokens(x, 2)
    with pytest.raises(ValueError):
        D.layer_norm(x, kind="batch")
    with pytest.raises(ValueError):
        D.route_tokens(x, 2, scores="relu")
    ex = D.B200KernelExperts(8, 4, expert_dim=4, bias="without_last", activation=torch.nn.ReLU)
    with pytest.raises(RuntimeError, match="CUDA"):
        ex.forward_weighted(x, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2))


@pytest.mark.gpu
def test_refusals_of_tensors():
    import d2dmoe_b200 as D
    c = dict(device="cuda")
    x, w = torch.zeros(4, 8, **c), torch.zeros(8, **c)
    h = x.half()
    i = torch.zeros(4, 2, dtype=torch.int32, **c)
    wt = torch.zeros(4, 2, **c)
    w1, w2 = torch.zeros(3, 8, 4, **c), torch.zeros(3, 4, 8, **c)
    st = torch.zeros(4, **c)
    bad = [
        (TypeError, lambda: D.layer_norm(h)), (TypeError, lambda: D.layer_norm(x, w.bfloat16())),
        (TypeError, lambda: D.layer_norm(x.bfloat16(), w, w.bfloat16())),
        (ValueError, lambda: D.layer_norm(x, w[:7])), (ValueError, lambda: D.layer_norm(x, w.view(1, 8))),
        (RuntimeError, lambda: D.layer_norm(x, w.cpu())), (ValueError, lambda: D.layer_norm(x[:, :0])),
        (D.ops._capi.D2DError, lambda: D.layer_norm(x, w, eps=-1.0)),
        (D.ops._capi.D2DError, lambda: D.layer_norm(torch.zeros(1, 16385, **c))),
        (TypeError, lambda: D.ops.layer_norm_backward(x.bfloat16(), x, w, st, st)),
        (ValueError, lambda: D.ops.layer_norm_backward(x[:3], x, w, st, st)),
        (ValueError, lambda: D.ops.layer_norm_backward(x, x, w, st[:3], st)),
        (ValueError, lambda: D.ops.layer_norm_backward(x, x, w, None, st)),
        (TypeError, lambda: D.ops.layer_norm_backward(x, x, w, st, None)),
        (TypeError, lambda: D.route_tokens(h, 2)), (TypeError, lambda: D.route_tokens(x, 2, bias=w.bfloat16())),
        (ValueError, lambda: D.route_tokens(x, 2, bias=w[:5])),
        (D.ops._capi.D2DError, lambda: D.route_tokens(x, 0)), (D.ops._capi.D2DError, lambda: D.route_tokens(x, 9)),
        (D.ops._capi.D2DError, lambda: D.route_tokens(x, 2, groups=3)),
        (D.ops._capi.D2DError, lambda: D.route_tokens(x, 5, groups=2, top_groups=1)),
        (D.ops._capi.D2DError, lambda: D.route_tokens(x, 2, scale=0.0)),
        (ValueError, lambda: D.ops.route(x, 2, wsp=D.ops.Workspace.allocate(4, 9, "cuda"))),
        (ValueError, lambda: D.ops.route(x, 2, wsp=D.ops.Workspace.allocate(2, 8, "cuda"))),
        (TypeError, lambda: D.ops.route_backward(wt, x, i.long(), wt)),
        (ValueError, lambda: D.ops.route_backward(wt[:, :1], x, i, wt)),
        (TypeError, lambda: D.ops.route_backward(wt.bfloat16(), x, i, wt)),
        (TypeError, lambda: D.ops.experts_weighted(x, i.long(), wt, w1, None, w2, "relu")),
        (TypeError, lambda: D.ops.experts_weighted(x, i, wt.bfloat16(), w1, None, w2, "relu")),
        (TypeError, lambda: D.ops.experts_weighted(x, i, wt, w1.bfloat16(), None, w2, "relu")),
        (ValueError, lambda: D.ops.experts_weighted(x, i[:3], wt, w1, None, w2, "relu")),
        (ValueError, lambda: D.ops.experts_weighted(x, i, wt[:, :1], w1, None, w2, "relu")),
        (ValueError, lambda: D.ops.experts_weighted(x[:, :7], i, wt, w1, None, w2, "relu")),
        (ValueError, lambda: D.ops.experts_weighted(x, i, wt, w1, None, w2[:2], "relu")),
        (ValueError, lambda: D.ops.experts_weighted(x, i, wt, w1, None, w2, "relu", packed=torch.zeros(8, **c))),
        (ValueError, lambda: D.ops.experts_weighted(x, i, wt, w1, None, w2, "relu", last_bias=w[:3])),
        (KeyError, lambda: D.ops.experts_weighted(x, i, wt, w1, None, w2, "sigmoid")),
        (D.ops._capi.D2DError, lambda: D.ops.experts_weighted(x, torch.cat([i, i], 1), torch.cat([wt, wt], 1), w1,
                                                              None, w2, "relu")),
    ]
    for n, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {n} was not refused")
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_second_derivatives_are_refused_for_plain_incoming_gradients():
    """y's gradient does not require one itself: the second derivative in x is there all the same."""
    import d2dmoe_b200 as D
    x, w, b, dy = norm_inputs(20, 96, "fp32", "same", "layer", 0)
    leaf = x.detach().clone().requires_grad_()
    for y in (D.layer_norm(leaf, w, b), D.route_tokens(leaf, 3)[0]):
        g, = torch.autograd.grad(y, leaf, torch.ones_like(y), create_graph=True)
        with pytest.raises(RuntimeError, match="first derivatives only"):
            (g.square().sum() + y.sum()).backward()


@pytest.mark.gpu
def test_weighted_status_word_is_checked():
    import d2dmoe_b200 as D
    g = gen(5)
    x, e, w = randn(g, 3, 64), torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, 1, device="cuda")
    w1, w2 = randn(g, 2, 64, 32), randn(g, 2, 32, 64)
    for status, error in ((torch.zeros(1, dtype=torch.int64, device="cuda"), TypeError),
                          (torch.zeros(0, dtype=torch.int32, device="cuda"), ValueError)):
        with pytest.raises(error, match="status"):
            D.ops.experts_weighted(x, e, w, w1, None, w2, "relu", status=status)


@pytest.mark.gpu
def test_weighted_layouts_are_not_made_in_a_capture():
    """The first call, and the first after the weights changed, lay out what later calls read: refused in a capture,
    and right afterwards."""
    import copy
    ex = weighted_layer().experts
    g = gen(6)
    x, w = randn(g, 700, 256).bfloat16(), torch.rand(700, 4, device="cuda")
    e = torch.randint(0, 24, (700, 4), device="cuda", dtype=torch.int32)

    def refused():
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                ex.forward_weighted(x, e, w)

    refused()
    before = ex.forward_weighted(x, e, w)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = ex.forward_weighted(x, e, w)
    gr.replay()
    assert torch.equal(out, before)
    with torch.no_grad():
        ex.w2.mul_(2.0)
    refused()
    with torch.no_grad():
        fresh = copy.deepcopy(ex).forward_weighted(x, e, w)
    assert torch.equal(ex.forward_weighted(x, e, w), fresh) and not torch.equal(fresh, before)
    ex.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    # N, d, E, H, k, biases: items of one CTA, of two and of four; one slice of hidden columns and sixteen, the last one
    # of four columns; one chunk of d and several; fewer 64-column blocks than CTAs; more items than run at a time
    (550, 768, 24, 128, 4, True), (1200, 768, 24, 128, 4, True), (3200, 768, 24, 128, 4, False),
    (2100, 68, 1, 100, 1, True), (2060, 64, 3, 160, 1, True), (1100, 4, 5, 36, 2, True), (2100, 132, 7, 512, 1, False),
    (2100, 36, 3, 4, 1, True), (3400, 68, 200, 64, 1, True), (2100, 200, 9, 516, 1, True),
    # the line between the two forms of few pairs and of lists
    (108, 768, 24, 128, 4, True), (116, 768, 24, 128, 4, True)], ids=str)
def test_weighted_experts_fp32_forms(case):
    import d2dmoe_b200 as D
    N, d, E, H, k, biases = case
    x, e, w, w1, b1, w2, _, lb = experts_case(N, d, E, H, k, "fp32", False, biases)
    if E == 200:         # 17 each: two items where one is expected and a half
        e = (torch.arange(N, device="cuda") % E).int().view(N, 1)
    e[3] = -1
    if k > 1:
        e[5] = e[5, 0]                                   # one expert several times
        e[::7, 1] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for act in ("relu", "gelu"):
        want, tol = experts_reference(x, e, w, w1, b1, w2, act, None, lb, act == "relu")
        args = dict(last_bias=lb, add_residual=act == "relu", status=status)
        got = D.ops.experts_weighted(x, e, w, w1, b1, w2, act, **args)
        within(got, want, tol, act)
        for _ in range(3):
            assert torch.equal(got, D.ops.experts_weighted(x, e, w, w1, b1, w2, act, **args))
        # weights that start anywhere
        off = torch.zeros(w1.numel() + 1, device="cuda")[1:].view(w1.shape)
        off.copy_(w1)
        within(D.ops.experts_weighted(x, e, w, off, b1, w2, act, **args), want, tol, "misaligned weights")
    assert int(status.item()) == 0
