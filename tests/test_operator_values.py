"""Norm, routing and weighted experts on values and calls where a plain implementation is easily right: rows in their
16-bit form, zeros of both signs, NaN through an activation, biases that cancel, rows wider than 2^16, tangents, streams."""
import math

import pytest
import torch

from test_operators import (ACTS, DT, U, check_route, experts_case, experts_reference, gen, half, norm_inputs,
                            norm_reference, randn, route_gradient, route_reference, weighted_layer, within)


# -- rows of pairs ------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("glu", [False, True])
def test_rows_of_pairs_keep_their_size(glu):
    """One expert per token, weight 1, hidden values that bf16 holds: what the 16-bit row of a pair loses is all that is
    lost, and last_bias takes the output's upper bits away, so that its own rounding does not hide it."""
    import d2dmoe_b200 as D
    N, d, E, H = 2100, 128, 24, 64
    g = gen(3)
    w1, w2 = randn(g, E, d, H).bfloat16(), randn(g, E, H, d).bfloat16()
    up = torch.exp2(torch.randint(-2, 3, (E, d, H), generator=g, device="cuda").float()).bfloat16() if glu else None
    packed = D.ops.prepack_experts(w1, None, w2, up)
    assert packed is not None
    ones = torch.ones(N, 1, device="cuda")
    along = size = 0.0
    for e in range(E):
        x = torch.zeros(N, d, dtype=torch.bfloat16, device="cuda")
        x[:, 5 * e] = 1.0
        h = torch.relu(w1[e, 5 * e]).double()
        if glu:
            h = h * up[e, 5 * e].double()                # (powers of two: still exact)
        y = h @ w2[e].double()
        lb = -y.bfloat16()
        got = D.ops.experts_weighted(x, torch.full((N, 1), e, dtype=torch.int32, device="cuda"), ones, w1, None, w2,
                                     "relu", w_up=up, packed=packed, last_bias=lb).double()
        want = y + lb.double()
        top = y.abs().view(-1, 8).amax(1, keepdim=True).expand(-1, 8).reshape(-1)
        # half a unit of the row, 2^-14 (1 + 2^-14) of the largest of eight; 32-bit sums of H terms; half a step of the output
        tol = (2.0 ** -14 * (1 + 2.0 ** -14) * top + (2 * H + 16) * U * (h @ w2[e].double().abs()) +
               half(torch.bfloat16) * want.abs())
        within(got, want.expand_as(got), tol.expand_as(got), e)
        along += float(((got[0] - want) * y).sum())
        size += float((y * y).sum())
    # E d errors of at most 2^-14 of about twice the value, either way: 2^-13 / sqrt(3 E d) = 1.3e-6 of the whole
    assert abs(along / size) <= 1e-5


# -- zeros of both signs ------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("E,k", [(2, 1), (7, 3), (24, 1), (24, 8), (24, 4), (64, 16), (96, 12), (128, 8), (130, 8),
                                 (256, 8), (1023, 16), (1024, 8), (40, 17)])
def test_route_between_zeros_of_both_signs(E, k, dtype):
    """-0 and +0 are equal: the lowest index is taken."""
    g = gen(E + k)
    N = 150
    kind = torch.rand(N, E, generator=g, device="cuda")
    size = randn(g, N, E).abs() + 0.1
    zero = torch.where(torch.rand(N, E, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    size[:20] *= 2.0 ** -128                             # numbers below the normal ones beside the zeros
    # fewer than k above the zeros, the others among them
    logits = torch.where(kind < 0.4 * k / E, size, torch.where(kind < 0.9, zero, -size)).to(DT[dtype])
    assert (torch.signbit(logits) & (logits == 0)).any()
    for how in (dict(), dict(scores="sigmoid"), dict(renormalise=False)):
        check_route(logits, k, randn(g, N, k), **how)
    if E % 4 == 0 and k <= E // 2:
        check_route(logits, k, groups=4, top_groups=2)
        check_route(logits, k, groups=4, top_groups=3, scores="sigmoid", renormalise=False)


# -- NaN and the activations ----------------------------------------------------------------------------
# N x 3 pairs; packed; weights off a 16-byte boundary: few pairs, lists on the tensor cores, lists of the general kernel, fp32 lists
FORMS = [("bf16", 5, True, False, False), ("bf16", 900, True, False, False), ("bf16", 900, False, False, False),
         ("bf16", 5, True, True, False), ("bf16", 900, True, True, False), ("fp32", 5, False, False, False),
         ("fp32", 900, False, False, False), ("fp32", 900, False, False, True), ("fp32", 900, False, True, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_a_nan_stays_one_through_every_activation(form, act):
    import d2dmoe_b200 as D
    dtype, N, pack, glu, off = form
    x, e, w, w1, b1, w2, up, _ = experts_case(N, 128, 12, 32, 3, dtype, glu, not glu, seed=7)
    x[2, 7] = math.nan
    if off:
        far = torch.zeros(w1.numel() + 1, dtype=w1.dtype, device="cuda")[1:].view(w1.shape)
        w1 = far.copy_(w1)
    packed = D.ops.prepack_experts(w1, b1, w2, up) if pack else None
    assert (packed is not None) == pack
    got = D.ops.experts_weighted(x, e, w, w1, b1, w2, act, w_up=up, packed=packed)
    want, tol = experts_reference(x, e, w, w1, b1, w2, act, up)
    assert torch.isnan(want[2]).all() and torch.isnan(got[2]).all()
    keep = torch.arange(N, device="cuda") != 2
    assert torch.isfinite(got[keep]).all()
    within(got[keep], want[keep], tol[keep], "other rows")


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 150, 900])
@pytest.mark.parametrize("dtype,d,H", [("bf16", 128, 32), ("bf16", 100, 20), ("fp32", 128, 32), ("fp32", 102, 33)])
def test_a_nan_stays_one_through_the_unweighted_layer(dtype, d, H, N):
    import d2dmoe_b200 as D
    moe = D.MoeficationMoE("ffn", d, 12, True, H, torch.nn.ReLU).to(DT[dtype]).cuda().eval()
    with torch.no_grad():
        for p in moe.parameters():
            p.copy_(randn(gen(p.numel()), *p.shape) / 8)
    x = randn(gen(N), 1, N, d).to(DT[dtype])
    x[0, 2, 7] = math.nan
    out = moe(x)[0].detach()                             # every expert on every token
    assert torch.isnan(out[0, 2]).all()
    out[0, 2] = 0.0
    assert torch.isfinite(out).all()


# -- a token whose logits are NaN, in the layer -----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,glu", [("bf16", False), ("bf16", True), ("fp32", False)])
@pytest.mark.parametrize("N", [3, 900])
def test_a_token_without_usable_logits_shows_in_the_layers_output(N, dtype, glu):
    """Its weights are NaN, and so is its row; a token that no expert is allowed for has the bias."""
    moe = weighted_layer(dtype, glu)
    bad = torch.zeros(24, device="cuda", dtype=DT[dtype])

    class Router(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, x):
            s = self.inner(x)
            s[0, 1, 3], s[0, 2, 4] = math.nan, math.inf
            s[0, 0] = -math.inf
            return s + bad
    x = randn(gen(2), 1, N, 256).to(DT[dtype])
    with torch.no_grad():
        moe.router = Router(moe.router)
        out, gating = moe(x)
        lb = moe.last_bias.view(-1) if moe.bias else torch.zeros(256, device="cuda", dtype=DT[dtype])
        assert torch.isnan(out[0, 1:3]).all() and torch.equal(out[0, 0], lb)
        assert torch.isfinite(out[0, 3:]).all() and not gating["ffn"][0][0, :3].any()
        other = x.clone()
        other[0, :3] = 0.5
        assert torch.equal(moe(other)[0][0, 3:], out[0, 3:])
    moe.experts.check_status()


# -- groups whose two best cancel --------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_groups_whose_scores_and_biases_cancel(scores, dtype):
    """A group counts as the sum of its two best score + bias, whose size says nothing about their roundings."""
    g = gen(21)
    logits = randn(g, 300, 16).to(DT[dtype])
    for big in (3.0, 1000.0, 30000.0):
        # (the larger c of the groups lie apart and within 4 of each other: only the groups are in question)
        bias = torch.empty(16, device="cuda")
        bias[0::2] = big + 0.4 * torch.randperm(8, generator=g, device="cuda")
        bias[1::2] = -bias[0::2]
        check_route(logits, 3, bias=bias, groups=8, top_groups=3, scores=scores)
        bias[5] = bias[8] = -1e9                         # groups far behind
        check_route(logits, 3, bias=bias, groups=8, top_groups=3, scores=scores)
    # sums that 32 bits do not hold, and cannot order
    for sign in (1.0, -1.0):
        bias = sign * 2e38 * (1 + 0.05 * torch.randperm(8, generator=g, device="cuda").float()).repeat_interleave(2)
        check_route(logits, 4, bias=bias, groups=8, top_groups=3, scores=scores)


# -- forward mode -------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_tangents_are_refused():
    """No operator has a forward-mode derivative; a result without its tangent would be wrong without a word."""
    import torch.autograd.forward_ad as fw
    import d2dmoe_b200 as D
    g = gen(9)
    x, w, b = randn(g, 20, 48), 1 + randn(g, 48), randn(g, 48)
    ex = weighted_layer(d=256).experts
    h = randn(g, 20, 256).bfloat16()
    wt, e = D.route_tokens(randn(g, 20, 24), 4)
    y, mean, rstd = D.ops.layer_norm(x, w, b)
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))
        calls = [lambda: D.layer_norm(dual(x), w, b), lambda: D.layer_norm(x, dual(w), b),
                 lambda: D.layer_norm(x, w, dual(b)), lambda: D.layer_norm(dual(x.requires_grad_()), w, b),
                 lambda: D.ops.layer_norm_backward(dual(y), x.detach(), w, mean, rstd),
                 lambda: D.route_tokens(dual(x), 3), lambda: D.route_tokens(x, 3, bias=dual(b)),
                 lambda: ex.forward_weighted(dual(h), e, wt), lambda: ex.forward_weighted(h, e, dual(wt))]
        for n, call in enumerate(calls):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
                pytest.fail(f"call {n} dropped its tangent")
    ex.forward_weighted(h, e, wt)


# -- the status word across streams ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("first", [False, True])
def test_status_of_calls_on_other_streams(first):
    """check_status knows what calls on any stream reported, and the word's first value is there before all of them."""
    from d2dmoe_b200._capi import D2DError
    ex = weighted_layer().experts
    ex.packed()
    torch.cuda.synchronize()
    x, w = randn(gen(1), 6, 256).bfloat16(), torch.ones(6, 4, device="cuda")
    good = torch.zeros(6, 4, dtype=torch.int32, device="cuda")
    wrong = torch.full_like(good, 99)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    if first:                                            # the word is made on a stream that is busy
        with torch.cuda.stream(a):
            torch.cuda._sleep(100_000_000)
            ex.forward_weighted(x, good, w)
        with torch.cuda.stream(b):
            ex.forward_weighted(x, wrong, w)
        torch.cuda.synchronize()
    else:
        ex.forward_weighted(x, good, w)
        torch.cuda.synchronize()
        with torch.cuda.stream(b):
            torch.cuda._sleep(100_000_000)
            ex.forward_weighted(x, wrong, w)
    with pytest.raises(D2DError):
        ex.check_status()
    ex.check_status()


@pytest.mark.gpu
def test_status_of_first_calls_from_several_threads():
    """They share one word, whichever of them makes it."""
    import threading
    from d2dmoe_b200._capi import D2DError
    x, w = randn(gen(1), 6, 256).bfloat16(), torch.ones(6, 4, device="cuda")
    good = torch.zeros(6, 4, dtype=torch.int32, device="cuda")
    wrong = torch.full_like(good, 99)
    for turn in range(8):
        ex = weighted_layer().experts
        ex.packed()
        torch.cuda.synchronize()
        start = threading.Barrier(8)

        def call(i):
            with torch.cuda.stream(torch.cuda.Stream()):
                torch.cuda._sleep(1_000_000 * (i + 1))
                start.wait()
                ex.forward_weighted(x, wrong if i == turn else good, w)
        threads = [threading.Thread(target=call, args=(i,)) for i in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        with pytest.raises(D2DError):
            ex.check_status()


# -- rows wider than 2^16 -----------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("fp32", 70001), ("bf16", 100003)])
def test_sum_of_rows_wider_than_a_quotients_range(dtype, d):
    """Odd widths past 2^16 in lists (one thread a column): the last columns are their own token's."""
    import d2dmoe_b200 as D
    N, H = 2060, 4
    x, e, w, w1, b1, w2, _, lb = experts_case(N, d, 3, H, 1, dtype, False, True)
    x[:, 64:] = 0.0                                      # (sums of 64 terms)
    w.uniform_(0.5, 2.0, generator=gen(8))
    got = D.ops.experts_weighted(x, e, w, w1, b1, w2, "relu", last_bias=lb)
    for t in (0, 1, 1000, N - 2, N - 1):
        i = int(e[t, 0])
        h = torch.relu(x[t, :64].double() @ w1[i, :64].double() + b1[i].double())
        h_abs = x[t, :64].double().abs() @ w1[i, :64].double().abs() + b1[i].double().abs()
        want = float(w[t, 0]) * (h @ w2[i].double()) + lb.double()
        size = float(w[t, 0]) * (h_abs @ w2[i].double().abs()) + lb.double().abs()
        within(got[t], want, half(DT[dtype]) * want.abs() + (2 * 64 + H + 16) * U * size, t)


# -- layers behind a kernel that lets them start early -----------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["all", "topk", "dynk", "dynk_max", "weighted"])
@pytest.mark.parametrize("dtype,d", [("bf16", 256), ("fp32", 256), ("bf16", 100)])
def test_layers_read_the_norm_of_this_replay(mode, dtype, d):
    """The layer's kernels may start while layer_norm still writes x; replays on new inputs must see the new rows."""
    import d2dmoe_b200 as D
    torch.manual_seed(3)
    norm = torch.nn.LayerNorm(d).to(DT[dtype]).cuda()
    for N in (7, 300, 3000):
        moe = weighted_layer(dtype, d=d, residual=True)
        moe.forward_mode, moe.tau, moe.k = mode, 0.5, 4
        h = randn(gen(N), 1, N, d).to(DT[dtype])

        def step():
            x = D.layer_norm(h, norm.weight.detach(), norm.bias.detach(), norm.eps)
            y, gating = moe(x)
            z, _ = moe.forward_block(x, norm)
            return x, y, gating["ffn"][0], z
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s), torch.no_grad():
            step()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr), torch.no_grad():
            x, y, rt, z = step()
        for turn in range(4):
            h.copy_(randn(gen(100 * turn + N), 1, N, d) * (1 + turn))
            gr.replay()
            torch.cuda.synchronize()
            with torch.no_grad():
                xs = D.layer_norm(h, norm.weight.detach(), norm.bias.detach(), norm.eps)
                torch.cuda.synchronize()
                ys, gating = moe(xs)
                torch.cuda.synchronize()
                zs, _ = moe.forward_block(xs, norm)
                torch.cuda.synchronize()
            assert torch.equal(x, xs) and torch.equal(rt, gating["ffn"][0])
            # (the 0/1 path adds in any order: about 2^-9 a sum; rows of another input differ by their own size)
            for a, c in ((y, ys), (z, zs)):
                assert ((a - c).float().norm(dim=-1) <= 0.1 * c.float().norm(dim=-1)).all()


# -- scales -------------------------------------------------------------------------------------------------------
def test_scales_without_a_reciprocal_are_refused():
    """The gradient divides the weights by their scale: one below the normal numbers has no finite reciprocal."""
    import ctypes as C
    from d2dmoe_b200 import _capi
    a = C.c_void_p(0x7f0000000000)
    for scale, want in ((1e-39, 1), (2.0 ** -149, 1), (2.0 ** -126, 0), (3e38, 0)):
        assert _capi.lib.d2d_route(a, None, 0, 4, 1, 1, 1, scale, a, a, None, None, 0, 24, 1, None) == want
        assert _capi.lib.d2d_route_backward(a, a, a, a, 0, 1, scale, a, 0, 24, 4, 1, None) == want


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** 100])
def test_gradient_at_extreme_scales(scale):
    g = gen(6)
    for how in (dict(), dict(scores="sigmoid"), dict(renormalise=False)):
        check_route(randn(g, 40, 24), 4, randn(g, 40, 4), scale=scale, **how)


# -- offsets past 32 bits -------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_routing_gradient_past_32_bits():
    """Rows of dlogits on either side of 2^31 elements and at the end, against the 64-bit gradient."""
    import d2dmoe_b200 as D
    g = gen(1)
    N, E, k = 17_000_000, 128, 2
    logits = torch.empty(N, E, dtype=torch.bfloat16, device="cuda")
    for part in logits.split(1 << 20):
        part.copy_(randn(g, *part.shape))
    dw = randn(g, N, k)
    rows = torch.tensor([0, 16_777_215, 16_777_216, N - 1], device="cuda")
    few = logits[rows].double().cpu()
    rel = (96 + 4 * (few.amax(1) - few.amin(1))[:, None]) * U
    for how in (dict(), dict(scores="sigmoid"), dict(renormalise=False)):
        how = dict(dict(scores="softmax", renormalise=True, scale=1.0), **how)
        w, e, _ = D.ops.route(logits, k, **how)
        got = D.ops.route_backward(dw, logits, e, w, **how)[rows].cpu()
        W, I, S = route_reference(logits[rows], k, **how)
        assert torch.equal(e[rows].cpu(), I)
        want = route_gradient(logits[rows], dw[rows], I, **how)
        gd = dw[rows].double().cpu().abs()
        dot = (W * gd).sum(1, keepdim=True)              # what cancels, per row
        size = torch.zeros_like(want).scatter_add_(1, I.long(), W * (gd + dot))
        if how["scores"] == "softmax" and not how["renormalise"]:
            size = S * dot + size
        within(got, want, half(logits.dtype) * want.abs() + 4 * rel * size + 1e-37, how)
        del w, e, got


# -- norms of long rows --------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,params", [("bf16", "same"), ("bf16", "fp32"), ("fp32", "same")])
def test_norms_of_rows_of_every_length(dtype, params):
    """Each number of vectors a thread can have, whole and ragged, up to the longest rows."""
    import d2dmoe_b200 as D
    for d in (4096, 4104, 6144, 6152, 8192, 8196, 8200, 9000, 10240, 12288, 12296, 14336, 16380, 16384, 8193, 12001):
        for kind in ("layer", "rms"):
            x, w, b, dy = norm_inputs(3, d, dtype, params, kind, 0)
            ref = norm_reference(x, w, b, 1e-5, kind, 0.0, dy)
            y, mean, rstd = D.ops.layer_norm(x, w, b, kind=kind)
            within(y, *ref["y"], d)
            dx, dw, db = D.ops.layer_norm_backward(dy, x, w, mean, rstd, kind=kind, bias=b is not None)
            within(dx, *ref["dx"], d)
            within(dw, *ref["dw"], d)
            if b is not None:
                within(db, *ref["db"], d)
            only, _, _ = D.ops.layer_norm_backward(dy, x, w, mean, rstd, kind=kind, bias=False, dweight=False)
            assert torch.equal(only, dx)


# -- shares of small sigmoids ------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("k", [8, 17])
def test_shares_of_sigmoids_that_underflow(k, dtype):
    """sigmoid(-95) is no 32-bit number, its share beside sigmoid(-50) is."""
    g = gen(k)
    for top in (-55.0, -30.0, -1.0, 2.0):
        logits = (top - 60 * torch.rand(100, 24, generator=g, device="cuda")).to(DT[dtype])
        check_route(logits, k, randn(g, 100, k), scores="sigmoid")
        check_route(logits, k, scores="sigmoid", bias=0.1 * randn(g, 24), scale=2.5)
