"""Norm, routing and weighted experts on values and calls where a plain implementation is easily right: rows in their
16-bit form, zeros of both signs, NaN through an activation, biases that cancel, rows wider than 2^16, tangents, streams."""
import pytest
import torch

from test_operators import U, gen, half, randn, within


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
    # 3072 errors of at most 2^-14 of about twice the value, either way: 2^-13 / sqrt(3 * 3072) = 1.3e-6 of the whole
    assert abs(along / size) <= 1e-5
