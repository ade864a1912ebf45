"""Rows that two masks leave nothing together (padding on the left under a diagonal; a query mask that opens only padding): out
is zero and there is no gradient, whatever the row's own query and output gradient hold.  Bounds: test_attention.reference."""
import math

import pytest
import torch

from test_attention import BF, F32, check, make, reference

# N, Lq, Lk, Hq, Hk, D, masks
CASES = [
    (2, 70, 70, 2, 1, 64, "left causal"),
    (2, 150, 200, 4, 2, 128, "left causal"),
    (3, 33, 40, 2, 2, 32, "left pair"),
    (1, 3, 5000, 4, 2, 96, "left pair"),        # keys in parts
    (2, 300, 290, 2, 2, 64, "left causal pair"),
]


def masks(N, Lq, Lk, kind, gen):
    """(mask, key mask, rows that have no open key): the last image has no padding."""
    key = torch.ones(N, Lk, dtype=torch.bool)
    for n in range(N):
        key[n, :(N - n) * Lk // (2 * N) if N == 1 or n < N - 1 else 0] = False
    mask = None
    open_ = key[:, None].expand(N, Lq, Lk).clone()
    if "pair" in kind:
        mask = torch.rand(N, 1, Lq, Lk, generator=gen) < 0.8
        mask[:, 0, ::3] &= ~key[:, None]          # only padding
        open_ &= mask[:, 0]
    if "causal" in kind:
        open_ &= torch.arange(Lk) <= torch.arange(Lq)[:, None] + (Lk - Lq)
    empty = ~open_.any(2)
    assert empty.any() and not empty.all()
    return None if mask is None else mask.cuda(), key.cuda(), empty.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=[str(c) for c in CASES])
def test_rows_closed_by_two_masks_may_hold_anything(case, dt, bad):
    from segk import functional as SF, ops
    N, Lq, Lk, Hq, Hk, D, kind = case
    q, k, v, dout, gen = make(N, Lq, Lk, Hq, Hk, D, dt, "plain", 41)
    mask, key, empty = masks(N, Lq, Lk, kind, gen)
    causal = "causal" in kind
    res, tol = reference(q, k, v, dout, mask, key, causal, D ** -0.5, dt)
    q, k, v, dout = (t.clone() for t in (q, k, v, dout))
    q[empty] = bad
    dout[empty] = bad
    k[~key] = bad
    v[~key] = bad
    got = torch.empty_like(q)
    lse = ops.attention_fwd(q, k, v, got, D ** -0.5, causal, mask, key, want_lse=True)
    check({"out": got, "lse": lse}, res, tol, "forward")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = SF.attention(*leaves, mask, key, causal)
    grads = torch.autograd.grad(out, leaves, dout)
    check(dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads)), res, tol, "training")
    assert not out.detach()[empty].any() and not grads[0][empty].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("lk", [1, 90, 6000])
def test_queries_that_are_not_finite_stay_visible(dt, masked, lk):
    """A row that has an open key and a query with NaN or an infinity is NaN, also where every score is -inf (one key); other
    rows are not touched by it."""
    from segk import functional as SF, ops
    q, k, v, _, gen = make(1, 40, lk, 2, 1, 64, dt, "plain", 43)
    key = None
    if masked:
        key = torch.rand(1, lk, generator=gen).cuda() < 0.5
        key[0, 0] = True
    want = SF.attention(q, k, v, key_mask=key)
    for bad in (math.nan, math.inf, -math.inf):
        q2 = q.clone()
        q2[0, 3, 1, 9] = bad
        q2[0, 30, 0] = bad
        out = torch.empty_like(q2)
        lse = ops.attention_fwd(q2, k, v, out, 0.125, key_mask=key, want_lse=True)
        for t, h in ((3, 1), (30, 0)):
            assert torch.isnan(out[0, t, h]).all() and torch.isnan(lse[0, h, t])
            out[0, t, h] = want[0, t, h]
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("lk", [500, 9000])
def test_an_empty_row_does_not_change_its_neighbours(dt, lk):
    """Not by a bit: a row without an open key needs no new reference for its exponents, which the rows beside it would share."""
    from segk import functional as SF
    q, k, v, _, gen = make(1, 40, lk, 1, 1, 64, dt, "plain", 47)
    mask = torch.rand(1, 1, 40, lk, generator=gen).cuda() < 0.9
    mask[..., 0] = True
    want = SF.attention(q, k, v, mask)
    for row in (0, 7, 39):
        less = mask.clone()
        less[0, 0, row] = False
        got = SF.attention(q, k, v, less)
        assert not got[0, row].any()
        got[0, row] = want[0, row]
        same = torch.equal(got, want)
        assert same


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("lk", [1, 70, 5000])
def test_scores_far_below_zero(dt, lk):
    """-1e30 and less, where one key lies so far above the others that the result is its value."""
    from segk import functional as SF
    _, _, v, _, _ = make(1, 33, lk, 1, 1, 32, dt, "plain", 53)
    for top in (0, lk // 2, lk - 1):
        q = torch.full((1, 33, 1, 32), 2.0 ** 50, device="cuda", dtype=dt)
        k = torch.full((1, lk, 1, 32), -2.0 ** 52, device="cuda", dtype=dt)
        k[0, top] = -2.0 ** 51
        out = SF.attention(q, k, v, scale=1.0)
        same = torch.equal(out, v[:, top:top + 1].expand_as(out))
        assert same
