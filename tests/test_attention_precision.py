"""How far bf16 results and gradients of the attention are from 64 bits, as the rms error relative to the result's own rms.
u = 2^-9 / sqrt(3) / 0.68 = 0.00166 is the rms of one rounding to bf16 relative to the rounded values (uniform within half a
step of 2^-8 to 2^-9 of the value).  Sampling: the final rounding is one of 10^4 to 10^6 elements, below 1 %.  Of the rounded
operands (p, ds) few large ones can carry a result.  Their mean square error is a mean of e^2 with weights w = p^2 (ds^2),
worth n = (sum w)^2 / sum w^2 independent terms; e^2 / u^2 has mean 1 and standard deviation sqrt(9 / 5 * 1.2 - 1) < 1.25
(uniform e, steps spread by the mantissa), so that four deviations are 5 / sqrt(n)."""
import pytest
import torch

from test_attention import BF, make

U = 0.00166


def errors(got, want):
    return {n: float((got[n].double() - want[n]).norm() / want[n].norm()) for n in got}


def spread(t):
    """Factor on the mean square of a rounding of t, weighted with t's squares: four deviations of its sampling."""
    w = t.square()
    return 1 + 5 * float(w.square().sum().sqrt() / w.sum())


def exact(q, k, v, dout, scale):
    """One head, float64."""
    q, k, v, dout = (t.double()[0, :, 0] for t in (q, k, v, dout))
    p = torch.softmax(q @ k.t() * scale, 1)
    out = p @ v
    ds = p * (dout @ v.t() - (dout * out).sum(1, keepdim=True)) * scale
    res = {n: t[None, :, None] for n, t in (("out", out), ("dq", ds @ k), ("dk", ds.t() @ q), ("dv", p.t() @ dout))}
    return dict(res, p=p, ds=ds)


def measured(q, k, v, dout, scale):
    from segk import functional as SF
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = SF.attention(*leaves, scale=scale)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + torch.autograd.grad(out, leaves, dout)))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
def test_gradients_of_keys_for_few_and_many_rows(D):
    """Up to 64 rows P and dS go into their products as two bf16 operands (the final rounding is left, u), above that rounded
    once (sqrt(2) u), the same at 65 rows as at more."""
    found = {}
    for rows in (21, 64, 65, 200):
        q, k, v, dout, _ = make(1, rows, 4096, 1, 1, D, BF, "plain", 51)
        want = exact(q, k, v, dout, D ** -0.5)
        found[rows] = errors(measured(q, k, v, dout, D ** -0.5), want)
        bound = 1.02 * U * (1 if rows <= 64 else 1 + spread(want["p"])) ** 0.5
        for name in ("dk", "dv"):
            assert found[rows][name] < bound, (rows, found)
    for name in ("dk", "dv"):
        assert abs(found[65][name] / found[200][name] - 1) < 0.1, found


@pytest.mark.gpu
def test_keys_that_one_row_reads():
    """Windows of few keys: a key's gradient is one term, and its roundings are its error (up to 64 rows: the final one's)."""
    from segk import functional as SF
    q, k, v, dout, gen = make(1, 21, 4096, 1, 1, 32, BF, "plain", 55)
    mask = torch.zeros(1, 1, 21, 4096, dtype=torch.bool)
    for i in range(21):
        mask[0, 0, i, 190 * i:190 * i + 3 + i] = True
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = SF.attention(*leaves, mask.cuda())
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout)))
    q, k, v, dout = (t.double()[0, :, 0] for t in (q, k, v, dout))
    p = torch.softmax((q @ k.t() * 32 ** -0.5).masked_fill(~mask.cuda()[0, 0], -torch.inf), 1)
    ds = p * (dout @ v.t() - (dout * (p @ v)).sum(1, keepdim=True)) * 32 ** -0.5
    want = {"dk": (ds.t() @ q)[None, :, None], "dv": (p.t() @ dout)[None, :, None]}
    # dk: u, and delta's part, u |p|_2 of ds' row norm (|p|_2 < 1); dv: u.  Sampling of 273 weights: 5 / sqrt(n)
    found = errors({n: got[n] for n in want}, want)
    assert found["dv"] < 1.02 * U * 1.05 and found["dk"] < 1.02 * U * (1 + spread(ds)) ** 0.5, found


def scaled(sd, Lq, Lk, H, Hk, D, seed=61):
    """Operands whose scores have the standard deviation sd (trained heads reach 3 to 10)."""
    q, k, v, dout, _ = make(1, Lq, Lk, H, Hk, D, BF, "plain", seed)
    return (q.float() * sd).to(BF), k, v, dout


SHARP = [
    (512, 1024, 64),
    (500, 1000, 128),
    (300, 700, 32),
    (33, 12000, 64),      # keys in parts
    (33, 12000, 96),
]


@pytest.mark.gpu
@pytest.mark.parametrize("sd", [1, 3, 5, 8])
@pytest.mark.parametrize("size", SHARP, ids=[str(s) for s in SHARP])
def test_sharp_scores(size, sd):
    """P is rounded to bf16 for its products; what the rounding does to out and, through delta, to dq and dk stays below one
    rounding of the result, however few keys carry a row.
      out    sum of rounded p v / sum of rounded p: sum_j p_j e_j (v_j - out), at most u |p|_2 (|p|_2 <= 1) of out's size
      delta  the same with dp in the place of v: sum_j ds_j e_j, rms u |ds_i|_2
      dq     delta's error times sum_j p_j k_j: u |p|_2 of dq's size
    so that out and dq have at most sqrt(2) u with the final rounding, dv (P rounded for its product) the same, and dk (dS
    rounded) sqrt(3) u.  With scores of standard deviation 1, |p|_2 is below a third, and dq has sqrt(1 + 1 / 9) u."""
    Lq, Lk, D = size
    q, k, v, dout = scaled(sd, Lq, Lk, 1, 1, D)
    want = exact(q, k, v, dout, D ** -0.5)
    got = errors(measured(q, k, v, dout, D ** -0.5), want)
    p, ds = spread(want["p"]), spread(want["ds"])
    square = {"out": 1 + p, "dq": 1 + ds / 9 if sd == 1 else 1 + ds, "dk": 1 + 2 * ds, "dv": 1 + p}
    bound = {n: 1.02 * U * x ** 0.5 for n, x in square.items()}
    print(size, sd, {n: "%.5f / %.5f" % (e, bound[n]) for n, e in got.items()})
    assert all(e < bound[n] for n, e in got.items()), got


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2, 150, 300, 4, 2, 64), (1, 3, 9000, 4, 2, 40), (2, 64, 200, 2, 2, 128)])
def test_what_the_rounding_left_over(size):
    """out_rest: at most half a step of out, zero in empty rows; out + out_rest is nearer to 64 bits than out."""
    from segk import ops
    N, Lq, Lk, Hq, Hk, D = size
    q, k, v, dout, gen = make(N, Lq, Lk, Hq, Hk, D, BF, "heads_first", 71)
    mask = torch.ones(N, 1, Lq, 1, dtype=torch.bool, device="cuda")
    mask[:, :, ::3] = False
    out, rest = torch.empty(N, Lq, Hq, D, dtype=BF, device="cuda"), torch.full((N, Lq, Hq, D), 7., dtype=BF, device="cuda")
    lse = ops.attention_fwd(q, k, v, out, D ** -0.5, mask=mask, want_lse=True, out_rest=rest)
    assert not out[:, ::3].any() and not rest[:, ::3].any()
    both = out.double() + rest.double()
    # (half a step of out is at most 2^-8 |out|; rest may round up to it, so that the sum need not round to out again)
    assert bool((rest.double().abs() <= 2.0 ** -8 * out.double().abs()).all())
    plain = torch.empty_like(out)
    ops.attention_fwd(q, k, v, plain, D ** -0.5, mask=mask)
    same = torch.equal(plain, out)
    assert same
    # the weights of the sum are rounded p over their own sum: |out - both| <= 2 half steps of sum p |v|, and what is left of
    # the result itself a quarter step of 2^-8 of |rest| <= 2^-8 |out|
    kk, vv = (t.double().repeat_interleave(Hq // Hk, 2) for t in (k, v))
    p = torch.softmax(torch.matmul(q.double().permute(0, 2, 1, 3), kk.permute(0, 2, 3, 1).contiguous()) * D ** -0.5, -1)
    want, size_ = (torch.matmul(p, t.permute(0, 2, 1, 3).contiguous()).permute(0, 2, 1, 3) for t in (vv, vv.abs()))
    live = torch.arange(Lq) % 3 != 0
    assert bool(((both - want).abs() <= 2.1 * 2.0 ** -8 * size_ + 2.0 ** -16 * want.abs())[:, live].all())
    assert float((both - want)[:, live].norm()) < 0.8 * float((out.double() - want)[:, live].norm())
    # and in the backward pass: nothing of it, or all of it
    ops.attention_bwd(q, k, v, out, lse, dout, D ** -0.5, mask=mask)
    got = ops.attention_bwd(q, k, v, out, lse, dout, D ** -0.5, mask=mask, out_rest=rest)
    assert all(torch.isfinite(g).all() for g in got)


@pytest.mark.gpu
def test_out_rest_is_refused_where_it_does_not_fit():
    from segk import ops
    q, k, v, _, _ = make(1, 4, 6, 2, 2, 16, BF, "plain", 1)
    out = torch.empty_like(q)
    for bad in (torch.empty_like(q, dtype=torch.float32), torch.empty(1, 4, 2, 8, dtype=BF, device="cuda"),
                torch.empty(1, 4, 16, 2, dtype=BF, device="cuda").transpose(2, 3), torch.empty(1, 4, 2, 16, dtype=BF)):
        with pytest.raises(ValueError):
            ops.attention_fwd(q, k, v, out, 0.25, out_rest=bad)
    f = [t.float() for t in (q, k, v, out)]
    with pytest.raises(ValueError, match="bfloat16"):
        ops.attention_fwd(*f, 0.25, out_rest=torch.empty_like(q))
