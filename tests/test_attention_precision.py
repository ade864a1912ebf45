"""How far bf16 results and gradients of the attention are from 64 bits, as the rms error relative to the result's own rms.
u = 2^-9 / sqrt(3) / 0.68 = 0.00166 is the rms of one rounding to bf16 relative to the rounded values (uniform within half a
step of 2^-8 to 2^-9 of the value), sampling errors over the 10^4 to 10^6 elements taken here are below 1 %."""
import pytest
import torch

from test_attention import BF, make

U = 0.00166


def errors(got, want):
    return {n: float((got[n].double() - want[n]).norm() / want[n].norm()) for n in want}


def exact(q, k, v, dout, scale):
    """One head, float64."""
    q, k, v, dout = (t.double()[0, :, 0] for t in (q, k, v, dout))
    p = torch.softmax(q @ k.t() * scale, 1)
    out = p @ v
    ds = p * (dout @ v.t() - (dout * out).sum(1, keepdim=True)) * scale
    return {n: t[None, :, None] for n, t in (("out", out), ("dq", ds @ k), ("dk", ds.t() @ q), ("dv", p.t() @ dout))}


def measured(q, k, v, dout, scale):
    from segk import functional as SF
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = SF.attention(*leaves, scale=scale)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + torch.autograd.grad(out, leaves, dout)))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
def test_gradients_of_keys_round_alike_for_few_and_many_rows(D):
    """P and dS are rounded to bf16 once for the products over the rows, however many rows there are."""
    found = []
    for rows in (21, 64, 65, 200):
        q, k, v, dout, _ = make(1, rows, 4096, 1, 1, D, BF, "plain", 51)
        found.append(errors(measured(q, k, v, dout, D ** -0.5), exact(q, k, v, dout, D ** -0.5)))
    for name in ("dk", "dv"):
        e = [f[name] for f in found]
        assert max(e) < 1.1 * min(e), (name, e)
        # the roundings of the operand and of the result, sqrt(2) u
        assert max(e) < 1.1 * 2 ** 0.5 * U, (name, e)
