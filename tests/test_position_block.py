"""Projection output -> norm and rotation -> attention over padded maps -> gradients in bf16, against float64 autograd of the same
inputs: rms error of every result relative to its own rms.

u = 0.00166, one rounding to bf16 (test_attention_precision).  The operands are exact; rounded are q and k behind the rotation
(heads of norm sqrt(D): a score's error is sqrt(2) u sqrt(sum q^2 k^2) / sqrt(D) = sqrt(2) u absolute, the same relative to its
probability), P for its product and in delta, dS for dk, and every result:
  out  2 + 1 (P) + 1                                                          = 4 u^2
  dv   2 + 1 (P) + 1                                                          = 4 u^2
  dq   2 + 1 (k) + 1 (delta) + 1 (dq) + 1 (behind the rotation)               = 6 u^2
  dk   2 + 1 (q) + 1 (delta) + 1 (dS) + 1 (dk) + 1 (behind the rotation)      = 7 u^2
  weights as dq and dk, over sums of independent terms, without the last rounding
Twice these roots are asked for: the norm's backward pass takes the part along a head out of its gradient and with it up to
half of the square it is measured against, and the sums behind the weights have few hundred terms an element."""
import math

import pytest
import torch

U = 0.00166


def rotate(x, w, cos, sin):
    n = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    a, b = n.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2, 9, 11, 4, 2, 32), (1, 21, 17, 4, 4, 64), (2, 13, 13, 8, 2, 128)])
def test_block_in_bf16(size):
    from segk import functional as SF
    N, H, W, Hq, Hk, D = size
    L = H * W
    gen = torch.Generator().manual_seed(91)
    qkv = torch.randn(N, L, Hq + 2 * Hk, D, generator=gen).cuda().bfloat16().requires_grad_(True)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=gen)).cuda().requires_grad_(True) for _ in range(2))
    pos = torch.cartesian_prod(torch.arange(H), torch.arange(W)).cuda()
    freq = (100.0 ** -(torch.arange(D // 4) / (D // 4))).repeat(2).cuda()
    key = torch.ones(N, H, W, dtype=torch.bool, device="cuda")
    key[0, 2 * H // 3:] = False
    key[N - 1, :, W - 3:] = False
    key = key.reshape(N, L)
    dout = torch.randn(N, L, Hq, D, generator=gen).cuda().bfloat16()

    q, k = SF.qk_norm_rotary(qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], wq, wk, pos, freq)
    out = SF.attention(q, k, qkv[:, :, Hq + Hk:], key_mask=key)
    dx, dwq, dwk = torch.autograd.grad(out, (qkv, wq, wk), dout)

    x, w1, w2 = (t.detach().double().requires_grad_(True) for t in (qkv, wq, wk))
    angle = pos.double()[:, [0] * (D // 4) + [1] * (D // 4)] * freq.double()
    cos, sin = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)
    q6 = rotate(x[:, :, :Hq], w1, cos, sin).transpose(1, 2)
    k6 = rotate(x[:, :, Hq:Hq + Hk], w2, cos, sin).repeat_interleave(Hq // Hk, 2).transpose(1, 2)
    v6 = x[:, :, Hq + Hk:].repeat_interleave(Hq // Hk, 2).transpose(1, 2)
    s = (q6 @ k6.transpose(2, 3).contiguous() * D ** -0.5).masked_fill(~key[:, None, None], -math.inf)
    out6 = (torch.softmax(s, -1) @ v6).transpose(1, 2)
    dx6, dw1, dw2 = torch.autograd.grad(out6, (x, w1, w2), dout.double())

    parts = {"out": (out, out6, 4), "dq": (dx[:, :, :Hq], dx6[:, :, :Hq], 6), "dk": (dx[:, :, Hq:Hq + Hk], dx6[:, :, Hq:Hq + Hk], 7),
             "dv": (dx[:, :, Hq + Hk:], dx6[:, :, Hq + Hk:], 4), "dwq": (dwq, dw1, 5), "dwk": (dwk, dw2, 6)}
    found = {n: (float((a.detach().double() - b).norm() / b.norm()), 2 * U * m ** 0.5) for n, (a, b, m) in parts.items()}
    print(size, {n: "%.5f / %.5f" % f for n, f in found.items()})
    assert all(e < bound for e, bound in found.values()), found
