"""Norm + rotation of queries and keys (segk.functional.qk_norm_rotary) against the definition in 64 bits.

Bounds, element by element.  v = 2^-24 (half a step of fp32), u the same of the operand type.  y = (x r w) turned:
  x r w   mean of D squares (D / 8 + 8) v halved by the root, root 2 v, three products 3 v       -> (D / 16 + 9) v relative
  angle   one rounding of a value up to 1 half turn: pi v absolute; sin / cos 4 v absolute      -> 8 v of |a| + |b|
  turn    2 products and a sum                                                                  -> 2 v of |a| + |b|
so |y error| <= ((D / 16 + 19) v (|a| + |b|) + u|y|), doubled.  Backward: dn = dy turned back carries 10 v (|a| + |b|) of dy;
dx = r (g - xr mean(g xr)): (D / 8 + 24) v (r (|g| + |xr| mean|g xr|)) + r (dn error and its mean) + u|dx|, doubled;
dw = sum dn xr over T terms: fp32 sums of at most T / 64 + 64 terms one after the other."""
import math

import pytest
import torch

BF, F32 = torch.bfloat16, torch.float32
V = 2.0 ** -24


def pairs_of(D, R, interleaved, dev):
    c = torch.arange(R, device=dev)
    return (2 * c, 2 * c + 1) if interleaved else (c, c + R)


def turn(x, cos, sin, ia, ib):
    y = x.clone()
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = a * cos - b * sin
    y[..., ib] = a * sin + b * cos
    return y


def both(x, ia, ib):
    """|a| + |b| of an element's pair at both places; twice |x| elsewhere."""
    y = 2 * x.abs()
    s = x[..., ia].abs() + x[..., ib].abs()
    y[..., ia] = s
    y[..., ib] = s
    return y


def reference(x, w, dy, pos, freq, sections, eps, interleaved, dt):
    u = torch.finfo(dt).eps / 2
    x, dy = x.double(), dy.double()
    D, R = x.shape[-1], freq.shape[0]
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(x.device)
    ang = pos.double()[..., axis] * freq.double()
    ang = ang.unsqueeze(-2) if ang.dim() == 3 else ang.unsqueeze(-2).unsqueeze(0)
    cos, sin = ang.cos(), ang.sin()
    ia, ib = pairs_of(D, R, interleaved, x.device)
    one = torch.ones(D, dtype=torch.float64, device=x.device)
    w = one if w is None else w.double()
    r = one.new_ones(()) if eps is None else (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r * w
    y = turn(n, cos, sin, ia, ib)
    ty = 2 * ((D / 16 + 19) * V * both(n, ia, ib) + u * y.abs())
    dn = turn(dy, cos, -sin, ia, ib)
    e_dn = 10 * V * both(dy, ia, ib)
    if eps is None:
        return y, ty, dn, 2 * (e_dn + u * dn.abs()), None, None
    xr = x * r
    g = dn * w
    dx = r * (g - xr * (g * xr).mean(-1, keepdim=True))
    big = g.abs() + xr.abs() * (g * xr).abs().mean(-1, keepdim=True)
    e_g = e_dn * w.abs()
    tx = 2 * ((D / 8 + 24) * V * r * big + r * (e_g + xr.abs() * (e_g * xr.abs()).mean(-1, keepdim=True)) + u * dx.abs())
    dw = (dn * xr).sum((0, 1, 2))
    T = x.shape[0] * x.shape[1] * x.shape[2]
    tw = 2 * (((e_dn + (D / 16 + 9) * V * dn.abs()) * xr.abs()).sum((0, 1, 2)) + (T / 64 + 64) * V * (dn * xr).abs().sum((0, 1, 2)))
    return y, ty, dx, tx, dw, tw


def close(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got.double() - want).abs() <= tol + 1e-37)
    if bad.any():
        i = int(bad.flatten().nonzero()[0])
        raise AssertionError("%s: %d of %d off, at %d got %g want %g bound %g" % (
            what, int(bad.sum()), bad.numel(), i, got.flatten()[i], want.flatten()[i], tol.expand_as(want).flatten()[i]))


CASES = [
    # N, L, Hq, Hk, D, sections, interleaved, positions, weights, eps
    (1, 1, 1, 1, 8, (4,), False, "int32", True, 1e-6),
    (1, 1, 16, 4, 64, (16, 16), False, "int32", True, 1e-6),
    (2, 35, 3, 1, 24, (4, 4, 4), True, "int64", True, 1e-6),
    (2, 77, 4, 2, 40, (8, 8), False, "float", False, 1e-5),
    (1, 129, 2, 2, 128, (24, 20, 20), False, "images", True, 1e-6),
    (3, 50, 5, 0, 96, (16, 16, 16), True, "far", True, 1e-6),
    (2, 31, 2, 3, 256, (32, 32, 32, 32), False, "int32", True, 1e-6),
    (2, 31, 2, 1, 64, (5, 0, 11), False, "int32", True, 1e-3),      # 16 of 32 pairs, ragged shares, one axis unused
    (2, 31, 2, 1, 64, (4, 4), True, "int64", True, 1e-6),           # 8 of 32 pairs
    (1, 64, 2, 2, 16, (8,), False, "far", False, None),             # rotation alone
    (4, 1089, 8, 8, 64, (16, 16), False, "int32", True, 1e-6),
    (1, 3000, 12, 4, 72, (18, 18), True, "float", True, 1e-6),
]


def make(case, dt, dev="cuda"):
    N, L, Hq, Hk, D, sections, interleaved, kind, weights, eps = case
    gen = torch.Generator().manual_seed(17)
    x = (torch.randn(N, L, Hq + Hk, D, generator=gen) * torch.rand(N, L, 1, 1, generator=gen)).to(dev).to(dt)
    A, R = len(sections), sum(sections)
    shape = (N, L, A) if kind in ("images", "far") else (L, A)
    if kind == "float":
        pos = (torch.rand(shape, generator=gen) * 200 - 50).to(dev)
    elif kind == "far":
        pos = torch.randint(-2 ** 40, 2 ** 40, shape, generator=gen).to(dev) if eps is None else \
            torch.randint(0, 2 ** 31 - 1, shape, generator=gen, dtype=torch.int64).to(torch.int32).to(dev)
    else:
        pos = torch.randint(0, 700, shape, generator=gen).to(torch.int32 if kind != "int64" else torch.int64).to(dev)
    freq = (10000.0 ** -torch.rand(R, generator=gen)).to(dev)
    if kind == "far" and eps is None:
        freq = freq * 2.0 ** -20
    wq = wk = None
    if weights:
        wq, wk = (1 + 0.3 * torch.randn(D, generator=gen)).to(dev), (1 + 0.3 * torch.randn(D, generator=gen)).to(dev)
    dy = torch.randn(N, L, Hq + Hk, D, generator=gen).to(dev).to(dt)
    return x, wq, wk, pos, freq, dy


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=[str(c) for c in CASES])
def test_forward_and_gradients(case, dt):
    from segk import functional as SF
    N, L, Hq, Hk, D, sections, interleaved, kind, weights, eps = case
    x, wq, wk, pos, freq, dy = make(case, dt)
    leaves = [x[:, :, :Hq].detach().requires_grad_(True), x[:, :, Hq:].detach().requires_grad_(True) if Hk else None,
              None if wq is None else wq.requires_grad_(True), None if wk is None or not Hk else wk.requires_grad_(True)]
    kw = dict(sections=sections, eps=eps, interleaved=interleaved)
    with torch.no_grad():
        plain = SF.qk_norm_rotary(*leaves, pos, freq, **kw)
    out = SF.qk_norm_rotary(*leaves, pos, freq, **kw)
    plain, out = (plain, out) if Hk else ((plain,), (out,))
    assert all(torch.equal(a, b) for a, b in zip(plain, out))
    wanted = [t for t in leaves if t is not None]
    dys = (dy[:, :, :Hq], dy[:, :, Hq:])[:len(out)]
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None], torch.autograd.grad(out, wanted, dys)))
    for i in range(len(out)):
        y, ty, dx, tx, dw, tw = reference((x[:, :, :Hq], x[:, :, Hq:])[i], leaves[2 + i] if weights else None, dys[i], pos,
                                          freq, sections, eps, interleaved, dt)
        close(out[i].detach(), y, ty, "result %d" % i)
        close(grads[i], dx, tx, "gradient %d" % i)
        if leaves[2 + i] is not None:
            close(grads[2 + i], dw, tw, "weight gradient %d" % i)


# Numbers of tokens at which a group of lanes takes one, some or all of a token's heads (10 and 23 of them).
SHARES = [
    (1, 500, 7, 3, 64, (16, 16), False, "int32", True, 1e-6),
    (1, 3001, 7, 3, 96, (16, 16, 16), False, "int64", True, 1e-6),
    (2, 6001, 7, 3, 64, (16, 16), True, "images", True, 1e-6),
    (1, 1777, 20, 3, 128, (32, 32), False, "int32", True, 1e-6),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", SHARES, ids=[str(c) for c in SHARES])
def test_shares_of_heads(case, dt):
    test_forward_and_gradients(case, dt)


@pytest.mark.gpu
def test_default_sections_layouts_and_types():
    from segk import functional as SF
    case = (2, 20, 4, 2, 32, (8, 8), False, "int32", True, 1e-6)
    x, wq, wk, pos, freq, _ = make(case, BF)
    q, k = x[:, :, :4], x[:, :, 4:]
    want = SF.qk_norm_rotary(q, k, wq, wk, pos, freq, sections=(8, 8))
    for other in (SF.qk_norm_rotary(q, k, wq, wk, pos, freq),
                  SF.qk_norm_rotary(q, k, wq, wk, pos.long().expand(2, 20, 2), freq),
                  SF.qk_norm_rotary(q, k, wq, wk, pos.float(), freq),
                  SF.qk_norm_rotary(q, k, wq, wk, pos.t().contiguous().t(), freq),
                  SF.qk_norm_rotary(q.transpose(1, 2).contiguous().transpose(1, 2), k.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2),
                                    wq, wk, pos, freq)):
        assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    alone = SF.qk_norm_rotary(k, None, wk, None, pos, freq)
    assert torch.equal(alone, want[1])
    wb = wq.to(BF).requires_grad_(True)
    out = SF.qk_norm_rotary(q, None, wb, None, pos, freq)
    (g,) = torch.autograd.grad(out.float().sum(), wb)
    assert g.dtype == BF and torch.isfinite(g).all()
    none = SF.qk_norm_rotary(q[:, :0], k[:, :0], wq, wk, pos[:0], freq)
    assert none[0].shape == (2, 0, 4, 32)
    zero = SF.qk_norm_rotary(torch.zeros_like(q), torch.zeros_like(k), wq, wk, pos, freq)
    assert not zero[0].any() and not zero[1].any()


@pytest.mark.gpu
def test_gradients_against_differences():
    from segk import functional as SF
    case = (1, 6, 2, 1, 16, (4, 4), False, "int32", True, 1e-6)
    x, wq, wk, pos, freq, dy = make(case, F32)
    x = x + 0.5
    leaves = [x[:, :, :2].detach().requires_grad_(True), x[:, :, 2:].detach().requires_grad_(True), wq.requires_grad_(True),
              wk.requires_grad_(True)]
    dys = (dy[:, :, :2], dy[:, :, 2:])
    grads = torch.autograd.grad(SF.qk_norm_rotary(*leaves, pos, freq), leaves, dys)
    gen = torch.Generator().manual_seed(1)
    eps = 2.0 ** -8
    for i, t in enumerate(leaves):
        step = torch.randn(t.shape, generator=gen).cuda()
        ends = []
        with torch.no_grad():
            for sign in (1, -1):
                at = [u + sign * eps * step if j == i else u for j, u in enumerate(leaves)]
                ends.append(sum(float((o.double() * d.double()).sum()) for o, d in zip(SF.qk_norm_rotary(*at, pos, freq), dys)))
        want = float((grads[i].double() * step.double()).sum())
        # central differences: eps^2 / 6 times a third derivative of at most ~100 per value, and rounding / (2 eps)
        size = float(dy.abs().sum()) * (eps ** 2 * 20 + 2 ** -22 / eps)
        assert abs((ends[0] - ends[1]) / (2 * eps) - want) < size, i


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
def test_position_attention_block(dt):
    """Projection output -> norm and rotation -> attention over a padded map -> gradients: the operators as they are used
    together, replayed from one graph between eager calls, and in fp32 against float64 autograd.  (Bound, relative to each
    result's largest value: heads of norm sqrt(32) with 25 v each give scores 2 * 25 * 5.7 v = 285 v, twice that in a
    probability, twice again in p (dp - delta), less than 4096 v in all.)"""
    from segk import functional as SF
    N, H, W, Hq, Hk, D = 2, 9, 11, 4, 2, 32
    L = H * W
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn(N, L, Hq + 2 * Hk, D, generator=gen).cuda().to(dt).requires_grad_(True)
    wq, wk = (torch.ones(D, device="cuda", requires_grad=True) for _ in range(2))
    pos = torch.cartesian_prod(torch.arange(H), torch.arange(W)).cuda()
    freq = (100.0 ** -(torch.arange(8) / 8)).repeat(2).cuda()
    key = torch.ones(N, H, W, dtype=torch.bool, device="cuda")
    key[0, 6:] = False
    key[1, :, 8:] = False
    key = key.reshape(N, L)
    dout = torch.randn(N, L, Hq, D, generator=gen).cuda().to(dt)

    def step():
        q, k = SF.qk_norm_rotary(qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], wq, wk, pos, freq)
        out = SF.attention(q, k, qkv[:, :, Hq + Hk:], key_mask=key)
        return (out.detach(),) + torch.autograd.grad(out, (qkv, wq, wk), dout)

    x64 = qkv.detach().double().requires_grad_(True)
    w64 = [w.detach().double().requires_grad_(True) for w in (wq, wk)]
    ang = pos.double()[:, [0] * 8 + [1] * 8] * freq.double()
    cos, sin = ang.cos().unsqueeze(1), ang.sin().unsqueeze(1)
    sides = []
    for part, w in ((x64[:, :, :Hq], w64[0]), (x64[:, :, Hq:Hq + Hk], w64[1])):
        n = part * (part.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        a, b = n[..., :16], n[..., 16:]
        sides.append(torch.cat((a * cos - b * sin, a * sin + b * cos), -1))
    q, k, v = sides[0], sides[1].repeat_interleave(2, 2), x64[:, :, Hq + Hk:].repeat_interleave(2, 2)
    s = (q.transpose(1, 2) @ k.transpose(1, 2).transpose(2, 3).contiguous()) * D ** -0.5
    s = s.masked_fill(~key[:, None, None], -math.inf)
    out64 = (torch.softmax(s, -1) @ v.transpose(1, 2)).transpose(1, 2)
    want = (out64.detach(),) + torch.autograd.grad(out64, [x64] + w64, dout.double())
    got = step()
    for g, r in zip(got, want):
        assert dt == BF or float((g.double() - r).abs().max() / r.abs().max()) < 4096 * V
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = step()
    for _ in range(3):
        with torch.no_grad():
            qkv.copy_(torch.randn_like(qkv))
        graph.replay()
        kept = [t.clone() for t in res]
        again = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, again))


def test_refuses_cpu_tensors():
    from segk import functional as SF
    q = torch.zeros(1, 4, 2, 16)
    with pytest.raises(ValueError, match="GPU"):
        SF.qk_norm_rotary(q, q, None, None, torch.zeros(4, 1, dtype=torch.int32), torch.ones(4))
    with pytest.raises(ValueError, match="heads, D"):
        SF.qk_norm_rotary(q[0], q, None, None, torch.zeros(4, 1, dtype=torch.int32), torch.ones(4))


@pytest.mark.gpu
def test_refusals():
    from segk import functional as SF
    from segk._lib import SegkError

    def t(*shape, dt=F32):
        return torch.zeros(*shape, dtype=dt, device="cuda")
    i32 = torch.int32
    q, k, w, p, f = t(2, 5, 4, 32), t(2, 5, 2, 32), t(32), t(5, 2, dt=i32), t(16)
    for args, kw, err in (
            ((q, t(2, 6, 2, 32), w, w, p, f), {}, ValueError),
            ((q, k.to(BF), w, w, p, f), {}, ValueError),
            ((q.half(), k.half(), w, w, p, f), {}, TypeError),
            ((q, k, t(16), w, p, f), {}, ValueError),
            ((q, k, w, w, t(4, 2, dt=i32), f), {}, ValueError),
            ((q, k, w, w, t(5, 5, dt=i32), f), {}, ValueError),
            ((q, k, w, w, t(5, 2, dt=torch.int16), f), {}, ValueError),
            ((q, k, w, w, p.cpu(), f), {}, ValueError),
            ((q, k, w, w, p, f.double()), {}, ValueError),
            ((q, k, w, w, p, t(15)), {}, ValueError),
            ((q, k, w, w, p, f), {"sections": (8, 9)}, ValueError),
            ((q, k, w, w, p, f), {"sections": (16,)}, ValueError),
            ((q, k, w, w, p, f), {"sections": (-4, 20)}, ValueError),
            ((q, k, w, w, p, t(18)), {}, SegkError),                      # more pairs than D / 2, not a multiple of 4
            ((q, k, w, w, p, f), {"eps": None}, ValueError),
            ((q, k, w, w, p, f), {"eps": -1.0}, SegkError),
            ((t(2, 5, 4, 20), None, None, None, p, t(4)), {}, SegkError),
            ((t(2, 5, 4, 264), None, None, None, p, f), {}, SegkError),
            ((q, k, w, w, p, f.clone().requires_grad_(True)), {}, ValueError)):
        with pytest.raises(err):
            SF.qk_norm_rotary(*args, **kw)
