"""Every key and every row counts once, however the work is cut up: with equal scores every weight of a row is 1 / n (n: its open
keys), and one channel of a result is given to one key (of out and dq) or to one row (of dk and dv) at a time, so that a key or
row that is left out, taken twice or taken for another shows as a whole value and not as one part in n.

Bounds (u: half a step of the operands' type, V: of fp32): the probabilities of the forward pass are exactly 1, their sums exact
whole numbers, so that out has u + 4 V, and lse, |lse| < 16, log2 and two products, 8 V * 16.  Gradients take p from lse: its
2^-20 absolute is 2^-20 of p, with what is left of delta's rounding less than 2^-14; dq rounds its result, u, dk and dv P or dS
as well, 2 u, of values up to scale * p * 2 (dv: p)."""
import math

import pytest
import torch

from test_attention import BF, F32, make_masks

V = 2.0 ** -24


def attend_plain(q, k, v, dout, scale, mask, key, causal, skip_key=None, skip_row=None):
    """out, lse, dq, dk, dv in 64 bits on the CPU, leaving out one key or one row if asked."""
    N, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1:3]
    G = Hq // Hk
    open_ = open_pairs(N, Hq, Lq, Lk, mask, key, causal, "cpu")
    if skip_key is not None:
        open_ = open_ & (torch.arange(Lk) != skip_key)
    q, k, v, dout = (t.double().transpose(1, 2) for t in (q, k, v, dout))
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = (q @ kk.transpose(2, 3) * scale).masked_fill(~open_, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(torch.isinf(lse), 0)[..., None])
    out = p @ vv
    dp = dout @ vv.transpose(2, 3)
    ds = p * (dp - (dout * out).sum(-1, keepdim=True)) * scale
    dq = ds @ kk
    if skip_row is not None:
        p, ds = p.clone(), ds.clone()
        p[:, :, skip_row], ds[:, :, skip_row] = 0, 0
    dk, dv = (t.transpose(2, 3) @ x for t, x in ((ds, q), (p, dout)))
    dk, dv = (t.unflatten(1, (Hk, G)).sum(2) for t in (dk, dv))
    return {"lse": lse, **{n: t.transpose(1, 2) for n, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv))}}


def attend(q, k, v, dout, scale, mask, key, causal):
    from segk import functional as SF, ops
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = SF.attention(*leaves, mask, key, causal, scale)
    grads = torch.autograd.grad(out, leaves, dout)
    lse = ops.attention_fwd(q, k, v, torch.empty_like(q), scale, causal, mask, key, want_lse=True)
    return dict(zip(("out", "dq", "dk", "dv", "lse"), (out.detach(),) + grads + (lse,)))


def open_pairs(N, Hq, Lq, Lk, mask, key, causal, dev):
    open_ = torch.ones(N, Hq, Lq, Lk, dtype=torch.bool, device=dev)
    if mask is not None:
        open_ &= mask
    if key is not None:
        open_ &= key[:, None, None]
    if causal:
        open_ &= torch.arange(Lk, device=dev) <= torch.arange(Lq, device=dev)[:, None] + (Lk - Lq)
    return open_


class Worst:
    """The largest error in units of its bound, kept on the device until the end."""

    def __init__(self):
        self.at = {}

    def add(self, name, got, want, bound):
        e = ((got.double() - want).abs() / bound).nan_to_num(math.inf, math.inf, math.inf).max()
        self.at[name] = torch.maximum(self.at[name], e) if name in self.at else e

    def check(self):
        found = {n: float(e) for n, e in self.at.items()}
        assert all(e <= 1 for e in found.values()), found


def every_key(f, case, dt, dev):
    N, Lq, Lk, Hq, Hk, D, kind = case
    gen = torch.Generator().manual_seed(81)
    mask, key, causal = make_masks(kind, N, Hq, Lq, Lk, gen, dev)
    n = torch.zeros(N, Hq, Lq, dtype=torch.int64, device=dev)
    for i in range(0, Lq, 64):       # (a whole map's pairs at once are too many)
        rows = None if mask is None else mask[:, :, i:i + 64] if mask.shape[2] > 1 else mask
        at = open_pairs(N, Hq, min(64, Lq - i), Lk, rows, key, False, dev)
        if causal:
            at &= torch.arange(Lk, device=dev) <= torch.arange(i, min(Lq, i + 64), device=dev)[:, None] + (Lk - Lq)
        n[:, :, i:i + 64] = at.sum(-1)
    p = torch.where(n > 0, 1.0 / n.double(), 0.0).transpose(1, 2)[..., None]       # [N, Lq, Hq, 1]
    u, scale = torch.finfo(dt).eps / 2, 0.5
    q = torch.zeros(N, Lq, Hq, D, dtype=dt, device=dev)
    dout = torch.ones_like(q)
    k, v = (torch.zeros(N, Lk, Hk, D, dtype=dt, device=dev) for _ in range(2))
    eye = torch.eye(D, dtype=dt, device=dev)[:, None]
    worst, some = Worst(), p + (p == 0)
    for j0 in range(0, Lk, D):
        j1 = min(Lk, j0 + D)
        for t in (k, v):
            t.zero_()
            t[:, j0:j1] = eye[:j1 - j0]
        got = f(q, k, v, dout, scale, mask, key, causal)
        at = torch.zeros(N, Hq, Lq, D, dtype=torch.bool, device=dev)
        at[..., :j1 - j0] = True
        if mask is not None:
            at[..., :j1 - j0] &= mask[..., j0:j1] if mask.shape[3] > 1 else mask
        if key is not None:
            at[..., :j1 - j0] &= key[:, None, None, j0:j1]
        if causal:
            at[..., :j1 - j0] &= torch.arange(j0, j1, device=dev) <= torch.arange(Lq, device=dev)[:, None] + (Lk - Lq)
        at = at.transpose(1, 2).double()
        worst.add("out", got["out"], at * p, (u + 4 * V) * some)
        delta = (at * p).sum(-1, keepdim=True)
        worst.add("dq", got["dq"], scale * at * p * (1 - delta), scale * some * (u + 2.0 ** -14))
        if j0 == 0:
            live = n > 0
            worst.add("lse", got["lse"][live], n[live].double().log(), 8 * V * 16)
            assert bool((got["lse"][~live] == -math.inf).all())
    worst.check()


def every_row(f, case, dt, dev):
    N, Lq, Lk, Hq, Hk, D, kind = case
    gen = torch.Generator().manual_seed(83)
    mask, key, causal = make_masks(kind, N, Hq, Lq, Lk, gen, dev)
    G, u, scale = Hq // Hk, torch.finfo(dt).eps / 2, 0.5
    k = torch.zeros(N, Lk, Hk, D, dtype=dt, device=dev)
    v = (torch.randint(0, 2, (N, Lk, Hk, D), generator=gen) * 2 - 1).to(dev).to(dt)
    worst = Worst()
    rows = Lq * G                    # of one key / value head: token r // G, head r % G of the group
    for r0 in range(0, rows, D):
        r = torch.arange(r0, min(rows, r0 + D), device=dev)
        c = torch.arange(r.numel(), device=dev)
        one = torch.zeros(N, Lq, G, Hk, D, dtype=dt, device=dev)
        one[:, r // G, r % G, :, c] = 1
        one = one.transpose(2, 3).reshape(N, Lq, Hq, D)
        got = f(one, k, v, one, scale, mask, key, causal)
        # [N, Hk, rows of the window, Lk]
        open_ = torch.ones(N, Hk, r.numel(), Lk, dtype=torch.bool, device=dev)
        if mask is not None:
            m = mask.expand(N, Hq, mask.shape[2], Lk).unflatten(1, (Hk, G))
            open_ &= m[:, :, r % G, (r // G) if mask.shape[2] > 1 else torch.zeros_like(r)]
        if key is not None:
            open_ &= key[:, None, None]
        if causal:
            open_ &= torch.arange(Lk, device=dev) <= (r // G)[:, None] + (Lk - Lq)
        n = open_.sum(-1, keepdim=True)
        p = torch.where(open_, 1.0 / n.clamp(min=1).double(), 0.0)
        vv = v[..., c].permute(0, 2, 3, 1).double()                    # [N, Hk, window, Lk]: dp of the window's rows
        dk = scale * p * (vv - (p * vv).sum(-1, keepdim=True))
        size = (p + (p == 0))
        for name, want, bound in (("dv", p, size * (2 * u + 2.0 ** -14)), ("dk", dk, 2 * scale * size * (2 * u + 2.0 ** -14))):
            worst.add(name, got[name][..., c].permute(0, 2, 3, 1), want, bound)
    worst.check()


KEYS = [
    (1, 1, 1, 1, 1, 8, ""),
    (1, 1, 70001, 8, 2, 64, "key"),
    (2, 2, 33333, 4, 4, 128, "causal"),
    (1, 1, 2053, 8, 2, 64, ""),
    (1, 5, 4099, 2, 2, 128, ""),
    (2, 21, 9001, 4, 4, 32, "pair"),
    (2, 21, 3001, 4, 2, 96, "pair key"),
    (1, 600, 4100, 104, 104, 128, ""),
    (1, 700, 1900, 8, 2, 64, "causal"),
    (8, 150, 300, 2, 1, 64, "causal key"),
    (4, 300, 700, 8, 4, 64, "key"),
    (2, 1089, 1089, 4, 4, 64, "causal"),
    (1, 1500, 1500, 8, 1, 64, "causal"),       # 94 tiles of rows
    (1, 40, 9000, 2, 2, 32, "causal"),         # 71 tiles of keys
]
ROWS = [
    (1, 1, 70, 1, 1, 8, ""),
    (1, 1500, 7, 2, 1, 64, ""),
    (1, 2100, 600, 104, 104, 128, ""),
    (1, 2100, 600, 104, 104, 128, "key"),
    (1, 1900, 700, 2, 2, 128, "causal"),
    (1, 700, 1900, 8, 2, 64, "causal"),
    (2, 5, 130, 200, 2, 32, "causal key"),
    (2, 21, 900, 2, 2, 32, "pair"),
    (2, 150, 333, 4, 4, 128, "pair key"),
    (6, 700, 300, 4, 4, 32, "key"),
    (2, 300, 70, 6, 2, 40, "causal"),
    (2, 1089, 1089, 4, 4, 64, "causal"),
    (1, 1500, 1500, 8, 1, 64, "causal"),
    (1, 40, 9000, 2, 2, 32, "causal"),
    (1, 9000, 40, 2, 2, 32, "causal"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", KEYS, ids=[str(c) for c in KEYS])
def test_every_key_counts_once(case, dt):
    every_key(attend, case, dt, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", ROWS, ids=[str(c) for c in ROWS])
def test_every_row_counts_once(case, dt):
    every_row(attend, case, dt, "cuda")


@pytest.mark.parametrize("kind", ["", "key", "pair", "causal"])
def test_a_key_or_row_left_out_is_seen(kind):
    """The checks themselves, on plain results, and on plain results that leave out one key or one row."""
    case = (1, 20, 300, 4, 2, 16, kind)
    every_key(attend_plain, case, F32, "cpu")
    every_row(attend_plain, case, F32, "cpu")
    with pytest.raises(AssertionError):
        every_key(lambda *a: attend_plain(*a, skip_key=299), case, F32, "cpu")
    with pytest.raises(AssertionError):
        every_row(lambda *a: attend_plain(*a, skip_row=18), case, F32, "cpu")
