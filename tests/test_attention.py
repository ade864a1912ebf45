"""Multi-head attention (segk.functional.attention): forward and gradients against the definition in 64 bits.

Bounds, element by element.  u = half a step of the operand type (eps / 2: bf16 2^-8, fp32 2^-24), v = 2^-24.
  rel     relative error of a probability from fp32 arithmetic: scores of magnitude S carry (D + 4) v S' (S' = the sum of
          the products' magnitudes times scale) plus the rounding of s * log2(e) and of lse (2 v S each way), exp2 4 v, and
          the row sum of Lk terms Lk v
  out     sum_j p|v| (u + rel) + u|out|            (probabilities rounded to the operand type, result rounded)
  dv      sum_i p|dout| (u + rel + rows v) + u|dv|
  ds      p (e_dp + e_delta) + |ds|(u + rel),  e_dp = D v sum|dout||v|,  e_delta = sum|dout| e_out + D v sum|dout||out|
  dq, dk  scale sum ds-error |k| (|q|) + (terms) v scale sum|ds||k| + u|dq|
Every bound is doubled once for second-order terms.
  underflow  probabilities below 2^-126 are zero in fp32: a gradient element misses at most (rows or keys) * 2^-126 *
          |dp - delta| |q or k| scale; 2^12 * 2^-126 covers 40 rows * 25 * 4 of the one test that gets there
          (test_large_scores: |dp - delta| <= 25, |q| <= 4, scale 1) and lies 30 orders below any other value here"""
import math

import pytest
import torch

BF, F32 = torch.bfloat16, torch.float32
V = 2.0 ** -24
FLOOR = 2.0 ** (12 - 126)


def make_masks(kind, N, Hq, Lq, Lk, gen, dev):
    """(mask, key_mask, causal)."""
    def rnd(*s):
        return torch.rand(*s, generator=gen).to(dev)
    mask = key = None
    causal = "causal" in kind
    if "key" in kind:
        key = rnd(N, Lk) < 0.7
        if N > 1:
            key[0] = False              # an image that is all padding
        key[N - 1, Lk - 1] = True
    if "pair" in kind:
        mask = rnd(N, 1, Lq, Lk) < 0.6
        mask[:, :, ::5] = False          # rows that are left nothing
    if "heads" in kind:
        mask = rnd(1, Hq, Lq, Lk) < 0.6
    if "rows" in kind:
        mask = (rnd(N, 1, Lq, 1) < 0.7)
    if "odd" in kind:                    # every second byte of a wider tensor
        mask = (rnd(N, Hq, Lq, 2 * Lk) < 0.8)[..., ::2]
    return mask, key, causal


def reference(q, k, v, dout, mask, key, causal, scale, dt):
    """float64 results and bounds, on the tensors' device."""
    N, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    u = torch.finfo(dt).eps / 2
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    dev = q.device
    res = {n: torch.zeros(s, dtype=torch.float64, device=dev) for n, s in
           (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", k.shape), ("lse", (N, Hq, Lq)))}
    tol = {n: torch.zeros_like(t) for n, t in res.items()}
    acc = {}
    for n in range(N):
        for h in range(Hq):
            g = h * Hk // Hq
            open_ = torch.ones(Lq, Lk, dtype=torch.bool, device=dev)
            if mask is not None:
                open_ &= mask.expand(N, Hq, Lq, Lk)[n, h]
            if key is not None:
                open_ &= key[n]
            if causal:
                i = torch.arange(Lq, device=dev).unsqueeze(1)
                open_ &= torch.arange(Lk, device=dev) <= i + (Lk - Lq)
            live = torch.ones(Lk, dtype=torch.bool, device=dev) if key is None else key[n]
            kk = torch.where(live.unsqueeze(1), k[n, :, g], torch.zeros((), dtype=torch.float64, device=dev))
            vv = torch.where(live.unsqueeze(1), v[n, :, g], torch.zeros((), dtype=torch.float64, device=dev))
            qq, dd = q[n, :, h], dout[n, :, h]
            any_ = open_.any(1, keepdim=True)
            qq, dd = torch.where(any_, qq, 0.0), torch.where(any_, dd, 0.0)
            s = (qq @ kk.t()) * scale
            sm = (qq.abs() @ kk.abs().t()) * scale
            s = torch.where(open_, s, -math.inf)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.where(open_ & any_, torch.exp(s - lse), 0.0)
            o = p @ vv
            big = float(sm.max()) if sm.numel() else 0.0
            rel = 2 * ((D + 4) * V * big + 4 * V * big + 4 * V + Lk * V)
            e_out = 2 * ((p @ vv.abs()) * (u + rel) + u * o.abs())
            dp = dd @ vv.t()
            delta = (dd * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e_dp = D * V * (dd.abs() @ vv.abs().t())
            e_delta = (dd.abs() * e_out).sum(1, keepdim=True) + D * V * (dd * o).abs().sum(1, keepdim=True)
            e_ds = 2 * (p * (e_dp + e_delta) + ds.abs() * (u + rel))
            res["out"][n, :, h], tol["out"][n, :, h] = o, e_out
            res["lse"][n, h] = lse.squeeze(1)
            tol["lse"][n, h] = 2 * rel + 4 * V * lse.squeeze(1).abs().nan_to_num(0, 0, 0)
            dq = scale * ds @ kk
            res["dq"][n, :, h] = dq
            tol["dq"][n, :, h] = 2 * scale * (e_ds @ kk.abs() + Lk * V * (ds.abs() @ kk.abs())) + 2 * u * dq.abs()
            res["dk"][n, :, g] += scale * ds.t() @ qq
            tol["dk"][n, :, g] += 2 * scale * (e_ds.t() @ qq.abs() + 2 * Lq * Hq // Hk * V * (ds.abs().t() @ qq.abs()))
            res["dv"][n, :, g] += p.t() @ dd
            tol["dv"][n, :, g] += 2 * (p.t() @ dd.abs()) * (u + rel + 2 * Lq * Hq // Hk * V)
    for name in ("dk", "dv"):
        tol[name] += 2 * u * res[name].abs()
    return res, tol


def check(got, res, tol, what):
    for name, g in got.items():
        r, t = res[name], tol[name]
        g = g.double()
        assert g.shape == r.shape, (what, name, g.shape, r.shape)
        assert not torch.isnan(g).any(), "%s: NaN in %s" % (what, name)
        inf = torch.isinf(r)
        assert torch.equal(torch.isinf(g), inf) and torch.equal(g[inf], r[inf]), "%s: infinities of %s" % (what, name)
        bad = ((g - r).abs() > t + FLOOR) & ~inf
        if bad.any():
            i = int(((g - r).abs() / (t + FLOOR)).masked_fill(inf, 0).argmax())
            raise AssertionError("%s: %s off at %d of %d: got %g, want %g, bound %g" % (
                what, name, int(bad.sum()), g.numel(), g.flatten()[i], r.flatten()[i], t.flatten()[i]))


def make(N, Lq, Lk, Hq, Hk, D, dt, layout, seed, dev="cuda"):
    gen = torch.Generator().manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, generator=gen).to(dev).to(dt)
    if layout == "fused" and Lq == Lk:
        qkv = rnd(N, Lq, Hq + 2 * Hk, D)
        q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
    elif layout == "heads_first":
        q, k, v = rnd(N, Hq, Lq, D).transpose(1, 2), rnd(N, Hk, Lk, D).transpose(1, 2), rnd(N, Hk, Lk, D).transpose(1, 2)
    elif layout == "tokens_first":
        q, k, v = rnd(Lq, N, Hq, D).transpose(0, 1), rnd(Lk, N, Hk, D).transpose(0, 1), rnd(Lk, N, Hk, D).transpose(0, 1)
    elif layout == "channels_first":     # unit stride over the tokens: copied before the kernels
        q = rnd(N, Hq, D, Lq).permute(0, 3, 1, 2)
        k, v = rnd(N, Hk, D, Lk).permute(0, 3, 1, 2), rnd(N, Hk, D, Lk).permute(0, 3, 1, 2)
    else:
        q, k, v = rnd(N, Lq, Hq, D), rnd(N, Lk, Hk, D), rnd(N, Lk, Hk, D)
    return q, k, v, rnd(N, Lq, Hq, D), gen


CASES = [
    # N, Lq, Lk, Hq, Hk, D, masks, layout
    (1, 1, 1, 1, 1, 8, "", "plain"),
    (2, 1, 1, 2, 1, 64, "key", "plain"),
    (2, 33, 33, 2, 2, 32, "", "fused"),
    (1, 64, 64, 1, 1, 64, "", "plain"),
    (1, 128, 129, 1, 1, 128, "", "plain"),
    (2, 65, 200, 2, 1, 40, "", "heads_first"),
    (2, 130, 61, 6, 2, 72, "", "tokens_first"),
    (1, 257, 257, 3, 3, 96, "", "channels_first"),
    (1, 31, 1000, 4, 1, 16, "", "plain"),
    (1, 1, 2053, 8, 2, 64, "", "plain"),
    (1, 5, 4099, 2, 2, 128, "", "heads_first"),
    (1, 1500, 7, 2, 1, 64, "", "plain"),
    (3, 100, 161, 2, 1, 24, "key", "plain"),
    (2, 90, 290, 4, 2, 64, "pair", "plain"),
    (2, 21, 900, 2, 2, 32, "pair key", "heads_first"),
    (2, 70, 70, 4, 2, 128, "heads", "fused"),
    (2, 40, 50, 2, 1, 80, "rows", "plain"),
    (1, 40, 50, 2, 1, 56, "odd", "plain"),
    (2, 200, 200, 4, 2, 64, "causal", "fused"),
    (1, 70, 300, 2, 1, 32, "causal", "plain"),
    (2, 300, 70, 2, 2, 64, "causal", "plain"),
    (1, 1, 333, 4, 4, 128, "causal", "plain"),
    (2, 150, 150, 3, 1, 88, "causal key", "fused"),
    (1, 1025, 129, 2, 1, 128, "causal pair", "plain"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=[str(c) for c in CASES])
def test_forward_and_gradients(case, dt):
    from segk import functional as SF, ops
    N, Lq, Lk, Hq, Hk, D, kind, layout = case
    q, k, v, dout, gen = make(N, Lq, Lk, Hq, Hk, D, dt, layout, 11)
    mask, key, causal = make_masks(kind, N, Hq, Lq, Lk, gen, "cuda")
    res, tol = reference(q, k, v, dout, mask, key, causal, D ** -0.5, dt)
    with torch.no_grad():
        check({"out": SF.attention(q, k, v, mask, key, causal)}, res, tol, "inference")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = SF.attention(*leaves, mask, key, causal)
    assert out.dtype == dt and out.is_contiguous()
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    check({"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}, res, tol, "training")
    if layout == "plain":
        got = torch.empty_like(q)
        lse = ops.attention_fwd(q, k, v, got, D ** -0.5, causal, mask, key, want_lse=True)
        check({"out": got, "lse": lse}, res, tol, "ops")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
def test_closed_keys_may_hold_anything(dt):
    """NaN and infinities where key_mask closes, and in the rows and gradients of queries that are left nothing."""
    from segk import functional as SF
    N, Lq, Lk, Hq, Hk, D = 2, 70, 150, 2, 1, 64
    q, k, v, dout, gen = make(N, Lq, Lk, Hq, Hk, D, dt, "plain", 3)
    key = torch.rand(N, Lk, generator=gen).cuda() < 0.5
    mask = torch.ones(N, 1, Lq, 1, dtype=torch.bool, device="cuda")
    mask[:, :, ::7] = False
    res, tol = reference(q, k, v, dout, mask, key, False, 0.3, dt)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2, q2, d2 = k.clone(), v.clone(), q.clone(), dout.clone()
        k2[~key], v2[~key] = bad, bad
        d2[:, ::7] = bad
        q2[:, ::7] = bad
        leaves = [t.requires_grad_(True) for t in (q2, k2, v2)]
        out = SF.attention(*leaves, mask, key, scale=0.3)
        grads = torch.autograd.grad(out, leaves, d2)
        check(dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads)), res, tol, str(bad))
        assert float(out.detach()[:, ::7].abs().max()) == 0 and float(grads[0][:, ::7].abs().max()) == 0
        assert float(grads[1][~key].abs().max()) == 0 and float(grads[2][~key].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
def test_large_scores(dt):
    """Scores of several hundreds, whose exponentials only exist relative to the row maximum, growing along the keys (the
    running maximum moves at every step) and falling."""
    from segk import functional as SF
    N, Lq, Lk, H, D = 1, 40, 500, 1, 32
    q, k, v, dout, _ = make(N, Lq, Lk, H, H, D, dt, "plain", 5)
    ramp = torch.linspace(-20, 20, Lk, device="cuda").reshape(1, Lk, 1, 1)
    for sign in (1, -1):
        q2 = q.abs()
        k2 = (k.float() + sign * ramp).to(dt)
        res, tol = reference(q2, k2, v, dout, None, None, False, 1.0, dt)
        leaves = [t.detach().requires_grad_(True) for t in (q2, k2, v)]
        out = SF.attention(*leaves, scale=1.0)
        grads = torch.autograd.grad(out, leaves, dout)
        check(dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads)), res, tol, str(sign))


@pytest.mark.gpu
def test_nan_and_infinity_stay_visible():
    from segk import functional as SF
    q, k, v, _, _ = make(1, 40, 100, 1, 1, 32, F32, "plain", 5)
    q[0, 3] = math.nan
    v[0, 7, 0, 5] = math.inf
    out = SF.attention(q, k, v)
    assert torch.isnan(out[0, 3]).all()
    assert torch.isinf(out[0, 4, 0, 5]) and torch.isfinite(out[0, 4, 0, :5]).all()


@pytest.mark.gpu
def test_gradients_against_differences():
    from segk import functional as SF
    q, k, v, dout, gen = make(1, 9, 14, 2, 1, 16, F32, "plain", 9)
    mask, key, _ = make_masks("pair key", 1, 2, 9, 14, gen, "cuda")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(SF.attention(*leaves, mask, key), leaves, dout)
    eps = 2.0 ** -6
    for which in range(3):
        step = torch.randn(leaves[which].shape, generator=gen).cuda()
        with torch.no_grad():
            at = [[t + sign * eps * step if i == which else t for i, t in enumerate(leaves)] for sign in (1, -1)]
            hi, lo = (float((SF.attention(*a, mask, key).double() * dout.double()).sum()) for a in at)
        want = float((grads[which].double() * step.double()).sum())
        # central differences: third-order term eps^2 times sums of O(1) values, and fp32 rounding of both sides / (2 eps)
        size = float(dout.abs().sum()) * (eps ** 2 * 4 + 2 ** -22 / eps)
        assert abs((hi - lo) / (2 * eps) - want) < size, (which, (hi - lo) / (2 * eps), want, size)


@pytest.mark.gpu
def test_broadcast_and_shared_operands():
    """Keys shared by the images through a stride of zero; one tensor as key and value; only some gradients wanted."""
    from segk import functional as SF
    N, Lq, Lk, Hq, Hk, D = 3, 20, 75, 4, 2, 32
    q, k, v, dout, _ = make(N, Lq, Lk, Hq, Hk, D, F32, "plain", 21)
    one = k[:1].clone().requires_grad_(True)
    both = one.expand(N, Lk, Hk, D)
    res, tol = reference(q, both.detach(), both.detach(), dout, None, None, False, D ** -0.5, F32)
    out = SF.attention(q, both, both)
    (got,) = torch.autograd.grad(out, one, dout)
    want = (res["dk"] + res["dv"]).sum(0, keepdim=True)
    bound = (tol["dk"] + tol["dv"]).sum(0, keepdim=True) + 8 * V * (res["dk"].abs() + res["dv"].abs()).sum(0, keepdim=True)
    assert ((got.double() - want).abs() <= bound).all()
    qg = q.clone().requires_grad_(True)
    (dq,) = torch.autograd.grad(SF.attention(qg, both.detach(), both.detach()), qg, dout)
    check({"dq": dq}, res, tol, "dq alone")
    dq2 = torch.autograd.grad(SF.attention(qg, both.detach(), both.detach()).sum(), qg)[0]     # an expanded gradient
    assert torch.isfinite(dq2).all()


@pytest.mark.gpu
def test_empty_sizes():
    from segk import functional as SF
    for N, Lq, Lk in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        q = torch.randn(N, Lq, 4, 16, device="cuda", requires_grad=True)
        k = torch.randn(N, Lk, 2, 16, device="cuda", requires_grad=True)
        v = torch.randn(N, Lk, 2, 16, device="cuda", requires_grad=True)
        out = SF.attention(q, k, v)
        assert out.shape == q.shape and not out.any()
        grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
        assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, (q, k, v)))


@pytest.mark.gpu
def test_same_bits_every_time():
    from segk import functional as SF
    for case in ((2, 300, 300, 4, 2, 64, ""), (1, 3, 5000, 4, 2, 64, "pair")):
        N, Lq, Lk, Hq, Hk, D, kind = case
        q, k, v, dout, gen = make(N, Lq, Lk, Hq, Hk, D, BF, "plain", 2)
        mask, key, _ = make_masks(kind, N, Hq, Lq, Lk, gen, "cuda")
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        runs = []
        for _ in range(3):
            out = SF.attention(*leaves, mask, key)
            runs.append((out.detach(),) + torch.autograd.grad(out, leaves, dout))
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


@pytest.mark.gpu
def test_streams_and_graph():
    """Forward and backward recorded into one graph and replayed between eager calls, on a stream of its own; two graphs
    that are replayed in turn."""
    from segk import functional as SF
    sets = []
    side = torch.cuda.Stream()
    for seed, (Lq, Lk) in ((1, (3, 4000)), (2, (200, 260))):
        q, k, v, dout, _ = make(2, Lq, Lk, 4, 2, 64, BF, "plain", seed)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]

        def step(leaves=leaves, dout=dout):
            out = SF.attention(*leaves)
            return (out.detach(),) + torch.autograd.grad(out, leaves, dout)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = step()
        sets.append((graph, res, leaves, dout, step))
    for turn in range(4):
        for graph, res, leaves, dout, step in sets:
            with torch.no_grad():
                for t in leaves:
                    t.copy_(torch.randn_like(t))
            graph.replay()
            got = [t.clone() for t in res]
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


@pytest.mark.gpu
def test_far_offsets():
    """Tokens whose rows lie more than 2^32 bytes apart."""
    from segk import functional as SF
    need = 10 * (1 << 30)
    if torch.cuda.get_device_properties(0).total_memory < 4 * need:
        pytest.skip("needs 10 GiB")
    L, D = 150, 64
    wide = torch.empty(need // 2, dtype=BF, device="cuda")
    ld = (wide.numel() // (2 * L)) // 64 * 64
    q, k, v, dout, _ = make(1, 10, L, 1, 1, D, BF, "plain", 4)
    far_k = torch.as_strided(wide, (1, L, 1, D), (0, ld, D, 1), 0)
    far_v = torch.as_strided(wide, (1, L, 1, D), (0, ld, D, 1), L * ld)
    far_k.copy_(k)
    far_v.copy_(v)
    res, tol = reference(q, k, v, dout, None, None, False, D ** -0.5, BF)
    leaves = [q.requires_grad_(True), far_k.detach().requires_grad_(True), far_v.detach().requires_grad_(True)]
    out = SF.attention(*leaves)
    grads = torch.autograd.grad(out, leaves, dout)
    check(dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads)), res, tol, "far")


# Sizes at which the work is dealt out in other ways: a last round of workgroups that is cut up (of queries, of keys; rounds
# are 256 times 1 to 5 workgroups), parts of equal length under the diagonal, images dealt out in turns, groups of more heads
# than a tile has rows, one token against a long cache.
DEALT = [
    (1, 600, 4100, 104, 104, 128, "", "plain"),
    (1, 2100, 600, 104, 104, 128, "", "plain"),
    (1, 600, 4100, 104, 104, 120, "pair", "plain"),
    (1, 2100, 600, 104, 104, 128, "key", "plain"),
    (1, 700, 1900, 8, 2, 64, "causal", "plain"),
    (1, 1900, 700, 2, 2, 128, "causal", "heads_first"),
    (8, 150, 300, 2, 1, 64, "causal key", "plain"),
    (4, 300, 700, 8, 4, 64, "key", "fused"),
    (6, 700, 300, 4, 4, 32, "key", "plain"),
    (2, 150, 333, 4, 4, 128, "pair key", "plain"),
    (1, 7, 200, 40, 1, 64, "", "plain"),
    (2, 5, 130, 200, 2, 32, "causal key", "plain"),
    (1, 1, 70001, 8, 2, 64, "key", "plain"),
    (2, 2, 33333, 4, 4, 128, "causal", "tokens_first"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", DEALT, ids=[str(c) for c in DEALT])
def test_ways_of_dealing_out(case, dt):
    from segk import functional as SF
    N, Lq, Lk, Hq, Hk, D, kind, layout = case
    q, k, v, dout, gen = make(N, Lq, Lk, Hq, Hk, D, dt, layout, 31)
    mask, key, causal = make_masks(kind, N, Hq, Lq, Lk, gen, "cuda")
    res, tol = reference(q, k, v, dout, mask, key, causal, D ** -0.5, dt)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = SF.attention(*leaves, mask, key, causal)
    grads = torch.autograd.grad(out, leaves, dout)
    check(dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads)), res, tol, str(case))


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls on two streams that run side by side, each with its own workspace, against the same calls one after the other."""
    from segk import functional as SF
    sets = []
    for seed, (Lq, Lk, kind) in ((1, (2, 9000, "key")), (2, (500, 700, "causal"))):
        q, k, v, dout, gen = make(2, Lq, Lk, 4, 2, 64, BF, "plain", seed)
        mask, key, causal = make_masks(kind, 2, 4, Lq, Lk, gen, "cuda")
        sets.append(([t.requires_grad_(True) for t in (q, k, v)], dout, key, causal))

    def step(leaves, dout, key, causal):
        out = SF.attention(*leaves, None, key, causal)
        return (out.detach(),) + torch.autograd.grad(out, leaves, dout)
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(8):
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(step(*s))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i % 2])), i


# ------------------------------------------------------------- refusals ----
def _meta(*shape, dt=F32):
    return torch.zeros(*shape, dtype=dt)


def test_refuses_cpu_tensors_and_bad_shapes():
    from segk import functional as SF
    q, k = _meta(1, 4, 2, 16), _meta(1, 5, 2, 16)
    with pytest.raises(ValueError, match="GPU"):
        SF.attention(q, k, k)
    with pytest.raises(ValueError, match="heads, D"):
        SF.attention(q[0], k, k)


@pytest.mark.gpu
def test_refusals():
    from segk import functional as SF, ops
    from segk._lib import SegkError

    def t(*shape, dt=F32):
        return torch.zeros(*shape, dtype=dt, device="cuda")
    q, k = t(2, 4, 4, 16), t(2, 5, 2, 16)
    for args, kw, err in (
            ((q, k, t(2, 6, 2, 16)), {}, ValueError),                          # key and value lengths differ
            ((q, t(2, 5, 3, 16), t(2, 5, 3, 16)), {}, ValueError),             # 4 heads over 3
            ((q, t(1, 5, 2, 16), t(1, 5, 2, 16)), {}, ValueError),             # images
            ((q, k.to(BF), k.to(BF)), {}, ValueError),                         # types
            ((q.half(), k.half(), k.half()), {}, TypeError),
            ((t(2, 4, 4, 12), t(2, 5, 2, 12), t(2, 5, 2, 12)), {}, SegkError),   # head sizes
            ((t(2, 4, 4, 136), t(2, 5, 2, 136), t(2, 5, 2, 136)), {}, SegkError),
            ((q, k, k), {"scale": 0.0}, SegkError),
            ((q, k, k), {"scale": -1.0}, SegkError),
            ((q, k, k), {"scale": math.inf}, SegkError),
            ((q, k, k), {"scale": math.nan}, SegkError),
            ((q, k, k), {"mask": t(2, 4, 4, 5)}, ValueError),                  # not bool
            ((q, k, k), {"mask": t(4, 5, dt=torch.bool)}, ValueError),
            ((q, k, k), {"mask": t(2, 4, 4, 6, dt=torch.bool)}, ValueError),
            ((q, k, k), {"mask": t(2, 4, 4, 5, dt=torch.bool).cpu()}, ValueError),
            ((q, k, k), {"key_mask": t(2, 4, dt=torch.bool)}, ValueError),
            ((q, k, k), {"key_mask": t(2, 5)}, ValueError)):
        with pytest.raises(err):
            SF.attention(*args, **kw)
    with pytest.raises(ValueError, match="aligned"):
        ops.attention_fwd(t(2, 4, 4, 17)[..., 1:], k, k, t(2, 4, 4, 16), 1.0)
    x = q.clone().requires_grad_(True)
    out = SF.attention(x, k, k)
    (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
