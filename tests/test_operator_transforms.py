"""attention and qk_norm_rotary under torch's own transforms: a recorded module (torch.jit.trace) computes what the call does,
and forward-mode differentiation, which the operators do not have, is refused rather than answered with no tangent.  On the
CPU with plain forms in the launches' place, and on the GPU as they are."""
import warnings

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from segk import functional as SF, ops


def _plain_attention(q, k, v, out, scale, causal=False, mask=None, key_mask=None, want_lse=False, **kw):
    # (numpy, which torch cannot see, as it cannot see a kernel's launch)
    n = [np.asarray(t.detach()) for t in (q, k, v)]
    g = q.shape[2] // k.shape[2]
    s = np.einsum("nihd,njhd->nhij", n[0], n[1].repeat(g, 2)) * scale
    if key_mask is not None:
        s = np.where(np.asarray(key_mask)[:, None, None], s, -np.inf)
    e = np.exp(s - s.max(-1, keepdims=True))
    out.detach().numpy()[...] = np.einsum("nhij,njhd->nihd", e / e.sum(-1, keepdims=True), n[2].repeat(g, 2))
    return torch.from_numpy(np.log(np.exp(s).sum(-1))) if want_lse else None


def _plain_rotary(q, k, q_weight, k_weight, positions, inv_freq, sections=None, eps=1e-6, interleaved=False):
    f = float(np.asarray(positions).sum()) + float(np.asarray(inv_freq).sum())
    res = []
    for x, w in ((q, q_weight), (k, k_weight)):
        res.append(torch.empty_like(x))
        res[-1].numpy()[...] = np.asarray(x.detach()) * np.asarray(w.detach()) * f
    return tuple(res)


def _attention_inputs(dev, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(2, n, h, 16, generator=gen).to(dev) for n, h in ((7, 4), (9, 2), (9, 2))] + \
        [(torch.rand(2, 9, generator=gen) < 0.7).to(dev)]


def _rotary_inputs(dev, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(2, 6, h, 16, generator=gen).to(dev) for h in (4, 2)] + \
        [torch.randn(16, generator=gen).to(dev) for _ in range(2)] + \
        [torch.randint(0, 50, (6, 2), generator=gen).to(dev), torch.rand(8, generator=gen).to(dev)]


class Attention(torch.nn.Module):
    def forward(self, q, k, v, key_mask):
        return SF.attention(q, k, v, key_mask=key_mask, scale=0.3)


class Rotary(torch.nn.Module):
    def forward(self, q, k, wq, wk, pos, freq):
        return SF.qk_norm_rotary(q, k, wq, wk, pos, freq, sections=(4, 4))


KINDS = [(Attention, _attention_inputs), (Rotary, _rotary_inputs)]


def recorded(module, inputs, dev):
    """The module recorded on one set of inputs, run on another, with and without gradients wanted."""
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with torch.no_grad():
            traced = torch.jit.trace(module(), tuple(inputs(dev, 1)))
        for seed in (2, 3):
            args = inputs(dev, seed)
            want = module()(*args)
            got = traced(*args)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert torch.equal(a, b)


def dual(module, inputs, dev):
    args = inputs(dev, 4)
    with torch.no_grad(), fwAD.dual_level():
        args[0] = fwAD.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            module()(*args)


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(ops, "attention_fwd", _plain_attention)
    monkeypatch.setattr(ops, "qk_norm_rotary_fwd", _plain_rotary)


@pytest.mark.parametrize("module,inputs", KINDS)
def test_recorded_module_on_the_cpu(plain, module, inputs):
    recorded(module, inputs, "cpu")


@pytest.mark.parametrize("module,inputs", KINDS)
def test_forward_mode_is_refused_on_the_cpu(plain, module, inputs):
    dual(module, inputs, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("module,inputs", KINDS)
def test_recorded_module(module, inputs):
    recorded(module, inputs, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("module,inputs", KINDS)
def test_forward_mode_is_refused(module, inputs):
    dual(module, inputs, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("module,inputs", KINDS)
def test_recorded_without_gradients_run_with_them(module, inputs):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with torch.no_grad():
            traced = torch.jit.trace(module(), tuple(inputs("cuda", 1)))
        args = inputs("cuda", 2)
        leaves = [t.requires_grad_(True) for t in args[:3]]
        grads = []
        for f in (module(), traced):
            out = f(*args)
            out = out if isinstance(out, tuple) else (out,)
            grads.append(torch.autograd.grad(sum(t.square().sum() for t in out), leaves))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
