"""Every library call of the attention and rotation operators, the sizing of their workspaces included, is made on the device
of their operands (occupancy is asked of the current device).  No GPU: the device and the library are stood in for."""
import contextlib

import pytest
import torch

from segk import ops


class OnDevice1(torch.Tensor):
    def get_device(self):
        return 1


def here(*shape):
    return torch.zeros(*shape).as_subclass(OnDevice1)


@pytest.mark.parametrize("current", [0, 1])
def test_library_calls_are_made_on_the_operands_device(monkeypatch, current):
    at, calls = [current], []

    @contextlib.contextmanager
    def device(index):
        before, at[0] = at[0], index
        yield
        at[0] = before

    def call(name, *args):
        calls.append((name, at[0]))
        return 64 if name.endswith("workspace") else 0
    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "call", call)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    q, k, out = here(1, 5, 4, 16), here(1, 6, 2, 16), here(1, 5, 4, 16)
    lse = ops.attention_fwd(q, k, k, out, 0.25, want_lse=True).as_subclass(OnDevice1)
    ops.attention_bwd(q, k, k, out, lse, out, 0.25)
    pos, freq, w = here(5, 1).int(), here(4), here(16)
    ops.qk_norm_rotary_fwd(q, out, w, w, pos, freq)
    ops.qk_norm_rotary_bwd(out, out, q, out, w, w, pos, freq)
    assert len(calls) >= 6 and all(index == 1 for _, index in calls), calls
    assert at[0] == current
