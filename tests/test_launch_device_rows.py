"""The row operators launch with the tensors' device current and on its stream, whatever device
the caller has current (on the CPU, with stand-ins for the tensors and the library call)."""
from __future__ import annotations

import contextlib

import pytest
import torch

from test_launch_device import _OnGpu1, _i32


class _Tensor(_OnGpu1):
    def element_size(self):
        return 1

    def __getattr__(self, name):  # (what follows the launch)
        raise AttributeError(name)


def _pools():
    return _Tensor(8, 2, 8, 16, 8), _Tensor(8, 2, 64, 16)


CALLS = {
    "ivakv_cross_attn": lambda o: o.paged_cross_attention(
        _Tensor(6, 4, 64), *_pools(), _i32(2, 4), _i32(2), _i32(3), max_query_len=3),
    "ivakv_prefix_decode_attn": lambda o: o.paged_prefix_decode_attention(
        _Tensor(2, 4, 64), *_pools(), _i32(2, 4), _i32(2), _i32(2), _i32(1), max_group=2),
}


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("entry", CALLS)
def test_row_launch_enters_the_tensors_device(iva, monkeypatch, entry, current):
    ops, state, seen = iva.ops, {"current": current}, []

    @contextlib.contextmanager
    def enter(dev):
        before, state["current"] = state["current"], dev.index
        yield
        state["current"] = before

    monkeypatch.setattr(torch.cuda, "device", enter)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
    monkeypatch.setattr(ops, "_current_device", lambda: state["current"], raising=False)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(ops, "_sized_workspace", lambda w, dev, n: _Tensor(max(n, 1)))
    monkeypatch.setattr(torch, "empty_like", lambda t: t)
    monkeypatch.setitem(ops._abi._FUNCS, entry,
                        lambda *a: seen.append((entry, state["current"], a[-1])) or ops._abi.OK)
    CALLS[entry](ops)
    assert seen == [(entry, 1, 101)]
    assert state["current"] == current
