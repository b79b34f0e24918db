"""How long the bucket maps live that `ops.attention_relpos` hands to its kernels, and who shares them.  On the CPU: the launches are replaced by a stub."""
import contextlib
import gc
import types
import weakref

import pytest
import torch

from synergize_motion_appearance_amd import lib as L
from synergize_motion_appearance_amd import ops, train_ops
from synergize_motion_appearance_amd.tape import Tape


@pytest.fixture
def calls(monkeypatch):
    """attention_relpos on CPU tensors: a launch only leaves its name and the map's address here"""
    seen = []

    def call(fn, d, index):
        seen.append((fn.__name__, d.map))
        return 0
    monkeypatch.setattr(ops, "_call", call)
    monkeypatch.setattr(ops, "_dev", lambda *a, **kw: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(synchronize=lambda: None))
    monkeypatch.setattr(torch.cuda, "device", lambda *a: contextlib.nullcontext())
    return seen


def test_the_tape_keeps_the_map(calls, monkeypatch):
    """a RelPos that nobody holds after the forward: its map is still there when the backward reads it"""
    maps, on = [], ops.RelPos.on

    def watched(self, device):
        t = on(self, device)
        maps.append(weakref.ref(t))
        return t
    monkeypatch.setattr(ops.RelPos, "on", watched)
    q, g = torch.randn(1, 6, 8), torch.ones(1, 6, 8)
    tp = Tape({"t": torch.zeros(8, 2)}, {"t": torch.zeros(8, 2)})
    o = train_ops.attention_relpos(tp, q, q, q, "t", ops.RelPos(8, 21), 2)
    gc.collect()
    assert maps[-1]() is not None and maps[-1]().data_ptr() == calls[-1][1]
    at = maps[-1]().data_ptr()
    tp._g[id(o)], tp._keep[id(o)] = [g, False], o
    monkeypatch.setattr(tp, "acc", lambda *a, **kw: None)
    tp.backward()
    assert calls[-1] == ("smx_attention_relpos_bwd_f32", at)
