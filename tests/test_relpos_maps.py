"""How long the bucket maps live that `ops.attention_relpos` hands to its kernels, and who shares them.  On the CPU: the launches are replaced by a stub."""
import contextlib
import gc
import types
import weakref

import pytest
import torch

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


def test_threads_at_the_first_use_share_one_map(calls, monkeypatch):
    """two threads that both find no map yet: what either is handed is what stays"""
    import threading
    meet, made, tensor = threading.Barrier(2, timeout=20), [], torch.tensor

    def both_in(*a, **kw):
        t = tensor(*a, **kw)
        made.append(t.data_ptr())
        meet.wait()
        return t
    rp, got = ops.RelPos(8, 22), []
    monkeypatch.setattr(torch, "tensor", both_in)
    ts = [threading.Thread(target=lambda: got.append(rp.on(torch.device("cpu")))) for _ in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert len(made) == 2 and len(got) == 2
    assert got[0] is got[1] and rp.on(torch.device("cpu")) is got[0]


def test_a_map_outlives_its_relpos(calls):
    """a launch on another stream than the one its memory belongs to, or a captured graph, may read a map after its RelPos is gone: maps are never freed,
    and equal ones are one"""
    q = torch.randn(1, 6, 8)
    rp = ops.RelPos(8, 23)
    ops.attention_relpos(q, q, q, torch.zeros(8, 2), rp, 2)
    at, m = calls[-1][1], weakref.ref(rp.on(q.device))
    assert m().data_ptr() == at
    del rp
    gc.collect()
    assert m() is not None and m().data_ptr() == at
    ops.attention_relpos(q, q, q, torch.zeros(8, 2), ops.RelPos(8, 23), 2)
    assert calls[-1][1] == at


def test_one_relpos_for_every_spelling():
    one = ops.relpos(32, 128, True)
    assert ops.relpos() is one and ops.relpos(32) is one and ops.relpos(32, 128) is one and ops.relpos(max_distance=128) is one
    assert ops.relpos(32, 128, two_sided=True) is one and ops.relpos(num_buckets=32, max_distance=128, two_sided=1) is one
    causal = ops.relpos(32, 128, False)
    assert causal is not one and ops.relpos(two_sided=False) is causal and ops.relpos(32, two_sided=0, max_distance=128) is causal
