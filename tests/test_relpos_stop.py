"""Which passes the attention's backward asks for where some tensors take no gradient.  On the CPU: the launches are replaced by a stub."""
import contextlib
import ctypes as C
import types

import pytest
import torch

from synergize_motion_appearance_amd import ops, train_ops
from synergize_motion_appearance_amd.tape import Tape
from tests.test_relpos_host import lib, relpos_desc


# what takes no gradient -> which of dq, dk, dv, dtable the library is asked for
@pytest.mark.parametrize("stopped,asked", [("", (1, 1, 1, 1)), ("q", (1, 1, 1, 1)), ("k", (1, 1, 1, 1)), ("kv", (1, 0, 0, 1)), ("t", (1, 1, 1, 1)), ("qt", (0, 1, 1, 0)),
                                           ("kvt", (1, 0, 0, 1)), ("qkv", (1, 0, 0, 1)), ("qkvt", None)])
def test_no_pass_for_what_takes_no_gradient(monkeypatch, stopped, asked):
    seen = []

    def call(fn, d, index):
        seen.append((fn.__name__, tuple(int(bool(p)) for p in (d.dq, d.dk, d.dv, d.dtable))))
        return 0
    monkeypatch.setattr(ops, "_call", call)
    monkeypatch.setattr(ops, "_dev", lambda *a, **kw: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(synchronize=lambda: None))
    monkeypatch.setattr(torch.cuda, "device", lambda *a: contextlib.nullcontext())
    q, k, v = (torch.randn(1, 6, 8) for _ in range(3))
    tp = Tape({"t": torch.zeros(8, 2)}, {} if "t" in stopped else {"t": torch.zeros(8, 2)})
    for n, t in (("q", q), ("k", k), ("v", v)):
        if n in stopped:
            tp.stop(t)
    o = train_ops.attention_relpos(tp, q, k, v, "t", ops.RelPos(8, 21), 2)
    tp._g[id(o)], tp._keep[id(o)] = [torch.ones(1, 6, 8), False], o
    tp.backward()
    assert seen[1:] == ([] if asked is None else [("smx_attention_relpos_bwd_f32", asked)])
    for n, t in (("q", q), ("k", k), ("v", v)):
        assert (tp.grad(t) is None) == (n in stopped)


@pytest.mark.parametrize("bad", [dict(dq=None, dtable=None, dk=None, dv=None), dict(dq=None, dk=None, dv=None), dict(dq=None), dict(dtable=None), dict(dk=None, dtable=None),
                                 dict(dv=None, dtable=None), dict(dq=None, dtable=None, dk=None)], ids=str)
def test_refused_without(bad):
    so = lib()
    for ok in (dict(dq=None, dtable=None), dict(dk=None, dv=None)):
        assert so.smx_attention_relpos_bwd_ws_bytes(C.byref(relpos_desc(**ok))) > 0
    assert so.smx_attention_relpos_bwd_f32(C.byref(relpos_desc(**bad)), None) == -22
