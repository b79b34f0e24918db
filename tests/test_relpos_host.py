"""CPU side of `ops.attention_relpos` / `ops.norm_residual`: the bucket map, the 64-bit form's own gradients against differences, and the refusals of
the library's entry points (host checks, nothing is launched)."""
import ctypes as C
import math

import pytest
import torch

from synergize_motion_appearance_amd import lib as L
from synergize_motion_appearance_amd import ops
from tests import layer_ref as R


@pytest.mark.parametrize("nb,md,two", [(32, 128, True), (32, 128, False), (8, 64, True), (24, 301, True), (64, 800, False), (3, 64, False), (4, 2, True),
                                       (16, 1024, False), (2, 1024, False)])
def test_bucket_map(nb, md, two):
    rp = ops.RelPos(nb, md, two)
    assert ops.relpos(nb, md, two) is ops.relpos(nb, md, two)
    for delta in list(range(-1200, 1201)) + [-2 ** 30, 2 ** 30]:
        assert rp.bucket(delta) == R.bucket(nb, md, two, delta), delta
    assert len(rp.map) <= 2049 and rp.lo <= 0 <= rp.lo + len(rp.map) - 1
    assert set(rp.map) <= set(range(nb))


def test_bucket_borders_are_exact():
    """half 8, max 128, 16 one-sided buckets: the borders 8 * 16^(t/8) include the whole numbers 16, 32, 64, which open their bucket"""
    rp = ops.RelPos(16, 128, False)
    for n, b in ((8, 8), (15, 9), (16, 10), (31, 11), (32, 12), (63, 13), (64, 14), (90, 14), (91, 15), (127, 15), (5000, 15)):
        assert rp.bucket(-n) == b, n


@pytest.mark.parametrize("a", [(7, 64, True), (2, 64, True), (32, 8, True), (32, 1025, True), (1, 64, False), (8192, 1024, False), (32, 16, False)])
def test_bucket_refusals(a):
    with pytest.raises(L.SmxError):
        ops.RelPos(*a)


def test_cpu_tensors_are_refused():
    z = torch.zeros(1, 4, 32)
    with pytest.raises(L.SmxError, match="no CPU fallback"):
        ops.attention_relpos(z, z, z, torch.zeros(32, 8), ops.relpos(), 8)
    with pytest.raises(L.SmxError, match="no CPU fallback"):
        ops.norm_residual(z, z)


@pytest.mark.parametrize("causal,two", [(False, True), (True, False)])
def test_reference_gradients_against_differences(causal, two):
    """the 64-bit form of the attention's backward, against central differences of its forward (step 1e-5: error 1e-10 from the cubic term, 1e-11 from rounding)"""
    g = torch.Generator().manual_seed(3)
    B, H, Hkv, Lq, S, dh = 2, 4, 2, 5, 9, 4
    rp = ops.RelPos(8, 16, two)
    t = {"q": torch.randn(B, Lq, H * dh, generator=g).double(), "k": torch.randn(B, S, Hkv * dh, generator=g).double(),
         "v": torch.randn(B, S, Hkv * dh, generator=g).double(), "table": torch.randn(8, H, generator=g).double()}
    go = torch.randn(B, Lq, H * dh, generator=g).double()
    mask = torch.rand(B, S, generator=g) < 0.3
    mask[1] = True
    kw = dict(nkv=Hkv, causal=causal, mask=mask)
    ref = R.attention(**t, rp=rp, nhead=H, g=go, **kw)
    for name in t:
        d = torch.randn(t[name].shape, generator=g).double()
        e = 1e-5
        up, dn = (R.attention(**{**t, name: t[name] + s * e * d}, rp=rp, nhead=H, **kw)["o"][0] for s in (1, -1))
        diff = float(((up - dn) * go).sum()) / (2 * e)
        assert abs(diff - float((ref["d" + name][0] * d).sum())) < 1e-7 * max(1.0, abs(diff)), name


def lib():
    so = C.CDLL(L.LIB_PATH)
    for name in L.SIGNATURES:
        if "relpos" in name or "norm_residual" in name:
            getattr(so, name).restype, getattr(so, name).argtypes = L.SIGNATURES[name]
    return so


FAKE = 0x7f0000000000                                    # 16-byte aligned, never dereferenced: the calls below end in the host's checks


def relpos_desc(**kw):
    d = L.RelposDesc(B=2, H=4, Hkv=2, L=5, S=7, dh=32, map_lo=-3, map_n=7, num_buckets=8, scale=0.1, ldq=128, ldk=64, ldv=64, ldo=128, q_bs=640, k_bs=448, v_bs=448,
                     o_bs=640)
    for n in ("q", "k", "v", "o", "table", "map", "lse", "ws", "d_o", "dq", "dk", "dv", "dtable"):
        setattr(d, n, FAKE)
    d.ws_bytes = 1 << 40
    for n, v in kw.items():
        setattr(d, n, v)
    return d


BAD = [dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(table=None), dict(map=None), dict(B=0), dict(H=0), dict(Hkv=0), dict(Hkv=3), dict(L=0), dict(S=0),
       dict(dh=0), dict(dh=30), dict(dh=132, H=1, Hkv=1, ldq=132, ldo=132, ldk=132, ldv=132), dict(map_n=0), dict(map_n=2050), dict(map_lo=1), dict(map_lo=-8),
       dict(num_buckets=0), dict(num_buckets=4097), dict(ldq=124), dict(ldk=60), dict(ldv=66), dict(ldo=130), dict(ldk=(1 << 24) + 4), dict(q_bs=642), dict(k_bs=-4), dict(v_bs=2), dict(o_bs=1),
       dict(q=FAKE + 4), dict(k=FAKE + 8), dict(v=FAKE + 2), dict(o=FAKE + 12), dict(bf16=2), dict(bf16=1, k=FAKE + 4), dict(scale=math.nan),
       dict(has_q_start=1, q_start=2 ** 30 + 1), dict(has_q_start=1, q_start=-2 ** 30 - 1), dict(L=2 ** 29 + 1), dict(S=2 ** 29 + 1)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_relpos_entry_point_refuses(bad):
    so = lib()
    assert so.smx_attention_relpos_ws_bytes(C.byref(relpos_desc())) >= 0
    assert so.smx_attention_relpos(C.byref(relpos_desc(**bad)), None) == -22
    assert so.smx_attention_relpos_ws_bytes(C.byref(relpos_desc(**bad))) == -1
    assert so.smx_attention_relpos_bwd_f32(C.byref(relpos_desc(**bad)), None) == -22
    assert so.smx_attention_relpos_bwd_ws_bytes(C.byref(relpos_desc(**bad))) == -1
    assert so.smx_attention_relpos(None, None) == -22


@pytest.mark.parametrize("bad", [dict(d_o=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(dtable=None), dict(lse=None), dict(ws=None), dict(ws_bytes=16),
                                 dict(ws=FAKE + 8), dict(bf16=1), dict(d_o=FAKE + 4), dict(dq=FAKE + 8), dict(dk=FAKE + 4), dict(dv=FAKE + 4), dict(ldo=132),
                                 dict(o_bs=644)], ids=str)
def test_relpos_backward_refuses(bad):
    so = lib()
    assert so.smx_attention_relpos_bwd_ws_bytes(C.byref(relpos_desc())) > 0
    assert so.smx_attention_relpos_bwd_f32(C.byref(relpos_desc(**bad)), None) == -22


def norm_desc(**kw):
    d = L.NormResidualDesc(T=12, groups=3, E=64, res_scale=1.0, eps=1e-5)
    for n in ("x", "h", "xo", "y", "post_gamma", "post_beta", "pre_gamma", "pre_beta", "gate", "gx", "gy", "dx", "dh", "dgate", "dpost_gamma", "dpost_beta",
              "dpre_gamma", "dpre_beta", "ws"):
        setattr(d, n, FAKE)
    d.ws_floats = 1 << 40
    for n, v in kw.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("bad,fwd,bwd", [(dict(x=None), 1, 0), (dict(h=None), 1, 1), (dict(xo=None), 1, 1), (dict(y=None), 1, 0), (dict(T=0), 1, 1), (dict(T=13), 1, 1),
                                         (dict(groups=0), 1, 1), (dict(groups=5), 1, 1), (dict(E=0), 1, 1), (dict(E=16385), 1, 1), (dict(gate=None), 1, 1),
                                         (dict(post_gamma=None), 1, 1), (dict(pre_gamma=None), 1, 1), (dict(eps=-1.0), 1, 1), (dict(eps=math.nan), 1, 1),
                                         (dict(res_scale=math.nan), 1, 1), (dict(bf16=3), 1, 1), (dict(bf16=1), 0, 1), (dict(gx=None, gy=None), 0, 1),
                                         (dict(ws=None), 0, 1), (dict(ws=FAKE + 4), 0, 1), (dict(ws_floats=4), 0, 1), (dict(T=2 ** 31), 1, 1)], ids=str)
def test_norm_residual_entry_points_refuse(bad, fwd, bwd):
    so = lib()
    if fwd:
        assert so.smx_norm_residual(C.byref(norm_desc(**bad)), None) == -22
    if bwd:
        assert so.smx_norm_residual_bwd_f32(C.byref(norm_desc(**bad)), None) == -22
    assert so.smx_norm_residual(None, None) == -22 and so.smx_norm_residual_bwd_f32(None, None) == -22
    assert so.smx_norm_residual_bwd_ws_floats(12, 3, 64) > 0 and so.smx_norm_residual_bwd_ws_floats(12, 5, 64) == -1
