"""The C entry points of `attention_relpos` and `norm_residual` write what they are given and nothing beside it: every output and workspace lies between
guards of a pattern that is compared bit for bit, and every output element is written."""
import ctypes as C

import pytest
import torch

from synergize_motion_appearance_amd import lib as L
from tests import layer_ref as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
PAD = 4096                                              # bytes of guard on either side, a multiple of every alignment asked for


class Guarded:
    """buffers between guards; `check` compares the guards and that no element of an output is as it was"""
    def __init__(self):
        self.all = []

    def new(self, shape, dtype=F32, off=0, out=True):
        """off: elements by which the buffer starts behind a 16-byte border"""
        n = dtype.itemsize * max(1, torch.Size(shape).numel())
        raw = torch.full((PAD + off * dtype.itemsize + n + PAD,), 0xA5, dtype=torch.uint8, device="cuda")
        at = PAD + off * dtype.itemsize
        self.all.append((raw, at, n, dtype.itemsize if out else 0))
        return raw[at:at + n].view(dtype)[:torch.Size(shape).numel()].view(shape)

    def check(self):
        torch.cuda.synchronize()
        for raw, at, n, size in self.all:
            assert bool((raw[:at] == 0xA5).all()) and bool((raw[at + n:] == 0xA5).all())
            if size:                                    # (the pattern as bf16 and fp32: -2.9e-16, far below any result's size here)
                assert not bool((raw[at:at + n].view(-1, size) == 0xA5).all(1).any()), "left unwritten"


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,E,off", [(1, 8, 0), (7, 96, 0), (11, 33, 0), (5, 250, 1), (13, 256, 3), (3, 1026, 0), (6, 2470, 1), (2, 4098, 0), (3, 8191, 1), (2, 16384, 0),
                                     (3, 16383, 0)])
def test_norm_residual_forward(dtype, T, E, off):
    lib, g, b = L.load(), torch.Generator().manual_seed(1), Guarded()
    x, h = (torch.randn(T, E, generator=g).to(dtype).cuda() for _ in range(2))
    w = [(1 + 0.1 * torch.randn(E, generator=g)).cuda() for _ in range(4)]
    xo, y = b.new((T, E), dtype, off), b.new((T, E), dtype, off)
    d = L.NormResidualDesc(T=T, groups=1, E=E, bf16=dtype is BF, res_scale=1.0, eps=1e-5, x=x.data_ptr(), h=h.data_ptr(), xo=xo.data_ptr(), y=y.data_ptr(),
                           post_gamma=w[0].data_ptr(), post_beta=w[1].data_ptr(), pre_gamma=w[2].data_ptr(), pre_beta=w[3].data_ptr())
    assert lib.smx_norm_residual(C.byref(d), stream()) == 0
    b.check()
    ref = R.norm_residual(x, h, post=(w[0], w[1]), pre=(w[2], w[3]))
    for a, r in ((xo, ref["x"]), (y, ref["y"])):         # (2-norm, as tests/test_gpu_norm_residual.py derives it)
        assert float((a.double().cpu() - r).norm() / r.norm()) < (24 + E / 256) * R.U32 + (3 * R.U[BF] if dtype is BF else 0)


@pytest.mark.parametrize("T,E,groups,off", [(1, 8, 1, 0), (7, 96, 7, 0), (11, 33, 1, 0), (6, 250, 2, 1), (14, 256, 2, 3), (3, 1026, 3, 0), (6, 2470, 1, 1), (2, 4098, 2, 0),
                                            (300, 8191, 1, 1), (2, 16384, 1, 0), (3, 16383, 3, 0), (777, 64, 1, 0)])
def test_norm_residual_backward(T, E, groups, off):
    lib, g, b = L.load(), torch.Generator().manual_seed(2), Guarded()
    x, h, gx, gy = (torch.randn(T, E, generator=g).cuda() for _ in range(4))
    w = [(1 + 0.1 * torch.randn(E, generator=g)).cuda() for _ in range(4)]
    gate = torch.randn(groups, E, generator=g).cuda()
    ref = R.norm_residual(x, h, post=(w[0], w[1]), pre=(w[2], w[3]), gate=gate, gx=gx, gy=gy)
    xo = ref["x"].float().cuda()
    dx, dh, dgate = b.new((T, E), off=off), b.new((T, E), off=off), b.new((groups, E))
    dp = [b.new((E,)).zero_() for _ in range(4)]
    n = lib.smx_norm_residual_bwd_ws_floats(T, groups, E)
    ws = b.new((n,), out=False)
    d = L.NormResidualDesc(T=T, groups=groups, E=E, res_scale=1.0, eps=1e-5, h=h.data_ptr(), xo=xo.data_ptr(), gate=gate.data_ptr(), gx=gx.data_ptr(), gy=gy.data_ptr(),
                           post_gamma=w[0].data_ptr(), post_beta=w[1].data_ptr(), pre_gamma=w[2].data_ptr(), pre_beta=w[3].data_ptr(), dx=dx.data_ptr(), dh=dh.data_ptr(),
                           dgate=dgate.data_ptr(), dpost_gamma=dp[0].data_ptr(), dpost_beta=dp[1].data_ptr(), dpre_gamma=dp[2].data_ptr(), dpre_beta=dp[3].data_ptr(),
                           ws=ws.data_ptr(), ws_floats=n)
    assert lib.smx_norm_residual_bwd_f32(C.byref(d), stream()) == 0
    b.check()
    t = 4 * (24 + E / 256 + T / 4) * R.U32 + 2 * R.U32   # (x' is the reference's, rounded)
    for a, r in ((dx, "dx"), (dh, "dh"), (dgate, "dgate"), (dp[0], "dpost0"), (dp[1], "dpost1"), (dp[2], "dpre0"), (dp[3], "dpre1")):
        assert float((a.double().cpu() - ref[r]).norm() / ref[r].norm()) < t, r


ATTENTION = [  # B, H, Hkv, L, S, dh, causal
    (1, 1, 1, 1, 1, 4, False), (2, 4, 2, 1, 301, 64, True), (3, 2, 1, 3, 600, 36, False), (2, 2, 2, 33, 65, 32, False), (1, 4, 1, 129, 700, 80, True), (2, 2, 1, 70, 70, 128, True),
    (1, 1, 1, 700, 700, 100, False)]


class Ops:
    """the arguments of a call"""
    def __init__(self, c, dtype):
        from synergize_motion_appearance_amd import ops
        B, H, Hkv, Lq, S, dh, causal = c
        g = torch.Generator().manual_seed(3)
        self.q, self.k, self.v = (torch.randn(B, n, h * dh, generator=g).to(dtype).cuda() for n, h in ((Lq, H), (S, Hkv), (S, Hkv)))
        self.rp = ops.relpos(32, 128, two_sided=not causal)
        self.table, self.map = torch.randn(32, H, generator=g).cuda(), self.rp.on(self.q.device)
        self.d = L.RelposDesc(B=B, H=H, Hkv=Hkv, L=Lq, S=S, dh=dh, map_lo=self.rp.lo, map_n=len(self.rp.map), num_buckets=32, causal=causal, bf16=dtype is BF,
                              scale=dh ** -0.5, ldq=H * dh, ldk=Hkv * dh, ldv=Hkv * dh, ldo=H * dh, q_bs=Lq * H * dh, k_bs=S * Hkv * dh, v_bs=S * Hkv * dh, o_bs=Lq * H * dh,
                              q=self.q.data_ptr(), k=self.k.data_ptr(), v=self.v.data_ptr(), table=self.table.data_ptr(), map=self.map.data_ptr())

    def forward(self, lib, b, c, dtype):
        B, H, Hkv, Lq, S, dh, causal = c
        o, lse = b.new((B, Lq, H * dh), dtype), b.new((B, H, Lq))
        self.d.o, self.d.lse = o.data_ptr(), lse.data_ptr()
        n = lib.smx_attention_relpos_ws_bytes(C.byref(self.d))
        ws = b.new((n,), torch.uint8, out=False)
        self.d.ws, self.d.ws_bytes = ws.data_ptr(), n
        assert lib.smx_attention_relpos(C.byref(self.d), stream()) == 0
        return o, lse


def near(got, ref, what):
    off = (got.double().cpu() - ref[0]).abs() - ref[1]
    assert float(off.max()) <= 0, what


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", ATTENTION, ids=str)
def test_attention_forward(dtype, c):
    lib, b = L.load(), Guarded()
    a = Ops(c, dtype)
    o, _ = a.forward(lib, b, c, dtype)
    b.check()
    near(o, R.attention(a.q, a.k, a.v, a.table, a.rp, c[1], nkv=c[2], causal=c[6], storage=dtype)["o"], "o")


@pytest.mark.parametrize("c", ATTENTION, ids=str)
def test_attention_backward(c):
    lib, b = L.load(), Guarded()
    B, H, Hkv, Lq, S, dh, causal = c
    a = Ops(c, F32)
    o, lse = a.forward(lib, b, c, F32)
    go = torch.randn(B, Lq, H * dh, generator=torch.Generator().manual_seed(4)).cuda()
    dq, dk, dv, dt = b.new((B, Lq, H * dh)), b.new((B, S, Hkv * dh)), b.new((B, S, Hkv * dh)), b.new((32, H)).zero_()
    d = a.d
    d.d_o, d.dq, d.dk, d.dv, d.dtable = (t.data_ptr() for t in (go, dq, dk, dv, dt))
    n = lib.smx_attention_relpos_bwd_ws_bytes(C.byref(d))
    ws = b.new((n,), torch.uint8, out=False)
    d.ws, d.ws_bytes = ws.data_ptr(), n
    assert lib.smx_attention_relpos_bwd_f32(C.byref(d), stream()) == 0
    b.check()
    ref = R.attention(a.q, a.k, a.v, a.table, a.rp, H, nkv=Hkv, causal=causal, g=go)
    for t, r in ((o, "o"), (dq, "dq"), (dk, "dk"), (dv, "dv"), (dt, "dtable")):
        near(t, ref[r], r)
