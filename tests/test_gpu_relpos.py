"""`ops.attention_relpos` and `train_ops.attention_relpos` on a real MI355X against the formula in fp64 (tests/layer_ref.py), every value within the bound that
rounding allows it: odd lengths and head sizes, shared heads, strides of a fused projection, masks, ragged samples, empty rows, single tokens,
what left-out places hold, other positions, other streams, replayed graphs."""
import math

import pytest
import torch

from synergize_motion_appearance_amd import lib as L
from tests import layer_ref as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs an MI355X"
    from synergize_motion_appearance_amd import ops as _ops
    return _ops


@pytest.fixture(scope="module")
def T():
    from synergize_motion_appearance_amd import train_ops
    return train_ops


def mk(seed, B, H, Hkv, Lq, S, dh, dtype=F32, std=1.0, fused=False):
    g = torch.Generator().manual_seed(seed)
    if fused:
        w = torch.randn(B, S, (H + 2 * Hkv) * dh, generator=g).mul(std).to(dtype).cuda()
        q, k, v = w[..., :H * dh], w[..., H * dh:(H + Hkv) * dh], w[..., (H + Hkv) * dh:]
    else:
        q, k, v = (torch.randn(B, n, h * dh, generator=g).mul(std).to(dtype).cuda() for n, h in ((Lq, H), (S, Hkv), (S, Hkv)))
    return q, k, v, g


def near(got, ref, what=""):
    val, bound = ref
    got = got.detach().double().cpu()
    assert got.shape == val.shape and torch.isfinite(got).all(), what
    off = (got - val).abs() - bound
    assert float(off.max()) <= 0 if off.numel() else True, f"{what}: over its bound by {float(off.max()):.3e} (value {float(val.flatten()[off.argmax()]):.3e}, " \
                                                          f"bound {float(bound.flatten()[off.argmax()]):.3e})"


def lengths(B, S):
    return torch.tensor([max(0, S - (b * S) // 2) if b != 2 else 0 for b in range(B)], dtype=torch.int32)


# B, H, Hkv, L, S, dh, causal, mask, ragged, fused
FORWARD = [
    (1, 1, 1, 1, 1, 4, False, False, False, False),
    (2, 2, 1, 1, 1, 32, True, False, False, False),
    (1, 8, 8, 1, 300, 32, True, False, False, False),            # one token
    (4, 8, 2, 1, 1025, 64, True, True, True, False),
    (2, 4, 1, 1, 777, 128, False, True, False, False),
    (3, 4, 2, 1, 63, 80, False, True, True, False),
    (3, 16, 2, 2, 517, 16, True, False, True, False),            # a few tokens
    (1, 8, 1, 5, 130, 4, True, False, False, False),
    (2, 2, 2, 31, 33, 32, False, False, False, False),
    (2, 4, 4, 64, 64, 64, True, True, False, True),
    (3, 6, 2, 129, 129, 80, False, True, True, True),
    (1, 2, 2, 200, 321, 128, True, False, False, False),
    (2, 2, 1, 65, 1000, 36, False, True, False, False),
    (1, 4, 2, 513, 513, 32, True, True, False, True),
    (3, 2, 2, 257, 700, 64, True, False, True, False),
    (1, 3, 1, 1100, 1100, 4, False, False, False, False),
    (2, 8, 4, 385, 385, 32, True, False, False, False),          # 16 heads: their order over the XCDs
    (1, 8, 8, 12, 2000, 100, True, True, False, False),          # the most query rows a kv head that fp32 token calls of more than two queries take
    (1, 1, 1, 13, 2000, 100, True, True, False, False),          # the fewest a tile call takes
    (1, 16, 1, 2, 700, 64, False, True, False, False),           # more query rows on a kv head than one block takes
    (2, 6, 2, 1, 700, 64, True, False, True, False),             # rows that leave some of a block's unused
    (1, 16, 1, 3, 700, 64, False, False, False, False),
]


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", FORWARD, ids=str)
def test_forward(ops, c, dtype):
    B, H, Hkv, Lq, S, dh, causal, masked, ragged, fused = c
    q, k, v, g = mk(5, B, H, Hkv, Lq, S, dh, dtype, fused=fused)
    rp = ops.relpos(24, 301, two_sided=True) if not causal else ops.relpos(32, 128, two_sided=False)
    table = torch.randn(rp.num_buckets, H, generator=g).cuda()
    mask = (torch.rand(B, S, generator=g) < 0.3).cuda() if masked else None
    kv_len = lengths(B, S).cuda() if ragged else None
    kw = dict(nkv=Hkv, causal=causal, mask=mask, kv_len=kv_len)
    o = ops.attention_relpos(q, k, v, table, rp, H, **kw)
    assert o.dtype == dtype and o.is_contiguous()
    near(o, R.attention(q, k, v, table, rp, H, storage=dtype, **kw)["o"])


BACKWARD = [
    (1, 1, 1, 1, 1, 4, False, False, False),
    (2, 2, 1, 1, 70, 32, True, False, False),
    (1, 2, 2, 33, 33, 32, False, True, False),
    (2, 4, 2, 64, 64, 64, True, True, False),
    (3, 4, 1, 100, 131, 80, False, True, True),
    (1, 2, 2, 129, 300, 128, True, False, False),
    (2, 2, 2, 257, 257, 32, False, True, False),
    (3, 3, 3, 190, 190, 4, True, False, True),
    (1, 4, 4, 640, 640, 64, True, False, False),
    (1, 2, 1, 70, 1500, 32, False, False, False),
    (1, 1, 1, 1500, 1500, 64, True, False, False),               # both sides in parts
    (2, 8, 4, 200, 200, 36, True, False, False),
    (4, 2, 1, 700, 1030, 100, False, True, True),
]


@pytest.mark.parametrize("c", BACKWARD, ids=str)
def test_backward(ops, T, c):
    from synergize_motion_appearance_amd.tape import Tape
    B, H, Hkv, Lq, S, dh, causal, masked, ragged = c
    q, k, v, g = mk(6, B, H, Hkv, Lq, S, dh)
    rp = ops.relpos(24, 301, two_sided=True) if not causal else ops.relpos(32, 128, two_sided=False)
    table = torch.randn(rp.num_buckets, H, generator=g).cuda()
    mask = (torch.rand(B, S, generator=g) < 0.3).to(torch.uint8).cuda() if masked else None
    kv_len = lengths(B, S).cuda() if ragged else None
    go = (torch.randn(B, Lq, H * dh, generator=g) * 1e-3).cuda()
    kw = dict(nkv=Hkv, causal=causal, mask=mask, kv_len=kv_len)
    old = torch.randn(rp.num_buckets, H, generator=g)
    G = {"table": old.cuda()}
    tp = Tape({"table": table}, G)
    o = T.attention_relpos(tp, q, k, v, "table", rp, H, **kw)
    tp.acc(o, go, owned=False)
    tp.backward()
    ref = R.attention(q, k, v, table, rp, H, g=go, **kw)
    near(o, ref["o"], "o")
    for n, t in (("dq", q), ("dk", k), ("dv", v)):
        near(tp.grad(t), ref[n], n)
    val, bound = ref["dtable"]                                   # accumulated into what was there: one more rounding
    near(G["table"], (val + old.double(), bound + 2 * R.U32 * (val.abs() + old.double().abs())), "dtable")
    for t in (q, k, v):                                          # the same call again answers the same bits
        t_old = tp.grad(t).clone()
        tp2 = Tape({"table": table}, {"table": torch.zeros_like(table)})
        o2 = T.attention_relpos(tp2, q, k, v, "table", rp, H, **kw)
        tp2.acc(o2, go, owned=False)
        tp2.backward()
        assert torch.equal(tp2.grad(t), t_old) and torch.equal(o, o2)


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_against_differences(ops, T, causal):
    """directional differences of the kernel's own forward; with steps of 2^-5 the cubic term of a softmax of unit scores is below 1e-3 of the slope's scale"""
    from synergize_motion_appearance_amd.tape import Tape
    B, H, Hkv, Lq, dh = 2, 4, 2, 70, 32
    q, k, v, g = mk(8, B, H, Hkv, Lq, Lq, dh)
    rp = ops.relpos(32, 128, two_sided=not causal)
    P = {"table": torch.randn(32, H, generator=g).cuda()}
    go = torch.randn(B, Lq, H * dh, generator=g).cuda()
    tp = Tape(P, {"table": torch.zeros_like(P["table"])})
    o = T.attention_relpos(tp, q, k, v, "table", rp, H, nkv=Hkv, causal=causal)
    tp.acc(o, go, owned=False)
    tp.backward()
    grads = {"q": tp.grad(q), "k": tp.grad(k), "v": tp.grad(v), "table": tp.G["table"]}
    have = {"q": q, "k": k, "v": v, "table": P["table"]}
    for n in have:
        d = torch.randn(have[n].shape, generator=g).cuda()
        e = 2.0 ** -5
        up, dn = (ops.attention_relpos(*({**have, n: have[n] + s * e * d}[m] for m in ("q", "k", "v", "table")), rp, H, nkv=Hkv, causal=causal).double()
                  for s in (1, -1))
        slope, want = float(((up - dn) * go).sum()) / (2 * e), float((grads[n].double() * d).sum())
        size = float(((up - dn).abs() * go.abs()).sum()) / (2 * e)
        assert abs(slope - want) < 2e-3 * size, (n, slope, want, size)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("Lq", [1, 4, 96])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_left_out_places_do_not_count(ops, dtype, Lq, bad):
    """NaN, infinities and huge values in masked keys and behind kv_len change nothing, bit for bit"""
    B, H, Hkv, S, dh = 3, 4, 2, 200, 64
    q, k, v, g = mk(9, B, H, Hkv, Lq, S, dh, dtype)
    rp = ops.relpos()
    table = torch.randn(32, H, generator=g).cuda()
    mask = (torch.rand(B, S, generator=g) < 0.3).cuda()
    kv_len = torch.tensor([200, 131, 64], dtype=torch.int32).cuda()
    gone = mask | (torch.arange(S).cuda()[None] >= kv_len[:, None])
    k, v = k.masked_fill(gone[..., None], 0), v.masked_fill(gone[..., None], 0)
    a = ops.attention_relpos(q, k, v, table, rp, H, nkv=Hkv, mask=mask, kv_len=kv_len)
    b = ops.attention_relpos(q, k.masked_fill(gone[..., None], bad), v.masked_fill(gone[..., None], bad), table, rp, H, nkv=Hkv, mask=mask, kv_len=kv_len)
    assert torch.isfinite(a).all() and torch.equal(a, b)


def test_left_out_places_do_not_count_in_the_backward(ops, T):
    from synergize_motion_appearance_amd.tape import Tape
    B, H, S, dh = 2, 2, 150, 32
    q, k, v, g = mk(10, B, H, H, S, S, dh)
    rp = ops.relpos()
    table = torch.randn(32, H, generator=g).cuda()
    mask = (torch.rand(B, S, generator=g) < 0.3).cuda()
    kv_len = torch.tensor([150, 77], dtype=torch.int32).cuda()
    gone = (mask | (torch.arange(S).cuda()[None] >= kv_len[:, None]))[..., None]
    go = torch.randn(B, S, H * dh, generator=g).cuda()

    def grads(kk, vv):
        tp = Tape({"t": table}, {"t": torch.zeros_like(table)})
        o = T.attention_relpos(tp, q, kk, vv, "t", rp, H, mask=mask, kv_len=kv_len, q_start=0)
        tp.acc(o, go, owned=False)
        tp.backward()
        return tp.grad(q), tp.grad(kk), tp.grad(vv), tp.G["t"]
    a = grads(k.masked_fill(gone, 0), v.masked_fill(gone, 0))
    for bad in (float("nan"), float("inf"), -3e38):
        for x, y in zip(a, grads(k.masked_fill(gone, bad), v.masked_fill(gone, bad))):
            assert torch.isfinite(x).all() and torch.equal(x, y)
    assert float(a[1].masked_select(gone.expand_as(a[1])).abs().max()) == 0.0 and float(a[2].masked_select(gone.expand_as(a[2])).abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("Lq", [1, 40])
def test_rows_without_a_key(ops, T, dtype, Lq):
    """a sample whose mask leaves nothing, a length of zero, and causal queries that stand before every key: zeros, and zero gradients"""
    B, H, S, dh = 3, 2, 90, 32
    q, k, v, g = mk(11, B, H, H, Lq, S, dh, dtype)
    rp = ops.relpos()
    table = torch.randn(32, H, generator=g).cuda()
    mask = torch.zeros(B, S, dtype=torch.uint8)
    mask[1] = 1
    kv_len = torch.tensor([S, S, -4], dtype=torch.int32).cuda()
    kw = dict(mask=mask.cuda(), kv_len=kv_len)
    o = ops.attention_relpos(q, k, v, table, rp, H, **kw)
    assert float(o[1:].abs().max()) == 0.0
    near(o, R.attention(q, k, v, table, rp, H, storage=dtype, **kw)["o"])
    o = ops.attention_relpos(q, k, v, table, rp, H, causal=True, q_start=-Lq + 1)         # only the last query sees key 0
    near(o, R.attention(q, k, v, table, rp, H, causal=True, q_start=-Lq + 1, storage=dtype)["o"])
    if Lq > 1:
        assert float(o[:, :-1].abs().max()) == 0.0
    if dtype == F32:
        from synergize_motion_appearance_amd.tape import Tape
        tp = Tape({"t": table}, {"t": torch.zeros_like(table)})
        o = T.attention_relpos(tp, q, k, v, "t", rp, H, **kw)
        tp.acc(o, torch.ones_like(o))
        tp.backward()
        ref = R.attention(q, k, v, table, rp, H, g=torch.ones_like(o), **kw)
        for n, t in (("dq", tp.grad(q)), ("dk", tp.grad(k)), ("dv", tp.grad(v)), ("dtable", tp.G["t"])):
            near(t, ref[n], n)
        assert float(tp.grad(q)[1:].abs().max()) == 0.0 and float(tp.grad(k)[1:].abs().max()) == 0.0


def test_table_gradient_of_many_pairs(ops, T):
    """a bucket of half a million pairs of mixed signs: independent errors of a few 2^-23 a pair (22-bit products, fp32 scores) stay that in the sum, 2^-19
    holds sixteen of them; an error of one sign a pair, as small as 2^-25 of it, would grow to 2^-15 of the sum"""
    from synergize_motion_appearance_amd.tape import Tape
    B, H, S, dh = 2, 2, 1024, 32
    q, k, v, g = mk(21, B, H, H, S, S, dh)
    rp = ops.relpos(32, 128)
    table, go = torch.randn(32, H, generator=g).cuda(), (torch.randn(B, S, H * dh, generator=g) * 1e-3).cuda()
    G = {"t": torch.zeros_like(table)}
    tp = Tape({"t": table}, G)
    o = T.attention_relpos(tp, q, k, v, "t", rp, H)
    tp.acc(o, go, owned=False)
    tp.backward()
    ref = R.attention(q, k, v, table, rp, H, g=go)["dtable"][0]
    assert float((G["t"].double().cpu() - ref).norm() / ref.norm()) < 2.0 ** -19


@pytest.mark.parametrize("a", [(64, 1024, True), (2, 1024, False), (512, 600, True)])
def test_largest_maps(ops, T, a):
    from synergize_motion_appearance_amd.tape import Tape
    B, H, S, dh = 1, 2, 1400, 32
    q, k, v, g = mk(22, B, H, H, S, S, dh)
    rp = ops.relpos(*a)
    table, go = torch.randn(a[0], H, generator=g).cuda(), torch.randn(B, S, H * dh, generator=g).cuda()
    G = {"t": torch.zeros_like(table)}
    tp = Tape({"t": table}, G)
    o = T.attention_relpos(tp, q, k, v, "t", rp, H)
    tp.acc(o, go, owned=False)
    tp.backward()
    ref = R.attention(q, k, v, table, rp, H, g=go)
    for n, t in (("o", o), ("dq", tp.grad(q)), ("dk", tp.grad(k)), ("dv", tp.grad(v)), ("dtable", G["t"])):
        near(t, ref[n], n)
    near(ops.attention_relpos(q[:, -1:], k, v, table, rp, H), (ref["o"][0][:, -1:], ref["o"][1][:, -1:]))


@pytest.mark.parametrize("start", [-70, 0, 13, 500, 2 ** 30, -2 ** 30])
def test_positions(ops, start):
    B, H, Lq, S, dh = 1, 2, 70, 140, 32
    q, k, v, g = mk(12, B, H, H, Lq, S, dh)
    rp = ops.relpos(32, 64)
    table = torch.randn(32, H, generator=g).cuda()
    near(ops.attention_relpos(q, k, v, table, rp, H, q_start=start), R.attention(q, k, v, table, rp, H, q_start=start)["o"])


@pytest.mark.parametrize("std", [1e-12, 1e-4, 30.0, 1e6])
def test_magnitudes(ops, T, std):
    """values and gradients far from one; the scores stay moderate through `scale`"""
    from synergize_motion_appearance_amd.tape import Tape
    B, H, S, dh = 1, 2, 150, 64
    q, k, v, g = mk(13, B, H, H, S, S, dh, std=std)
    v[:, ::7] *= 1e-3                                            # keys of small values among large ones
    k[:, 5::11] *= 1e-3
    rp = ops.relpos()
    table = torch.randn(32, H, generator=g).cuda()
    go = (torch.randn(B, S, H * dh, generator=g) * std).cuda()
    scale = dh ** -0.5 / std / std
    tp = Tape({"t": table}, {"t": torch.zeros_like(table)})
    o = T.attention_relpos(tp, q, k, v, "t", rp, H, scale=scale)
    tp.acc(o, go, owned=False)
    tp.backward()
    ref = R.attention(q, k, v, table, rp, H, scale=scale, g=go)
    for n, t in (("o", o), ("dq", tp.grad(q)), ("dk", tp.grad(k)), ("dv", tp.grad(v)), ("dtable", tp.G["t"])):
        near(t, ref[n], n)


def test_large_scores_pick_one_key(ops):
    """scores of thousands: the softmax is a selection, nothing overflows"""
    B, H, S, dh = 1, 2, 300, 32
    q, k, v, g = mk(14, B, H, H, S, S, dh, std=40.0)
    rp = ops.relpos()
    table = (torch.randn(32, H, generator=g) * 100).cuda()
    near(ops.attention_relpos(q, k, v, table, rp, H), R.attention(q, k, v, table, rp, H)["o"])


def test_broadcast_and_repeated_operands(ops, T):
    """one context for all samples (sample stride 0), and the same tensor as key and value"""
    from synergize_motion_appearance_amd.tape import Tape
    B, H, Lq, S, dh = 3, 2, 40, 77, 32
    q, k, v, g = mk(15, B, H, H, Lq, S, dh)
    rp = ops.relpos()
    table = torch.randn(32, H, generator=g).cuda()
    ke, ve = k[:1].expand(B, -1, -1), v[:1].expand(B, -1, -1)
    near(ops.attention_relpos(q, ke, ve, table, rp, H, q_start=3), R.attention(q, ke, ve, table, rp, H, q_start=3)["o"])
    go = torch.randn(B, Lq, H * dh, generator=g).cuda()
    tp = Tape({"t": table}, {"t": torch.zeros_like(table)})
    o = T.attention_relpos(tp, q, k, k, "t", rp, H)
    tp.acc(o, go, owned=False)
    tp.backward()
    ref = R.attention(q, k, k, table, rp, H, g=go)
    both = ref["dk"][0] + ref["dv"][0], ref["dk"][1] + ref["dv"][1] + 2 * R.U32 * (ref["dk"][0].abs() + ref["dv"][0].abs())
    near(tp.grad(k), both)


def test_gradient_through_views_and_without_gradients(ops, T):
    """a key that needs no gradient, and an output gradient whose rows are strided"""
    from synergize_motion_appearance_amd.tape import Tape
    B, H, S, dh = 2, 2, 65, 32
    q, k, v, g = mk(16, B, H, H, S, S, dh)
    rp = ops.relpos()
    table = torch.randn(32, H, generator=g).cuda()
    wide = torch.randn(B, S, 2 * H * dh, generator=g).cuda()
    go = wide[..., H * dh:]
    tp = Tape({"t": table}, {"t": torch.zeros_like(table)})
    tp.stop(k)
    o = T.attention_relpos(tp, q, k, v, "t", rp, H)
    tp._g[id(o)], tp._keep[id(o)] = [go, False], o
    tp.backward()
    ref = R.attention(q, k, v, table, rp, H, g=go)
    assert tp.grad(k) is None
    near(tp.grad(q), ref["dq"])
    near(tp.grad(v), ref["dv"])


def test_empty_operands(ops):
    rp, z = ops.relpos(), lambda *s: torch.zeros(s, device="cuda")
    t = z(32, 2)
    assert ops.attention_relpos(z(2, 0, 64), z(2, 5, 64), z(2, 5, 64), t, rp, 2).shape == (2, 0, 64)
    o = ops.attention_relpos(torch.ones(2, 3, 64, device="cuda"), z(2, 0, 64), z(2, 0, 64), t, rp, 2)
    assert o.shape == (2, 3, 64) and float(o.abs().max()) == 0.0


def test_refusals(ops):
    rp = ops.relpos()
    q = torch.zeros(2, 8, 64, device="cuda")
    t = torch.zeros(32, 2, device="cuda")
    ok = dict(q=q, k=q, v=q, table=t, rp=rp, nhead=2)
    for bad in (dict(q=q.half()), dict(k=q.bfloat16()), dict(v=q[:, :7]), dict(k=q[:1]), dict(nhead=3), dict(nhead=64), dict(table=t[:31]), dict(table=t.double()),
                dict(table=t.cpu()), dict(rp=None), dict(nkv=3), dict(mask=torch.zeros(2, 7, device="cuda", dtype=torch.uint8)),
                dict(mask=torch.zeros(2, 8, device="cuda")), dict(kv_len=torch.zeros(2, device="cuda", dtype=torch.int64)), dict(q_start=2 ** 31),
                dict(q=torch.zeros(2, 64, 8, device="cuda").transpose(1, 2)), dict(q=torch.zeros(2, 8, 65, device="cuda")[..., 1:]),
                dict(q=torch.zeros(2 * 8 * 64 + 2, device="cuda")[2:].view(2, 8, 64)), dict(q=q[0])):
        with pytest.raises(L.SmxError):
            ops.attention_relpos(**{**ok, **bad})


def test_other_stream_and_graph(ops, T):
    """a captured forward and backward replayed several times with eager work between, new inputs copied in, against the eager result"""
    from synergize_motion_appearance_amd.tape import Tape
    B, H, S, dh = 2, 2, 130, 64
    q, k, v, g = mk(17, B, H, H, S, S, dh)
    rp = ops.relpos()
    table, go = torch.randn(32, H, generator=g).cuda(), torch.randn(B, S, H * dh, generator=g).cuda()
    G = {"t": torch.zeros_like(table)}

    def step():
        G["t"].zero_()
        tp = Tape({"t": table}, G)
        o = T.attention_relpos(tp, q, k, v, "t", rp, H, causal=True)
        tp.acc(o, go, owned=False)
        tp.backward()
        return o, tp.grad(q), tp.grad(k), tp.grad(v), G["t"]
    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(step(), eager):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                           # two graphs of the same inputs: neither touches what the other works in
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for n in range(4):
        q.copy_(torch.randn(q.shape, generator=g).cuda())
        want = [t.clone() for t in step()]
        for gr, out in graphs:
            for t in out:
                t.fill_(float("nan")) if t is not G["t"] else None
            gr.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), n


@pytest.mark.parametrize("scales", [(0.0, 1e-6), (1e-9, 0.0, 1.0), (1.0, 1e-9), (1.0, 1e-9, 1e9, 1e-3, 0.0, 1e-12)], ids=str)
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
def test_tiles_of_very_different_sizes(ops, T, which, scales):
    """rows of 64 that are zeros (a loss over some tokens only) or 2^30 and more apart; a channel of its own for each 64 keys keeps the weights across them
    below 2^-50, so that every row's results are of its own tile's size and have that size's accuracy"""
    from synergize_motion_appearance_amd.tape import Tape
    n = len(scales)
    B, H, S, dh = 1, 1, 64 * n, 64
    q, k, v, g = mk(25, B, H, H, S, S, dh)
    go = torch.randn(B, S, dh, generator=g).cuda()
    scale = 1.0
    for j, f in enumerate(scales):
        own = slice(64 * j, 64 * j + 64)
        if which in ("v", "do"):
            for t in (q, k):
                t[:, own] *= 0.2
                t[:, own, :n] = 0.0
                t[:, own, j] = 7.0                                   # score 49 on the own tile
        {"q": q, "k": k, "v": v, "do": go}[which][:, own] *= f
    rp = ops.relpos(32, 128)
    table = torch.randn(32, H, generator=g).cuda() * 0.1
    G = {"t": torch.zeros_like(table)}
    tp = Tape({"t": table}, G)
    o = T.attention_relpos(tp, q, k, v, "t", rp, H, scale=scale if which in ("v", "do") else None)
    tp.acc(o, go, owned=False)
    tp.backward()
    ref = R.attention(q, k, v, table, rp, H, g=go, scale=scale if which in ("v", "do") else None, apart=8)
    for name, t in (("o", o), ("dq", tp.grad(q)), ("dk", tp.grad(k)), ("dv", tp.grad(v)), ("dtable", G["t"])):
        near(t, ref[name], name)


@pytest.mark.parametrize("Lq, S, dtype", [(1, 40, F32), (1, 3000, F32), (1, 3000, BF), (70, 70, F32), (70, 70, BF), (70, 3000, F32), (70, 3000, BF)])
def test_no_number_in_no_number_out(ops, Lq, S, dtype):
    """a query that is no number gives a row of none, and only that; an infinite value or key is seen in every row that sees it"""
    B, H, dh = 2, 2, 32
    q, k, v, g = mk(26, B, H, H, Lq, S, dh, dtype)
    rp = ops.relpos()
    table = torch.randn(32, H, generator=g).cuda()
    good = ops.attention_relpos(q, k, v, table, rp, H)
    bad = q.clone()
    bad[1, Lq // 2, :dh] = math.nan
    o = ops.attention_relpos(bad, k, v, table, rp, H)
    assert torch.isnan(o[1, Lq // 2, :dh]).all()
    o[1, Lq // 2, :dh] = good[1, Lq // 2, :dh]
    assert torch.equal(o, good)
    for t in (k, v) if Lq > 1 else (v,):                             # (a single query's score of an infinite key may be -inf: no weight)
        w = t.clone()
        w[1, 5, 3] = math.inf
        o = ops.attention_relpos(q, w if t is k else k, w if t is v else v, table, rp, H)
        assert not torch.isfinite(o[1, :, 3]).any() if t is v else not torch.isfinite(o[1, :, :dh]).all(-1).all()
        assert torch.equal(o[0], good[0]) and torch.equal(o[1, :, dh:], good[1, :, dh:])


def test_two_calls_at_once(ops):
    """calls on two streams, each with workspaces of its own"""
    B, H, S, dh = 2, 2, 1300, 64
    q, k, v, g = mk(23, B, H, H, S, S, dh)
    q2, k2, v2, _ = mk(24, B, H, H, S, S, dh)
    rp = ops.relpos()
    table = torch.randn(32, H, generator=g).cuda()
    want = ops.attention_relpos(q, k, v, table, rp, H).clone(), ops.attention_relpos(q2, k2, v2, table, rp, H).clone()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(a):
            x = ops.attention_relpos(q, k, v, table, rp, H)
        with torch.cuda.stream(b):
            y = ops.attention_relpos(q2, k2, v2, table, rp, H)
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_profile_names_the_launch(ops):
    rp, z = ops.relpos(), torch.zeros(1, 40, 64, device="cuda")
    with ops.profile() as rec:
        ops.attention_relpos(z, z, z, torch.zeros(32, 2, device="cuda"), rp, 2)
        ops.norm_residual(z, z)
    assert [r[0] for r in rec.rows] == ["attention_relpos", "norm_residual"] and rec.rows[0][1]["flops"] > 0 and rec.rows[1][1]["bytes"] > 0


def test_single_tokens_answer_what_the_prompt_answers(ops):
    """streaming: the newest token against the keys so far, one step after the other, equals the causal pass over the whole clip (fp32 bounds of both)"""
    B, H, Hkv, S, dh = 2, 4, 2, 70, 32
    q, k, v, g = mk(18, B, H, Hkv, S, S, dh)
    rp = ops.relpos(32, 64, two_sided=False)
    table = torch.randn(32, H, generator=g).cuda()
    whole = R.attention(q, k, v, table, rp, H, nkv=Hkv, causal=True)["o"]
    near(ops.attention_relpos(q, k, v, table, rp, H, nkv=Hkv, causal=True), whole)
    for n in (1, 2, 33, 64, 65, 70):
        lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
        near(ops.attention_relpos(q[:, n - 1:n], k, v, table, rp, H, nkv=Hkv, causal=True, kv_len=lens), (whole[0][:, n - 1:n], whole[1][:, n - 1:n]))


def test_far_offsets(ops):
    """a cache whose last sample starts beyond 2^31 elements"""
    H, dh, S = 2, 128, 4000
    bs = 2 ** 31 + 4096
    buf = torch.zeros(bs + S * 2 * H * dh, device="cuda", dtype=BF)
    kv = buf.as_strided((2, S, 2 * H * dh), (bs, 2 * H * dh, 1))
    g = torch.Generator().manual_seed(19)
    kv.copy_(torch.randn(2, S, 2 * H * dh, generator=g).cuda())
    k, v = kv[..., :H * dh], kv[..., H * dh:]
    rp = ops.relpos(32, 128, two_sided=False)
    table = torch.randn(32, H, generator=g).cuda()
    for Lq in (1, 40):
        q = torch.randn(2, Lq, H * dh, generator=g).to(BF).cuda()
        near(ops.attention_relpos(q, k, v, table, rp, H, causal=True), R.attention(q, k, v, table, rp, H, causal=True, storage=BF)["o"])
