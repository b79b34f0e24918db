"""`ops.norm_residual` and `train_ops.norm_residual` on a real MI355X against fp64: both norms, gates of every shape, odd widths, one token to many, both storage
types, the backward with every parameter's gradient."""
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


def mk(seed, T_, E, dtype, kind, post, pre, groups, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    w = {"x": (r(T_, E) * 2 + shift).to(dtype).cuda(), "h": (r(T_, E) + shift).to(dtype).cuda()}
    w["gate"] = None if groups is None else (r(E) if groups == 0 else r(groups, E)).cuda()
    for n, on in (("post", post), ("pre", pre)):
        w[n] = None if not on else ((1 + 0.1 * r(E)).cuda(), (0.1 * r(E)).cuda()) if kind == "layer" else ((1 + 0.1 * r(E)).cuda(),)
    return w, g


def rel(a, b):
    return float((a.double().cpu() - b).norm() / b.norm().clamp_min(1e-300)) if b.numel() else 0.0


# fp32: a value is a chain of some 12 roundings around two row sums of E terms (pairwise within lanes and waves: depth <= 16 + E / 256) -- 2^-24 each, and the
# parameters' sums run over at most T tokens in a chain; taken in the 2-norm, all adding up
def tol(E, T_, dtype, sums=False):
    return (24 + E / 256 + (T_ / 4 if sums else 0)) * R.U32 + (3 * R.U[BF] if dtype == BF else 0)     # bf16: x' rounded, y of the rounded x' rounded


CASES = [  # T, E, kind, post, pre, groups (None: no gate, 0: [E]), res_scale
    (1, 1, "rms", True, True, None, 1.0),
    (1, 4, "layer", True, True, 0, 1.0),
    (3, 33, "layer", True, True, 3, 0.5),
    (7, 256, "layer", True, True, 0, 1.0),
    (64, 32, "layer", True, False, 1, 1.0),
    (65, 100, "rms", False, True, 5, 1.25),
    (130, 255, "layer", True, True, 130, 1.0),
    (40, 512, "layer", False, False, 0, -1.0),
    (33, 1000, "rms", True, True, 0, 1.0),
    (12, 1026, "layer", True, True, 2, 1.0),
    (9, 2048, "rms", True, True, 3, 0.5),
    (5, 4100, "layer", True, True, 0, 1.0),
    (3, 8192, "rms", True, True, None, 1.0),
    (2, 16384, "layer", True, True, 0, 1.0),
    (2000, 256, "layer", True, True, 4, 1.0),
    (5001, 64, "rms", True, True, 3, 1.0),
    (3001, 2049, "layer", True, True, 0, 1.0),
]


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", CASES, ids=str)
def test_forward(ops, c, dtype):
    T_, E, kind, post, pre, groups, rs = c
    w, _ = mk(1, T_, E, dtype, kind, post, pre, groups)
    x0, h0 = w["x"].clone(), w["h"].clone()
    xo, y = ops.norm_residual(**w, res_scale=rs, kind=kind)
    ref = R.norm_residual(**w, res_scale=rs, kind=kind)
    assert xo.dtype == dtype and rel(xo, ref["x"]) < tol(E, T_, dtype)
    assert (y is None) == (not pre)
    if pre and E > 1:
        # a row whose variance is far below its values' size loses what it loses in any arithmetic: the rows here have none
        assert rel(y, ref["y"]) < tol(E, T_, dtype)
    assert torch.equal(w["x"], x0) and torch.equal(w["h"], h0)


@pytest.mark.parametrize("c", CASES, ids=str)
def test_backward(ops, T, c):
    from synergize_motion_appearance_amd.tape import Tape
    T_, E, kind, post, pre, groups, rs = c
    w, g = mk(2, T_, E, F32, kind, post, pre, groups)
    gx, gy = (torch.randn(T_, E, generator=g).cuda() for _ in range(2))
    P = {n + str(i): t for n in ("post", "pre") if w[n] for i, t in enumerate(w[n])}
    P["gate"] = w["gate"] if w["gate"] is not None else torch.zeros(1, device="cuda")
    old = {n: torch.randn(t.shape, generator=g).cuda() for n, t in P.items()}
    refs = {n: tuple(f"{n}{i}" for i in range(len(w[n]))) if w[n] else None for n in ("post", "pre")}
    for with_gx, with_gy, as_param in ((True, True, True), (False, True, False), (True, False, True)):
        if with_gy and not pre:
            if not with_gx:
                continue
            with_gy = False
        G = {n: t.clone() for n, t in old.items()}
        tp = Tape(P, G)
        gate = None if w["gate"] is None else "gate" if as_param else w["gate"]
        xo, y = T.norm_residual(tp, w["x"], w["h"], gate=gate, res_scale=rs, kind=kind, **refs)
        if with_gx:
            tp.acc(xo, gx, owned=False)
        if with_gy:
            tp.acc(y, gy, owned=False)
        tp.backward()
        ref = R.norm_residual(**w, res_scale=rs, kind=kind, gx=gx if with_gx else None, gy=gy if with_gy else None)
        t, ts = 2 * tol(E, T_, F32), 2 * tol(E, T_, F32, True)
        # (E = 1 under a norm: the gradient is a difference of equal numbers)
        scale = float(gx.norm()) if E == 1 else 0.0
        near = lambda a, b, tt: float((a.double().cpu() - b).norm()) <= tt * (float(b.norm()) + scale)  # noqa: E731
        assert near(tp.grad(w["x"]), ref["dx"], t)
        # dh is a difference: what it cancels is of the size of the gradient that enters, through r
        assert near(tp.grad(w["h"]), ref["dh"], 2 * t), rel(tp.grad(w["h"]), ref["dh"])
        for n in ("post", "pre"):
            for i in range(len(w[n]) if w[n] else 0):
                want = ref.get(f"d{n}{i}", torch.zeros(E).double()) + old[f"{n}{i}"].double().cpu()
                assert near(G[f"{n}{i}"], want, ts), f"{n}{i}"
        if w["gate"] is not None:
            got = G["gate"].double().cpu() - old["gate"].double().cpu() if as_param else tp.grad(w["gate"]).double().cpu()
            assert float((got - ref["dgate"]).norm()) <= ts * (float(ref["dgate"].norm()) + float(old["gate"].norm())) + scale * ts


def test_offset_rows_keep_their_variance(ops):
    """values around 300 with deviations around one: the variance is of the deviations, not a difference of squares (its loss here: 300 * 2^-24 per value)"""
    w, _ = mk(3, 50, 777, F32, "layer", True, True, None, shift=300.0)
    xo, y = ops.norm_residual(**w)
    ref = R.norm_residual(**w)
    assert rel(y, ref["y"]) < 300 * 12 * R.U32


def test_batched_shapes_and_same_tensor(ops, T):
    """[B, H, W, E] tokens; x and h the same tensor: its gradient is the sum of both"""
    from synergize_motion_appearance_amd.tape import Tape
    w, g = mk(4, 2 * 6 * 5, 64, F32, "layer", True, True, 2)
    x = w["x"].view(2, 6, 5, 64)
    xo, y = ops.norm_residual(x, x, post=w["post"], pre=w["pre"], gate=w["gate"])
    assert xo.shape == y.shape == x.shape
    gx, gy = (torch.randn(60, 64, generator=g).cuda() for _ in range(2))
    P = {"a": w["post"][0], "b": w["post"][1], "c": w["pre"][0], "d": w["pre"][1]}
    tp = Tape(P, {n: torch.zeros_like(t) for n, t in P.items()})
    xo, y = T.norm_residual(tp, x, x, post=("a", "b"), pre=("c", "d"), gate=w["gate"])
    tp.acc(xo, gx.view(x.shape), owned=False)
    tp.acc(y, gy.view(x.shape), owned=False)
    tp.backward()
    ref = R.norm_residual(w["x"], w["x"], post=w["post"], pre=w["pre"], gate=w["gate"], gx=gx, gy=gy)
    assert rel(tp.grad(x).view(60, 64), ref["dx"] + ref["dh"]) < 4 * tol(64, 60, F32)


def test_left_over_rows_and_empty(ops):
    """nothing behind the last token is written"""
    for dtype in (F32, BF):
        w, _ = mk(5, 11, 96, dtype, "layer", True, True, None)
        xo, y = ops.norm_residual(w["x"][:7], w["h"][:7], post=w["post"], pre=w["pre"])
        full, fy = ops.norm_residual(w["x"], w["h"], post=w["post"], pre=w["pre"])
        assert torch.equal(xo, full[:7]) and torch.equal(y, fy[:7])
        a, b = ops.norm_residual(w["x"][:0], w["h"][:0], post=w["post"], pre=w["pre"])
        assert a.shape == b.shape == (0, 96)


@pytest.mark.parametrize("E", [5, 7, 33, 66, 100, 260, 1025, 2470, 4099, 8191, 16383])
def test_rows_that_start_anywhere(ops, T, E):
    """contiguous views behind an odd number of rows: no 16-byte alignment to rely on"""
    from synergize_motion_appearance_amd.tape import Tape
    for dtype in (F32, BF):
        w, g = mk(8, 11, E, dtype, "layer", True, True, 0)
        v = {**w, "x": w["x"][1:], "h": w["h"][1:]}
        xo, y = ops.norm_residual(**v)
        ref = R.norm_residual(**v)
        assert rel(xo, ref["x"]) < tol(E, 10, dtype) and rel(y, ref["y"]) < tol(E, 10, dtype)
    w, g = mk(9, 11, E, F32, "layer", True, True, 0)
    gx, gy = (torch.randn(11, E, generator=g).cuda()[1:] for _ in range(2))
    x, h = w["x"][1:], w["h"][1:]
    P = {"a": w["post"][0], "b": w["post"][1], "c": w["pre"][0], "d": w["pre"][1], "gate": w["gate"]}
    G = {n: torch.zeros_like(t) for n, t in P.items()}
    tp = Tape(P, G)
    xo, y = T.norm_residual(tp, x, h, post=("a", "b"), pre=("c", "d"), gate="gate")
    tp.acc(xo, gx, owned=False)
    tp.acc(y, gy, owned=False)
    tp.backward()
    ref = R.norm_residual(x, h, post=w["post"], pre=w["pre"], gate=w["gate"], gx=gx, gy=gy)
    t = 2 * tol(E, 11, F32, True)
    for a, b in ((tp.grad(x), "dx"), (tp.grad(h), "dh"), (G["gate"], "dgate"), (G["a"], "dpost0"), (G["b"], "dpost1"), (G["c"], "dpre0"), (G["d"], "dpre1")):
        assert rel(a, ref[b]) < 2 * t, b


def test_a_gate_row_for_every_token(ops, T):
    """as many gate rows as tokens, and a residual stream that takes no gradient"""
    from synergize_motion_appearance_amd.tape import Tape
    n, E = 700, 64
    w, g = mk(10, n, E, F32, "rms", True, True, n)
    gx, gy = (torch.randn(n, E, generator=g).cuda() for _ in range(2))
    P = {"a": w["post"][0], "c": w["pre"][0]}
    G = {k: torch.zeros_like(t) for k, t in P.items()}
    tp = Tape(P, G)
    tp.stop(w["x"])
    xo, y = T.norm_residual(tp, w["x"], w["h"], post=("a",), pre=("c",), gate=w["gate"], kind="rms")
    tp.acc(xo, gx, owned=False)
    tp.acc(y, gy, owned=False)
    tp.backward()
    ref = R.norm_residual(**w, kind="rms", gx=gx, gy=gy)
    assert tp.grad(w["x"]) is None
    for a, b in ((tp.grad(w["h"]), "dh"), (tp.grad(w["gate"]), "dgate"), (G["a"], "dpost0"), (G["c"], "dpre0")):
        assert rel(a, ref[b]) < 4 * tol(E, n, F32, True), b


def test_one_parameter_in_two_places(ops, T):
    """tied norms: a parameter's gradient is the sum of both places'; a gate that is a norm's scale too"""
    from synergize_motion_appearance_amd.tape import Tape
    n, E = 900, 100
    w, g = mk(11, n, E, F32, "layer", True, True, 0)
    gx, gy = (torch.randn(n, E, generator=g).cuda() for _ in range(2))
    P = {"a": w["post"][0], "b": w["post"][1]}
    for gate in (None, "a"):
        G = {k: torch.zeros_like(t) for k, t in P.items()}
        tp = Tape(P, G)
        xo, y = T.norm_residual(tp, w["x"], w["x"], post=("a", "b"), pre=("a", "b"), gate=gate)
        tp.acc(xo, gx, owned=False)
        tp.acc(y, gy, owned=False)
        tp.backward()
        ref = R.norm_residual(w["x"], w["x"], post=w["post"], pre=w["post"], gate=None if gate is None else w["post"][0], gx=gx, gy=gy)
        t = 8 * tol(E, n, F32, True)
        a = ref["dpost0"] + ref["dpre0"] + (0 if gate is None else ref["dgate"].view(E))
        assert rel(G["a"], a) < t and rel(G["b"], ref["dpost1"] + ref["dpre1"]) < t and rel(tp.grad(w["x"]), ref["dx"] + ref["dh"]) < t


def test_refusals(ops):
    w, _ = mk(6, 12, 64, F32, "layer", True, True, 3)
    for bad in (dict(x=w["x"].half()), dict(h=w["h"].bfloat16()), dict(h=w["h"][:6]), dict(x=w["x"][:, ::2], h=w["h"][:, ::2]), dict(kind="batch"),
                dict(gate=torch.ones(5, 64, device="cuda")), dict(gate=torch.ones(3, 32, device="cuda")), dict(gate=torch.ones(3, 64)),
                dict(gate=torch.ones(3, 64, device="cuda", dtype=BF)), dict(post=w["post"][0]), dict(pre=(w["pre"][0][:32],)), dict(post=(w["post"][0].cpu(),)),
                dict(x=w["x"].cpu())):
        with pytest.raises(L.SmxError):
            ops.norm_residual(**{**w, **bad})


def test_graph_replays(ops, T):
    from synergize_motion_appearance_amd.tape import Tape
    w, g = mk(7, 300, 256, F32, "layer", True, True, 2)
    gx, gy = (torch.randn(300, 256, generator=g).cuda() for _ in range(2))
    P = {"a": w["post"][0], "b": w["post"][1], "c": w["pre"][0], "d": w["pre"][1], "gate": w["gate"]}
    G = {n: torch.zeros_like(t) for n, t in P.items()}

    def step():
        for t in G.values():
            t.zero_()
        tp = Tape(P, G)
        xo, y = T.norm_residual(tp, w["x"], w["h"], post=("a", "b"), pre=("c", "d"), gate="gate")
        tp.acc(xo, gx, owned=False)
        tp.acc(y, gy, owned=False)
        tp.backward()
        return [xo, y, tp.grad(w["x"]), tp.grad(w["h"])] + [G[n] for n in sorted(G)]
    step()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step()
    for _ in range(4):
        w["x"].copy_(torch.randn(300, 256, generator=g).cuda())
        want = [t.clone() for t in step()]
        for t in out[:4]:
            t.fill_(float("nan"))
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_one_layer(ops, T):
    """the run of them as a layer uses them: x, y = norms(x, attention(y)), twice, forward and backward against fp64 autograd"""
    from synergize_motion_appearance_amd.tape import Tape
    B, S, H, dh = 2, 90, 4, 16
    E = H * dh
    g = torch.Generator().manual_seed(20)
    rp = ops.relpos(32, 64)
    P = {"table": torch.randn(32, H, generator=g), "gate": torch.randn(E, generator=g) * 0.3}
    for n in ("n1", "n2", "n3"):
        P[n + ".w"], P[n + ".b"] = 1 + 0.1 * torch.randn(E, generator=g), 0.1 * torch.randn(E, generator=g)
    x, y, go = (torch.randn(B, S, E, generator=g) for _ in range(3))
    mask = torch.rand(B, S, generator=g) < 0.2
    D = {n: t.cuda() for n, t in P.items()}
    G = {n: torch.zeros_like(t) for n, t in D.items()}
    tp = Tape(D, G)
    xd, yd = x.cuda(), y.cuda()
    a, b = xd, yd
    for n in ("n1", "n2"):
        a, b = T.norm_residual(tp, a, T.attention_relpos(tp, b, b, b, "table", rp, H, mask=mask.cuda()), post=(n + ".w", n + ".b"), pre=("n3.w", "n3.b"), gate="gate")
    tp.acc(b, go.cuda(), owned=False)
    tp.backward()
    Q = {n: t.double().requires_grad_() for n, t in P.items()}
    X, Y = x.double().requires_grad_(), y.double().requires_grad_()
    idx = torch.tensor([[rp.bucket(j - i) for j in range(S)] for i in range(S)])
    u, w = X, Y
    for n in ("n1", "n2"):
        z = w.view(B, S, H, dh).transpose(1, 2)
        s = z @ z.transpose(-1, -2) * dh ** -0.5 + Q["table"][idx].permute(2, 0, 1)
        h = (torch.softmax(s.masked_fill(mask[:, None, None, :], float("-inf")), -1) @ z).transpose(1, 2).reshape(B, S, E)
        u = u + Q["gate"] * torch.nn.functional.layer_norm(h, (E,), Q[n + ".w"], Q[n + ".b"], 1e-5)
        w = torch.nn.functional.layer_norm(u, (E,), Q["n3.w"], Q["n3.b"], 1e-5)
    names = sorted(Q)
    want = torch.autograd.grad((w * go.double()).sum(), [X, Y] + [Q[n] for n in names])
    # two layers of some 40 roundings on a path, each amplified by the norms' 1 / deviation (attention's averages: about 4 a layer)
    t = 2 * 40 * 16 * R.U32
    assert rel(b, w.detach()) < t
    for have, ref in zip([tp.grad(xd), tp.grad(yd)] + [G[n] for n in names], want):
        assert rel(have, ref) < t
