"""`norm_residual` and `attention_relpos` at the ends of their shapes, against fp64: the widest rows with several of them a block, a gate row for each of
thousands of tokens, hundreds of short samples."""
import pytest
import torch

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


def norms(T, n, E, kind, groups):
    """one forward and backward -> ({name: got}, the fp64 ones)"""
    from synergize_motion_appearance_amd.tape import Tape
    g = torch.Generator().manual_seed(n + E)
    x, h, gx, gy = (torch.randn(n, E, generator=g).cuda() for _ in range(4))
    w = {p: tuple((1 - i + 0.1 * torch.randn(E, generator=g)).cuda() for i in range(2 if kind == "layer" else 1)) for p in ("post", "pre")}
    gate = None if groups is None else torch.randn(groups, E, generator=g).cuda()
    P = {p + str(i): t for p in w for i, t in enumerate(w[p])}
    G = {k: torch.zeros_like(t) for k, t in P.items()}
    tp = Tape(P, G)
    xo, y = T.norm_residual(tp, x, h, post=tuple(k for k in P if k.startswith("post")), pre=tuple(k for k in P if k.startswith("pre")), gate=gate, kind=kind)
    tp.acc(xo, gx, owned=False)
    tp.acc(y, gy, owned=False)
    tp.backward()
    got = {"x": xo, "y": y, "dx": tp.grad(x), "dh": tp.grad(h), **{"d" + k: t for k, t in G.items()}}
    if gate is not None:
        got["dgate"] = tp.grad(gate)
    return got, R.norm_residual(x, h, gate=gate, kind=kind, gx=gx, gy=gy, **w), x, h, gx, gy


# a value is a chain of some 12 roundings around two row sums of E terms, a gradient two of them; a parameter's sum adds one of T terms at most (2-norms, all adding up)
@pytest.mark.parametrize("n,E,kind,groups", [(700, 4100, "layer", 1), (700, 8192, "rms", 2), (600, 8200, "layer", None), (700, 16384, "layer", 1), (520, 16383, "rms", 2),
                                             (1030, 2050, "layer", 1)])
def test_several_wide_rows_a_block(T, n, E, kind, groups):
    got, ref, *_ = norms(T, n, E, kind, groups)
    for k, t in got.items():
        sums = k[1:].startswith(("post", "pre", "gate"))
        tol = 4 * (24 + E / 256 + (n / 4 if sums else 0)) * R.U32
        assert float((t.double().cpu() - ref[k]).norm()) < tol * float(ref[k].norm()), k


@pytest.mark.parametrize("n,E,kind", [(5000, 64, "layer"), (3001, 200, "rms"), (9000, 33, "layer")])
def test_a_gate_row_for_each_of_thousands_of_tokens(T, n, E, kind):
    """every element of the parameters' sums within n / 32 + 64 roundings of the sum of its terms' sizes (32 runs of the tokens and their joint) and two of each term's
    own chain"""
    got, ref, x, h, gx, gy = norms(T, n, E, kind, n)
    for k, t in got.items():
        if not k[1:].startswith(("post", "pre")):
            assert float((t.double().cpu() - ref[k]).norm()) < 8 * (24 + E / 256) * R.U32 * float(ref[k].norm()), k
    y = ref["x"] - (ref["x"].mean(-1, keepdim=True) if kind == "layer" else 0)
    hat = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    sizes = {"dpre0": (gy.double().cpu() * hat).abs().sum(0), "dpre1": gy.double().cpu().abs().sum(0)}
    for k, size in sizes.items():
        if k in got:
            off = (got[k].double().cpu() - ref[k]).abs() - (n / 32 + 64 + 2 * (24 + E / 256)) * R.U32 * size
            assert float(off.max()) <= 0, k


def near(got, ref, what=""):
    val, bound = ref
    off = (got.double().cpu() - val).abs() - bound
    assert torch.isfinite(got).all() and float(off.max()) <= 0, what


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,S,causal", [(300, 16, False), (257, 33, True)])
def test_hundreds_of_short_samples(ops, T, dtype, B, S, causal):
    """attention over the frames of a clip, one sample for every place of the token grid, ragged and masked; one token a sample too"""
    from synergize_motion_appearance_amd.tape import Tape
    H, dh = 2, 32
    g = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(B, S, H * dh, generator=g).to(dtype).cuda() for _ in range(3))
    rp = ops.RelPos(16, 24, not causal)
    table = torch.randn(16, H, generator=g).cuda()
    kw = dict(causal=causal, mask=(torch.rand(B, S, generator=g) < 0.2).cuda(), kv_len=torch.randint(0, S + 1, (B,), generator=g, dtype=torch.int32).cuda())
    ref = R.attention(q, k, v, table, rp, H, storage=dtype, **kw)["o"]
    near(ops.attention_relpos(q, k, v, table, rp, H, **kw), ref)
    near(ops.attention_relpos(q[:, -1:], k, v, table, rp, H, **kw), (ref[0][:, -1:], ref[1][:, -1:]))
    if dtype is F32:
        go = torch.randn(B, S, H * dh, generator=g).cuda()
        tp = Tape({"t": table}, {"t": torch.zeros_like(table)})
        o = T.attention_relpos(tp, q, k, v, "t", rp, H, **kw)
        tp.acc(o, go, owned=False)
        tp.backward()
        ref = R.attention(q, k, v, table, rp, H, g=go, **kw)
        for t, n in ((tp.grad(q), "dq"), (tp.grad(k), "dk"), (tp.grad(v), "dv")):
            near(t, ref[n], n)
        # (the bound counts (L + S) / 4 + 64 roundings of the sum of sizes; a bucket's sum runs over the samples' blocks too, B more)
        val, bound = ref["dtable"]
        near(tp.G["t"], (val, bound * (1 + B / (S / 2 + 64))), "dtable")
