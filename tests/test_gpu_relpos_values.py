"""`ops.attention_relpos` and `train_ops.attention_relpos` on a real MI355X: values where arithmetic of fewer bits, very different sizes and places that
do not count could show, against the formula in fp64 (tests/layer_ref.py)."""
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


def mk(seed, B, H, Hkv, Lq, S, dh, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (*(torch.randn(B, n, h * dh, generator=g).to(dtype).cuda() for n, h in ((Lq, H), (S, Hkv), (S, Hkv))), g)


def near(got, val, bound, what=""):
    got = got.detach().double().cpu()
    assert got.shape == val.shape and torch.isfinite(got).all(), what
    off = (got - val).abs() - bound
    assert float(off.max()) <= 0, f"{what}: over its bound by {float(off.max()):.3e}, {int((off > 0).sum())} of {off.numel()}"


# B, H, Hkv, L, S, dh, causal, masked, ragged
PROMPTS = [(1, 2, 1, 2, 40, 32, False, False, False), (2, 4, 2, 70, 70, 64, True, True, False), (3, 2, 2, 33, 300, 80, False, True, True),
           (1, 2, 1, 130, 2000, 128, False, False, False), (2, 2, 2, 40, 1300, 4, True, False, False), (1, 8, 2, 600, 600, 32, True, False, False)]


@pytest.mark.parametrize("c", PROMPTS, ids=str)
def test_bf16_prompts_are_rounded_once(ops, c):
    """bf16 storage of several queries: what the weights' two bf16 parts leave (2^-8 of 2^-8 of a weight) and the output's own rounding, next to the bound of fp32
    arithmetic.  One part alone would be off by up to 2^-8 of a weight."""
    B, H, Hkv, Lq, S, dh, causal, masked, ragged = c
    q, k, v, g = mk(31, B, H, Hkv, Lq, S, dh, BF)
    rp = ops.relpos(32, 128, two_sided=not causal)
    table = torch.randn(32, H, generator=g).cuda()
    kw = dict(nkv=Hkv, causal=causal, mask=(torch.rand(B, S, generator=g) < 0.3).cuda() if masked else None,
              kv_len=torch.tensor([S, S // 2, 1][:B], dtype=torch.int32).cuda() if ragged else None)
    val, bound = R.attention(q, k, v, table, rp, H, **kw)["o"]
    spread = R.attention(q, k, v.abs(), table, rp, H, **kw)["o"][0]
    near(ops.attention_relpos(q, k, v, table, rp, H, **kw), val, bound + 2.0 ** -16 * spread + R.U[BF] * val.abs())


def step(T, q, k, v, table, rp, H, go, **kw):
    from synergize_motion_appearance_amd.tape import Tape
    G = {"t": torch.zeros_like(table)}
    tp = Tape({"t": table}, G)
    o = T.attention_relpos(tp, q, k, v, "t", rp, H, **kw)
    tp.acc(o, go, owned=False)
    tp.backward()
    return o, tp.grad(q), tp.grad(k), tp.grad(v), G["t"]


def test_a_map_that_only_the_tape_holds(ops, T):
    """a RelPos made for one call, its map's size of memory written over between the forward and the backward"""
    from synergize_motion_appearance_amd.tape import Tape
    B, H, S, dh = 2, 2, 100, 32
    q, k, v, g = mk(35, B, H, H, S, S, dh)
    table, go = torch.randn(24, H, generator=g).cuda(), torch.randn(B, S, H * dh, generator=g).cuda()
    want = step(T, q, k, v, table, ops.relpos(24, 301), H, go)
    G = {"t": torch.zeros_like(table)}
    tp = Tape({"t": table}, G)
    o = T.attention_relpos(tp, q, k, v, "t", ops.RelPos(24, 301), H)
    n = len(ops.relpos(24, 301).map)
    over = [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(8)]
    tp.acc(o, go, owned=False)
    tp.backward()
    for x, y in zip((o, tp.grad(q), tp.grad(k), tp.grad(v), G["t"]), want):
        assert torch.equal(x, y)
    assert len(over) == 8


@pytest.mark.parametrize("dh", [32, 64, 128])
def test_dk_of_far_smaller_gradients(ops, T, dh):
    """output gradients of 64 rows 2^-110 of those before them, and a key that so far has met exact zeros only: its dk is of the small ones' size.  A dS of some 2^-113
    is carried times 2^100 in two halves, off by at most half of the lowest bit 2^-24: 2^-125."""
    q, k, v, g = mk(32, 1, 1, 1, 128, 128, dh)
    go = torch.randn(1, 128, dh, generator=g)
    go[:, 63] = 0
    go[:, 64:] *= 2.0 ** -110
    go = go.cuda()
    rp = ops.relpos(32, 128, two_sided=False)
    table = torch.randn(32, 1, generator=g).cuda()
    out = step(T, q, k, v, table, rp, 1, go, causal=True)
    val, bound = R.attention(q, k, v, table, rp, 1, causal=True, g=go)["dk"]
    for t in out:
        assert torch.isfinite(t).all()
    near(out[2], val, bound + dh ** -0.5 * 2.0 ** -125 * q.double().cpu().abs().sum(1, keepdim=True), "dk")


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3e38])
@pytest.mark.parametrize("which", ["q", "do"])
def test_queries_without_a_key_do_not_count_in_the_backward(ops, T, which, bad):
    """padding in front of a short sample, a sample whose mask leaves nothing: what those queries and their output gradients hold changes no gradient by a bit,
    and their own is zero"""
    B, H, S, dh = 3, 2, 150, 32
    q, k, v, g = mk(33, B, H, H, S, S, dh)
    go = torch.randn(B, S, H * dh, generator=g).cuda()
    rp = ops.relpos(32, 128, two_sided=False)
    table = torch.randn(32, H, generator=g).cuda()
    mask = torch.zeros(B, S, dtype=torch.uint8)
    mask[1] = 1
    kw = dict(causal=True, mask=mask.cuda(), kv_len=torch.tensor([S, S, 77], dtype=torch.int32).cuda())
    empty = torch.zeros(B, S, 1, dtype=torch.bool)
    empty[1], empty[2, :S - 77] = True, True
    empty = empty.cuda()

    def with_(x):
        return step(T, q.masked_fill(empty, x if which == "q" else 0.0), k, v, table, rp, H, go.masked_fill(empty, x if which == "do" else 0.0), **kw)
    a, b = with_(0.0), with_(bad)
    for x, y, n in zip(a, b, ("o", "dq", "dk", "dv", "dtable")):
        assert torch.isfinite(y).all() and torch.equal(x, y), n
    assert float(b[1].masked_select(empty.expand_as(b[1])).abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("Lq", [1, 4, 96])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3e38])
def test_keys_behind_the_last_query_do_not_count(ops, T, dtype, Lq, bad):
    """a cache that is longer than what has been written, with a causal rule and the first query's position: no result changes by a bit with what lies behind the
    last query, and those keys' gradients are zeros"""
    B, H, S, dh, start = 2, 2, 300, 64, 103
    q, k, v, g = mk(34, B, H, H, Lq, S, dh, dtype)
    rp = ops.relpos(32, 128, two_sided=False)
    table = torch.randn(32, H, generator=g).cuda()
    go = torch.randn(B, Lq, H * dh, generator=g).cuda()
    kw = dict(causal=True, q_start=start)

    def with_(x):
        kk, vv = k.clone(), v.clone()
        kk[:, start + Lq:], vv[:, start + Lq:] = x, x
        return step(T, q, kk, vv, table, rp, H, go, **kw) if dtype == F32 else (ops.attention_relpos(q, kk, vv, table, rp, H, **kw),)
    a, b = with_(0.0), with_(bad)
    for x, y in zip(a, b):
        assert torch.isfinite(y).all() and torch.equal(x, y)
    if dtype == F32:
        assert float(b[2][:, start + Lq:].abs().max()) == 0.0 and float(b[3][:, start + Lq:].abs().max()) == 0.0
    ref = R.attention(q, k[:, :start + Lq], v[:, :start + Lq], table, rp, H, storage=dtype, **kw)["o"]
    near(b[0], *ref)


@pytest.mark.parametrize("stopped", ["q", "k", "kv", "t", "qt", "kvt", "qkv", "qkvt"])
@pytest.mark.parametrize("S", [90, 1500])                        # (1500: both sides in parts)
def test_gradients_that_are_wanted_do_not_depend_on_the_others(ops, T, stopped, S):
    from synergize_motion_appearance_amd.tape import Tape
    q, k, v, g = mk(36, 1, 2, 1, S, S, 32)
    table, go = torch.randn(32, 2, generator=g).cuda(), torch.randn(1, S, 64, generator=g).cuda()
    rp = ops.relpos()
    want = step(T, q, k, v, table, rp, 2, go, nkv=1)
    G = {} if "t" in stopped else {"t": torch.zeros_like(table)}
    tp = Tape({"t": table}, G)
    for n, t in (("q", q), ("k", k), ("v", v)):
        if n in stopped:
            tp.stop(t)
    o = T.attention_relpos(tp, q, k, v, "t", rp, 2, nkv=1)
    tp.acc(o, go, owned=False)
    tp.backward()
    for n, got, ref in zip("qkvt", (tp.grad(q), tp.grad(k), tp.grad(v), G.get("t")), want[1:]):
        assert got is None if n in stopped else torch.equal(got, ref), n


@pytest.mark.parametrize("Lq", [1, 100])
@pytest.mark.parametrize("S", [500, 2000])
@pytest.mark.parametrize("e", [-115, -90, 90])
def test_far_values_keep_their_bits(ops, T, Lq, S, e):
    """values (and, in the other direction, output gradients) of size 2^e: results of their size are as accurate as those of size one"""
    q, k, v, g = mk(37, 2, 2, 1, Lq, S, 32)
    rp = ops.relpos()
    table, go = torch.randn(32, 2, generator=g).cuda(), torch.randn(2, Lq, 64, generator=g).cuda()
    f = 2.0 ** e
    near(ops.attention_relpos(q, k, v * f, table, rp, 2, nkv=1), *R.attention(q, k, v * f, table, rp, 2, nkv=1)["o"], "o")
    if abs(e) < 100:                                             # (dS of size 2^-91 and more)
        out = step(T, q, k, v, table, rp, 2, go * f, nkv=1)
        ref = R.attention(q, k, v, table, rp, 2, nkv=1, g=go * f)
        for t, n in zip(out[1:], ("dq", "dk", "dv", "dtable")):
            val, bound = ref[n]
            near(t, val, bound + 2.0 ** -125 * S, n)
