"""fp64 forms of `ops.attention_relpos` and `ops.norm_residual` from their formulas, with the bounds that rounding puts on the kernels' errors."""
import math

import torch

U32 = 2.0 ** -24                                       # half a step of fp32, relative
U = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}


def bucket(num_buckets, max_distance, two_sided, delta):
    """bucket of one whole distance: the largest t with (n / half)^(nb - half) >= (max / half)^t, in whole numbers"""
    nb = num_buckets // 2 if two_sided else num_buckets
    half, n = nb // 2, abs(delta)
    side = 0
    if delta > 0:
        if not two_sided:
            return 0
        side = nb
    if n < half:
        return side + n
    t = max(t for t in range(nb - half) if n ** (nb - half) * half ** t >= max_distance ** t * half ** (nb - half))
    return side + half + t


def attention(q, k, v, table, rp, nhead, nkv=None, causal=False, mask=None, kv_len=None, q_start=None, scale=None, g=None, storage=torch.float32, apart=0):
    """-> {"o", ("dq", "dk", "dv", "dtable")}, each with its bound: (value, largest error that rounding allows), fp64 on the CPU.
    Left-out keys are not used, queries with no key give zeros.  fp32 storage: a factor w of a sum over rows (weights, dS) is two halves of w 2^s; the second
    half's lowest bit is 2^-24, so that w is off by up to 2^-25 2^-s, or by w itself if it is smaller.  2^s brings a row's largest weight to 2^6 at least in the
    forward (2^-31 of it), weights to 2^14 in dv (2^-39), a column's largest |dS| to 2^9 at least (2^-34 of it); apart: binary orders less where staged
    tiles differ in size."""
    nkv = nhead if nkv is None else nkv
    B, L, E = q.shape
    S, dh, G = k.shape[1], E // nhead, nhead // nkv
    scale = dh ** -0.5 if scale is None else scale
    q, k, v, table = (t.detach().double().cpu() for t in (q, k, v, table))
    lens = [S] * B if kv_len is None else [max(0, min(int(n), S)) for n in kv_len.cpu()]
    u = U[storage]
    # half a step of each product's factors where they are kept in fewer bits than fp32's 24 (22 at the least: two halves of 11), the sums in any order
    prod = 2.0 ** -21 if storage == torch.float32 else 0.0
    names = ["o"] + (["dq", "dk", "dv", "dtable"] if g is not None else [])
    out = {n: [torch.zeros(s, dtype=torch.float64), torch.zeros(s, dtype=torch.float64)] for n, s in
           zip(names, [(B, L, E), (B, L, E), (B, S, nkv * dh), (B, S, nkv * dh), tuple(table.shape)])}
    g = None if g is None else g.detach().double().cpu()
    for b in range(B):
        n = lens[b]
        see = torch.zeros((S,), dtype=torch.bool)
        see[:n] = True
        if mask is not None:
            see &= mask[b].cpu() == 0
        pos = torch.arange(L) + (n - L if q_start is None else q_start)
        delta = torch.arange(S)[None, :] - pos[:, None]
        see = see[None, :].expand(L, S).clone()
        gone = ~see[0] if L else torch.ones(S, dtype=torch.bool)
        if causal:
            see &= delta <= 0
        lo = int(delta.min()) if delta.numel() else 0
        which = torch.tensor([rp.bucket(x) for x in range(lo, lo + L + S)], dtype=torch.long)[delta - lo]
        for h in range(nhead):
            c, ck = slice(h * dh, (h + 1) * dh), slice(h // G * dh, (h // G + 1) * dh)
            Q, K, V = q[b, :, c], k[b, :, ck].masked_fill(gone[:, None], 0.0), v[b, :, ck].masked_fill(gone[:, None], 0.0)
            s = scale * Q @ K.t() + table[which, h]
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True) if S else torch.full((L, 1), -math.inf)
            p = torch.exp(s - torch.where(top.isinf(), torch.zeros_like(top), top))
            tot = p.sum(-1, keepdim=True)
            p = p / torch.where(tot == 0, torch.ones_like(tot), tot)
            o = p @ V
            # |ds| <= (products + sums over dh) sum |q k| + a few roundings of s itself; exp, the row's sum and the weighted sum follow
            es = (prod + (dh + 4) * U32) * scale * (Q.abs() @ K.abs().t()) + 6 * U32 * s.masked_fill(~see, 0.0).abs()
            T = (es * see).amax(-1, keepdim=True) if S else torch.zeros(L, 1, dtype=torch.float64)
            acc = (S / 4 + 64) * U32 + prod
            pv = p @ V.abs()
            out["o"][0][b, :, c] = o
            out["o"][1][b, :, c] = (2 * T + acc + (u if storage != torch.float32 else 0.0)) * pv + u * o.abs()
            low = 2.0 ** apart * (1 if storage == torch.float32 else 0)
            if S:
                out["o"][1][b, :, c] += torch.minimum(p, low * 2.0 ** -31 * p.amax(-1, keepdim=True)) @ V.abs()
            if g is None:
                continue
            dO = g[b, :, c]
            dP, D = dO @ V.t(), (dO * o).sum(-1, keepdim=True)
            ds = p * (dP - D)
            ep = (2 * T + 16 * U32) * p
            edP = (prod + (dh + 4) * U32) * (dO.abs() @ V.abs().t())
            eD = (dh + 4) * U32 * (dO * o).abs().sum(-1, keepdim=True) + (dO.abs() * out["o"][1][b, :, c]).sum(-1, keepdim=True)
            eds = ep * (dP - D).abs() + p * (edP + eD) + 4 * U32 * ds.abs()
            accq = (L * G / 4 + 64) * U32 + prod
            out["dq"][0][b, :, c] = scale * ds @ K
            size = ds.abs()
            fq, fk = (torch.minimum(size, low * 2.0 ** -34 * size.amax(d, keepdim=True)) for d in (-1, 0))
            out["dq"][1][b, :, c] = scale * (eds + acc * ds.abs() + fq) @ K.abs()
            out["dk"][0][b, :, ck] += scale * ds.t() @ Q
            out["dk"][1][b, :, ck] += scale * (eds + accq * ds.abs() + fk).t() @ Q.abs()
            out["dv"][0][b, :, ck] += p.t() @ dO
            out["dv"][1][b, :, ck] += (ep + accq * p + p.clamp(max=low * 2.0 ** -39)).t() @ dO.abs()
            # a bucket's sum: in fp32 over a tile's diagonal and a block's tiles, then over the blocks
            out["dtable"][0][:, h].index_add_(0, which.flatten(), ds.flatten())
            out["dtable"][1][:, h].index_add_(0, which.flatten(), (eds + ((L + S) / 4 + 64) * U32 * ds.abs()).flatten())
    return {n: tuple(w) for n, w in out.items()}


def norm_residual(x, h, post=None, gate=None, res_scale=1.0, pre=None, kind="layer", eps=1e-5, gx=None, gy=None):
    """fp64 values by autograd: {"x", "y", "dx", "dh", "dgate", "dpost0", "dpost1", "dpre0", "dpre1"}"""
    store = x.dtype
    leaf = {}

    def mk(name, t):
        leaf[name] = t.detach().double().cpu().requires_grad_()
        return leaf[name]
    E = x.shape[-1]
    X, Hh = mk("x", x), mk("h", h)

    def norm(v, w, name):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        y = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * mk(name + "0", w[0])
        return y + mk(name + "1", w[1]) if len(w) > 1 and w[1] is not None else y
    n = norm(Hh, post, "post") if post is not None else Hh
    if gate is not None:
        gt = mk("gate", gate).reshape(-1, E)
        n = (n.reshape(gt.shape[0], -1, E) * gt[:, None]).reshape(X.shape)
    xo = res_scale * X + n
    out = {"x": xo.detach()}
    loss = 0.0 if gx is None else (xo * gx.double().cpu()).sum()
    if pre is not None:
        stored = xo if store == torch.float32 else xo.detach().to(store).double()
        y = norm(stored, pre, "pre")
        out["y"] = y.detach()
        if gy is not None:
            loss = loss + (y * gy.double().cpu()).sum()
    if gx is not None or gy is not None:
        names = [a for a in leaf if gy is not None or not a.startswith("pre")]
        for a, d in zip(names, torch.autograd.grad(loss, [leaf[a] for a in names])):
            out["d" + a] = d
    return out
