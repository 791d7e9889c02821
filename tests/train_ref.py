"""The operators of atlas_amd.train_ops in 64 bits, by their formulas, each with a bound on how far a right kernel can be off.

A bound counts what the kernels' contract allows: u = finfo(dtype).eps / 2 for every value that is rounded to the tensors' dtype (results; the
probabilities, dS and dz that feed a second product; the saved pre-activation), and fp32 arithmetic of n terms as 2 (n + 8) 2^-24 of the sum
of the terms' magnitudes. `tiny` is half the smallest step of the dtype: what a value near zero may lose (fp16: 2^-25).
"""
import math

import torch

U32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]


def check(name, got, want, bound):
    """got (kernel) against want (64 bits), element by element"""
    assert tuple(got.shape) == tuple(want.shape), (name, got.shape, want.shape)
    got, want, bound = got.detach().double().cpu(), want.cpu(), bound.cpu()
    assert bool(torch.isfinite(got).all()), f"{name}: {int((~torch.isfinite(got)).sum())} values are not finite"
    if got.numel() == 0:
        return
    over = (got - want).abs() - bound
    at = int(over.argmax())
    assert float(over.max()) <= 0, (f"{name}: off by {float((got - want).abs().flatten()[at]):.3e} at {at} (of {got.numel()}), bound {float(bound.flatten()[at]):.3e}, "
                                    f"value {float(want.flatten()[at]):.3e}; {int((over > 0).sum())} values are over")


# ---- attention -----------------------------------------------------------------------------------------------------------
def attention(q, k, v, dout, q_off, k_off, scale, key_mask=None, keep=None, keep_scale=1.0):
    """-> {name: (value, bound)} of out, dq, dk, dv; offsets are lists"""
    dtype = q.dtype
    u, t = unit(dtype), tiny(dtype)
    q, k, v, do = (x.detach().double().cpu() for x in (q, k, v, dout))
    heads, kv, dim = q.shape[1], k.shape[1], q.shape[2]
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    e_out, e_dq, e_dk, e_dv = (torch.zeros_like(x) for x in (q, q, k, v))
    for b in range(len(q_off) - 1):
        qs, ks = slice(q_off[b], q_off[b + 1]), slice(k_off[b], k_off[b + 1])
        lq, lk = q_off[b + 1] - q_off[b], k_off[b + 1] - k_off[b]
        if lq <= 0 or lk <= 0:
            continue
        seen = torch.ones(lk, dtype=torch.bool) if key_mask is None else key_mask[ks].cpu().bool()
        if not bool(seen.any()):
            continue
        at = torch.nonzero(seen).flatten()
        for h in range(heads):
            g = h * kv // heads
            Q, K, V, D = q[qs, h], k[ks, g][at], v[ks, g][at], do[qs, h]
            S = scale * Q @ K.T
            dS_in = scale * 2 * (dim + 8) * U32 * (Q.abs() @ K.abs().T) + 8 * U32 * S.abs()          # error of an exponent
            P = torch.softmax(S, dim=1)
            rel = 2 * dS_in.amax(1, keepdim=True) + (lk + 16) * 2 * U32                              # relative error of a probability
            M = torch.full_like(P, 1.0)
            if keep is not None:
                M = torch.zeros_like(P)
                cols = at[at < keep.shape[2]]
                M[:, : len(cols)] = keep[qs, h].cpu()[:, cols].double() * keep_scale
            low = t * P.amax(1, keepdim=True)                                                        # probabilities are held relative to the row's largest
            O = (P * M) @ V
            eO = (P * M * (u + rel)) @ V.abs() + low * (M @ V.abs()) + u * O.abs() + t
            dP = D @ V.T
            edP = 2 * (dim + 8) * U32 * (D.abs() @ V.abs().T)
            delta = (D * O).sum(1, keepdim=True)
            edelta = (D.abs() * eO).sum(1, keepdim=True) + 2 * (dim + 8) * U32 * (D * O).abs().sum(1, keepdim=True)
            X = M * dP - delta
            dS = P * X
            edS = P * (rel * X.abs() + M * edP + edelta + 4 * U32 * ((M * dP).abs() + delta.abs()))
            edS = edS + u * (dS.abs() + edS) + t
            out[qs, h], e_out[qs, h] = O, eO
            dq[qs, h] = scale * dS @ K
            e_dq[qs, h] = scale * (edS @ K.abs() + 2 * (lk + 8) * U32 * (dS.abs() @ K.abs()))
            rows = torch.arange(ks.start, ks.stop)[at]
            dk[rows, g] += scale * dS.T @ Q
            e_dk[rows, g] += scale * (edS.T @ Q.abs() + 2 * (lq * heads // kv + 8) * U32 * (dS.abs().T @ Q.abs()))
            PM = P * M
            dv[rows, g] += PM.T @ D
            e_dv[rows, g] += (PM * (u + rel + 2 * (lq * heads // kv + 8) * U32) + t * M).T @ D.abs()
    r = {"out": (out, e_out)}
    for n, x, e in (("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv)):
        r[n] = (x, e + u * x.abs() + u * e + t)
    return r


# ---- 8-bit values ----------------------------------------------------------------------------------------------------------
def eight_bits(x, largest=torch.finfo(torch.float32).max):
    """the values that 8 bits hold of a 64-bit tensor, by arithmetic, none beyond the type's `largest`; values that are not finite: NaN"""
    n = x.shape[-1]
    bad = ~torch.isfinite(x)
    x = torch.nn.functional.pad(torch.where(bad, 0.0, x), (0, -n % 32)).unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    part, power = torch.frexp(most)                          # most = part 2^power, part in [0.5, 1)
    power = torch.where(most > 0, power - 9 + (part > 0.875), torch.full_like(power, -126)).clamp(-126, 120).double()
    own = (torch.frexp(x)[1] - 1).double()                   # a value's own power of two
    step = torch.exp2(torch.maximum(own - 3, power - 9))
    y = torch.round(x / step) * step
    y = torch.where(y.abs() > largest, y.sign() * 240 * torch.exp2(power), y).flatten(-2)[..., :n]
    return torch.where(bad, math.nan, y)


# ---- dense layer -----------------------------------------------------------------------------------------------------------
def _slope(z):
    return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def linear(x, w, b, dy, gelu=False, keep=None, keep_scale=1.0, residual=None, checkpoint=False, device="cpu"):
    """-> {name: (value, bound)} of y, dx, dw, db"""
    dtype = x.dtype
    u, t = unit(dtype), tiny(dtype)
    x, w, dy = (a.detach().double().to(device) for a in (x, w, dy))
    m, k = x.shape
    n = w.shape[0]
    fp32 = lambda terms: 2 * (terms + 8) * U32  # noqa: E731
    z = x @ w.T
    A = x.abs() @ w.abs().T
    if b is not None:
        bb = b.detach().double().to(device)
        z, A = z + bb, A + bb.abs()
    ez = fp32(k) * A
    M = torch.ones_like(z) if keep is None else keep.to(device).double() * keep_scale
    act, s = (z * torch.special.ndtr(z), _slope(z)) if gelu else (z, torch.ones_like(z))
    y = act * M
    ey = M * ((1.13 if gelu else 1.0) * ez + 16 * U32 * act.abs())          # |gelu'| <= 1.13
    if residual is not None:
        rr = residual.detach().double().to(device)
        y, ey = y + rr, ey + 2 * U32 * (act.abs() * M + rr.abs())
    ey = ey + u * (y.abs() + ey) + t
    es = torch.zeros_like(z)
    xs = x
    if gelu:                                                                # |gelu''| <= 0.8
        if checkpoint:
            zs = eight_bits(z)
            moved = [(eight_bits(z + d) - zs).abs() for d in (ez, -ez, ez * z.sign(), -ez * z.sign())]     # where a rounding can go the other way
            es = 0.8 * torch.stack(moved).amax(0) + 16 * U32
            s = _slope(zs)
        else:
            es = 0.8 * (ez + u * z.abs() + t) + 16 * U32
    if checkpoint:
        xs = eight_bits(x)
    g = dy * M
    dz = g * s
    edz = g.abs() * es + 4 * U32 * dz.abs()
    db, edb = dz.sum(0), edz.sum(0) + fp32(m) * dz.abs().sum(0)
    if gelu or keep is not None:
        edz = edz + u * (dz.abs() + edz) + t                                # dz is rounded for the products
    dx, edx = dz @ w, edz @ w.abs() + fp32(n) * (dz.abs() @ w.abs())
    dw, edw = dz.T @ xs, edz.T @ xs.abs() + fp32(m) * (dz.abs().T @ xs.abs())
    r = {"y": (y, ey)}
    for name, v, e in (("dx", dx, edx), ("dw", dw, edw), ("db", db, edb)):
        r[name] = (v, e + u * (v.abs() + e) + t)
    if b is None:
        del r["db"]
    return r


# ---- layer norm ------------------------------------------------------------------------------------------------------------
def layer_norm(x, w, b, dy, eps):
    dtype = x.dtype
    u, t = unit(dtype), tiny(dtype)
    x, w, b, dy = (a.detach().double().cpu() for a in (x, w, b, dy))
    m, n = x.shape
    f = 2 * (n + 16) * U32
    mu = x.mean(1, keepdim=True)
    q = x.square().mean(1, keepdim=True)
    r = 1 / torch.sqrt(q + eps)
    c = x - mu
    emu = f * x.abs().mean(1, keepdim=True)
    er = f * r                                               # q is a sum of squares: its relative error is that of the sum
    ec = emu + 2 * U32 * c.abs()
    xh = c * r
    exh = ec * r + c.abs() * er + 2 * U32 * xh.abs()
    y = w * xh + b
    ey = w.abs() * exh + 4 * U32 * (w * xh).abs() + 4 * U32 * b.abs()
    g = w * dy
    gm = g.mean(1, keepdim=True)
    gc = (g * c).mean(1, keepdim=True)
    egm = f * g.abs().mean(1, keepdim=True)
    egc = (g.abs() * ec).mean(1, keepdim=True) + f * (g * c).abs().mean(1, keepdim=True)
    dx = r * (g - gm) - x * r ** 3 * gc
    edx = er * (g - gm).abs() + r * (egm + 4 * U32 * (g.abs() + gm.abs())) + x.abs() * (r ** 3 * egc + 3 * r ** 2 * er * gc.abs() + 8 * U32 * r ** 3 * gc.abs())
    fm = 2 * (m + 16) * U32
    dw, edw = (dy * xh).sum(0), (dy.abs() * exh).sum(0) + fm * (dy * xh).abs().sum(0)
    db, edb = dy.sum(0), fm * dy.abs().sum(0)
    return {name: (v, e + u * (v.abs() + e) + t) for name, v, e in (("y", y, ey), ("dx", dx, edx), ("dw", dw, edw), ("db", db, edb))}
