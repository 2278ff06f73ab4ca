"""Plain 64-bit forms of the feed-forward operators, with bounds on how far a correctly rounded 32-bit computation may be off.

The bounds count roundings, with u = 2^-24 half a step of float32 and h half a step of the operands' type
(``torch.finfo(t).eps / 2``):

  a sum of n products in float32            (n + 2) u sum |products|      (products rounded or fused, any order)
  act(z), z off by e, in float32            1.13 e + 16 u |z|             (no slope is above 1.13; a few roundings of factors <= |z|)
  act'(z), z off by e                       0.85 e + 32 u (1 + |z|)       (no curvature is above 0.8)
  storing v in type t                       h |v| + half the smallest subnormal of t
"""
import math

import numpy as np
import torch

U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def stored(v, dtype):
    return half_step(dtype) * v.abs() + TINY[dtype]


def act(z, kind, clip=32.0):
    if kind == "none":
        return z.clone()
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "clip":
        return z.clamp(0, clip)
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def slope(z, kind, clip=32.0):
    if kind == "none":
        return torch.ones_like(z)
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "clip":
        return ((z > 0) & (z < clip)).to(z.dtype)
    if kind == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    a, b = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(a * (z + b * z ** 3))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * b * z * z)


def corners(z, off, kind, clip=32.0):
    """1 where a pre-activation off by ``off`` may be on the other side of a corner."""
    near = torch.zeros_like(z)
    if kind in ("relu", "clip"):
        near = near + (z.abs() <= off)
    if kind == "clip":
        near = near + ((z - clip).abs() <= off)
    return (near > 0).to(z.dtype)


def dense(rows, w, inputs):
    """[inputs, outputs] of a set of weights [outputs, slots] in canonical order (rows < 0: no connection)."""
    rows = torch.as_tensor(np.asarray(rows), device=w.device).long()
    keep = rows >= 0
    out = torch.arange(rows.shape[0], device=w.device)[:, None].expand_as(rows)[keep]
    W = torch.zeros(inputs, rows.shape[0], dtype=torch.float64, device=w.device)
    W.index_put_((rows[keep], out), w.double()[keep], accumulate=True)
    return W


class Forward:
    """y, the pre-activations z, and their bounds.  x, ws, bs: tensors of any float type, on one device."""

    def __init__(self, rows, inputs, x, ws, bs, kind, clip=32.0, out_dtype=None):
        self.rows, self.inputs, self.kind, self.clip, self.x, self.ws = rows, inputs, kind, clip, x, ws
        n = np.asarray(rows).shape[1]
        xd = x.double()
        self.z, self.dz = [], []
        for w, b in zip(ws, bs):
            bd = torch.zeros(len(rows), dtype=torch.float64, device=x.device) if b is None else b.double()
            self.z.append(xd @ dense(rows, w, inputs) + bd)
            self.dz.append((n + 3) * U * (xd.abs() @ dense(rows, w.double().abs(), inputs) + bd.abs()) + 2.0 ** -140)
        a = act(self.z[0], kind, clip)
        da = 1.13 * self.dz[0] + 16 * U * self.z[0].abs()
        if len(ws) == 2:
            self.y = a * self.z[1]
            dy = da * (self.z[1].abs() + self.dz[1]) + a.abs() * self.dz[1] + U * self.y.abs()
        else:
            self.y, dy = a, da
        t = out_dtype or x.dtype
        self.bound = dy * (1 + half_step(t)) + stored(self.y, t)


def backward(f, dy):
    """dx, dw, db with their bounds, for the operands of a Forward, d held in x's type on its way to dx."""
    t = f.x.dtype
    n = np.asarray(f.rows).shape[1]
    dyd = dy.double()
    off = [e + U * z.abs() for z, e in zip(f.z, f.dz)]
    s, ds = slope(f.z[0], f.kind, f.clip), 0.85 * off[0] + 32 * U * (1 + f.z[0].abs())
    if f.kind in ("none", "relu", "clip"):
        ds = corners(f.z[0], f.dz[0], f.kind, f.clip)
    if len(f.ws) == 1:
        d, dd = [dyd * s], [dyd.abs() * ds]
    else:
        a, da = act(f.z[0], f.kind, f.clip), 1.13 * off[0] + 16 * U * f.z[0].abs()
        d = [dyd * s * f.z[1], dyd * a]
        dd = [dyd.abs() * (ds * (f.z[1].abs() + off[1]) + s.abs() * off[1]), dyd.abs() * da]
    dd = [e * (1 + 4 * U) + 4 * U * v.abs() for v, e in zip(d, dd)]
    dd_stored = [e * (1 + half_step(t)) + stored(v, t) for v, e in zip(d, dd)]
    tokens, xd = dy.shape[0], f.x.double()
    rows = torch.as_tensor(np.asarray(f.rows), device=dy.device).long()
    fan = int((rows >= 0).sum()) and int(torch.bincount(rows[rows >= 0]).max())
    dx = torch.zeros(tokens, f.inputs, dtype=torch.float64, device=dy.device)
    dx_bound = torch.zeros_like(dx)
    dws, dbs = [], []
    for v, e, es, w in zip(d, dd, dd_stored, f.ws):
        W = dense(f.rows, w, f.inputs)
        A = dense(f.rows, w.double().abs(), f.inputs)
        dx += v @ W.t()
        dx_bound += es @ A.t() + (fan * len(f.ws) + 2) * U * ((v.abs() + es) @ A.t())
        at = rows.clamp(min=0)
        pick = lambda m: torch.gather(m.t(), 1, at) * (rows >= 0)  # noqa: E731
        dws.append((pick(xd.t() @ v), pick(xd.abs().t() @ e) + (tokens + 8) * U * pick(xd.abs().t() @ (v.abs() + e)) + 2.0 ** -140))
        dbs.append((v.sum(0), e.sum(0) + (tokens + 8) * U * (v.abs() + e).sum(0) + 2.0 ** -140))
    return (dx, dx_bound * (1 + half_step(t)) + stored(dx, t)), dws, dbs


def within(got, want, bound):
    """Whether every element is within its bound; the worst ratio for the message."""
    off = (got.double() - want).abs()
    worst = float((off / bound.clamp(min=1e-300)).max()) if off.numel() else 0.0
    return bool((off <= bound).all()), worst


# ---- microscaled 4-bit floats -------------------------------------------------------------

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mx4_reference(v):
    """(codes, scales, values) of a float matrix from the definition, numpy in 64 bits; non-finite blocks become NaN."""
    v = np.asarray(v, dtype=np.float64)
    rows, cols = v.shape
    blocks = (cols + 31) // 32
    p = np.zeros((rows, blocks * 32))
    p[:, :cols] = v
    p = p.reshape(rows, blocks, 32)
    with np.errstate(all="ignore"):
        top = np.abs(p).max(axis=2)
        finite = np.isfinite(top)
        e = np.where(finite & (top > 0), np.frexp(np.where(finite, top, 1.0))[1] - 3, -127)
        e = np.clip(e, -127, 127)
        a = np.abs(np.where(finite[:, :, None], p, 0.0)) * np.exp2(-e.astype(np.float64))[:, :, None]
    gap = np.abs(a[..., None] - E2M1)
    best = gap.min(axis=-1, keepdims=True)
    tie = gap == best                                     # one or two candidates; of two the even code
    even = tie & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), tie.argmax(-1))
    code = code + 8 * (np.signbit(p) & finite[:, :, None])
    values = E2M1[code & 7] * np.where(code >= 8, -1.0, 1.0) * np.exp2(e.astype(np.float64))[:, :, None]
    values = np.where(finite[:, :, None], values, np.nan).reshape(rows, -1)[:, :cols]
    code = code.reshape(rows, blocks, 16, 2)
    return (code[..., 0] | (code[..., 1] << 4)).astype(np.uint8), np.where(finite, e + 127, 255).astype(np.uint8), values
