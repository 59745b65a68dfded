"""float64 restatement of the dense-block operators of onto_vae_amd.ops.  TEST INFRASTRUCTURE ONLY.

The reference has no counterpart (its blocks are torch's Linear, BatchNorm1d, Dropout, ReLU: onto_vae/modules.py:43-64); the
formulas are those of include/ontovae_hip.h.  numpy on the host, Philox from philox_oracle (pinned by Random123's vectors).
"""
import math

import numpy as np

from philox_oracle import philox4x32_10

STREAM_OP = 6


def quantize_rows(x):
    """(q int8, scale float32, both of [M, K] float64 input holding the element type's values)."""
    x = np.asarray(x, np.float64)
    M, K = x.shape
    amax = np.abs(x).max(1) if K else np.zeros(M)
    bad = ~np.isfinite(x).all(1)
    with np.errstate(all="ignore"):
        s = (amax.astype(np.float32) * (np.float32(1) / np.float32(127))).astype(np.float32)
        q = np.rint(x / s.astype(np.float64)[:, None])
    q = np.where(np.isfinite(q) & ~bad[:, None] & (s > 0)[:, None], q, 0)
    s[bad] = np.nan
    return np.clip(q, -127, 127).astype(np.int8), s


def int8_matmul(a, sa, b, sb, bias=None):
    acc = a.astype(np.float64) @ b.astype(np.float64).T
    y = acc * np.asarray(sa, np.float64)[:, None] * np.asarray(sb, np.float64)[None, :]
    return y if bias is None else y + np.asarray(bias, np.float64)


def keep_mask(R, C, p, seed, offset):
    """(keep [R, C] bool, factor of the kept elements)."""
    nb = -(-C // 8)
    t = int(np.rint(float(np.float32(p)) * 65536))
    i = np.arange(R * nb, dtype=np.uint64)
    c = philox4x32_10((i & np.uint64(0xFFFFFFFF), (i >> np.uint64(32)) ^ np.uint64(STREAM_OP << 24), np.uint64(offset & 0xFFFFFFFF),
                       np.uint64(offset >> 32)), (seed & 0xFFFFFFFF, seed >> 32))
    u = np.stack([h for w in c for h in (w & np.uint32(0xFFFF), w >> np.uint32(16))], 1).reshape(R, nb * 8)[:, :C]
    return u >= t, 65536.0 / (65536 - t) if t < 65536 else 0.0


def dropout(x, p, seed, offset):
    keep, f = keep_mask(*x.shape, p, seed, offset)
    return np.where(keep, np.asarray(x, np.float64) * f, 0.0)


_erf = np.vectorize(math.erf, otypes=[np.float64])


def act(v, name):
    if name == "relu":
        return np.maximum(v, 0)
    if name == "silu":
        return v / (1 + np.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + _erf(v / math.sqrt(2)))
    return v


def act_grad(v, name):
    if name == "relu":
        return (v > 0).astype(np.float64)
    if name == "silu":
        s = 1 / (1 + np.exp(-v))
        return s * (1 + v * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + _erf(v / math.sqrt(2))) + v * np.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    return np.ones_like(v)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, name="none", drop=0.0, seed=0, offset=0, dy=None):
    """x [N, S, C] float64.  dict of y, mean, rstd and, with dy, dx, dweight, dbias; also what a tolerance needs: xhat, v, and
    the magnitudes the sums run over (dweight_abs, dbias_abs)."""
    x = np.asarray(x, np.float64)
    N, S, C = x.shape
    cg = C // groups
    xg = x.reshape(N, S, groups, cg)
    mu = xg.mean((1, 3), keepdims=True)
    r = 1 / np.sqrt(((xg - mu) ** 2).mean((1, 3), keepdims=True) + eps)
    xhat = ((xg - mu) * r).reshape(N, S, C)
    w = np.ones(C) if weight is None else np.asarray(weight, np.float64)
    b = np.zeros(C) if bias is None else np.asarray(bias, np.float64)
    v = xhat * w + b
    keep, f = (np.ones((N, S, C), bool), 1.0)
    if drop > 0:
        keep, f = keep_mask(N * S, C, drop, seed, offset)
        keep = keep.reshape(N, S, C)
    out = dict(y=np.where(keep, act(v, name) * f, 0.0), mean=mu[:, 0, :, 0], rstd=r[:, 0, :, 0], xhat=xhat, v=v, w=w, f=f)
    if dy is not None:
        dv = np.where(keep, np.asarray(dy, np.float64) * act_grad(v, name) * f, 0.0)
        e = (dv * w).reshape(N, S, groups, cg)
        xh = xhat.reshape(N, S, groups, cg)
        dx = r * (e - e.mean((1, 3), keepdims=True) - xh * (e * xh).mean((1, 3), keepdims=True))
        out.update(dx=dx.reshape(N, S, C), dweight=(dv * xhat).sum((0, 1)), dbias=dv.sum((0, 1)),
                   dweight_abs=np.abs(dv * xhat).sum((0, 1)), dbias_abs=np.abs(dv).sum((0, 1)), dv=dv)
    return out
