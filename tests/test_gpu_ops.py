"""Dense-block operators (onto_vae_amd.ops) on the GPU against oracle/ops_oracle.py in float64.

Tolerances, u = 2^-24 (half a step of float32), h = half a step of the output type, relative to the value or, below the
smallest normal number `tiny` where the steps stop shrinking (float16 subnormals: steps of tiny * eps), to `tiny`:
  8-bit operands: equal.  Products: the integer sum is exact, its conversion, two products by scales and the bias are four
    float32 roundings of at most |t| + |b|: (|t| + |b|) 5 u, then one rounding to the output: h |y|.
  Group norm: a mean of n values by 64-fold unrolled threads and trees has at most 64 + 30 additions on a path: 94 u max|x|, and so
    has the second moment; v = (x - mu) r gamma + beta then carries K = 2 * 94 + 8 roundings, each of a magnitude of at most
    A = (max|x - mu| + |mu|) r |gamma| + |beta|.  Activations have slopes within 1.13; silu / gelu themselves add (|v| + 8) u
    of exp / erf.  dx: the same count on E = r (|e| + mean|e| + |xhat| mean|e xhat|), plus the error of v through act'' (<= 1).
    dweight, dbias: at most rows / 64 + 200 additions in a path are NOT assumed: the bound is
    (sqrt(rows) + 200) u times the sum of magnitudes, plus v's error through act''.
  Dropout: one rounding of the factor, one of the product, one to the output; zeros and NaN exactly where they belong."""
import numpy as np
import pytest
import torch

import ops_oracle as oo
from onto_vae_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(t):
    return torch.finfo(t).eps / 2


def last(t, want):
    """The rounding to the output type: half a step of the value, of `tiny` among the subnormals."""
    return half(t) * np.maximum(np.abs(want), torch.finfo(t).tiny)


def f64(t):
    return t.detach().double().cpu().numpy()


def rnd(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    rng = np.random.default_rng(seed)
    return torch.as_tensor(rng.standard_normal(shape) * scale + shift).to(dtype).to(DEV)


def close(got, want, tol):
    got = f64(got)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], np.broadcast_to(tol, want.shape)[bad][:4])


# ---------------------------------------------------------------- quantiser
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 20000), (3, 7), (2, 64), (5, 1000), (130, 360), (300, 5893), (2, 40001), (1, 131071), (2000, 40)])
def test_quantize_rows(M, K, dtype):
    x = rnd(M * 7 + K, M, K, dtype=DT[dtype])
    q, s = ops.quantize_rows(x)
    qr, sr = oo.quantize_rows(f64(x))
    assert q.shape == (M, K) and s.shape == (M,)
    np.testing.assert_array_equal(s.cpu().numpy(), sr)
    np.testing.assert_array_equal(q.cpu().numpy(), qr)
    pad = torch.as_strided(q, (M, q.stride(0)), (q.stride(0), 1))[:, K:]
    assert q.stride(0) % 64 == 0 and not pad.any()


@pytest.mark.parametrize("dtype", DT)
def test_quantize_rows_borders(dtype):
    """Exact ties, quotients one step beside a border, zero, tiny, huge and non-finite rows."""
    t = DT[dtype]
    K = 300
    base = torch.arange(K, dtype=torch.float64) % 255 - 127
    rows = [base + 0.5, base * 0.5, base * 1.0, torch.zeros(K).double(), base * torch.finfo(t).tiny * 0.25, base * (torch.finfo(t).max / 254),
            torch.where(torch.arange(K) == 7, float("inf"), 1.0).double(), torch.where(torch.arange(K) == 299, float("nan"), 1.0).double(),
            torch.where(torch.arange(K) == 0, -float("inf"), 1.0).double(), base / 3, torch.nextafter(base.float() + 0.5, torch.zeros(K)).double()]
    x = torch.stack(rows).to(t).to(DEV)
    q, s = ops.quantize_rows(x)
    qr, sr = oo.quantize_rows(f64(x))
    np.testing.assert_array_equal(s.cpu().numpy(), sr)
    np.testing.assert_array_equal(q.cpu().numpy(), qr)


def test_quantize_rows_gather_strides_and_shapes():
    x = rnd(1, 50, 96)
    rows = torch.tensor([3, 49, 3, 0, 50, -1], device=DEV)
    for dt in (torch.int32, torch.int64):
        q, s = ops.quantize_rows(x, rows.to(dt))
        qr, sr = oo.quantize_rows(f64(x)[[3, 49, 3, 0]])
        np.testing.assert_array_equal(q.cpu().numpy()[:4], qr)
        np.testing.assert_array_equal(s.cpu().numpy()[:4], sr)
        assert torch.isnan(s[4:]).all() and not q[4:].any()
    q, s = ops.quantize_rows(x, torch.tensor([2 ** 32 + 3], device=DEV))
    assert torch.isnan(s).all()
    for v in (x[:, 1:38], x[::2, 3:], x.t(), x.view(5, 10, 96), x[0], x[:, :0], x[:0], x[:1].expand(4, 96)):
        q, s = ops.quantize_rows(v)
        assert q.shape == v.shape and s.shape == v.shape[:-1]
        qr, sr = oo.quantize_rows(f64(v).reshape(-1, v.shape[-1]) if v.numel() else np.zeros((s.numel(), v.shape[-1])))
        np.testing.assert_array_equal(q.cpu().numpy().reshape(qr.shape), qr)
        np.testing.assert_array_equal(s.cpu().numpy().reshape(-1), sr)


# ---------------------------------------------------------------- 8-bit product
def _check_product(a, sa, b, sb, bias, dtype):
    y = ops.int8_matmul(a, sa, b, sb, bias, dtype)
    t = oo.int8_matmul(a.cpu().numpy(), f64(sa), b.cpu().numpy(), f64(sb))
    bb = np.zeros(b.shape[0]) if bias is None else f64(bias)
    want = t + bb
    close(y, want, (np.abs(t) + np.abs(bb)) * 5 * U + last(dtype, want))


def _int8(seed, *shape):
    return torch.as_tensor(np.random.default_rng(seed).integers(-128, 128, shape, dtype=np.int8)).to(DEV)


SHAPES = [(1, 1, 1), (1, 360, 20000), (2, 3, 5), (7, 229, 5893), (16, 16, 64), (17, 33, 63), (32, 128, 512), (33, 129, 257), (64, 1, 1000),
          (100, 360, 4096), (128, 360, 20000), (129, 257, 385), (256, 256, 64), (257, 255, 128), (300, 1000, 96), (513, 260, 1024), (1, 8192, 64),
          (8192, 16, 100), (640, 700, 2048), (5, 7, 0), (3, 4, 131071)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_int8_matmul(M, N, K):
    a, b = _int8(M + K, M, K), _int8(N + K + 1, N, K)
    sa, sb = rnd(1, M).abs() + 0.1, rnd(2, N).abs() + 0.1
    for dtype, bias in ((torch.float32, None), (torch.bfloat16, rnd(3, N) * 10), (torch.float16, rnd(3, N))):
        _check_product(a, sa * (1e-3 if dtype == torch.float16 else 1.0) * (1e-3 if K > 1e4 else 1.0), b, sb, bias, dtype)


@pytest.mark.parametrize("M,N,K", [(1, 40, 333), (20, 130, 1111), (200, 300, 640)])
def test_int8_matmul_layouts(M, N, K):
    """Padded rows with junk behind K, odd row strides, odd first bytes, leading dimensions."""
    for ldx, off in ((K, 0), (K + 1, 1), ((K + 63) // 64 * 64 + 64, 0), ((K + 15) // 16 * 16 + 16, 16), (K + 5, 3)):
        ab, bb = _int8(5, M * ldx + 64), _int8(6, N * ldx + 64)
        a = torch.as_strided(ab, (M, K), (ldx, 1), off)
        b = torch.as_strided(bb, (N, K), (ldx, 1), off)
        _check_product(a, rnd(1, M), b, rnd(2, N), None, torch.float32)
    a = _int8(9, 2, 3, K)
    y = ops.int8_matmul(a, rnd(1, 2, 3), _int8(8, N, K), rnd(2, N))
    assert y.shape == (2, 3, N)


def test_int8_extremes_are_exact():
    """The largest sums: K = 131071 products of -128 * -128, and of 127 * -127."""
    K = 131071
    for va, vb in ((-128, -128), (127, -127)):
        a = torch.full((3, K), va, dtype=torch.int8, device=DEV)
        b = torch.full((2, K), vb, dtype=torch.int8, device=DEV)
        one = torch.ones(3, device=DEV)
        y = ops.int8_matmul(a, one, b, one[:2])
        assert (y == float(np.float32(va * vb * K))).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,K,N", [(1, 360, 720), (130, 1000, 129), (40, 5893, 229), (9, 20000, 360), (1, 20000, 360), (2, 5893, 700), (3, 333, 41),
                                   (4, 20000, 9), (2, 32768, 5), (1, 32769, 5), (4, 1, 600), (3, 17, 2000), (5, 64, 3)])
def test_int8_linear(M, K, N, dtype):
    t = DT[dtype]
    x, w, bias = rnd(1, M, K, dtype=t), rnd(2, N, K, scale=K ** -0.5), rnd(3, N)
    qw, sw = ops.quantize_rows(w)
    y = ops.int8_linear(x, qw, sw, bias)
    assert y.dtype == t
    qx, sx = oo.quantize_rows(f64(x))
    tt = oo.int8_matmul(qx, sx, *oo.quantize_rows(f64(w)))
    want = tt + f64(bias)
    close(y, want, (np.abs(tt) + np.abs(f64(bias))) * 5 * U + last(t, want))
    # and it is the layer: each 8-bit operand is off by at most half a step of its scale
    full = f64(x) @ f64(w).T + f64(bias)
    bound = (np.abs(f64(x)).sum(1)[:, None] * f64(sw)[None] / 2 + np.abs(f64(w)).sum(1)[None] * sx.astype(np.float64)[:, None] / 2 +
             K * sx.astype(np.float64)[:, None] * f64(sw)[None] / 4)
    assert (np.abs(want - full) <= bound).all()
    assert torch.equal(y, ops.int8_matmul(*ops.quantize_rows(x), qw, sw, bias, dtype=t))      # the fused form of few rows, bit for bit
    idx = torch.tensor([M - 1, 0, -1, M], device=DEV)
    yr = ops.int8_linear(x, qw, sw, bias, rows=idx)
    assert torch.equal(yr[:2], y[[M - 1, 0]]) and torch.isnan(yr[2:]).all()
    x[0, K // 2] = float("nan")
    y = ops.int8_linear(x, qw, sw, bias, dtype=torch.float32)
    assert torch.isnan(y[0]).all() and torch.isfinite(y[1:]).all() and y.dtype == torch.float32


# ---------------------------------------------------------------- group norm
GN_CASES = [   # N, S, C, groups
    (1, 1, 360, 8), (1, 1, 8, 1), (3, 1, 8, 8), (5, 1, 1000, 8), (130, 1, 1000, 40), (70, 1, 96, 1), (33, 1, 130, 13), (2, 1, 5893, 1),
    (9, 1, 5000, 5), (2, 1, 20000, 1), (3, 1, 40000, 2), (1, 1, 70001, 1), (700, 1, 64, 32),
    (2, 2, 8, 2), (3, 5, 30, 3), (2, 49, 320, 32), (1, 64, 128, 8), (4, 100, 77, 7), (2, 1024, 320, 32), (3, 1000, 96, 1), (1, 4096, 512, 32),
    (2, 4097, 24, 4), (1, 20000, 16, 2), (1, 1, 3, 3), (1, 2, 3, 1), (2, 1, 2, 2), (40, 1, 9000, 1), (3, 1, 16384, 1), (2, 1, 16385, 1), (17, 1, 4100, 2), (2, 3, 5000, 2), (700, 40, 24, 3),
    (2, 333, 1000, 8), (1, 7, 5893, 1), (64, 16, 320, 32), (1, 70000, 3, 3), (300, 3, 40, 4)]


def _gn_tol(o, x, t):
    """(tolerance of v, of y) in the module docstring's terms."""
    K = 2 * 94 + 8
    xa = np.abs(f64(x))
    N, S, C = x.shape
    G = o["mean"].shape[1]
    big = (xa.reshape(N, S, G, C // G).max((1, 3)) + np.abs(o["mean"])) * o["rstd"]
    big = np.repeat(big, C // G, 1)[:, None, :]
    tv = K * U * (big * np.abs(o["w"]) + np.abs(o["v"])) * np.maximum(1, np.abs(o["xhat"]))
    return tv, o["f"] * (1.13 * tv + (np.abs(o["v"]) + 8) * U * np.abs(o["v"])) + last(t, o["y"])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("i", range(len(GN_CASES)), ids=["x".join(map(str, c)) for c in GN_CASES])
def test_group_norm_act(i, dtype):
    N, S, C, G = GN_CASES[i]
    t = DT[dtype]
    act = ("none", "relu", "silu", "gelu")[i % 4]
    drop = (0.0, 0.3, 0.0)[i % 3]
    x, dy = rnd(i, N, S, C, dtype=t, shift=0.5), rnd(i + 100, N, S, C, dtype=t)
    wt = t if i % 2 else torch.float32
    w, b = rnd(i + 200, C, dtype=wt, scale=0.2, shift=1.0), rnd(i + 300, C, dtype=wt)
    kw = dict(act=act, drop=drop, seed=11 + i, offset=5 + 2 ** 33 * (i % 2))
    y, mean, rstd = ops.group_norm_act(x, G, w, b, **kw)
    kn = dict(kw, name=act)
    del kn["act"]
    o = oo.group_norm_act(f64(x), G, f64(w), f64(b), dy=f64(dy), **kn)
    tv, ty = _gn_tol(o, x, t)
    amax = np.abs(f64(x)).max((1, 2))[:, None] + 1e-30
    close(mean, o["mean"], 94 * U * amax)
    close(rstd, o["rstd"], 200 * U * o["rstd"] * np.maximum(1, (amax * o["rstd"]) ** 2))
    close(y, o["y"], ty)
    # relu's gradient jumps where v is 0: those elements are left out of dy (kept at 0) so that every sum has one right value
    if act == "relu":
        near = np.abs(o["v"]) <= 2 * tv
        dy = dy.masked_fill(torch.as_tensor(near).to(DEV), 0.0)
        o = oo.group_norm_act(f64(x), G, f64(w), f64(b), dy=f64(dy), **kn)
    dx, dw, db = ops.group_norm_act_backward(dy, x, mean, rstd, G, w, b, **kw)
    eg = np.abs(o["dv"] * o["w"]).reshape(N, S, G, C // G)
    xg = np.abs(o["xhat"]).reshape(N, S, G, C // G)
    r = o["rstd"][:, None, :, None]
    E = r * (eg + eg.mean((1, 3), keepdims=True) + xg * (eg * xg).mean((1, 3), keepdims=True))
    curv = 0.0 if act in ("none", "relu") else 1.0
    tdv = curv * o["f"] * tv * np.abs(f64(dy))
    tg = (tdv * np.abs(o["w"])).reshape(N, S, G, C // G)
    tve = tv.reshape(N, S, G, C // G) / np.maximum(1e-3, np.abs(o["w"]).reshape(1, 1, G, C // G))
    T = (400 * U * E + r * (tg + tg.mean((1, 3), keepdims=True) + xg * (tg * xg + eg * tve).mean((1, 3), keepdims=True) +
                            tve * (eg * xg).mean((1, 3), keepdims=True))).reshape(N, S, C)
    close(dx, o["dx"], T + last(t, o["dx"]))
    n = np.sqrt(N * S) + 200
    tx = tv / np.maximum(1e-3, np.abs(o["w"]))
    close(dw, o["dweight"], n * U * o["dweight_abs"] + (tdv * np.abs(o["xhat"]) + np.abs(o["dv"]) * tx).sum((0, 1)) + 1e-30)
    close(db, o["dbias"], n * U * o["dbias_abs"] + tdv.sum((0, 1)) + 1e-30)


def test_group_norm_large_mean_keeps_its_digits():
    """Mean 1000 times the spread: the second moment is taken about the mean."""
    for N, S, C, G in ((4, 1, 1000, 8), (2, 64, 64, 4), (2, 4096, 64, 4), (1, 30000, 8, 1)):
        x = rnd(1, N, S, C, shift=1000.0)
        y, mean, rstd = ops.group_norm_act(x, G)
        o = oo.group_norm_act(f64(x), G)
        # the mean is off by at most 94 u 1000 and with it every xhat
        close(y, o["y"], 94 * U * 1010 * 1.2 + 200 * U * np.abs(o["y"]))
        close(rstd, o["rstd"], 300 * U * o["rstd"] + (94 * U * 1010) ** 2)


@pytest.mark.parametrize("N,S,C,G", [(4, 1, 96, 4), (2, 64, 96, 4), (1, 8192, 96, 4)])
def test_group_norm_special_values(N, S, C, G):
    """A constant group (rstd = 1 / sqrt(eps), dx finite), a NaN or an infinity stays in its own sample and group."""
    x = rnd(5, N, S, C)
    x[0, :, :C // G] = 3.0
    x[-1, 0, C - 1] = float("nan")
    y, mean, rstd = ops.group_norm_act(x, G, act="silu")
    assert torch.isnan(y[-1, :, C - C // G:]).all()
    ok = torch.ones_like(x, dtype=torch.bool)
    ok[-1, :, C - C // G:] = False
    assert torch.isfinite(y[ok]).all()
    assert (y[0, :, :C // G] == 0).all() and abs(float(rstd[0, 0]) - 1e-5 ** -0.5) < 1e-3
    dy = rnd(6, N, S, C)
    dx, _, _ = ops.group_norm_act_backward(dy, x, mean, rstd, G, act="silu")
    assert torch.isfinite(dx[ok]).all() and torch.isnan(dx[-1, :, C - C // G:]).all()
    x[-1, 0, C - 1] = float("inf")
    assert torch.isfinite(ops.group_norm_act(x, G)[0][ok]).all()


def test_group_norm_shapes_optional_parameters_and_empty():
    x = rnd(1, 2, 4, 6, 32)
    y, mean, rstd = ops.group_norm_act(x, 4)
    close(y.view(2, 24, 32), oo.group_norm_act(f64(x).reshape(2, 24, 32), 4)["y"], 1e-4)
    dx, dw, db = ops.group_norm_act_backward(x, x, mean, rstd, 4)
    assert dx.shape == x.shape and dw is None and db is None
    w = rnd(2, 32)
    _, dw, db = ops.group_norm_act_backward(x, x, mean, rstd, 4, weight=w)
    assert dw.shape == (32,) and db is None
    _, dw, db = ops.group_norm_act_backward(x, x, mean, rstd, 4, bias=w)
    assert dw is None and db.shape == (32,)
    # channels last in memory, seen as [N, C, H, W]
    m = rnd(3, 2, 32, 5, 5).to(memory_format=torch.channels_last)
    assert m.permute(0, 2, 3, 1).is_contiguous()
    y = ops.group_norm_act(m.permute(0, 2, 3, 1), 8)[0].permute(0, 3, 1, 2)
    torch.testing.assert_close(y, torch.nn.functional.group_norm(m, 8), rtol=1e-4, atol=1e-5)
    for shape in ((0, 5, 32), (3, 0, 32)):
        e = torch.empty(shape, device=DEV)
        y, mean, rstd = ops.group_norm_act(e, 4, w, w)
        assert y.shape == shape and mean.shape == (shape[0], 4)
        dx, dw, db = ops.group_norm_act_backward(e, e, mean, rstd, 4, w, w)
        assert dx.shape == shape and not dw.any() and not db.any()
    # a view with other strides gives what its copy gives
    big = rnd(4, 6, 40)
    assert torch.equal(ops.group_norm_act(big[::2, 4:36], 4)[0], ops.group_norm_act(big[::2, 4:36].contiguous(), 4)[0])


def test_group_norm_is_deterministic():
    for N, S, C, G in ((300, 1, 1000, 8), (8, 1024, 320, 32), (1, 16384, 64, 8)):
        x, dy, w = rnd(1, N, S, C), rnd(2, N, S, C), rnd(3, C)
        runs = []
        for _ in range(3):
            y, mean, rstd = ops.group_norm_act(x, G, w, w, act="gelu", drop=0.1, seed=3, offset=4)
            runs.append((y, mean, rstd, *ops.group_norm_act_backward(dy, x, mean, rstd, G, w, w, act="gelu", drop=0.1, seed=3, offset=4)))
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


# ---------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("R,C", [(1, 1), (1, 8), (3, 7), (128, 360), (37, 5893), (5, 20000), (1000, 9), (2, 16), (64, 24)])
def test_dropout(R, C, dtype):
    t = DT[dtype]
    x = rnd(R + C, R, C, dtype=t)
    for p, seed, offset in ((0.5, 1, 0), (0.1, 2 ** 63 + 5, 2 ** 40 + 3), (0.0, 3, 3), (1.0, 3, 3), (2.0 ** -18, 3, 3)):
        y = ops.dropout(x, p, seed, offset)
        keep, f = oo.keep_mask(R, C, p, seed, offset)
        want = np.where(keep, f64(x) * f, 0.0)
        close(y, want, np.abs(want) * 3 * U + last(t, want))
        assert ((y == 0).cpu().numpy() == (~keep | (f64(x) == 0))).all()
        assert torch.equal(ops.dropout_backward(x, p, seed, offset), y)


def test_dropout_rows_strides_and_special_values():
    x = rnd(1, 40, 100)
    rows = torch.tensor([39, 0, 5, 5, 40, -3], device=DEV)
    y = ops.dropout(x, 0.25, 9, 2, rows=rows)
    want = oo.dropout(f64(x)[[39, 0, 5, 5]], 0.25, 9, 2)
    close(y[:4], want, np.abs(want) * 4 * U)
    assert torch.isnan(y[4:]).all()                    # a row index outside the matrix
    for v in (x[:, 3:77], x[1::3], x.t(), x.view(4, 10, 100), x[:0], x[:, :0], x[0]):
        y = ops.dropout(v, 0.5, 4)
        assert y.shape == v.shape and y.is_contiguous()
        if v.numel():
            want = oo.dropout(f64(v).reshape(-1, v.shape[-1]), 0.5, 4, 0)
            close(y.reshape(want.shape), want, np.abs(want) * 4 * U)
    x.fill_(float("inf"))
    x[::2] = float("nan")
    y = ops.dropout(x, 0.5, 7)
    keep = torch.as_tensor(oo.keep_mask(40, 100, 0.5, 7, 0)[0]).to(DEV)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()


def test_dropout_mask_is_group_norms_mask():
    x = rnd(1, 6, 7, 44)
    y, _, _ = ops.group_norm_act(x, 4, drop=0.4, seed=8, offset=3)
    one = ops.dropout(torch.ones_like(x), 0.4, 8, 3)
    assert torch.equal(y == 0, one == 0)


def test_dropout_rate():
    y = ops.dropout(torch.ones(1000, 4000, device=DEV), 0.3, 123)
    n = y.numel()
    assert abs(float((y == 0).sum()) / n - 0.3) < 5 * (0.21 / n) ** 0.5
    assert abs(float(y.double().mean()) - 1.0) < 5 * (0.3 / 0.7 / n) ** 0.5


# ---------------------------------------------------------------- as they are used together
def _block(x, qw, sw, bias, w, b, off):
    h = ops.int8_linear(ops.dropout(x, 0.1, 5, off), qw, sw, bias)
    a, mean, rstd = ops.group_norm_act(h, 8, w, b, act="silu", drop=0.2, seed=5, offset=off + 1)
    return a, h, mean, rstd


@pytest.mark.parametrize("dtype", DT)
def test_a_dense_block(dtype):
    """dropout -> 8-bit linear -> group norm, activation, dropout -> 8-bit linear, and the block's backward down to the linear."""
    t = DT[dtype]
    x, W, bias = rnd(1, 70, 333, dtype=t), rnd(2, 96, 333, scale=0.1), rnd(3, 96)
    w, b, W2 = rnd(4, 96, shift=1.0), rnd(5, 96), rnd(6, 50, 96, scale=0.1)
    qw, sw = ops.quantize_rows(W)
    qw2, sw2 = ops.quantize_rows(W2)
    a, h, mean, rstd = _block(x, qw, sw, bias, w, b, 100)
    y = ops.int8_linear(a, qw2, sw2)
    dh, dw, db = ops.group_norm_act_backward(a, h, mean, rstd, 8, w, b, act="silu", drop=0.2, seed=5, offset=101)
    xd = oo.dropout(f64(x), 0.1, 5, 100)
    hd = oo.int8_matmul(*oo.quantize_rows(f64(torch.as_tensor(xd).to(t))), *oo.quantize_rows(f64(W)), f64(bias))
    close(h, hd, 2 * last(t, hd) + 40 * U * 30)
    o = oo.group_norm_act(f64(h)[:, None], 8, f64(w), f64(b), name="silu", drop=0.2, seed=5, offset=101, dy=f64(a)[:, None])
    close(a[:, None], o["y"], _gn_tol(o, h[:, None], t)[1])
    want = oo.int8_matmul(*oo.quantize_rows(f64(a)), *oo.quantize_rows(f64(W2)))
    close(y, want, 5 * U * np.abs(want) + last(t, want))
    assert dh.shape == h.shape and torch.isfinite(dh.float()).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()


def test_streams_and_graph_replays():
    """The block on a side stream, two interleaved streams, and captured: every replay equals the eager result on new inputs."""
    x, W, bias = rnd(1, 130, 5893), rnd(2, 360, 5893, scale=0.02), rnd(3, 360)
    w, b = rnd(4, 360, shift=1.0), rnd(5, 360)
    qw, sw = ops.quantize_rows(W)
    want = _block(x, qw, sw, bias, w, b, 7)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(_block(x, qw, sw, bias, w, b, 7))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))
    m = rnd(6, 2, 4096, 64)
    graphs = []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        xs = x.clone()
        with torch.cuda.graph(g):
            a, h, mean, rstd = _block(xs, qw, sw, bias, w, b, 7)
            dh, dw, db = ops.group_norm_act_backward(a, h, mean, rstd, 8, w, b, act="silu", drop=0.2, seed=5, offset=8)
            ym, mm, rm = ops.group_norm_act(m, 8, act="silu")
            dm = ops.group_norm_act_backward(ym, m, mm, rm, 8, act="silu")[0]
        graphs.append((g, xs, (a, h, mean, rstd, dh, dw, db, ym, dm)))
    for rep in range(4):
        fresh = rnd(50 + rep, 130, 5893)
        a, h, mean, rstd = _block(fresh, qw, sw, bias, w, b, 7)
        ym, mm, rm = ops.group_norm_act(m, 8, act="silu")
        want = (a, h, mean, rstd, *ops.group_norm_act_backward(a, h, mean, rstd, 8, w, b, act="silu", drop=0.2, seed=5, offset=8), ym,
                ops.group_norm_act_backward(ym, m, mm, rm, 8, act="silu")[0])
        for g, xs, outs in graphs:
            xs.copy_(fresh)
            g.replay()
        torch.cuda.synchronize()
        for g, xs, outs in graphs:
            assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_refusals():
    x = rnd(1, 4, 16)
    q, s = ops.quantize_rows(x)
    for bad in (lambda: ops.quantize_rows(x.double()), lambda: ops.quantize_rows(x, rows=torch.tensor([0.5], device=DEV)),
                lambda: ops.quantize_rows(x, rows=torch.tensor([0])), lambda: ops.quantize_rows(x.view(2, 2, 16), rows=torch.tensor([0], device=DEV)),
                lambda: ops.quantize_rows(x.sum()), lambda: ops.int8_matmul(x, s, q, s), lambda: ops.int8_matmul(q, s, q[:, :8], s),
                lambda: ops.int8_matmul(q, s[:2], q, s), lambda: ops.int8_matmul(q, s, q, s[:2]), lambda: ops.int8_matmul(q, s, q, s, bias=s[:1]),
                lambda: ops.int8_matmul(q, s.half(), q, s), lambda: ops.int8_matmul(q, s, q, s, dtype=torch.float64),
                lambda: ops.int8_matmul(q, s, q.cpu(), s), lambda: ops.int8_linear(x, q, s[:1]), lambda: ops.int8_linear(x, x, s),
                lambda: ops.int8_linear(x[:, :8], q, s), lambda: ops.int8_linear(x, q, s, bias=s[:2]), lambda: ops.int8_linear(x, q, s, dtype=torch.int8),
                lambda: ops.int8_linear(x.double(), q, s), lambda: ops.int8_linear(x.view(2, 2, 16), q, s, rows=torch.tensor([0], device=DEV)), lambda: ops.group_norm_act(x, 3), lambda: ops.group_norm_act(x, 0),
                lambda: ops.group_norm_act(x[0], 4), lambda: ops.group_norm_act(x, 4, act="tanh"), lambda: ops.group_norm_act(x, 4, drop=1.5),
                lambda: ops.group_norm_act(x, 4, drop=float("nan")), lambda: ops.group_norm_act(x, 4, eps=-1.0), lambda: ops.group_norm_act(x, 4, seed=-1),
                lambda: ops.group_norm_act(x, 4, weight=x[0, :8]), lambda: ops.group_norm_act(x, 4, weight=x[0].double()),
                lambda: ops.group_norm_act(x.half(), 4, weight=x[0], bias=x[0].half()), lambda: ops.group_norm_act(x.long(), 4),
                lambda: ops.group_norm_act_backward(x[:2], x, s, s, 4), lambda: ops.group_norm_act_backward(x, x, s, s, 4),
                lambda: ops.dropout(x, -0.1, 1), lambda: ops.dropout(x, 0.5, 2 ** 64), lambda: ops.dropout(x, 0.5, 1, -1),
                lambda: ops.dropout(x.int(), 0.5, 1)):
        with pytest.raises(ValueError):
            bad()
