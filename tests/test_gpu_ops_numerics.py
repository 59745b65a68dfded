"""Group norm on the GPU where digits are lost first: values far from 0 against their spread, long sums.  Against oracle/ops_oracle.py in
float64; u = 2^-24 (half a step of float32)."""
import numpy as np
import pytest
import torch

import ops_oracle as oo
from onto_vae_amd import ops
from test_gpu_ops import U, close, f64, last, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,S,C,G", [(4, 1, 96, 4), (3, 5, 30, 3), (2, 64, 96, 4), (1, 4097, 24, 4), (1, 16385, 64, 4), (2, 3, 5000, 2)])
def test_means_whose_square_passes_float32(N, S, C, G):
    """Values around 1e20, spread 1e16: every square about the mean and every sum of squares is a float32, the mean's own square is not.
    (16385 rows end in a tile of fewer rows than a workgroup takes at a time.)"""
    x = rnd(N + S + C, N, S, C, scale=1e16, shift=1e20)
    y, mean, rstd = ops.group_norm_act(x, G)
    o = oo.group_norm_act(f64(x), G)
    # a mean of n values is off by at most 94 u of the largest value, and with it xhat by that over the spread
    off = 94 * U * 1.001e20
    close(mean, o["mean"], off)
    close(y, o["y"], off * o["rstd"].max() + 200 * U * np.abs(o["y"]))
    dy = rnd(1, N, S, C)
    dx, _, _ = ops.group_norm_act_backward(dy, x, mean, rstd, G)
    assert torch.isfinite(dx).all()


FAR = [(4, 1, 1000, 8), (3, 1, 8200, 1), (2, 1, 16384, 1), (2, 1, 20000, 1), (70, 1, 96, 3), (2, 64, 64, 4), (3, 5, 30, 3), (1, 300, 24, 24), (2, 4096, 64, 4),
       (1, 30000, 8, 1), (1, 16385, 64, 4), (2, 3000, 320, 32), (2, 3, 5000, 2), (1, 40, 2500, 1)]


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("shift,dtype", [(1e3, torch.float32), (1e5, torch.float32), (100.0, torch.bfloat16), (100.0, torch.float16)])
@pytest.mark.parametrize("N,S,C,G", FAR)
def test_a_large_mean_costs_no_digits(N, S, C, G, shift, dtype, act):
    """Spread 1 around 1e3 and 1e5, where a float32 mean is off by up to 3e-5 and 4e-3 of the spread.  Every group has another mean, some
    groups are around 0, and a group's first value stands far from the rest.

    x - mean - rest: the difference of neighbouring float32s is exact or off by u of itself, the rest is a mean of differences of
    the spread's size, 94 additions on a path: 94 u (mean |xhat| <= 1).  The second moment has the same count, half of it in rstd:
    err_x = 100 u (1 + |xhat|) leaves room for the products.  The backward pass of a 16-bit x may use the saved mean as it is, nearest to
    the mean: u |mean| rstd more."""
    rng = np.random.default_rng(N + S + C)
    sh = np.repeat(shift * rng.uniform(0.5, 1.0, (N, 1, G)) * rng.choice([-1, 1, 1, 0], (N, 1, G)), C // G, 2)
    x = torch.as_tensor(rng.standard_normal((N, S, C)) + sh)
    x[:, 0, ::C // G] += 20.0
    x = x.to(dtype).to("cuda:0")
    dy, w, b = rnd(1, N, S, C, dtype=dtype), rnd(2, C, scale=0.2, shift=1.0), rnd(3, C)
    y, mean, rstd = ops.group_norm_act(x, G, w, b, act=act)
    o = oo.group_norm_act(f64(x), G, f64(w), f64(b), name=act, dy=f64(dy))
    xh = np.abs(o["xhat"])
    err = 100 * U * (1 + xh)
    close(mean, o["mean"], U * np.abs(o["mean"]) + 100 * U / o["rstd"])
    close(rstd, o["rstd"], 100 * U * o["rstd"])
    tv = err * np.abs(o["w"]) + 6 * U * (xh * np.abs(o["w"]) + np.abs(f64(b)))
    close(y, o["y"], 1.13 * tv + (np.abs(o["v"]) + 8) * U * np.abs(o["v"]) + last(dtype, o["y"]))
    if dtype != torch.float32:
        err = err + np.repeat(U * np.abs(o["mean"]) * o["rstd"], C // G, 1)[:, None]
        tv = tv + np.repeat(U * np.abs(o["mean"]) * o["rstd"], C // G, 1)[:, None] * np.abs(o["w"])
    dx, dw, db = ops.group_norm_act_backward(dy, x, mean, rstd, G, w, b, act=act)
    shape = (N, S, G, C // G)
    mean_g = lambda a: a.mean((1, 3), keepdims=True)
    curv = 0.0 if act == "none" else 1.0
    tdv = curv * tv * np.abs(f64(dy))
    e, x4, t4, e4 = (np.abs(a).reshape(shape) for a in (o["dv"] * o["w"], xh, tdv * o["w"], err))
    r = o["rstd"][:, None, :, None]
    E = r * (e + mean_g(e) + x4 * mean_g(e * x4))
    T = 400 * U * E + r * (t4 + mean_g(t4) + x4 * mean_g(t4 * x4 + e * e4) + e4 * mean_g(e * x4))
    close(dx, o["dx"], T.reshape(N, S, C) + last(dtype, o["dx"]))
    n = np.sqrt(N * S) + 200
    close(dw, o["dweight"], n * U * o["dweight_abs"] + (tdv * xh + np.abs(o["dv"]) * err).sum((0, 1)))
    close(db, o["dbias"], n * U * o["dbias_abs"] + tdv.sum((0, 1)))


@pytest.mark.parametrize("S,C,G", [(4096, 4096, 1), (2000, 5893, 1), (65536, 2050, 1), (1, 3000000, 1), (512, 9000, 3)])
def test_long_sums_of_wide_groups(S, C, G):
    """Groups too wide for the tiles, one workgroup each.  All squares about the mean are alike, and so are all terms of the gradients'
    sums: in one chain of additions their roundings would all go the same way.  In three levels of 64 a path has at most
    64 + 64 + n / 4096 / 1024 + 30 < 200 additions: 200 u of the sum of magnitudes, half of it in rstd."""
    g = torch.Generator(device="cuda:0").manual_seed(S + C)
    sign = torch.randint(0, 2, (1, S, C), generator=g, device="cuda:0", dtype=torch.int8).mul_(2).sub_(1)
    x, dy = 0.3 * sign.float() + 0.7, 0.37 * sign.float() + 0.11
    y, mean, rstd = ops.group_norm_act(x, G)
    w = torch.ones(C, device="cuda:0")
    dx, dw, db = ops.group_norm_act_backward(dy, x, mean, rstd, G, w, w)
    for k in range(G):
        sl = slice(k * C // G, (k + 1) * C // G)
        xd, dd = x[..., sl].double(), dy[..., sl].double()
        mu = xd.mean()
        xd -= mu
        r = float(1 / torch.sqrt((xd * xd).mean() + 1e-5))
        assert abs(float(mean[0, k]) - float(mu)) <= U * abs(float(mu)) + 200 * U / r
        assert abs(float(rstd[0, k]) - r) <= 105 * U * r
        xd *= r
        assert float(((y[..., sl].double() - xd).abs() - 210 * U * (1 + xd.abs())).max()) <= 0
        p = dd * xd
        for got, terms in ((dw[sl], p), (db[sl], dd)):
            assert float(((got.double() - terms.sum((0, 1))).abs() - 320 * U * terms.abs().sum((0, 1))).max()) <= 0      # and xhat's 100 u
        s1, s2 = dd.mean(), p.mean()
        E = r * (dd.abs() + dd.abs().mean() + xd.abs() * p.abs().mean())
        want = r * (dd - s1 - xd * s2)
        assert float(((dx[..., sl].double() - want).abs() - 600 * U * E).max()) <= 0


@pytest.mark.parametrize("N,S,C,G", [(1 << 22, 2, 8, 2), (1 << 20, 1, 8, 2)])
def test_parameter_gradients_of_many_samples(N, S, C, G):
    """Two-valued groups, so that all terms of a channel's sums are alike: 8 summands of one sample's or slot's rows, then the same 200 additions."""
    pat = torch.tensor([1.0, -1.0], device="cuda:0").repeat(S * C // 2).view(1, S, C)
    x, dy = (0.3 * pat).repeat(N, 1, 1), (0.37 * pat + 0.11).repeat(N, 1, 1)
    w = torch.ones(C, device="cuda:0")
    _, mean, rstd = ops.group_norm_act(x, G)
    _, dw, db = ops.group_norm_act_backward(dy, x, mean, rstd, G, w, w)
    r = 1 / np.sqrt(float(x[0, 0, 0].double() ** 2) + 1e-5)
    d = dy[0].double()
    close(dw, f64((d * x[0].double() * r).sum(0)) * N, 320 * U * f64((d * x[0].double() * r).abs().sum(0)) * N)
    close(db, f64(d.sum(0)) * N, 208 * U * f64(d.abs().sum(0)) * N)


@pytest.mark.parametrize("B", [1, 2, 3])
def test_a_model_of_few_units_takes_a_short_batch(B):
    """A batch of less than 8 elements takes the general form, whose workspace a model sized for 128 rows has to hold as well."""
    from test_gpu_dense_block import check_step
    check_step(B, 0.0, 0.0, enc=(5,), dec=(4,), Z=3, groups=1)


def test_int8_linear_of_more_columns_than_tiles():
    """One row against 2^30 + 64 weights of one column each: more 64 x 64 tiles than a launch takes, but the few-row form has none.  Its last
    weights and results stand past 32-bit byte offsets."""
    N = (1 << 30) + 64
    x = torch.full((1, 1), 2.0, device="cuda:0")
    w = torch.empty(N, 1, dtype=torch.int8, device="cuda:0")
    w.view(-1).copy_(torch.arange(7, dtype=torch.int8, device="cuda:0").sub_(3).repeat(N // 7 + 1)[:N])
    y = ops.int8_linear(x, w, torch.ones(N, device="cuda:0"))
    s = float(ops.quantize_rows(x)[1])
    step = 1 << 26
    for k in list(range(0, N, step)):
        got, want = y[0, k:k + step].double(), w[k:k + step, 0].double() * (127 * s)
        assert float(((got - want).abs() - 3 * U * want.abs()).max()) <= 0
