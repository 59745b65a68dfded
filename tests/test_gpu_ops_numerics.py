"""Group norm on the GPU where digits are lost first: values far from 0 against their spread, long sums.  Against oracle/ops_oracle.py in
float64; u = 2^-24 (half a step of float32)."""
import numpy as np
import pytest
import torch

import ops_oracle as oo
from onto_vae_amd import ops
from test_gpu_ops import U, close, f64, rnd

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
