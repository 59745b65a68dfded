"""The data-parallel BatchNorm forward against the formula where its mean is far from 0: simulated ranks on one GPU, the collectives by hand."""
import numpy as np
import pytest
import torch

from test_gpu_parity import make_model, medium

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("parts", [[(0, 1100), (1100, 2213)], [(0, 1030), (1030, 1731)], [(0, 300), (300, 800)]])
def test_a_constant_unit_stays_constant_over_the_ranks(parts):
    """A first layer of zero weights: every row of the global batch has the same h, its mean is that value and xhat is 0.  What a float32 sum
    over the rows leaves of the mean would be blown up by rstd = 1 / sqrt(eps) = 316 (1e-2 at h around 500) and reach the gradient of
    gamma; a rank's nearest mean is h itself, and what the combination over the ranks rounds is taken off to 2^-24 of itself.
    (Ranks of 1024 rows and more, of fewer, one of each.)"""
    masks, sd = medium()
    L, B = 60, parts[-1][1]
    rng = np.random.RandomState(3)
    x = torch.as_tensor(np.log1p(rng.poisson(0.5, size=(B, 1000))).astype(np.float32)).cuda()
    eps = torch.as_tensor(rng.standard_normal((B, L)).astype(np.float32)).cuda()
    h = torch.as_tensor((500 + 100 * rng.standard_normal(L)).astype(np.float32)).cuda()
    ranks = []
    for _ in parts:
        m, _ = make_model(masks, 3, sd)
        e = m._engine
        lay = e.plan.layout
        e.view("W0").zero_()
        e.P[int(lay.b0):int(lay.b0) + L] = h
        ranks.append(m)
    stats = [torch.zeros(2 * L + 1, device="cuda") for _ in ranks]
    bstats = [torch.zeros(2, L, device="cuda") for _ in ranks]
    louts = [torch.zeros(3, device="cuda") for _ in ranks]
    for r, (m, (a, b)) in enumerate(zip(ranks, parts)):
        stats[r][2 * L] = float(b - a)
        m._engine.train_step_dp(0, x[a:b], None, B, eps[a:b], 1e-4, stats[r][:2 * L].view(2, L), bstats[r], louts[r], 1)
        assert torch.equal(stats[r][:L], h) and float(stats[r][L:2 * L].max()) <= 1e-9
    gathered = torch.cat(stats)
    dy, dyx = 0, 0
    for r, (m, (a, b)) in enumerate(zip(ranks, parts)):
        m._engine.train_step_dp(16 + len(parts), x[a:b], None, B, eps[a:b], 1e-4, gathered, bstats[r], louts[r], 1)
        dy, dyx = dy + bstats[r][0].double(), dyx + bstats[r][1].double()
    # what is left: |xhat| <= 316 * 2^-23 * (a step of the mean, 6e-5) = 3e-9
    assert float(dyx.abs().max()) <= 1e-6 * float(dy.abs().max() + 1)
    e = ranks[0]._engine
    for m in ranks[1:]:
        assert torch.equal(m._engine.rmean, e.rmean) and torch.equal(m._engine.rvar, e.rvar)       # replicas stay alike
