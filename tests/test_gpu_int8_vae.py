"""VAE.set_precision('int8'): the latent means of an inference pass against the 8-bit first layer in float64, from one row on."""
import numpy as np
import pytest
import torch

import ops_oracle as oo

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
G, H, Z, GROUPS = 333, 64, 16, 8


@pytest.mark.parametrize("norm", ["batch", "group"])
@pytest.mark.parametrize("B", [1, 3, 5, 37, 300])
def test_latent_means(B, norm):
    """The product is off by five float32 roundings of |t| (its sum is exact), the bias adds one; the norm scales that by rstd and adds its
    own (BatchNorm with running statistics 6 u of its terms, group norm 100 u (1 + |xhat|) and what the statistics feel of h), a
    product of 64 terms at most 74 u of its sum of magnitudes."""
    from onto_vae_amd.vae_model import VAE
    torch.manual_seed(B)
    model = VAE(np.zeros((2, G)), [H], [H], Z, drop=0.0, z_drop=0.0, norm=norm, groups=GROUPS)
    sd = model.state_dict()
    g = torch.Generator().manual_seed(3)
    rand = lambda k, shift, scale: sd.__setitem__(k, shift + scale * torch.randn(sd[k].shape, generator=g))
    rand("encoder.encoder.0.1.weight", 1.0, 0.3)
    rand("encoder.encoder.0.1.bias", 0.0, 0.3)
    if norm == "batch":
        rand("encoder.encoder.0.1.running_mean", 0.0, 0.3)
        sd["encoder.encoder.0.1.running_var"] = 0.1 + torch.rand(H, generator=g)
    model.load_state_dict(sd)
    sd = {k: v.double().cpu().numpy() for k, v in model.state_dict().items()}
    model.eval()
    model.set_precision("int8")
    rng = np.random.RandomState(B)
    X = np.log1p(rng.poisson(0.7, size=(B + 5, G))).astype(np.float32)
    idx = rng.permutation(B + 5)[:B].astype(np.int32)
    Xd = torch.as_tensor(X).cuda()
    for x, xi, rows in ((Xd[:B].contiguous(), None, X[:B]), (Xd, torch.as_tensor(idx).cuda(), X[idx])):
        got = model._engine.forward(x, xi, eps=torch.zeros(B, Z), want=("mu",))["mu"].cpu().numpy()
        W, b = sd["encoder.encoder.0.0.weight"], sd["encoder.encoder.0.0.bias"]
        t = oo.int8_matmul(*oo.quantize_rows(rows), *oo.quantize_rows(W))
        h, err = t + b, 5 * U * np.abs(t) + U * (np.abs(t) + np.abs(b))
        ga, be = sd["encoder.encoder.0.1.weight"], sd["encoder.encoder.0.1.bias"]
        if norm == "batch":
            rm, r = sd["encoder.encoder.0.1.running_mean"], 1 / np.sqrt(sd["encoder.encoder.0.1.running_var"] + 1e-5)
            xh = (h - rm) * r
            err = (err + 2 * U * (np.abs(h) + np.abs(rm))) * r + 4 * U * np.abs(xh)
        else:
            o = oo.group_norm_act(h[:, None], GROUPS)
            xh, per = o["xhat"][:, 0], (B, GROUPS, H // GROUPS)
            e, x3 = err.reshape(per), np.abs(xh).reshape(per)
            r = o["rstd"][:, :, None]
            err = (r * (e + e.mean(2, keepdims=True)) + x3 * r * (x3 * e).mean(2, keepdims=True)).reshape(B, H) + 100 * U * (1 + np.abs(xh))
        a = np.maximum(xh * ga + be, 0)
        err = np.abs(ga) * err + 2 * U * (np.abs(xh * ga) + np.abs(be))
        Wm, bm = sd["encoder.mu.0.weight"], sd["encoder.mu.0.bias"]
        want = a @ Wm.T + bm
        tol = err @ np.abs(Wm).T + 75 * U * (a @ np.abs(Wm).T + np.abs(bm))
        assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
