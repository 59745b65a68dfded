"""The models' paths through the dense-block operators: set_precision('int8') of OntoVAE and VAE, VAE(norm='group', input_drop=...),
against the float64 oracle of the operators and a plain torch model in float64."""
import ctypes as C

import numpy as np
import pytest
import torch

import ops_oracle as oo
from test_gpu_parity import make_model, medium

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def cosines(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return (a * b).sum(1) / (np.linalg.norm(a, axis=1) * np.linalg.norm(b, axis=1))


# ---------------------------------------------------------------- OntoVAE in 8 bits
@pytest.mark.parametrize("B", [1, 3, 37, 128, 1100])
def test_ontovae_int8_first_product(B):
    """The cached product of a batch is the operator's, to five float32 roundings, through a row index list as well."""
    masks, sd = medium()
    model, _ = make_model(masks, 3, sd)
    e = model._engine
    model.set_precision("int8")
    rng = np.random.RandomState(B)
    X = torch.as_tensor(np.log1p(rng.poisson(0.5, size=(B + 9, 1000))).astype(np.float32)).cuda()
    idx = torch.as_tensor(rng.permutation(B + 9)[:B].astype(np.int32)).cuda()
    ld = (B + 3) // 4 * 4
    W = e.view("W0").cpu().numpy()
    for x, xi, rows in ((X[:B].contiguous(), None, X[:B]), (X, idx, X[idx.long()])):
        h = torch.zeros(e.plan.L, ld, device="cuda")
        e.encode_pre(x, xi, h, 0)
        want = oo.int8_matmul(*oo.quantize_rows(rows.cpu().numpy()), *oo.quantize_rows(W)).T
        got = h.cpu().numpy()[:, :B].astype(np.float64)
        assert (np.abs(got - want) <= 5 * U * np.abs(want)).all()


def test_ontovae_int8_inference_close_and_training_untouched():
    masks, sd = medium()
    rng = np.random.RandomState(1)
    X = np.log1p(rng.poisson(0.5, size=(300, 1000))).astype(np.float32)
    eps = [rng.standard_normal((300, 60)).astype(np.float32) for _ in range(2)]
    acts, recs, grads = {}, {}, {}
    for prec in ("f32", "int8"):
        model, onto = make_model(masks, 3, sd)
        model.set_precision(prec)
        for key, store in (("act", acts), ("rec", recs)):
            q = [torch.as_tensor(a) for a in eps]
            model.eps_source = lambda B: q.pop(0)
            store[prec] = model._pass_data(X, key)
        model.set_precision("f32")           # and back (before the training pass moves the running statistics)
        q = [torch.as_tensor(a) for a in eps]
        assert np.array_equal(model._pass_data(X, "act"), acts["f32"])
        model.set_precision(prec)
        model.eps_source = None
        out = torch.zeros(3, device="cuda")
        model._engine.train_step(torch.as_tensor(X), None, torch.as_tensor(eps[0]), 1e-4, None, out, apply_update=False)
        grads[prec] = (model._engine.Gr.clone(), out.clone())
    assert cosines(acts["int8"], acts["f32"]).min() >= 0.999 and cosines(recs["int8"], recs["f32"]).min() >= 0.999
    assert not np.array_equal(acts["int8"], acts["f32"])
    assert torch.equal(grads["f32"][0], grads["int8"][0]) and torch.equal(grads["f32"][1], grads["int8"][1])
    with pytest.raises(ValueError):
        model.set_precision("int4")


def test_int8_and_bf16_exclude_each_other():
    from onto_vae_amd import _lib
    masks, sd = medium()
    model, _ = make_model(masks, 3, sd)
    model.set_precision("int8")
    model._engine.flags |= _lib.FLAG_BF16_GEMM
    model._engine.invalidate()
    with pytest.raises(ValueError, match="exclude"):
        model._engine.eval_step(torch.zeros(4, 1000), None, None, 1e-4, torch.zeros(3, device="cuda"))


# ---------------------------------------------------------------- the plain VAE with group norm
class Plain(torch.nn.Module):
    """The same model in plain torch, float64, dropout by given factors."""

    def __init__(self, G, enc, dec, Z, groups):
        super().__init__()
        def stack(dims):
            return torch.nn.ModuleList([torch.nn.ModuleList([torch.nn.Linear(a, b), torch.nn.GroupNorm(groups, b)]) for a, b in zip(dims, dims[1:])])
        self.enc, self.dec = stack([G] + enc), stack([Z] + dec)
        self.mu, self.lv, self.out = torch.nn.Linear(enc[-1], Z), torch.nn.Linear(enc[-1], Z), torch.nn.Linear(dec[-1], G)
        self.double()

    def forward(self, x, eps, masks=None):
        k = 0
        def run(blocks, h):
            nonlocal k
            for lin, norm in blocks:
                h = norm(lin(h))
                if masks is not None:
                    h = h * masks[k]
                h, k = torch.relu(h), k + 1
            return h
        h = run(self.enc, x)
        mu, lv = self.mu(h), self.lv(h)
        return self.out(run(self.dec, mu + eps * torch.exp(lv / 2))), mu, lv


def build(G=200, enc=(96, 48), dec=(64,), Z=12, groups=8, drop=0.0, seed=3, **kw):
    from onto_vae_amd.vae_model import VAE
    torch.manual_seed(seed)
    model = VAE(np.zeros((2, G)), list(enc), list(dec), Z, drop=drop, z_drop=0.0, norm="group", groups=groups, **kw)
    sd = model.state_dict()
    g = torch.Generator().manual_seed(seed)
    for k in sd:
        if ".1." in k:          # norm weights and biases away from 1 and 0
            sd[k] = (1.0 if k.endswith("weight") else 0.0) + 0.3 * torch.randn(sd[k].shape, generator=g)
    model.load_state_dict(sd)
    plain = Plain(G, list(enc), list(dec), Z, groups)
    sd = {k: v.cpu().double() for k, v in model.state_dict().items()}
    new = {}
    for i in range(len(enc)):
        for j in (0, 1):
            for n in ("weight", "bias"):
                new[f"enc.{i}.{j}.{n}"] = sd[f"encoder.encoder.{i}.{j}.{n}"]
    for i in range(len(dec)):
        for j in (0, 1):
            for n in ("weight", "bias"):
                new[f"dec.{i}.{j}.{n}"] = sd[f"decoder.decoder.{i}.{j}.{n}"]
    for n in ("weight", "bias"):
        new[f"mu.{n}"], new[f"lv.{n}"], new[f"out.{n}"] = sd[f"encoder.mu.0.{n}"], sd[f"encoder.logvar.0.{n}"], sd[f"decoder.decoder.{len(dec)}.0.{n}"]
    plain.load_state_dict(new)
    return model, plain


def grads_of(model, plain):
    e = model._engine
    for i, (lin, norm) in enumerate(plain.enc):
        yield from zip(e.block_views("enc", i, e.Gr), (lin.weight, lin.bias, norm.weight, norm.bias))
    for i, (lin, norm) in enumerate(plain.dec):
        yield from zip(e.block_views("dec", i, e.Gr), (lin.weight, lin.bias, norm.weight, norm.bias))
    yield from zip(e.head_views(e.Gr), (plain.mu.weight, plain.mu.bias, plain.lv.weight, plain.lv.bias))
    yield from zip(e.out_views(e.Gr), (plain.out.weight, plain.out.bias))


def plain_loss(plain, x, xin, eps, kc, masks=None):
    rec, mu, lv = plain(xin, eps, masks)
    r = ((rec - x) ** 2).sum()
    kl = -0.5 * (1 + lv - mu ** 2 - lv.exp()).sum()
    return r, kl, r + kc * kl


def check_step(B, drop, input_drop, **kw):
    model, plain = build(drop=drop, input_drop=input_drop, **kw)
    rng = np.random.RandomState(B + 5)
    x = np.log1p(rng.poisson(0.7, size=(B, model.in_features))).astype(np.float32)
    eps = rng.standard_normal((B, model.latent_dim)).astype(np.float32)
    e = model._engine
    out = torch.zeros(3, device="cuda")
    off = e.rng_offset + 1
    e.train_step(torch.as_tensor(x), None, torch.as_tensor(eps), 0.3, None, out, apply_update=False)
    masks = None
    if drop > 0:
        masks = []
        for k, w in enumerate(list(e.enc) + list(e.dec)):
            keep, f = oo.keep_mask(B, w, drop, e.seed, off ^ ((k + 1) << 48))
            masks.append(torch.as_tensor(keep * f))
    xd = torch.as_tensor(x).double()
    xin = torch.as_tensor(oo.dropout(x, input_drop, e.seed, off)) if input_drop > 0 else xd
    rec, kl, loss = plain_loss(plain, xd, xin, torch.as_tensor(eps).double(), 0.3, masks)
    loss.backward()
    np.testing.assert_allclose(out.cpu().numpy(), [float(rec), float(kl), float(loss)], rtol=1e-4)
    for got, want in grads_of(model, plain):
        want = want.grad.numpy()
        assert np.abs(got.cpu().numpy() - want).max() <= 2e-5 * np.abs(want).max() + 1e-30
    return model, plain


@pytest.mark.parametrize("B", [1, 2, 37, 128, 530])
def test_group_norm_vae_gradients(B):
    """Every gradient within 2e-5 of its own scale of a float64 torch model, as for the models with BatchNorm; one row is a batch."""
    check_step(B, 0.0, 0.0)


def test_group_norm_vae_gradients_with_dropout_and_input_dropout():
    check_step(64, 0.25, 0.0)
    check_step(64, 0.0, 0.3)
    check_step(37, 0.25, 0.3, groups=4, enc=(1000,), dec=(40, 24), Z=5)


def test_group_norm_vae_steps_against_torch_adamw():
    """Five fused AdamW steps: the loss of each, and the parameters behind the last."""
    model, plain = build()
    from onto_vae_amd.vae_model import FusedAdamW
    opt, popt = FusedAdamW(model, lr=1e-3), torch.optim.AdamW(plain.parameters(), lr=1e-3)
    rng = np.random.RandomState(2)
    out = torch.zeros(5, 3, device="cuda")
    for s in range(5):
        x = np.log1p(rng.poisson(0.7, size=(96, 200))).astype(np.float32)
        eps = rng.standard_normal((96, 12)).astype(np.float32)
        model._engine.train_step(torch.as_tensor(x), None, torch.as_tensor(eps), 1e-2, opt.next_hyper(), out[s])
        popt.zero_grad()
        xd = torch.as_tensor(x).double()
        loss = plain_loss(plain, xd, xd, torch.as_tensor(eps).double(), 1e-2)[2]
        loss.backward()
        popt.step()
        assert abs(float(out[s, 2]) - float(loss)) <= 1e-4 * abs(float(loss))
    model._engine.Gr = model._engine.P
    for got, want in grads_of(model, plain):       # the parameters themselves: an AdamW step is at most lr, noise of tiny gradients a fraction of it
        assert np.abs(got.cpu().numpy() - want.detach().numpy()).max() <= 5e-4


def test_group_norm_vae_eval_is_per_row_and_like_training():
    model, plain = build(drop=0.0)
    model.eval()
    rng = np.random.RandomState(4)
    x = torch.as_tensor(np.log1p(rng.poisson(0.7, size=(50, 200))).astype(np.float32))
    eps = rng.standard_normal((50, 12)).astype(np.float32)
    model.eps_source = lambda B: torch.as_tensor(eps[:B])
    rec, mu, lv = (t.cpu().double().numpy() for t in model(x))
    want = [t.detach().numpy() for t in plain(x.double(), torch.as_tensor(eps).double())]
    for a, b in zip((rec, mu, lv), want):
        assert np.abs(a - b).max() <= 1e-4 * np.abs(b).max()
    one = model(x[:1])[0].cpu().double().numpy()
    assert np.abs(one - rec[:1]).max() <= 1e-5 * np.abs(rec).max()
    model.train()
    assert np.abs(model(x)[0].cpu().double().numpy() - rec).max() <= 1e-6 * np.abs(rec).max()
    keys = list(model.state_dict())
    assert "encoder.encoder.0.1.weight" in keys and not any("running" in k for k in keys)


def test_vae_int8_inference():
    for kw in (dict(), dict(norm="group")):
        from onto_vae_amd.vae_model import VAE
        torch.manual_seed(1)
        model = VAE(np.zeros((2, 333)), [64], [64], 16, drop=0.0, z_drop=0.0, **kw)
        model.eval()
        rng = np.random.RandomState(4)
        for B in (2, 150):
            x = torch.as_tensor(np.log1p(rng.poisson(0.7, size=(B, 333))).astype(np.float32))
            model.eps_source = lambda b: torch.zeros(b, 16)
            model.set_precision("f32")
            a = model(x)[0].cpu().numpy()
            model.set_precision("int8")
            b = model(x)[0].cpu().numpy()
            assert cosines(a, b).min() >= 0.999 and not np.array_equal(a, b)


def test_input_drop_leaves_inference_and_plain_models_alone():
    from onto_vae_amd.vae_model import VAE
    outs = []
    for kw in (dict(), dict(input_drop=0.4)):
        torch.manual_seed(1)
        model = VAE(np.zeros((2, 120)), [32], [32], 8, drop=0.0, z_drop=0.0, **kw)
        model.eval()
        model.eps_source = lambda b: torch.zeros(b, 8)
        outs.append(model(torch.ones(5, 120))[0])
    assert torch.equal(*outs)


def test_train_model_with_the_new_blocks(tmp_path):
    """The whole training loop with group norm, dropout and input dropout runs, logs a finite loss, and its checkpoint loads."""
    from onto_vae_amd.vae_model import VAE
    rng = np.random.RandomState(0)
    X = np.log1p(rng.poisson(0.7, size=(330, 120)))
    torch.manual_seed(5)
    model = VAE(X, [48], [48], 8, drop=0.2, z_drop=0.2, norm="group", groups=6, input_drop=0.2)
    path = str(tmp_path / "m.pt")
    model.train_model(path, lr=1e-3, batch_size=65, epochs=2)
    ck = torch.load(path, map_location="cpu", weights_only=True)
    other = VAE(X, [48], [48], 8, norm="group", groups=6)
    other.load_state_dict(ck["model_state_dict"])
    assert np.isfinite(ck["loss"])


def test_refusals():
    from onto_vae_amd import _lib
    from onto_vae_amd.vae_model import VAE
    X = np.zeros((4, 20))
    for kw in (dict(norm="layer"), dict(norm="group", groups=7), dict(norm="group", groups=0), dict(input_drop=1.0), dict(input_drop=-0.1)):
        with pytest.raises(ValueError):
            VAE(X, [16], [16], 4, **kw)
    model = VAE(X, [16], [16], 4, norm="group", groups=4)
    with pytest.raises(ValueError):
        model.set_precision("bf16")
    e = model._engine
    ctx = e.ctx(4)
    ext = _lib.VaeExt(groups=4)
    rc = _lib.lib().ontovae_vae_forward_ext(C.byref(ctx), C.byref(ext), C.c_void_p(1 << 20), None, 4, None, 1, 0, 0.0, None, None, None, None, None, None)
    assert rc == -1 and b"workspace" in _lib.lib().ontovae_last_error()
