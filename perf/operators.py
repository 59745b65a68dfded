"""The dense-block operators of onto_vae_amd.ops as measurable cases: int8_linear (row quantiser + 8-bit product),
group_norm_act with its backward, dropout with its backward.  `run` computes a case in plain torch operations, or, where
`own` is true, through the framework's entry points."""
import math

import torch

own = False
DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one cell through the first encoder layer of the 20000-gene model: a latency
        dict(name="int8_one_cell", op="int8", M=1, K=20000, N=360, dtype="f32", bias=False, log1p=True),
        # a training-sized batch of cells, same layer
        dict(name="int8_batch128", op="int8", M=128, K=20000, N=360, dtype="f32", bias=False, log1p=True),
        # the inference batch of the pass over a whole dataset: the read of x bounds it
        dict(name="int8_inference_batch", op="int8", M=16384, K=20000, N=360, dtype="f32", bias=False, log1p=True),
        # a square layer in bf16: the matrix cores bound it
        dict(name="int8_square_bf16", op="int8", M=8192, K=4096, N=4096, dtype="bf16", bias=True, log1p=False),
        # ragged: a validation tail over an odd gene count, odd width
        dict(name="int8_ragged_f16", op="int8", M=777, K=5893, N=229, dtype="f16", bias=True, log1p=False),
        # the hidden vector of one cell: a latency
        dict(name="gn_one_cell", op="gn", N=1, S=1, C=360, G=8, dtype="f32", act="relu", drop=0.0, train=False),
        # the plain VAE's hidden layer (1000 wide) over a large batch, trained, with the block's dropout
        dict(name="gn_hidden_train", op="gn", N=8192, S=1, C=1000, G=8, dtype="f32", act="silu", drop=0.2, train=True),
        # feature maps, 10 channels a group (a group ends inside a 16-byte piece), inference
        dict(name="gn_maps_infer", op="gn", N=16, S=4096, C=320, G=32, dtype="bf16", act="silu", drop=0.0, train=False),
        # feature maps, trained: larger than the last-level cache
        dict(name="gn_maps_train", op="gn", N=32, S=4096, C=512, G=32, dtype="bf16", act="silu", drop=0.0, train=True),
        # the dropout of one batch's latent rows: a latency
        dict(name="drop_latent", op="drop", R=128, C=360, dtype="f32", p=0.5, train=True),
        # odd width, trained (forward and backward)
        dict(name="drop_ragged_train", op="drop", R=1023, C=5893, dtype="f32", p=0.2, train=True),
        # input corruption of a whole inference batch
        dict(name="drop_input_bf16", op="drop", R=16384, C=20000, dtype="bf16", p=0.1, train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("int8", "gn", "drop"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "int8":
        while True:
            M, K, N = _log(rng, 1, 16384), _log(rng, 64, 24000), _log(rng, 16, 8192)
            if M * K * N <= 16384 * 20000 * 360 and M * K + M * N + N * K <= 3.3e8:
                return dict(op=op, M=M, K=K, N=N, dtype=dtype, bias=rng.random() < 0.5, log1p=rng.random() < 0.5)
    if op == "gn":
        train = rng.random() < 0.6
        act = rng.choice(("none", "silu", "gelu") if train else ("none", "relu", "silu", "gelu"))   # relu's gradient jumps at 0
        drop = rng.choice((0.0, 0.0, 0.2, 0.5))
        while True:
            S = 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
            G = rng.choice((1, 4, 8, 32, 40))
            C = G * _log(rng, 2, 256)
            N = _log(rng, 1, 8192 if S == 1 else 64)
            if S * C // G >= 8 and N * S * C <= (3.3e7 if dtype == "f32" else 6.7e7):
                return dict(op=op, N=N, S=S, C=C, G=G, dtype=dtype, act=act, drop=drop, train=train)
    while True:
        R, C = _log(rng, 1, 16384), _log(rng, 1, 20000)
        train = rng.random() < 0.5
        if R * C * (2 if train else 1) * (2 if dtype == "f32" else 1) <= 3.2e8:
            return dict(op=op, R=R, C=C, dtype=dtype, p=rng.choice((0.1, 0.2, 0.5, round(rng.uniform(0.01, 0.9), 3))), train=train)


# ---------------------------------------------------------------- inputs
def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)
    if case["op"] == "int8":
        M, K, N = case["M"], case["K"], case["N"]
        if case["log1p"]:          # log counts: most are 0
            x = torch.log1p(torch.floor(torch.rand(M, K, generator=g, device=DEV).mul_(-1).add_(1).log_().mul_(-0.8)))
        else:
            x = randn(M, K)
        return dict(x=x.to(dt), w=randn(N, K) / math.sqrt(K), bias=0.1 * randn(N) if case["bias"] else None)
    if case["op"] == "gn":
        N, S, C = case["N"], case["S"], case["C"]
        x = (randn(N, S, C) + 0.5 * randn(C)).to(dt)
        d = dict(x=x, w=1.0 + 0.1 * randn(C), b=0.1 * randn(C), seed=seed * 7919 + 11, offset=seed + 1)
        if case["train"]:
            d["dy"] = randn(N, S, C).to(dt)
        return d
    d = dict(x=randn(case["R"], case["C"]).to(dt), seed=seed * 7919 + 13, offset=seed + 2)
    if case["train"]:
        d["dy"] = randn(case["R"], case["C"]).to(dt)
    return d


def _quantize(x):
    """Rows of x in 8 bits: scale = max|x| / 127 in 32 bits, values x / scale rounded to the nearest, ties to even (the
    quotient in 64 bits: it decides next to a border)."""
    x = x.float()
    s = x.abs().amax(1) / 127.0
    sd = s.double()[:, None]
    return torch.where(sd > 0, torch.round(x.double() / sd), torch.zeros((), dtype=torch.float64, device=x.device)).clamp(-127, 127).float(), s


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if case["op"] == "int8":       # a program keeps the layer's weights in 8 bits
        w = st.pop("w")
        if own:
            from onto_vae_amd import ops
            st["qw"], st["sw"] = ops.quantize_rows(w)
        else:
            q, st["sw"] = _quantize(w)
            st["qw"] = q.to(torch.int8)
    return st


# ---------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    if own:
        from onto_vae_amd import ops
        if case["op"] == "int8":
            return ops.int8_linear(st["x"], st["qw"], st["sw"], st["bias"])
        if case["op"] == "gn":
            kw = dict(act=case["act"], drop=case["drop"], seed=st["seed"], offset=st["offset"])
            y, mean, rstd = ops.group_norm_act(st["x"], case["G"], st["w"], st["b"], **kw)
            if not case["train"]:
                return y
            return (y, *ops.group_norm_act_backward(st["dy"], st["x"], mean, rstd, case["G"], st["w"], st["b"], **kw))
        y = ops.dropout(st["x"], case["p"], st["seed"], st["offset"])
        if not case["train"]:
            return y
        return y, ops.dropout_backward(st["dy"], case["p"], st["seed"], st["offset"])
    if case["op"] == "int8":
        q, s = _quantize(st["x"])
        y = (q @ st["qw"].float().t()) * s[:, None] * st["sw"]
        if st["bias"] is not None:
            y = y + st["bias"]
        return y.to(st["x"].dtype)
    if case["op"] == "gn":
        return _plain_group_norm(st, case)
    keep, scale = _keep(st["x"].shape, case["p"], st["seed"], st["offset"])
    zero = torch.zeros((), device=DEV)
    y = torch.where(keep, st["x"].float() * scale, zero).to(st["x"].dtype)
    if not case["train"]:
        return y
    return y, torch.where(keep, st["dy"].float() * scale, zero).to(st["dy"].dtype)


def _plain_group_norm(st, case):
    N, S, C, G = case["N"], case["S"], case["C"], case["G"]
    x = st["x"].float().view(N, S, G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean((1, 3), keepdim=True) + 1e-5)
    xhat = (xc * rstd).view(N, S, C)
    v = xhat * st["w"] + st["b"]
    act = case["act"]
    if act == "none":
        a, da = v, torch.ones_like(v)
    elif act == "relu":
        a, da = torch.clamp(v, min=0), (v > 0).float()
    elif act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-v))
        a, da = v * sg, sg * (1.0 + v * (1.0 - sg))
    else:
        cdf = 0.5 * (1.0 + torch.erf(v * 0.7071067811865476))
        a, da = v * cdf, cdf + v * torch.exp(-0.5 * v * v) * 0.3989422804014327
    keep = None
    if case["drop"] > 0:
        keep, scale = _keep(v.shape, case["drop"], st["seed"], st["offset"])
        a = torch.where(keep, a * scale, torch.zeros((), device=DEV))
    y = a.to(st["x"].dtype)
    if not case["train"]:
        return y
    dv = st["dy"].float() * da
    if keep is not None:
        dv = torch.where(keep, dv * scale, torch.zeros((), device=DEV))
    dw, db = (dv * xhat).sum((0, 1)), dv.sum((0, 1))
    e = (dv * st["w"]).view(N, S, G, C // G)
    xh = xhat.view(N, S, G, C // G)
    dx = rstd * (e - e.mean((1, 3), keepdim=True) - xh * (e * xh).mean((1, 3), keepdim=True))
    return y, dx.view(N, S, C).to(st["x"].dtype), dw, db


def _keep(shape, p, seed, offset):
    """Which elements dropout keeps, and the factor of the kept ones.  Eight neighbours of a row share one Philox4x32-10
    block (16 bits each); 64-bit integers hold the 32-bit words."""
    C = shape[-1]
    R = math.prod(shape[:-1])
    nb = (C + 7) // 8
    m32 = 0xFFFFFFFF
    idx = torch.arange(R * nb, device=DEV, dtype=torch.int64)
    c = [idx & m32, (idx >> 32) ^ (6 << 24), torch.full_like(idx, offset & m32), torch.full_like(idx, (offset >> 32) & m32)]
    k0, k1 = seed & m32, (seed >> 32) & m32
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57      # the low 64 bits: both 32-bit halves
        c = [((p1 >> 32) & m32) ^ c[1] ^ k0, p1 & m32, ((p0 >> 32) & m32) ^ c[3] ^ k1, p0 & m32]
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    u = torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], 1).view(R, nb * 8)[:, :C].reshape(shape)
    t = round(p * 65536)
    return u >= t, 65536.0 / (65536 - t) if t < 65536 else 0.0


# ---------------------------------------------------------------- least work
def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "int8":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K * e + N * K + 4 * N + M * N * e + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    if case["op"] == "gn":
        n = case["N"] * case["S"] * case["C"]
        return {"bytes": n * e * (4 if case["train"] else 2) + 8 * case["C"] * (2 if case["train"] else 1), "flops": n * (30 if case["train"] else 10)}
    n = case["R"] * case["C"]
    return {"bytes": n * e * (4 if case["train"] else 2), "flops": n * (2 if case["train"] else 1)}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "int8":
        def q8(t):
            t = t.double()
            s = (t.abs().max(dim=1, keepdim=True).values / 127).float().double()      # the scale is held in 32 bits
            return torch.nan_to_num(t / s, nan=0.0).round().clamp(-127, 127), s
        (qx, sx), (qw, sw) = q8(d["x"]), q8(d["w"])
        y = torch.mm(qx, qw.t().contiguous()) * (sx * sw.t())
        return y if d["bias"] is None else y + d["bias"].double()
    t, sc = None, 1.0
    p = case.get("p", case.get("drop", 0.0))
    if p > 0:
        t = int(round(p * 65536))
        sc = 65536 / (65536 - t) if t < 65536 else 0.0
    if case["op"] == "drop":
        m = _mask_exact(d["x"].shape, t, d["seed"], d["offset"])
        y = (d["x"].double() * sc).masked_fill(~m, 0.0)
        return (y, (d["dy"].double() * sc).masked_fill(~m, 0.0)) if case["train"] else y
    N, S, C, G = case["N"], case["S"], case["C"], case["G"]
    m = _mask_exact(d["x"].shape, t, d["seed"], d["offset"]) if t else None
    outs, dw, db = ([], []), 0, 0
    w, b = d["w"].double(), d["b"].double()
    step = max(1, (1 << 25) // (S * C))
    for i in range(0, N, step):                # sample by sample: nothing couples them but the sums of dw and db
        x = d["x"][i:i + step].double()
        z = x.reshape(x.shape[0], S, G, -1).permute(0, 2, 1, 3).reshape(x.shape[0], G, -1)
        var, mu = torch.var_mean(z, dim=2, unbiased=False)
        spread = lambda a: a.repeat_interleave(C // G, dim=1)[:, None, :]
        r = spread((var + 1e-5) ** -0.5)
        xh = (x - spread(mu)) * r
        v = (xh * w + b).requires_grad_(case["train"])
        with torch.enable_grad():
            y = {"none": lambda u: u * 1.0, "relu": torch.relu, "silu": lambda u: u * torch.sigmoid(u),
                 "gelu": lambda u: u * torch.special.ndtr(u)}[case["act"]](v)
            if m is not None:
                y = (y * sc).masked_fill(~m[i:i + step], 0.0)
        outs[0].append(y.detach())
        if case["train"]:
            dv, = torch.autograd.grad(y, v, d["dy"][i:i + step].double())
            dw, db = dw + (dv * xh).sum((0, 1)), db + dv.sum((0, 1))
            e = dv * w
            tog = lambda a: spread(a.sum(1).view(-1, G, C // G).sum(2) / (S * (C // G)))
            outs[1].append(r * (e - tog(e) - xh * tog(e * xh)))
    y = torch.cat(outs[0])
    return (y, torch.cat(outs[1]), dw, db) if case["train"] else y


def _mask_exact(shape, t, seed, offset):
    """The kept elements from Philox4x32-10 with every 32 x 32-bit product built from 16-bit halves."""
    C, R = shape[-1], math.prod(shape[:-1])
    nb = -(-C // 8)

    def mul(a, x):
        a0, a1, x0, x1 = a & 0xFFFF, a >> 16, x & 0xFFFF, x >> 16
        mid = a1 * x0 + ((a0 * x0) >> 16)
        mid2 = a0 * x1 + (mid & 0xFFFF)
        return a1 * x1 + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((a0 * x0) & 0xFFFF)

    out = torch.empty(R * nb, 8, dtype=torch.bool, device=DEV)
    for lo in range(0, R * nb, 1 << 23):
        i = torch.arange(lo, min(lo + (1 << 23), R * nb), device=DEV, dtype=torch.int64)
        x0, x1 = i % (1 << 32), (i // (1 << 32)) ^ 0x06000000
        x2, x3 = torch.zeros_like(i) + offset % (1 << 32), torch.zeros_like(i) + (offset // (1 << 32)) % (1 << 32)
        for r in range(10):
            ka, kb = (seed + r * 0x9E3779B9) % (1 << 32), (seed // (1 << 32) + r * 0xBB67AE85) % (1 << 32)
            (h0, l0), (h1, l1) = mul(0xD2511F53, x0), mul(0xCD9E8D57, x2)
            x0, x1, x2, x3 = h1 ^ x1 ^ ka, l1, h0 ^ x3 ^ kb, l0
        for j, wd in enumerate((x0, x1, x2, x3)):
            out[lo:lo + i.numel(), 2 * j] = wd % 65536 >= t
            out[lo:lo + i.numel(), 2 * j + 1] = wd // 65536 >= t
    return out.view(R, nb * 8)[:, :C].reshape(shape)
