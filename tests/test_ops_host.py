"""Dense-block operators, what needs no GPU: the oracle against torch and finite differences, and every refusal of the C entry
points (the checks come before any pointer is used)."""
import ctypes as C

import numpy as np
import pytest
import torch

import ops_oracle as oo


def test_oracle_group_norm_against_torch_and_differences():
    rng = np.random.default_rng(3)
    N, S, Cn, G = 2, 3, 12, 4
    x, dy = rng.standard_normal((N, S, Cn)), rng.standard_normal((N, S, Cn))
    w, b = 1 + 0.3 * rng.standard_normal(Cn), rng.standard_normal(Cn)
    fns = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}
    for name, fn in fns.items():
        t = [torch.tensor(a, requires_grad=True) for a in (x, w, b)]
        y = fn(torch.nn.functional.group_norm(t[0].permute(0, 2, 1), G, t[1], t[2], 1e-5)).permute(0, 2, 1)
        y.backward(torch.tensor(dy))
        o = oo.group_norm_act(x, G, w, b, 1e-5, name, dy=dy)
        for got, want in ((o["y"], y), (o["dx"], t[0].grad), (o["dweight"], t[1].grad), (o["dbias"], t[2].grad)):
            np.testing.assert_allclose(got, want.detach().numpy(), rtol=1e-10, atol=1e-12)
    # differences, with the dropout mask in place
    kw = dict(eps=1e-5, name="silu", drop=0.3, seed=7, offset=9)
    o = oo.group_norm_act(x, G, w, b, dy=dy, **kw)
    for idx in ((0, 0, 0), (1, 2, 11), (0, 1, 5)):
        d = np.zeros_like(x)
        d[idx] = 1e-6
        num = ((oo.group_norm_act(x + d, G, w, b, **kw)["y"] - oo.group_norm_act(x - d, G, w, b, **kw)["y"]) * dy).sum() / 2e-6
        assert abs(num - o["dx"][idx]) < 1e-7


def test_oracle_quantizer_and_mask():
    x = np.array([[0.5, -1.0, 0.25, 0.0], [0, 0, 0, 0], [np.inf, 1, 2, 3], [np.nan, 1, 2, 3]])
    q, s = oo.quantize_rows(x)
    assert q.tolist()[:2] == [[64, -127, 32, 0], [0, 0, 0, 0]] and s[1] == 0 and np.isnan(s[2:]).all() and not q[2:].any()
    keep, f = oo.keep_mask(2000, 13, 0.25, 5, 1)
    assert abs(keep.mean() - 0.75) < 5 * np.sqrt(0.25 * 0.75 / keep.size) and f == 65536 / 49152
    assert not oo.keep_mask(4, 9, 1.0, 5, 1)[0].any() and oo.keep_mask(4, 9, 0.0, 5, 1)[0].all()


@pytest.fixture(scope="module")
def L():
    from onto_vae_amd import _lib
    return _lib.lib()


P = C.c_void_p(1 << 20)      # never dereferenced: the refusal comes first
NULL = C.c_void_p(0)


@pytest.mark.parametrize("change", [dict(M=-1), dict(K=-1), dict(ldx=3), dict(ldq=3), dict(dtype=3), dict(dtype=-1), dict(n_src=1), dict(x=NULL),
                                    dict(q=NULL), dict(scale=NULL), dict(n_src=-1), dict(K=(1 << 30) + 1, ldx=1 << 31, ldq=1 << 31)])
def test_quantize_rows_refusals(L, change):
    a = dict(x=P, dtype=0, ldx=4, rows=NULL, n_src=2, M=2, K=4, q=P, ldq=4, scale=P, stream=NULL)
    a.update(change)
    assert L.ontovae_quantize_rows(*a.values()) == -1
    assert b"quantize_rows" in L.ontovae_last_error()


@pytest.mark.parametrize("change", [dict(M=-1), dict(N=-1), dict(K=-1), dict(lda=3), dict(ldb=3), dict(ldy=2), dict(K=131072, lda=1 << 20, ldb=1 << 20),
                                    dict(dtype=7), dict(M=2 ** 31 - 1), dict(M=2 ** 30, N=2 ** 20, ldy=2 ** 20), dict(a=NULL), dict(b=NULL), dict(sa=NULL), dict(sb=NULL), dict(y=NULL)])
def test_int8_matmul_refusals(L, change):
    a = dict(a=P, lda=4, sa=P, b=P, ldb=4, sb=P, bias=NULL, M=2, N=3, K=4, y=P, dtype=0, ldy=3, ws=NULL, nbytes=0, stream=NULL)
    a.update(change)
    assert L.ontovae_int8_matmul(*a.values()) == -1
    assert b"int8_matmul" in L.ontovae_last_error()


def test_int8_matmul_needs_its_workspace(L):
    for M, N, K in ((1, 360, 20000), (128, 360, 20000)):
        need = L.ontovae_int8_matmul_workspace_bytes(M, N, K)
        if need > 0:
            assert L.ontovae_int8_matmul(P, K, P, P, K, P, NULL, M, N, K, P, 0, N, P, need - 1, NULL) == -1
            assert L.ontovae_int8_matmul(P, K, P, P, K, P, NULL, M, N, K, P, 0, N, NULL, need, NULL) == -1


@pytest.mark.parametrize("change", [dict(M=-1), dict(N=-1), dict(K=-1), dict(ldx=3), dict(ldw=3), dict(ldy=2), dict(n_src=1), dict(dtype=3), dict(ydtype=-1),
                                    dict(K=131072, ldx=1 << 20, ldw=1 << 20), dict(x=NULL), dict(w=NULL), dict(sw=NULL), dict(y=NULL),
                                    dict(M=9, n_src=9, nbytes=8), dict(M=9, n_src=9, ws=NULL), dict(M=9, n_src=9, ws=C.c_void_p((1 << 20) + 16))])
def test_int8_linear_refusals(L, change):
    a = dict(x=P, dtype=0, ldx=4, rows=NULL, n_src=2, w=P, ldw=4, sw=P, bias=NULL, M=2, N=3, K=4, y=P, ydtype=0, ldy=3, ws=P, nbytes=1 << 30, stream=NULL)
    a.update(change)
    assert L.ontovae_int8_linear(*a.values()) == -1
    assert b"int8_linear" in L.ontovae_last_error()


GN = dict(x=P, dtype=0, N=2, S=3, C=8, groups=2, w=P, b=P, wdtype=0, eps=1e-5, act=0, drop=0.0, seed=0, offset=0, y=P, mean=P, rstd=P, ws=P,
          nbytes=1 << 30, stream=NULL)


@pytest.mark.parametrize("change", [dict(N=-1), dict(S=-1), dict(C=-8), dict(N=2 ** 31 - 1), dict(S=2 ** 31 - 1), dict(C=2 ** 31 - 2), dict(groups=0), dict(groups=3), dict(groups=-2), dict(dtype=3), dict(wdtype=5),
                                    dict(act=4), dict(act=-1), dict(drop=-0.1), dict(drop=1.5), dict(drop=float("nan")), dict(eps=-1.0),
                                    dict(eps=float("nan")), dict(x=NULL), dict(y=NULL), dict(mean=NULL), dict(rstd=NULL)])
def test_group_norm_act_refusals(L, change):
    a = dict(GN)
    a.update(change)
    assert L.ontovae_group_norm_act(*a.values()) == -1
    assert b"group_norm_act" in L.ontovae_last_error()


@pytest.mark.parametrize("change", [dict(N=-1), dict(groups=3), dict(dtype=3), dict(act=9), dict(drop=2.0), dict(dy=NULL), dict(x=NULL), dict(mean=NULL),
                                    dict(rstd=NULL), dict(dx=NULL)])
def test_group_norm_act_backward_refusals(L, change):
    a = dict(dy=P, x=P, dtype=0, N=2, S=3, C=8, groups=2, w=P, b=P, wdtype=0, mean=P, rstd=P, act=0, drop=0.0, seed=0, offset=0, dx=P, dw=P, db=P,
             ws=P, nbytes=1 << 30, stream=NULL)
    a.update(change)
    assert L.ontovae_group_norm_act_backward(*a.values()) == -1
    assert b"group_norm_act_backward" in L.ontovae_last_error()


def test_group_norm_act_needs_its_workspace(L):
    for S, backward in ((1, 1), (4096, 0), (4096, 1)):
        need = L.ontovae_group_norm_act_workspace_bytes(0, 64, S, 512, 32, backward)
        assert need >= 0
        if need == 0:
            continue
        for ws, nbytes in ((P, need - 1), (NULL, need)):
            if backward:
                rc = L.ontovae_group_norm_act_backward(P, P, 0, 64, S, 512, 32, P, P, 0, P, P, 0, 0.0, 0, 0, P, P, P, ws, nbytes, NULL)
            else:
                rc = L.ontovae_group_norm_act(P, 0, 64, S, 512, 32, P, P, 0, 1e-5, 0, 0.0, 0, 0, P, P, P, ws, nbytes, NULL)
            assert rc == -1 and b"workspace" in L.ontovae_last_error()


@pytest.mark.parametrize("change", [dict(R=-1), dict(C=-1), dict(ldx=3), dict(n_src=1), dict(p=-0.5), dict(p=1.1), dict(p=float("nan")), dict(dtype=9),
                                    dict(x=NULL), dict(y=NULL), dict(n_src=-1)])
def test_dropout_refusals(L, change):
    a = dict(x=P, dtype=0, ldx=4, rows=NULL, n_src=2, R=2, C=4, p=0.5, seed=1, offset=1, y=P, stream=NULL)
    a.update(change)
    assert L.ontovae_dropout(*a.values()) == -1
    assert b"dropout" in L.ontovae_last_error()


def test_empty_calls_launch_nothing(L):
    assert L.ontovae_quantize_rows(NULL, 0, 4, NULL, 0, 0, 4, NULL, 4, NULL, NULL) == 0
    assert L.ontovae_int8_matmul(NULL, 4, NULL, NULL, 4, NULL, NULL, 0, 3, 4, NULL, 0, 3, NULL, 0, NULL) == 0
    assert L.ontovae_int8_matmul(NULL, 4, NULL, NULL, 4, NULL, NULL, 3, 0, 4, NULL, 0, 0, NULL, 0, NULL) == 0
    assert L.ontovae_group_norm_act(NULL, 0, 0, 3, 8, 2, NULL, NULL, 0, 1e-5, 0, 0.0, 0, 0, NULL, NULL, NULL, NULL, 0, NULL) == 0
    assert L.ontovae_dropout(NULL, 0, 4, NULL, 0, 0, 4, 0.5, 1, 1, NULL, NULL) == 0
    assert L.ontovae_dropout(NULL, 0, 0, NULL, 5, 5, 0, 0.5, 1, 1, NULL, NULL) == 0


def test_python_entry_points_refuse_host_tensors():
    from onto_vae_amd import _lib, ops
    x = torch.zeros(2, 8)
    for fn in (lambda: ops.quantize_rows(x), lambda: ops.dropout(x, 0.5, 1), lambda: ops.group_norm_act(x, 2),
               lambda: ops.int8_matmul(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0])):
        with pytest.raises(_lib.OntoVAEHipError, match="no CPU path"):
            fn()


def test_vae_ext_sizing_and_refusals(L):
    from onto_vae_amd import _lib
    d = _lib.VaeDims()
    d.G, d.Z, d.n_enc, d.n_dec = 500, 8, 1, 1
    d.enc[0], d.dec[0] = 96, 64
    size = lambda **kw: L.ontovae_vae_ext_workspace_bytes(C.byref(d), C.byref(_lib.VaeExt(**kw)), 128)
    assert size() == 0
    assert size(groups=8) > 0 and size(input_drop=0.5) >= 4 * 128 * 500 and size(flags=_lib.VAE_FLAG_INT8_INPUT) > 96 * 500
    for bad in (dict(groups=-1), dict(groups=7), dict(input_drop=1.0), dict(input_drop=-0.5), dict(input_drop=float("nan")), dict(flags=2), dict(reserved=1)):
        assert size(**bad) == -1
    # enough for every smaller batch
    top = size(groups=8)
    for b in (1, 2, 64, 127):
        assert L.ontovae_vae_ext_workspace_bytes(C.byref(d), C.byref(_lib.VaeExt(groups=8)), b) <= top


def test_int8_workspace_of_a_model_covers_every_batch(L):
    from onto_vae_amd import _lib
    dims = _lib.Dims()
    for L_, G, top in ((360, 20000, 700), (60, 1000, 5000), (228, 5892, 300)):
        dims.L, dims.G = L_, G
        have = L.ontovae_int8_workspace_bytes(C.byref(dims), top)
        for b in list(range(1, top, 7)) + [top]:
            fixed = have - L.ontovae_int8_linear_workspace_bytes(b, L_, G)
            assert fixed >= L_ * G + 4 * L_ + 4 * L_ * b
    assert L.ontovae_int8_workspace_bytes(C.byref(dims), 0) == -1
