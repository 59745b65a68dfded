"""onto_vae_amd.ops inside autograd: no graph is recorded, and a call that would cut one says so."""
import warnings

import pytest
import torch

from onto_vae_amd import ops
from test_gpu_ops import rnd

pytestmark = pytest.mark.gpu


def calls(x):
    qw, sw = ops.quantize_rows(rnd(2, 24, 16))
    return ((lambda: ops.group_norm_act(x, 4)[0], "group_norm_act"), (lambda: ops.dropout(x, 0.5, 1), "dropout"), (lambda: ops.int8_linear(x, qw, sw), "int8_linear"))


def test_a_cut_graph_is_named():
    x = rnd(1, 6, 16)
    leaf = x.clone().requires_grad_()
    for (plain, _), (cut, name) in zip(calls(x), calls(leaf * 1.0)):
        with pytest.warns(UserWarning, match=f"{name} records no autograd graph"):
            y = cut()
        assert not y.requires_grad
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            assert torch.equal(plain(), y)
            with torch.no_grad():
                assert torch.equal(cut(), y)
    with warnings.catch_warnings():          # a layer's parameters may require grad: their gradients come from explicit calls
        warnings.simplefilter("error")
        w = torch.nn.Parameter(torch.ones(16, device="cuda:0"))
        ops.quantize_rows(torch.nn.Parameter(x))
        ops.group_norm_act(x, 4, w, w)


def test_the_operators_in_an_autograd_function():
    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, b):
            y, mean, rstd = ops.group_norm_act(x, 4, w, b, act="silu")
            ctx.save_for_backward(x, w, b, mean, rstd)
            return y

        @staticmethod
        def backward(ctx, dy):
            x, w, b, mean, rstd = ctx.saved_tensors
            return ops.group_norm_act_backward(dy, x, mean, rstd, 4, w, b, act="silu")

    x, w, b = (t.requires_grad_() for t in (rnd(1, 6, 16), rnd(2, 16), rnd(3, 16)))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        Norm.apply(x, w, b).square().sum().backward()
    got = [t.grad.clone() for t in (x, w, b)]
    leaves = [t.detach().double().requires_grad_() for t in (x, w, b)]
    torch.nn.functional.silu(torch.nn.functional.group_norm(leaves[0], 4, leaves[1], leaves[2])).square().sum().backward()
    for g, l in zip(got, leaves):
        torch.testing.assert_close(g.double(), l.grad, rtol=1e-4, atol=1e-5)
