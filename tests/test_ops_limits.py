"""Sizes at the ends of the integer types: the sizing functions and the refusals of the dense-block operators, no GPU needed (a
refusal comes before any pointer is used).  Where a wrapped size could end the process, the calls run in one of their own."""
import ctypes as C
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOP = 2 ** 31 - 1


def call(*exprs):
    """The values of expressions in L (the library), P (a pointer that nobody follows), NULL and err() (the last error's text)."""
    code = ("import ctypes as C\nfrom onto_vae_amd import _lib\nL = _lib.lib()\nP, NULL = C.c_void_p(1 << 20), C.c_void_p(0)\n"
            "err = lambda: L.ontovae_last_error().decode()\n" + "".join(f"print(repr({e}), flush=True)\n" for e in exprs))
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, exprs[len(r.stdout.splitlines())], r.stderr[-500:])
    return [eval(line) for line in r.stdout.splitlines()]


def test_group_norm_sizing_of_many_groups():
    """groups * 8 threads pass 32 bits from 2^28 groups on.  One sample fills the card then: one row of gradient sums, two
    float32 a channel, however many samples follow."""
    for groups in (2 ** 28, 2 ** 29 - 1, 2 ** 29, 2 ** 29 + 1, 2 ** 30, 2 ** 31 - 1 - 65536):
        got = call(f"L.ontovae_group_norm_act_workspace_bytes(0, 1, 1, {groups}, {groups}, 1)",
                   f"L.ontovae_group_norm_act_workspace_bytes(0, 1, 1, {groups}, {groups}, 0)",
                   f"L.ontovae_group_norm_act_workspace_bytes(1, 17, 1, {groups}, {groups}, 1)")
        assert got == [8 * groups, 0, 8 * groups], groups


@pytest.mark.parametrize("N,S,Cn,groups", [(TOP, 1, 8, 8), (1, TOP, 8, 8), (1, 1, TOP, 1), (TOP, TOP, TOP, 1)])
def test_group_norm_sizing_past_the_sizes_it_takes(N, S, Cn, groups):
    """Sizes that the entry points refuse: no workspace, nothing divided by what wrapped to 0."""
    assert call(f"L.ontovae_group_norm_act_workspace_bytes(0, {N}, {S}, {Cn}, {groups}, 1)") == [0]


@pytest.mark.parametrize("name", ["int8_matmul", "int8_linear"])
def test_int8_sizing_at_the_ends(name):
    """M or N next to 2^31: rounded up to whole tiles it passes 32 bits.  0 for the sizes that the entry points refuse; below them
    the rows in 8 bits (linear) and no slabs, as there are tiles enough."""
    f = f"L.ontovae_{name}_workspace_bytes"
    assert call(f"{f}({TOP}, 64, 64)", f"{f}(64, {TOP}, 64)", f"{f}({TOP}, {TOP}, 64)", f"{f}({TOP - 1023}, 64, 64)") == [0] * 4
    big = TOP - 1024
    row = (big * 128 + 255) // 256 * 256 + (big * 4 + 255) // 256 * 256 if name == "int8_linear" else 0
    few = 64 * 128 + 256 if name == "int8_linear" else 0
    assert call(f"{f}({big}, 64, 64)", f"{f}(64, {big}, 64)") == [row, few]


def test_int8_workspace_of_a_model_at_the_ends():
    """What a model asks for its largest batch is enough for the largest batch itself."""
    got = call(*(f"(lambda d: (setattr(d, 'L', {L}), setattr(d, 'G', {G}), L.ontovae_int8_workspace_bytes(C.byref(d), {B}), "
                 f"L.ontovae_int8_linear_workspace_bytes({B}, {L}, {G}))[2:])(_lib.Dims())" for L, G, B in
                 ((360, 1000, TOP - 1024), (360, 20000, 2 ** 30), (1, 1, TOP - 1024), (360, 20000, 16384))))
    for (have, need), (L_, G, B) in zip(got, ((360, 1000, TOP - 1024), (360, 20000, 2 ** 30), (1, 1, TOP - 1024), (360, 20000, 16384))):
        assert have >= need + L_ * G + 4 * L_ + 4 * L_ * B > 0


@pytest.mark.parametrize("M", [1, 2, 4, 5])
def test_int8_linear_refuses_more_columns_than_its_indexes_hold(M):
    """The few-row form walks the weight rows with 32-bit steps of its grid: past 2^31 - 1024 rows they would wrap to negative ones.  (Its
    refusal is read from the message: where there is no card a launch fails, too.)"""
    for N in (TOP - 1023, TOP):
        rc, text = call(f"L.ontovae_int8_linear(P, 0, 1, NULL, {M}, P, 1, P, NULL, {M}, {N}, 1, P, 0, {N}, P, 1 << 40, NULL)", "err()")
        assert rc == -1 and "int8_linear" in text and str(N) in text


def refused(expr, *words):
    from onto_vae_amd import _lib
    L = _lib.lib()
    rc = eval(expr, dict(L=L, P=C.c_void_p(1 << 20), NULL=C.c_void_p(0)))
    text = L.ontovae_last_error().decode()
    assert rc == -1, (rc, text)           # the library's refusal, not the runtime's
    assert all(w in text for w in words), text


@pytest.mark.parametrize("R,Cn,dtype", [(2 ** 29, 64, 0), (2 ** 29, 57, 1), (TOP, 16, 2), (TOP, TOP, 0), (16, TOP - 7, 1), (17, TOP, 1)])
def test_dropout_of_more_than_one_launch(R, Cn, dtype):
    """One thread per 8 elements, less than 2^32 of them."""
    refused(f"L.ontovae_dropout(P, {dtype}, {Cn}, NULL, {R}, {R}, {Cn}, 0.5, 1, 1, P, NULL)", "dropout", "too many")


@pytest.mark.parametrize("N,S,Cn,groups", [
    (1, 1, 2 ** 29, 2 ** 29),          # one sample of 2^32 threads
    (1, 1, 2 ** 30, 2 ** 30),
    (2 ** 24, 2, 8, 2),                # a workgroup a sample
    (2 ** 24, 2, 8, 8),
    (2 ** 22, 1, 16385, 1),            # the general form: 1024 threads a group
    (2 ** 22, 2, 2049, 1),
    (TOP - 65536, TOP - 65536, 8, 1)])
def test_group_norm_of_more_than_one_launch(N, S, Cn, groups):
    refused(f"L.ontovae_group_norm_act(P, 0, {N}, {S}, {Cn}, {groups}, P, P, 0, 1e-5, 0, 0.0, 0, 0, P, P, P, P, 1 << 62, NULL)",
            "group_norm_act", "too many")
    refused(f"L.ontovae_group_norm_act_backward(P, P, 0, {N}, {S}, {Cn}, {groups}, P, P, 0, P, P, 0, 0.0, 0, 0, P, P, P, P, 1 << 62, NULL)",
            "group_norm_act_backward", "too many")


def test_group_norm_parameter_gradients_of_more_than_one_launch():
    """64 threads a channel: the gradient sums of 2^26 channels are refused before anything is written."""
    for dw, db in (("P", "P"), ("P", "NULL"), ("NULL", "P")):
        refused(f"L.ontovae_group_norm_act_backward(P, P, 0, 1, 1, {2 ** 26}, {2 ** 13}, P, P, 0, P, P, 0, 0.0, 0, 0, P, {dw}, {db}, P, 1 << 62, NULL)",
                "group_norm_act_backward", "too many")


@pytest.mark.parametrize("M,K,dtype", [(2 ** 26, 8, 0), (TOP, 1, 1), (2 ** 24, 2000, 0), (2 ** 23, 20000, 1), (2 ** 22, 50000, 1), (2 ** 24, 1 << 30, 1)])
def test_quantizing_more_rows_than_one_launch_takes(M, K, dtype):
    refused(f"L.ontovae_quantize_rows(P, {dtype}, {K}, NULL, {M}, {M}, {K}, P, {K}, P, NULL)", "quantize_rows", "too many")


@pytest.mark.parametrize("M,N,K", [(2 ** 30, 2 ** 12, 64), (2 ** 20, 2 ** 17, 16), (32, TOP - 1024, 16)])
def test_int8_products_of_more_than_one_launch(M, N, K):
    """In tiles of 256 x 256, of 64 x 64 where the rows do not start on 16 bytes (the last two)."""
    lda = K + 1 if K == 16 else K
    refused(f"L.ontovae_int8_matmul(P, {lda}, P, P, {lda}, P, NULL, {M}, {N}, {K}, P, 0, {N}, P, 1 << 62, NULL)", "int8_matmul", "too many")
    refused(f"L.ontovae_int8_linear(P, 0, {K}, NULL, {M}, P, {lda}, P, NULL, {M}, {N}, {K}, P, 0, {N}, P, 1 << 62, NULL)", "int8_linear", "too many")


def test_int8_linear_of_more_rows_than_its_quantizer_takes():
    refused(f"L.ontovae_int8_linear(P, 0, 8, NULL, {2 ** 26}, P, 8, P, NULL, {2 ** 26}, 1, 8, P, 0, 1, P, 1 << 62, NULL)", "int8_linear", "too many")


@pytest.mark.parametrize("p", [1.0, 1 - 1e-9, -0.1, float("nan")])
def test_input_drop_is_refused_where_the_library_would_refuse_it(p):
    """1 - 1e-9 is 1 in float32: refused when the model is built, not in its first training step."""
    import numpy as np
    from onto_vae_amd.vae_model import VAE
    with pytest.raises(ValueError, match="input_drop"):
        VAE(np.zeros((2, 12)), [8], [8], 4, input_drop=p)
