"""Sizes at the ends of the integer types: the sizing functions and the refusals of the dense-block operators, no GPU needed (a
refusal comes before any pointer is used).  The calls run in a process of their own, so that one that ends its process fails
its own test only."""
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


@pytest.mark.parametrize("N,S,C,groups", [(TOP, 1, 8, 8), (1, TOP, 8, 8), (1, 1, TOP, 1), (TOP, TOP, TOP, 1)])
def test_group_norm_sizing_past_the_sizes_it_takes(N, S, C, groups):
    """Sizes that the entry points refuse: no workspace, nothing divided by what wrapped to 0."""
    assert call(f"L.ontovae_group_norm_act_workspace_bytes(0, {N}, {S}, {C}, {groups}, 1)") == [0]


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
