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
