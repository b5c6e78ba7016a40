"""What a CTA of gated_mix leaves where one of its waits has run out (csrc/gated_give_up.h, compiled for the host): NaN in every row that it was to write, of
dx and of the residual's gradient alike, and nothing elsewhere."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("shim") / "libgive_up.so")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-o", out, "-I", os.path.join(ROOT, "permutohedral_lattice_b200", "csrc"),
                           os.path.join(ROOT, "tests", "helpers", "gated_give_up_shim.cpp")])
    lib = ctypes.CDLL(out)
    p, i, ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
    lib.give_up_as.argtypes = [p, i, p, i, ll, i, ll, ll, i]
    lib.give_up_as.restype = None
    return lib


@pytest.mark.parametrize("rows,tile,ctas", [(1, 128, 1), (128, 128, 1), (129, 128, 2), (1000, 64, 3), (1000, 128, 5), (5000, 64, 148)])
@pytest.mark.parametrize("k,n", [(64, 64), (21, 5), (1, 128)])
def test_all_rows_of_a_cta_in_all_outputs(shim, rows, tile, ctas, k, n):
    for cta in {0, ctas // 2, ctas - 1}:
        dx, dresidual = np.ones((rows + 1, k), np.float32), np.ones((rows + 1, n), np.float32)      # (a row behind the last)
        shim.give_up_as(dx.ctypes.data, k, dresidual.ctypes.data, n, rows, tile, cta, ctas, 96)
        own = (np.arange(rows + 1) // tile % ctas == cta) & (np.arange(rows + 1) < rows)
        for t in (dx, dresidual):
            assert np.isnan(t[own]).all() and (t[~own] == 1).all()


def test_an_output_that_is_not_wanted(shim):
    dx = np.ones((300, 7), np.float32)
    shim.give_up_as(dx.ctypes.data, 7, None, 5, 300, 128, 1, 2, 640)
    assert np.isnan(dx[128:256]).all() and (dx[:128] == 1).all() and (dx[256:] == 1).all()


def test_both_outputs_of_the_rows_pass_are_given_up():
    """The kernel hands over dx and, where it writes one, the residual's gradient."""
    with open(os.path.join(ROOT, "permutohedral_lattice_b200", "csrc", "gated.cuh")) as f:
        source = f.read()
    dead = source[source.index("if (b.dead) {"):]
    dead = dead[:dead.index("tensor_before_sync")]
    assert "p.out" in dead and "p.dresidual" in dead and "give_up(" in dead
