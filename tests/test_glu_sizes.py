"""Calls of the gated block with more tiles than a launch takes: refused as such, also without a workspace, and no size is given for
them (decided on the host before anything is launched; the pointers are never followed)."""
import ctypes as C

import pytest

import ggemm as G

P = 0x7f0000000000      # an address, aligned to everything


def block(rows, d, f, groups):
    return G.Glu(groups, rows, d, f, G.BF16, G.SILU, rows, P, d, None, P, P, P, d, f * d, P, f, d * f, P, P, f, P, d)


def grad(d, f, weights=True):
    w = P if weights else None
    return G.GluGrad(P, d, P, d, G.F32, 0.0, w, w, d, f * d, w, f, d * f)


ROWS = [(2 ** 29, 64, 64, 1), (2 ** 30, 40, 2 ** 18, 3), (2 ** 20, 64, 2 ** 16, 4096)]


@pytest.mark.parametrize("rows,d,f,groups", ROWS)
def test_too_many_tiles_of_rows(rows, d, f, groups):
    p, q = block(rows, d, f, groups), grad(d, f, False)
    assert G.lib().ggemm_glu_workspace(C.byref(p)) == 0
    assert G.lib().ggemm_glu_backward_workspace(C.byref(p), C.byref(q)) == 0
    for ws, size in ((None, 0), (P, 0), (P, 1 << 60)):
        assert G.lib().ggemm_glu(C.byref(p), ws, size, None) == G.GGEMM_ERR_INVALID
        assert G.lib().ggemm_glu_backward(C.byref(p), C.byref(q), ws, size, None) == G.GGEMM_ERR_INVALID


def test_too_many_tiles_of_weights():
    """3 x 4096 x 32 x 32 of 128 x 128: only where the weights' gradients are wanted."""
    p = block(64, 4096, 4096, 4096)
    assert G.lib().ggemm_glu_workspace(C.byref(p)) == 64 * 4096 * 2
    assert G.lib().ggemm_glu_backward_workspace(C.byref(p), C.byref(grad(4096, 4096, False))) == 3 * 64 * 4096 * 2
    q = grad(4096, 4096)
    assert G.lib().ggemm_glu_backward_workspace(C.byref(p), C.byref(q)) == 0
    for ws, size in ((None, 0), (P, 0), (P, 1 << 60)):
        assert G.lib().ggemm_glu_backward(C.byref(p), C.byref(q), ws, size, None) == G.GGEMM_ERR_INVALID


def test_the_largest_that_fit():
    p = block(2 ** 29 - 64, 64, 64, 1)      # 2^23 - 1 tiles
    assert G.lib().ggemm_glu_workspace(C.byref(p)) == (2 ** 29 - 64) * 64 * 2
    assert G.lib().ggemm_glu(C.byref(p), None, 0, None) == G.GGEMM_ERR_WORKSPACE
