"""Workspaces and limits of the 4-bit operators and the router, as the host decides them.  Every call here is refused:
the pointers are addresses of nothing."""
import ctypes as C

import pytest

import ggemm as G

P = 0x7f0000000000


def product(**kw):
    """A product whose inner dimension is computed in parts: it needs a workspace."""
    f = dict(form=G.MX4_ROWS, groups=1, m=64, n=1024, k=16384, dtype=G.F32, alpha=1.0, beta=0.0, a=P, lda=8192, a_scales=P,
             lda_scales=512, b=P, ldb=8192, b_stride=0, b_scales=P, ldb_scales=512, b_scales_stride=0, offsets=None, c=P,
             ldc=1024, c_stride=0)
    f.update(kw)
    return G.Mx4Gemm(**f)


def test_product_workspace_refusals():
    p = product()
    size = G.lib().ggemm_mx4_gemm_workspace(C.byref(p))
    assert size > 0 and size % 16 == 0
    for ws, n, rc in ((P, size - 1, G.GGEMM_ERR_WORKSPACE), (P, 0, G.GGEMM_ERR_WORKSPACE), (None, 0, G.GGEMM_ERR_WORKSPACE),
                      (None, size, G.GGEMM_ERR_INVALID), (P + 4, size, G.GGEMM_ERR_INVALID)):
        assert G.lib().ggemm_mx4_gemm(C.byref(p), ws, n, None) == rc, (ws, n)


def test_router_token_limit():
    T = G.ROUTE_MAX_TOKENS
    assert T == 2 ** 30 and G.lib().ggemm_route_workspace(T, 1, 1) > 0 and G.lib().ggemm_route_workspace(T + 1, 1, 1) == 0
    r = G.Router(T + 1, 2, 1, 1, G.BF16, 0, 0.0, T + 1, P, 2, None, P, P, P, P, P, P, P, P, P)
    assert G.lib().ggemm_route(C.byref(r), P, 1 << 40, None) == G.GGEMM_ERR_INVALID
    assert G.lib().ggemm_route_backward(C.byref(r), P, P, P, 2, None) == G.GGEMM_ERR_INVALID


@pytest.mark.parametrize("form", [G.MX4_ROWS, G.MX4_INNER])
@pytest.mark.parametrize("groups,m", [(1, 64), (1, 256), (2, 100)])
def test_product_workspace_by_sizes(form, groups, m):
    """The same before the operands and the offsets exist as with them."""
    kw = dict(form=form, groups=groups, m=m, b_stride=8192 * 1024, b_scales_stride=512 * 1024, c_stride=m * 1024)
    full = product(offsets=P, **kw)
    none = product(a=None, a_scales=None, b=None, b_scales=None, c=None, offsets=None, **kw)
    size = G.lib().ggemm_mx4_gemm_workspace(C.byref(full))
    assert size > 0 and G.lib().ggemm_mx4_gemm_workspace(C.byref(none)) == size
    if groups == 1:
        assert G.lib().ggemm_mx4_gemm_workspace(C.byref(product(**kw))) == size      # one group without offsets
    assert G.lib().ggemm_mx4_gemm(C.byref(none), P, size, None) == G.GGEMM_ERR_INVALID
    assert G.lib().ggemm_mx4_gemm(C.byref(full), P, size - 1, None) == G.GGEMM_ERR_WORKSPACE
    for bad in (dict(lda=16), dict(ldb=8184), dict(lda_scales=511), dict(ldc=1023), dict(dtype=9), dict(k=-1), dict(form=2)):
        assert G.lib().ggemm_mx4_gemm_workspace(C.byref(product(**{**kw, **bad}))) == 0, bad


def quant(**kw):
    f = dict(rows=4, cols=64, dtype=G.BF16, x_rows=4, x=P, ld=64, index=P, codes=P, ld_codes=32, scales=P, ld_scales=4)
    f.update(kw)
    return G.lib().ggemm_mx4_quantize(C.byref(G.Mx4Quant(**f)), None)


def test_quantise_without_a_matrix():
    """x may be NULL only where an index picks from no rows."""
    assert quant(x=None) == quant(x=None, index=None, x_rows=0) == quant(x=None, x_rows=1) == G.GGEMM_ERR_INVALID
    assert quant(x=None, x_rows=0, ld=63) == quant(x=None, x_rows=0, codes=None) == G.GGEMM_ERR_INVALID


def test_quantised_row_limit():
    """One column more than a quantised row can have, along the rows, down the columns and back to values."""
    n = G.MX4_MAX_COLS + 1
    long = dict(ld_codes=2 ** 25, ld_scales=2 ** 21)
    assert G.MX4_MAX_COLS == 2 ** 25
    assert quant(cols=n, ld=n, **long) == G.GGEMM_ERR_INVALID
    assert quant(rows=n, codes_t=P, scales_t=P, ld_codes_t=2 ** 25, ld_scales_t=2 ** 21) == G.GGEMM_ERR_INVALID
    d = G.Mx4Dequant(4, n, G.BF16, P, 2 ** 25, P, 2 ** 21, P, n)
    assert G.lib().ggemm_mx4_dequantize(C.byref(d), None) == G.GGEMM_ERR_INVALID
