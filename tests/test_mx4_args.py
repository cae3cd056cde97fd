"""What the 4-bit operators and the router refuse, and what they accept without work: all decided on the
host before anything is launched (no GPU here; the pointers are never followed)."""
import ctypes as C
import sys
from pathlib import Path

import pytest

import ggemm as G

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "coding-basic-hw-2_amd" / "apps"))
import moe_mx4   # noqa: E402

P = 0x7f0000000000      # an address, aligned to everything


def quant(**kw):
    f = dict(rows=4, cols=64, dtype=G.BF16, x_rows=4, x=P, ld=64, index=None, codes=P, ld_codes=32, scales=P, ld_scales=4,
             codes_t=None, ld_codes_t=0, scales_t=None, ld_scales_t=0)
    f.update(kw)
    return G.lib().ggemm_mx4_quantize(C.byref(G.Mx4Quant(**f)), None)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(cols=-1), dict(cols=2 ** 26 + 1, ld=2 ** 27), dict(dtype=3), dict(dtype=-1), dict(x=None), dict(ld=63),
    dict(x=P + 1), dict(dtype=G.F32, x=P + 2), dict(codes=None), dict(scales=None), dict(codes=None, scales=None),
    dict(codes=P + 8), dict(scales=P + 2), dict(ld_codes=16), dict(ld_codes=40), dict(ld_scales=0), dict(ld_scales=6),
    dict(index=P, x_rows=-1), dict(index=P + 2),
    dict(codes_t=P, scales_t=None, ld_codes_t=16, ld_scales_t=4), dict(codes_t=P, scales_t=P, ld_codes_t=8, ld_scales_t=4),
    dict(codes_t=P, scales_t=P, ld_codes_t=16, ld_scales_t=2),
])
def test_quantise_refusals(bad):
    assert quant(**bad) == G.GGEMM_ERR_INVALID


def test_quantise_nothing_to_do():
    assert quant(rows=0) == G.GGEMM_OK and quant(cols=0, x=None) == G.GGEMM_OK
    assert G.lib().ggemm_mx4_quantize(None, None) == G.GGEMM_ERR_INVALID


def dequant(**kw):
    f = dict(rows=4, cols=64, dtype=G.BF16, codes=P, ld_codes=32, scales=P, ld_scales=4, y=P, ld=64)
    f.update(kw)
    return G.lib().ggemm_mx4_dequantize(C.byref(G.Mx4Dequant(**f)), None)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(cols=-1), dict(cols=2 ** 26 + 1, ld=2 ** 27), dict(dtype=5), dict(codes=None), dict(scales=None),
    dict(y=None), dict(y=P + 1), dict(ld=60), dict(codes=P + 4), dict(scales=P + 1), dict(ld_codes=30), dict(ld_scales=1),
])
def test_dequantise_refusals(bad):
    assert dequant(**bad) == G.GGEMM_ERR_INVALID


def test_dequantise_nothing_to_do():
    assert dequant(rows=0) == G.GGEMM_OK and dequant(cols=0) == G.GGEMM_OK
    assert G.lib().ggemm_mx4_dequantize(None, None) == G.GGEMM_ERR_INVALID


def gemm(ws=P, ws_bytes=1 << 40, **kw):
    f = dict(form=G.MX4_ROWS, groups=3, m=8, n=40, k=64, dtype=G.F32, alpha=1.0, beta=0.0, a=P, lda=32, a_scales=P, lda_scales=4,
             b=P, ldb=32, b_stride=32 * 40, b_scales=P, ldb_scales=4, b_scales_stride=160, offsets=P, c=P, ldc=40, c_stride=0)
    f.update(kw)
    p = G.Mx4Gemm(**f)
    return G.lib().ggemm_mx4_gemm(C.byref(p), ws, ws_bytes, None), G.lib().ggemm_mx4_gemm_workspace(C.byref(p))


@pytest.mark.parametrize("bad", [
    dict(form=2), dict(form=-1), dict(groups=0), dict(groups=G.MX4_MAX_GROUPS + 1), dict(m=-1), dict(n=-1), dict(k=-1),
    dict(dtype=7), dict(offsets=None), dict(offsets=P + 2), dict(c=None), dict(c=P + 2), dict(ldc=39), dict(a=None), dict(b=None),
    dict(a_scales=None), dict(b_scales=None), dict(a=P + 8), dict(b=P + 1), dict(a_scales=P + 2), dict(lda=24), dict(lda=16),
    dict(ldb=40), dict(lda_scales=1), dict(ldb_scales=6), dict(b_stride=8), dict(b_scales_stride=2),
    dict(form=G.MX4_INNER, c_stride=100), dict(form=G.MX4_INNER, c_stride=-400),
])
def test_gemm_refusals(bad):
    rc, size = gemm(**bad)
    assert rc == G.GGEMM_ERR_INVALID and size == 0


def test_gemm_workspace_and_empty():
    rc, size = gemm(ws_bytes=0)
    assert size % 16 == 0 and rc == (G.GGEMM_ERR_WORKSPACE if size else rc)
    assert gemm(ws=None)[0] == G.GGEMM_ERR_INVALID or size == 0
    assert gemm(m=0)[0] == G.GGEMM_OK and gemm(n=0)[0] == G.GGEMM_OK
    assert G.lib().ggemm_mx4_gemm(None, P, 1 << 30, None) == G.GGEMM_ERR_INVALID
    assert G.lib().ggemm_mx4_gemm_workspace(None) == 0


def router(call="forward", ws=P, ws_bytes=1 << 40, d_logits=P, ld_d=16, **kw):
    f = dict(tokens=10, experts=16, topk=2, row_align=4, dtype=G.F32, renormalize=1, balance_coef=0.1, max_rows=20 + 16 * 3,
             logits=P, ld=16, mask=None, ids=P, gates=P, pos=P, counts=P, offsets=P, order=P, used=P, probs=P, loss=P)
    f.update(kw)
    r = G.Router(**f)
    if call == "forward":
        return G.lib().ggemm_route(C.byref(r), ws, ws_bytes, None)
    return G.lib().ggemm_route_backward(C.byref(r), P, P, d_logits, ld_d, None)


BOTH = [dict(tokens=-1), dict(experts=0), dict(experts=1025), dict(topk=0), dict(topk=17), dict(topk=65, experts=100, ld=100, ld_d=100),
        dict(dtype=3), dict(logits=None), dict(ld=15), dict(logits=P + 2), dict(ids=None), dict(gates=None), dict(counts=None),
        dict(used=None), dict(tokens=2 ** 31 - 1)]


@pytest.mark.parametrize("bad", BOTH + [
    dict(row_align=0), dict(row_align=3), dict(row_align=2048), dict(max_rows=67), dict(pos=None), dict(offsets=None),
    dict(order=None), dict(probs=None), dict(loss=None), dict(ws=None), dict(ws=P + 4),
])
def test_route_refusals(bad):
    bad = {k: v for k, v in bad.items() if k != "ld_d"}
    assert router(**bad) == G.GGEMM_ERR_INVALID


@pytest.mark.parametrize("bad", BOTH + [dict(d_logits=None), dict(d_logits=P + 1), dict(ld_d=15)])
def test_route_backward_refusals(bad):
    assert router("backward", **bad) == G.GGEMM_ERR_INVALID


def test_route_workspace():
    size = G.lib().ggemm_route_workspace(10, 16, 2)
    assert size > 0 and size % 16 == 0
    assert router(ws_bytes=size - 1) == G.GGEMM_ERR_WORKSPACE
    assert G.lib().ggemm_route_workspace(10, 16, 17) == 0 and G.lib().ggemm_route_workspace(-1, 16, 2) == 0
    assert router("backward", tokens=0) == G.GGEMM_OK
    assert G.lib().ggemm_route(None, P, 1 << 30, None) == G.GGEMM_ERR_INVALID
    assert G.lib().ggemm_route_backward(None, P, P, P, 16, None) == G.GGEMM_ERR_INVALID


@pytest.mark.parametrize("bad", [["--tokens", "0"], ["--topk", "17"], ["--topk", "0"], ["--d-model", "100"], ["--d-ff", "64"],
                                 ["--experts", "2000"], ["--steps", "0"]])
def test_app_refuses(bad, capsys):
    with pytest.raises(SystemExit):
        moe_mx4.parse_args(bad)
    assert "error" in capsys.readouterr().err
