"""The router on the GPU against a 64-bit reference: choices, ranks, counts and order exactly, gates, sums, loss
and gradients within bounds of 32-bit arithmetic."""
import ctypes as C

import numpy as np
import pytest
import torch

import ggemm as G
import mx4_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu

# Relative error of a softmax entry in 32 bits with |x - max| <= 40: the exponent's argument (x - max) log2 e
# carries two roundings, 58 * 2^-23 * ln 2 < 5e-6; sums of at most 1024 terms in trees and chains of at most
# 32 add 3e-6, the divisions and products below 1e-6.
REL = 2e-5


def _logits(rng, T, E, dtype, ties=False, barred=0.0):
    x = rng.standard_normal((T, E)) * 2
    if ties:
        x = np.round(x)
        x[rng.random((T, E)) < 0.1] = -0.0
    t = torch.from_numpy(x.astype(np.float32)).to(R.TORCH[dtype])
    if barred:
        t[torch.from_numpy(rng.random((T, E)) < barred)] = -float("inf")
    return t


def _compare(o, w, what):
    for n in ("ids", "pos", "counts", "offsets", "order"):
        assert np.array_equal(o[n].cpu().numpy(), w[n]), (what, n)
    assert int(o["used"]) == w["used"], what
    for n in ("gates", "probs"):
        g = o[n].cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(g), np.isnan(w[n])), (what, n)
        f = ~np.isnan(w[n])
        assert (np.abs(g - w[n])[f] <= REL * np.abs(w[n])[f] + 1e-30).all(), (what, n)
    l = float(o["loss"])
    assert (np.isnan(l) and np.isnan(w["loss"])) or abs(l - w["loss"]) <= 2 * REL * abs(w["loss"]), (what, l, w["loss"])


CASES = [  # tokens, experts, topk, align
    (1, 1, 1, 1), (1, 8, 2, 1), (1, 64, 8, 1), (3, 7, 7, 4), (64, 16, 2, 32), (65, 17, 3, 1), (200, 32, 4, 128), (130, 33, 33, 2),
    (257, 64, 8, 1), (300, 65, 5, 16), (129, 128, 6, 1), (513, 200, 8, 32), (100, 256, 8, 1), (70, 511, 10, 8), (90, 1024, 64, 1024),
    (1000, 60, 4, 1),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k,align", CASES)
def test_forward(dtype, T, E, k, align):
    rng = np.random.default_rng(T + 7 * E + k)
    for renorm, ties, masked, barred in ((True, False, False, 0.0), (False, True, True, 0.2)):
        say(f"route {dtype} {T} {E} {k} {align} {renorm}")
        x = _logits(rng, T, E, dtype, ties, barred)
        mask = (rng.random(T) < 0.7).astype(np.uint8) if masked else None
        w = R.route(x.double().numpy(), mask, k, align, renorm, 0.01)
        _, o, _ = R.gpu_route(x.cuda(), R.dev(mask) if masked else None, k, align, renorm, 0.01)
        _compare(o, w, (dtype, T, E, k, align, renorm))


def test_forward_many_tokens():
    """More tokens than one span: long starting ranks and sums over many workgroups."""
    for T, E, k in ((5000, 12, 2), (33000, 16, 2)):
        say(f"route many {T}")
        rng = np.random.default_rng(T)
        x = _logits(rng, T, E, "bf16")
        w = R.route(x.double().numpy(), None, k, 32, True, 1.0)
        _, o, _ = R.gpu_route(x.cuda(), None, k, 32, True, 1.0)
        _compare(o, w, T)


def test_odd_rows():
    """All barred, one expert left, NaN, +Inf, the type's lowest value, NaN in rows left out."""
    say("route odd rows")
    E, k = 20, 3
    x = np.random.default_rng(1).standard_normal((10, E))
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, 13] = 0.5
    x[2, 5] = np.nan
    x[3, 7] = np.inf
    x[4] = np.finfo(np.float32).min
    x[5, 3:] = np.finfo(np.float32).min
    x[6] = 0.0
    x[6, ::2] = -0.0
    x[7] = np.nan
    x[8] = np.inf
    mask = np.ones(10, dtype=np.uint8)
    t = torch.from_numpy(x.astype(np.float32))
    w = R.route(t.double().numpy(), mask, k, 4, True, 0.5)
    _, o, _ = R.gpu_route(t.cuda(), R.dev(mask), k, 4, True, 0.5)
    _compare(o, w, "odd")
    mask[[2, 3, 7, 8]] = 0          # the NaN rows left out: everything finite
    w = R.route(t.double().numpy(), mask, k, 4, False, 0.5)
    assert np.isfinite(w["loss"])
    _, o, _ = R.gpu_route(t.cuda(), R.dev(mask), k, 4, False, 0.5)
    _compare(o, w, "odd, left out")
    mask[:] = 0                     # nothing left
    w = R.route(t.double().numpy(), mask, k, 4, False, 0.5)
    r, o, _ = R.gpu_route(t.cuda(), R.dev(mask), k, 4, False, 0.5)
    _compare(o, w, "all left out")
    d = torch.full((10, E), 3.0, device="cuda")
    one = torch.ones(10 * k, device="cuda")
    assert G.lib().ggemm_route_backward(C.byref(r), one.data_ptr(), one.data_ptr(), d.data_ptr(), E, R.stream()) == 0
    torch.cuda.synchronize()
    assert (d == 0).all()


def test_no_tokens():
    say("route no tokens")
    _, o, _ = R.gpu_route(torch.zeros(0, 12, device="cuda"), None, 2, 8, True, 0.5, max_rows=100)
    assert (o["counts"] == 0).all() and (o["offsets"] == 0).all() and (o["order"] == -1).all()
    assert int(o["used"]) == 0 and float(o["loss"]) == 0.0 and (o["probs"] == 0).all()


def test_strided_logits_same_bits_twice():
    say("route strided")
    rng = np.random.default_rng(2)
    base = _logits(rng, 3000, 75, "f32")
    x = base.cuda()[:, 3:70]
    w = R.route(base.double().numpy()[:, 3:70], None, 4, 1, True, 0.1)
    runs = [R.gpu_route(x, None, 4, 1, True, 0.1)[1] for _ in range(3)]
    _compare(runs[0], w, "strided")
    for o in runs[1:]:
        for n in o:
            assert torch.equal(o[n], runs[0][n]), n


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 3), (5, 17, 4), (70, 64, 8), (33, 130, 5), (40, 256, 8), (9, 700, 20), (2100, 24, 3)])
def test_backward_formula(dtype, T, E, k):
    rng = np.random.default_rng(T * 3 + E)
    for renorm in (True, False):
        say(f"route backward {dtype} {T} {E} {k} {renorm}")
        x = _logits(rng, T, E, dtype, barred=0.15)
        mask = (rng.random(T) < 0.9).astype(np.uint8)
        w = R.route(x.double().numpy(), mask, k, 1, renorm, 0.3)
        r, o, _ = R.gpu_route(x.cuda(), (md := R.dev(mask)), k, 1, renorm, 0.3)
        xd = x.cuda()
        r.logits = xd.data_ptr()
        dg, dl = rng.standard_normal((T, k)), 1.7
        dgd, dld = R.dev(dg.astype(np.float32)), torch.full((1,), dl, device="cuda")
        dg = dg.astype(np.float32).astype(np.float64)
        dl = float(np.float32(dl))
        for gates, loss in ((True, True), (True, False), (False, True), (False, False)):
            grad, mag = R.route_gradient(w, k, renorm, 0.3, dg if gates else 0 * dg, dl if loss else 0.0)
            out = torch.full((T, E + 3), 9.0, dtype=R.TORCH[dtype], device="cuda")
            rc = G.lib().ggemm_route_backward(C.byref(r), dgd.data_ptr() if gates else None, dld.data_ptr() if loss else None,
                                              out.data_ptr(), E + 3, R.stream())
            assert rc == G.GGEMM_OK
            got = out.double().cpu().numpy()
            tol = 3 * REL * mag + R.UNIT[dtype] * np.abs(grad) + R.TINY[dtype]
            assert (np.abs(got[:, :E] - grad) <= tol).all(), (dtype, T, E, k, renorm, gates, loss)
            assert (got[:, E:] == 9.0).all()
            assert (got[:, :E][x.double().numpy() == -np.inf] == 0).all() and (got[:, :E][mask == 0] == 0).all()


@pytest.mark.parametrize("renorm", [True, False])
def test_backward_differences(renorm):
    """Against central differences of the 64-bit objective.  Step 1e-5: truncation about 1e-10 of the third
    derivative, rounding 1e-16 / 1e-5 of the objective's size, both far below the 32-bit gradient's error."""
    say(f"route differences {renorm}")
    rng = np.random.default_rng(12)
    T, E, k = 6, 11, 3
    x = _logits(rng, T, E, "f32")
    w = R.route(x.double().numpy(), None, k, 1, renorm, 0.2)
    dg, dl = rng.standard_normal((T, k)).astype(np.float32), 0.7
    xd, dgd, dld = x.cuda(), R.dev(dg), torch.full((1,), dl, device="cuda")
    r, o, _ = R.gpu_route(xd, None, k, 1, renorm, 0.2)
    out = torch.zeros(T, E, device="cuda")
    assert G.lib().ggemm_route_backward(C.byref(r), dgd.data_ptr(), dld.data_ptr(), out.data_ptr(), E, R.stream()) == 0
    got, h = out.double().cpu().numpy(), 1e-5
    for t in range(T):
        for e in range(E):
            a, b = x.double().numpy(), x.double().numpy()
            a[t, e] += h
            b[t, e] -= h
            d = (R.route_objective(a, w, k, renorm, 0.2, dg.astype(np.float64), dl) -
                 R.route_objective(b, w, k, renorm, 0.2, dg.astype(np.float64), dl)) / (2 * h)
            assert abs(d - got[t, e]) <= 1e-4 * np.abs(dg[t]).max(), (t, e, d, got[t, e])


def test_graph_replay():
    """Captured once, replayed on new logits; each replay against the reference."""
    say("route graph")
    rng = np.random.default_rng(13)
    T, E, k = 700, 40, 4
    x = torch.zeros(T, E, device="cuda")
    r, o, ws = R.gpu_route(x, None, k, 8, True, 0.1)
    dg, out = torch.randn(T, k, device="cuda"), torch.zeros(T, E, device="cuda")
    dl = torch.ones(1, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        assert G.lib().ggemm_route(C.byref(r), ws.data_ptr(), ws.numel(), side.cuda_stream) == 0
        assert G.lib().ggemm_route_backward(C.byref(r), dg.data_ptr(), dl.data_ptr(), out.data_ptr(), E, side.cuda_stream) == 0
    for i in range(3):
        v = _logits(rng, T, E, "f32")
        x.copy_(v.cuda())
        for t in o.values():
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        w = R.route(v.double().numpy(), None, k, 8, True, 0.1)
        _compare(o, w, ("replay", i))
        grad, mag = R.route_gradient(w, k, True, 0.1, dg.double().cpu().numpy(), 1.0)
        assert (np.abs(out.double().cpu().numpy() - grad) <= 3 * REL * mag + 1e-30).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_logits_far_from_zero(dtype):
    """Softmax depends on differences only: rows of large logits that differ by a few units or of the type's spacings, alone
    and beside ordinary rows; gates as they are, sums and gradients.  Differences stay exact in 32 bits."""
    say(f"route far from zero {dtype}")
    rng = np.random.default_rng(8)
    E, k = 40, 4
    centres = [20.0, -40.0, 90.0, 1e3, -1e3, 3e4] + ([] if dtype == "f16" else [1e6, 1e10, -1e10, 1e25, -3e29, 2e30])
    x = rng.standard_normal((40 * len(centres), E)) * 2
    for i, c in enumerate(centres):
        spacing = 2.0 ** np.floor(np.log2(abs(c))) * 2 * R.UNIT[dtype]
        rows = x[40 * i:40 * i + 30]
        rows[:] = c + (np.round(rows / spacing) if spacing < 0.5 else np.round(rows)) * spacing
    x = torch.from_numpy(x).to(R.TORCH[dtype])
    T = x.shape[0]
    dg, dl = rng.standard_normal((T, k)).astype(np.float32), np.float32(0.6)
    xd, dgd, dld = x.cuda(), R.dev(dg), torch.full((1,), float(dl), device="cuda")
    for renorm in (False, True):
        w = R.route(x.double().numpy(), None, k, 1, renorm, 0.3)
        r, o, _ = R.gpu_route(xd, None, k, 1, renorm, 0.3)
        _compare(o, w, (dtype, renorm))
        grad, mag = R.route_gradient(w, k, renorm, 0.3, dg.astype(np.float64), float(dl))
        out = torch.full((T, E), 9.0, dtype=R.TORCH[dtype], device="cuda")
        assert G.lib().ggemm_route_backward(C.byref(r), dgd.data_ptr(), dld.data_ptr(), out.data_ptr(), E, R.stream()) == 0
        tol = 3 * REL * mag + R.UNIT[dtype] * np.abs(grad) + R.TINY[dtype]
        assert (np.abs(out.double().cpu().numpy() - grad) <= tol).all(), (dtype, renorm)
