"""The gated block's gradients (include/ggemm_glu.h) against differences of its 64-bit forward form: every entry of a small block, and
of larger ones the slope along the gradient itself, which is as large as the gradient.  Wrong factors, signs and missing terms
cannot hide: on the CPU both checks are shown to reject those."""
import pytest
import torch

import glu_ref as R
from gpu_util import say

CASES = [("bf16", "silu"), ("f16", "gelu"), ("bf16", "gelu_tanh")]
GRADS = (("x", "dx"), ("wg", "dwg"), ("wu", "dwu"), ("wd", "dwd"))
SMALL = ([0, 9, 9, 23], 16, 24)      # offsets, d, f


def allowed(dtype):
    """Of the gradient's norm.  A gradient is dg^T x (dy^T h, dg Wg + du Wu): an entry of dg carries at most four roundings to the type
    (kept gate by way of the slope, kept up, itself, the result).  So the error is at most 4 unit |dg| |x|_2, and |x|_2 of R x C
    random entries is about sqrt R + sqrt C where |dg^T x| is about |dg| times the larger root: 8 units with all errors in line.  Half
    as much again for the matrices being these."""
    return 12 * R.UNIT[dtype]


def leaves(b):
    return {"x": b.x64().cpu(), **{n: getattr(b, n)[:, :c].double().cpu() for n, c in (("wg", b.d), ("wu", b.d), ("wd", b.f))}}


def loss(b, t, dy):
    """sum dy y in 64 bits"""
    tot, d, f = 0.0, b.d, b.f
    for g, r in b.spans():
        gate, u = t["x"][r] @ t["wg"][g * f:(g + 1) * f].t(), t["x"][r] @ t["wu"][g * f:(g + 1) * f].t()
        h = gate * R.act_parts(gate, b.act)[0] * u
        tot += float(((h @ t["wd"][g * d:(g + 1) * d].t()) * dy[r]).sum())
    return tot


def slope(b, t, dy, n, v, step):
    """(L(+ step v) - L(- step v)) / 2 step; third derivatives are of order one, so it is off by about step^2."""
    keep = t[n]
    t[n] = keep + step * v
    up = loss(b, t, dy)
    t[n] = keep - step * v
    down = loss(b, t, dy)
    t[n] = keep
    return (up - down) / (2 * step)


def flat(b, got, n, like):
    return got[n].double().cpu().reshape(-1, got[n].shape[-1])[:like.shape[0], :like.shape[1]]


def entrywise(b, got):
    """{leaf: |got - differences| / |differences|}, every entry by its own difference."""
    return {n: float((flat(b, got, grad, d) - d).norm() / d.norm()) for (n, grad), d in zip(GRADS, differences(b))}


def differences(b):
    t, dy = leaves(b), b.dy[:b.rows, :b.d].double().cpu()
    for n, _ in GRADS:
        d, v = torch.zeros_like(t[n]), torch.zeros_like(t[n])
        for i in range(d.numel()):
            v.view(-1)[i] = 1.0
            d.view(-1)[i] = slope(b, t, dy, n, v, 1e-4)
            v.view(-1)[i] = 0.0
        yield d


def along(b, got):
    """{leaf: |<got, v> - slope along v| / slope}, v = got / |got|: a multiple of the gradient has another slope than length."""
    t, dy, out = leaves(b), b.dy[:b.rows, :b.d].double().cpu(), {}
    for n, grad in GRADS:
        g = flat(b, got, grad, t[n])
        v = g / g.norm()
        s = slope(b, t, dy, n, v, 1e-4)
        out[n] = abs(float((g * v).sum()) - s) / abs(s)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,act", CASES + [("f16", "silu")])
def test_every_entry_of_a_small_block(dtype, act):
    say("differences", dtype, act)
    offsets, d, f = SMALL
    b = R.Block(offsets, offsets[-1], d, f, dtype, act, seed=15)
    gate, u, _ = b.forward()
    e = entrywise(b, b.backward(gate, u))
    say(e)
    assert max(e.values()) <= allowed(dtype), e


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,act", CASES)
@pytest.mark.parametrize("offsets,d,f", [([0, 30, 30, 90], 48, 72), ([0, 400, 700], 136, 264), ([0, 5000], 264, 520)])
def test_along_the_gradient(dtype, act, offsets, d, f):
    say("differences", dtype, act, offsets)
    b = R.Block(offsets, offsets[-1], d, f, dtype, act, seed=15)
    gate, u, _ = b.forward()
    e = along(b, b.backward(gate, u))
    say(e)
    assert max(e.values()) <= allowed(dtype), e


@pytest.mark.parametrize("dtype,act", CASES)
def test_the_checks_take_the_gradient_and_nothing_else(dtype, act):
    offsets, d, f = SMALL
    b = R.Block(offsets, offsets[-1], d, f, dtype, act, seed=15, device="cpu")
    fwd, most = b.forward64(), allowed(dtype)
    gate, u = (fwd[n][0].to(R.TORCH[dtype]).double() for n in ("gate", "up"))
    right = {n: v for n, (v, _) in b.backward64(gate, u).items()}
    rounded = {n: v.to(R.TORCH[dtype]) for n, v in right.items()}
    ref = dict(zip((n for n, _ in GRADS), differences(b)))

    def far(got, n):
        return float((flat(b, got, dict(GRADS)[n], ref[n]) - ref[n]).norm() / ref[n].norm())
    assert max(entrywise(b, rounded).values()) <= most and max(along(b, rounded).values()) <= most
    for factor in (-1.0, 0.0625, 0.5, 0.9, 1.1, 2.0):
        wrong = {n: factor * v for n, v in right.items()}
        assert min(along(b, wrong).values()) > most and min(far(wrong, n) for n in ref) > most, factor
    # in one group: terms and factors left out or exchanged
    p, slope_ = R.act_parts(gate, act)
    for g, r in b.spans():
        wg, wu, wd = b.w64(g)
        x, dy, a, c = b.x64()[r], b.dy[r, :b.d].double(), gate[r], u[r]
        dh = R.mm(dy, wd)
        dg, du = dh * c * slope_[r], dh * a * p[r]
        for n, v in (("wg", R.mm((dh * c * p[r]).t(), x)), ("wg", R.mm((dh * slope_[r]).t(), x)), ("wu", R.mm((dh * a).t(), x)), ("wd", R.mm(dy.t(), a * c)),
                     ("wd", R.mm(dy.t(), a * p[r])), ("x", R.mm(dg, wg)), ("x", R.mm(du, wu)), ("x", R.mm(dg, wu) + R.mm(du, wg))):
            wrong = {k: t.clone() for k, t in right.items()}
            wrong[dict(GRADS)[n]][r if n == "x" else g] = v
            assert far(wrong, n) > most, (g, n)
