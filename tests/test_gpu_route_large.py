"""The router on calls large enough for the paths that small ones do not take, against references on the GPU."""
import ctypes as C

import pytest
import torch

import ggemm as G
import mx4_gpu_ref as M
import mx4_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def test_rows_and_lanes_past_31_bits():
    """216e6 tokens to all 8 of 8 experts: 1.728e9 rows, and 4.32e8 lanes that look for rows after the last one.  Every
    expert gets every token, so a pair's row is expert tokens + token.  The sums of probabilities run over 1.69e6
    workgroups, 64 chains of 26368 and each workgroup's 128 tokens: relative error below 27000 2^-24."""
    T, E = 216_000_000, 8
    say("route past 31 bits")
    x = torch.empty(T, E, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    step = 2 ** 25
    for t in range(0, T, step):
        x[t:t + step] = torch.randn(min(step, T - t), E, device="cuda", generator=gen)
    _, o, _ = R.gpu_route(x, None, E, 1, False, 0.5, max_rows=T * E + 9)
    torch.cuda.synchronize()
    say("route past 31 bits: compared")
    assert o["counts"].tolist() == [T] * E and o["offsets"].tolist() == [e * T for e in range(E + 1)] and int(o["used"]) == T
    assert bool((o["order"][T * E:] == -1).all())
    tol, probs = 27000 * 2.0 ** -24, torch.zeros(E, dtype=torch.float64, device="cuda")
    for t in range(0, T, step):
        v = x[t:t + step].float()
        top, ids = torch.sort(v, dim=1, descending=True, stable=True)
        assert torch.equal(o["ids"][t:t + step], ids.int())
        tok = torch.arange(t, t + v.shape[0], device="cuda")
        assert torch.equal(o["pos"][t:t + step], (ids * T + tok[:, None]).int())
        for e in range(E):
            assert torch.equal(o["order"][e * T + t:e * T + t + v.shape[0]], tok.int())
        del ids, tok
        p = torch.softmax(top.double(), 1)
        assert bool(((o["gates"][t:t + step] - p).abs() <= 2e-5 * p).all())
        probs += torch.softmax(v.double(), 1).sum(0)
        del p, top, v
    probs /= T
    assert bool(((o["probs"] - probs).abs() <= tol * probs).all())
    assert abs(float(o["loss"]) - 0.5) <= 2 * tol * 0.5       # every f is 1 / 8, and the probabilities sum to 1


def test_order_of_2_31_rows():
    """An order with the most entries it can have, by the one-workgroup form and the others."""
    for T in (3, 100, 70000):
        say(f"route order of 2^31 - 1 rows, {T} tokens")
        x = torch.zeros(T, 2, device="cuda")
        _, o, _ = R.gpu_route(x, None, 1, 1, True, 0.5, max_rows=2 ** 31 - 1)
        torch.cuda.synchronize()
        assert torch.equal(o["order"][:T].long(), torch.arange(T, device="cuda"))
        for i in range(T, 2 ** 31 - 1, 2 ** 28):
            assert bool((o["order"][i:i + 2 ** 28] == -1).all())


def test_most_tokens():
    """2^30 tokens, the most there can be: 2^31 lanes in the last launch.  Logits are one of two rows, so the choice, the
    rows and the gradient of the balance loss follow from which one a token has."""
    T, E = G.ROUTE_MAX_TOKENS, 2
    say("route 2^30 tokens")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(6)
    ids = torch.empty(T, dtype=torch.bool, device="cuda")
    x = torch.empty(T, E, dtype=torch.bfloat16, device="cuda")
    step = 2 ** 27
    for t in range(0, T, step):
        ids[t:t + step] = torch.rand(step, device="cuda", generator=gen) < 0.3
        x[t:t + step, 0], x[t:t + step, 1] = 0.0, ids[t:t + step] * 2.0 - 1.0
    coef = 1e9          # the gradient goes with 1 / T
    r, o, _ = R.gpu_route(x, None, 1, 32, False, coef)
    d = torch.full((T, E), 9.0, dtype=torch.bfloat16, device="cuda")
    one = torch.ones(1, device="cuda")
    assert G.lib().ggemm_route_backward(C.byref(r), None, one.data_ptr(), d.data_ptr(), E, R.stream()) == G.GGEMM_OK
    torch.cuda.synchronize()
    say("route 2^30 tokens: compared")
    n1 = int(ids.sum())
    counts = [T - n1, n1]
    first = R.up(T - n1, 32)
    assert o["counts"].tolist() == counts and o["offsets"].tolist() == [0, first, first + R.up(n1, 32)]
    seen = [0, 0]
    s = [coef * E * c / T ** 2 for c in counts]
    p = torch.softmax(torch.tensor([[0.0, -1.0], [0.0, 1.0]], dtype=torch.float64), 1)
    grad = (p * (torch.tensor(s) - (p * torch.tensor(s)).sum(1, keepdim=True))).cuda()
    for t in range(0, T, step):
        on = ids[t:t + step]
        assert torch.equal(o["ids"][t:t + step, 0], on.int())
        for e, at in ((0, 0), (1, first)):
            tok = torch.nonzero((on == bool(e)))[:, 0]
            rows = torch.arange(at + seen[e], at + seen[e] + len(tok), device="cuda", dtype=torch.int32)
            assert torch.equal(o["pos"][t + tok, 0], rows)
            assert torch.equal(o["order"][at + seen[e]:at + seen[e] + len(tok)], (t + tok).int())
            seen[e] += len(tok)
        want = torch.where(on[:, None], grad[1], grad[0])
        # the formula's terms are below 2 |s|; one rounding to 16 bits
        assert bool(((d[t:t + step].double() - want).abs() <= 1e-4 * max(s) + R.UNIT["bf16"] * want.abs()).all())
    assert bool((o["order"][T - n1:first] == -1).all()) and bool((o["order"][first + n1:] == -1).all())


def _case(T, E, dtype, seed, masked=0.1, barred=0.05):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.randn(T, E, device="cuda", generator=gen) * 2
    x[torch.rand(T, E, device="cuda", generator=gen) < barred] = -torch.inf
    mask = (torch.rand(T, device="cuda", generator=gen) >= masked).to(torch.uint8) if masked else None
    return x.to(R.TORCH[dtype]), mask, gen


# Sums of probabilities: at most 128 tokens in 4 or more chains, 4 to 64 partial sums, 9 workgroups a chain and 64 chains:
# 109 additions of positive terms, 109 2^-24 < 7e-6, beside the entries' own 9e-6; together below the 2e-5 that the
# smaller calls have.
REL = 2e-5


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k,align,renorm", [(70001, 200, 8, 32, True), (66000, 1000, 10, 1, False), (90000, 5, 2, 16, False),
                                                (131072, 64, 6, 128, True), (33001, 129, 3, 1, True), (68000, 24, 12, 4, False)])
def test_forward_long_spans(dtype, T, E, k, align, renorm):
    """Spans of 64 and 128 tokens, with tokens left out and experts barred; choices, ranks and order exactly."""
    say(f"route long spans {dtype} {T} {E} {k}")
    x, mask, _ = _case(T, E, dtype, T + E)
    w = M.route(x, mask, k, align, renorm, 0.01)
    _, o, _ = R.gpu_route(x, mask, k, align, renorm, 0.01)
    for n in ("ids", "counts", "offsets", "pos", "order"):
        assert torch.equal(o[n].long(), w[n]), n
    assert int(o["used"]) == w["used"]
    for n in ("gates", "probs"):
        assert bool(((o[n] - w[n]).abs() <= REL * w[n] + 1e-30).all()), n
    assert abs(float(o["loss"]) - w["loss"]) <= 2 * REL * w["loss"]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k", [(70000, 24, 3), (140001, 7, 2), (40000, 200, 8), (9001, 700, 20), (70, 32, 20), (50, 33, 33), (17, 8, 8),
                                   (33000, 60, 17), (300, 1024, 64)])
def test_backward_long_and_many_places(dtype, renorm, T, E, k):
    """More tokens than the grid covers at once, and more places than a token has lanes."""
    say(f"route backward long {dtype} {T} {E} {k} {renorm}")
    x, mask, gen = _case(T, E, dtype, T + E + k)
    w = M.route(x, mask, k, 1, renorm, 0.3)
    r, o, _ = R.gpu_route(x, mask, k, 1, renorm, 0.3)
    assert torch.equal(o["ids"].long(), w["ids"])
    dg, dl = torch.randn(T, k, device="cuda", generator=gen), torch.full((1,), 1.75, device="cuda")
    for gates, loss in ((True, True), (True, False), (False, True)):
        grad, mag = M.route_gradient(w, k, renorm, 0.3, dg.double() * gates, 1.75 * loss)
        out = torch.full((T, E + 1), 9.0, dtype=R.TORCH[dtype], device="cuda")
        assert G.lib().ggemm_route_backward(C.byref(r), dg.data_ptr() if gates else None, dl.data_ptr() if loss else None,
                                            out.data_ptr(), E + 1, R.stream()) == G.GGEMM_OK
        got = out[:, :E].double()
        assert bool(((got - grad).abs() <= 3 * REL * mag + R.UNIT[dtype] * grad.abs() + R.TINY[dtype]).all()), (gates, loss)
        assert bool((got[x == -torch.inf] == 0).all()) and bool((got[~w["on"]] == 0).all()) and bool((out[:, E] == 9.0).all())
