"""The 4-bit expert layer (coding-basic-hw-2_amd/apps/moe_mx4.py) end to end: products within the bound of a 32-bit
sum, the layer near its 64-bit form, gradients that agree with the 64-bit layer's, a loss that falls."""
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from gpu_util import say

APPS = Path(__file__).resolve().parents[1] / "coding-basic-hw-2_amd" / "apps"
sys.path.insert(0, str(APPS))
import moe_mx4 as M   # noqa: E402

pytestmark = pytest.mark.gpu


def _exact(lay):
    """The same layer in 64 bits from the unquantised weights, the routing taken over: (out, gradients)."""
    a = lay.a
    leaf = lambda t: t.double().cpu().requires_grad_(True)   # noqa: E731
    x, W1, W2, Wr = leaf(lay.x), leaf(lay.W1), leaf(lay.W2), leaf(lay.Wr)
    ids = lay.ids.cpu().long()
    logits = x @ Wr
    gates = torch.softmax(logits.gather(1, ids), 1)
    out = torch.zeros(a.tokens, a.d_model, dtype=torch.float64)
    W1e, W2e = W1.view(a.experts, a.d_ff, a.d_model), W2.view(a.experts, a.d_model, a.d_ff)
    for j in range(a.topk):
        for e in range(a.experts):
            at = (ids[:, j] == e).nonzero()[:, 0]
            if len(at):
                y = torch.tanh(x[at] @ W1e[e].t()) @ W2e[e].t()
                out = out.index_add(0, at, y * gates[at, j:j + 1])
    f = lay.counts.cpu().double() / (a.topk * a.tokens)
    balance = a.balance * a.experts * (f * torch.softmax(logits, 1).mean(0)).sum()
    loss = ((out - lay.target.double().cpu()) ** 2).mean() / 2 + balance
    loss.backward()
    return out.detach(), dict(gx=x.grad, gW1=W1.grad, gW2=W2.grad, gWr=Wr.grad), float(balance.detach())


def _cosine(a, b):
    a, b = a.double().cpu().reshape(-1), b.reshape(-1)
    return float(a @ b / (a.norm() * b.norm()))


def test_training_step_against_64_bits():
    """4-bit operands carry relative errors of about a tenth per value, independent across values: a product's
    relative error is about 0.15, the layer's two in a row and its gradients' up to four 0.3, cosines above
    1 / sqrt(1 + 0.3^2) = 0.957; the router's parts are 32-bit but for the gates' gradient, which sees the outputs'."""
    a = M.parse_args(["--tokens", "300", "--experts", "5", "--topk", "2", "--d-model", "128", "--d-ff", "256", "--seed", "3"])
    lay = M.Layer(a, torch)
    say("moe_mx4 step")
    lay.forward()
    lay.backward()
    assert lay.product_error() <= 1.0
    out, grads, balance = _exact(lay)
    assert abs(float(lay.balance) - balance) <= 1e-4 * balance
    assert _cosine(lay.out, out) > 0.95
    for n in ("gx", "gW1", "gW2", "gWr"):
        c = _cosine(getattr(lay, n), grads[n])
        say(n, c)
        assert c > 0.9, (n, c)


def test_training_reduces_the_loss():
    say("moe_mx4 train")
    rec = M.main(["--tokens", "512", "--experts", "6", "--topk", "2", "--d-model", "128", "--d-ff", "256", "--steps", "12",
                  "--lr", "1.0"])
    assert rec["product_error_over_bound"] <= 1.0
    assert rec["loss"][-1] < 0.97 * rec["loss"][0] and np.isfinite(rec["loss"]).all()


@pytest.mark.parametrize("tokens", [1, 37])
def test_serving(tokens):
    say("moe_mx4 serve", tokens)
    rec = M.main(["--tokens", str(tokens), "--experts", "16", "--topk", "4", "--d-model", "256", "--d-ff", "512", "--steps", "2", "--serve"])
    assert rec["product_error_over_bound"] <= 1.0 and rec["mode"] == "serve"
