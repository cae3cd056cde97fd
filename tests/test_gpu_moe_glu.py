"""The gated expert layer (coding-basic-hw-2_amd/apps/moe_glu.py) end to end: router, dispatch, block, combine and every gradient
against the layer in 64 bits, training in bf16 and serving in 8-bit integers."""
import sys
from pathlib import Path

import pytest
import torch

from gpu_util import say

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "coding-basic-hw-2_amd" / "apps"))
import moe_glu as M   # noqa: E402

pytestmark = pytest.mark.gpu

SIZES = ["--tokens", "300", "--experts", "5", "--topk", "2", "--d-model", "128", "--d-ff", "272", "--seed", "3"]


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_training_step_against_64_bits(act):
    """bf16 values are off by 2^-8 at most, 2^-8 / sqrt 3 at root mean square, at random.  The output takes six such roundings in a row
    (weights three, h, y; x is given in bf16) and the gradients at most as many again (dy, kept gate and up, dh's factors, dx): twelve
    in squares, sqrt(12) 2^-8 / sqrt 3 = 2^-7 of the norm.  Twice that is allowed."""
    say("moe_glu step", act)
    lay = M.Layer(M.parse_args([*SIZES, "--act", act]), torch)
    lay.forward()
    lay.backward()
    out, balance, leaf = lay.exact()
    assert abs(float(lay.balance) - float(balance.detach())) <= 1e-4 * float(balance.detach())
    loss = ((out - lay.target.double()) ** 2).mean() / 2 + balance
    loss.backward()
    got = {"x": lay.gx, "Wr": lay.gWr, "Wg": lay.gWg, "Wu": lay.gWu, "Wd": lay.gWd}
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())   # noqa: E731
    assert rel(lay.out, out.detach()) < 2.0 ** -6
    for n, t in leaf.items():
        r = rel(got[n], t.grad)
        say(n, r)
        assert r < 2.0 ** -6, (n, r)


def test_serving_against_64_bits():
    """8-bit rounding is uniform within half a step of max / 127; a row's maximum is about 3.5 deviations: 3.5 / 254 / sqrt 3 = 0.008 of each
    operand.  Five quantised operands (x, three weights, h; the pair's product doubles two of them): below 0.008 sqrt 8 = 0.023."""
    say("moe_glu serve")
    for tokens in (1, 37, 300):
        rec = M.main(["--tokens", str(tokens), "--experts", "16", "--topk", "4", "--d-model", "256", "--d-ff", "512", "--steps", "2", "--serve"])
        assert rec["relative_error"] < 0.03 and rec["mode"] == "serve"


def test_command_runs():
    say("moe_glu train")
    rec = M.main([*SIZES, "--steps", "2"])
    assert rec["relative_error"] < 2.0 ** -6 and len(rec["loss"]) == 3 and rec["mode"] == "train"
