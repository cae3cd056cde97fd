"""Gradients of weights with few tiles and many rows (include/ggemm_glu.h): sums over thousands of rows in one tile."""
import pytest
import torch

import glu_ref as R
from gpu_util import say
from test_gpu_glu import check_backward, kept

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offsets,d,f", [([0, 16384], 256, 256), ([0, 16384], 128, 128), ([0, 16383], 64, 40), ([0, 1, 1, 12001], 129, 136)])
@pytest.mark.parametrize("dw_dtype,beta", [("f32", 1.0), ("bf16", 0.0)])
def test_many_rows_of_few_tiles(offsets, d, f, dw_dtype, beta):
    say("deep", offsets, d, f, dw_dtype, beta)
    b = R.Block(offsets, offsets[-1], d, f, "bf16", "gelu", seed=23)
    gate, u = kept(b)
    check_backward(b, gate, u, dw_dtype=dw_dtype, beta=beta)


@pytest.mark.parametrize("groups,d,f", [(64, 100, 300), (40, 136, 264), (20, 520, 1032)])
def test_many_groups_whose_edges_waste_large_tiles(groups, d, f):
    say("edges", groups, d, f)
    b = R.Block([9 * g for g in range(groups)] + [9 * groups + 200], 9 * groups + 200, d, f, "bf16", "silu", seed=25)
    gate, u = kept(b)
    for dw_dtype, beta in (("bf16", 0.0), ("f32", -1.0)):
        check_backward(b, gate, u, dw_dtype=dw_dtype, beta=beta)


def test_deep_sums_of_picked_rows():
    say("deep, picked")
    rows, d, f = 16384, 136, 72
    gen = torch.Generator()
    gen.manual_seed(2)
    index = torch.randint(-500, 6000, (rows,), generator=gen).clamp(min=-1).numpy()
    b = R.Block([0, 64, rows], rows, d, f, "f16", "silu", index, 6000, seed=24)
    b.dy *= 0.0625       # sums of f16 results within its range
    gate, u = kept(b)
    check_backward(b, gate, u, dw_dtype="f32")
