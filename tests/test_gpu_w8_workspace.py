"""The integer products need no workspace (include/ggemm_w8.h): every kernel gives the same bits with none as with some."""
import ctypes as C

import numpy as np
import pytest
import torch

import ggemm as G
from gpu_util import say
from test_gpu_w8 import Operands, cut, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k,groups", [(3, 40, 96, 2), (200, 136, 264, 3), (700, 513, 384, 2), (3000, 2600, 136, 2), (5, 7, 0, 1)])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_no_workspace(m, n, k, groups, act):
    say("no workspace", m, n, k, groups, act)
    o = Operands(m, m, n, k, groups, act is not None)
    off = cut(np.random.default_rng(m), m, groups)
    want = o.run(off, "bf16", act)
    c = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    t = lambda v: v.data_ptr() if v is not None else None   # noqa: E731
    p = G.W8Gemm(groups, m, n, k, G.BF16, G.ACTS[act] if act else 0, t(o.a), o.a.stride(0), t(o.sa), t(o.b), t(o.u), o.b.stride(0), n * o.b.stride(0),
                 t(o.sb), t(o.su), n, t(o.off), t(c), n)
    assert G.lib().ggemm_w8_gemm_workspace(C.byref(p)) == 0
    for ws, size in ((None, 0), (None, 4096), (8, 0)):
        c.fill_(7.0)
        assert G.lib().ggemm_w8_gemm(C.byref(p), ws, size, stream()) == G.GGEMM_OK
        torch.cuda.synchronize()
        assert torch.equal(c, want)
