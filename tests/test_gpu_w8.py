"""8-bit integer quantisation and products (include/ggemm_w8.h): quantisation bit for bit as its definition says, products
within the roundings that follow their exact sums."""
import ctypes as C

import numpy as np
import pytest
import torch

import ggemm as G
import glu_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def quantise(x, index=None, ldq=None, shift=0):
    """(q, scales) by the library; q's rows ldq apart, shifted by some bytes from an aligned address."""
    rows, cols = (x.shape[0] if index is None else len(index)), x.shape[1]
    ldq = ldq or R.up(max(cols, 1), 16)
    store = torch.full((rows * ldq + shift,), 99, dtype=torch.int8, device="cuda")
    s = torch.full((rows + 1,), 5.0, device="cuda")
    kind = {v: k for k, v in R.TORCH.items()}[x.dtype]
    p = G.W8Quant(rows, cols, G.DTYPES[kind], x.shape[0], x.data_ptr(), x.stride(0), index.data_ptr() if index is not None else None,
                  store.data_ptr() + shift, ldq, s.data_ptr())
    G.check(G.lib().ggemm_w8_quantize(C.byref(p), stream()), "ggemm_w8_quantize")
    q = store[shift:].view(rows, ldq)
    assert bool((q[:, cols:] == 99).all()) and bool((store[:shift] == 99).all()) and float(s[-1]) == 5.0
    return q[:, :cols], s[:-1]


def same(got, want):
    (q, s), (wq, ws) = got, want
    assert torch.equal(torch.nan_to_num(s, nan=-1.0), torch.nan_to_num(ws, nan=-1.0)), (s, ws)
    assert torch.equal(q, wq), (q != wq).nonzero()[:5]


def values(gen, rows, cols, dtype):
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    x *= torch.exp(3 * torch.randn(rows, 1, device="cuda", generator=gen))
    return x.to(R.TORCH[dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (5, 64), (17, 1000), (257, 33), (64, 8192), (9, 12345), (2, 131071),
                                       (4000, 520), (1000, 2049), (300, 16384), (3000, 1500), (2100, 4000), (5000, 3999)])
def test_quantise(rows, cols, dtype):
    say("quantise", rows, cols, dtype)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows + cols)
    x = values(gen, rows, cols, dtype)
    same(quantise(x), R.quantise64(x))
    wide = torch.zeros(rows, cols + 5, dtype=x.dtype, device="cuda")     # rows at any element
    wide[:, 1:cols + 1] = x
    same(quantise(wide[:, 1:cols + 1], ldq=cols + 3, shift=1), R.quantise64(x))


@pytest.mark.parametrize("rows,cols", [(20000, 4096), (9000, 8200), (70000, 1001), (300000, 250)])
def test_quantise_large(rows, cols):
    """More integers than are stored by way of the caches."""
    say("quantise large", rows, cols)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows)
    for dtype in ("f32", "bf16"):
        x = values(gen, rows, cols, dtype)
        same(quantise(x), R.quantise64(x))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantise_halves(dtype):
    """Values at and next to halves of the scale: 127 of them make the scale 1 (and other powers of two); scales that are no
    powers of two, with the 32-bit neighbours of every half."""
    say("halves", dtype)
    k = torch.arange(-126, 127, device="cuda", dtype=torch.float64) + 0.5
    for e in (-20, 0, 3) if dtype != "f16" else (-3, 0, 3):
        x = torch.cat([k, torch.tensor([127.0], device="cuda", dtype=torch.float64)]) * 2.0 ** e
        x = x[None].to(R.TORCH[dtype])
        same(quantise(x), R.quantise64(x))
    if dtype != "f32":
        return
    rng = np.random.default_rng(3)
    rows = []
    for _ in range(300):
        top = np.float32(rng.uniform(0.5, 4.0) * 2.0 ** rng.integers(-60, 60))
        s = np.float64(np.float32(np.float64(top) / 127))
        h = ((np.arange(0, 127) + 0.5) * s).astype(np.float32)
        h = np.concatenate([h, np.nextafter(h, np.float32(np.inf)), np.nextafter(h, np.float32(0))])
        rows.append(np.concatenate([[top], np.minimum(h, top) * rng.choice([-1, 1], h.shape).astype(np.float32)]))
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda()
    same(quantise(x), R.quantise64(x))


def test_quantise_edges():
    say("edges")
    f = float
    rows = [[0.0, -0.0, 0.0], [f("nan"), 1.0, 2.0], [1.0, f("inf"), 2.0], [f("-inf"), 0.0, 0.0], [2.0 ** -149, 0.0, -2.0 ** -149],
            [2.0 ** -126, 2.0 ** -127, -2.0 ** -140], [127 * 2.0 ** -126, 2.0 ** -126, 3 * 2.0 ** -127], [3.4028234e38, -3.4028234e38, 1e38],
            [1e-37, 1e-38, 5e-40], [126 * 2.0 ** -126, -125.5 * 2.0 ** -126, 0.5 * 2.0 ** -126]]
    x = torch.tensor(rows, device="cuda")
    same(quantise(x), R.quantise64(x))
    for dtype in ("bf16", "f16"):
        y = x.to(R.TORCH[dtype])
        same(quantise(y), R.quantise64(y))


def test_quantise_gathered():
    say("gather")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    for cols in (40, 5000):
        x = values(gen, 50, cols, "bf16")
        x[7] = float("nan")                                        # no index names it
        i = torch.tensor([3, -1, 49, 50, 0, 3, -2 ** 31, 2 ** 31 - 1, 8], dtype=torch.int32, device="cuda")
        ok = (i >= 0) & (i < 50)
        want = torch.where(ok[:, None], x[torch.where(ok, i, 0).long()], torch.zeros_like(x[:1]))
        same(quantise(x, i), R.quantise64(want))


def test_nothing_to_quantise():
    say("nothing")
    i = torch.full((5,), -1, dtype=torch.int32, device="cuda")
    q, s = torch.full((5, 16), 9, dtype=torch.int8, device="cuda"), torch.zeros(5, device="cuda")
    p = G.W8Quant(5, 16, G.BF16, 0, None, 16, i.data_ptr(), q.data_ptr(), 16, s.data_ptr())
    assert G.lib().ggemm_w8_quantize(C.byref(p), stream()) == G.GGEMM_OK
    assert bool((q == 0).all()) and bool((s == 2.0 ** -126).all())
    s.zero_()
    p = G.W8Quant(5, 0, G.F32, 5, None, 0, None, None, 0, s.data_ptr())
    assert G.lib().ggemm_w8_quantize(C.byref(p), stream()) == G.GGEMM_OK
    assert bool((s == 2.0 ** -126).all())


def test_dequantise():
    say("dequantise")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    for rows, cols, pad in ((1, 1, 0), (300, 4096, 0), (77, 1001, 3), (5, 131071, 1), (4000, 64, 0)):
        q = torch.randint(-128, 128, (rows, cols + pad), dtype=torch.int8, device="cuda", generator=gen)
        s = torch.exp(torch.randn(rows, device="cuda", generator=gen))
        if rows > 2:
            s[1] = float("nan")
        for dtype in ("f32", "bf16", "f16"):
            y = torch.full((rows, cols + pad), 7.0, dtype=R.TORCH[dtype], device="cuda")
            p = G.W8Dequant(rows, cols, G.DTYPES[dtype], q.data_ptr(), cols + pad, s.data_ptr(), y.data_ptr(), cols + pad)
            G.check(G.lib().ggemm_w8_dequantize(C.byref(p), stream()), "ggemm_w8_dequantize")
            want = (q[:, :cols].float() * s[:, None]).to(y.dtype)
            assert torch.equal(torch.nan_to_num(y[:, :cols], nan=-3.0), torch.nan_to_num(want, nan=-3.0))
            assert bool((y[:, cols:] == 7.0).all())


# ------------------------------------------------------------------ products

class Operands:
    def __init__(self, seed, m, n, k, groups, gated, pad=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.m, self.n, self.k, self.groups, self.pad = m, n, k, groups, pad

        def rand(rows):
            q = torch.randint(-128, 128, (max(rows, 1), R.up(max(k, 1), 16) + pad), dtype=torch.int8, device="cuda", generator=gen)
            return q, torch.exp(torch.randn(max(rows, 1), device="cuda", generator=gen)) / (5000 * max(k, 1) ** 0.5)
        self.a, self.sa = rand(m)
        self.b, self.sb = rand(groups * n)
        self.u, self.su = rand(groups * n) if gated else (None, None)

    def run(self, off, dtype="f32", act=None, ldc=None, shift=0, stream_=None):
        ldc = ldc or self.n
        store = torch.full((max(self.m, 1) * ldc + shift,), 7.0, dtype=R.TORCH[dtype], device="cuda")
        t = lambda v: v.data_ptr() if v is not None else None   # noqa: E731
        self.off = None if off is None else torch.tensor(off, dtype=torch.int32, device="cuda")
        p = G.W8Gemm(self.groups, self.m, self.n, self.k, G.DTYPES[dtype], G.ACTS[act] if act else 0, t(self.a), self.a.stride(0),
                     t(self.sa), t(self.b), t(self.u), self.b.stride(0), self.n * self.b.stride(0), t(self.sb), t(self.su), self.n,
                     t(self.off), store.data_ptr() + shift * store.element_size(), ldc)
        size = G.lib().ggemm_w8_gemm_workspace(C.byref(p))
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        ws.fill_(255)
        G.check(G.lib().ggemm_w8_gemm(C.byref(p), ws.data_ptr(), size, stream_ or stream()), "ggemm_w8_gemm")
        return store[shift:].view(max(self.m, 1), ldc)[:self.m]

    def want(self, off, act=None):
        spans = []
        for g in range(self.groups):
            lo, hi = (min(max(int(v), 0), self.m) for v in off[g:g + 2])
            if lo < hi:
                spans.append((g, slice(lo, hi)))
        k = self.k
        u = (self.u[:, :k], self.su) if act else (None, None)
        v, e = R.product64(self.a[:, :k], self.sa, self.b[:, :k], self.sb, spans, self.n, act, *u)
        cov = torch.zeros(self.m, dtype=torch.bool, device="cuda")
        for _, r in spans:
            cov[r] = True
        return v, e, cov


def check(o, off, dtype, act, ldc=None, shift=0):
    got = o.run(off, dtype, act, ldc, shift)
    v, e, cov = o.want(off, act)
    bound = e + R.UNIT[dtype] * (v.abs() + e) + R.TINY[dtype]
    bad = R.worst(got[cov][:, :o.n], v[cov], bound[cov])
    assert bad <= 1.0, (bad, o.m, o.n, o.k, o.groups, dtype, act)
    assert bool((got[~cov] == 7.0).all()) and bool((got[:, o.n:] == 7.0).all())
    return got


def cut(rng, rows, groups, empty=0.3):
    c = np.sort(rng.integers(0, rows + 1, max(groups - 1, 0)))
    for i in range(1, len(c)):
        if rng.random() < empty:
            c[i] = c[i - 1]
    return [0, *map(int, c), rows]


SHAPES = [  # m, n, k, groups
    (1, 1, 1, 1), (1, 64, 64, 1), (3, 5, 17, 1), (2, 100, 4096, 7), (16, 33, 128, 1), (17, 130, 100, 2), (30, 260, 1000, 5),
    (64, 128, 256, 1), (65, 129, 257, 1), (128, 300, 512, 9), (300, 100, 33, 3), (1000, 513, 384, 2), (700, 70, 1001, 60),
    (5000, 1500, 300, 2), (4097, 2049, 144, 1), (8, 520, 20000, 1), (40, 64, 30000, 1), (260, 260, 8200, 1), (9, 40, 64, 900),
    (9000, 1032, 640, 6), (100, 77, 131071, 1), (5, 16, 131071, 2),
]


@pytest.mark.parametrize("m,n,k,groups", SHAPES)
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_product(m, n, k, groups, act):
    say("product", m, n, k, groups, act)
    rng = np.random.default_rng(m + 3 * n + 7 * k)
    o = Operands(m + n + k, m, n, k, groups, act is not None, pad=16 * (k % 3))
    check(o, cut(rng, m, groups), "f32", act)
    check(o, cut(rng, m, groups), "bf16", act, ldc=n + 3, shift=1)


def test_result_types_and_the_last_activation():
    say("types")
    rng = np.random.default_rng(5)
    for m, n, k, groups in ((7, 40, 96, 2), (200, 136, 264, 3), (1500, 1200, 160, 2), (3000, 2600, 136, 2), (8200, 4100, 200, 3)):
        o = Operands(m, m, n, k, groups, True)
        for dtype in ("f32", "bf16", "f16"):
            for act in (None, "gelu_tanh"):
                check(o, cut(rng, m, groups), dtype, act)


def test_extreme_integers():
    """-128 throughout: the largest sums, 2^14 k."""
    say("extremes")
    for m, n, k in ((4, 40, 131071), (300, 260, 131071)):
        o = Operands(1, m, n, k, 1, False)
        o.a.fill_(-128)
        o.b.fill_(-128)
        check(o, [0, m], "f32", None)
        o.b.fill_(127)
        check(o, [0, m], "f32", None)


def test_groups_and_offsets():
    say("offsets")
    o = Operands(6, 50, 72, 80, 2, False)
    for off in ([3, 20, 44], [0, 0, 50], [50, 50, 50], [-9, 10, 60], [0, 2 ** 31 - 1, 2 ** 31 - 1], [30, 10, 40]):
        check(o, off, "f32", None)
    one = Operands(7, 50, 72, 80, 1, False)
    assert torch.equal(one.run(None), one.run([0, 50]))


def test_offsets_that_name_rows_many_times():
    """Not ascending: results of rows named twice are anybody's, but nothing outside C is touched and the call ends."""
    say("offsets over and over")
    for m, groups in ((40, 9), (2000, 300), (50000, 2001)):
        n, k = 40, 32
        o = Operands(16, m, n, k, groups, False)
        store = torch.full((m + 64, n), 7.0, device="cuda")
        off = torch.tensor([0 if g % 2 == 0 else m for g in range(groups + 1)], dtype=torch.int32, device="cuda")
        p = G.W8Gemm(groups, m, n, k, G.F32, 0, o.a.data_ptr(), o.a.stride(0), o.sa.data_ptr(), o.b.data_ptr(), None, o.b.stride(0),
                     n * o.b.stride(0), o.sb.data_ptr(), None, n, off.data_ptr(), store[32:].data_ptr(), n)
        G.check(G.lib().ggemm_w8_gemm(C.byref(p), None, 0, stream()), "ggemm_w8_gemm")
        torch.cuda.synchronize()
        assert bool((store[:32] == 7.0).all()) and bool((store[m + 32:] == 7.0).all())


def test_offsets_past_32_bits():
    """Weights of more than 4 GiB with rows in the first and the last group, and operands whose rows lie 2^23 bytes apart."""
    say("large weights")
    m, n, k, groups = 70, 8192, 8192, 72
    o = Operands(17, m, 1, k, 1, False)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    o.n, o.groups = n, groups
    o.b = torch.randint(-128, 128, (groups * n, k), dtype=torch.int8, device="cuda", generator=gen)
    o.sb = torch.exp(torch.randn(groups * n, device="cuda", generator=gen)) / 1e6
    check(o, [0] + [30] * (groups - 1) + [m], "f32", None)
    del o
    say("long rows")
    for m, n in ((300, 40), (9, 300), (300, 300)):
        o = Operands(18, m, n, 100, 1, False)
        for name, rows in (("a", m), ("b", n)):
            wide = torch.empty(rows, G.W8_MAX_LD, dtype=torch.int8, device="cuda")
            wide[:, :112] = getattr(o, name)[:, :112]
            setattr(o, name, wide)
        check(o, [0, m], "bf16", None)


def test_no_inner_dimension():
    say("k = 0")
    o = Operands(8, 20, 40, 0, 2, True)
    assert bool((o.run([0, 5, 20]) == 0).all()) and bool((o.run([0, 5, 20], "bf16", "silu") == 0).all())


def test_nan_rows():
    """A row that could not be quantised (NaN scale) is NaN as a whole, others are not."""
    say("nan rows")
    for m, n, k in ((9, 40, 64), (400, 300, 136)):
        o = Operands(9, m, n, k, 1, True)
        o.sa[3] = float("nan")
        for act in (None, "silu"):
            got = o.run([0, m], "bf16", act)
            bad = torch.zeros(m, dtype=torch.bool, device="cuda")
            bad[3] = True
            assert bool(torch.isnan(got[bad]).all()) and bool(torch.isfinite(got[~bad]).all())


def test_same_bits_streams_and_a_graph():
    say("bits, streams, graph")
    for m, n, k in ((3, 520, 8192), (40, 64, 30000), (600, 520, 264)):
        o, o2 = Operands(10, m, n, k, 1, True), Operands(11, m, n, k, 1, True)
        want, want2 = o.run([0, m], "bf16", "silu"), o2.run([0, m], "bf16", "silu")
        torch.cuda.synchronize()
        for op, w in ((o, want), (o2, want2)):
            with torch.cuda.stream(torch.cuda.Stream()):
                runs = [op.run([0, m], "bf16", "silu") for _ in range(3)]
            op.runs = runs, w
        torch.cuda.synchronize()
        for op in (o, o2):
            assert all(torch.equal(r, op.runs[1]) for r in op.runs[0])
    m, n, k = 300, 264, 520
    o = Operands(12, m, n, k, 1, False)
    x = torch.randn(m, k, device="cuda", generator=(gen := torch.Generator(device="cuda"))).bfloat16()
    c = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    qp = G.W8Quant(m, k, G.BF16, m, x.data_ptr(), k, None, o.a.data_ptr(), o.a.stride(0), o.sa.data_ptr())
    gp = G.W8Gemm(1, m, n, k, G.BF16, 0, o.a.data_ptr(), o.a.stride(0), o.sa.data_ptr(), o.b.data_ptr(), None, o.b.stride(0), 0,
                  o.sb.data_ptr(), None, 0, None, c.data_ptr(), n)
    size = G.lib().ggemm_w8_gemm_workspace(C.byref(gp))
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")

    def step():
        G.check(G.lib().ggemm_w8_quantize(C.byref(qp), stream()))
        G.check(G.lib().ggemm_w8_gemm(C.byref(gp), ws.data_ptr(), size, stream()))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(4):
        x.copy_(torch.randn(m, k, device="cuda", generator=gen))
        c.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        got = c.clone()
        step()
        assert torch.equal(got, c)


def test_quantised_block():
    """Serving as a layer does it: rows quantised, the gated pair, its result quantised, the down product; against the same
    chain in 64 bits from the library's integers (each step's own bound is tested above; here the steps meet)."""
    say("block")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(13)
    T, d, f = 90, 136, 264
    x = torch.randn(T, d, device="cuda", generator=gen).bfloat16()
    w = [torch.randn(r, c, device="cuda", generator=gen) / c ** 0.5 for r, c in ((f, d), (f, d), (d, f))]
    q = [quantise(t) for t in w]
    stored = lambda p: p[0].as_strided((p[0].shape[0], p[0].stride(0)), (p[0].stride(0), 1))   # noqa: E731
    o = Operands(0, T, f, d, 1, True)
    xq = quantise(x)
    o.a, o.sa, o.b, o.sb, o.u, o.su = stored(xq), xq[1], stored(q[0]), q[0][1], stored(q[1]), q[1][1]
    h = check(o, [0, T], "bf16", "silu")
    hq = quantise(h)
    same(hq, R.quantise64(h))
    o2 = Operands(0, T, d, f, 1, False)
    o2.a, o2.sa, o2.b, o2.sb = stored(hq), hq[1], stored(q[2]), q[2][1]
    y = check(o2, [0, T], "f32", None)
    g, u = x.double() @ w[0].double().t(), x.double() @ w[1].double().t()
    want = (g * torch.sigmoid(g) * u) @ w[2].double().t()
    # 8-bit rounding: uniform within half a step of max / 127, max about 3.5 deviations: 3.5 / 254 / sqrt 3 = 0.008 of each operand,
    # two operands a product, three products whose errors add in squares and the gated pair's doubling: below 0.03
    assert float((y - want).norm() / want.norm()) < 0.03
