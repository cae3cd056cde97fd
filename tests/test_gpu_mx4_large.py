"""The 4-bit operators on calls large enough for the paths that small ones do not take, and on empty ones; exact against
references on the GPU."""
import ctypes as C

import numpy as np
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


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_layer_without_tokens(dtype):
    """No tokens: the router's order holds padding only, the matrix that it picks rows from has none (and no address)."""
    say(f"no tokens {dtype}")
    E, d, f, align = 5, 200, 96, 32
    rows = E * (align - 1)
    _, o, _ = R.gpu_route(torch.zeros(0, E, device="cuda"), None, 2, align, True, 0.5)
    x = torch.zeros(0, d, dtype=R.TORCH[dtype], device="cuda")
    assert x.data_ptr() == 0 and o["order"].shape[0] == rows
    c, s, ct, st = R.gpu_quantise(x, index=o["order"], down=True)
    nb, nr = R.up(d, 32) // 32, R.up(rows, 32) // 32
    assert (c == 0).all() and (s[:, :nb] == 0).all() and (ct == 0).all() and (st[:, :nr] == 0).all()
    a, at = (R.dev(c), R.dev(s)), (R.dev(ct), R.dev(st))
    w = torch.full((E * f, 16 * nb), 0x22, dtype=torch.uint8, device="cuda"), torch.full((E * f, R.up(nb, 4)), 127, dtype=torch.uint8, device="cuda")
    out = R.gemm(G.MX4_ROWS, a, w, rows, f, d, torch.full((rows, f), 5.0, device="cuda"), o["offsets"], E,
                 b_strides=(f * w[0].shape[1], f * w[1].shape[1]))
    assert bool((out == 5.0).all())
    out = R.gemm(G.MX4_INNER, at, at, d, d, rows, torch.full((E, d, d), 5.0, device="cuda"), o["offsets"], E, c_stride=d * d)
    assert bool((out == 0.0).all())


def test_older_error_is_not_the_calls():
    """An error that an earlier call of the program left behind (here: a device that does not exist) is not reported as a
    failed launch."""
    say("older error")
    hip = C.CDLL("libamdhip64.so")
    x = torch.randn(70, 96, device="cuda")
    y = torch.zeros(70, 96, device="cuda")
    c, s = torch.zeros(70, 48, dtype=torch.uint8, device="cuda"), torch.zeros(70, 4, dtype=torch.uint8, device="cuda")
    out = torch.zeros(70, 70, device="cuda")
    q = G.Mx4Quant(70, 96, G.F32, 70, x.data_ptr(), 96, None, c.data_ptr(), 48, s.data_ptr(), 4, None, 0, None, 0)
    d = G.Mx4Dequant(70, 96, G.F32, c.data_ptr(), 48, s.data_ptr(), 4, y.data_ptr(), 96)
    p = G.Mx4Gemm(G.MX4_ROWS, 1, 70, 70, 96, G.F32, 1.0, 0.0, c.data_ptr(), 48, s.data_ptr(), 4, c.data_ptr(), 48, 0,
                  s.data_ptr(), 4, 0, None, out.data_ptr(), 70, 0)
    ws = torch.zeros(max(16, G.lib().ggemm_mx4_gemm_workspace(C.byref(p))), dtype=torch.uint8, device="cuda")
    r, o, rws = R.gpu_route(x, None, 2, 1, True, 0.1)
    dx = torch.zeros(70, 96, device="cuda")
    calls = {"quantize": lambda: G.lib().ggemm_mx4_quantize(C.byref(q), R.stream()),
             "dequantize": lambda: G.lib().ggemm_mx4_dequantize(C.byref(d), R.stream()),
             "gemm": lambda: G.lib().ggemm_mx4_gemm(C.byref(p), ws.data_ptr(), ws.numel(), R.stream()),
             "route": lambda: G.lib().ggemm_route(C.byref(r), rws.data_ptr(), rws.numel(), R.stream()),
             "route_backward": lambda: G.lib().ggemm_route_backward(C.byref(r), None, None, dx.data_ptr(), 96, R.stream())}
    torch.cuda.synchronize()
    rc = {}
    for name, call in calls.items():
        assert hip.hipSetDevice(9999) != 0
        rc[name] = call()
        hip.hipGetLastError()
    torch.cuda.synchronize()
    assert rc == {name: G.GGEMM_OK for name in calls}
    assert bool(((y - x).abs() <= 0.5 * x.abs().amax(1, keepdim=True)).all()) and bool(out.any())


@pytest.mark.parametrize("m", [3, 100, 9000])
def test_products_of_subnormal_size(m):
    """A single product of 1.5 2^e, and two that leave 2^(e - 1), down to e = -152: exact where a 32-bit number holds it
    (multiples of 2^-149), rounded there below."""
    say(f"subnormal products {m}")
    n, k = 64, 64
    e = np.arange(-152, -152 + n)
    ac = torch.zeros(m, 32, dtype=torch.uint8, device="cuda")
    asc = torch.full((m, 4), 127 - 60, dtype=torch.uint8, device="cuda")
    bsc = R.dev(np.repeat((e + 60 + 127).astype(np.uint8)[:, None], 4, 1))
    for a0, b0, want in ((0x02, 0x03, np.ldexp(1.5, e)), (0x22, 0xA3, np.ldexp(0.5, e))):      # 1, 1.5;  1 1, 1.5 -1
        ac[:, 0] = a0
        bc = torch.zeros(n, 32, dtype=torch.uint8, device="cuda")
        bc[:, 0] = b0
        out = R.gemm(G.MX4_ROWS, (ac, asc), (bc, bsc), m, n, k, torch.zeros(m, n, device="cuda"))
        got = out.double().cpu().numpy()
        held = np.ldexp(np.round(np.ldexp(want, 149)), -149) == want
        assert (got[:, held] == want[held]).all() and held.sum() >= 60
        assert (np.abs(got - want) <= 2.0 ** -149).all()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _quantised(x, index=None, along=True, down=False, spare=0):
    """The kernel's codes and scales on the GPU; rows as long as the format needs and `spare` 128-byte lines more."""
    rows, cols = (x.shape[0] if index is None else index.shape[0]), x.shape[1]
    bufs, put = [], []
    for on, r, k in ((along, rows, cols), (down, cols, rows)):
        for n in (R.up(k, 32) // 2 + 128 * spare, R.up(k, 128) // 32 + 4 * spare):
            t = torch.full((r, n), 0xA5, dtype=torch.uint8, device="cuda") if on else None
            bufs.append(t)
            put += [R.ptr(t), n if on else 0]
    dt = {v: k for k, v in R.TORCH.items()}[x.dtype]
    q = G.Mx4Quant(rows, cols, G.DTYPES[dt], x.shape[0], x.data_ptr(), x.stride(0), R.ptr(index), *put)
    assert G.lib().ggemm_mx4_quantize(C.byref(q), R.stream()) == G.GGEMM_OK
    return bufs


def _same(got, x):
    """Codes and scales of x's rows, and nothing written past a row's blocks."""
    codes, scales = got
    nb = R.up(x.shape[1], 32) // 32
    step = max(1, 2 ** 23 // x.shape[1])
    for r in range(0, x.shape[0], step):
        c, s = M.quantise(x[r:r + step])
        assert torch.equal(codes[r:r + step, :16 * nb], c) and torch.equal(scales[r:r + step, :nb], s), r
    assert bool((codes[:, 16 * nb:] == 0xA5).all()) and bool((scales[:, nb:] == 0xA5).all())


# rows, cols, spare lines at a row's end.  Along the rows the grid covers 4096 (1024 columns) or 2048 rows at once; down the
# columns 256 tiles of 256 (f32: 128) x 128 and more are dealt to the dies in runs; rows of whole 128-byte lines are stored
# past the caches.
QUANT = [(20000, 1024, 0), (20001, 1003, 0), (8192, 2048, 0), (8192, 2048, 1), (8191, 2047, 0), (16640, 1280, 0), (65537, 96, 0), (300, 40000, 0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,spare", QUANT)
def test_quantise_large(dtype, rows, cols, spare):
    say(f"quantise large {dtype} {rows}x{cols}+{spare}")
    gen = _gen(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=gen) * torch.exp(torch.randn(rows, 1, device="cuda", generator=gen))
    x = x.to(R.TORCH[dtype])
    xt = x.t().contiguous()
    c, s, ct, st = _quantised(x, down=True, spare=spare)
    _same((c, s), x)
    _same((ct, st), xt)
    c, s, _, _ = _quantised(x, spare=spare)
    _same((c, s), x)
    _, _, ct, st = _quantised(x, along=False, down=True, spare=spare)
    _same((ct, st), xt)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(8192, 1024), (30000, 520)])
def test_quantise_gather_large(dtype, rows, cols):
    say(f"quantise gather large {dtype} {rows}x{cols}")
    gen = _gen(rows)
    x = torch.randn(rows // 2, cols, device="cuda", generator=gen).to(R.TORCH[dtype])
    index = torch.randint(-1, rows // 2, (rows,), device="cuda", generator=gen, dtype=torch.int32)
    picked = torch.where((index >= 0)[:, None], x[index.clamp(min=0).long()], torch.zeros((), dtype=x.dtype, device="cuda"))
    c, s, ct, st = _quantised(x, index, down=True)
    _same((c, s), picked)
    _same((ct, st), picked.t().contiguous())
    c, s, _, _ = _quantised(x, index)
    _same((c, s), picked)


def test_quantise_past_31_bits():
    """2.8e9 values: rows at both ends, around the 2^31st value and in the middle; columns at both ends."""
    rows, cols = 70000, 40000
    say("quantise past 31 bits")
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    gen = _gen(4)
    for r in range(0, rows, 4096):
        x[r:r + 4096] = torch.randn(min(4096, rows - r), cols, device="cuda", generator=gen)
    c, s, ct, st = _quantised(x, down=True)
    c2, s2, _, _ = _quantised(x)
    assert torch.equal(c, c2) and torch.equal(s[:, :cols // 32], s2[:, :cols // 32])
    torch.cuda.synchronize()
    say("quantise past 31 bits: compared")
    for r in (0, 31000, 2 ** 31 // cols - 100, rows - 200):
        wc, ws = M.quantise(x[r:r + 200])
        assert torch.equal(c[r:r + 200], wc) and torch.equal(s[r:r + 200, :cols // 32], ws), r
    nr = R.up(rows, 32) // 32
    for k in (0, 20000, cols - 100):
        wc, ws = M.quantise(x[:, k:k + 100].t().contiguous())
        assert torch.equal(ct[k:k + 100, :16 * nr], wc) and torch.equal(st[k:k + 100, :nr], ws), k
    y = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    d = G.Mx4Dequant(rows, cols, G.BF16, c.data_ptr(), c.shape[1], s.data_ptr(), s.shape[1], y.data_ptr(), cols)
    assert G.lib().ggemm_mx4_dequantize(C.byref(d), R.stream()) == G.GGEMM_OK
    for r in (0, 2 ** 31 // cols - 100, rows - 200):
        assert torch.equal(y[r:r + 200].double(), M.values(c[r:r + 200], s[r:r + 200], cols)), r


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,ld", [(20000, 1024, 1024), (20001, 1003, 1003), (20000, 1000, 1024), (9000, 4096, 4096), (33000, 40, 64)])
def test_dequantise_large(dtype, rows, cols, ld):
    say(f"dequantise large {dtype} {rows}x{cols}")
    gen = _gen(cols)
    codes, scales = M.operand(gen, rows, cols, 100, 150)      # 16-bit values: subnormal ones and some beyond the largest
    scales[::7, 0] = 255
    y = torch.full((rows, ld), 7.0, dtype=R.TORCH[dtype], device="cuda")
    d = G.Mx4Dequant(rows, cols, G.DTYPES[dtype], codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1],
                     y.data_ptr(), ld)
    assert G.lib().ggemm_mx4_dequantize(C.byref(d), R.stream()) == G.GGEMM_OK
    want = M.values(codes, scales, cols).to(R.TORCH[dtype])
    assert torch.equal(torch.nan_to_num(y[:, :cols].float(), nan=12345.0), torch.nan_to_num(want.float(), nan=12345.0))
    assert bool((y[:, cols:] == 7.0).all())


def _near(got, want, mass, k, dtype, what):
    """Each of k additions off by one 32-bit truncation of at most the sum of magnitudes; the output's rounding."""
    tol = (k + 4) * 2.0 ** -23 * mass + 2 * R.UNIT[dtype] * want.abs() + R.TINY[dtype]
    assert bool(((got.double() - want).abs() <= tol).all()), what


def _rows_case(gen, m, n, k, off, dtype, ldc, beta, lo=123, hi=132):
    groups = len(off) - 1
    a, b = M.operand(gen, m, k, lo, hi), M.operand(gen, groups * n, k, lo, hi)
    out = torch.empty(m, ldc, dtype=R.TORCH[dtype], device="cuda")
    for r in range(0, m, 4096):
        out[r:r + 4096] = torch.randn(min(4096, m - r), ldc, device="cuda", generator=gen)
    before = out.clone() if beta or ldc > n else None
    R.gemm(G.MX4_ROWS, a, b, m, n, k, out, R.dev(np.array(off, dtype=np.int32)), groups, beta=beta,
           b_strides=(n * b[0].shape[1], n * b[1].shape[1]), ldc=ldc)
    torch.cuda.synchronize()
    for g in range(groups):
        w = M.values(b[0][g * n:(g + 1) * n], b[1][g * n:(g + 1) * n], k).t().contiguous()
        for r in range(off[g], off[g + 1], 2048):
            e = min(r + 2048, off[g + 1])
            av = M.values(a[0][r:e], a[1][r:e], k)
            want, mass = av @ w, av.abs() @ w.abs()
            if beta:
                want, mass = want + beta * before[r:e, :n].double(), mass + abs(beta) * before[r:e, :n].double().abs()
            _near(out[r:e, :n], want, mass, k, dtype, (g, r))
    if ldc > n:
        assert torch.equal(out[:, n:], before[:, n:])


@pytest.mark.parametrize("dtype,m,n,k,off,ldc,beta", [
    ("f32", 9000, 8192, 300, (0, 3000, 3001, 9000), 8192, 0.0),
    ("f32", 8300, 8200, 320, (0, 8300), 8208, -0.5),
    ("bf16", 17000, 8192, 256, (0, 5, 9000, 9000, 17000), 8192, 0.0),
    ("bf16", 17000, 8010, 96, (0, 8500, 17000), 8032, 1.0),
    ("f16", 17000, 8192, 288, (0, 17000), 8192, 0.0),
])
def test_rows_stored_past_the_caches(dtype, m, n, k, off, ldc, beta):
    """C of more than 256 MB with rows at multiples of 64 bytes."""
    say(f"rows streamed {dtype} {m} {n} {k}")
    assert m * n * (4 if dtype == "f32" else 2) > 2 ** 28 and ldc * (4 if dtype == "f32" else 2) % 64 == 0
    _rows_case(_gen(m + n + k), m, n, k, off, dtype, ldc, beta, *((115, 123) if dtype == "f16" else (123, 132)))


def test_rows_results_past_31_bits():
    """2.3e9 results."""
    say("rows results past 31 bits")
    _rows_case(_gen(1), 70000, 32800, 64, (0, 100, 69000, 70000), "bf16", 32800, 0.0)


def test_rows_weights_past_32_bits():
    """4.6e9 bytes of codes in the weights of 70 groups, a few rows each."""
    say("rows weights past 32 bits")
    off = [9 * g for g in range(71)]
    _rows_case(_gen(2), 630, 8192, 16000, off, "f32", 8192, 0.0)


@pytest.mark.parametrize("dtype,groups,m,n,k,pad,beta", [
    ("f32", 3, 4100, 6000, 3200, 0, 0.0), ("f32", 5, 4096, 4096, 4000, 16, 1.0), ("bf16", 9, 4096, 4096, 5000, 0, 0.0),
    ("f16", 9, 4000, 4112, 5000, 16, 0.0),                       # more than 256 MB
    ("f16", 2, 2048, 4096, 2000, 0, 0.0), ("f16", 3, 1000, 700, 2500, 1, 0.5), ("f16", 5, 20, 500, 3000, 0, 0.0),
    ("f16", 1, 16, 33, 640, 0, 0.0), ("f16", 1, 128, 130, 30000, 0, 0.0), ("f16", 70, 64, 64, 2000, 3, 0.0),
])
def test_inner_large_and_f16(dtype, groups, m, n, k, pad, beta):
    say(f"inner {dtype} {groups} {m} {n} {k}")
    gen = _gen(m + n + k)
    lo, hi = (113, 121) if dtype == "f16" else (123, 132)
    a, b = M.operand(gen, m, k, lo, hi), M.operand(gen, n, k, lo, hi)
    cut = np.sort(np.random.default_rng(k).integers(0, k // 32 + 1, groups - 1)) * 32
    off, ldc = np.concatenate([[0], cut, [k]]).astype(np.int32), n + pad
    out = torch.randn(groups, m, ldc, device="cuda", generator=gen).to(R.TORCH[dtype])
    before = out.clone()
    R.gemm(G.MX4_INNER, a, b, m, n, k, out, R.dev(off), groups, ldc=ldc, c_stride=m * ldc, beta=beta)
    av, bv = M.values(*a, k), M.values(*b, k)
    for g in range(groups):
        s = slice(int(off[g]), int(off[g + 1]))
        w = bv[:, s].t().contiguous()
        want, mass = av[:, s] @ w, av[:, s].abs() @ w.abs()
        if beta:
            want, mass = want + beta * before[g, :, :n].double(), mass + beta * before[g, :, :n].double().abs()
        _near(out[g, :, :n], want, mass, k, dtype, g)
        assert torch.equal(out[g, :, n:], before[g, :, n:])


@pytest.mark.parametrize("E,n,k,m", [(5, 128, 100, 77), (3, 384, 257, 1000), (40, 256, 1000, 60), (2, 2048, 1024, 6000), (16, 128, 32, 3)])
def test_input_gradient_on_transposed_weights(E, n, k, m):
    """dX[r] = dH[r] W_e by ROWS on the columns n e .. of the stacked weights' transposed quantisation, whose rows hold all
    experts; accumulated too."""
    say(f"input gradient {E} {n} {k} {m}")
    gen = _gen(E + n + k)
    W = torch.randn(E * n, k, device="cuda", generator=gen)
    _, _, wt, wts = _quantised(W, along=False, down=True)
    a = M.operand(gen, m, n)
    off = np.concatenate([[0], np.sort(np.random.default_rng(m).integers(0, m + 1, E - 1)), [m]]).astype(np.int32)
    first = R.gemm(G.MX4_ROWS, a, (wt, wts), m, k, n, torch.zeros(m, k, device="cuda"), R.dev(off), E, b_strides=(n // 2, n // 32))
    again = R.gemm(G.MX4_ROWS, a, (wt, wts), m, k, n, first.clone(), R.dev(off), E, b_strides=(n // 2, n // 32), beta=1.0)
    av, wv = M.values(*a, n), M.values(wt, wts, E * n)
    for g in range(E):
        s = slice(int(off[g]), int(off[g + 1]))
        w = wv[:, g * n:(g + 1) * n].t().contiguous()
        want, mass = av[s] @ w, av[s].abs() @ w.abs()
        _near(first[s], want, mass, n, "f32", g)
        _near(again[s], want + first[s].double(), mass + first[s].double().abs(), n, "f32", g)


def _at(t, skip, spare):
    """t's rows in a buffer that begins `skip` bytes late and has `spare` more bytes a row, all of them 255."""
    rows, n = t.shape
    buf = torch.full((skip + rows * (n + spare),), 255, dtype=torch.uint8, device="cuda")
    v = buf[skip:].view(rows, n + spare)
    v[:, :n] = t
    return v


@pytest.mark.parametrize("m,n,k,groups", [(5, 70, 3000, 2), (40, 300, 1500, 3), (700, 500, 1300, 4), (300, 260, 20000, 1),
                                          (9000, 4100, 1200, 3), (2000, 515, 2050, 9)])
def test_products_at_least_alignment(m, n, k, groups):
    """Codes at odd multiples of 16 bytes and scales at odd multiples of 4, rows and weights further apart than they are
    long; every tile shape, with whole and ragged windows of scales."""
    say(f"least alignment {m} {n} {k} {groups}")
    gen = _gen(m + n + k)
    a, b = M.operand(gen, m, k), M.operand(gen, groups * n, k)
    av, bv = M.values(*a, k), M.values(*b, k)
    off = np.concatenate([[0], np.sort(np.random.default_rng(n).integers(0, m + 1, groups - 1)), [m]]).astype(np.int32)
    a2, b2 = (_at(a[0], 16, 48), _at(a[1], 4, 4)), (_at(b[0], 48, 16), _at(b[1], 12, 20))
    assert a2[0].data_ptr() % 32 == 16 and a2[1].data_ptr() % 8 == 4 and b2[1].data_ptr() % 8 == 4
    for dtype, skip in (("f32", 1), ("bf16", 3), ("f16", 1)):
        ldc = n + 3
        out = torch.full((m * ldc + skip,), 5.0, dtype=R.TORCH[dtype], device="cuda")
        c = out[skip:].view(m, ldc)
        R.gemm(G.MX4_ROWS, a2, b2, m, n, k, c, R.dev(off), groups, b_strides=(n * b2[0].stride(0), n * b2[1].stride(0)), ldc=ldc,
               alpha=2.0 ** -9 if dtype == "f16" else 1.0)
        for g in range(groups):
            s, w = slice(int(off[g]), int(off[g + 1])), bv[g * n:(g + 1) * n].t().contiguous()
            want, mass = av[s] @ w, av[s].abs() @ w.abs()
            f = 2.0 ** -9 if dtype == "f16" else 1.0
            _near(c[s, :n], f * want, f * mass, k, dtype, (dtype, g))
        assert bool((c[:, n:] == 5.0).all())
    if groups * m * n < 2 ** 25:       # the same operands' columns cut into groups
        b3 = (b2[0][:n], b2[1][:n])
        cut = np.concatenate([[0], np.sort(np.random.default_rng(m).integers(0, k // 32 + 1, groups - 1)) * 32, [k]]).astype(np.int32)
        out = torch.full((groups, m, n + 1), 5.0, device="cuda")
        R.gemm(G.MX4_INNER, a2, b3, m, n, k, out, R.dev(cut), groups, ldc=n + 1, c_stride=m * (n + 1))
        for g in range(groups):
            s = slice(int(cut[g]), int(cut[g + 1]))
            w = bv[:n, s].t().contiguous()
            _near(out[g, :, :n], av[:, s] @ w, av[:, s].abs() @ w.abs(), k, "f32", ("inner", g))
        assert bool((out[..., n:] == 5.0).all())
