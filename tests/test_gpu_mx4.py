"""4-bit quantisation and grouped products on the GPU against 64-bit references: codes and scales bit for bit,
products within the bound of a 32-bit sum."""
import ctypes as C

import numpy as np
import pytest
import torch

import ggemm as G
import mx4_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu

QSHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (1, 4096), (33, 64), (64, 40), (127, 100), (130, 257), (300, 72)]


def _x(rng, rows, cols, dtype):
    v = rng.standard_normal((rows, cols)) * np.exp(2 * rng.standard_normal((rows, 1)))
    t = torch.from_numpy(v.astype(np.float32)).to(R.TORCH[dtype])
    return t.cuda(), t.double().numpy()


def _check_side(got, x64):
    codes, scales = got
    code, s = R.quantise(x64)
    nb = s.shape[1]
    assert np.array_equal(scales[:, :nb], s)
    assert np.array_equal(codes[:, :16 * nb], R.pack(code))
    assert (codes[:, 16 * nb:] == 0xA5).all() and (scales[:, nb:] == 0xA5).all()   # nothing past the blocks


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", QSHAPES)
def test_quantise_sizes(dtype, rows, cols):
    say(f"quantise {dtype} {rows}x{cols}")
    rng = np.random.default_rng(rows * 1000 + cols)
    x, x64 = _x(rng, rows, cols, dtype)
    c, s, ct, st = R.gpu_quantise(x, down=True, pad=1)
    _check_side((c, s), x64)
    _check_side((ct, st), x64.T)
    c, s, _, _ = R.gpu_quantise(x)
    _check_side((c, s), x64)
    _, _, ct, st = R.gpu_quantise(x, along=False, down=True)
    _check_side((ct, st), x64.T)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantise_strided_unaligned(dtype):
    rng = np.random.default_rng(5)
    base = torch.from_numpy(rng.standard_normal((70, 145)).astype(np.float32)).to(R.TORCH[dtype]).cuda()
    for c0, cols in ((0, 96), (1, 96), (3, 141)):
        say(f"quantise strided {dtype} {c0} {cols}")
        x = base[:, c0:c0 + cols]
        got = R.gpu_quantise(x, down=True)
        _check_side(got[:2], x.double().cpu().numpy())
        _check_side(got[2:], x.double().cpu().numpy().T)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantise_gather(dtype):
    rng = np.random.default_rng(6)
    x, x64 = _x(rng, 50, 200, dtype)
    idx = rng.integers(-1, 51, 171).astype(np.int32)     # -1 and 50: rows that do not exist
    idx[[3, 70]] = [-2 ** 31, 2 ** 31 - 1]
    say(f"quantise gather {dtype}")
    ok = (idx >= 0) & (idx < 50)
    want = np.where(ok[:, None], x64[np.where(ok, idx, 0)], 0.0)
    got = R.gpu_quantise(x, index=R.dev(idx), down=True)
    _check_side(got[:2], want)
    _check_side(got[2:], want.T)


def _bits(u, dtype):
    if dtype == "f32":
        return torch.from_numpy(u.astype(np.uint32).view(np.int32)).view(torch.float32)
    return torch.from_numpy(u.astype(np.uint16).view(np.int16)).view(R.TORCH[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_quantise_every_16_bit_value(dtype):
    """Every value as the first of a block, the others its multiples by quarters of the grid's steps (ties
    among them), zeros of both signs and much smaller ones."""
    say(f"quantise every {dtype}")
    first = _bits(np.arange(65536), dtype)
    f = np.concatenate([np.arange(1, 25) / 24.0, [0.0, -0.0, 1e-3, -0.5, -0.25, -0.75, 2.0 ** -20]])
    x = (first.double().numpy()[:, None] * np.concatenate([[1.0], f])[None])
    with np.errstate(invalid="ignore", over="ignore"):
        t = torch.from_numpy(x).to(R.TORCH[dtype])
    t[:, 0] = first
    assert t.shape[1] == 32
    c, s, ct, st = R.gpu_quantise(t.cuda(), down=False)
    _check_side((c, s), t.double().numpy())
    tt = t.t().contiguous()
    _, _, ct, st = R.gpu_quantise(tt.cuda(), along=False, down=True)
    _check_side((ct, st), t.double().numpy())


def test_quantise_f32_ranges():
    """Blocks over the whole range of exponents, subnormals, values just beside the rounding points, zeros, NaN, Inf."""
    say("quantise f32 ranges")
    rng = np.random.default_rng(8)
    e = np.repeat(np.arange(-149, 128), 4)
    lead = np.ldexp(1 + rng.random(e.size), e)
    mid = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0])           # ties, in units of the scale
    unit = np.ldexp(1.0, np.clip(np.frexp(lead)[1] - 3, -127, 127))
    x = np.zeros((e.size, 32))
    x[:, 0] = lead
    x[:, 1:8] = mid * unit[:, None]
    x[:, 8:15] = np.nextafter((mid * unit[:, None]).astype(np.float32), np.float32(0))
    x[:, 15:22] = np.nextafter((mid * unit[:, None]).astype(np.float32), np.float32(np.inf))
    x[:, 22:] = rng.uniform(-1, 1, (e.size, 10)) * lead[:, None]
    x[np.abs(x) > 2 * lead[:, None]] = 0
    extra = np.zeros((8, 32))
    extra[1, 5] = np.nan
    extra[2, 31] = np.inf
    extra[3, 0] = -np.inf
    extra[4] = -0.0
    extra[5] = np.finfo(np.float32).max
    extra[6] = 2.0 ** -149
    extra[7, 9], extra[7, 10] = np.finfo(np.float32).max, 2.0 ** -149
    x = np.concatenate([x, extra])
    with np.errstate(over="ignore"):
        t = torch.from_numpy(x.astype(np.float32))
    c, s, _, _ = R.gpu_quantise(t.cuda())
    _check_side((c, s), t.double().numpy())
    _, _, ct, st = R.gpu_quantise(t.t().contiguous().cuda(), along=False, down=True)
    _check_side((ct, st), t.double().numpy())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,ld", [(1, 1, 1), (3, 45, 45), (70, 256, 264), (9, 8 * 33, 8 * 33 + 1)])
def test_dequantise(dtype, rows, cols, ld):
    say(f"dequantise {dtype} {rows}x{cols}")
    rng = np.random.default_rng(cols)
    nb = R.up(cols, 32) // 32
    codes = rng.integers(0, 256, (rows, 16 * nb)).astype(np.uint8)
    scales = rng.integers(0, 256, (rows, R.up(nb, 4))).astype(np.uint8)
    scales[0, 0] = 255
    y = torch.full((rows, ld), 7.0, dtype=R.TORCH[dtype], device="cuda")
    cd, sd = R.dev(codes), R.dev(scales)
    d = G.Mx4Dequant(rows, cols, G.DTYPES[dtype], cd.data_ptr(), cd.shape[1], sd.data_ptr(), sd.shape[1], y.data_ptr(), ld)
    assert G.lib().ggemm_mx4_dequantize(C.byref(d), R.stream()) == G.GGEMM_OK
    with np.errstate(over="ignore"):
        want = torch.from_numpy(R.values(codes, scales)[:, :cols].astype(np.float32)).to(R.TORCH[dtype])
    got = y.cpu()
    assert torch.equal(torch.nan_to_num(got[:, :cols].double(), nan=1e300), torch.nan_to_num(want.double(), nan=1e300))
    assert (got[:, cols:] == 7.0).all()


def _operand(rng, rows, cols, spread=4):
    """Random codes and scales with blocks that fill up with zeros, on the GPU and as float64 values."""
    nb = R.up(max(cols, 1), 32) // 32
    nib = rng.integers(0, 16, (rows, 32 * nb))
    nib[:, cols:] = 0
    codes = R.pack(nib.reshape(rows, nb, 32))
    scales = np.full((rows, R.up(nb, 4)), 255, dtype=np.uint8)     # bytes past the blocks must not matter
    scales[:, :nb] = rng.integers(127 - spread, 128 + spread, (rows, nb))
    return (R.dev(codes), R.dev(scales)), R.values(codes, scales[:, :nb])[:, :cols]


def _groups(rng, total, groups, empty=0.3):
    w = rng.random(groups) * (rng.random(groups) >= empty)
    if w.sum() == 0:
        w[groups // 2] = 1.0
    c = np.floor(w / w.sum() * total).astype(np.int64)
    c[int(np.argmax(w))] += total - c.sum()
    return np.concatenate([[0], np.cumsum(c)])


ROWS = [  # m, n, k, groups
    (1, 1, 1, 1), (1, 1, 32, 1), (1, 130, 64, 3), (2, 64, 4096, 2), (5, 100, 96, 4), (16, 256, 512, 1), (17, 31, 33, 5),
    (33, 129, 255, 2), (64, 64, 64, 1), (65, 257, 160, 70), (128, 512, 1024, 8), (200, 300, 31, 3), (257, 255, 417, 2),
    (300, 1000, 1001, 23), (513, 384, 256, 4), (1000, 192, 2048, 130), (1024, 1024, 320, 2), (777, 515, 1056, 1),
]


@pytest.mark.parametrize("m,n,k,groups", ROWS)
def test_rows_product(m, n, k, groups):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a, av = _operand(rng, m, k)
    b, bv = _operand(rng, groups * n, k)
    off = _groups(rng, m, groups)
    offs = R.dev(off.astype(np.int32))
    strides = (n * b[0].shape[1], n * b[1].shape[1])
    want = np.concatenate([av[off[g]:off[g + 1]] @ bv[g * n:(g + 1) * n].T for g in range(groups)])
    mass = np.concatenate([np.abs(av[off[g]:off[g + 1]]) @ np.abs(bv[g * n:(g + 1) * n]).T for g in range(groups)])
    for dtype in ("f32", "bf16", "f16"):
        say(f"rows {m} {n} {k} {groups} {dtype}")
        ldc = n + (3 if dtype == "bf16" else 8 if dtype == "f16" else 0)
        out = torch.full((m, ldc), 5.0, dtype=R.TORCH[dtype], device="cuda")
        R.gemm(G.MX4_ROWS, a, b, m, n, k, out, offs, groups, b_strides=strides, ldc=ldc)
        got = out.float().cpu().numpy()
        if dtype == "f16":
            sel = mass < 3e4      # beyond it a 16-bit value may round to Inf
            R.check_product(np.where(sel, got[:, :n], 0), np.where(sel, want, 0), mass, k, dtype, (m, n, k, groups, dtype))
        else:
            R.check_product(got[:, :n], want, mass, k, dtype, (m, n, k, groups, dtype))
        assert (got[:, n:] == 5.0).all()
    # C = alpha A B + beta C
    c0 = rng.standard_normal((m, n)).astype(np.float32)
    out = R.dev(c0)
    R.gemm(G.MX4_ROWS, a, b, m, n, k, out, offs, groups, alpha=-1.5, beta=0.75, b_strides=strides)
    R.check_product(out.cpu().numpy(), -1.5 * want + 0.75 * c0, 1.5 * mass + np.abs(c0), k, "f32", ("beta", m, n, k))


INNER = [  # m, n, total k, groups
    (1, 1, 32, 1), (3, 5, 64, 2), (64, 64, 256, 3), (65, 130, 96, 4), (100, 200, 1024, 7), (256, 256, 2048, 5),
    (257, 300, 4096, 66), (512, 96, 800, 2),
]


@pytest.mark.parametrize("m,n,k,groups", INNER)
def test_inner_product(m, n, k, groups):
    rng = np.random.default_rng(m * 11 + n * 5 + k)
    a, av = _operand(rng, m, k)
    b, bv = _operand(rng, n, k)
    off = 32 * _groups(rng, k // 32, groups)
    want = np.stack([av[:, off[g]:off[g + 1]] @ bv[:, off[g]:off[g + 1]].T for g in range(groups)])
    mass = np.stack([np.abs(av[:, off[g]:off[g + 1]]) @ np.abs(bv[:, off[g]:off[g + 1]]).T for g in range(groups)])
    for dtype in ("f32", "bf16"):
        say(f"inner {m} {n} {k} {groups} {dtype}")
        ldc = n + (5 if dtype == "bf16" else 0)
        out = torch.full((groups, m, ldc), 5.0, dtype=R.TORCH[dtype], device="cuda")
        R.gemm(G.MX4_INNER, a, b, m, n, k, out, R.dev(off.astype(np.int32)), groups, ldc=ldc, c_stride=m * ldc)
        got = out.float().cpu().numpy()
        R.check_product(got[..., :n], want, mass, k, dtype, (m, n, k, groups, dtype))
        assert (got[..., n:] == 5.0).all()
    c0 = rng.standard_normal((groups, m, n)).astype(np.float32)
    out = R.dev(c0)
    R.gemm(G.MX4_INNER, a, b, m, n, k, out, R.dev(off.astype(np.int32)), groups, alpha=0.5, beta=1.0, c_stride=m * n)
    R.check_product(out.cpu().numpy(), 0.5 * want + c0, 0.5 * mass + np.abs(c0), k, "f32", ("beta", m, n, k))


@pytest.mark.parametrize("m,n,k", [(1, 48, 77), (40, 33, 500), (300, 290, 100), (260, 300, 2048)])
def test_one_group_without_offsets(m, n, k):
    say(f"dense {m} {n} {k}")
    rng = np.random.default_rng(m + n + k)
    a, av = _operand(rng, m, k)
    b, bv = _operand(rng, n, k)
    for form in (G.MX4_ROWS, G.MX4_INNER):
        out = torch.zeros(m, n, dtype=torch.float32, device="cuda")
        R.gemm(form, a, b, m, n, k, out)
        R.check_product(out.cpu().numpy(), av @ bv.T, np.abs(av) @ np.abs(bv).T, k, "f32", (form, m, n, k))


def test_rows_outside_groups_stay():
    """Rows before the first and past the last offset are not written; offsets out of range are clamped."""
    say("rows outside groups")
    rng = np.random.default_rng(3)
    m, n, k = 100, 70, 64
    a, av = _operand(rng, m, k)
    b, bv = _operand(rng, 3 * n, k)
    for off in ([10, 40, 40, 90], [0, 0, 0, 0], [100, 100, 100, 100], [-50, 20, 60, 1000], [60, 20, 80, 80]):
        out = torch.full((m, n), 5.0, device="cuda")
        R.gemm(G.MX4_ROWS, a, b, m, n, k, out, R.dev(np.array(off, dtype=np.int32)), 3,
               b_strides=(n * b[0].shape[1], n * b[1].shape[1]))
        want, mass = np.full((m, n), 5.0), np.zeros((m, n))
        o = np.clip(off, 0, m)
        for g in range(3):
            s = slice(o[g], max(o[g], o[g + 1]))
            want[s] = av[s] @ bv[g * n:(g + 1) * n].T
            mass[s] = np.abs(av[s]) @ np.abs(bv[g * n:(g + 1) * n]).T
        R.check_product(out.cpu().numpy(), want, mass, k, "f32", off)


def test_inner_offsets_clamped_and_rounded():
    say("inner offsets")
    rng = np.random.default_rng(4)
    m, n, k = 70, 90, 200       # ends inside a block
    a, av = _operand(rng, m, k)
    b, bv = _operand(rng, n, k)
    for off, used in (([0, 64, 200], [0, 64, 200]), ([0, 70, 199], [0, 64, 192]), ([-5, 64, 9999], [0, 64, 200]),
                      ([200, 200, 200], [200, 200, 200]), ([96, 32, 200], [96, 32, 200])):
        out = torch.full((2, m, n), 5.0, device="cuda")
        R.gemm(G.MX4_INNER, a, b, m, n, k, out, R.dev(np.array(off, dtype=np.int32)), 2, c_stride=m * n)
        for g in range(2):
            s = slice(used[g], max(used[g], used[g + 1]))
            R.check_product(out[g].cpu().numpy(), av[:, s] @ bv[:, s].T, np.abs(av[:, s]) @ np.abs(bv[:, s]).T, k, "f32", (off, g))


@pytest.mark.parametrize("m", [1, 20, 300])
def test_k_zero_and_empty_inner(m):
    say(f"k zero {m}")
    n = 40
    z = torch.zeros(m, 16, dtype=torch.uint8, device="cuda"), torch.zeros(m, 4, dtype=torch.uint8, device="cuda")
    w = torch.zeros(n, 16, dtype=torch.uint8, device="cuda"), torch.zeros(n, 4, dtype=torch.uint8, device="cuda")
    for form in (G.MX4_ROWS, G.MX4_INNER):
        out = torch.full((m, n), 3.0, device="cuda")
        R.gemm(form, z, w, m, n, 0, out, beta=0.5)
        assert (out == 1.5).all()
        out = torch.full((m, n), float("nan"), device="cuda")
        R.gemm(form, z, w, m, n, 0, out)
        assert (out == 0.0).all()      # beta = 0: C is not read


@pytest.mark.parametrize("m,n,k", [(3, 70, 96), (200, 300, 256), (300, 520, 600)])
def test_product_nan_blocks_and_extreme_scales(m, n, k):
    """A NaN block makes its row (A) or column (B) NaN and nothing else; scales at both ends of the range."""
    say(f"nan and scales {m} {n} {k}")
    rng = np.random.default_rng(m)
    a, _ = _operand(rng, m, k)
    b, _ = _operand(rng, n, k)
    ac, asc, bc, bsc = (t.cpu().numpy().copy() for t in (*a, *b))
    nb = R.up(k, 32) // 32
    asc[m // 2, nb - 1] = 255
    bsc[n - 1, 0] = 255
    asc[0, :nb], bsc[0, :nb] = 0, 140       # 2^-127 times 2^13
    asc[1, :nb], bsc[1, :nb] = 230, 20      # 2^103 times 2^-107
    asc[2, :nb], bsc[2, :nb] = 14, 230
    av, bv = R.values(ac, asc)[:, :k], R.values(bc, bsc)[:, :k]
    out = torch.zeros(m, n, device="cuda")
    R.gemm(G.MX4_ROWS, (R.dev(ac), R.dev(asc)), (R.dev(bc), R.dev(bsc)), m, n, k, out)
    got = out.cpu().numpy()
    want = av @ bv.T
    mass = np.abs(av) @ np.abs(bv).T
    keep = mass < 2.0 ** 120       # sums that stay in range; a product below 2^-126 may count as zero
    keep |= np.isnan(want)
    R.check_product(np.where(keep, got, 0), np.where(keep, want, 0), np.where(keep, mass, 0) + 2.0 ** -103 * (mass < 2.0 ** -100), k, "f32", (m, n, k))


def test_other_stream_and_graph_replay():
    """Calls on another stream and their replays from a captured graph on new inputs."""
    say("graph")
    rng = np.random.default_rng(9)
    m, n, k, groups = 96, 160, 192, 4
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    b, bv = _operand(rng, groups * n, k)
    offs = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    codes, scales = torch.zeros(m, 96, dtype=torch.uint8, device="cuda"), torch.zeros(m, 8, dtype=torch.uint8, device="cuda")
    out = torch.zeros(m, n, device="cuda")
    q = G.Mx4Quant(m, k, G.BF16, m, x.data_ptr(), k, None, codes.data_ptr(), 96, scales.data_ptr(), 8, None, 0, None, 0)
    p = G.Mx4Gemm(G.MX4_ROWS, groups, m, n, k, G.F32, 1.0, 0.0, codes.data_ptr(), 96, scales.data_ptr(), 8,
                  b[0].data_ptr(), b[0].shape[1], n * b[0].shape[1], b[1].data_ptr(), b[1].shape[1], n * b[1].shape[1],
                  offs.data_ptr(), out.data_ptr(), n, 0)
    ws = torch.zeros(max(16, G.lib().ggemm_mx4_gemm_workspace(C.byref(p))), dtype=torch.uint8, device="cuda")

    def call(s):
        assert G.lib().ggemm_mx4_quantize(C.byref(q), s) == G.GGEMM_OK
        assert G.lib().ggemm_mx4_gemm(C.byref(p), ws.data_ptr(), ws.numel(), s) == G.GGEMM_OK

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call(side.cuda_stream)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call(side.cuda_stream)
    for i in range(4):
        v = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(torch.bfloat16)
        off = _groups(rng, m, groups)
        x.copy_(v.cuda())
        offs.copy_(R.dev(off.astype(np.int32)))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        code, s = R.quantise(v.double().numpy())
        av = R.values(R.pack(code), s)
        want = np.concatenate([av[off[g]:off[g + 1]] @ bv[g * n:(g + 1) * n].T for g in range(groups)])
        mass = np.concatenate([np.abs(av[off[g]:off[g + 1]]) @ np.abs(bv[g * n:(g + 1) * n]).T for g in range(groups)])
        R.check_product(out.cpu().numpy(), want, mass, k, "f32", ("replay", i))
