"""64-bit references of the 4-bit quantisation, the grouped products and the router, and the torch
side of calling them (include/ggemm_mx4.h, include/ggemm_route.h)."""
import ctypes as C

import numpy as np
import torch

import ggemm as G

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # unit roundoffs
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}   # smallest subnormals


def up(x, a):
    return -(-x // a) * a


def quantise(x):
    """x (rows x cols, float64) -> codes (rows x blocks x 32 ints), scale bytes."""
    rows, cols = x.shape
    v = np.zeros((rows, up(cols, 32)))
    v[:, :cols] = x
    v = v.reshape(rows, -1, 32)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    amax = np.abs(v).max(-1)
    e = np.where(amax > 0, np.clip(np.frexp(amax)[1] - 3, -127, 127), -127)
    a = np.abs(v) / np.ldexp(1.0, e)[..., None]
    d = np.abs(a[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = code | (np.signbit(v).astype(np.int64) << 3)
    return code, np.where(bad, 255, e + 127).astype(np.uint8)


def pack(code):
    c = code.reshape(code.shape[0], -1, 2)
    return (c[..., 0] | c[..., 1] << 4).astype(np.uint8)


def values(codes, scales):
    """The values of packed codes and scale bytes (float64)."""
    nib = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1, 32)
    mag = GRID[nib & 7] * np.where(nib & 8, -1.0, 1.0)
    s = scales[:, :nib.shape[1]].astype(np.int64)
    v = np.ldexp(mag, (s - 127)[..., None])
    return np.where((s == 255)[..., None], np.nan, v).reshape(codes.shape[0], -1)


def ptr(t):
    return t.data_ptr() if t is not None else None


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def stream():
    return torch.cuda.current_stream().cuda_stream


def gpu_quantise(x, index=None, along=True, down=False, ld=None, pad=0, rows=None):
    """Runs the kernel on a torch matrix; codes and scales as numpy (along, down), None where not asked.
    Buffers are filled with 0xA5 and have `pad` spare bytes (times 16 / 4) at each row's end."""
    R, K = (index.shape[0] if index is not None else x.shape[0]), x.shape[1]
    bufs = []
    for on, r, k in ((along, R, K), (down, K, R)):
        if on:
            c = torch.full((max(r, 1), 16 * (up(max(k, 1), 32) // 32 + pad)), 0xA5, dtype=torch.uint8, device="cuda")
            s = torch.full((max(r, 1), up(up(max(k, 1), 32) // 32, 4) + 4 * pad), 0xA5, dtype=torch.uint8, device="cuda")
            bufs += [c, s]
        else:
            bufs += [None, None]
    put = []
    for t in bufs:
        put += [ptr(t), t.shape[1] if t is not None else 0]
    dt = {v: k for k, v in TORCH.items()}[x.dtype]
    q = G.Mx4Quant(R, K, G.DTYPES[dt], x.shape[0], x.data_ptr(), x.stride(0) if ld is None else ld, ptr(index), *put)
    rc = G.lib().ggemm_mx4_quantize(C.byref(q), stream())
    torch.cuda.synchronize()
    assert rc == G.GGEMM_OK, rc
    return [t.cpu().numpy() if t is not None else None for t in bufs]


def gemm(form, a, b, m, n, k, out, offsets=None, groups=1, alpha=1.0, beta=0.0, b_strides=(0, 0), ldc=None, c_stride=0):
    """One ggemm_mx4_gemm call; a, b: (codes, scales) torch tensors; out: a torch tensor."""
    dt = {v: x for x, v in TORCH.items()}[out.dtype]
    p = G.Mx4Gemm(form, groups, m, n, k, G.DTYPES[dt], alpha, beta, ptr(a[0]), a[0].stride(0), ptr(a[1]), a[1].stride(0),
                  ptr(b[0]), b[0].stride(0), b_strides[0], ptr(b[1]), b[1].stride(0), b_strides[1], ptr(offsets),
                  out.data_ptr(), n if ldc is None else ldc, c_stride)
    size = G.lib().ggemm_mx4_gemm_workspace(C.byref(p))
    ws = torch.full((max(size, 16),), 0xA5, dtype=torch.uint8, device="cuda")
    rc = G.lib().ggemm_mx4_gemm(C.byref(p), ws.data_ptr(), size, stream())
    assert rc == G.GGEMM_OK, rc
    return out


def check_product(got, want, mass, k, dtype, what):
    """|got - want| <= k 2^-23 mass (each of k additions off by one 32-bit truncation of at most the sum of
    magnitudes `mass`) + the output's rounding; NaN exactly where want is NaN."""
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    fine = np.isfinite(want)
    err = np.abs(got - want)[fine]
    tol = ((k + 4) * 2.0 ** -23 * mass + 2 * UNIT[dtype] * np.abs(want) + TINY[dtype])[fine]
    bad = err > tol
    assert not bad.any(), (what, int(bad.sum()), float((err / tol).max()))


# ------------------------------------------------------------------ router

def route(x, mask, k, align, renorm, coef):
    """Everything ggemm_route writes, from float64 logits (tokens x experts)."""
    T, E = x.shape
    ids = np.full((T, k), -1, dtype=np.int64)
    gates = np.zeros((T, k))
    p = np.zeros((T, E))
    used = np.zeros(T, dtype=bool)
    for t in range(T):
        if (mask is not None and not mask[t]) or not (x[t] != -np.inf).any():
            continue
        used[t] = True
        order = sorted((e for e in range(E) if x[t, e] != -np.inf),
                       key=lambda e: (0, 0.0, e) if np.isnan(x[t, e]) else (1, -x[t, e], e))
        ch = order[:k]
        ids[t, :len(ch)] = ch
        with np.errstate(invalid="ignore"):
            mx = x[t, order[0]]
            w = np.where(x[t] == -np.inf, 0.0, np.exp(x[t] - mx))
            p[t] = w / w.sum()
            g = p[t, ch]
            gates[t, :len(ch)] = g / g.sum() if renorm else g
    n = int(used.sum())
    counts = np.bincount(ids[ids >= 0], minlength=E)[:E]
    offsets = np.concatenate([[0], np.cumsum(up(counts, align))])
    pos = np.full((T, k), -1, dtype=np.int64)
    cap = T * k + E * (align - 1)
    order = np.full(cap, -1, dtype=np.int64)
    fill = offsets[:-1].copy()
    for t in range(T):
        for j in range(k):
            e = ids[t, j]
            if e >= 0:
                pos[t, j] = fill[e]
                order[fill[e]] = t
                fill[e] += 1
    probs = p.sum(0) / n if n else np.zeros(E)
    loss = coef * E * float((counts * probs).sum()) / (k * n) if n else 0.0
    return dict(ids=ids, gates=gates, pos=pos, counts=counts, offsets=offsets, order=order, used=n, probs=probs,
                loss=loss, p=p, on=used)


def route_objective(x, r, k, renorm, coef, d_gates, d_loss):
    """d_loss loss + sum d_gates gates as a function of the logits, the choice and the counts held fixed."""
    T, E = x.shape
    total, P = 0.0, np.zeros(E)
    for t in np.flatnonzero(r["on"]):
        w = np.exp(x[t] - x[t].max())
        p = w / w.sum()
        P += p
        ch = r["ids"][t][r["ids"][t] >= 0]
        g = p[ch] / p[ch].sum() if renorm else p[ch]
        total += float((g * d_gates[t, :len(ch)]).sum())
    n = r["used"]
    return total + d_loss * coef * E * float((r["counts"] / (k * n) * P / n).sum())


def route_gradient(r, k, renorm, coef, d_gates, d_loss):
    """The gradient by its formula, and the magnitude of its terms (for tolerances)."""
    p, on, n = r["p"], r["on"], max(r["used"], 1)
    T, E = p.shape
    s = d_loss * coef * E * r["counts"] / (k * n * n)
    grad, mag = np.zeros((T, E)), np.zeros((T, E))
    for t in np.flatnonzero(on):
        d, c, cm = np.array(s), np.zeros(E), np.zeros(E)
        dm = np.abs(d)
        for j, e in enumerate(r["ids"][t]):
            if e < 0:
                continue
            if renorm:
                g, ok = r["gates"][t], r["ids"][t] >= 0
                c[e] = g[j] * (d_gates[t, j] - (g * d_gates[t])[ok].sum())
                cm[e] = g[j] * (abs(d_gates[t, j]) + (g * np.abs(d_gates[t]))[ok].sum())
            else:
                d[e] += d_gates[t, j]
                dm[e] += abs(d_gates[t, j])
        grad[t] = p[t] * (d - (p[t] * d).sum()) + c
        mag[t] = p[t] * (dm + (p[t] * dm).sum()) + cm
    return grad, mag


def gpu_route(logits, mask, k, align, renorm, coef, max_rows=None):
    """Runs ggemm_route on a torch matrix (leading dimension stride(0)); returns the struct and its tensors."""
    T, E = logits.shape
    dt = {v: x for x, v in TORCH.items()}[logits.dtype]
    cap = T * k + E * (align - 1) if max_rows is None else max_rows
    i32 = lambda *s: torch.full(s, -77, dtype=torch.int32, device="cuda")   # noqa: E731
    f32 = lambda *s: torch.full(s, float("nan"), dtype=torch.float32, device="cuda")   # noqa: E731
    o = dict(ids=i32(T, k), gates=f32(T, k), pos=i32(T, k), counts=i32(E), offsets=i32(E + 1), order=i32(cap), used=i32(1),
             probs=f32(E), loss=f32(1))
    r = G.Router(T, E, k, align, G.DTYPES[dt], int(renorm), coef, cap, logits.data_ptr(), logits.stride(0), ptr(mask),
                 *[ptr(o[n]) for n in ("ids", "gates", "pos", "counts", "offsets", "order", "used", "probs", "loss")])
    size = G.lib().ggemm_route_workspace(T, E, k)
    ws = torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda")
    rc = G.lib().ggemm_route(C.byref(r), ws.data_ptr(), size, stream())
    assert rc == G.GGEMM_OK, rc
    return r, o, ws
