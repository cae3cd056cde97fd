"""64-bit references of the gated feed-forward block, its gradients and the 8-bit integer operators, with bounds on what
the kernels' roundings may add, entry by entry."""
import math

import numpy as np
import torch

import ggemm as G

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {k: torch.finfo(v).eps / 2 for k, v in TORCH.items()}     # half a step, relative
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -24}          # where a type runs out of exponents
ACT_REL = 2.0 ** -20   # of p = act(v) / v: exponential, reciprocal, polynomial (1.5e-7 absolute for GELU), a few roundings each


def up(x, a):
    return -(-x // a) * a


def act_parts(v, act):
    """p = act(v) / v and act'(v), in 64 bits."""
    if act == "silu":
        p = torch.sigmoid(v)
        return p, p + v * p * torch.sigmoid(-v)
    if act == "gelu":
        p = 0.5 * torch.special.erfc(-v / math.sqrt(2))
        return p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    z = math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3)
    p = torch.sigmoid(z)
    return p, p + v * p * torch.sigmoid(-z) * math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * v * v)


def mm(a, b):
    return torch.matmul(a, b.contiguous())


class Block:
    """A block's operands in a type, in rows as wide as the alignment asks (or `pad` more), and the same in 64 bits."""

    def __init__(self, offsets, rows, d, f, dtype="bf16", act="silu", index=None, x_rows=None, seed=0, pad=0, device="cuda", scale=1.0):
        self.offsets, self.rows, self.d, self.f, self.dtype, self.act = list(offsets), rows, d, f, dtype, act
        self.E, self.device, self.pad = len(offsets) - 1, device, pad
        self.gen = torch.Generator(device=device)
        self.gen.manual_seed(seed)
        self.index = None if index is None else torch.tensor(np.asarray(index), dtype=torch.int32, device=device)
        self.x_rows = x_rows if index is not None else rows
        self.x = self.matrix(max(self.x_rows, 1), d)
        self.wg, self.wu = self.matrix(self.E * f, d, scale * d ** -0.5), self.matrix(self.E * f, d, scale * d ** -0.5)
        self.wd = self.matrix(self.E * d, f, f ** -0.5)
        self.dy = self.matrix(max(rows, 1), d)
        self.offs = torch.tensor(self.offsets, dtype=torch.int32, device=device)   # lives as long as graphs that read it

    def matrix(self, rows, cols, scale=1.0):
        """Random values; what lies past the columns is NaN, so that nothing may come of it."""
        t = torch.full((rows, up(cols, 8) + self.pad), float("nan"), dtype=TORCH[self.dtype], device=self.device)
        t[:, :cols] = (torch.randn(rows, cols, device=self.device, generator=self.gen) * scale).to(t.dtype)
        return t

    def spans(self):
        for g in range(self.E):
            lo, hi = (min(max(int(v), 0), self.rows) for v in self.offsets[g:g + 2])
            if lo < hi:
                yield g, slice(lo, hi)

    def covered(self):
        """Rows that belong to a group."""
        c = torch.zeros(self.rows, dtype=torch.bool, device=self.device)
        for _, r in self.spans():
            c[r] = True
        return c

    def live(self):
        if self.index is None:
            return torch.ones(self.rows, dtype=torch.bool, device=self.device)
        return (self.index >= 0) & (self.index < self.x_rows)

    def x64(self):
        x = self.x[:, :self.d].double()
        if self.index is None:
            return x[:self.rows]
        out = torch.zeros(self.rows, self.d, dtype=torch.float64, device=self.device)
        out[self.live()] = x[self.index[self.live()].long()]
        return out

    def w64(self, g):
        d, f = self.d, self.f
        return (self.wg[g * f:(g + 1) * f, :d].double(), self.wu[g * f:(g + 1) * f, :d].double(), self.wd[g * d:(g + 1) * d, :f].double())

    def zeros(self, *n):
        return torch.zeros(*n, dtype=torch.float64, device=self.device)

    def forward64(self, x=None):
        """{name: (value, bound)} of gate, up and y."""
        u, tiny, d, f = UNIT[self.dtype], TINY[self.dtype], self.d, self.f
        x = self.x64() if x is None else x
        out = {n: (self.zeros(self.rows, w), self.zeros(self.rows, w)) for n, w in (("gate", f), ("up", f), ("y", d))}
        for g, r in self.spans():
            wg, wu, wd = self.w64(g)
            a, b = mm(x[r], wg.t()), mm(x[r], wu.t())
            ea, eb = ((d + 4) * 2.0 ** -23 * mm(x[r].abs(), w.abs().t()) for w in (wg, wu))
            p, _ = act_parts(a, self.act)
            h = a * p * b
            # |act'| <= 1.13
            eh = u * h.abs() + 1.13 * ea * (b.abs() + eb) + (a * p).abs() * eb + ACT_REL * (a * b).abs() + tiny
            y = mm(h, wd.t())
            ey = mm(eh, wd.abs().t()) * (1 + u) + (f + 4) * 2.0 ** -23 * mm(h.abs() + eh, wd.abs().t()) + u * y.abs() * 1.01 + tiny
            for n, v, e in (("gate", a, ea + u * (a.abs() + ea) + tiny), ("up", b, eb + u * (b.abs() + eb) + tiny), ("y", y, ey)):
                out[n][0][r], out[n][1][r] = v, e
        return out

    def backward64(self, gate, up_, dw_dtype="f32", beta=0.0, dw0=None):
        """{name: (value, bound)} of dx and the weights' gradients, from kept projections (64 bits)."""
        u, tiny, d, f = UNIT[self.dtype], TINY[self.dtype], self.d, self.f
        uw, tw, live = UNIT[dw_dtype], TINY[dw_dtype], self.live()[:, None].double()
        x, dy = self.x64(), self.dy[:self.rows, :d].double()
        dy = torch.where(live > 0, dy, 0.0)
        pair = lambda *n: (self.zeros(*n), self.zeros(*n))   # noqa: E731
        out = {"dx": pair(self.rows, d), "dwg": pair(self.E, f, d), "dwu": pair(self.E, f, d), "dwd": pair(self.E, d, f)}
        for g, r in self.spans():
            wg, wu, wd = self.w64(g)
            a, b, s = gate[r], up_[r], live[r]
            a, b = torch.where(s > 0, a, 0.0), torch.where(s > 0, b, 0.0)
            p, slope = act_parts(a, self.act)
            dh = mm(dy[r], wd)
            edh = (d + 4) * 2.0 ** -23 * mm(dy[r].abs(), wd.abs())
            dg, du, h = dh * b * slope, dh * a * p, a * p * b
            # the slope's error: p's, and v p' with |v p'| <= 1.2 and a relative one alike
            edg = u * dg.abs() * 1.01 + 1.2 * edh * b.abs() + 4 * ACT_REL * (dh * b).abs() * (1 + a.abs()) + tiny
            edu = u * du.abs() * 1.01 + edh * a.abs() + 2 * ACT_REL * (dh * a).abs() + tiny
            eh = u * h.abs() * 1.01 + 2 * ACT_REL * (a * b).abs() + tiny
            both = mm(dg.abs() + edg, wg.abs()) + mm(du.abs() + edu, wu.abs())
            v = mm(dg, wg) + mm(du, wu)
            out["dx"][0][r] = v
            out["dx"][1][r] = mm(edg, wg.abs()) + mm(edu, wu.abs()) + (2 * f + 4) * 2.0 ** -23 * both + u * v.abs() * 1.01 + tiny
            k = (r.stop - r.start + 4) * 2.0 ** -23
            for n, left, el, right, er in (("dwg", dg, edg, x[r], 0 * x[r]), ("dwu", du, edu, x[r], 0 * x[r]), ("dwd", dy[r], 0 * dy[r], h, eh)):
                v, mass = mm(left.t(), right), mm((left.abs() + el).t(), right.abs() + er)
                e = mm(el.t(), right.abs() + er) + mm(left.abs().t(), er)
                out[n][0][g], out[n][1][g] = v, e + k * mass
        for n in ("dwg", "dwu", "dwd"):
            v, e = out[n]
            if beta:
                b0 = beta * dw0[n]
                e += 2.0 ** -23 * (v.abs() + b0.abs())
                v += b0
            e += uw * (v.abs() + e) + tw
        return out

    # ------------------------------------------------------------ the library's calls

    def struct(self, gate=None, up_=None, y=None, offsets=True):
        t = lambda v: v.data_ptr() if v is not None else None   # noqa: E731
        return G.Glu(self.E, self.rows, self.d, self.f, G.DTYPES[self.dtype], G.ACTS[self.act], self.x_rows, t(self.x),
                     self.x.stride(0), t(self.index), t(self.offs) if offsets is True else offsets, t(self.wg), t(self.wu),
                     self.wg.stride(0), self.f * self.wg.stride(0), t(self.wd), self.wd.stride(0), self.d * self.wd.stride(0), t(gate),
                     t(up_), gate.stride(0) if gate is not None else 0, t(y), y.stride(0) if y is not None else 0)

    def out(self, rows, cols, dtype=None, pad=0, fill=7.0):
        return torch.full((max(rows, 1), cols + pad), fill, dtype=TORCH[dtype or self.dtype], device=self.device)

    def forward(self, keep=True, pad=0, stream=None, offsets=True):
        """(gate, up, y) by the library; rows that it leaves alone hold 7."""
        y = self.out(self.rows, self.d, pad=pad)
        gate, u = (self.out(self.rows, self.f, pad=pad) if keep else None for _ in range(2))
        run_forward(self.struct(gate, u, y, offsets), stream)
        return gate, u, y

    def backward(self, gate, up_, want=("dx", "dw", "dwd"), dw_dtype="f32", beta=0.0, dw0=None, pad=0, stream=None):
        d, f, E = self.d, self.f, self.E
        dx = self.out(self.rows, d, pad=pad) if "dx" in want else None
        new = lambda n, r, c: self.out(E * r, c, dw_dtype, pad)   # noqa: E731
        dwg, dwu = (new("dwg", f, d), new("dwu", f, d)) if "dw" in want else (None, None)
        dwd = new("dwd", d, f) if "dwd" in want else None
        for n, t in (("dwg", dwg), ("dwu", dwu), ("dwd", dwd)):
            if t is not None and dw0 is not None:
                t[:, :dw0[n].shape[-1]] = dw0[n].reshape(t.shape[0], -1).to(t.dtype)
        q = grad_struct(self, dx, dwg, dwu, dwd, dw_dtype, beta)
        run_backward(self.struct(gate, up_, None), q, stream)
        return {"dx": dx, "dwg": dwg, "dwu": dwu, "dwd": dwd}


def grad_struct(b, dx, dwg, dwu, dwd, dw_dtype="f32", beta=0.0):
    t = lambda v: v.data_ptr() if v is not None else None   # noqa: E731
    ld = lambda v: v.stride(0) if v is not None else 0      # noqa: E731
    return G.GluGrad(t(b.dy), b.dy.stride(0), t(dx), ld(dx), G.DTYPES[dw_dtype], beta, t(dwg), t(dwu), ld(dwg), b.f * ld(dwg),
                     t(dwd), ld(dwd), b.d * ld(dwd))


def run_forward(p, stream=None):
    import ctypes as C
    n = G.lib().ggemm_glu_workspace(C.byref(p))
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    ws.fill_(255)     # NaN in either type: what is not written first may not come through
    G.check(G.lib().ggemm_glu(C.byref(p), ws.data_ptr(), n, stream or torch.cuda.current_stream().cuda_stream), "ggemm_glu")


def run_backward(p, q, stream=None):
    import ctypes as C
    n = G.lib().ggemm_glu_backward_workspace(C.byref(p), C.byref(q))
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    ws.fill_(255)
    G.check(G.lib().ggemm_glu_backward(C.byref(p), C.byref(q), ws.data_ptr(), n, stream or torch.cuda.current_stream().cuda_stream),
            "ggemm_glu_backward")


def worst(got, want, bound):
    """Largest error over its bound; NaN counts as infinite."""
    r = (got.double() - want).abs() / bound
    return float(torch.nan_to_num(r, nan=math.inf).max()) if r.numel() else 0.0


# ------------------------------------------------------------------ 8-bit integers

def quantise64(x):
    """(q, scales) of rows of x from the definition: scales rounded to 32 bits, q the nearest whole number, ties to even."""
    x = x.double()
    top = x.abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    s = (top / 127).float().clamp(min=2.0 ** -126)     # 64 bits round once to 32: the quotient is no tie of both
    bad = ~torch.isfinite(x).all(1)
    q = torch.round(torch.where(bad[:, None], 0.0, x / s.double()[:, None]))
    return q.to(torch.int8), torch.where(bad, torch.nan, s)


def product64(a, sa, b, sb, spans, n, act=None, b_up=None, sb_up=None):
    """(value, bound before the last rounding) of the grouped product; spans: (group, rows)."""
    m = a.shape[0]
    out, err = (torch.zeros(m, n, dtype=torch.float64, device=a.device) for _ in range(2))
    for g, r in spans:
        def one(q, s):
            v = mm(a[r].double(), q[g * n:(g + 1) * n].double().t()) * sa[r].double()[:, None] * s[g * n:(g + 1) * n].double()
            return v, 3.01 * 2.0 ** -24 * v.abs()     # the sum to 32 bits, two products
        v, e = one(b, sb)
        if act:
            w, ew = one(b_up, sb_up)
            p, _ = act_parts(v, act)
            e = 1.13 * e * (w.abs() + ew) + (v * p).abs() * ew + (ACT_REL + 2.0 ** -23) * (v * w).abs()
            v = v * p * w
        out[r], err[r] = v, e
    return out, err
