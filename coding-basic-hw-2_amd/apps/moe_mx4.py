"""Mixture-of-experts feed-forward layer with 4-bit expert products: router, dispatch, up, activation, down, combine,
and in training the whole backward pass and an update, on the library's router (include/ggemm_route.h) and 4-bit
operators (include/ggemm_mx4.h).  The FP64 layer on the grouped DGEMM is moe_ffn.py.

Layer (T tokens, width d, hidden width f, E experts, k per token, rows R = T k and padding):
  route     logits = x Wr;  gates, counts, offsets, order, balance loss               ggemm_route
  dispatch  rows x[order] quantised (training: along the rows and down the columns)   ggemm_mx4_quantize
  up, act   H = Xq W1_e^T, Ha = tanh H, quantised                                     ggemm_mx4_gemm, ROWS
  down      Y = Haq W2_e^T                                                            ggemm_mx4_gemm, ROWS
  combine   out[t] = sum_j gates[t, j] Y[pos[t, j]]
Backward (loss = mean (out - target)^2 / 2 + balance loss), every product on operands quantised along its own
inner dimension: dHa = dYq W2_e and dX = dHq W1_e (ROWS on the transposed weights), dW2_e = dY^T Ha and
dW1_e = dH^T X (INNER: the tokens of each expert), gates and loss back to the logits (ggemm_route_backward).
Weights are kept in 32 bits and quantised once per step, both ways at once; a step moves each matrix by lr / 50 of
its norm.

Usage: python3 moe_mx4.py [--tokens 4096] [--experts 16] [--topk 2] [--d-model 1024] [--d-ff 2048] [--steps 10]
                          [--lr 0.5] [--balance 0.01] [--seed 7] [--serve]
--serve: forward only (no padding, no transposed operands); --tokens 1 is one decoding step.
Prints one JSON line: time per step and stage (us), losses, and the largest error of sampled product entries in
units of their bound (k + 4) 2^-23 sum |a b| against 64-bit sums of the same quantised operands.
"""
import argparse
import ctypes as C
import json
import sys

import app_util as AU

G = AU.G
STAGES = ("route", "dispatch", "up", "down", "combine", "backward", "update")


def parse_args(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--topk", type=int, default=2)
    ap.add_argument("--d-model", type=int, default=1024)
    ap.add_argument("--d-ff", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=10)
    ap.add_argument("--lr", type=float, default=0.5)
    ap.add_argument("--balance", type=float, default=0.01)
    ap.add_argument("--seed", type=int, default=7)
    ap.add_argument("--serve", action="store_true")
    a = ap.parse_args(argv)
    if min(a.tokens, a.experts, a.steps) < 1 or not 1 <= a.topk <= min(a.experts, G.ROUTE_MAX_TOPK):
        ap.error("--tokens, --experts and --steps must be positive, --topk in [1, --experts]")
    if a.experts > G.ROUTE_MAX_EXPERTS:
        ap.error(f"at most {G.ROUTE_MAX_EXPERTS} experts")
    # the transposed weights of an expert start at a multiple of its rows: whole scale words
    if a.d_model < 128 or a.d_ff < 128 or a.d_model % 128 or a.d_ff % 128:
        ap.error("--d-model and --d-ff must be multiples of 128")
    return a


class Quantised:
    """A matrix in 4 bits along its rows (codes, scales) and, where asked, down its columns (codes_t, scales_t)."""

    def __init__(self, torch, rows, cols, along=True, down=False):
        u8 = lambda r, c: torch.zeros(r, c, dtype=torch.uint8, device="cuda")   # noqa: E731
        up = lambda x, m: -(-x // m) * m                                        # noqa: E731
        self.rows, self.cols = rows, cols
        self.codes, self.scales = (u8(rows, up(cols, 32) // 2), u8(rows, up(cols, 128) // 32)) if along else (None, None)
        self.codes_t, self.scales_t = (u8(cols, up(rows, 32) // 2), u8(cols, up(rows, 128) // 32)) if down else (None, None)

    def of(self, x, index=None):
        """Quantises x (rows, cols), or its rows index[0], index[1], ... (-1: zeros)."""
        put = []
        for t in (self.codes, self.scales, self.codes_t, self.scales_t):
            put += [t.data_ptr(), t.shape[1]] if t is not None else [None, 0]
        kind = {"torch.float32": G.F32, "torch.bfloat16": G.BF16, "torch.float16": G.F16}[str(x.dtype)]
        q = G.Mx4Quant(self.rows, self.cols, kind, x.shape[0], x.data_ptr(), x.stride(0),
                       index.data_ptr() if index is not None else None, *put)
        G.check(G.lib().ggemm_mx4_quantize(C.byref(q), stream()), "ggemm_mx4_quantize")
        return self


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


class Layer:
    def __init__(self, a, torch):
        self.a, self.torch = a, torch
        gen = torch.Generator(device="cuda")
        gen.manual_seed(a.seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)   # noqa: E731
        T, E, k, d, f = a.tokens, a.experts, a.topk, a.d_model, a.d_ff
        self.align = 1 if a.serve else 32
        self.R = T * k + E * (self.align - 1)      # rows at most; the real number is on the device
        self.x, self.target = rand(T, d).bfloat16(), rand(T, d)
        self.Wr, self.W1, self.W2 = rand(d, E) / d ** 0.5, rand(E * f, d) / d ** 0.5, rand(E * d, f) / f ** 0.5
        train = not a.serve
        new = lambda r, c: Quantised(torch, r, c, down=train)             # noqa: E731
        self.W1q, self.W2q = new(E * f, d), new(E * d, f)
        self.Xq, self.Haq, self.dYq, self.dHq = new(self.R, d), new(self.R, f), new(self.R, d), new(self.R, f)
        i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")   # noqa: E731
        f32 = lambda *s: torch.empty(*s, device="cuda")                      # noqa: E731
        self.ids, self.pos, self.gates = i32(T, k), i32(T, k), f32(T, k)
        self.counts, self.offsets, self.order, self.used = i32(E), i32(E + 1), i32(max(self.R, 1)), i32(1)
        self.probs, self.balance = f32(E), f32(1)
        self.H, self.Y = (torch.zeros(self.R, n, dtype=torch.bfloat16, device="cuda") for n in (f, d))
        self.route_ws = torch.empty(G.lib().ggemm_route_workspace(T, E, k), dtype=torch.uint8, device="cuda")
        self.ws = torch.empty(0, dtype=torch.uint8, device="cuda")
        self.quantise_weights()

    def quantise_weights(self):
        self.W1q.of(self.W1)
        self.W2q.of(self.W2)

    def product(self, form, m, n, k, A, As, B, Bs, out, b_stride=0, bs_stride=0, c_stride=0):
        kind = {"torch.float32": G.F32, "torch.bfloat16": G.BF16}[str(out.dtype)]
        p = G.Mx4Gemm(form, self.a.experts, m, n, k, kind, 1.0, 0.0, A.data_ptr(), A.stride(0), As.data_ptr(), As.stride(0),
                      B.data_ptr(), B.stride(0), b_stride, Bs.data_ptr(), Bs.stride(0), bs_stride, self.offsets.data_ptr(),
                      out.data_ptr(), n, c_stride)
        need = G.lib().ggemm_mx4_gemm_workspace(C.byref(p))
        if need > self.ws.numel():
            self.ws = self.torch.empty(need, dtype=self.torch.uint8, device="cuda")
        G.check(G.lib().ggemm_mx4_gemm(C.byref(p), self.ws.data_ptr(), self.ws.numel(), stream()), "ggemm_mx4_gemm")
        return out

    def rows(self, Aq, Wq, n, k, out):
        """out[r] = A[r] W_e^T, W_e: n x k."""
        return self.product(G.MX4_ROWS, self.R, n, k, Aq.codes, Aq.scales, Wq.codes, Wq.scales, out,
                            n * Wq.codes.shape[1], n * Wq.scales.shape[1])

    def rows_t(self, Aq, Wq, n, k, out):
        """out[r] = A[r] W_e, W_e: k x n, by the transposed quantisation: expert e's columns k e .. of n rows."""
        return self.product(G.MX4_ROWS, self.R, n, k, Aq.codes, Aq.scales, Wq.codes_t, Wq.scales_t, out, k // 2, k // 32)

    def inner(self, Aq, Bq, m, n):
        """out_e = A_e^T B_e over expert e's rows (m x n each)."""
        out = self.torch.empty(self.a.experts * m, n, device="cuda")
        return self.product(G.MX4_INNER, m, n, self.R, Aq.codes_t, Aq.scales_t, Bq.codes_t, Bq.scales_t, out, c_stride=m * n)

    def forward(self, mark=lambda i: None):
        a, t = self.a, self.torch
        T, d, f = a.tokens, a.d_model, a.d_ff
        self.logits = self.x.float() @ self.Wr
        self.r = G.Router(T, a.experts, a.topk, self.align, G.F32, 1, a.balance, self.R, self.logits.data_ptr(), a.experts,
                          None, *[v.data_ptr() for v in (self.ids, self.gates, self.pos, self.counts, self.offsets,
                                                         self.order, self.used, self.probs, self.balance)])
        G.check(G.lib().ggemm_route(C.byref(self.r), self.route_ws.data_ptr(), self.route_ws.numel(), stream()), "ggemm_route")
        mark(0)
        self.Xq.of(self.x, self.order)
        mark(1)
        self.rows(self.Xq, self.W1q, f, d, self.H)
        self.Ha = t.tanh(self.H)
        self.Haq.of(self.Ha)
        mark(2)
        self.rows(self.Haq, self.W2q, d, f, self.Y)
        mark(3)
        self.picked = self.Y[self.pos.clamp(min=0).long()].float()          # T x k x d
        self.out = (self.picked * self.gates[..., None]).sum(1)
        mark(4)
        return self.out

    def backward(self):
        a, t = self.a, self.torch
        T, E, d, f = a.tokens, a.experts, a.d_model, a.d_ff
        d_out = (self.out - self.target) / (T * d)
        d_gates = (self.picked * d_out[:, None]).sum(-1).contiguous()
        # each row's gradient: its token's, times its gate (rows of padding: zeros)
        gate = t.zeros(self.R, device="cuda")
        gate[self.pos.view(-1).long()] = self.gates.view(-1)
        dY = d_out[self.order.clamp(min=0).long()] * gate[:, None]
        self.dYq.of(dY)
        dHa = self.rows_t(self.dYq, self.W2q, f, d, t.zeros(self.R, f, device="cuda"))
        self.gW2 = self.inner(self.dYq, self.Haq, d, f)
        Ha = self.Ha.float()
        self.dHq.of(dHa * (1 - Ha * Ha))
        dX = self.rows_t(self.dHq, self.W1q, d, f, t.zeros(self.R, d, device="cuda"))
        self.gW1 = self.inner(self.dHq, self.Xq, f, d)
        d_logits, one = t.empty(T, E, device="cuda"), t.ones(1, device="cuda")
        G.check(G.lib().ggemm_route_backward(C.byref(self.r), d_gates.data_ptr(), one.data_ptr(), d_logits.data_ptr(), E, stream()),
                "ggemm_route_backward")
        self.gWr = self.x.float().t() @ d_logits
        self.gx = dX[self.pos.clamp(min=0).long()].sum(1) + d_logits @ self.Wr.t()

    def update(self):
        """Each matrix moves against its gradient by lr / 50 of its own norm, whatever the gradient's."""
        for w, g in ((self.W1, self.gW1), (self.W2, self.gW2), (self.Wr, self.gWr)):
            w -= (0.02 * self.a.lr * w.norm() / (g.norm() + 1e-30)) * g
        self.quantise_weights()

    def loss(self):
        return float(((self.out - self.target) ** 2).mean() / 2), float(self.balance)

    def values(self, codes, scales):
        """What codes and scales stand for, by the library, in 64 bits."""
        y = self.torch.empty(codes.shape[0], 2 * codes.shape[1], device="cuda")
        q = G.Mx4Dequant(y.shape[0], y.shape[1], G.F32, codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1],
                         y.data_ptr(), y.shape[1])
        G.check(G.lib().ggemm_mx4_dequantize(C.byref(q), stream()), "ggemm_mx4_dequantize")
        return y.double()

    def product_error(self):
        """Largest error of the fullest expert's part of H (and of its dW1) over its bound."""
        a, t = self.a, self.torch
        e = int(self.counts.argmax())
        lo = int(self.offsets[e])
        hi, d, f, worst = lo + int(self.counts[e]), a.d_model, a.d_ff, 0.0

        def over(got, A, B, k, unit):
            want, mass = A @ B.t().contiguous(), A.abs() @ B.abs().t().contiguous()
            return float(((got.double() - want).abs() / ((k + 4) * 2.0 ** -23 * mass + unit * want.abs() + 1e-38)).max())
        X, W = self.values(self.Xq.codes[lo:hi], self.Xq.scales[lo:hi]), self.values(self.W1q.codes[e * f:(e + 1) * f],
                                                                                   self.W1q.scales[e * f:(e + 1) * f])
        worst = max(worst, over(self.H[lo:hi], X, W, d, 2.0 ** -7))
        if not a.serve:
            end = int(self.offsets[e + 1])
            A = self.values(self.dHq.codes_t, self.dHq.scales_t)[:, lo:end].contiguous()
            B = self.values(self.Xq.codes_t, self.Xq.scales_t)[:, lo:end].contiguous()
            worst = max(worst, over(self.gW1[e * f:(e + 1) * f], A, B, end - lo, 2.0 ** -23))
        return worst


def main(argv=None):
    a = parse_args(argv)
    import torch
    if not torch.cuda.is_available():
        sys.exit("moe_mx4: no GPU")
    lay = Layer(a, torch)
    stages = STAGES[:5] if a.serve else STAGES
    timer, losses = AU.StageTimer(torch, stages), []
    for step in range(a.steps + 1):      # the first one warms up
        timer.start()
        lay.forward(timer.mark)
        if not a.serve:
            losses.append(lay.loss())
            lay.backward()
            timer.mark(5)
            lay.update()
            timer.mark(6)
        timer.stop()
        if step == 0:
            timer.ms = {s: [] for s in timer.ms}
    lay.forward()
    if not a.serve:
        lay.backward()
    error = lay.product_error()
    us = {s: round(1e3 * v, 1) for s, v in timer.mean().items()}
    rec = {"app": "moe_mx4", "tokens": a.tokens, "experts": a.experts, "topk": a.topk, "d_model": a.d_model, "d_ff": a.d_ff,
           "mode": "serve" if a.serve else "train", "total_us": us.pop("total"), **{f"{s}_us": v for s, v in us.items()},
           "loss": [round(l, 5) for l, _ in losses], "balance_loss": [round(b, 6) for _, b in losses],
           "product_error_over_bound": error}
    print(json.dumps(rec), flush=True)
    return rec


if __name__ == "__main__":
    main()
