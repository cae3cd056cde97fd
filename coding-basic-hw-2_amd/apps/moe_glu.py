"""Mixture-of-experts feed-forward layer with gated experts: router, dispatch, gate and up projections, activation, product,
down projection, combine, and in training the whole backward pass and an update, on the library's router
(include/ggemm_route.h) and gated block (include/ggemm_glu.h); in serving on its 8-bit integer products (include/ggemm_w8.h).
The layer with a tanh and 4-bit products is moe_mx4.py, the FP64 layer moe_ffn.py.

Layer (T tokens, width d, hidden width f, E experts, k per token, rows R = T k and padding):
  route    logits = x Wr;  gates, counts, offsets, order, balance loss                        ggemm_route
  block    Y = (act(X Wg_e^T) * (X Wu_e^T)) Wd_e^T of the rows X = x[order]                   ggemm_glu
  combine  out[t] = sum_j gates[t, j] Y[pos[t, j]]
Backward (loss = mean (out - target)^2 / 2 + balance loss): dY from the combine, then every gradient of the block
(ggemm_glu_backward), gates and loss back to the logits (ggemm_route_backward).  Weights are kept in 32 bits and rounded to
bf16 once per step; a step moves each matrix by lr / 50 of its norm.
Serving (--serve): weights as 8-bit integers with a scale for each output channel, made once; per step the rows x[order] are
quantised (ggemm_w8_quantize), gate and up in one product (ggemm_w8_gemm with an activation), its rows quantised again, the
down product.  --tokens 1 is one decoding step.

Usage: python3 moe_glu.py [--tokens 4096] [--experts 16] [--topk 2] [--d-model 1024] [--d-ff 2048] [--steps 10]
                          [--act silu|gelu|gelu_tanh] [--lr 0.5] [--balance 0.01] [--seed 7] [--serve]
Prints one JSON line: time per step and stage (us), losses, and the relative error of the layer's output against the same
layer in 64 bits from the unrounded weights (routing taken over).
"""
import argparse
import ctypes as C
import json
import sys

import app_util as AU

G = AU.G
STAGES = ("route", "block", "combine", "backward", "update")


def parse_args(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--topk", type=int, default=2)
    ap.add_argument("--d-model", type=int, default=1024)
    ap.add_argument("--d-ff", type=int, default=2048)
    ap.add_argument("--act", choices=sorted(G.ACTS), default="silu")
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
    # rows of every operand begin at multiples of 16 bytes without padding
    if a.d_model < 16 or a.d_ff < 16 or a.d_model % 16 or a.d_ff % 16:
        ap.error("--d-model and --d-ff must be multiples of 16")
    return a


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


class Integers:
    """Rows as 8-bit integers with a scale each."""

    def __init__(self, torch, rows, cols):
        self.rows, self.cols = rows, cols
        self.q, self.scales = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")

    def of(self, x, index=None):
        """Quantises the rows of x, or its rows index[0], index[1], ... (-1: zeros)."""
        kind = {"torch.float32": G.F32, "torch.bfloat16": G.BF16}[str(x.dtype)]
        p = G.W8Quant(self.rows, self.cols, kind, x.shape[0], x.data_ptr(), x.stride(0), index.data_ptr() if index is not None else None,
                      self.q.data_ptr(), self.cols, self.scales.data_ptr())
        G.check(G.lib().ggemm_w8_quantize(C.byref(p), stream()), "ggemm_w8_quantize")
        return self


class Layer:
    def __init__(self, a, torch):
        self.a, self.torch = a, torch
        gen = torch.Generator(device="cuda")
        gen.manual_seed(a.seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)   # noqa: E731
        T, E, k, d, f = a.tokens, a.experts, a.topk, a.d_model, a.d_ff
        self.R = T * k                              # the grouped products need no padding
        self.x, self.target = rand(T, d).bfloat16(), rand(T, d)
        self.Wr, self.Wg, self.Wu = rand(d, E) / d ** 0.5, rand(E * f, d) / d ** 0.5, rand(E * f, d) / d ** 0.5
        self.Wd = rand(E * d, f) / f ** 0.5
        i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")   # noqa: E731
        f32 = lambda *s: torch.empty(*s, device="cuda")                      # noqa: E731
        b16 = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")   # noqa: E731
        self.ids, self.pos, self.gates = i32(T, k), i32(T, k), f32(T, k)
        self.counts, self.offsets, self.order, self.used = i32(E), i32(E + 1), i32(self.R), i32(1)
        self.probs, self.balance = f32(E), f32(1)
        self.Y = b16(self.R, d)
        self.route_ws = torch.empty(G.lib().ggemm_route_workspace(T, E, k), dtype=torch.uint8, device="cuda")
        self.ws = torch.empty(0, dtype=torch.uint8, device="cuda")
        if a.serve:
            self.Wgq, self.Wuq, self.Wdq = (Integers(torch, *w.shape).of(w) for w in (self.Wg, self.Wu, self.Wd))
            self.Xq, self.Hq, self.H = Integers(torch, self.R, d), Integers(torch, self.R, f), b16(self.R, f)
        else:
            self.gate, self.up, self.dx = b16(self.R, f), b16(self.R, f), b16(self.R, d)
            self.gWg, self.gWu, self.gWd = f32(E * f, d), f32(E * f, d), f32(E * d, f)
            self.round_weights()

    def round_weights(self):
        self.Wgb, self.Wub, self.Wdb = (w.bfloat16() for w in (self.Wg, self.Wu, self.Wd))

    def workspace(self, need):
        if need > self.ws.numel():
            self.ws = self.torch.empty(need, dtype=self.torch.uint8, device="cuda")
        return self.ws.data_ptr(), self.ws.numel()

    def route(self):
        a = self.a
        self.logits = self.x.float() @ self.Wr
        self.r = G.Router(a.tokens, a.experts, a.topk, 1, G.F32, 1, a.balance, self.R, self.logits.data_ptr(), a.experts, None,
                          *[v.data_ptr() for v in (self.ids, self.gates, self.pos, self.counts, self.offsets, self.order, self.used,
                                                   self.probs, self.balance)])
        G.check(G.lib().ggemm_route(C.byref(self.r), self.route_ws.data_ptr(), self.route_ws.numel(), stream()), "ggemm_route")

    def block(self):
        """The library's description of the experts' block."""
        a, p = self.a, lambda t: t.data_ptr()   # noqa: E731
        d, f = a.d_model, a.d_ff
        return G.Glu(a.experts, self.R, d, f, G.BF16, G.ACTS[a.act], a.tokens, p(self.x), d, p(self.order), p(self.offsets), p(self.Wgb),
                     p(self.Wub), d, f * d, p(self.Wdb), f, d * f, p(self.gate), p(self.up), f, p(self.Y), d)

    def product(self, A, B, n, k, out, act=0, B2=None):
        """out = A B_e^T for each expert's rows, or act of it times A B2_e^T."""
        p = G.W8Gemm(self.a.experts, self.R, n, k, G.BF16, act, A.q.data_ptr(), k, A.scales.data_ptr(), B.q.data_ptr(),
                     B2.q.data_ptr() if B2 else None, k, n * k, B.scales.data_ptr(), B2.scales.data_ptr() if B2 else None, n,
                     self.offsets.data_ptr(), out.data_ptr(), n)
        G.check(G.lib().ggemm_w8_gemm(C.byref(p), *self.workspace(G.lib().ggemm_w8_gemm_workspace(C.byref(p))), stream()), "ggemm_w8_gemm")

    def forward(self, mark=lambda i: None):
        a = self.a
        self.route()
        mark(0)
        if a.serve:
            self.Xq.of(self.x, self.order)
            self.product(self.Xq, self.Wgq, a.d_ff, a.d_model, self.H, G.ACTS[a.act], self.Wuq)
            self.Hq.of(self.H)
            self.product(self.Hq, self.Wdq, a.d_model, a.d_ff, self.Y)
        else:
            p = self.block()
            G.check(G.lib().ggemm_glu(C.byref(p), *self.workspace(G.lib().ggemm_glu_workspace(C.byref(p))), stream()), "ggemm_glu")
        mark(1)
        self.picked = self.Y[self.pos.long()].float()                       # T x k x d
        self.out = (self.picked * self.gates[..., None]).sum(1)
        mark(2)
        return self.out

    def backward(self):
        a, t = self.a, self.torch
        T, E, d, f = a.tokens, a.experts, a.d_model, a.d_ff
        d_out = (self.out - self.target) / (T * d)
        d_gates = (self.picked * d_out[:, None]).sum(-1).contiguous()
        gate = t.empty(self.R, device="cuda")
        gate[self.pos.view(-1).long()] = self.gates.view(-1)
        # bf16 has the exponents of 32 bits: gradients of this size need no scale of their own
        self.dY = (d_out[self.order.long()] * gate[:, None]).bfloat16()
        p = self.block()
        q = G.GluGrad(self.dY.data_ptr(), d, self.dx.data_ptr(), d, G.F32, 0.0, self.gWg.data_ptr(), self.gWu.data_ptr(), d, f * d,
                      self.gWd.data_ptr(), f, d * f)
        need = G.lib().ggemm_glu_backward_workspace(C.byref(p), C.byref(q))
        G.check(G.lib().ggemm_glu_backward(C.byref(p), C.byref(q), *self.workspace(need), stream()), "ggemm_glu_backward")
        d_logits, one = t.empty(T, E, device="cuda"), t.ones(1, device="cuda")
        G.check(G.lib().ggemm_route_backward(C.byref(self.r), d_gates.data_ptr(), one.data_ptr(), d_logits.data_ptr(), E, stream()),
                "ggemm_route_backward")
        self.gWr = self.x.float().t() @ d_logits
        self.gx = self.dx[self.pos.long()].float().sum(1) + d_logits @ self.Wr.t()

    def update(self):
        """Each matrix moves against its gradient by lr / 50 of its own norm, whatever the gradient's."""
        for w, g in ((self.Wg, self.gWg), (self.Wu, self.gWu), (self.Wd, self.gWd), (self.Wr, self.gWr)):
            w -= (0.02 * self.a.lr * w.norm() / (g.norm() + 1e-30)) * g
        self.round_weights()

    def loss(self):
        return float(((self.out - self.target) ** 2).mean() / 2), float(self.balance)

    def exact(self):
        """The layer's output in 64 bits from the unrounded weights, the routing taken over; also the leaves it was made of."""
        a, t = self.a, self.torch
        d, f = a.d_model, a.d_ff
        leaf = {n: getattr(self, n).double().requires_grad_(True) for n in ("x", "Wr", "Wg", "Wu", "Wd")}
        ids, logits = self.ids.long(), leaf["x"] @ leaf["Wr"]
        gates = t.softmax(logits.gather(1, ids), 1)
        act = {"silu": t.nn.functional.silu, "gelu": t.nn.functional.gelu,
               "gelu_tanh": lambda v: t.nn.functional.gelu(v, approximate="tanh")}[a.act]
        out = t.zeros(a.tokens, d, dtype=t.float64, device="cuda")
        for e in range(a.experts):
            at, j = (ids == e).nonzero(as_tuple=True)
            if len(at):
                xe = leaf["x"][at]
                g, u = xe @ leaf["Wg"][e * f:(e + 1) * f].t(), xe @ leaf["Wu"][e * f:(e + 1) * f].t()
                out = out.index_add(0, at, ((act(g) * u) @ leaf["Wd"][e * d:(e + 1) * d].t()) * gates[at, j][:, None])
        share = self.counts.double() / (a.topk * a.tokens)
        balance = a.balance * a.experts * (share * t.softmax(logits, 1).mean(0)).sum()
        return out, balance, leaf


def main(argv=None):
    a = parse_args(argv)
    import torch
    if not torch.cuda.is_available():
        sys.exit("moe_glu: no GPU")
    lay = Layer(a, torch)
    stages = STAGES[:3] if a.serve else STAGES
    timer, losses = AU.StageTimer(torch, stages), []
    for step in range(a.steps + 1):      # the first one warms up
        timer.start()
        lay.forward(timer.mark)
        if not a.serve:
            losses.append(lay.loss())
            lay.backward()
            timer.mark(3)
            lay.update()
            timer.mark(4)
        timer.stop()
        if step == 0:
            timer.ms = {s: [] for s in timer.ms}
    out = lay.forward().double()
    with torch.no_grad():
        want = lay.exact()[0]
    us = {s: round(1e3 * v, 1) for s, v in timer.mean().items()}
    rec = {"app": "moe_glu", "tokens": a.tokens, "experts": a.experts, "topk": a.topk, "d_model": a.d_model, "d_ff": a.d_ff, "act": a.act,
           "mode": "serve" if a.serve else "train", "total_us": us.pop("total"), **{f"{s}_us": v for s, v in us.items()},
           "loss": [round(v, 5) for v, _ in losses], "balance_loss": [round(b, 6) for _, b in losses],
           "relative_error": float((out - want).norm() / want.norm())}
    print(json.dumps(rec), flush=True)
    return rec


if __name__ == "__main__":
    main()
