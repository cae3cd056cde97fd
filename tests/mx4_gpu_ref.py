"""64-bit references of the 4-bit operators and the router in torch, on the device of their inputs, for calls of many
rows."""
import torch

import mx4_ref as R

GRID = tuple(float(v) for v in R.GRID)


def scale64(e):
    """2^e in 64 bits, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantise(x):
    """x (rows x cols, finite) -> packed codes and scale bytes, blocks along the rows."""
    x = x.double()
    v = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).view(x.shape[0], -1, 32)
    amax = v.abs().amax(-1)
    e = torch.where(amax > 0, (torch.frexp(amax)[1] - 3).clamp(-127, 127), -127)
    a = v.abs() / scale64(e)[..., None]
    code, dist = torch.zeros_like(a, dtype=torch.uint8), a.clone()
    for i in range(1, 8):
        d = (a - GRID[i]).abs()
        take = (d < dist) | ((d == dist) & (i % 2 == 0))
        code, dist = torch.where(take, i, code), torch.where(take, d, dist)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).view(x.shape[0], -1, 2)
    return code[..., 0] | code[..., 1] << 4, (e + 127).to(torch.uint8)


def values(codes, scales, cols):
    """What packed codes and scale bytes stand for; a byte of 255 makes its block NaN."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=codes.device)
    nib = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1, 32).int()
    s = scales[:, :nib.shape[1]].int()
    v = grid[nib] * torch.where(s < 255, scale64(s - 127), torch.nan)[..., None]
    return v.view(codes.shape[0], -1)[:, :cols].contiguous()


def operand(gen, rows, cols, lo=123, hi=132):
    """Random codes (the last block filled up with zeros) and scale bytes in [lo, hi)."""
    nb = R.up(cols, 32) // 32
    codes = torch.randint(0, 256, (rows, 16 * nb), dtype=torch.uint8, device="cuda", generator=gen)
    if cols % 32:
        keep = torch.arange(32 * nb, device="cuda") < cols
        codes &= (keep[0::2].to(torch.uint8) * 15) | (keep[1::2].to(torch.uint8) * 240)
    scales = torch.full((rows, R.up(nb, 4)), 255, dtype=torch.uint8, device="cuda")
    scales[:, :nb] = torch.randint(lo, hi, (rows, nb), dtype=torch.uint8, device="cuda", generator=gen)
    return codes, scales


def route(x, mask, k, align, renorm, coef):
    """What ggemm_route writes, from logits without NaN and +Inf; also p and the tokens that take part."""
    x = x.double()
    T, E = x.shape
    on = (x > -torch.inf).any(1)
    if mask is not None:
        on &= mask != 0
    top, ids = torch.sort(x, dim=1, descending=True, stable=True)
    ok = on[:, None] & (top[:, :k] > -torch.inf)
    ids = torch.where(ok, ids[:, :k], -1)
    p = torch.where(on[:, None], torch.softmax(torch.where(on[:, None], x, 0.0), 1), 0.0)
    g = torch.where(ok, p.gather(1, ids.clamp(min=0)), 0.0)
    if renorm:
        g = torch.where(ok, g / g.sum(1, keepdim=True), 0.0)
    hit = torch.zeros(T, E, dtype=torch.int64, device=x.device).scatter_add_(1, ids.clamp(min=0), ok.long())
    counts = hit.sum(0)
    offsets = torch.zeros(E + 1, dtype=torch.int64, device=x.device)
    offsets[1:] = ((counts + align - 1) // align * align).cumsum(0)
    row = offsets[:-1] + hit.cumsum(0) - hit                       # of a pair (t, e), if it is one
    pos = torch.where(ok, row.gather(1, ids.clamp(min=0)), -1)
    order = torch.full((T * k + E * (align - 1),), -1, dtype=torch.int64, device=x.device)
    order[pos[ok]] = torch.arange(T, device=x.device)[:, None].expand(T, k)[ok]
    n = int(on.sum())
    probs = p.sum(0) / max(n, 1)
    loss = coef * E * float((counts * probs).sum()) / (k * max(n, 1))
    return dict(ids=ids, gates=g, counts=counts, offsets=offsets, pos=pos, order=order, used=n, probs=probs, loss=loss, p=p, on=on)


def route_gradient(w, k, renorm, coef, d_gates, d_loss):
    """Of d_loss loss + sum d_gates gates; and the magnitude of the formula's terms."""
    p, ids, g = w["p"], w["ids"], w["gates"]
    T, E = p.shape
    n = max(w["used"], 1)
    s = (d_loss * coef * E / (k * n * n) * w["counts"].double()).expand(T, E)
    put = lambda v: torch.zeros_like(p).scatter_add_(1, ids.clamp(min=0), torch.where(ids >= 0, v, 0.0))   # noqa: E731
    if renorm:
        c = put(g * (d_gates - (g * d_gates).sum(1, keepdim=True)))
        cm = put(g * (d_gates.abs() + (g * d_gates.abs()).sum(1, keepdim=True)))
        d, dm = s, s.abs()
    else:
        c = cm = torch.zeros_like(p)
        d, dm = s + put(d_gates), s.abs() + put(d_gates.abs())
    return p * (d - (p * d).sum(1, keepdim=True)) + c, p * (dm + (p * dm).sum(1, keepdim=True)) + cm
