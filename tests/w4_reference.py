"""4-bit weights in 64 bits, and how far the products may be from them.

Bars, each from the roundings that the entry points document. With
S = sum |w x| and M = sum over 128-column chunks of max |x| sum |w|:
  - an fp32 or bf16 activation is off by at most 2^-23 of its chunk's largest
    value (int8 ones are exact): 2^-23 M;
  - codes times digits are summed exactly in a group; joining the digits'
    sums rounds at most 5 times, a scale and an activation scale once each, and
    the fp32 additions are at most 4 per chunk, ceil(K / 128) chunks, 4 parts
    and 2 residuals, each rounding a partial sum of size at most S (plus the
    residuals): (4 ceil(K / 128) + 16) 2^-24 (S + |a| + |b|).
    Calls of many fp32 or bf16 tokens sum a chunk's products of fp16 values in
    fp32 instead, which may round 128 or 256 times per chunk; they are held to
    the same bar, since roundings of either sign seldom add up to four steps.
silu(g) has a slope of at most 1.1 and is formed with at most 8 roundings."""
import math

import torch

U = 2.0 ** -24


def make(g, rows, cols, group, experts=0, zeros=False, scales=torch.bfloat16, device="cuda",
         scale=0.01):
    """Codes, scales and zero points of one matrix or of one per expert."""
    lead = (experts,) if experts else ()
    codes = torch.randint(0, 256, (*lead, rows, cols // 2), generator=g, dtype=torch.uint8)
    s = scale * torch.exp(0.3 * torch.randn(*lead, rows, cols // group, generator=g))
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    return tuple(None if t is None else t.to(device) for t in (codes, s.to(scales), z))


def dense(codes, scales, zeros=None):
    codes, scales = codes.cpu(), scales.cpu()
    cols = 2 * codes.shape[-1]
    q = torch.empty(*codes.shape[:-1], cols, dtype=torch.float64)
    q[..., 0::2] = (codes & 15).double()
    q[..., 1::2] = (codes >> 4).double()
    of = torch.arange(cols) // (cols // scales.shape[-1])
    q -= 8.0 if zeros is None else zeros.cpu().clamp(max=127).double()[..., of]
    return q * scales.double()[..., of]


def values(x, x_scales=None):
    x = x.cpu().double()
    if x_scales is None:
        return x
    s = x_scales.cpu().double()
    return x * s[:, torch.arange(x.shape[1]) // (x.shape[1] // s.shape[1])]


def linear(w, x, rounded=True, extra=0.0, x_err=None):
    """(x w^T, its bar); x_err: how far each x may be off by itself."""
    K = x.shape[1]
    C = math.ceil(K / 128)
    a = w.abs()
    bar = (4 * C + 16) * U * (x.abs() @ a.T + extra)
    if rounded:
        pad = torch.nn.functional.pad(x.abs(), (0, 128 * C - K)).view(-1, C, 128)
        top = pad.amax(2).repeat_interleave(128, 1)[:, :K]
        bar = bar + 2.0 ** -23 * (top @ a.T)
    if x_err is not None:
        bar = bar + x_err @ a.T
    return x @ w.T, bar


def swiglu(wg, wu, x, rounded=True):
    g, dg = linear(wg, x, rounded)
    u, du = linear(wu, x, rounded)
    s = g * torch.sigmoid(g)
    return s * u, 1.1 * dg * u.abs() + s.abs() * du + 1.1 * dg * du + 8 * U * (s * u).abs()


def moe(gate, up, down, x, ids, weights, k, rounded=True):
    """Routed experts and their bar; ids of no expert count nothing. gate, up
    and down are lists of one matrix per expert."""
    T = x.shape[0]
    out = torch.zeros(T, down[0].shape[0], dtype=torch.float64)
    bar = torch.zeros_like(out)
    size = torch.zeros_like(out)
    ids, weights = ids.view(T, k).cpu(), weights.view(T, k).cpu().double()
    for e in range(len(gate)):
        t, r = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        h, dh = swiglu(gate[e], up[e], x[t], rounded)
        w = weights[t, r].unsqueeze(1)
        h, dh = h * w, dh * w.abs() + 2 * U * (h * w).abs()
        y, dy = linear(down[e], h, True, x_err=dh)
        out.index_add_(0, t, y)
        bar.index_add_(0, t, dy)
        size.index_add_(0, t, y.abs())
    return out, bar + (k + 1) * U * size
