"""MXFP4 and products grouped by expert in 64 bits, on the CPU, and the bars of
their results."""
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


def quantize(x):
    """(codes, scales, values in 64 bits) of rows, from the definition: the nearest
    of the grid's values by distance, of two as near the one with an even code."""
    rows, cols = x.shape
    v = x.double().cpu().view(rows, cols // 32, 32)
    top = v.abs().amax(2)
    bad = ~torch.isfinite(v).all(2)
    _, e = torch.frexp(torch.where(bad | (top == 0), torch.ones_like(top), top))
    power = torch.where(top == 0, torch.full_like(e, -127), e - 3).clamp(min=-127)
    unit = torch.ldexp(torch.ones_like(top), power).unsqueeze(2)
    m = torch.where(bad.unsqueeze(2), torch.zeros_like(v), v / unit)
    far = (m.abs().unsqueeze(3) - GRID).abs()
    near = far == far.amin(3, keepdim=True)
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(3), even.double().argmax(3), near.double().argmax(3))
    value = torch.where(torch.signbit(m), -GRID[code], GRID[code]) * unit
    code = code + 8 * (torch.signbit(m) & ~bad.unsqueeze(2))
    value = torch.where(bad.unsqueeze(2), torch.full_like(value, float("nan")), value)
    code = code.view(rows, cols).to(U8)
    scales = torch.where(bad, torch.full_like(power, 255), power + 127).to(U8)
    return code[:, 0::2] | code[:, 1::2] << 4, scales, value.view(rows, cols)


def values(codes, scales):
    """What codes and scales stand for, in 64 bits."""
    codes, scales = codes.cpu(), scales.cpu()
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = torch.where(q >= 8, -GRID[q & 7], GRID[q & 7])
    s = torch.exp2(scales.double() - 127.0)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return v * s.repeat_interleave(32, -1)


class Mats:
    """Weights of E experts (0: one matrix) in bf16 or MXFP4 and their values."""

    def __init__(self, g, N, K, E=0, fp4=False, device="cuda"):
        shape = ((E,) if E else ()) + (N,)
        if fp4:
            codes = torch.randint(0, 256, (*shape, K // 2), generator=g, dtype=U8)
            scales = torch.randint(118, 123, (*shape, K // 32), generator=g, dtype=U8)
            self.parts = (codes.to(device), scales.to(device))
            self.values = values(codes, scales)
        else:
            w = (0.05 * torch.randn(*shape, K, generator=g)).to(BF16)
            self.parts, self.values = (w.to(device),), w.double()

    def of(self, e):
        return self.values if self.values.dim() == 2 else self.values[e]


def rows(g, R, K, fp4=False, device="cuda"):
    """(the call's x and x_scales, values in 64 bits) of R rows with loud channels."""
    x = torch.randn(R, K, generator=g)
    x[:, ::61] *= 8.0
    if not fp4:
        x = x.to(BF16)
        return (x.to(device),), x.double()
    codes, scales, v = quantize(x)
    return (codes.to(device), scales.to(device)), v


def groups(g, T, k, E, empty=()):
    """Offsets and sorted assignments of T tokens with k different experts each,
    none of them in `empty`."""
    score = torch.randn(T, E, generator=g) + torch.randn(E, generator=g)
    score[:, list(empty)] = -1e9
    ids = score.topk(k, 1).indices.reshape(-1)
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[1:] = torch.bincount(ids, minlength=E).cumsum(0)
    return offsets, ids.argsort(stable=True).to(torch.int32)


# Sums of K exact products in fp32, each addition off by at most a step (2^-23) of
# a partial sum, which the sum of magnitudes S bounds: K 2^-23 S, or less.
def product(w, x, e, r):
    y = x[r] @ w.of(e).T
    return y, w.values.shape[-1] * 2.0 ** -23 * (x[r].abs() @ w.of(e).abs().T)


def expected(mats, x, A, k, offsets, sorted_, dtype):
    """(values, bars, rows that are written) of a grouped product, or with two
    matrices of silu(x gate^T) * (x up^T)."""
    out = torch.zeros(A, mats[0].values.shape[-2], dtype=torch.float64)
    bar, hit = torch.zeros_like(out), torch.zeros(A, dtype=torch.bool)
    begin = [0, A] if offsets is None else offsets.tolist()
    for e in range(len(begin) - 1):
        c = torch.arange(begin[e], max(begin[e], begin[e + 1]))
        a = c if sorted_ is None else sorted_[c].long()
        y, d = product(mats[0], x, e, a // k)
        if len(mats) == 2:
            u, du = product(mats[1], x, e, a // k)
            s = torch.sigmoid(y)
            # |d silu / dg| <= 1.1; the exponential of an argument rounded to 24
            # bits and four more operations
            y, d = y * s * u, 1.1 * d * (u.abs() + du) + (y * s).abs() * du + \
                (8 + y.abs()) * 2.0 ** -23 * (y * s * u).abs()
        out[a], bar[a], hit[a] = y, d, True
    step = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    return out, bar + step * (out.abs() + bar) + 1e-38, hit


def near(got, want, bar):
    worst = ((got.cpu().double() - want).abs() / bar).max().item() if want.numel() else 0.0
    assert worst <= 1.0, worst
