"""Residual addition, RMSNorm and 8-bit activations (inferno_add_rms_norm_q8)
against the definition in 64 bits.

Bars. The sum is one fp32 addition: equal. q is the rounded quotient of two
products that 64 bits hold exactly, one division: equal. The root, if the
squares were summed in 32 bits: a thread adds at most ceil(H / 256) of them one
after another and the 256 sums are added in at most 12 steps, each rounding by
2^-24 of the (positive) sum; the square root halves that, and mean, eps, root,
quotient and product round once each. So y and the scales are within ((ceil(H / 256) + 12) / 2 + 6) 2^-24 of
themselves, y in bf16 within 2^-8 more."""
import math

import pytest
import torch

from inferno_amd import InfernoError, lib, ops

EPS = 1e-6


def _definition(x, residual, w, eps, group):
    s = x.float() if residual is None else x.float() + residual
    d = s.double()
    root = torch.sqrt(d.square().mean(1, keepdim=True) + eps)
    p = d * w.double()
    v = p.unflatten(1, (-1, group or p.shape[1]))
    top = v.abs().amax(2, keepdim=True)
    q = torch.where(top > 0, torch.round(127.0 * v / top), 0.0).flatten(1).to(torch.int8)
    return s, p / root, q, top.squeeze(2) / root / 127.0


def _bar(H):
    return ((math.ceil(H / 256) + 12) / 2 + 6) * 2.0 ** -24


def _check(x, residual, w, group, act, eps=EPS, out=None):
    s, y, q, sc = _definition(x, residual, w, eps, group)
    got = ops.add_rms_norm_q8(x, residual, w, eps, group=group, act_dtype=act, out=out)
    bar = _bar(x.shape[1])
    assert torch.equal(got[0], s)
    assert got[1].dtype == act
    wide = bar + (2.0 ** -8 if act == torch.bfloat16 else 0.0)
    assert ((got[1].double() - y).abs() <= wide * y.abs() + 1e-44).all()
    assert torch.equal(got[2], q)
    assert ((got[3].double() - sc).abs() <= bar * sc + 1e-44).all()
    return got


def _inputs(T, H, x_dtype, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (std * torch.randn(T, H, generator=g, device="cuda")).to(x_dtype)
    r = std * torch.randn(T, H, generator=g, device="cuda")
    r[:, ::97] *= 20.0  # a few loud channels
    w = 1.0 + 0.2 * torch.randn(H, generator=g, device="cuda")
    return x, r, w


@pytest.mark.gpu
@pytest.mark.parametrize("x_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,group", [(1, 2048, 0), (1, 2048, 128), (3, 1, 0), (2, 7, 0),
                                       (5, 96, 32), (61, 2816, 128), (17, 320, 64), (4, 4097, 0),
                                       (2, 6144, 0), (3, 8192, 32), (2, 9216, 128), (2, 20000, 0),
                                       (1, 33000, 0), (1, 65536, 128), (300, 512, 0)])
def test_against_the_definition(cuda, T, H, group, x_dtype, act):
    x, r, w = _inputs(T, H, x_dtype)
    _check(x, r, w, group, act)
    _check(x, None, w, group, act)


@pytest.mark.gpu
@pytest.mark.parametrize("H,group", [(512, 0), (512, 128), (4099, 0), (512, 32)])
@pytest.mark.parametrize("std", [1e-30, 1e-12, 1e12, 1e18])
def test_sizes_of_the_values(cuda, H, group, std):
    # squares leave fp32's range on both sides
    x, r, w = _inputs(4, H, torch.float32, seed=3, std=std)
    _check(x, r, w, group, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [0, 32, 128])
def test_borders_between_two_values(cuda, group):
    # the largest value is 254 steps, so that the odd ones lie on borders
    # exactly: ties go to even
    H = 512
    i = torch.arange(H, device="cuda")
    x = ((i * 37) % 509 - 254).clamp(-254, 254).float().unsqueeze(0).repeat(3, 1)
    x[:, ::32] = 254.0
    got = _check(x * 2.0 ** -5, None, torch.ones(H, device="cuda"), group, torch.float32)
    assert (got[2].double() * 2 == x.double()).float().mean() < 0.6  # there were ties


@pytest.mark.gpu
@pytest.mark.parametrize("H,group", [(512, 0), (512, 64), (515, 0)])
def test_rows_of_zeros_and_not_finite(cuda, H, group):
    x, r, w = _inputs(6, H, torch.float32, seed=5)
    x[1], r[1] = 0.0, 0.0
    x[2, 5] = float("nan")
    x[3, 100] = float("inf")
    x[4, 100] = float("-inf")
    s, y, q, sc = ops.add_rms_norm_q8(x, r, w, EPS, group=group)
    assert not y[1].any() and not q[1].any() and not sc[1].any()
    n = group or H
    for t, c in ((2, 5), (3, 100), (4, 100)):
        at = c // n
        assert not q[t, at * n:(at + 1) * n].any()
        assert not sc[t, at].isfinite()
    for t in (0, 5):  # the other rows are as if alone
        one = ops.add_rms_norm_q8(x[t:t + 1].clone(), r[t:t + 1].clone(), w, EPS, group=group)
        for a, b in zip((s, y, q, sc), one):
            assert torch.equal(a[t:t + 1], b)


@pytest.mark.gpu
@pytest.mark.parametrize("H,group", [(512, 0), (512, 64), (515, 0), (16384, 128)])
def test_rows_of_zeros_without_eps(cuda, H, group):
    x, r, w = _inputs(4, H, torch.float32, seed=6)
    x[1], r[1] = 0.0, -0.0
    x[2, :] = -r[2]  # a sum of zeros
    s, y, q, sc = ops.add_rms_norm_q8(x, r, w, 0.0, group=group)
    for t in (1, 2):
        assert not s[t].any() and not y[t].any() and not q[t].any() and not sc[t].any()
    _check(x[[0, 3]], r[[0, 3]], w, group, torch.float32, eps=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("H,group", [(512, 0), (512, 64), (515, 0), (16384, 128)])
@pytest.mark.parametrize("size", [1e-44, 1e-42, 1e-40, 1e-38, 1e37, 9e37])
def test_rows_whose_factor_leaves_the_range(cuda, H, group, size):
    # 1 / sqrt(mean(s^2)) beyond fp32's largest value, or below its normal ones
    g = torch.Generator(device="cuda").manual_seed(H)
    x = size * (1.0 + torch.rand(3, H, generator=g, device="cuda"))
    w = 1.0 + 0.2 * torch.randn(H, generator=g, device="cuda")
    for act in (torch.float32, torch.bfloat16):
        _check(x, None, w, group, act, eps=0.0)
        _check(x, torch.full_like(x, -0.5 * size), w, group, act, eps=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("H,group", [(2048, 128), (515, 0), (40000, 0)])
def test_the_sum_in_place(cuda, H, group):
    x, r, w = _inputs(3, H, torch.float32, seed=7)
    want = ops.add_rms_norm_q8(x, r, w, EPS, group=group)
    stream = r.clone()
    got = ops.add_rms_norm_q8(x, stream, w, EPS, group=group, out=stream)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(stream, want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("H,group", [(2048, 128), (515, 0), (1028, 0), (6144, 32), (40000, 0)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_the_sum_over_x(cuda, H, group, with_residual):
    x, r, w = _inputs(7, H, torch.float32, seed=8)
    r = r if with_residual else None
    want = ops.add_rms_norm_q8(x, r, w, EPS, group=group)
    for _ in range(3):
        stream = x.clone()
        got = ops.add_rms_norm_q8(stream, r, w, EPS, group=group, out=stream)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(stream, want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("H,group", [(256, 64), (259, 0)])
def test_outputs_left_out_and_pointers_off_alignment(cuda, H, group):
    # every output but one left out; inputs and outputs one element past an
    # aligned address; what lies around the outputs stays
    T = 3
    x, r, w = _inputs(T, H, torch.float32, seed=9)
    s, y, q, sc = ops.add_rms_norm_q8(x, r, w, EPS, group=group)

    def off(t):
        buf = torch.full((t.numel() + 2,), 77, dtype=t.dtype, device="cuda")
        buf[1:-1] = t.flatten()
        return buf, buf[1:].data_ptr()

    (bx, px), (br, pr), (bw, pw) = off(x), off(r), off(w)
    st = torch.cuda.current_stream().cuda_stream
    for keep in ("s", "y", "q"):
        outs = {n: off(torch.zeros_like(t)) for n, t in dict(s=s, y=y, q=q, sc=sc).items()}
        ptr = {n: o[1] if n == keep or (keep == "q" and n == "sc") else None
               for n, o in outs.items()}
        assert lib().inferno_add_rms_norm_q8(st, px, 0, pr, pw, EPS, T, H, group, 0, ptr["s"],
                                             ptr["y"], ptr["q"], ptr["sc"]) == 0
        torch.cuda.synchronize()
        for n, t in dict(s=s, y=y, q=q, sc=sc).items():
            buf = outs[n][0]
            assert buf[0] == 77 and buf[-1] == 77
            assert torch.equal(buf[1:-1].view(t.shape), t if ptr[n] else torch.zeros_like(t))


def test_refusals():
    x, w = torch.zeros(2, 96), torch.zeros(96)
    with pytest.raises(ValueError, match="GPU tensors"):
        ops.add_rms_norm_q8(x, None, w, EPS)
    with pytest.raises(ValueError, match="group"):
        ops.add_rms_norm_q8(x, None, w, EPS, group=48)
    with pytest.raises(ValueError, match="group"):
        ops.add_rms_norm_q8(x, None, w, EPS, group=128)
    with pytest.raises(ValueError, match="contiguous"):
        ops.add_rms_norm_q8(torch.zeros(96, 2).T, None, w, EPS)
    with pytest.raises(ValueError, match="residual"):
        ops.add_rms_norm_q8(x, torch.zeros(2, 95), w, EPS)
    with pytest.raises(ValueError, match="residual"):
        ops.add_rms_norm_q8(x, torch.zeros(2, 96, dtype=torch.bfloat16), w, EPS)
    with pytest.raises(ValueError, match="out"):
        ops.add_rms_norm_q8(x, None, w, EPS, out=torch.zeros(3, 96))
    with pytest.raises(ValueError, match="x must"):
        ops.add_rms_norm_q8(x.half(), None, w, EPS)
    with pytest.raises(ValueError, match="act_dtype"):
        ops.add_rms_norm_q8(x, None, w, EPS, act_dtype=torch.float16)
    f = lib().inferno_add_rms_norm_q8
    assert f(None, 16, 0, None, 16, EPS, 1, 96, 0, 0, 16, 16, 16, None) == -1
    assert b"together" in lib().inferno_last_error()
    assert f(None, 16, 2, None, 16, EPS, 1, 96, 0, 0, 16, 16, 16, 16) == -1
    assert f(None, 16, 0, None, 16, EPS, 1, 96, 48, 0, 16, 16, 16, 16) == -1
    assert f(None, 16, 0, None, 16, float("nan"), 1, 96, 0, 0, 16, 16, 16, 16) == -1
    assert f(None, 16, 0, None, 16, EPS, 1, 0, 0, 0, 16, 16, 16, 16) == -1
    assert f(None, None, 0, None, 16, EPS, 1, 96, 0, 0, 16, 16, 16, 16) == -1
    assert f(None, 16, 0, None, 16, EPS, 1 << 24, 96, 0, 0, 16, 16, 16, 16) == -1
    assert f(None, None, 0, None, None, EPS, 0, 96, 0, 0, None, None, None, None) == 0


@pytest.mark.gpu
def test_no_rows(cuda):
    out = ops.add_rms_norm_q8(torch.zeros(0, 64, device=cuda), None, torch.ones(64, device=cuda),
                              EPS, group=32)
    assert [tuple(t.shape) for t in out] == [(0, 64), (0, 64), (0, 64), (0, 2)]
    with pytest.raises(InfernoError, match="eps"):
        ops.add_rms_norm_q8(torch.zeros(1, 64, device=cuda), None, torch.ones(64, device=cuda), -1.0)
