"""Quantisation to MXFP4 against its definition in 64 bits: codes, scales and the
values that they stand for are equal."""
import pytest
import torch

import experts_reference as ref
from inferno_amd import InfernoError, lib, ops

F32, BF16, U8 = torch.float32, torch.bfloat16, torch.uint8


def _check(x):
    codes, scales, held = ops.mxfp4_quantize(x, values=True)
    c, s = ops.mxfp4_quantize(x)
    assert torch.equal(c, codes) and torch.equal(s, scales)
    want_c, want_s, want_v = ref.quantize(x)
    assert torch.equal(scales.cpu(), want_s)
    assert torch.equal(codes.cpu(), want_c)
    assert held.dtype == x.dtype
    got = held.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want_v))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want_v))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 2048), (3, 96), (5, 64), (77, 2848), (300, 160)])
def test_quantize(cuda, rows, cols, dtype):
    g = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(6.0 * torch.randn(rows, 1, generator=g))
    x[:, ::61] *= 12.0
    _check(x.to(dtype).cuda())


@pytest.mark.gpu
def test_every_bf16_value(cuda):
    """All finite values, each in blocks where it is the largest, and where a
    larger one makes it small, subnormal or half of a code's step."""
    bits = torch.arange(65536, dtype=torch.int32)
    v = (bits << 16).view(F32)
    v = v[torch.isfinite(v)]
    x = torch.zeros(v.numel(), 32)
    x[:, 0] = v
    for j, f in enumerate([1.0, 0.75, 0.5, 0.4375, 0.375, 0.3125, 0.25, 0.21875, 0.1875, 0.125,
                           0.09375, 0.0625, 0.03125, 0.015625]):
        x[:, 1 + 2 * j] = f * v
        x[:, 2 + 2 * j] = -f * v
    _check(x.to(BF16).cuda())
    _check(x.cuda())


@pytest.mark.gpu
def test_values_next_to_a_border(cuda):
    """fp32 values at halfway points, and one step to either side."""
    half = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0])
    near = torch.stack([half, torch.nextafter(half, half * 2), torch.nextafter(half, half * 0)], 1)
    block = torch.zeros(32)
    block[:27] = near.reshape(-1)
    block[27] = torch.nextafter(torch.tensor(8.0), torch.tensor(0.0))
    block[28:] = torch.tensor([4.0, -0.0, 1e-30, -1e-30])
    scale = torch.exp2(torch.arange(-126, 124, dtype=torch.float64)).float()
    x = torch.cat([block * s for s in scale]).view(-1, 32)
    _check(torch.cat([x, -x]).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_zeros_subnormals_and_not_finite(cuda, dtype):
    x = torch.zeros(12, 64)
    x[1, :32] = -0.0
    x[2, 5] = 1e-45 if dtype == F32 else 1e-40
    x[3] = torch.linspace(-1e-38, 1e-38, 64)
    x[4] = torch.linspace(-3e-38, 3e-38, 64)
    x[5, 40] = float("inf")
    x[6, 3] = float("nan")
    x[6, 40:] = 1.0
    x[7, 31], x[7, 32] = float("-inf"), 2.0
    x[8] = torch.finfo(dtype).max
    x[9, ::2] = -torch.finfo(dtype).max
    x[10, 7] = torch.finfo(dtype).tiny
    _check(x.to(dtype).cuda())


@pytest.mark.gpu
def test_quantize_no_rows_and_only_its_own_output(cuda):
    codes, scales = ops.mxfp4_quantize(torch.empty(0, 64, device="cuda"))
    assert codes.shape == (0, 32) and scales.shape == (0, 2)
    # the library writes nothing behind the last value
    x = torch.randn(3, 96, device="cuda")
    c = torch.full((3 * 48 + 64,), 171, dtype=U8, device="cuda")
    s = torch.full((9 + 64,), 171, dtype=U8, device="cuda")
    v = torch.full((3 * 96 + 64,), 7.0, device="cuda")
    st = lib().inferno_mxfp4_quantize(torch.cuda.current_stream().cuda_stream, x.data_ptr(), 0, 3, 96,
                                      c.data_ptr(), s.data_ptr(), v.data_ptr())
    assert st == 0
    assert (c[144:] == 171).all() and (s[9:] == 171).all() and (v[288:] == 7.0).all()
    want_c, want_s, _ = ref.quantize(x)
    assert torch.equal(c[:144].cpu(), want_c.view(-1)) and torch.equal(s[:9].cpu(), want_s.view(-1))


def test_reference_agrees_with_itself():
    g = torch.Generator().manual_seed(0)
    codes, scales, v = ref.quantize(torch.randn(9, 96, generator=g))
    assert torch.equal(ref.values(codes, scales), v)


def test_quantize_refusals():
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.mxfp4_quantize(torch.zeros(2, 48))
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.mxfp4_quantize(torch.zeros(2, 0))
    with pytest.raises(ValueError, match="contiguous 2-D"):
        ops.mxfp4_quantize(torch.zeros(2, 64, dtype=torch.float16))
    with pytest.raises(ValueError, match="contiguous 2-D"):
        ops.mxfp4_quantize(torch.zeros(64))
    with pytest.raises(ValueError, match="not contiguous"):
        ops.mxfp4_quantize(torch.zeros(64, 64).t())
    with pytest.raises(ValueError, match="GPU"):
        ops.mxfp4_quantize(torch.zeros(2, 64))
    q, at = lib().inferno_mxfp4_quantize, 4096
    for args in [(at, 2, 1, 64, at, at, None), (at, 0, 1, 48, at, at, None),
                 (at, 0, 1, 0, at, at, None), (None, 0, 1, 64, at, at, None),
                 (at, 0, 1, 64, None, at, None), (at, 0, 1, 64, at, None, None),
                 (at + 4, 0, 1, 64, at, at, None), (at, 0, 1, 64, at + 8, at, None),
                 (at, 0, 1, 64, at, at, at + 4), (at, 0, 1 << 31, 1 << 31, at, at, None),
                 (at, 0, 1 << 33, 32, at, at, None)]:
        assert q(None, *args) == -1 and lib().inferno_last_error()
    assert q(None, None, 0, 0, 64, None, None, None) == 0  # no rows
