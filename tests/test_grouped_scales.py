"""Products of what mxfp4_quantize gives, in every form: blocks of zeros, whose scale is
2^-127, among the weights and the rows, and rows of every magnitude."""
import pytest
import torch

import experts_reference as ref
from inferno_amd import ops
from test_grouped_forms import FORMS, TYPES, _call

F32, U8 = torch.float32, torch.uint8
MX = [(t, f) for t, f in FORMS if t != "bf16" and f.endswith("/1")]


class Given:
    """One matrix per expert, or one: codes, scales and what they stand for."""

    def __init__(self, codes, scales):
        self.parts, self.values = (codes.cuda(), scales.cuda()), ref.values(codes, scales)

    def of(self, e):
        return self.values if self.values.dim() == 2 else self.values[e]


def _sparse(g, *shape):
    """Normal values, of which whole blocks of 32, whole rows and single values are 0,
    of either sign."""
    v = torch.randn(*shape, generator=g)
    v.view(*shape[:-1], -1, 32)[torch.rand(*shape[:-1], shape[-1] // 32, generator=g) < 0.4] *= 0.0
    v[..., ::7, :] *= 0.0
    v[torch.rand(*shape, generator=g) < 0.1] *= 0.0
    return v


@pytest.mark.gpu
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("types,form", MX)
def test_blocks_of_zeros(cuda, monkeypatch, types, form, mats):
    monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
    x4 = TYPES[types][1]
    g = torch.Generator().manual_seed(mats)
    E, N, K, counts = 4, 149, 608, [1, 150, 0, 49]
    m = []
    for _ in range(mats):
        codes, scales = ops.mxfp4_quantize(_sparse(g, E * N, K).cuda())
        assert (scales == 0).float().mean() > 0.3 and (codes & 8).any()
        m.append(Given(codes.view(E, N, K // 2).cpu(), scales.view(E, N, K // 32).cpu()))
    x = _sparse(g, sum(counts), K)
    if x4:
        given = ops.mxfp4_quantize(x.cuda())
        xv = ref.values(*given)
    else:
        given, xv = (x.to(torch.bfloat16).cuda(),), x.to(torch.bfloat16).double()
    offsets = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32)
    got = _call(m, given, offsets=offsets.cuda(), out_dtype=F32)
    want, bar, hit = ref.expected(m, xv, len(x), 1, offsets, None, F32)
    assert hit.all() and (want == 0).all(1).any() and (want[1:151] == 0).all(0).any()
    ref.near(got, want, bar)
    assert torch.equal(got.cpu() == 0, want == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("types,form", MX)
def test_zeros_of_any_scale(cuda, monkeypatch, types, form):
    """The scale of a block of zeros counts for nothing."""
    monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
    x4 = TYPES[types][1]
    g = torch.Generator().manual_seed(3)
    N, K, T = 255, 96, 100
    m = ref.Mats(g, N, K, 0, True)
    codes, scales = (t.cpu() for t in m.parts)
    codes[:, 16:32] = torch.tensor([0x00, 0x80, 0x08, 0x88], dtype=U8).repeat(4)
    scales[:, 1] = torch.arange(N, dtype=U8)  # 0 to 254
    given, xv = ref.rows(g, T, K, x4)
    want, bar, _ = ref.expected([Given(codes, scales)], xv, T, 1, None, None, F32)
    got = _call([Given(codes, scales)], given)
    ref.near(got, want, bar)
    if x4:
        c, s = (t.cpu() for t in given)
        c[:, :16], s[:, 0] = 0, torch.linspace(0, 254, T).to(U8)
        want, bar, _ = ref.expected([Given(codes, scales)], ref.values(c, s), T, 1, None, None, F32)
        ref.near(_call([Given(codes, scales)], (c.cuda(), s.cuda())), want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("types,form", [(t, f) for t, f in MX if TYPES[t][1]])
def test_rows_of_every_magnitude(cuda, monkeypatch, types, form):
    """A row's scales from 2^-127 to 2^105, as of values from fp32's subnormal ones on,
    by weights of 2^-9 to 2^-5 (and by 2^90, where small rows come out in the middle of
    the range)."""
    monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
    g = torch.Generator().manual_seed(9)
    N, K, T = 70, 160, 233
    codes = torch.randint(0, 256, (T, K // 2), generator=g, dtype=U8)
    scales = torch.arange(T, dtype=U8).view(T, 1).expand(T, K // 32).contiguous()
    xv, given = ref.values(codes, scales), (codes.cuda(), scales.cuda())
    m = ref.Mats(g, N, K, 0, True)
    want, bar, _ = ref.expected([m], xv, T, 1, None, None, F32)
    ref.near(_call([m], given), want, bar)
    loud = Given(m.parts[0].cpu(), m.parts[1].cpu() + 97)
    few = 120  # rows up to 2^-8: products below 2^100
    want, bar, _ = ref.expected([loud], xv[:few], few, 1, None, None, F32)
    ref.near(_call([loud], tuple(t[:few].contiguous() for t in given)), want, bar)
