"""Products grouped by expert at the ends of their stated ranges: many results per input
row, long columns, many weight rows."""
import pytest
import torch

import experts_reference as ref
from inferno_amd import ops

F32, BF16, U8 = torch.float32, torch.bfloat16, torch.uint8
TYPES = {"bf16": (False, False), "mxfp4": (True, False), "mxfp4-mxfp4": (True, True)}


@pytest.fixture(params=["rule", "tiles", "rows"])
def kernels(request, monkeypatch):
    """The kernel that the rule takes, and either one for all sizes."""
    if request.param != "rule":
        monkeypatch.setenv("INFERNO_EXPERTS_TILES", "1" if request.param == "tiles" else "0")


def _whole(g, *shape):
    """Whole numbers from -3 to 3, which bf16 and, with scales of 1, MXFP4 hold."""
    return torch.randint(-3, 4, shape, generator=g).float()


def _packed(v, fp4):
    """A tensor of such values as a product takes it."""
    if not fp4:
        return (v.to(BF16).cuda(),)
    code = torch.tensor([0, 2, 4, 5], dtype=U8)[v.abs().long()] + 8 * (v < 0).to(U8)
    return ((code[..., 0::2] | code[..., 1::2] << 4).contiguous().cuda(),
            torch.full((*v.shape[:-1], v.shape[-1] // 32), 127, dtype=U8, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("T,k", [(3, 13), (7, 1000), (5, 1023), (4098, 1023), (4096, 1024), (9, 1025),
                                 (4092, 1025), (2, 1 << 21), (1, 1 << 22), (1397, 3001)])
def test_many_results_of_an_input_row(cuda, kernels, types, T, k):
    """Sums of whole numbers are exact: each result is its input row's, to the bit."""
    w4, x4 = TYPES[types]
    g = torch.Generator().manual_seed(k)
    E, N, K, A = 3, 4, 32, T * k
    w, x = _whole(g, E, N, K), _whole(g, T, K)
    on_gpu = torch.Generator(device="cuda").manual_seed(k)
    order = torch.randperm(A, generator=on_gpu, device="cuda")
    offsets = torch.tensor([0, A // 3, A // 2, A], dtype=torch.int32, device="cuda")
    got = ops.grouped_matmul(ops.Experts(*_packed(w, w4)), *_packed(x, x4), offsets=offsets,
                             sorted_=order.to(torch.int32), k=k)
    each = torch.stack([x @ w[e].T for e in range(E)]).cuda()  # [E, T, N], exact in fp32
    expert = torch.empty(A, dtype=torch.long, device="cuda")
    expert[order] = (torch.arange(A, device="cuda") >= offsets[1]).long() + \
        (torch.arange(A, device="cuda") >= offsets[2]).long()
    assert torch.equal(got, each[expert, torch.arange(A, device="cuda") // k])


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("T", [1, 37])
def test_long_columns(cuda, kernels, types, mats, T):
    w4, x4 = TYPES[types]
    g = torch.Generator().manual_seed(T)
    N, K = 21, (1 << 20) + 32
    m = [ref.Mats(g, N, K, 0, w4) for _ in range(mats)]
    x, xv = ref.rows(g, T, K, x4)
    if mats == 2:  # gates of some size
        xv = xv * 2.0 ** -6
        if x4:
            x[1].sub_(6)
        else:
            x[0].mul_(2.0 ** -6)
    call = ops.grouped_matmul if mats == 1 else ops.grouped_gate_up_swiglu
    got = call(*(ops.Experts(*t.parts) for t in m), *x, out_dtype=F32)
    want, bar, _ = ref.expected(m, xv, T, 1, None, None, F32)
    ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("T", [1, 20])
def test_many_weight_rows(cuda, kernels, types, T):
    """As many as a matrix may have in bf16, a quarter of them in MXFP4."""
    w4, x4 = TYPES[types]
    N, K = ((1 << 22) - 1, 32) if w4 else (1 << 24, 8)
    g = torch.Generator().manual_seed(T)
    w, x = _whole(g, N, K), _whole(g, T, K)
    got = ops.grouped_matmul(ops.Experts(*_packed(w, w4)), *_packed(x, x4))
    assert torch.equal(got.cpu(), x @ w.T)
