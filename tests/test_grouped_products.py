"""Products of rows grouped by expert, weights in bf16 and MXFP4, against 64 bits
(bars: experts_reference.py), their refusals, and the calls that share a GPU."""
import pytest
import torch

import experts_reference as ref
from inferno_amd import ExpertsDesc, InfernoError, lib, ops

F32, BF16, U8 = torch.float32, torch.bfloat16, torch.uint8
FORMATS = [(False, False), (True, False), (True, True)]  # weights, rows in MXFP4
IDS = ["bf16", "mxfp4", "mxfp4-mxfp4"]


@pytest.fixture(params=["rule", "tiles", "rows"])
def kernels(request, monkeypatch):
    """The kernel that the rule takes, and either one for all sizes."""
    if request.param != "rule":
        monkeypatch.setenv("INFERNO_EXPERTS_TILES", "1" if request.param == "tiles" else "0")


def _call(mats, x, **kw):
    w = [ops.Experts(*m.parts) for m in mats]
    return (ops.grouped_matmul if len(w) == 1 else ops.grouped_gate_up_swiglu)(*w, *x, **kw)


def _cuda(t):
    return None if t is None else t.cuda()


SHAPES = [  # T, k, E, N, K, empty experts
    (1, 1, 1, 16, 32, ()), (1, 1, 1, 1, 256, ()), (1, 2, 4, 17, 96, ()), (1, 8, 64, 48, 160, ()),
    (2, 3, 5, 33, 128, ()), (3, 1, 7, 64, 288, (0, 6)), (5, 2, 3, 130, 512, ()),
    (13, 4, 40, 31, 352, (1, 2, 3, 20)), (16, 1, 2, 128, 1024, (1,)), (17, 1, 1, 20, 640, ()),
    (40, 2, 3, 257, 416, ()), (64, 8, 256, 16, 64, ()), (70, 3, 4, 96, 256, (2,)),
    (130, 1, 2, 256, 384, ()), (300, 2, 5, 129, 224, ()), (257, 4, 6, 272, 544, (0,)),
    (700, 2, 3, 384, 192, ()), (1100, 1, 1, 192, 320, ()), (600, 8, 16, 64, 128, (3, 15))]


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMATS, ids=IDS)
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("T,k,E,N,K,empty", SHAPES)
def test_grouped(cuda, kernels, T, k, E, N, K, empty, mats, w4, x4):
    """Tokens that serve k experts, rows of their own, and rows in the experts' order."""
    g = torch.Generator().manual_seed(T + N + K)
    m = [ref.Mats(g, N, K, E, w4) for _ in range(mats)]
    offsets, sorted_ = ref.groups(g, T, k, E, empty)
    for dtype, by in ((F32, "token"), (BF16, "assignment"), (BF16, "grouped")):
        R, kk = (T, k) if by == "token" else (T * k, 1)
        x, xv = ref.rows(g, R, K, x4)
        s = None if by == "grouped" else sorted_
        got = _call(m, x, offsets=offsets.cuda(), sorted_=_cuda(s), k=kk, out_dtype=dtype)
        want, bar, hit = ref.expected(m, xv, T * k, kk, offsets, s, dtype)
        assert hit.all() and got.dtype == dtype and got.shape == (T * k, N)
        ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMATS, ids=IDS)
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("T,N,K", [(1, 48, 2048), (1, 1285, 96), (2, 16, 32), (9, 40, 1056), (16, 70, 4096),
                                   (33, 96, 224), (65, 33, 512), (129, 260, 192), (520, 300, 160)])
def test_one_matrix(cuda, kernels, T, N, K, mats, w4, x4):
    g = torch.Generator().manual_seed(T + N + K)
    m = [ref.Mats(g, N, K, 0, w4) for _ in range(mats)]
    x, xv = ref.rows(g, T, K, x4)
    for dtype in (F32, BF16):
        got = _call(m, x, out_dtype=dtype)
        want, bar, _ = ref.expected(m, xv, T, 1, None, None, dtype)
        ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("T,N,K", [(1, 5, 8), (3, 16, 24), (20, 33, 136), (150, 130, 72), (260, 24, 1032)])
def test_bf16_columns_of_eight(cuda, kernels, T, N, K, mats):
    g = torch.Generator().manual_seed(T + N + K)
    m = [ref.Mats(g, N, K, 3) for _ in range(mats)]
    offsets, sorted_ = ref.groups(g, T, 2, 3)
    x, xv = ref.rows(g, T, K)
    got = _call(m, x, offsets=offsets.cuda(), sorted_=sorted_.cuda(), k=2, out_dtype=F32)
    want, bar, _ = ref.expected(m, xv, 2 * T, 2, offsets, sorted_, F32)
    ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMATS, ids=IDS)
@pytest.mark.parametrize("counts", [[0, 0, 0, 200], [200, 0, 0, 0], [1, 198, 1, 0], [0, 0, 0, 0],
                                    [16, 16, 16, 16], [17, 15, 33, 31], [128, 1, 129, 127]])
def test_uneven_groups(cuda, kernels, counts, w4, x4):
    g = torch.Generator().manual_seed(sum(counts))
    m = [ref.Mats(g, 80, 192, 4, w4)]
    A = 400  # rows behind the last group stay as they are
    offsets = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32)
    x, xv = ref.rows(g, A, 192, x4)
    for sorted_ in (None, torch.randperm(A, generator=g).to(torch.int32)):
        out = torch.full((A, 80), 7.0, device="cuda")
        got = _call(m, x, offsets=offsets.cuda(), sorted_=_cuda(sorted_), out=out)
        assert got is out
        want, bar, hit = ref.expected(m, xv, A, 1, offsets, sorted_, F32)
        want[~hit], bar[~hit] = 7.0, 1e-30
        ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMATS, ids=IDS)
@pytest.mark.parametrize("A", [40, 900])
def test_offsets_and_indices_out_of_range(cuda, kernels, A, w4, x4):
    """Offsets that no dispatch gives (behind the last row, running back, so that two
    experts' ranges overlap) and indices behind the last row: nothing is read or written
    out of range, and a value is one of its experts' results or left as it was."""
    g = torch.Generator().manual_seed(A)
    m = [ref.Mats(g, 48, 128, 5, w4)]
    x, xv = ref.rows(g, A, 128, x4)
    sorted_ = torch.randperm(A, generator=g).to(torch.int32)
    sorted_[::7] = torch.tensor([A, A + 1, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32).repeat(
        A)[: (A + 6) // 7]
    offsets = torch.tensor([0, A // 2, A // 4, A // 4, A + 100, 2 ** 31 - 1], dtype=torch.int32)
    out = torch.full((A + 64, 48), 7.0, device="cuda")
    _call(m, x, offsets=offsets.cuda(), sorted_=sorted_.cuda(), out=out[:A])
    assert (out[A:] == 7.0).all()
    fine = out[:A].cpu() == 7.0
    for e, (b, c) in enumerate([(0, A // 2), (0, 0), (0, 0), (A // 4, A), (0, 0)]):
        a = sorted_[b:c].long()
        a = a[(a >= 0) & (a < A)]
        y, d = ref.product(m[0], xv, e, a)
        fine[a] |= (out[a.cuda()].cpu() - y).abs() <= d + 2.0 ** -24 * y.abs()
    assert fine.all()


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMATS, ids=IDS)
@pytest.mark.parametrize("T", [3, 40, 500])
def test_not_finite_rows_change_their_own_results(cuda, kernels, T, w4, x4):
    g = torch.Generator().manual_seed(T)
    m = [ref.Mats(g, 40, 160, 2, w4)]
    x, _ = ref.rows(g, T, 160, x4)
    offsets = torch.tensor([0, T // 2, T], dtype=torch.int32).cuda()
    clean = _call(m, x, offsets=offsets)
    bad = [t.clone() for t in x]
    if x4:
        bad[1][1, 4] = 255
    else:
        bad[0][1, 159] = float("nan")
        bad[0][T - 1, 3] = float("inf")
    got = _call(m, bad, offsets=offsets)
    assert torch.isnan(got[1]).all()
    last = T - (0 if x4 else 1)
    assert not torch.isfinite(got[last:]).any()
    assert torch.equal(got[2:last], clean[2:last]) and torch.equal(got[0], clean[0])


@pytest.mark.gpu
@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("T", [2, 40, 300])
def test_weights_of_scale_255_are_nan(cuda, kernels, T, x4):
    g = torch.Generator().manual_seed(T)
    m = ref.Mats(g, 50, 256, 2, True)
    x, _ = ref.rows(g, T, 256, x4)
    offsets = torch.tensor([0, T // 2, T], dtype=torch.int32).cuda()
    clean = _call([m], x, offsets=offsets)
    m.parts[1][1, 17, 3] = 255
    got = _call([m], x, offsets=offsets)
    assert torch.isnan(got[T // 2:, 17]).all()
    got[T // 2:, 17] = clean[T // 2:, 17]
    assert torch.equal(got, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("T", [1, 30, 300])
def test_scales_over_the_stated_range(cuda, kernels, T, x4):
    """Weights of scales from 2^-100 to 2^100, one size a row."""
    g = torch.Generator().manual_seed(T)
    m = ref.Mats(g, 201, 96, 0, True)
    m.parts[1].copy_((27 + torch.arange(201, dtype=U8)).view(201, 1).expand(201, 3))
    m.values = ref.values(*m.parts)
    x, xv = ref.rows(g, T, 96, x4)
    got = _call([m], x)
    want, bar, _ = ref.expected([m], xv, T, 1, None, None, F32)
    ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMATS, ids=IDS)
def test_swiglu_of_large_gates(cuda, kernels, w4, x4):
    """Gates far from zero on both sides: no overflow of the exponential."""
    g = torch.Generator().manual_seed(5)
    m = [ref.Mats(g, 64, 128, 0, w4) for _ in range(2)]
    x, xv = ref.rows(g, 20, 128, x4)
    if x4:
        x[1].add_(6)
        xv = xv * 64.0
    else:
        x[0].mul_(64.0)
        xv = xv * 64.0
    got = _call(m, x, out_dtype=F32)
    want, bar, _ = ref.expected(m, xv, 20, 1, None, None, F32)
    assert want.abs().max() > 1e3 and torch.isfinite(got).all()
    ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMATS, ids=IDS)
@pytest.mark.parametrize("T", [1, 8, 200, 1500])
def test_same_bits_again_and_in_a_graph(cuda, kernels, T, w4, x4):
    """Replayed with other inputs in the same buffers, eager work between."""
    g = torch.Generator().manual_seed(T)
    up = [ref.Mats(g, 96, 160, 6, w4) for _ in range(2)]
    down = ref.Mats(g, 160, 96, 6, w4)
    wu, wd = [ops.Experts(*m.parts) for m in up], ops.Experts(*down.parts)
    batches = []
    for _ in range(3):
        offsets, sorted_ = ref.groups(g, T, 2, 6)
        batches.append(([t for t in ref.rows(g, T, 160, x4)[0]], offsets.cuda(), sorted_.cuda()))

    def step(x, offsets, sorted_):
        h = ops.grouped_gate_up_swiglu(*wu, *x, offsets=offsets, sorted_=sorted_, k=2)
        h = ops.mxfp4_quantize(h) if x4 else (h,)
        return ops.grouped_matmul(wd, *h, offsets=offsets, sorted_=sorted_)

    eager = [step(*b) for b in batches]
    for b, y in zip(batches, eager):
        assert torch.equal(step(*b), y)
    held = [t.clone() for t in batches[0][0]], batches[0][1].clone(), batches[0][2].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(*held)
    for b, want in list(zip(batches, eager)) * 2:
        for to, new in zip([*held[0], held[1], held[2]], [*b[0], b[1], b[2]]):
            to.copy_(new)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        step(*batches[0])


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMATS, ids=IDS)
def test_no_rows(cuda, w4, x4):
    g = torch.Generator().manual_seed(1)
    m = [ref.Mats(g, 32, 64, 2, w4)]
    x, _ = ref.rows(g, 0, 64, x4)
    offsets = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert _call(m, x, offsets=offsets).shape == (0, 32)


@pytest.mark.gpu
def test_other_stream(cuda):
    g = torch.Generator().manual_seed(1)
    m = [ref.Mats(g, 96, 128, 3, True)]
    offsets, sorted_ = ref.groups(g, 50, 2, 3)
    x, xv = ref.rows(g, 50, 128)
    offsets_, sorted__ = offsets.cuda(), sorted_.cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _call(m, x, offsets=offsets_, sorted_=sorted__, k=2)
    side.synchronize()
    want, bar, _ = ref.expected(m, xv, 100, 2, offsets, sorted_, F32)
    ref.near(got, want, bar)


@pytest.mark.gpu
def test_refusals_of_the_wrappers(cuda):
    w = ops.Experts(torch.zeros(3, 16, 64, dtype=BF16, device="cuda"))
    q = ops.Experts(torch.zeros(3, 16, 32, dtype=U8, device="cuda"),
                    torch.full((3, 16, 2), 127, dtype=U8, device="cuda"))
    x = torch.zeros(4, 64, dtype=BF16, device="cuda")
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad, match in [
            (dict(x=x.float()), "x must be"), (dict(x=x[:, :32].contiguous()), r"\[rows, 64\]"),
            (dict(x=x.t()), "contiguous"), (dict(x=x.cpu()), "device"), (dict(x=x[0]), "2-D"),
            (dict(offsets=offsets[:3]), "offsets"), (dict(offsets=offsets.long()), "offsets"),
            (dict(sorted_=offsets[:3]), "sorted_"), (dict(k=0), "k must"), (dict(k=2), "k must"),
            (dict(x_scales=torch.zeros(4, 2, dtype=U8, device="cuda")), "x_scales"),
            (dict(out_dtype=torch.float16), "out_dtype"),
            (dict(out=torch.zeros(4, 15, device="cuda")), "out"),
            (dict(out=torch.zeros(4, 16, dtype=torch.float16, device="cuda")), "out")]:
        kw = dict(dict(x=x, offsets=offsets), **bad)
        with pytest.raises(ValueError, match=match):
            ops.grouped_matmul(w, kw.pop("x"), kw.pop("x_scales", None), **kw)
    codes, scales = ops.mxfp4_quantize(x)
    with pytest.raises(ValueError, match="x must be"):
        ops.grouped_matmul(w, codes, scales, offsets=offsets)
    with pytest.raises(ValueError, match="x_scales"):
        ops.grouped_matmul(q, codes, offsets=offsets)
    with pytest.raises(ValueError, match="x_scales"):
        ops.grouped_matmul(q, codes, scales[:3], offsets=offsets)
    with pytest.raises(InfernoError, match="several experts"):
        ops.grouped_matmul(w, x)
    with pytest.raises(InfernoError, match="same sizes and format"):
        ops.grouped_gate_up_swiglu(w, q, x, offsets=offsets)
    one = ops.Experts(torch.zeros(16, 64, dtype=BF16, device="cuda"))
    with pytest.raises(InfernoError, match="offsets"):
        ops.grouped_matmul(one, x, sorted_=offsets[:4])
    with pytest.raises(InfernoError, match="16 bytes"):
        ops.grouped_matmul(one, torch.zeros(4 * 64 + 1, dtype=BF16, device="cuda")[1:].view(4, 64))
    with pytest.raises(InfernoError, match="16 bytes"):
        ops.Experts(torch.zeros(16 * 64 + 1, dtype=BF16, device="cuda")[1:].view(16, 64))
    for bad in [(torch.zeros(16, 60, dtype=BF16), None), (torch.zeros(16, 64), None),
                (torch.zeros(16, dtype=BF16), None), (torch.zeros(16, 128, dtype=BF16)[:, ::2], None),
                (torch.zeros(16, 24, dtype=U8), torch.zeros(16, 1, dtype=U8)),
                (torch.zeros(16, 32, dtype=U8), torch.zeros(16, 1, dtype=U8)),
                (torch.zeros(16, 32, dtype=U8), torch.zeros(16, 2))]:
        with pytest.raises(ValueError):
            ops.Experts(*(t if t is None else t.cuda() if t.is_contiguous() else t.cuda()[:, ::2]
                          for t in bad))
    with pytest.raises(ValueError, match="GPU"):
        ops.Experts(torch.zeros(16, 64, dtype=BF16))


def test_refusals_of_the_library():
    L, at = lib(), 1 << 20

    def desc(E=2, N=16, K=64, fmt=1, data=at, nbytes=None):
        d = ExpertsDesc(E, N, K, fmt, data, 0)
        d.data_bytes = nbytes if nbytes is not None else L.inferno_experts_packed_bytes(d)
        return d

    def call(w, x=at, dt=1, xs=None, rows=4, offsets=at, sorted_=None, k=1, od=0, out=at, up=None, ws=None, n=0):
        if up is not None:
            return L.inferno_grouped_gate_up_swiglu(None, w, up, x, dt, xs, rows, offsets, sorted_, k,
                                                    od, out, ws, n)
        return L.inferno_grouped_matmul(None, w, x, dt, xs, rows, offsets, sorted_, k, od, out, ws, n)

    ok = desc()
    for w in (None, desc(fmt=0), desc(fmt=2), desc(E=0), desc(E=257), desc(N=0), desc(K=0), desc(K=60),
              desc(K=48, fmt=3), desc(N=(1 << 24) + 1), desc(N=1 << 20, K=1 << 20), desc(data=None),
              desc(data=at + 8)):
        assert call(w) == -1 and L.inferno_last_error(), w
    assert call(desc(nbytes=100)) == -2 and call(desc(fmt=3, nbytes=100)) == -2
    for bad in (dict(x=None), dict(x=at + 2), dict(dt=0), dict(dt=3, xs=at), dict(xs=at),
                dict(offsets=None), dict(offsets=None, sorted_=at), dict(offsets=at + 2),
                dict(sorted_=at + 1), dict(k=0), dict(k=2), dict(od=2), dict(out=None),
                dict(out=at + 4), dict(rows=(1 << 22) + 1), dict(rows=1 << 40),
                dict(rows=1 << 20, k=8, sorted_=at)):
        assert call(ok, **bad) == -1 and L.inferno_last_error(), bad
    assert call(desc(fmt=3), dt=3) == -1  # codes without scales
    for up in (None, desc(N=32), desc(K=128), desc(E=3), desc(fmt=3)):
        assert L.inferno_grouped_gate_up_swiglu(None, ok, up, at, 1, None, 4, at, None, 1, 0, at, None,
                                                0) == -1
    assert call(ok, rows=0, x=None, out=None) == 0 and call(ok, up=desc(), rows=0) == 0
    pack, size = L.inferno_experts_pack, L.inferno_experts_packed_bytes
    w = desc(fmt=3)
    assert size(desc(fmt=3, K=48, nbytes=0)) == 0 and L.inferno_last_error()
    # two experts of one tile: one step of codes and the scales of four, two steps of bf16
    assert size(w) == 2 * (1024 + 256) and size(ok) == 2 * 2 * 1024
    assert size(desc(N=17, K=40)) == 2 * 2 * 2 * 1024
    assert pack(None, ok, at, 4096, at, 0, at) == -1  # scales of bf16
    assert pack(None, ok, at, 4095, None, 0, at) == -2 and pack(None, ok, at, 4096, None, 8, at) == -2
    assert pack(None, w, at, 1023, at, 64, at) == -2 and pack(None, w, at, 1024, at, 63, at) == -2
    assert pack(None, desc(fmt=3, nbytes=7), at, 1024, at, 64, at) == -2
    for a, b, c in ((None, at, at), (at, None, at), (at, at, None), (at + 4, at, at), (at, at, at + 8)):
        assert pack(None, w, a, 1024, b, 64, c) == -1
