"""Products of rows grouped by expert at sizes that reach each form of tiles and the
shares of long columns, against 64 bits (bars: experts_reference.py)."""
import pytest
import torch

import experts_reference as ref
from inferno_amd import BF16 as ABI_BF16
from inferno_amd import MXFP4, ExpertsDesc, lib, ops

F32, BF16 = torch.float32, torch.bfloat16
FORMS = {"bf16": (False, False), "mxfp4": (True, False), "mxfp4-mxfp4": (True, True)}

GROUPED = [  # form, T, k, E, N of all matrices, K
    ("bf16", 2240, 2, 64, 1500, 72), ("bf16", 900, 2, 40, 1030, 64), ("bf16", 400, 2, 48, 1540, 40),
    ("bf16", 250, 2, 64, 1540, 96), ("mxfp4", 640, 2, 64, 2000, 96), ("mxfp4", 1120, 2, 64, 1000, 160),
    ("mxfp4", 200, 2, 64, 900, 32), ("mxfp4-mxfp4", 2240, 2, 64, 2000, 96),
    ("mxfp4-mxfp4", 2240, 2, 64, 1000, 4096), ("mxfp4-mxfp4", 640, 2, 64, 400, 544),
    ("mxfp4-mxfp4", 200, 2, 64, 900, 1056)]
DENSE = [("bf16", 8190, 2000, 40), ("bf16", 2950, 2000, 2056), ("bf16", 1990, 1500, 2056),
         ("bf16", 1590, 1000, 64), ("mxfp4", 4090, 2000, 96), ("mxfp4", 1990, 1900, 64),
         ("mxfp4-mxfp4", 8190, 2000, 64), ("mxfp4-mxfp4", 790, 1900, 32)]


def _call(m, x, **kw):
    w = [ops.Experts(*t.parts) for t in m]
    return (ops.grouped_matmul if len(w) == 1 else ops.grouped_gate_up_swiglu)(*w, *x, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("form,T,k,E,N,K", GROUPED)
def test_grouped_tiles(cuda, form, T, k, E, N, K, mats):
    w4, x4 = FORMS[form]
    g = torch.Generator().manual_seed(T + N + K)
    m = [ref.Mats(g, N // mats, K, E, w4) for _ in range(mats)]
    offsets, sorted_ = ref.groups(g, T, k, E)
    x, xv = ref.rows(g, T, K, x4)
    got = _call(m, x, offsets=offsets.cuda(), sorted_=sorted_.cuda(), k=k, out_dtype=F32)
    want, bar, hit = ref.expected(m, xv, T * k, k, offsets, sorted_, F32)
    assert hit.all()
    ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("T,k,E,N,K", [(40, 2, 16, 600, 1600), (140, 2, 4, 1000, 1600), (40, 2, 16, 600, 160),
                                       (200, 2, 4, 1300, 96)])
def test_rows_and_their_shares(cuda, monkeypatch, form, T, k, E, N, K, mats):
    """The kernel of few rows with one, two and four wavefronts on the same weights."""
    monkeypatch.setenv("INFERNO_EXPERTS_TILES", "0")
    test_grouped_tiles(cuda, form, T, k, E, N, K, mats)


@pytest.mark.gpu
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("form,T,N,K", DENSE)
def test_tiles_of_one_matrix(cuda, form, T, N, K, mats):
    w4, x4 = FORMS[form]
    g = torch.Generator().manual_seed(T + N + K)
    m = [ref.Mats(g, N // mats, K, 0, w4) for _ in range(mats)]
    x, xv = ref.rows(g, T, K, x4)
    got = _call(m, x, out_dtype=BF16)
    want, bar, _ = ref.expected(m, xv, T, 1, None, None, BF16)
    ref.near(got, want, bar)


def _workspace(w4, N, K, E, mats, rows, k, grouped):
    d = ExpertsDesc(E, N, K, MXFP4 if w4 else ABI_BF16, None, 0)
    return lib().inferno_grouped_workspace_bytes(d, mats, ABI_BF16, rows, k, grouped)


SHARED = [(2, 40, 4128), (4, 33, 6432), (8, 70, 12832)]  # shares of the columns, N, K


@pytest.mark.parametrize("w4", [False, True])
@pytest.mark.parametrize("shares,N,K", SHARED)
def test_workspace_of_shared_columns(monkeypatch, shares, N, K, w4):
    monkeypatch.setenv("INFERNO_EXPERTS_TILES", "1")
    for mats in (1, 2):
        for rows, k, grouped in ((5, 1, 0), (90, 1, 0), (20, 3, 1)):
            want = shares * mats * rows * k * ((N + 3) // 4 * 4) * 4
            assert _workspace(w4, N, K, 3 if grouped else 1, mats, rows, k, grouped) == want
    L, at = lib(), 1 << 20
    d = ExpertsDesc(1, N, K, MXFP4 if w4 else ABI_BF16, at, 0)
    d.data_bytes = L.inferno_experts_packed_bytes(d)
    need = _workspace(w4, N, K, 1, 1, 5, 1, 0)
    for ws, n in ((None, 0), (at, need - 1)):
        assert L.inferno_grouped_matmul(None, d, at, 1, None, 5, None, None, 1, 0, at, ws, n) == -2
        assert L.inferno_last_error()
    assert L.inferno_grouped_matmul(None, d, at, 1, None, 5, None, None, 1, 0, at, at + 8, need) == -1


def test_most_products_need_no_workspace():
    for w4 in (False, True):
        for rows in (1, 8, 300, 5000):
            assert _workspace(w4, 1024, 2048, 64, 2, rows, 1, 1) == 0
            assert _workspace(w4, 2048, 1024, 1, 1, rows, 1, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("w4", [False, True])
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("shares,N,K", SHARED)
def test_shared_columns(cuda, monkeypatch, shares, N, K, mats, w4):
    """One matrix; groups of all sizes, tokens of several experts; and groups that leave
    rows and indices out, whose results stay as they were."""
    monkeypatch.setenv("INFERNO_EXPERTS_TILES", "1")
    g = torch.Generator().manual_seed(N + K)
    m = [ref.Mats(g, N, K, 0, w4) for _ in range(mats)]
    for T, dtype in ((1, F32), (90, BF16)):
        x, xv = ref.rows(g, T, K)
        want, bar, _ = ref.expected(m, xv, T, 1, None, None, dtype)
        ref.near(_call(m, x, out_dtype=dtype), want, bar)
    m = [ref.Mats(g, N, K, 3, w4) for _ in range(mats)]
    offsets, sorted_ = ref.groups(g, 20, 2, 3)
    x, xv = ref.rows(g, 20, K)
    got = _call(m, x, offsets=offsets.cuda(), sorted_=sorted_.cuda(), k=2, out_dtype=F32)
    want, bar, _ = ref.expected(m, xv, 40, 2, offsets, sorted_, F32)
    ref.near(got, want, bar)
    offsets = torch.tensor([3, 3, 9, 15], dtype=torch.int32)
    order = torch.randperm(20, generator=g).to(torch.int32)
    order[5] = 20
    for s in (None, order):
        out = torch.full((20, N), 7.0, device="cuda")
        _call(m, x, offsets=offsets.cuda(), sorted_=None if s is None else s.cuda(), out=out)
        if s is not None:
            s = s.clone()
            spared = torch.tensor([c for c in range(20) if c not in order.tolist()])
            s[5] = spared[0]  # in the oracle: a row that is then left out
        want, bar, hit = ref.expected(m, xv, 20, 1, offsets, s, F32)
        if s is not None:
            hit[spared[0]] = False
        want[~hit], bar[~hit] = 7.0, 1e-30
        ref.near(out, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("w4", [False, True])
def test_the_rule_shares_long_columns(cuda, w4):
    assert _workspace(w4, 640, 12832, 3, 1, 60, 1, 1) > 0
    g = torch.Generator().manual_seed(2)
    m = [ref.Mats(g, 640, 12832, 3, w4)]
    offsets, sorted_ = ref.groups(g, 60, 1, 3)
    x, xv = ref.rows(g, 60, 12832)
    got = _call(m, x, offsets=offsets.cuda(), sorted_=sorted_.cuda())
    want, bar, _ = ref.expected(m, xv, 60, 1, offsets, sorted_, F32)
    ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("tiles", [None, "1"])
@pytest.mark.parametrize("form,K", [("bf16", 488), ("bf16", 520), ("mxfp4", 480), ("mxfp4-mxfp4", 1984),
                                    ("mxfp4-mxfp4", 2080)])
def test_rows_far_behind_the_first(cuda, monkeypatch, form, K, tiles):
    """Rows of 4.1e9 bytes in all, and of more than 2^32, which tiles do not take."""
    if tiles:
        monkeypatch.setenv("INFERNO_EXPERTS_TILES", tiles)
    w4, x4 = FORMS[form]
    g = torch.Generator().manual_seed(K)
    m = ref.Mats(g, 24, K, 0, w4)
    A = (1 << 22) - 5
    on_gpu = torch.Generator(device="cuda").manual_seed(K)
    if x4:
        x = (torch.randint(0, 256, (A, K // 2), generator=on_gpu, device="cuda", dtype=torch.uint8),
             torch.randint(120, 124, (A, K // 32), generator=on_gpu, device="cuda", dtype=torch.uint8))
    else:
        x = (torch.empty(A, K, dtype=BF16, device="cuda").normal_(generator=on_gpu),)
    got = _call([m], x)
    at = torch.cat([torch.arange(40), torch.arange(A // 2, A // 2 + 40), torch.arange(A - 200, A)])
    part = [t[at.cuda()].cpu() for t in x]
    xv = ref.values(*part) if x4 else part[0].double()
    want, bar = ref.product(m, xv, 0, torch.arange(len(at)))
    ref.near(got[at.cuda()], want, bar + 2.0 ** -24 * want.abs() + 1e-38)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 300])
def test_weights_far_behind_the_first(cuda, rows):
    """The last of experts of 5e9 bytes."""
    E, N, K = 200, 2040, 6144
    w = torch.empty(E, N, K, dtype=BF16, device="cuda")
    w.normal_(0.0, 0.05, generator=torch.Generator(device="cuda").manual_seed(rows))
    handle = ops.Experts(w)
    last = w[E - 1].cpu().double()
    del w
    x, xv = ref.rows(torch.Generator().manual_seed(rows), rows, K)
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[E] = rows
    got = ops.grouped_matmul(handle, *x, offsets=offsets.cuda())
    want, bar = xv @ last.T, K * 2.0 ** -23 * (xv.abs() @ last.abs().T)
    ref.near(got, want, bar + 2.0 ** -24 * want.abs())


@pytest.mark.gpu
def test_quantised_rows_far_behind_the_first(cuda):
    x = torch.empty((1 << 21) + 3, 2048, dtype=BF16, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(4))
    codes, scales, held = ops.mxfp4_quantize(x, values=True)
    for at in (slice(0, 3), slice((1 << 20) - 2, (1 << 20) + 2), slice((1 << 21) - 1, None)):
        c, s, v = ref.quantize(x[at])
        assert torch.equal(codes[at].cpu(), c) and torch.equal(scales[at].cpu(), s)
        assert torch.equal(held[at].cpu().double(), v)


@pytest.mark.gpu
@pytest.mark.parametrize("form,T,E,N,K,tiles", [("mxfp4-mxfp4", 2240, 64, 2000, 96, None),
                                                ("mxfp4-mxfp4", 2240, 64, 1000, 4096, None),
                                                ("bf16", 2240, 64, 1500, 72, None),
                                                ("bf16", 11, 3, 40, 6432, "1"),
                                                ("mxfp4", 11, 3, 40, 6432, "1")])
def test_in_a_graph(cuda, monkeypatch, form, T, E, N, K, tiles):
    """The forms that ask for much shared memory or a workspace, captured before any
    eager call and replayed with other rows, eager work between."""
    if tiles:
        monkeypatch.setenv("INFERNO_EXPERTS_TILES", tiles)
    w4, x4 = FORMS[form]
    g = torch.Generator().manual_seed(K)
    w = ops.Experts(*ref.Mats(g, N, K, E, w4).parts)
    batches = []
    for _ in range(3):
        offsets, sorted_ = ref.groups(g, T, 2, E)
        batches.append([*ref.rows(g, T, K, x4)[0], offsets.cuda(), sorted_.cuda()])

    def step(b):
        return ops.grouped_matmul(w, *b[:-2], offsets=b[-2], sorted_=b[-1], k=2)

    held = [t.clone() for t in batches[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(held)
    for b in batches * 2:
        for to, new in zip(held, b):
            to.copy_(new)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, step(b))
