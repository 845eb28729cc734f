"""A decoder layer's feed-forward half from the operators that belong together
(residual norm with 8-bit activations, grouped routing, 4-bit products), eager,
captured, on other streams and from two threads, and the products over the sizes
at which their kernels change."""
import threading

import numpy as np
import pytest
import torch

import w4_reference as ref
from inferno_amd import GROUP_TOP2, SCORE_SIGMOID, lib, ops
from test_group_topk import _definition as routing

F32, BF16, I8 = torch.float32, torch.bfloat16, torch.int8
EPS = 1e-6


class Layer:
    """Norm, router, routed experts on bf16 or int8 tokens, a shared expert on
    int8 tokens and both residuals."""

    def __init__(self, seed, E=16, k=4, H=512, I=256, shared=384, group=64, zeros=False,
                 experts_on=BF16):
        g = torch.Generator().manual_seed(seed)
        self.E, self.k, self.H, self.on = E, k, H, experts_on
        self.norm = (1.0 + 0.2 * torch.randn(H, generator=g)).cuda()
        self.router = (0.1 * torch.randn(E, H, generator=g)).cuda()
        self.bias = (0.1 * torch.randn(E, generator=g)).cuda()
        kw = dict(zeros=zeros)
        self.mats = [ref.make(g, I, H, group, E, **kw), ref.make(g, I, H, group, E, **kw),
                     ref.make(g, H, I, group, E, **kw)]
        self.side = [ref.make(g, shared, H, group, **kw), ref.make(g, shared, H, group, **kw),
                     ref.make(g, H, shared, group, **kw)]
        self.w = [ops.W4(*m) for m in self.mats]
        self.s = [ops.W4(*m) for m in self.side]

    def __call__(self, x, residual):
        total, y, q, sc = ops.add_rms_norm_q8(x, residual, self.norm, EPS, act_dtype=BF16)
        logits = ops.router_logits(y, self.router)
        ids, w, _ = ops.router_group_topk(logits, self.bias, self.k, SCORE_SIGMOID, True, 2.5, 4, 2,
                                          GROUP_TOP2)
        routed = ops.w4_moe(*self.w, q if self.on == I8 else y, ids, w, self.k,
                            x_scales=sc if self.on == I8 else None)
        h = ops.w4_gate_up_swiglu(*self.s[:2], q, x_scales=sc)
        out = ops.w4_matvec_add2(self.s[2], h, total, routed)
        return out, (total, y, q, sc, logits, ids, w, h)

    def check(self, x, residual, out, parts):
        """Each stage against 64 bits from what the stage before it gave."""
        total, y, q, sc, logits, ids, w, h = (p.cpu() for p in parts)
        T = x.shape[0]
        s = (x.float() + residual).cpu()
        assert torch.equal(total, s)
        d = s.double()
        p = d * self.norm.cpu().double()
        root = torch.sqrt(d.square().mean(1, keepdim=True) + EPS)
        # half a step of bf16, and fewer than 32 fp32 roundings
        assert ((y.double() - p / root).abs() <= (2.0 ** -8 + 2.0 ** -19) * (p / root).abs()).all()
        top = p.abs().amax(1, keepdim=True)
        assert torch.equal(q, torch.round(127.0 * p / top).to(I8))
        want_ids, want_w = routing(logits.numpy(), self.bias.cpu().numpy(), self.k, SCORE_SIGMOID,
                                   True, 2.5, 4, 2, GROUP_TOP2)
        assert np.array_equal(ids.view(T, -1).numpy(), want_ids)
        np.testing.assert_allclose(w.view(T, -1).numpy(), want_w, rtol=24 * 2.0 ** -24)
        acts = ref.values(q, sc)
        side = [ref.dense(*m) for m in self.side]
        want, bar = ref.swiglu(side[0], side[1], acts, False)
        assert ((h.double() - want).abs() <= bar).all()
        mats = [[ref.dense(*(None if v is None else v[e] for v in m)) for e in range(self.E)]
                for m in self.mats]
        routed, routed_bar = ref.moe(*mats, acts if self.on == I8 else y.double(), ids, w, self.k,
                                     self.on != I8)
        want, bar = ref.linear(side[2], h.double(), extra=d.abs() + routed.abs() + routed_bar)
        assert ((out.cpu().double() - want - d - routed).abs() <= bar + routed_bar).all()


def _tokens(T, H, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, H, generator=g).to(BF16).cuda(), torch.randn(T, H, generator=g).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 4, 5, 16, 17, 67, 300])
@pytest.mark.parametrize("on,zeros,group", [(BF16, False, 64), (I8, True, 128), (I8, False, 32),
                                            (BF16, True, 128)])
def test_a_layer(cuda, T, on, zeros, group):
    layer = Layer(T, group=group, zeros=zeros, experts_on=on)
    x, r = _tokens(T, layer.H, T + 1)
    layer.check(x, r, *layer(x, r))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 40, 300, 700])
def test_captured_layers(cuda, T):
    # two graphs of one layer and a third of another, replayed in turn with new
    # tokens, eager calls and synchronizations between them
    one, other = Layer(1), Layer(2, group=32, zeros=True, experts_on=I8)
    x, r = _tokens(T, one.H, 5)
    for layer in (one, other):
        layer(x, r)
    torch.cuda.synchronize()
    held = []
    for layer in (one, one, other):
        sx, sr = x.clone(), r.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(sx, sr)[0]
        held.append((graph, layer, sx, sr, out))
    for i in range(5):
        for j, (graph, layer, sx, sr, out) in enumerate(held):
            x, r = _tokens(T, layer.H, 10 * i + j)
            sx.copy_(x)
            sr.copy_(r)
            graph.replay()
            want = layer(x, r)[0]
            assert torch.equal(out, want), (i, j)
            if i % 2:
                torch.cuda.synchronize()
    graphs = [h[0] for h in held]
    for g in graphs + graphs:
        g.replay()
    torch.cuda.synchronize()
    for graph, layer, sx, sr, out in held:
        assert torch.equal(out, layer(sx, sr)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 24, 200])
def test_two_streams_and_two_threads(cuda, T):
    layer = Layer(3)
    inputs = [_tokens(T, layer.H, s) for s in range(2)]
    want = [layer(*i)[0] for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [[], []]

    def work(n):
        with torch.cuda.stream(streams[n]):
            for _ in range(20):
                got[n].append(layer(*inputs[n])[0])

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for n in range(2):
        assert len(got[n]) == 20
        for o in got[n]:
            assert torch.equal(o, want[n])


# Products at the sizes where the kernels change: row tiles taken together (from
# 384, 2048, 8192 and 16384 tiles of 16 rows), shares of the chunks (below 128 and
# 256 workgroups), chunks that no share or wavefront has, and rows of few tokens
# that do not fit a workgroup's memory.
@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,group", [
    (1, 6160, 512, 128), (1, 40, 40960, 128), (2, 40, 49152, 32), (4, 17, 40992, 32),
    (4, 33, 131072, 1024), (5, 6160, 640, 64), (9, 32773, 128, 128), (6, 262149, 64, 64),
    (12, 131077, 160, 32), (16, 50, 16384, 128), (20, 4100, 128, 128), (300, 8200, 160, 32),
    (300, 16385, 256, 256), (200, 300, 1184, 32), (90, 2050, 896, 128), (65, 129, 33024, 256)])
@pytest.mark.parametrize("dtype,zeros", [(BF16, False), (I8, True), (F32, True), (I8, False)])
def test_where_kernels_change(cuda, T, N, K, group, dtype, zeros):
    g = torch.Generator().manual_seed(N)
    m = ref.make(g, N, K, group, zeros=zeros, scales=BF16 if dtype != F32 else F32)
    w = ops.W4(*m)
    x = torch.randn(T, K, generator=g)
    xs = None
    if dtype == I8:
        xs = torch.rand(T, 1, generator=g) + 0.5
        x = torch.randint(-128, 128, (T, K), generator=g)
    x = x.to(dtype).cuda()
    xs = None if xs is None else xs.cuda()
    pick = torch.randint(0, N, (min(N, 600),), generator=g).unique()
    pick[-1] = N - 1
    d = ref.dense(*(None if v is None else v[pick.cuda()] for v in m))
    want, bar = ref.linear(d, ref.values(x, xs), dtype != I8)
    got = ops.w4_matvec_add2(w, x, x_scales=xs)
    assert got.isfinite().all()
    assert ((got[:, pick.cuda()].cpu().double() - want).abs() <= bar).all()
    want, bar = ref.swiglu(d, d, ref.values(x, xs), dtype != I8)
    got = ops.w4_gate_up_swiglu(w, w, x, x_scales=xs)
    assert ((got[:, pick.cuda()].cpu().double() - want).abs() <= bar).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,H,I,group", [
    (1, 12, 4, 8192, 1184, 32), (1, 4, 1, 16384, 64, 64), (1, 20, 16, 1024, 4096, 128),
    (60, 100, 2, 1024, 1056, 32), (100, 16, 1, 4128, 64, 32), (300, 40, 4, 128, 2048, 128),
    (3000, 3, 2, 96, 32, 32), (2100, 1, 1, 64, 160, 32), (5000, 250, 8, 64, 64, 64)])
@pytest.mark.parametrize("dtype", [BF16, I8])
def test_experts_where_kernels_change(cuda, T, E, k, H, I, group, dtype):
    g = torch.Generator().manual_seed(T)
    mats = [ref.make(g, I, H, group, E), ref.make(g, I, H, group, E), ref.make(g, H, I, group, E)]
    x = torch.randn(T, H, generator=g)
    xs = None
    if dtype == I8:
        xs = (torch.rand(T, 1, generator=g) + 0.5).cuda()
        x = torch.randint(-128, 128, (T, H), generator=g)
    x = x.to(dtype).cuda()
    ids = torch.rand(T, E, generator=g).topk(k, 1).indices.int()
    ids[T // 2:, 0] = 0  # one expert has most of the tokens
    ids = ids.flatten().cuda()
    w = torch.rand(T * k, generator=g).cuda()
    got = ops.w4_moe(*(ops.W4(*m) for m in mats), x, ids, w, k, x_scales=xs)
    d = [[ref.dense(m[0][e], m[1][e]) for e in range(E)] for m in mats]
    want, bar = ref.moe(*d, ref.values(x, xs), ids, w, k, dtype != I8)
    assert ((got.cpu().double() - want).abs() <= bar).all()


@pytest.mark.gpu
def test_many_tokens(cuda):
    # more tokens than a grid has rows
    T = 70001
    g = torch.Generator().manual_seed(0)
    m = ref.make(g, 16, 32, 32)
    w = ops.W4(*m)
    x = torch.randn(T, 32, generator=g).to(BF16).cuda()
    want, bar = ref.linear(ref.dense(*m), ref.values(x))
    assert ((ops.w4_matvec_add2(w, x).cpu().double() - want).abs() <= bar).all()
    mats = [ref.make(g, 32, 32, 32, 2) for _ in range(3)]
    ids = torch.randint(0, 2, (T,), generator=g).int().cuda()
    wt = torch.ones(T).cuda()
    got = ops.w4_moe(*(ops.W4(*v) for v in mats), x, ids, wt, 1)
    d = [[ref.dense(v[0][e], v[1][e]) for e in range(2)] for v in mats]
    want, bar = ref.moe(*d, ref.values(x), ids, wt, 1)
    assert ((got.cpu().double() - want).abs() <= bar).all()


@pytest.mark.gpu
@pytest.mark.parametrize("E,k,I,group", [
    # k rows of I digits in one workgroup's memory: 62312 bytes, 66192 twice (past the
    # default limit of 65536), 78608, 80936 of the 81920 that it may take, then more
    (12, 10, 1920, 128), (12, 10, 2016, 32), (12, 10, 2048, 128), (16, 16, 1536, 64),
    (20, 11, 2304, 128), (20, 16, 1664, 32)])
@pytest.mark.parametrize("dtype,zeros", [(BF16, False), (F32, True)])
def test_one_token_of_large_sums(cuda, E, k, I, group, dtype, zeros):
    g = torch.Generator().manual_seed(I + k)
    H = 160 if group == 32 else 256
    mats = [ref.make(g, I, H, group, E, zeros), ref.make(g, I, H, group, E, zeros),
            ref.make(g, H, I, group, E, zeros, scales=F32 if zeros else BF16)]
    x = torch.randn(1, H, generator=g).to(dtype).cuda()
    ids = torch.randperm(E, generator=g)[:k].int().cuda()
    w = torch.rand(k, generator=g).cuda()
    handles = [ops.W4(*m) for m in mats]
    got = ops.w4_moe(*handles, x, ids, w, k)
    d = [[ref.dense(*(None if v is None else v[e] for v in m)) for e in range(E)] for m in mats]
    want, bar = ref.moe(*d, ref.values(x), ids, w, k)
    assert ((got.cpu().double() - want).abs() <= bar).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = ops.w4_moe(*handles, x, ids, w, k)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, ops.w4_moe(*handles, x, ids, w, k))


@pytest.mark.gpu
def test_a_handle_packed_behind_other_work_is_used_on_another_stream(cuda):
    # packing waits behind some milliseconds of products on its stream; the caller's
    # tensors are overwritten and the handle is used elsewhere right afterwards
    g = torch.Generator().manual_seed(4)
    m = ref.make(g, 300, 1024, 64, zeros=True)
    x = torch.randn(6, 1024, generator=g).to(BF16).cuda()
    want, bar = ref.linear(ref.dense(*m), ref.values(x))
    a = torch.randn(4096, 4096, device=cuda)
    b = a @ a
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(10):
            torch.mm(a, a, out=b)
        w = ops.W4(*m)
    with torch.cuda.stream(other):
        for t in m:
            t.zero_()
        got = ops.w4_matvec_add2(w, x)
    torch.cuda.synchronize()
    assert ((got.cpu().double() - want).abs() <= bar).all()


@pytest.mark.gpu
def test_a_handle_packed_in_a_graph(cuda):
    g = torch.Generator().manual_seed(5)
    first, second = (ref.make(g, 40, 256, 128) for _ in range(2))
    x = torch.randn(3, 256, generator=g).cuda()
    held = [t.clone() if t is not None else None for t in first]
    ops.w4_matvec_add2(ops.W4(*first), x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.w4_matvec_add2(ops.W4(*held), x)
    for m in (first, second, first):
        for t, v in zip(held, m):
            if t is not None:
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, ops.w4_matvec_add2(ops.W4(*m), x))


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,mats,one", [
    # bytes of a workgroup: T ceil(K / 128) 388 + 1024 mats + 16, of 54272
    (4, 4096, 2, True), (4, 4352, 2, False), (4, 4352, 1, True), (3, 5632, 2, True),
    (3, 5888, 2, False), (2, 8704, 1, True), (1, 17536, 1, True), (1, 17664, 1, False)])
def test_few_tokens_that_fit_take_one_launch(cuda, T, K, mats, one):
    # the launch that stages its tokens by itself leaves the workspace as it was
    g = torch.Generator().manual_seed(K)
    m = ref.make(g, 24, K, 128)
    w = ops.W4(*m)
    x = torch.randn(T, K, generator=g).cuda()
    n = lib().inferno_w4_workspace_bytes(T, K)
    ws = torch.full((n,), 171, dtype=torch.uint8, device=cuda)
    out = torch.empty(T, 24, device=cuda)
    s = torch.cuda.current_stream().cuda_stream
    tail = (x.data_ptr(), 0, None, 0)
    if mats == 2:
        st = lib().inferno_w4_gate_up_swiglu(s, w.ref, w.ref, *tail, T, out.data_ptr(),
                                             ws.data_ptr(), n)
        want, bar = ref.swiglu(ref.dense(*m), ref.dense(*m), ref.values(x))
    else:
        st = lib().inferno_w4_matvec_add2(s, w.ref, *tail, None, None, T, out.data_ptr(),
                                          ws.data_ptr(), n)
        want, bar = ref.linear(ref.dense(*m), ref.values(x))
    assert st == 0
    assert bool((ws == 171).all()) == one
    assert ((out.cpu().double() - want).abs() <= bar).all()
