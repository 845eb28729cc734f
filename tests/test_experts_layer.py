"""A routed layer with a shared expert, made of the router, the dispatch, the products
grouped by expert and the combine, each step against 64 bits from the step before it."""
import threading

import pytest
import torch

import experts_reference as ref
from inferno_amd import ops

F32, BF16 = torch.float32, torch.bfloat16
FORMS = [(False, False), (True, False), (True, True)]  # weights, rows in MXFP4
IDS = ["bf16", "mxfp4", "mxfp4-mxfp4"]
E, K_TOP, H, I, I_SHARED = 24, 4, 416, 160, 224


class Layer:
    def __init__(self, w4, x4, seed=3):
        g = torch.Generator().manual_seed(seed)
        self.x4 = x4
        self.up = [ref.Mats(g, I, H, E, w4) for _ in range(2)]
        self.down = ref.Mats(g, H, I, E, w4)
        self.shared_up = [ref.Mats(g, I_SHARED, H, 0, w4) for _ in range(2)]
        self.shared_down = ref.Mats(g, H, I_SHARED, 0, w4)
        self.router = (0.05 * torch.randn(E, H, generator=g)).cuda()
        self.w_up = [ops.Experts(*m.parts) for m in self.up]
        self.w_down = ops.Experts(*self.down.parts)
        self.w_shared_up = [ops.Experts(*m.parts) for m in self.shared_up]
        self.w_shared_down = ops.Experts(*self.shared_down.parts)

    def rows(self, x):
        return ops.mxfp4_quantize(x) if self.x4 else (x,)

    def __call__(self, x):
        """Every step's results, by name."""
        T, s = x.shape[0], {}
        s["ids"], s["weights"], _ = ops.router_topk(ops.router_logits(x, self.router), None, K_TOP, 0,
                                                    True, 1.0)
        s["offsets"], s["sorted"], _ = ops.dispatch(s["ids"], T, K_TOP, E)
        s["x"] = self.rows(x)
        at = dict(offsets=s["offsets"], sorted_=s["sorted"])
        s["mid"] = ops.grouped_gate_up_swiglu(*self.w_up, *s["x"], k=K_TOP, **at)
        s["h"] = self.rows(s["mid"])
        s["y"] = ops.grouped_matmul(self.w_down, *s["h"], **at)
        s["shared_mid"] = ops.grouped_gate_up_swiglu(*self.w_shared_up, *s["x"])
        s["shared_h"] = self.rows(s["shared_mid"])
        s["shared"] = ops.grouped_matmul(self.w_shared_down, *s["shared_h"])
        s["out"] = ops.topk_combine_residual(s["shared"], x.float(), s["y"], s["weights"], K_TOP)
        return s

    def held(self, x, given):
        """Values in 64 bits of the rows that a product takes, checked against x."""
        if not self.x4:
            return x.double().cpu()
        codes, scales, values = ref.quantize(x)
        assert torch.equal(given[0].cpu(), codes) and torch.equal(given[1].cpu(), scales)
        return values


def _x(seed, T):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, H, generator=g).to(BF16).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMS, ids=IDS)
@pytest.mark.parametrize("T", [1, 2, 7, 64, 301])
def test_steps(cuda, T, w4, x4):
    layer = Layer(w4, x4)
    x = _x(T, T)
    s = layer(x)
    A, offsets, sorted_ = T * K_TOP, s["offsets"].cpu(), s["sorted"].cpu()
    ids = s["ids"].cpu().long()
    assert torch.equal(offsets.long(), torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(
        ids, minlength=E).cumsum(0)]))
    assert torch.equal(sorted_.long(), ids.argsort(stable=True))
    xv = layer.held(x, s["x"])
    want, bar, hit = ref.expected(layer.up, xv, A, K_TOP, offsets, sorted_, BF16)
    assert hit.all()
    ref.near(s["mid"], want, bar)
    want, bar, _ = ref.expected([layer.down], layer.held(s["mid"], s["h"]), A, 1, offsets, sorted_, F32)
    ref.near(s["y"], want, bar)
    want, bar, _ = ref.expected(layer.shared_up, xv, T, 1, None, None, BF16)
    ref.near(s["shared_mid"], want, bar)
    want, bar, _ = ref.expected([layer.shared_down], layer.held(s["shared_mid"], s["shared_h"]), T, 1,
                                None, None, F32)
    ref.near(s["shared"], want, bar)
    parts = s["y"].double().cpu().view(T, K_TOP, H) * s["weights"].double().cpu().view(T, K_TOP, 1)
    want = s["shared"].double().cpu() + x.double().cpu() + parts.sum(1)
    # k products and k + 1 sums, each off by half a step of a partial sum
    size = s["shared"].double().cpu().abs() + x.double().cpu().abs() + parts.abs().sum(1)
    ref.near(s["out"], want, (2 * K_TOP + 1) * 2.0 ** -24 * 1.01 * size + 1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMS, ids=IDS)
@pytest.mark.parametrize("T", [1, 64, 301])
def test_in_a_graph(cuda, T, w4, x4):
    layer = Layer(w4, x4)
    xs = [_x(seed, T) for seed in range(3)]
    eager = [layer(x)["out"] for x in xs]
    held = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(held)["out"]
    for x, want in list(zip(xs, eager)) * 2:
        held.copy_(x)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(layer(x)["out"], want)


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMS, ids=IDS)
def test_threads_with_streams_of_their_own(cuda, w4, x4):
    """Four threads drive one layer's weights at once."""
    layer = Layer(w4, x4)
    xs = [_x(seed, T) for seed, T in enumerate((1, 17, 130, 301))]
    eager = [layer(x)["out"] for x in xs]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(4)

    def drive(i):
        try:
            start.wait(30)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    out = layer(xs[i])["out"]
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(out, eager[i]):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001 (told to the main thread)
            wrong.append(repr(e))

    threads = [threading.Thread(target=drive, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMS, ids=IDS)
@pytest.mark.parametrize("T", [5, 200])
def test_only_results_are_written(cuda, T, w4, x4):
    """Guards around a result, and inputs that stay as they were."""
    layer = Layer(w4, x4)
    x = _x(T, T)
    s = layer(x)
    inputs = [x, s["offsets"], s["sorted"], *s["x"]]
    before = [t.clone() for t in inputs]
    for dtype in (F32, BF16):
        room = torch.full((T * K_TOP + 64, I), 5.0, dtype=dtype, device="cuda")
        out = room[32: 32 + T * K_TOP]
        ops.grouped_gate_up_swiglu(*layer.w_up, *s["x"], offsets=s["offsets"], sorted_=s["sorted"],
                                   k=K_TOP, out=out)
        assert (room[:32] == 5.0).all() and (room[32 + T * K_TOP:] == 5.0).all()
        assert torch.equal(out, s["mid"]) if dtype == BF16 else torch.isfinite(out).all()
    assert all(torch.equal(a, b) for a, b in zip(inputs, before))


@pytest.mark.gpu
def test_handles_outlive_their_tensors(cuda):
    """Packed weights stand for themselves; a handle made on another stream is ready."""
    g = torch.Generator().manual_seed(0)
    m = ref.Mats(g, 96, 128, 3)
    x, xv = ref.rows(g, 30, 128)
    offsets, sorted_ = ref.groups(g, 30, 1, 3)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        w = ops.Experts(*m.parts)
    m.parts[0].zero_()
    got = ops.grouped_matmul(w, *x, offsets=offsets.cuda(), sorted_=sorted_.cuda())
    want, bar, _ = ref.expected([m], xv, 30, 1, offsets, sorted_, F32)
    ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("w4", [False, True])
def test_packed_inside_a_graph(cuda, w4):
    """A handle that a graph packs holds its matrices after the first replay, and those
    that the tensors hold at a later one."""
    g = torch.Generator().manual_seed(1)
    m, other = (ref.Mats(g, 70, 160, 3, w4) for _ in range(2))
    x, xv = ref.rows(g, 33, 160)
    offsets, sorted_ = ref.groups(g, 33, 1, 3)
    offsets_, sorted__ = offsets.cuda(), sorted_.cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w = ops.Experts(*m.parts)
        y = ops.grouped_matmul(w, *x, offsets=offsets_, sorted_=sorted__)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        got = ops.grouped_matmul(w, *x, offsets=offsets_, sorted_=sorted__)
        want, bar, _ = ref.expected([m], xv, 33, 1, offsets, sorted_, F32)
        ref.near(got, want, bar)
        assert torch.equal(got, y)
        for to, new in zip(m.parts, other.parts):
            to.copy_(new)
        m.values = other.values


@pytest.mark.gpu
@pytest.mark.parametrize("w4,x4", FORMS, ids=IDS)
def test_the_same_assignment_twice(cuda, w4, x4):
    """An index that comes twice: its row is one of its two experts' results, value by
    value, and all others are as ever."""
    g = torch.Generator().manual_seed(6)
    m = [ref.Mats(g, 48, 192, 2, w4)]
    x, xv = ref.rows(g, 40, 192, x4)
    offsets = torch.tensor([0, 20, 40], dtype=torch.int32)
    order = torch.randperm(40, generator=g).to(torch.int32)
    order[30] = order[3]
    w = ops.Experts(*m[0].parts)
    out = torch.full((40, 48), 7.0, device="cuda")
    got = ops.grouped_matmul(w, *x, offsets=offsets.cuda(), sorted_=order.cuda(), out=out).cpu().double()
    fine = got == 7.0
    for e in range(2):
        a = order[20 * e: 20 * e + 20].long()
        y, d = ref.product(m[0], xv, e, a)
        near = (got[a] - y).abs() <= d + 2.0 ** -24 * y.abs()
        fine[a] |= near
    assert fine.all() and (got[torch.tensor([i for i in range(40) if i not in order.tolist()])] == 7.0).all()
