"""Packed weights (Experts, W4) and the streams that use them: a handle may go while a
call on another stream is queued."""
import contextlib
import weakref
from types import SimpleNamespace

import pytest
import torch

import experts_reference as ref
from inferno_amd import ops

F32, BF16, U8 = torch.float32, torch.bfloat16, torch.uint8


class _Bytes:
    """Stands for packed bytes; notes the streams that it is told of."""

    def __init__(self):
        self.told = []

    def record_stream(self, stream):
        self.told.append(stream)


@pytest.mark.parametrize("kind", [ops.Experts, ops.W4])
def test_each_other_stream_is_told_of_once(monkeypatch, kind):
    now = {"stream": 5, "capturing": False}
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: now["stream"])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    h = kind.__new__(kind)
    h.device, data = torch.device("cuda:0"), _Bytes()
    x, calls = SimpleNamespace(is_cuda=True, get_device=lambda: 0), []
    now["capturing"] = True  # (nothing to wait for here)
    h._hold(data)
    for stream, capturing, told in [(5, False, []), (7, True, []), (7, False, [7]), (7, False, [7]),
                                    (5, False, [7]), (9, False, [7, 9]), (7, True, [7, 9])]:
        now.update(stream=stream, capturing=capturing)
        ops._run(x, lambda s, a: calls.append((s, a)) or 0, "a", held=(h, h))
        assert calls.pop() == (stream, "a") and data.told == told


def _experts(g, fp4):
    m = ref.Mats(g, 2080, 2048, 8, fp4)
    x, xv = ref.rows(g, 24, 2048)
    offsets, sorted_ = ref.groups(g, 24, 2, 8)
    o, s = offsets.cuda(), sorted_.cuda()
    want, bar, _ = ref.expected([m], xv, 48, 2, offsets, sorted_, F32)
    return ops.Experts, m.parts, lambda w: ops.grouped_matmul(w, *x, offsets=o, sorted_=s, k=2), \
        want, bar


def _w4(g):
    codes = torch.randint(0, 256, (8192, 1024), generator=g, dtype=U8)
    scales = 0.01 * (1.0 + torch.rand(8192, 16, generator=g))
    x = torch.randn(1, 2048, generator=g).to(BF16)
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double() - 8.0
    w = q * scales.double().repeat_interleave(128, -1)
    # x is exact in bf16: sums of 128 exact products, times a scale, in fp32
    bar = 2048 * 2.0 ** -23 * (x.double().abs() @ w.abs().T) + 1e-30
    xs = x.cuda()
    return ops.W4, (codes.cuda(), scales.cuda()), lambda h: ops.w4_matvec_add2(h, xs), \
        x.double() @ w.T, bar


def _product(kind, seed):
    """A handle's type and tensors, a product with a handle, its result and bar."""
    g = torch.Generator().manual_seed(seed)
    return _w4(g) if kind == "w4" else _experts(g, kind == "mxfp4")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "mxfp4", "w4"])
def test_a_handle_goes_while_its_call_is_queued(cuda, kind):
    """Its bytes are given to nobody before the other stream has read them."""
    make, tensors, call, want, bar = _product(kind, 11)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        long = torch.zeros(8192, 8192, dtype=BF16, device="cuda")
        warm = make(*tensors)
        call(warm)
        long @ long
    del warm
    torch.cuda.synchronize()
    w = make(*tensors)
    data = w.packed if kind == "w4" else w.data
    size, at = data.numel(), data.data_ptr()
    del data
    with torch.cuda.stream(side):
        for _ in range(60):
            long @ long
        got = call(w)
        busy = torch.cuda.Event()
        busy.record()
    del w
    other = torch.full((size,), 255, dtype=U8, device="cuda")
    assert not busy.query()  # the call was queued all that while
    assert other.data_ptr() != at
    side.synchronize()
    ref.near(got, want, bar)


@pytest.mark.gpu
def test_captured_on_another_stream(cuda):
    """A graph's call tells the allocator nothing; the handle outlives the graph."""
    make, tensors, call, want, bar = _product("mxfp4", 12)
    w = make(*tensors)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(w)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        ref.near(y, want, bar)
        ref.near(call(w), want, bar)



@pytest.mark.parametrize("capturing", [True, False])
@pytest.mark.parametrize("kind", [ops.Experts, ops.W4])
def test_tensors_are_kept_while_a_stream_is_captured(monkeypatch, kind, capturing):
    waits = []
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 5)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: SimpleNamespace(
        synchronize=lambda: waits.append(dev)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    h, source = kind.__new__(kind), torch.zeros(3)
    h.device = torch.device("cuda:0")
    h._hold(_Bytes(), source, None)
    gone = weakref.ref(source)
    del source
    assert (gone() is not None) == capturing and len(waits) == (0 if capturing else 1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "mxfp4", "w4"])
def test_a_handle_made_in_a_graph_keeps_its_tensors(cuda, kind):
    """Each replay packs again, from tensors that nothing else holds."""
    make, tensors, call, want, bar = _product(kind, 13)
    gone = [weakref.ref(t) for t in tensors]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w = make(*tensors)
        y = call(w)
    del tensors
    assert all(t() is not None for t in gone)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        ref.near(y, want, bar)
        ref.near(call(w), want, bar)
    del w
    assert all(t() is None for t in gone)
