"""Products with 4-bit group-scaled weights against 64 bits (bars:
w4_reference.py), their refusals, and the calls that share a GPU."""
import pytest
import torch

import w4_reference as ref
from inferno_amd import InfernoError, W4Desc, lib, ops

F32, BF16, I8 = torch.float32, torch.bfloat16, torch.int8


def _x(g, T, K, dtype, x_group=0, device="cuda", std=1.0):
    x = std * torch.randn(T, K, generator=g)
    x[:, ::61] *= 12.0  # loud channels
    if dtype != I8:
        return x.to(dtype).to(device), None
    n = x_group or K
    v = x.view(T, K // n, n)
    s = v.abs().amax(2, keepdim=True) / 127.0
    q = torch.round(v / s).clamp(-128, 127).to(I8).view(T, K).contiguous()
    q[:, 5::50] = -128
    return q.to(device), s.view(T, K // n).contiguous().to(device)


def _near(got, want, bar):
    got = got.cpu().double()
    worst = ((got - want).abs() / (bar + 1e-300)).max().item()
    assert worst <= 1.0, worst


SHAPES = [  # T, rows, cols, group
    (1, 16, 128, 128), (1, 1, 32, 32), (1, 17, 96, 32), (2, 33, 160, 32), (3, 250, 192, 64),
    (4, 64, 2048, 128), (5, 16, 1056, 32), (7, 130, 640, 128), (16, 48, 512, 256), (17, 31, 384, 64),
    (33, 20, 1024, 1024), (64, 96, 256, 64), (70, 257, 288, 32), (128, 128, 512, 128),
    (130, 70, 1152, 384), (300, 129, 448, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,group", SHAPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, I8])
def test_matvec_add2(cuda, T, N, K, group, zeros, dtype):
    g = torch.Generator().manual_seed(T * 1000 + N + K)
    for scales in (F32, BF16):
        m = ref.make(g, N, K, group, zeros=zeros, scales=scales)
        w = ops.W4(*m)
        assert (w.rows, w.cols, w.group) == (N, K, group)
        x, xs = _x(g, T, K, dtype, 128 if K % 128 == 0 and scales == F32 else 0)
        a, b = (torch.randn(T, N, generator=g).cuda() for _ in range(2))
        want, bar = ref.linear(ref.dense(*m), ref.values(x, xs), dtype != I8)
        _near(ops.w4_matvec_add2(w, x, x_scales=xs), want, bar)
        want, bar = ref.linear(ref.dense(*m), ref.values(x, xs), dtype != I8,
                               extra=(a.abs() + b.abs()).cpu().double())
        _near(ops.w4_matvec_add2(w, x, a, b, x_scales=xs), want + (a.cpu().double() + b.cpu()), bar)
        want = want + b.cpu()
        _near(ops.w4_matvec_add2(w, x, residual_b=b, x_scales=xs), want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,group", SHAPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, I8])
def test_gate_up_swiglu(cuda, T, N, K, group, zeros, dtype):
    g = torch.Generator().manual_seed(T * 1000 + N + K + 1)
    mg, mu = (ref.make(g, N, K, group, zeros=zeros) for _ in range(2))
    x, xs = _x(g, T, K, dtype)
    want, bar = ref.swiglu(ref.dense(*mg), ref.dense(*mu), ref.values(x, xs), dtype != I8)
    _near(ops.w4_gate_up_swiglu(ops.W4(*mg), ops.W4(*mu), x, x_scales=xs), want, bar)


def _experts(g, E, H, I, group, group2=None, zeros=False, zeros2=False, scales=BF16):
    return (ref.make(g, I, H, group, E, zeros, scales), ref.make(g, I, H, group, E, zeros, scales),
            ref.make(g, H, I, group2 or group, E, zeros2))


def _moe(mats, x, xs, ids, w, k):
    """The entry point's result, checked against 64 bits."""
    got = ops.w4_moe(*(ops.W4(*m) for m in mats), x, ids, w, k, x_scales=xs)
    d = [[ref.dense(*(None if v is None else v[e] for v in m)) for e in range(m[0].shape[0])]
         for m in mats]
    want, bar = ref.moe(*d, ref.values(x, xs), ids, w, k, x.dtype != I8)
    _near(got, want, bar)
    return got


def _routing(g, T, E, k):
    top = torch.randn(T, E, generator=g).topk(k, 1)
    return (top.indices.int().flatten().cuda(),
            torch.softmax(top.values, 1).flatten().contiguous().cuda())


MOE = [  # T, E, k, H, I, group of gate and up, of down
    (1, 8, 2, 128, 64, 64, 32), (1, 256, 16, 64, 32, 32, 32), (1, 16, 4, 2048, 768, 128, 128),
    (2, 8, 8, 96, 160, 32, 32), (3, 5, 2, 256, 384, 128, 128), (5, 16, 3, 288, 96, 32, 32),
    (16, 4, 2, 512, 256, 128, 64), (20, 64, 6, 384, 192, 64, 64), (40, 3, 1, 160, 224, 32, 32),
    (70, 2, 2, 256, 128, 256, 128), (130, 8, 3, 384, 256, 128, 128), (257, 6, 2, 224, 288, 32, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,H,I,group,group2", MOE)
@pytest.mark.parametrize("dtype,zeros", [(F32, False), (BF16, True), (I8, False), (BF16, False)])
def test_moe(cuda, T, E, k, H, I, group, group2, dtype, zeros):
    g = torch.Generator().manual_seed(T + E + H)
    mats = _experts(g, E, H, I, group, group2, zeros, not zeros, F32 if zeros else BF16)
    x, xs = _x(g, T, H, dtype, 128 if H % 128 == 0 else 0)
    _moe(mats, x, xs, *_routing(g, T, E, k), k)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 6, 90])
def test_moe_any_ids(cuda, T):
    # repeated experts in a token, ids of no expert, one expert for all, none
    g = torch.Generator().manual_seed(T)
    E, k, H, I = 7, 4, 256, 160
    mats = _experts(g, E, H, I, 32)
    x, _ = _x(g, T, H, BF16)
    w = torch.rand(T * k, generator=g).cuda()
    some = torch.randint(0, E, (T * k,), generator=g).int()
    some[1::5] = E
    some[3::7] = -1
    some[::11] = 2 ** 31 - 1
    _moe(mats, x, None, some.cuda(), w, k)
    _moe(mats, x, None, torch.full((T * k,), 3).int().cuda(), w, k)
    out = _moe(mats, x, None, torch.full((T * k,), E).int().cuda(), w, k)
    assert not out.any()
    for e in (2, E):
        _moe(mats, x, None, torch.full((T,), e).int().cuda(), w[:T].contiguous(), 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("std", [1e-38, 1e-30, 1e-18, 1e18, 1e30])
def test_sizes_of_the_values(cuda, dtype, std):
    # activations below 2^-96 share the step of that size: 2^-118 and half of
    # it as an error, which the bar takes in as such
    g = torch.Generator().manual_seed(5)
    for T in (1, 20):
        m = ref.make(g, 40, 416, 32)
        x, _ = _x(g, T, 416, dtype, std=std)
        w, v = ref.dense(*m), ref.values(x)
        want, bar = ref.linear(w, v)
        bar = bar + 2.0 ** -119 * w.abs().sum(1) + 2.0 ** -149 * 20
        _near(ops.w4_matvec_add2(ops.W4(*m), x), want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 9, 40, 300])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_vanishing_activations(cuda, T, group, dtype):
    # down to fp32's smallest normal values a chunk's largest sets its step, as the
    # header says; below, half of 2^-148. Results round to a multiple of 2^-149,
    # (4 * 3 + 16) times
    g = torch.Generator().manual_seed(T + group)
    m = ref.make(g, 40, 384, group, scales=F32, scale=3.0)
    w, handle = ref.dense(*m), ops.W4(*m)
    for std in (1e-28, 1e-30, 1e-33, 1e-35, 1e-36, 1e-37, 1e-38, 1e-40, 1e-43):
        x, _ = _x(g, T, 384, dtype, std=std)
        want, bar = ref.linear(w, ref.values(x))
        bar = bar + 2.0 ** -149 * (w.abs().sum(1) + 28)
        _near(ops.w4_matvec_add2(handle, x), want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 128])
def test_extreme_codes_and_zero_points(cuda, group):
    # the largest sums: every code 0 or 15, zero points of any byte, digits of
    # one sign
    for T in (1, 8, 40):
        for code in (0x00, 0xff, 0xf0):
            for z in (None, 0, 15, 255):
                codes = torch.full((24, 128), code, dtype=torch.uint8, device=cuda)
                s = torch.full((24, 256 // group), 0.5, device=cuda)
                zp = None if z is None else torch.full_like(s, z).to(torch.uint8)
                for x, xs in ((torch.full((T, 256), 127, dtype=I8, device=cuda),
                               torch.ones(T, 1, device=cuda)),
                              (torch.full((T, 256), -128, dtype=I8, device=cuda),
                               torch.ones(T, 1, device=cuda)),
                              (torch.full((T, 256), 1.9921875, device=cuda), None),
                              (torch.full((T, 256), -1.9999999, device=cuda), None)):
                    want, bar = ref.linear(ref.dense(codes, s, zp), ref.values(x, xs), xs is None)
                    _near(ops.w4_matvec_add2(ops.W4(codes, s, zp), x, x_scales=xs), want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 128])
def test_zero_points_above_127_count_as_127(cuda, group):
    g = torch.Generator().manual_seed(group)
    codes, s, z = ref.make(g, 40, 256, group, zeros=True)
    z[::2] += 100
    z[1::4] = 127
    z[::3, 0] = 255
    plain = ops.W4(codes, s, z.clamp(max=127))
    w = ops.W4(codes, s, z)
    assert int(z.max()) == 255
    for T in (1, 8, 40):
        for dtype in (F32, BF16, I8):
            x, xs = _x(g, T, 256, dtype)
            got = ops.w4_matvec_add2(w, x, x_scales=xs)
            assert torch.equal(got, ops.w4_matvec_add2(plain, x, x_scales=xs))
            # the definition's matrix, of the zero points that count
            q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).cpu().double()
            zz = z.cpu().double().clamp(max=127).repeat_interleave(group, 1)
            d = (q - zz) * s.cpu().double().repeat_interleave(group, 1)
            want, bar = ref.linear(d, ref.values(x, xs), dtype != I8)
            _near(got, want, bar)


@pytest.mark.gpu
def test_digits_hold_bf16_whole(cuda):
    # one column at a time through a matrix of ones: values down to 2^-14 of
    # their chunk's largest come back as they are
    K = 128
    x = torch.zeros(64, K)
    i = torch.arange(64)
    x[:, 0] = 1.9921875                                # the chunk's largest
    x[i, 1 + i] = (1 + i / 64.0) * 2.0 ** -(i % 15)
    x = x.to(BF16)
    codes = torch.full((16, K // 2), 0x99, dtype=torch.uint8)  # 9 - 8 = 1
    codes[:, 0] = 0x98                                 # column 0: 0
    w = ops.W4(codes.cuda(), torch.ones(16, 1, device=cuda))
    want = x[:, 1:].double().sum(1, keepdim=True).expand(-1, 16)
    for T in (1, 4, 64):
        assert torch.equal(ops.w4_matvec_add2(w, x[:T].cuda()).cpu().double(), want[:T])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 9, 40, 100])
@pytest.mark.parametrize("group", [32, 128])
def test_not_finite_and_zero_rows(cuda, T, group):
    g = torch.Generator().manual_seed(T)
    E, k, H, I = 6, 2, 256, 128
    mats = _experts(g, E, H, I, group)
    ws = [ops.W4(*m) for m in mats]
    x, _ = _x(g, T, H, F32)
    ids, w = _routing(g, T, E, k)
    clean = ops.w4_moe(*ws, x, ids, w, k)
    bad = x.clone()
    bad[0, 200] = float("nan")
    bad[T // 2, 3] = float("inf")
    if T > 2:
        bad[T - 1] = 0.0
    out = ops.w4_moe(*ws, bad, ids, w, k)
    lin = ops.w4_matvec_add2(ops.W4(*(v[0].contiguous() for v in mats[0] if v is not None)), bad)
    for t in range(T):
        if t in (0, T // 2):
            assert out[t].isnan().all() and lin[t].isnan().all()
        elif t == T - 1 and T > 2:
            assert not out[t].any() and not lin[t].any()
        else:
            assert torch.equal(out[t], clean[t])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 16, 65, 200])
def test_same_bits_again_and_rows_by_themselves(cuda, T):
    # the same call twice gives the same bits
    g = torch.Generator().manual_seed(2)
    mats = _experts(g, 8, 256, 192, 64)
    ws = [ops.W4(*m) for m in mats]
    x, _ = _x(g, T, 256, BF16)
    ids, w = _routing(g, T, 8, 3)
    a = ops.w4_moe(*ws, x, ids, w, 3)
    for _ in range(3):
        assert torch.equal(a, ops.w4_moe(*ws, x, ids, w, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("few,many", [(1, 4), (2, 3), (5, 16), (7, 13), (17, 64), (65, 200)])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype", [F32, BF16, I8])
def test_a_row_does_not_depend_on_the_others(cuda, few, many, group, dtype):
    # between sizes that take one kernel, in another order, and among other tokens
    g = torch.Generator().manual_seed(few)
    w, u = (ops.W4(*ref.make(g, 200, 1152, group)) for _ in range(2))
    x, xs = _x(g, many, 1152, dtype)
    y, ys = _x(g, many, 1152, dtype)
    y[:few] = x[:few]
    if xs is not None:
        ys[:few] = xs[:few]
    order = torch.randperm(many, generator=g).cuda()
    for f in (lambda a, s: ops.w4_matvec_add2(w, a, x_scales=s),
              lambda a, s: ops.w4_gate_up_swiglu(w, u, a, x_scales=s)):
        whole = f(x, xs)
        part = f(x[:few].contiguous(), None if xs is None else xs[:few].contiguous())
        assert torch.equal(whole[:few], part)
        assert torch.equal(f(y, ys)[:few], part)
        moved = f(x[order].contiguous(), None if xs is None else xs[order].contiguous())
        assert torch.equal(moved, whole[order])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 6, 40, 150])
@pytest.mark.parametrize("dtype", [F32, BF16, I8])
def test_a_routed_token_does_not_depend_on_the_others(cuda, T, dtype):
    g = torch.Generator().manual_seed(T)
    mats = _experts(g, 8, 256, 192, 64)
    ws = [ops.W4(*m) for m in mats]
    x, xs = _x(g, T, 256, dtype)
    ids, w = _routing(g, T, 8, 3)
    whole = ops.w4_moe(*ws, x, ids, w, 3, x_scales=xs)
    order = torch.randperm(T, generator=g).cuda()
    moved = ops.w4_moe(*ws, x[order].contiguous(), ids.view(T, 3)[order].flatten(),
                       w.view(T, 3)[order].flatten(), 3,
                       x_scales=None if xs is None else xs[order].contiguous())
    assert torch.equal(moved, whole[order])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [17, 70, 300])
@pytest.mark.parametrize("K", [32, 128, 1152])
@pytest.mark.parametrize("dtype,group,planes", [(BF16, 32, 1), (BF16, 128, 1), (F32, 32, 2)])
def test_fp16_sums_of_one_sign(cuda, T, K, dtype, group, planes):
    # Many tokens sum a chunk's products of fp16 values in fp32. Whatever the order
    # inside a matrix instruction, a chunk has at most 128 additions a plane, each off
    # by at most 2^-23 (were it cut off) of a partial sum of one sign; the rest as in
    # w4_reference.py
    group = min(group, K) if K % 128 else group
    g = torch.Generator().manual_seed(K)
    codes = torch.randint(9, 16, (50, K), generator=g, dtype=torch.uint8)
    packed = (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous()
    s = 0.01 * (1.0 + torch.rand(50, K // group, generator=g))
    x = (0.5 + torch.rand(T, K, generator=g)).to(dtype)
    w = ref.dense(packed, s)
    want, bar = ref.linear(w, x.double())
    bar = bar + 256 * planes * ref.U * want
    _near(ops.w4_matvec_add2(ops.W4(packed.cuda(), s.cuda()), x.cuda()), want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 33])
def test_only_the_outputs_are_written(cuda, T):
    # the library's call with outputs inside a larger buffer and a workspace of
    # exactly the size asked for, both with a border that has to stay
    g = torch.Generator().manual_seed(8)
    E, k, H, I = 5, 2, 160, 96
    mats = _experts(g, E, H, I, 32, zeros=True)
    ws = [ops.W4(*m) for m in mats]
    x, _ = _x(g, T, H, F32)
    ids, w = _routing(g, T, E, k)
    want = ops.w4_moe(*ws, x, ids, w, k)
    n = lib().inferno_w4_moe_workspace_bytes(T, k, E, H, I)
    buf = torch.full((n + 512,), 171, dtype=torch.uint8, device=cuda)
    out = torch.full((T + 2, H), 5.0, device=cuda)
    s = torch.cuda.current_stream().cuda_stream
    assert lib().inferno_w4_moe(s, ws[0].ref, ws[1].ref, ws[2].ref, x.data_ptr(), 0, None, 0,
                                ids.data_ptr(), w.data_ptr(), T, k, out[1:].data_ptr(),
                                buf[256:].data_ptr(), n) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[1:-1], want) and (out[0] == 5).all() and (out[-1] == 5).all()
    assert (buf[:256] == 171).all() and (buf[-256:] == 171).all()


@pytest.mark.gpu
def test_residual_in_place(cuda):
    g = torch.Generator().manual_seed(9)
    m = ref.make(g, 64, 256, 64)
    w = ops.W4(*m)
    for T in (1, 20, 100):
        x, _ = _x(g, T, 256, BF16)
        r = torch.randn(T, 64, generator=g).cuda()
        want = ops.w4_matvec_add2(w, x, r)
        n = lib().inferno_w4_workspace_bytes(T, 256)
        ws = torch.empty(n, dtype=torch.uint8, device=cuda)
        s = torch.cuda.current_stream().cuda_stream
        assert lib().inferno_w4_matvec_add2(s, w.ref, x.data_ptr(), 1, None, 0, r.data_ptr(), None,
                                            T, r.data_ptr(), ws.data_ptr(), n) == 0
        torch.cuda.synchronize()
        assert torch.equal(r, want)


@pytest.mark.gpu
def test_no_tokens(cuda):
    g = torch.Generator().manual_seed(1)
    mats = _experts(g, 4, 64, 32, 32)
    ws = [ops.W4(*m) for m in mats]
    x = torch.zeros(0, 64, device=cuda)
    ids, w = torch.zeros(0, dtype=torch.int32, device=cuda), torch.zeros(0, device=cuda)
    assert ops.w4_moe(*ws, x, ids, w, 2).shape == (0, 64)
    one = ops.W4(*ref.make(g, 48, 64, 32))
    assert ops.w4_matvec_add2(one, x).shape == (0, 48)
    assert ops.w4_gate_up_swiglu(one, one, x).shape == (0, 48)


def _cpu(rows=16, cols=64, group=32, experts=0, **kw):
    return ref.make(torch.Generator().manual_seed(0), rows, cols, group, experts, device="cpu", **kw)


def _unpacked(rows=16, cols=64, experts=1):
    """A handle of these sizes without its matrix: the checks come first."""
    w = object.__new__(ops.W4)
    w.rows, w.cols, w.experts, w.device = rows, cols, experts, torch.device("cpu")
    w.ref = _desc(experts, rows, cols)
    return w


def test_refusals_of_the_wrappers():
    codes, scales, _ = _cpu()
    with pytest.raises(ValueError, match="codes"):
        ops.W4(codes.int(), scales)
    with pytest.raises(ValueError, match="codes"):
        ops.W4(codes.T, scales)
    with pytest.raises(ValueError, match="scales"):
        ops.W4(codes, scales.half())
    with pytest.raises(ValueError, match="scales"):
        ops.W4(codes, scales[:-1])
    with pytest.raises(ValueError, match="do not divide"):
        ops.W4(codes, torch.zeros(16, 3))
    with pytest.raises(ValueError, match="zeros"):
        ops.W4(codes, scales, torch.zeros(16, 2, dtype=torch.int8))
    with pytest.raises(ValueError, match="GPU tensors"):
        ops.W4(codes, scales)
    w = _unpacked()
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="GPU tensors"):
        ops.w4_matvec_add2(w, x)
    with pytest.raises(ValueError, match="x must"):
        ops.w4_matvec_add2(w, torch.zeros(2, 32))
    with pytest.raises(ValueError, match="x must"):
        ops.w4_matvec_add2(w, x.half())
    with pytest.raises(ValueError, match="contiguous"):
        ops.w4_matvec_add2(w, torch.zeros(64, 2).T)
    with pytest.raises(ValueError, match="x_scales"):
        ops.w4_matvec_add2(w, x.to(I8))
    with pytest.raises(ValueError, match="x_scales"):
        ops.w4_matvec_add2(w, x.to(I8), x_scales=torch.zeros(2, 3))
    with pytest.raises(ValueError, match="x_scales"):
        ops.w4_matvec_add2(w, x.to(I8), x_scales=torch.zeros(3, 1))
    with pytest.raises(ValueError, match="belong"):
        ops.w4_matvec_add2(w, x, x_scales=torch.zeros(2, 1))
    with pytest.raises(ValueError, match="residual_a"):
        ops.w4_matvec_add2(w, x, torch.zeros(2, 15))
    mats = [_unpacked(32, 64, 4), _unpacked(32, 64, 4), _unpacked(64, 32, 4)]
    ids, wt = torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    with pytest.raises(ValueError, match="ids"):
        ops.w4_moe(*mats, x, ids.long(), wt, 2)
    with pytest.raises(ValueError, match="ids"):
        ops.w4_moe(*mats, x, ids, wt, 3)
    with pytest.raises(ValueError, match="weights"):
        ops.w4_moe(*mats, x, ids, wt[:3], 2)
    with pytest.raises(ValueError, match="k must"):
        ops.w4_moe(*mats, x, ids, wt, 0)


def _desc(experts=1, rows=16, cols=64, group=32, p=16, **more):
    d = W4Desc(experts, rows, cols, group, 0, 0, p, 0)
    d.packed_bytes = lib().inferno_w4_packed_bytes(d)
    for name, v in more.items():
        setattr(d, name, v)
    return d


BAD_SIZES = [dict(rows=0), dict(cols=0), dict(experts=0), dict(group=0), dict(group=48),
             dict(group=128), dict(group=96, cols=96), dict(cols=48, group=16),
             dict(scale_dtype=2), dict(experts=257), dict(rows=1 << 20, cols=1 << 13, group=128),
             dict(rows=1 << 31), dict(cols=1 << 31), dict(rows=(1 << 25) + 1)]


def test_packed_bytes():
    L = lib()

    def size(zeros=0, dtype=0, **kw):
        d = _desc(**kw)
        d.has_zeros, d.scale_dtype = zeros, dtype
        return L.inferno_w4_packed_bytes(d)

    # 16 rows by 128 columns: 1024 bytes of codes, 16 scales or 16 times 4
    assert size(rows=16, cols=128, group=128, dtype=1) == 1024 + 256
    assert size(rows=17, cols=160, group=32, dtype=1) == 4 * 1024 + 4 * 128
    assert size(rows=64, cols=1024, group=64, dtype=0, zeros=1) == 32 * (1024 + 256 + 64)
    assert size(experts=3, rows=16, cols=256, group=256, dtype=0, zeros=1) == 6 * 1024 + 512 + 256
    for kw in BAD_SIZES:
        assert L.inferno_w4_packed_bytes(_desc(**kw)) == 0, kw


def test_refusals_of_the_library():
    # every one before any device work
    L = lib()

    def pack(d, codes=16, nc=512, scales=16, ns=128, zeros=None, nz=0, to=16):
        return L.inferno_w4_pack(None, d, codes, nc, scales, ns, zeros, nz, to)

    d = _desc()
    for bad in (dict(codes=None), dict(codes=18), dict(scales=None), dict(scales=18), dict(to=None),
                dict(to=24)):
        assert pack(d, **bad) == -1, bad
    for bad in (dict(nc=511), dict(ns=64)):
        assert pack(d, **bad) == -2, bad
    z = _desc(has_zeros=1)
    z.packed_bytes = L.inferno_w4_packed_bytes(z)
    assert pack(z, nz=32) == -1 and pack(z, zeros=16, nz=31) == -2
    assert pack(_desc(packed_bytes=10)) == -2
    for kw in BAD_SIZES:
        assert pack(_desc(**kw)) == -1, kw

    def matvec(d, x=16, dt=0, xs=None, xg=0, T=1, out=16, ws=16, n=1 << 30):
        return L.inferno_w4_matvec_add2(None, d, x, dt, xs, xg, None, None, T, out, ws, n)

    for kw in BAD_SIZES + [dict(packed=None), dict(packed=24), dict(experts=2)]:
        assert matvec(_desc(**kw)) == -1, kw
    assert matvec(_desc(packed_bytes=1024)) == -2 and matvec(_desc(has_zeros=1)) == -2
    assert matvec(d, x=None) == -1 and matvec(d, x=20) == -1 and matvec(d, dt=3) == -1
    assert matvec(d, out=None) == -1 and matvec(d, ws=None) == -2 and matvec(d, n=100) == -2
    assert matvec(d, ws=24) == -1 and matvec(d, T=1 << 31) == -1
    assert matvec(d, dt=2) == -1  # no scales
    big = _desc(cols=512, group=128)
    for xg in (64, 192, 1024, 32):
        assert matvec(big, dt=2, xs=16, xg=xg) == -1
    assert matvec(d, x=None, T=0, out=None, ws=None, n=0) == 0

    def pair(a, b):
        return L.inferno_w4_gate_up_swiglu(None, a, b, 16, 0, None, 0, 1, 16, 16, 1 << 30)

    half = _desc()
    half.scale_dtype = 1
    half.packed_bytes = L.inferno_w4_packed_bytes(half)
    for b in (_desc(rows=32), _desc(cols=128), _desc(group=64), z, half):
        assert pair(d, b) == -1 and b"same" in L.inferno_last_error()

    def moe(g, u, dn, ids=16, k=2, T=1, n=1 << 30):
        return L.inferno_w4_moe(None, g, u, dn, 16, 0, None, 0, ids, 16, T, k, 16, 16, n)

    g, dn = _desc(4, 32, 64), _desc(4, 64, 32)
    for down in (_desc(3, 64, 32), _desc(4, 32, 32), _desc(4, 64, 64)):
        assert moe(g, g, down) == -1 and b"changed over" in L.inferno_last_error()
    assert moe(g, g, dn, k=0) == -1 and moe(g, g, dn, k=17) == -1
    assert moe(g, g, dn, ids=None) == -1 and moe(g, g, dn, n=10) == -2
    assert moe(g, g, dn, T=1 << 27) == -1
    assert moe(g, g, dn, T=0) == 0


def test_workspace_does_not_fall():
    L = lib()
    for K in (32, 160, 4096):
        need = [L.inferno_w4_workspace_bytes(T, K) for T in range(0, 300)]
        assert need == sorted(need)
        need = [L.inferno_w4_moe_workspace_bytes(T, 8, 64, K, 96) for T in range(0, 300)]
        assert need == sorted(need)


@pytest.mark.gpu
def test_library_errors_reach_the_caller(cuda):
    g = torch.Generator().manual_seed(1)
    a, b = ops.W4(*ref.make(g, 16, 64, 32)), ops.W4(*ref.make(g, 16, 64, 64))
    with pytest.raises(InfernoError, match="same group"):
        ops.w4_gate_up_swiglu(a, b, torch.zeros(1, 64, device=cuda))
    with pytest.raises(InfernoError, match="group"):
        ops.W4(*ref.make(g, 16, 96, 96))
    with pytest.raises(InfernoError, match="plain product"):
        ops.w4_matvec_add2(ops.W4(*ref.make(g, 16, 64, 32, 2)), torch.zeros(1, 64, device=cuda))
    buf = torch.zeros(65, device=cuda)
    with pytest.raises(InfernoError, match="multiple of 16"):
        ops.w4_matvec_add2(a, buf[1:].view(1, 64))
