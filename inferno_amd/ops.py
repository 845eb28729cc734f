"""Torch-tensor wrappers over the C ABI (device memory and streams only).

Every function here calls straight into libinferno_moe.so; tensors must live
on the GPU. uint32 outputs of the ABI are held in torch.int32 tensors.
"""
import ctypes as C

import torch

from ._lib import BF16, F32, I8, Q8_0, LayerDesc, W4Desc, check, lib

_DT = {torch.float32: F32, torch.bfloat16: BF16}

# a device's current stream as an integer, without a Stream object (3 us each)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _s():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dev(t):
    if not t.is_cuda:
        raise ValueError("inferno_amd ops need GPU tensors")
    return t


def block_bytes(quant):
    return lib().inferno_block_bytes(quant)


def block_values(quant):
    return lib().inferno_block_values(quant)


def matrix_bytes(quant, rows, cols):
    return rows * (cols // block_values(quant)) * block_bytes(quant)


def dequantize(quant, blocks):
    n_blocks = blocks.numel() // block_bytes(quant)
    out = torch.empty(n_blocks * block_values(quant), dtype=torch.float32, device=blocks.device)
    check(lib().inferno_gguf_dequantize(_s(), quant, _p(_dev(blocks)), n_blocks, _p(out)))
    return out


def router_logits(x, w_router):
    T, H = x.shape
    E = w_router.shape[0]
    out = torch.empty(T, E, dtype=torch.float32, device=x.device)
    check(lib().inferno_router_logits(_s(), _p(_dev(x)), _DT[x.dtype], _p(w_router), T, H, E,
                                      _p(out)))
    return out


def router_topk(logits, bias, k, score_fn, norm, scale):
    T, E = logits.shape
    ids = torch.empty(T * k, dtype=torch.int32, device=logits.device)
    w = torch.empty(T * k, dtype=torch.float32, device=logits.device)
    tok = torch.empty(T * k, dtype=torch.int32, device=logits.device)
    check(lib().inferno_moe_router_topk(_s(), _p(_dev(logits)), _p(bias), T, E, k, score_fn,
                                        int(norm), float(scale), _p(ids), _p(w), _p(tok)))
    return ids, w, tok


def dispatch(ids, T, k, E):
    dev = ids.device
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    sorted_ = torch.empty(max(T * k, 1), dtype=torch.int32, device=dev)
    active = torch.empty(E + 1, dtype=torch.int32, device=dev)
    check(lib().inferno_moe_dispatch(_s(), _p(_dev(ids)), T, k, E, _p(offsets), _p(sorted_),
                                     _p(active)))
    return offsets, sorted_[: T * k], active


def gguf_moe(quant, down_quant, gate, up, down, x, ids, weights, k, E, I):
    T, H = x.shape
    ws_bytes = lib().inferno_gguf_moe_workspace_bytes(T, k, E, H, I)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
    out = torch.empty(T, H, dtype=torch.float32, device=x.device)
    check(lib().inferno_gguf_moe(_s(), quant, down_quant, _p(gate), gate.numel(), _p(up),
                                 up.numel(), _p(down), down.numel(), _p(_dev(x)), _DT[x.dtype],
                                 _p(ids), _p(weights), T, k, E, H, I, _p(out), _p(ws), ws_bytes))
    return out


def gemv_workspace(rows, K, device):
    n = lib().inferno_gemv_workspace_bytes(rows, K)
    return torch.empty(max(n, 1), dtype=torch.uint8, device=device)


def expert_gate_up_swiglu(quant, gate, up, x, offsets, sorted_, active, weights, k, E, I,
                          out=None, ws=None):
    T, H = x.shape
    if out is None:
        out = torch.empty(T * k, I, dtype=torch.float32, device=x.device)
    if ws is None:
        ws = gemv_workspace(T, H, x.device)
    check(lib().inferno_moe_expert_gate_up_swiglu(
        _s(), quant, _p(gate), gate.numel(), _p(up), up.numel(), _p(_dev(x)), _DT[x.dtype],
        _p(offsets), _p(sorted_), _p(active), _p(weights), T, k, E, H, I, _p(out), _p(ws),
        ws.numel()))
    return out


def expert_down(down_quant, down, h, offsets, sorted_, active, T, k, E, H, out=None, ws=None):
    I = h.shape[1]
    if out is None:
        out = torch.empty(T * k, H, dtype=torch.float32, device=h.device)
    if ws is None:
        ws = gemv_workspace(T * k, I, h.device)
    check(lib().inferno_moe_expert_down(_s(), down_quant, _p(down), down.numel(), _p(_dev(h)),
                                        _p(offsets), _p(sorted_), _p(active), T, k, E, H, I,
                                        _p(out), _p(ws), ws.numel()))
    return out


def q8_0_gate_up_swiglu(gate, up, x, Is):
    T, H = x.shape
    out = torch.empty(T, Is, dtype=torch.float32, device=x.device)
    ws = gemv_workspace(T, H, x.device)
    check(lib().inferno_q8_0_gate_up_swiglu(_s(), _p(gate), gate.numel(), _p(up), up.numel(),
                                            _p(_dev(x)), _DT[x.dtype], T, H, Is, _p(out), _p(ws),
                                            ws.numel()))
    return out


def q8_0_matvec_add2(w, inp, residual_a, residual_b, O):
    T, In = inp.shape
    out = torch.empty(T, O, dtype=torch.float32, device=inp.device)
    ws = gemv_workspace(T, In, inp.device)
    check(lib().inferno_q8_0_matvec_add2(_s(), _p(w), w.numel(), _p(_dev(inp)), _p(residual_a),
                                         _p(residual_b), T, In, O, _p(out), _p(ws), ws.numel()))
    return out


def topk_combine_residual(shared, residual, expert_outputs, expert_weights, k):
    A, H = expert_outputs.shape
    T = A // k
    out = torch.empty(T, H, dtype=torch.float32, device=expert_outputs.device)
    check(lib().inferno_moe_topk_combine_residual(_s(), _p(shared), _p(residual),
                                                  _p(_dev(expert_outputs)), _p(expert_weights),
                                                  T, H, k, _p(out)))
    return out


def weighted_index_add_combine(acc, token_indices, expert_outputs, expert_weights):
    T, H = acc.shape
    A = token_indices.numel()
    out = torch.empty_like(acc)
    check(lib().inferno_moe_weighted_index_add_combine(_s(), _p(_dev(acc)), _p(token_indices),
                                                       _p(expert_outputs), _p(expert_weights),
                                                       T, H, A, _p(out)))
    return out


def gather_tokens(x, token_indices):
    T, H = x.shape
    A = token_indices.numel()
    out = torch.empty(A, H, dtype=torch.float32, device=x.device)
    check(lib().inferno_moe_gather_tokens(_s(), _p(_dev(x)), _p(token_indices), T, H, A, _p(out)))
    return out


def rms_norm(x, w, eps):
    rows, H = x.shape
    out = torch.empty_like(x)
    check(lib().inferno_rms_norm(_s(), _p(_dev(x)), _p(w), rows, H, float(eps), _p(out)))
    return out


def _like(x, name, t, dtype, *shape):
    """Refuses a tensor that an entry point cannot take: on another device than
    x, not of this type and shape, or not contiguous."""
    if t.dtype != dtype or t.shape != shape or t.device != x.device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on "
                         f"{x.device}, got {t.dtype} {tuple(t.shape)} on {t.device}"
                         f"{'' if t.is_contiguous() else ', not contiguous'}")


def _rows_of(x, name, dtypes):
    if x.dim() != 2 or x.dtype not in dtypes or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 2-D tensor of one of {dtypes}, got "
                         f"{x.dtype} {tuple(x.shape)}"
                         f"{'' if x.is_contiguous() else ', not contiguous'}")


def _at(t):
    return None if t is None else t.data_ptr()


def _run(x, fn, *args):
    """fn(stream, *args) on x's device and that device's current stream."""
    dev = _dev(x).get_device()
    if dev == torch.cuda.current_device():
        check(fn(_raw_stream(dev), *args))
    else:
        with torch.cuda.device(dev):
            check(fn(_raw_stream(dev), *args))


def add_rms_norm_q8(x, residual, w, eps, group=0, act_dtype=torch.float32, out=None):
    """Residual addition, RMSNorm and 8-bit activations (inferno_add_rms_norm_q8):
    s = x + residual (None: x), y = s / sqrt(mean(s^2) + eps) * w, and y in int8
    with one fp32 scale per ``group`` columns (32, 64, 128; 0: the row; the 4-bit
    products take those of 128 and of the row). Returns
    (s, y in act_dtype, q, scales); ``out`` (fp32, may be ``residual``) receives s."""
    _rows_of(x, "x", tuple(_DT))
    T, H = x.shape
    if group and (group not in (32, 64, 128) or H % group):
        raise ValueError(f"group must be 0, 32, 64 or 128 and divide the width {H}, got {group}")
    if act_dtype not in _DT:
        raise ValueError(f"act_dtype must be one of {tuple(_DT)}, got {act_dtype}")
    if residual is not None:
        _like(x, "residual", residual, torch.float32, T, H)
    _like(x, "w", w, torch.float32, H)
    if out is None:
        out = torch.empty(T, H, dtype=torch.float32, device=x.device)
    else:
        _like(x, "out", out, torch.float32, T, H)
    normed = torch.empty(T, H, dtype=act_dtype, device=x.device)
    q = torch.empty(T, H, dtype=torch.int8, device=x.device)
    scales = torch.empty(T, H // group if group else 1, dtype=torch.float32, device=x.device)
    _run(x, lib().inferno_add_rms_norm_q8, _at(x), _DT[x.dtype], _at(residual), _at(w), float(eps), T,
         H, group, _DT[act_dtype], _at(out), _at(normed), _at(q), _at(scales))
    return out, normed, q, scales


def router_group_topk(logits, bias, k, score_fn, norm, scale, n_group, topk_group, group_score):
    """``router_topk`` over the ``topk_group`` best of ``n_group`` groups of
    experts (inferno_moe_router_group_topk). With softmax, experts and groups are
    ranked by logit + bias, as ``router_topk`` does, not by their scores."""
    _rows_of(logits, "logits", (torch.float32,))
    T, E = logits.shape
    if bias is not None:
        _like(logits, "bias", bias, torch.float32, E)
    if k < 0 or n_group < 0 or topk_group < 0:
        raise ValueError("k, n_group and topk_group must not be negative")
    ids = torch.empty(T * k, dtype=torch.int32, device=logits.device)
    w = torch.empty(T * k, dtype=torch.float32, device=logits.device)
    tok = torch.empty(T * k, dtype=torch.int32, device=logits.device)
    _run(logits, lib().inferno_moe_router_group_topk, _at(logits), _at(bias), T, E, k, score_fn,
         int(norm), float(scale), n_group, topk_group, group_score, _at(ids), _at(w), _at(tok))
    return ids, w, tok


class W4:
    """4-bit weights with group scales (struct inferno_w4): one matrix [rows,
    cols], or one per expert [E, rows, cols]. ``codes`` holds two columns a byte
    (uint8 [..., cols / 2], the even column in the low nibble), ``scales`` one
    factor per cols / scales.shape[-1] columns (fp32 or bf16), ``zeros`` a zero
    point for each scale (uint8; None: 8), of which one above 127 counts as 127.
    Packed once, here, on the current stream (inferno_w4_pack), which is waited for:
    the handle may be used on any stream at once, and the tensors are not kept. While
    the stream is being captured nothing is waited for; such a handle holds its matrix
    after the graph's first replay."""

    def __init__(self, codes, scales, zeros=None):
        if codes.dtype != torch.uint8 or codes.dim() not in (2, 3) or not codes.is_contiguous():
            raise ValueError("codes must be a contiguous 2-D or 3-D uint8 tensor, got "
                             f"{codes.dtype} {tuple(codes.shape)}")
        if scales.dtype not in _DT:
            raise ValueError(f"scales must be one of {tuple(_DT)}, got {scales.dtype}")
        rows, cols = codes.shape[-2], 2 * codes.shape[-1]
        groups = scales.shape[-1] if scales.dim() else 0
        if groups == 0 or cols % groups:
            raise ValueError(f"{groups} scales a row do not divide {cols} columns")
        _like(codes, "scales", scales, scales.dtype, *codes.shape[:-1], groups)
        if zeros is not None:
            _like(codes, "zeros", zeros, torch.uint8, *codes.shape[:-1], groups)
        self.device = codes.device
        self.experts = codes.shape[0] if codes.dim() == 3 else 1
        self.rows, self.cols, self.group = rows, cols, cols // groups
        d = W4Desc(self.experts, rows, cols, self.group, _DT[scales.dtype], int(zeros is not None),
                   None, 0)
        self.desc, self.ref = d, C.byref(d)
        d.packed_bytes = lib().inferno_w4_packed_bytes(self.ref)
        self.packed = torch.empty(d.packed_bytes, dtype=torch.uint8, device=codes.device)
        _run(codes, lib().inferno_w4_pack, self.ref, _at(codes), codes.numel(), _at(scales),
             scales.numel() * scales.element_size(), _at(zeros),
             zeros.numel() if zeros is not None else 0, _at(self.packed))
        d.packed = self.packed.data_ptr()
        stream = torch.cuda.current_stream(self.device)
        with torch.cuda.device(self.device):
            if not torch.cuda.is_current_stream_capturing():
                stream.synchronize()


_ACT = {torch.float32: F32, torch.bfloat16: BF16, torch.int8: I8}


def _w4_x(w, x, x_scales):
    """Checks activations of a 4-bit product; their type, scales and group."""
    _rows_of(x, "x", tuple(_ACT))
    if x.shape[1] != w.cols or x.device != w.device:
        raise ValueError(f"x must be [tokens, {w.cols}] on {w.device}, got {tuple(x.shape)} on "
                         f"{x.device}")
    if x.dtype != torch.int8:
        if x_scales is not None:
            raise ValueError("x_scales belong to int8 activations")
        return _ACT[x.dtype], None, 0
    if x_scales is None or x_scales.dim() != 2 or not x_scales.shape[1] or \
            w.cols % x_scales.shape[1]:
        raise ValueError("int8 activations need x_scales [tokens, groups], groups dividing "
                         f"{w.cols}")
    _like(x, "x_scales", x_scales, torch.float32, x.shape[0], x_scales.shape[1])
    return I8, _at(x_scales), w.cols // x_scales.shape[1]


def _w4_ws(x, n):
    return torch.empty(n, dtype=torch.uint8, device=x.device)


def w4_matvec_add2(w, x, residual_a=None, residual_b=None, x_scales=None):
    """residual_a + residual_b + x W^T for a 4-bit matrix (inferno_w4_matvec_add2).
    x: fp32, bf16, or int8 with ``x_scales`` (add_rms_norm_q8's, group 128 or 0)."""
    dt, xs, xg = _w4_x(w, x, x_scales)
    T = x.shape[0]
    for name, r in (("residual_a", residual_a), ("residual_b", residual_b)):
        if r is not None:
            _like(x, name, r, torch.float32, T, w.rows)
    out = torch.empty(T, w.rows, dtype=torch.float32, device=x.device)
    n = lib().inferno_w4_workspace_bytes(T, w.cols)
    ws = _w4_ws(x, n)
    _run(x, lib().inferno_w4_matvec_add2, w.ref, _at(x), dt, xs, xg, _at(residual_a),
         _at(residual_b), T, _at(out), _at(ws), n)
    return out


def w4_gate_up_swiglu(gate, up, x, x_scales=None):
    """silu(x W_gate^T) * (x W_up^T) for 4-bit matrices (inferno_w4_gate_up_swiglu)."""
    dt, xs, xg = _w4_x(gate, x, x_scales)
    if up.device != x.device:
        raise ValueError(f"the up matrix must be on {x.device}, got {up.device}")
    T = x.shape[0]
    out = torch.empty(T, gate.rows, dtype=torch.float32, device=x.device)
    n = lib().inferno_w4_workspace_bytes(T, gate.cols)
    ws = _w4_ws(x, n)
    _run(x, lib().inferno_w4_gate_up_swiglu, gate.ref, up.ref, _at(x), dt, xs, xg, T, _at(out),
         _at(ws), n)
    return out


def w4_moe(gate, up, down, x, ids, weights, k, x_scales=None):
    """Routed experts with 4-bit weights (inferno_w4_moe): gate and up [E, I, H],
    down [E, H, I]; ids and weights [T * k] as ``router_topk`` returns them."""
    dt, xs, xg = _w4_x(gate, x, x_scales)
    if up.device != x.device or down.device != x.device:
        raise ValueError(f"the expert matrices must be on {x.device}")
    T, H = x.shape
    if k < 1:
        raise ValueError(f"k must be positive, got {k}")
    _like(x, "ids", ids, torch.int32, T * k)
    _like(x, "weights", weights, torch.float32, T * k)
    out = torch.empty(T, H, dtype=torch.float32, device=x.device)
    n = lib().inferno_w4_moe_workspace_bytes(T, k, gate.experts, H, gate.rows)
    ws = _w4_ws(x, n)
    _run(x, lib().inferno_w4_moe, gate.ref, up.ref, down.ref, _at(x), dt, xs, xg, _at(ids),
         _at(weights), T, k, _at(out), _at(ws), n)
    return out


class NormRouter:
    """RMSNorm -> router logits (-> top-k) of decode tokens in one launch
    (inferno_rms_norm_router_topk; Backend::laguna_xs_rms_norm_router_device
    followed by the decode top-k). Holds the zero-filled ticket workspace the
    top-k needs; calls through one instance must not overlap."""

    def __init__(self, max_tokens=1, device="cuda"):
        self._ws = torch.zeros(lib().inferno_rms_norm_router_topk_workspace_bytes(max_tokens),
                               dtype=torch.uint8, device=device)
        self.max_tokens = max_tokens

    def __call__(self, x, norm_weight, eps, router, bias=None, k=0, score_fn=0, norm=True,
                 scale=1.0, act_dtype=torch.float32, topk=True):
        T, H = x.shape
        E = router.shape[0]
        if T > self.max_tokens:
            self.__init__(T, x.device)
        normed = torch.empty(T, H, dtype=act_dtype, device=x.device)
        logits = torch.empty(T, E, dtype=torch.float32, device=x.device)
        ids = torch.empty(T * k, dtype=torch.int32, device=x.device) if topk else None
        w = torch.empty(T * k, dtype=torch.float32, device=x.device) if topk else None
        check(lib().inferno_rms_norm_router_topk(
            _s(), _p(_dev(x)), _p(norm_weight), float(eps), _p(router), _p(bias), T, H, E, k,
            score_fn, int(norm), float(scale), _DT[act_dtype], _p(normed), _p(logits), _p(ids),
            _p(w), _p(self._ws), self._ws.numel()))
        return normed, logits, ids, w


TIMER_GATE_UP, TIMER_DOWN, TIMER_ROUTE, TIMER_SELECT = 0, 1, 2, 3


def kernel_timing(enable):
    """Turns the event timing of the layer's launches (route, select, gate/up,
    down) on or off. Events are recorded around each launch without a wait;
    ``kernel_timing_read`` settles and sums them (measurement only)."""
    check(lib().inferno_kernel_timing_enable(1 if enable else 0))


def kernel_timing_read(which):
    """(total ms, launches) accumulated by one timer since the last read."""
    ms, n = C.c_double(0.0), C.c_uint64(0)
    check(lib().inferno_kernel_timing_read(which, C.byref(ms), C.byref(n)))
    return ms.value, n.value


def kernel_timing_label(which):
    """Label of the last launch a timer measured: "<kind>: <kernel> (...)"."""
    buf = C.create_string_buffer(256)
    check(lib().inferno_kernel_timing_label(which, buf, len(buf)))
    return buf.value.decode()


def synth_normal(seed, stddev, n, dtype=torch.float32, device="cuda"):
    out = torch.empty(n, dtype=dtype, device=device)
    check(lib().inferno_synth_normal(_s(), seed, float(stddev), n, _DT[dtype], _p(out)))
    return out


def synth_quantized(quant, seed, stddev, rows, cols, device="cuda"):
    out = torch.empty(matrix_bytes(quant, rows, cols), dtype=torch.uint8, device=device)
    check(lib().inferno_synth_quantized(_s(), quant, seed, float(stddev), rows, cols, _p(out)))
    return out


def synth_normal_host(seed, stddev, n):
    out = torch.empty(n, dtype=torch.float32)
    check(lib().inferno_synth_normal_host(seed, float(stddev), n, _p(out)))
    return out


def synth_quantized_host(quant, seed, stddev, rows, cols):
    out = torch.empty(matrix_bytes(quant, rows, cols), dtype=torch.uint8)
    check(lib().inferno_synth_quantized_host(quant, seed, float(stddev), rows, cols, _p(out)))
    return out


def quantize_rows_host(quant, x):
    rows, cols = x.shape
    x = x.contiguous().float()
    out = torch.empty(matrix_bytes(quant, rows, cols), dtype=torch.uint8)
    check(lib().inferno_quantize_rows_host(quant, _p(x), rows, cols, _p(out)))
    return out


class MoELayer:
    """One MoE FFN layer resident on the GPU (inferno_moe_layer_forward).

    Holds device tensors for the router, routed experts and optional Q8_0
    shared expert, and a reusable workspace sized for `max_tokens`.
    """

    def __init__(self, *, hidden, experts, intermediate, top_k, quant, down_quant, score_fn,
                 norm_topk_prob, routed_scaling_factor, router, router_bias, gate, up, down,
                 shared_intermediate=0, shared_gate=None, shared_up=None, shared_down=None,
                 shared_quant=Q8_0, shared_down_quant=Q8_0, max_tokens=1):
        self.tensors = [router, router_bias, gate, up, down, shared_gate, shared_up, shared_down]
        d = LayerDesc()
        d.hidden, d.experts, d.intermediate, d.top_k = hidden, experts, intermediate, top_k
        d.quant, d.down_quant, d.score_fn = quant, down_quant, score_fn
        d.norm_topk_prob, d.routed_scaling_factor = int(norm_topk_prob), routed_scaling_factor
        d.router, d.router_bias = _p(router), _p(router_bias)
        d.gate, d.up, d.down = _p(gate), _p(up), _p(down)
        d.gate_bytes, d.up_bytes, d.down_bytes = gate.numel(), up.numel(), down.numel()
        d.shared_intermediate = shared_intermediate
        if shared_intermediate:
            d.shared_gate, d.shared_up, d.shared_down = _p(shared_gate), _p(shared_up), _p(shared_down)
            d.shared_gate_bytes = shared_gate.numel()
            d.shared_up_bytes = shared_up.numel()
            d.shared_down_bytes = shared_down.numel()
            d.shared_quant, d.shared_down_quant = shared_quant, shared_down_quant
        self.desc = d
        self.hidden, self.top_k = hidden, top_k
        self.device = gate.device
        self._ws = None
        self.reserve(max_tokens)

    def reserve(self, T):
        need = lib().inferno_moe_layer_workspace_bytes(C.byref(self.desc), T)
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)

    def forward(self, x, residual=None, out=None, ids=None, weights=None):
        T = x.shape[0]
        self.reserve(T)
        if out is None:
            out = torch.empty(T, self.hidden, dtype=torch.float32, device=x.device)
        check(lib().inferno_moe_layer_forward(
            _s(), C.byref(self.desc), _p(_dev(x)), _DT[x.dtype], _p(residual), T, _p(out),
            _p(ids), _p(weights), _p(self._ws), self._ws.numel()))
        return out


class MoEStack:
    """Consecutive MoE layers on one residual stream (inferno_moe_stack_forward):
    for each layer, RMSNorm of the stream (rounded to ``act_dtype``), then
    stream += routed + shared expert outputs of the normalised activations."""

    def __init__(self, layers, norm_weights, eps=1e-6, act_dtype=torch.bfloat16, max_tokens=1):
        if len(layers) != len(norm_weights) or not layers:
            raise ValueError("one RMSNorm weight per layer is needed")
        self.layers = list(layers)
        self.norm_weights = list(norm_weights)
        self.eps, self.act_dtype = float(eps), act_dtype
        n = len(layers)
        self.descs = (LayerDesc * n)(*[l.desc for l in layers])
        self.norm_ptrs = (C.c_void_p * n)(*[w.data_ptr() for w in norm_weights])
        self.hidden = layers[0].hidden
        self.device = layers[0].device
        self._ws = None
        self.reserve(max_tokens)

    def reserve(self, T):
        need = lib().inferno_moe_stack_workspace_bytes(self.descs, len(self.layers), T)
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)

    def forward(self, hidden, out=None, ids=None):
        """hidden: fp32 [T, H] residual stream. ids (optional int32 tensor of
        sum_l T*k_l) receives every layer's routing, layer after layer."""
        T = hidden.shape[0]
        self.reserve(T)
        if out is None:
            out = torch.empty(T, self.hidden, dtype=torch.float32, device=hidden.device)
        check(lib().inferno_moe_stack_forward(
            _s(), self.descs, len(self.layers), self.norm_ptrs, self.eps, _DT[self.act_dtype],
            _p(_dev(hidden)), T, _p(out), _p(ids), _p(self._ws), self._ws.numel()))
        return out


def layer_forward_noalloc(layer, x, residual=None, out=None, ids=None, weights=None):
    """``layer``'s forward through inferno_moe_layer_forward_noalloc: the
    library's fixed device scratch instead of a workspace (no allocation in
    the library; ``out`` is allocated here when not given)."""
    T = x.shape[0]
    if out is None:
        out = torch.empty(T, layer.hidden, dtype=torch.float32, device=x.device)
    check(lib().inferno_moe_layer_forward_noalloc(
        _s(), C.byref(layer.desc), _p(_dev(x)), _DT[x.dtype], _p(residual), T, _p(out), _p(ids),
        _p(weights)))
    return out
