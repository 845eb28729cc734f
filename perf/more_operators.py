"""Performance cases of the operators around experts in bfloat16 and in
microscaled 4-bit floating point: quantisation and products grouped by expert.

Each case is a dict of plain values. ``op`` names the operator:

  quantize  ops.mxfp4_quantize: rows to 4-bit floating point
  matmul    ops.grouped_matmul: rows grouped by expert, each times its expert
  swiglu    ops.grouped_gate_up_swiglu: the same for gate and up matrices

MXFP4 is one code per value (sign, two bits of exponent, one of mantissa: 0, 0.5,
1, 1.5, 2, 3, 4, 6), two a byte, the even column in the low nibble, and one scale
2^(byte - 127) per 32 columns.

``w`` is the type of the weights and ``x`` of the rows, bf16 or mxfp4. A batch is
``tokens`` of ``top_k`` experts each, hence tokens * top_k rows, ragged among
``experts`` matrices; ``rows`` says where a grouped row comes from: "token" (a
token's row serves all its experts), "assignment" (a row of its own, in the order
of the assignments) or "grouped" (rows that lie in the order of the experts).
experts = 0 is one matrix for all rows. ``out`` is the type of the result.
"""
import math

import numpy as np
import torch

own = False  # True: run() calls the framework's kernels

BLOCK = 32

# Layer shapes of the package's configurations.
SMALL = dict(hidden=2048, experts=64, inter=768, top_k=8)
LAGUNA = dict(hidden=4096, experts=128, inter=1536, top_k=10)
GLM = dict(hidden=6144, experts=256, inter=2048, top_k=8)


def _up(layer, **more):
    """The gate and up product of a layer: rows are tokens."""
    return dict(op="swiglu", experts=layer["experts"], top_k=layer["top_k"], cols=layer["hidden"],
                width=layer["inter"], rows="token", **more)


def _down(layer, **more):
    """The down product: rows are assignments."""
    return dict(op="matmul", experts=layer["experts"], top_k=layer["top_k"], cols=layer["inter"],
                width=layer["hidden"], rows="assignment", **more)


def listed():
    return [
        # one decode token, with what its codes stand for: pure latency
        dict(name="quantize_t1", op="quantize", tokens=1, cols=2048, x="f32", values=True),
        # the rows of a large prompt chunk: bandwidth
        dict(name="quantize_t8192", op="quantize", tokens=8192, cols=6144, x="bf16", values=False),
        # gate and up of one decode token, the smallest layer in bf16
        dict(_up(SMALL, w="bf16", x="bf16", out="bf16"), name="swiglu_bf16_t1", tokens=1),
        # a shared expert in 4 bits, one decode token
        dict(name="swiglu_shared_t1", op="swiglu", experts=0, top_k=1, cols=4096, width=1536,
             rows="token", w="mxfp4", x="bf16", out="bf16", tokens=1),
        # down of one decode token, the largest layer in 4 bits
        dict(_down(GLM, w="mxfp4", x="bf16", out="f32"), name="matmul_t1", tokens=1),
        # sizes off every tile, few rows of many experts, rows in the experts' order
        dict(name="matmul_odd_t211", op="matmul", experts=37, top_k=1, cols=2848, width=1285,
             rows="grouped", w="mxfp4", x="bf16", out="bf16", tokens=211),
        # batched decode of the smallest layer, all in 4 bits
        dict(_up(SMALL, w="mxfp4", x="mxfp4", out="bf16"), name="swiglu_fp4_t16", tokens=16),
        # a full decode batch in bf16: the bytes of all experts
        dict(_up(LAGUNA, w="bf16", x="bf16", out="bf16"), name="swiglu_bf16_t64", tokens=64),
        # a prompt chunk of the largest layer, all in 4 bits: 16 rows an expert
        dict(_up(GLM, w="mxfp4", x="mxfp4", out="bf16"), name="swiglu_fp4_t512", tokens=512),
        # down of a prompt chunk in bf16: bytes and matrix cores
        dict(_down(LAGUNA, w="bf16", x="bf16", out="f32"), name="matmul_bf16_t2048", tokens=2048),
        # down of a large prompt chunk, all in 4 bits
        dict(_down(GLM, w="mxfp4", x="mxfp4", out="f32"), name="matmul_fp4_t4096", tokens=4096),
        # gate and up of a large prompt chunk, 4-bit weights: the matrix cores
        dict(_up(LAGUNA, w="mxfp4", x="bf16", out="bf16"), name="swiglu_t4096", tokens=4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most_bytes = max(work(c)["bytes"] for c in listed())
    most_flops = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(["quantize", "matmul", "matmul", "swiglu", "swiglu"])
        if op == "quantize":
            c = dict(op=op, tokens=_log_int(rng, 1, 16384), cols=BLOCK * rng.randint(1, 256),
                     x=rng.choice(["f32", "bf16"]), values=rng.random() < 0.5)
        else:
            w = rng.choice(["bf16", "mxfp4"])
            x = rng.choice(["bf16", "mxfp4"]) if w == "mxfp4" else "bf16"
            if rng.random() < 0.4:
                layer = rng.choice([SMALL, LAGUNA, GLM])
                c = _up(layer) if op == "swiglu" else _down(layer)
            else:
                step = 8 if w == "bf16" else BLOCK
                experts = rng.choice([0, rng.randint(2, 256), rng.randint(2, 256)])
                c = dict(op=op, experts=experts, cols=step * rng.randint(256 // step, 6144 // step),
                         top_k=rng.randint(1, min(12, experts)) if experts else 1,
                         width=rng.randint(64, 6144),
                         rows=rng.choice(["token", "assignment", "grouped"]))
            c = dict(c, tokens=_log_int(rng, 1, 8192), w=w, x=x, out=rng.choice(["f32", "bf16"]))
        got = work(c)
        if got["flops"] <= most_flops and got["bytes"] <= most_bytes and \
                (op == "quantize" or max(c["experts"], 1) * c["cols"] * c["width"] <= 256 * 6144 * 2048):
            return c


# ------------------------------------------------------------------ inputs

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _activations(g, tokens, width):
    """Normal values with a few channels of outliers, as a residual stream has."""
    x = _normal(g, tokens, width)
    loud = torch.randint(0, width, (max(1, width // 256),), generator=g, device="cuda")
    x[:, loud] *= 8.0
    return x


def _code_pairs():
    """Bytes of two codes, as often among 65536 as quantised normal values have them."""
    share = np.array([0.078, 0.152, 0.141, 0.124, 0.192, 0.169, 0.103, 0.041])
    edge = np.round(np.cumsum(share / share.sum()) * 128).astype(int)
    one = np.searchsorted(edge, np.arange(128), side="right")
    one = np.concatenate([one, one + 8])
    return torch.from_numpy((one[:, None] * 16 + one[None, :]).reshape(-1).astype(np.uint8)).cuda()


def _matrix(g, c):
    """The weights of one matrix, or of one per expert: a bf16 tensor, or codes and scales."""
    shape = ((c["experts"],) if c["experts"] else ()) + (c["width"],)
    if c["w"] == "bf16":
        w = torch.empty(*shape, c["cols"], dtype=torch.bfloat16, device="cuda")
        return (w.normal_(0.0, 0.02, generator=g),)
    pick = torch.randint(0, 65536, (*shape, c["cols"] // 2), generator=g, device="cuda",
                         dtype=torch.int32)
    codes = torch.index_select(_code_pairs(), 0, pick.view(-1)).view(pick.shape)
    scales = torch.randint(119, 122, (*shape, c["cols"] // BLOCK), generator=g, device="cuda",
                           dtype=torch.uint8)
    return codes, scales


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    T = c["tokens"]
    s = {"case": c}
    if c["op"] == "quantize":
        s["x"] = _activations(g, T, c["cols"]).to(DTYPE[c["x"]])
        return s
    names = ("w",) if c["op"] == "matmul" else ("gate", "up")
    for n in names:
        s[n] = _matrix(g, c)
    E, k = c["experts"], c["top_k"]
    x = _activations(g, T if c["rows"] == "token" else T * k, c["cols"])
    s["x"] = _quantize(x) if c["x"] == "mxfp4" else (x.to(torch.bfloat16),)
    s["offsets"], s["sorted"], s["most"] = None, None, T * k
    if E:
        score = _normal(g, T, E) + _normal(g, E, std=0.3)
        ids = score.topk(k, dim=1).indices.reshape(-1)
        count = torch.bincount(ids, minlength=E)
        s["offsets"] = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        s["offsets"][1:] = count.cumsum(0)
        s["most"] = int(count.max())  # rows of the largest expert, for the plain form's padding
        if c["rows"] != "grouped":
            s["sorted"] = ids.argsort(stable=True).to(torch.int32)
    return s


# --------------------------------------------------------------------- run

def _power_of_two(byte):
    """2^(byte - 127) of bytes from 1 to 254."""
    return (byte.int() << 23).view(torch.float32)


def _quantize(x):
    """Codes and scales of rows in MXFP4."""
    v = x.float().unflatten(-1, (-1, BLOCK))
    largest = v.abs().amax(-1, keepdim=True)
    power = torch.where(largest > 0, torch.frexp(largest).exponent - 3, -127).clamp(-127, 126)
    m = v.abs() * _power_of_two(127 - power)
    # halfway values go to the code whose last bit is 0
    code = (m > 0.25).byte() + (m >= 0.75).byte() + (m > 1.25).byte() + (m >= 1.75).byte() + \
        (m > 2.5).byte() + (m >= 3.5).byte() + (m > 5.0).byte()
    code = (code + 8 * torch.signbit(v).byte()).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], (power.squeeze(-1) + 127).to(torch.uint8)


def _values(t):
    """What a bf16 tensor, or codes and scales, stand for, in 32 bits."""
    if len(t) == 1:
        return t[0].float()
    codes, scales = t
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    e, m = (q >> 1) & 3, q & 1
    halves = torch.where(e == 0, m, ((2 + m) << e) >> 1)
    v = torch.where(q >= 8, -0.5, 0.5).mul_(halves).unflatten(-1, (-1, BLOCK))
    return v.mul_(_power_of_two(scales).unsqueeze(-1)).flatten(-2)


def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _plain(s, c):
    if c["op"] == "quantize":
        codes, scales = _quantize(s["x"])
        out = {"codes": codes, "scales": scales}
        if c["values"]:
            out["values"] = _values((codes, scales)).to(s["x"].dtype)
        return out
    names = ("w",) if c["op"] == "matmul" else ("gate", "up")
    x, E, A = _values(s["x"]), c["experts"], c["tokens"] * c["top_k"]
    if not E:
        y = [x @ _values(s[n]).T for n in names]
        return (y[0] if len(y) == 1 else _silu(y[0]) * y[1]).to(DTYPE[c["out"]])
    at = torch.arange(A, device=x.device) if s["sorted"] is None else s["sorted"].long()
    offsets = s["offsets"].long()
    place = torch.arange(A, device=x.device)
    expert = torch.searchsorted(offsets, place, right=True) - 1
    rows = x[at // c["top_k"] if c["rows"] == "token" else at]
    if A <= E:  # the selected experts' matrices alone
        y = [torch.bmm(_values(tuple(v[expert] for v in s[n])), rows.unsqueeze(-1)).squeeze(-1)
             for n in names]
    else:  # every expert's rows, as many as the largest has
        slot = place - offsets[expert]
        wide = x.new_zeros(E, s["most"], c["cols"])
        wide[expert, slot] = rows
        y = [torch.bmm(wide, _values(s[n]).transpose(1, 2))[expert, slot] for n in names]
    y = y[0] if len(y) == 1 else _silu(y[0]) * y[1]
    out = torch.empty(A, c["width"], dtype=DTYPE[c["out"]], device=x.device)
    out[at] = y.to(out.dtype)
    return out


def _handles(s):
    """The weights' handles, which a program makes once when it loads them."""
    from inferno_amd import ops
    if "handles" not in s:
        s["handles"] = [ops.Experts(*s[n]) for n in ("w", "gate", "up") if n in s]
    return s["handles"]


def run(state):
    s, c = state, state["case"]
    if not own:
        return _plain(s, c)
    from inferno_amd import ops
    if c["op"] == "quantize":
        got = ops.mxfp4_quantize(s["x"], values=c["values"])
        return dict(zip(("codes", "scales", "values"), got))
    call = ops.grouped_matmul if c["op"] == "matmul" else ops.grouped_gate_up_swiglu
    return call(*_handles(s), *s["x"], offsets=s["offsets"], sorted_=s["sorted"],
                k=c["top_k"] if c["rows"] == "token" else 1, out_dtype=DTYPE[c["out"]])


# -------------------------------------------------------------------- work

def _bytes(kind, rows, cols):
    return rows * cols * 2 if kind == "bf16" else rows * (cols // 2 + cols // BLOCK)


def _experts_used(c):
    """Experts that a batch selects, for scores of the inputs' distribution."""
    if not c["experts"]:
        return 1
    r = np.random.default_rng(7)
    key = r.standard_normal((c["tokens"], c["experts"])) + 0.3 * r.standard_normal(c["experts"])
    return len(np.unique(np.argpartition(-key, c["top_k"] - 1, axis=1)[:, :c["top_k"]]))


def work(case):
    c = case
    T = c["tokens"]
    if c["op"] == "quantize":
        each = (4 if c["x"] == "f32" else 2) * (2 if c["values"] else 1)
        return {"bytes": T * (c["cols"] * each + c["cols"] // 2 + c["cols"] // BLOCK),
                "flops": 4 * T * c["cols"]}
    n = 1 if c["op"] == "matmul" else 2
    A, K, N = T * c["top_k"], c["cols"], c["width"]
    moved = n * _experts_used(c) * _bytes(c["w"], N, K) + A * N * (4 if c["out"] == "f32" else 2)
    moved += _bytes(c["x"], T if c["rows"] == "token" else A, K)
    if c["experts"]:
        moved += 4 * (c["experts"] + 1) + (4 * A if c["rows"] != "grouped" else 0)
    return {"bytes": moved, "flops": 2 * n * A * N * K}


# ------------------------------------------------------------------- exact

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _dense64(t):
    """One matrix's values in 64 bits, from the format's definition."""
    if len(t) == 1:
        return t[0].double()
    codes, scales = t
    table = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device=codes.device)
    w = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    w[:, 0::2] = table[(codes % 16).long()]
    w[:, 1::2] = table[torch.div(codes, 16, rounding_mode="floor").long()]
    return w * torch.exp2(scales.double() - 127.0).repeat_interleave(BLOCK, 1)


def _nearest64(x):
    """Rows' nearest values in MXFP4."""
    v = x.double().view(x.shape[0], -1, BLOCK)
    unit = torch.frexp(v.abs().amax(2, keepdim=True)).exponent.double() - 3.0
    unit = torch.exp2(unit)
    q = v / unit
    # steps of a half below 2, of 1 below 4, of 2 above
    step = torch.where(q.abs() < 2.0, 0.5, torch.where(q.abs() < 4.0, 1.0, 2.0))
    return ((torch.round(q / step) * step).clamp(-6.0, 6.0) * unit).view(x.shape)


def exact(case, seed):
    c = case
    if c["op"] == "quantize" and not c["values"]:
        return None
    s = prepare(case, seed)
    if c["op"] == "quantize":
        return {"codes": None, "scales": None, "values": _nearest64(s["x"])}
    names = ("w",) if c["op"] == "matmul" else ("gate", "up")
    x, k = _dense64(s["x"]), c["top_k"]
    A = c["tokens"] * k
    out = torch.zeros(A, c["width"], dtype=torch.float64, device=x.device)
    at = torch.arange(A, device=x.device) if s["sorted"] is None else s["sorted"].long()
    begin = [0, A] if s["offsets"] is None else s["offsets"].tolist()
    for e in range(len(begin) - 1):
        if begin[e] == begin[e + 1]:
            continue
        to = at[begin[e]:begin[e + 1]]
        rows = x[torch.div(to, k, rounding_mode="floor") if c["rows"] == "token" else to]
        y = [rows @ _dense64(s[n] if s["offsets"] is None else tuple(v[e] for v in s[n])).T
             for n in names]
        out[to] = y[0] if len(y) == 1 else y[0] * torch.sigmoid(y[0]) * y[1]
    return out
