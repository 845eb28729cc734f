"""Every form of the products grouped by expert, by name: ragged groups, remainders of
columns and rows, tokens of several experts, values that are not finite; and the forms
that ask for much shared memory, captured before anything else runs.

Run as a program it does the latter: one form after the other, each captured first.
"""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import experts_reference as ref
from inferno_amd import BF16 as ABI_BF16
from inferno_amd import MXFP4, ExpertsDesc, lib, ops

F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"bf16": (False, False), "mxfp4": (True, False), "mxfp4-mxfp4": (True, True)}
ROWS = ["r%d/%d" % (width, shares) for width in (1, 2) for shares in (1, 2, 4)]
SPLIT = {  # tiles, those with shares of the columns among them
    "bf16": ["t4-128/1"] + ["t2-%d/%d" % (h, s) for h in (128, 64, 32) for s in (1, 2, 4, 8)],
    "mxfp4": ["t4-64/1"] + ["t2-%d/%d" % (h, s) for h in (64, 32) for s in (1, 2, 4, 8)],
    "mxfp4-mxfp4": ["t4-128/1", "t2-128/1", "t2-64/1", "t2-32/1"]}
FORMS = [(t, f) for t in TYPES for f in SPLIT[t] + ROWS]
LONG = {"2": 4128, "4": 6432, "8": 12832}  # columns that so many shares need


def _shapes(types, form):
    """(N, K) of one matrix: rows off every tile, columns that end inside a step, a
    stage and a chunk."""
    shares = form.split("/")[1] if form[0] == "t" else "1"
    if shares != "1":
        return [(37, LONG[shares])]
    return {"bf16": [(1, 8), (261, 72), (530, 296)], "mxfp4": [(1, 32), (261, 96), (530, 416)],
            "mxfp4-mxfp4": [(1, 32), (261, 480), (530, 544), (69, 2080)]}[types]


COUNTS = [1, 16, 0, 17, 33, 64, 65, 128, 129, 0, 300, 97]  # rows of each expert


def _call(m, x, **kw):
    w = [ops.Experts(*t.parts) for t in m]
    return (ops.grouped_matmul if len(w) == 1 else ops.grouped_gate_up_swiglu)(*w, *x, **kw)


def _offsets(first, counts):
    return torch.tensor([first] + counts, dtype=torch.int32).cumsum(0).to(torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("types,form", FORMS)
def test_ragged_groups(cuda, monkeypatch, types, form, mats):
    """Two results a token, in any order, into fp32; and rows in the experts' order,
    some before the first group and behind the last, into bf16. All of the groups' rows
    are written, and no others."""
    monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
    w4, x4 = TYPES[types]
    E, A = len(COUNTS), sum(COUNTS)
    for N, K in _shapes(types, form):
        g = torch.Generator().manual_seed(N + K)
        m = [ref.Mats(g, N, K, E, w4) for _ in range(mats)]
        x, xv = ref.rows(g, A // 2, K, x4)
        offsets, order = _offsets(0, COUNTS), torch.randperm(A, generator=g).to(torch.int32)
        got = _call(m, x, offsets=offsets.cuda(), sorted_=order.cuda(), k=2, out_dtype=F32)
        want, bar, hit = ref.expected(m, xv, A, 2, offsets, order, F32)
        assert hit.all()
        ref.near(got, want, bar)
        first, R = 5, A + 12
        x, xv = ref.rows(g, R, K, x4)
        offsets = _offsets(first, COUNTS)
        room = torch.full((R + 32, N), 7.0, dtype=BF16, device="cuda")
        out = room.flatten()[16 * N: (16 + R) * N].view(R, N)  # at a multiple of 16 bytes
        _call(m, x, offsets=offsets.cuda(), out=out)
        want, bar, hit = ref.expected(m, xv, R, 1, offsets, None, BF16)
        assert int(hit.sum()) == A
        want[~hit], bar[~hit] = 7.0, 1e-30
        ref.near(out, want, bar)
        assert (room[:16] == 7.0).all() and (room[16 + R:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("types,form", FORMS)
def test_one_matrix(cuda, monkeypatch, types, form, mats):
    monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
    w4, x4 = TYPES[types]
    for N, K in _shapes(types, form):
        for T in (1, 15, 150):
            g = torch.Generator().manual_seed(T + N + K)
            m = [ref.Mats(g, N, K, 0, w4) for _ in range(mats)]
            x, xv = ref.rows(g, T, K, x4)
            got = _call(m, x, out_dtype=F32)
            want, bar, _ = ref.expected(m, xv, T, 1, None, None, F32)
            ref.near(got, want, bar)


@pytest.mark.gpu
@pytest.mark.parametrize("types,form", FORMS)
def test_not_finite(cuda, monkeypatch, types, form):
    """A row that is not finite changes its own results, a weight row its own column."""
    monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
    w4, x4 = TYPES[types]
    N, K = _shapes(types, form)[-1]
    g = torch.Generator().manual_seed(N)
    m = [ref.Mats(g, N, K, 2, w4)]
    T = 200
    x, _ = ref.rows(g, T, K, x4)
    offsets = torch.tensor([0, 70, T], dtype=torch.int32).cuda()
    clean = _call(m, x, offsets=offsets)
    assert torch.isfinite(clean).all()
    bad = [t.clone() for t in x]
    if x4:
        bad[1][1, K // 32 - 1] = 255
        bad[1][T - 1, 0] = 255
    else:
        bad[0][1, K - 1] = float("nan")
        bad[0][T - 1, 0] = float("inf")
    got = _call(m, bad, offsets=offsets)
    assert torch.isnan(got[1]).all() and not torch.isfinite(got[T - 1]).any()
    assert torch.equal(got[2: T - 1], clean[2: T - 1]) and torch.equal(got[0], clean[0])
    if w4:
        m[0].parts[1][1, N - 1, K // 32 - 1] = 255
    else:
        m[0].parts[0][1, N - 1, K - 1] = float("nan")
    got = _call(m, x, offsets=offsets)
    assert torch.isnan(got[70:, N - 1]).all()
    got[70:, N - 1] = clean[70:, N - 1]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("types", TYPES)
def test_names(monkeypatch, types):
    """Of no form, or of one that other types or longer columns have: refused."""
    L, at = lib(), 1 << 20
    w4, x4 = TYPES[types]
    dt = MXFP4 if x4 else ABI_BF16

    def desc(K):
        d = ExpertsDesc(1, 40, K, MXFP4 if w4 else ABI_BF16, at, 0)
        d.data_bytes = L.inferno_experts_packed_bytes(d)
        return d

    def workspace(d):
        return L.inferno_grouped_workspace_bytes(d, 1, dt, 50, 1, 0)

    for form in SPLIT[types] + ROWS:
        monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
        shares = form.split("/")[1] if form[0] == "t" else "1"
        long = desc(LONG.get(shares, 64))
        assert workspace(long) == (int(shares) * 50 * 40 * 4 if shares != "1" else 0)
        assert L.inferno_last_error() == b""
        if shares != "1":
            assert workspace(desc(LONG[shares] // 2 // 32 * 32)) == 0 and L.inferno_last_error()
    other = {"bf16": "t4-64/1", "mxfp4": "t4-128/1", "mxfp4-mxfp4": "t2-64/2"}[types]
    for form in ("", "x", "t", "t4-128", "t2-32/0", "t2-32/3", "t4-32/1", "t3-64/1", "r1", "r3/1", "r1/8",
                 "r0/1", "t-2-32/1", other):
        monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
        d = desc(12832)
        assert workspace(d) == 0 and b"INFERNO_EXPERTS_FORM" in L.inferno_last_error(), form
        assert L.inferno_grouped_matmul(None, d, at, dt, at if x4 else None, 50, None, None, 1, 0, at, at,
                                        1 << 30) == -1
        assert b"INFERNO_EXPERTS_FORM" in L.inferno_last_error(), form


# ------------------------------------------------- captured before anything else

CAPTURED = [(t, f, mats) for t in TYPES for f in SPLIT[t] if f.startswith(("t4", "t2-128")) and
            f.endswith("/1") for mats in (1, 2)]


def _capture_first():
    for types, form, mats in CAPTURED:
        print(types, form, mats, flush=True)
        os.environ["INFERNO_EXPERTS_FORM"] = form
        w4, x4 = TYPES[types]
        g = torch.Generator().manual_seed(mats)
        N, K, E, A = 261, 544, len(COUNTS), sum(COUNTS)
        m = [ref.Mats(g, N, K, E, w4) for _ in range(mats)]
        w = [ops.Experts(*t.parts) for t in m]
        call = ops.grouped_matmul if mats == 1 else ops.grouped_gate_up_swiglu
        offsets = _offsets(0, COUNTS)
        batches = [ref.rows(g, A, K, x4) for _ in range(3)]
        held, o = [t.clone() for t in batches[0][0]], offsets.cuda()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(*w, *held, offsets=o, out_dtype=F32)
        for x, xv in batches:
            for to, new in zip(held, x):
                to.copy_(new)
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            want, bar, _ = ref.expected(m, xv, A, 1, offsets, None, F32)
            ref.near(y, want, bar)
            assert torch.equal(y, call(*w, *x, offsets=o, out_dtype=F32))


@pytest.mark.gpu
def test_first_used_in_a_graph(cuda):
    """In a process of its own, where nothing else has used these kernels."""
    r = subprocess.run([sys.executable, "-u", __file__], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert sum(line.split(" ")[0] in TYPES for line in r.stdout.splitlines()) == len(CAPTURED)


if __name__ == "__main__":
    _capture_first()
