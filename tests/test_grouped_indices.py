"""Products grouped by expert with indices and offsets that no dispatch gives, in every
form: rows that the call does define are written as ever, and nothing behind the last."""
import pytest
import torch

import experts_reference as ref
from inferno_amd import ops
from test_grouped_forms import FORMS, LONG, TYPES

F32 = torch.float32
N, E = 53, 3


def _case(types, form, A):
    w4, x4 = TYPES[types]
    shares = form.split("/")[1] if form[0] == "t" else "1"
    K = LONG.get(shares, 224)
    g = torch.Generator().manual_seed(A + K)
    m = ref.Mats(g, N, K, E, w4)
    x, xv = ref.rows(g, A, K, x4)
    return m, x, xv, torch.randperm(A, generator=g).to(torch.int32)


def _run(m, x, A, offsets, order):
    room = torch.full((A + 64, N), 7.0, device="cuda")
    ops.grouped_matmul(ops.Experts(*m.parts), *x, offsets=offsets.cuda(), sorted_=order.cuda(),
                       out=room[:A])
    assert (room[A:] == 7.0).all()
    return room[:A].cpu().double()


def _near(got, m, xv, e, a):
    """Where got, of rows a, is expert e's result."""
    y, d = ref.product(m, xv, e, a)
    return (got - y).abs() <= d + 2.0 ** -24 * y.abs()


@pytest.mark.gpu
@pytest.mark.parametrize("types,form", FORMS)
def test_an_index_twice_and_indices_out_of_range(cuda, monkeypatch, types, form):
    monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
    A = 190
    m, x, xv, order = _case(types, form, A)
    begin = [0, 20, 150, 190]
    order[160], order[170] = order[3], order[40]  # of two experts each
    order[[0, 33, 34, 149, 189]] = torch.tensor([A, A + 1, -1, 2 ** 31 - 1, -2 ** 31],
                                                dtype=torch.int32)
    got = _run(m, x, A, torch.tensor(begin, dtype=torch.int32), order)
    times = torch.zeros(A, dtype=torch.long)
    fine = torch.zeros(A, N, dtype=torch.bool)
    for e in range(E):
        a = order[begin[e]:begin[e + 1]].long()
        a = a[(a >= 0) & (a < A)]
        times[a] += 1
        fine[a] |= _near(got[a], m, xv, e, a)
    assert (times == 2).sum() == 2 and (times == 0).sum() == 7
    assert fine[times > 0].all() and (got[times == 0] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("A", [40, 900])
@pytest.mark.parametrize("types,form", FORMS)
def test_offsets_that_run_back_or_behind_the_last_row(cuda, monkeypatch, types, form, A):
    """Nothing is read or written out of range. Where ranges overlap a launch may have too
    few workgroups, and what they do not reach is left as it was. (Where workgroups share
    the columns, their sums may meet in rows of two experts or be of nothing, and rows
    before the first offset get no result.)"""
    split = form[0] == "t" and not form.endswith("/1")
    monkeypatch.setenv("INFERNO_EXPERTS_FORM", form)
    m, x, xv, order = _case(types, form, A)
    offsets = torch.tensor([A // 2, A // 4, A - 3, 2 ** 31 - 1], dtype=torch.int32)
    got = _run(m, x, A, offsets, order)  # the second and third expert's rows, none left out
    a1, a2 = order[A // 4: A - 3].long(), order[A - 3:].long()
    before = order[:A // 4].long()
    assert (got[before] == 7.0).all()
    if not split:
        assert _near(got[a1], m, xv, 1, a1).all() and _near(got[a2], m, xv, 2, a2).all()
    offsets = torch.tensor([0, A // 2, A // 4, A + 100], dtype=torch.int32)
    got = _run(m, x, A, offsets, order)  # the first and third expert share rows
    if split:
        return
    fine = got == 7.0
    for e, c in ((0, slice(0, A // 2)), (2, slice(A // 4, A))):
        a = order[c].long()
        fine[a] |= _near(got[a], m, xv, e, a)
    assert fine.all() and (got != 7.0).all(1).sum() > A // 2
