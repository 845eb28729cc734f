"""Workspace of the products grouped by expert: what a product would refuse has none, and
an error says why."""
import pytest

from inferno_amd import BF16, F32, I8, MXFP4, ExpertsDesc, lib


def _bytes(fmt=BF16, E=1, N=40, K=12832, mats=1, dt=BF16, rows=5, k=1, grouped=0):
    return lib().inferno_grouped_workspace_bytes(ExpertsDesc(E, N, K, fmt, None, 0), mats, dt, rows, k,
                                                 grouped)


@pytest.mark.parametrize("bad,match", [
    (dict(mats=0), "matrices"), (dict(mats=3), "matrices"), (dict(mats=-1), "matrices"),
    (dict(dt=F32), "dtype"), (dict(dt=I8), "dtype"), (dict(dt=7), "dtype"), (dict(dt=MXFP4), "dtype"),
    (dict(fmt=F32), "format"), (dict(K=12836), "multiple of 8"), (dict(N=0), "sizes"),
    (dict(rows=(1 << 22) + 1), "rows"), (dict(rows=1 << 20, k=8), "rows"), (dict(rows=1 << 40), "rows"),
    (dict(k=1 << 62, rows=8), "rows")])
def test_refused(monkeypatch, bad, match):
    monkeypatch.setenv("INFERNO_EXPERTS_TILES", "1")
    assert _bytes() > 0 and lib().inferno_last_error() == b""
    assert _bytes(**bad) == 0 and match in lib().inferno_last_error().decode()


def test_none_needed():
    for kw in (dict(rows=0), dict(k=0), dict(K=64), dict(fmt=MXFP4, dt=MXFP4, mats=2)):
        assert _bytes(**kw) == 0 and lib().inferno_last_error() == b"", kw
