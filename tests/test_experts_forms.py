"""The model of perf/experts_forms.py against the rule in the library: the shares of the
columns that either takes, which the library's workspace tells."""
import math
import random
import sys
from pathlib import Path

import pytest

from inferno_amd import BF16, MXFP4, ExpertsDesc, lib

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import perf.experts_forms as F  # noqa: E402


def _model(c, t):
    stages = math.ceil((c["cols"] // 2 if t == 2 else 2 * c["cols"]) / 256)
    P = F.constants()[t]
    fit = [f for f in F.forms(t) if f[0] == "r" or f.endswith("/1") or
           12 * int(f.split("/")[1]) <= stages]
    return min(fit, key=lambda f: F.cost(P, t, c, f))


@pytest.mark.parametrize("t", range(3))
def test_same_shares_of_the_columns(t):
    w, x = F.TYPES[t]
    r, taken = random.Random(t), set()
    for _ in range(1500):
        E = r.choice([0, 0, 2, 8, 32])
        c = dict(op=r.choice(["matmul", "swiglu"]), experts=E, cols=32 * int(2 ** r.uniform(3, 9.5)),
                 top_k=r.choice([1, 2]) if E else 1, width=int(2 ** r.uniform(4, 12)),
                 tokens=int(2 ** r.uniform(0, 11)), w=w, x=x)
        if E and F.rows_of_one(c)[0] <= 8:
            continue
        A, N, mats = c["tokens"] * c["top_k"], c["width"], 2 if c["op"] == "swiglu" else 1
        d = ExpertsDesc(max(E, 1), N, c["cols"], MXFP4 if w == "mxfp4" else BF16, None, 0)
        got = lib().inferno_grouped_workspace_bytes(d, mats, MXFP4 if x == "mxfp4" else BF16, c["tokens"],
                                                    c["top_k"], int(E > 0))
        assert lib().inferno_last_error() == b""
        form = _model(c, t)
        shares = int(form.split("/")[1]) if form[0] == "t" else 1
        assert got == (shares * mats * A * ((N + 3) // 4 * 4) * 4 if shares > 1 else 0), (c, form)
        taken.add(shares)
    assert taken == ({1} if t == 2 else {1, 2, 4, 8})
