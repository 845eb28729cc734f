"""How good the rule between the forms of a product grouped by expert is, and the fit of
its costs (plan_product in inferno_amd/csrc/experts_rows.hip).

    python perf/experts_forms.py time --draw 200 --seed 1 --few 60 > FILE
    python perf/experts_forms.py loss FILE [FILE ...]
    python perf/experts_forms.py fit FILE [FILE ...]

``time`` times products in every form that takes them and as the rule has them: products
drawn as in perf/more_operators.py, and --few of each type of one matrix or few experts
by up to 1024 tokens, half of them of long columns. A line each: the case, and the
microseconds of a call, the least of six rows of eight calls over copies of the
weights. ``loss`` says how much slower than the best form the rule's was. ``fit``
changes the costs in the source by random steps, keeps what lessens the mean of
log(loss) + max(0, loss - 1.08), and prints what it ends with, in units of a tenth of a
stage of a tile of 64 by 128; its model of the costs is plan_product's.
"""
import argparse
import json
import math
import os
import random
import re
import sys
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))

TYPES = [("bf16", "bf16"), ("mxfp4", "bf16"), ("mxfp4", "mxfp4")]  # of weights and rows
TILES = [[(4, 128), (2, 128), (2, 64), (2, 32)], [(4, 64), (2, 64), (2, 32)],
         [(4, 128), (2, 128), (2, 64), (2, 32)]]
ROWS = ["r%d/%d" % (width, shares) for width in (1, 2) for shares in (1, 2, 4)]


def forms(types):
    """Names of the forms of a pair of types, tiles first."""
    tiles = ["t%d-%d/%d" % (w, h, s) for w, h in TILES[types] for s in (1, 2, 4, 8)
             if s == 1 or (w == 2 and types < 2)]
    return tiles + ROWS


def types_of(c):
    return TYPES.index((c["w"], c["x"]))


# -------------------------------------------------------------------- timing

def _products(a):
    import perf.more_operators as M
    r, out = random.Random(a.seed), []
    while len(out) < a.draw:
        c = M.draw(r)
        if c["op"] != "quantize":
            out.append(dict(c, out="bf16"))
    for w, x in TYPES:
        for i in range(a.few):
            E = r.choice([0, 0, 4, 8, 16, 32, 64, 128])
            cols = 32 * int(2 ** (r.uniform(7, 8.6) if i % 2 else r.uniform(4, 7.6)))
            out.append(dict(op=r.choice(["matmul", "swiglu"]), experts=E, cols=cols,
                            top_k=r.choice([1, 2, 4]) if E else 1, width=int(2 ** r.uniform(8, 12)),
                            rows="token", w=w, x=x, out="bf16", tokens=int(2 ** r.uniform(0, 10))))
    return out


def _time(states, run):
    import torch
    a, b = torch.cuda.Event(True), torch.cuda.Event(True)
    a.record()
    for i in range(8):
        run(states[i % len(states)])
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / 8 * 1e3


def time_forms(a):
    import torch
    import perf.more_operators as M
    from inferno_amd import InfernoError
    M.own = True
    for c in _products(a):
        work = M.work(c)
        copies = max(1, min(4, int(4e8 / work["bytes"])))  # (more than the caches hold)
        states = [M.prepare(c, 100 + i) for i in range(copies)]
        per_expert = c["tokens"] * c["top_k"] / max(1, c["experts"])
        best = {}
        for _ in range(6):
            for f in ["rule"] + [f for f in forms(types_of(c)) if f[0] == "t" or per_expert <= 150]:
                os.environ.pop("INFERNO_EXPERTS_FORM", None)
                if f != "rule":
                    os.environ["INFERNO_EXPERTS_FORM"] = f
                try:
                    if f not in best:
                        for s in states:
                            M.run(s)
                    best[f] = min(best.get(f, 1e9), _time(states, M.run))
                except InfernoError:  # a form that such columns do not have
                    continue
        os.environ.pop("INFERNO_EXPERTS_FORM", None)
        print(json.dumps({"case": c, "work": work, "us": {f: round(t, 2) for f, t in best.items()}}),
              flush=True)
        del states
        torch.cuda.empty_cache()


def read(files):
    return [json.loads(line) for f in files for line in open(f) if line.startswith("{")]


# ---------------------------------------------------------------------- loss

def loss(a):
    got = read(a.files)
    for t, pair in enumerate(TYPES):
        rows = [d for d in got if types_of(d["case"]) == t]
        if not rows:
            continue
        lost = [d["us"]["rule"] / min(d["us"].values()) for d in rows]
        print("%s by %s: %d products, %.1f%% slower than the best form on the mean, %.0f%% at the "
              "95th percentile" % (*pair, len(rows), 100 * (np.exp(np.log(lost).mean()) - 1),
                                   100 * (np.quantile(lost, 0.95) - 1)))
        for i in np.argsort(lost)[::-1][:4]:
            us = rows[i]["us"]
            best = min(us, key=us.get)
            print("   %.2f: %.1f, by %s %.1f: %s" % (lost[i], us["rule"], best, us[best], rows[i]["case"]))
        rate = 1.35e15 * (4 if t == 2 else 1)
        for name, by_ops in (("operations", True), ("bytes", False)):
            over = []
            for d in rows:
                floor = [d["work"]["flops"] / rate * 1e6, d["work"]["bytes"] / 4.94e12 * 1e6]
                if max(floor) > 15 and (floor[0] > floor[1]) == by_ops:
                    over.append(d["us"]["rule"] / (max(floor) + 6.2))
            if over:
                print("   floor of more than 15 us by %s: %d, %.2f times floor and launch on the mean, %.2f "
                      "at most" % (name, len(over), np.exp(np.log(over).mean()), max(over)))


# ----------------------------------------------------------------------- fit

def constants():
    """The costs of the source: per pair of types {name: value}."""
    text = (ROOT / "inferno_amd/csrc/experts_rows.hip").read_text()

    def numbers(name):
        body = re.search(r"\b%s(?:\[\d*\])+ = (.*?);" % name, text, re.S).group(1)
        return [float(v) for v in re.findall(r"-?\d+\.?\d*(?:e-?\d+)?", body)]

    tile, rows, start = numbers("kTileCosts"), numbers("kRowsCosts"), numbers("kRowsStart")
    join = re.search(r"kJoin\[2\] = \{(.*?)\}, kJoinValue\[2\] = \{(.*?)\};", text)
    join, value = ([float(v) for v in join.group(i).split(",")] for i in (1, 2))
    out = []
    for t in range(3):
        P = {"start": start[t], "join": join[min(t, 1)], "value": value[min(t, 1)]}
        for w, h in TILES[t]:
            at = [i for i in range(0, len(tile), 5)
                  if tile[i: i + 2] == [w, h] and i >= 5 * (0, len(TILES[0]), 7)[t]][0]
            P.update({"%s%d-%d" % (n, w, h): v for n, v in zip(("first", "stage", "tile"),
                                                               tile[at + 2: at + 5])})
        for width in (1, 2):
            at = 6 * t + 3 * (width - 1)
            P.update({"%s%d" % (n, width): v for n, v in zip(("chunk", "turn_chunk", "turn"),
                                                             rows[at: at + 3])})
        out.append(P)
    return out


def rows_of_one(c):
    """Rows of an expert that has any, and how many have, by chance."""
    A, E = c["tokens"] * c["top_k"], c["experts"]
    used = E * (1 - (1 - 1 / E) ** A) if E else 1.0
    return A / used, used


def cost(P, t, c, form):
    A, E, K = c["tokens"] * c["top_k"], c["experts"], c["cols"]
    N = c["width"] * (2 if c["op"] == "swiglu" else 1)
    rows, used = rows_of_one(c)
    if form[0] == "r":
        width, shares = int(form[1]), int(form[3:])
        chunks = math.ceil(K / (128 * shares))
        turns = math.ceil(used * math.ceil(rows / (16 * width)) * math.ceil(N * shares / 128) / 256)
        return P["start"] + P["chunk%d" % width] * chunks + \
            turns * (P["turn_chunk%d" % width] * chunks + P["turn%d" % width])
    key, splits = form[1:].split("/")
    (width, height), splits = map(int, key.split("-")), int(splits)
    part = 0.3 if t == 2 else 0.7
    n = used * max(1.0, rows / height + (part if rows > height / 2 else 0)) if E else math.ceil(A / height)
    n = n * math.ceil(N / (64 * width)) * splits / 256
    turns = max(1.0, n) if E else math.ceil(n)
    mine = math.ceil(math.ceil((K // 2 if t == 2 else 2 * K) / 256) / splits)
    join = P["join"] + P["value"] * splits * A * N if splits > 1 else 0
    return P["first" + key] * mine + turns * (P["stage" + key] * mine + P["tile" + key]) + join


def fit(a):
    got = read(a.files)
    # (groups of up to eight rows an expert go by thresholds, not by costs)
    got = [d for d in got if not d["case"]["experts"] or rows_of_one(d["case"])[0] > 8]
    for t, pair in enumerate(TYPES):
        rows = [d for d in got if types_of(d["case"]) == t]
        if not rows:
            continue

        def score(P):
            lost = []
            for d in rows:
                us = {f: v for f, v in d["us"].items() if f != "rule"}
                lost.append(us[min(us, key=lambda f: cost(P, t, d["case"], f))] / min(us.values()))
            return np.mean(np.log(lost) + np.maximum(0, np.array(lost) - 1.08)), np.mean(np.log(lost))

        P, rng = constants()[t], np.random.default_rng(a.seed)
        best, mean = score(P)
        print("%s by %s: %d products, mean loss %.2f%%" % (*pair, len(rows), 100 * mean), flush=True)
        for step in range(a.steps):
            Q = dict(P)
            for k in rng.choice(sorted(Q), rng.integers(1, 4), replace=False):
                Q[k] = Q[k] + rng.normal(0, 8) if k == "start" else \
                    Q[k] * math.exp(rng.normal(0, 0.25 if step < a.steps // 2 else 0.1))
            s, m = score(Q)
            if s < best:
                best, mean, P = s, m, Q
        unit = P["stage2-64"] / 10
        print("   then %.2f%%: %s" % (100 * mean, {k: float("%.2g" % (v / unit)) for k, v in P.items()}),
              flush=True)


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("do", choices=("time", "loss", "fit"))
    p.add_argument("files", nargs="*")
    p.add_argument("--draw", type=int, default=200)
    p.add_argument("--few", type=int, default=60)
    p.add_argument("--seed", type=int, default=1)
    p.add_argument("--steps", type=int, default=4000)
    a = p.parse_args()
    {"time": time_forms, "loss": loss, "fit": fit}[a.do](a)


if __name__ == "__main__":
    main()
