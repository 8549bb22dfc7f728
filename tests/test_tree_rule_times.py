"""What "attention_tree" loses by the way that tree_rule (launch_rules.hpp) takes, over the times that the rule was fitted to
(profiles/tree_rule_times.csv): a call's way against the fastest of those measured."""
import os

import pytest

from test_launch_rules import ROOT, run_program

TIMES = os.path.join(ROOT, "profiles", "tree_rule_times.csv")


def measured():
    with open(TIMES) as f:
        rows = [line.rstrip("\n").split(",") for line in f if not line.startswith("#")][1:]
    for kind, *sizes, times in rows:
        ways = dict((tuple(map(int, w.split("=")[0].split(":"))), float(w.split("=")[1])) for w in times.split())
        yield kind, tuple(map(int, sizes)), ways


def runs_fit(kind, d):
    """The rows' kernels take the head size (attention_kernels.hpp: runs_fit)."""
    padded = 64 if d <= 64 else 128 if d <= 128 else 256
    run = 4 if kind == "f32" else min(128 // {"f16": 16, "q8": 8, "fp8": 8, "q4": 4}[kind], padded // 4)
    return d % run == 0 and d % (padded // 16) == 0


@pytest.mark.skipif(not os.path.exists(TIMES), reason="no measured times here")
def test_ways_taken(tmp_path):
    calls = list(measured())
    assert len(calls) >= 600
    lines = []
    for kind, (rows, keys, heads, kv, d, window), _ in calls:
        padded = 64 if d <= 64 else 128 if d <= 128 else 256
        lines.append(f"  one(TreeCall{{{rows}, {min(window or keys, keys)}, {heads}, {kv}, {d}, {padded}, {int(kind == 'f32')} != 0, "
                     f"{int(kind in ('q8', 'q4', 'fp8'))} != 0, {int(runs_fit(kind, d))} != 0, true}});")
    out = run_program(tmp_path, "  auto one = [](const TreeCall& c) { const TreeShape s = tree_rule(c, 256, 64, size_t{16} << 20);"
                      " std::printf(\"%zu %zu\\n\", static_cast<size_t>(s.pairs), static_cast<size_t>(s.parts)); };\n" + "\n".join(lines))
    loss = []
    for (_, _, ways), line in zip(calls, out.split("\n")):
        pairs, parts = map(int, line.split())
        at = sorted(p for e, p in ways if e == pairs)
        if not at:
            continue        # (not run in the way taken)
        below, above = max([p for p in at if p <= parts], default=at[0]), min([p for p in at if p >= parts], default=at[-1])
        part = (parts - below) / (above - below) if above > below else 0.0
        loss.append((ways[pairs, below] * (1 - part) + ways[pairs, above] * part) / min(ways.values()))
    loss.sort()
    print(len(loss), sum(loss) / len(loss), loss[len(loss) * 9 // 10], loss[-1])
    assert len(loss) >= 595
    assert sum(loss) / len(loss) <= 1.02 and loss[len(loss) * 9 // 10] <= 1.06 and loss[-1] <= 1.4
