"""Shared memory of another CTA may be reached only once that CTA runs: a kernel whose CTAs write or read each other's meets at a
barrier of its cluster first.  A missing one shows as a lost partial sum now and then, or not at all on an idle
device, so the order is checked where it stands: in the sources."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "approxtrain_b200", "csrc")


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    return re.sub(r"//[^\n]*", "", text)


def _body(text, at):
    """The braces that open behind `at`."""
    begin = text.index("{", at)
    depth = 0
    for i in range(begin, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[begin:i + 1]
    raise AssertionError("unbalanced braces")


def _functions(text):
    """name -> body of what is defined at the file's or a class's level."""
    out = {}
    for m in re.finditer(r"\b(\w+|operator\(\))\s*\(([^;{}]*)\)\s*(?:const\s*)?\{", text):
        if m.group(1) not in ("if", "for", "while", "switch"):
            out.setdefault(m.group(1), _body(text, m.end() - 1))
    return out


@pytest.mark.parametrize("file", sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))))
def test_clusters_meet_before_they_reach_each_other(file):
    text = _code(file)
    functions = _functions(text)
    mapped = {n for n, b in functions.items() if "mapa." in b}
    waits = {n for n, b in functions.items() if "barrier.cluster.wait" in b and "mapa." not in b}
    kernels = [(m.group(1), _body(text, m.end())) for m in re.finditer(r"__global__[^;{]*?\b(\w+)\(const __grid_constant__", text)]
    # functions of the file that reach another CTA, directly or through others
    reach = set(mapped)
    grown = True
    while grown:
        more = {n for n, b in functions.items() if n not in reach and any(re.search(rf"\b{re.escape(r)}\(", b) for r in reach if r != "operator()")}
        grown = bool(more)
        reach |= more
    if "operator()" in reach:       # RowSum's, called by the name of the object
        reach |= {"sum"} | {n for n, b in functions.items() if re.search(r"\bsum\(", b) and n not in dict(kernels)}
    for name, body in kernels:
        used = [m.start() for r in reach - {name, "operator()"} for m in re.finditer(rf"\b{re.escape(r)}\b\s*[(<]", body)]
        if not used:
            continue
        met = [m.start() for n in waits for m in re.finditer(rf"\b{re.escape(n)}\(", body)]
        assert met and min(met) < min(used), f"{file}: {name} reaches another CTA's shared memory before its cluster has met"
