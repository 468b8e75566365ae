"""Kernels whose blocks write into one another's shared memory: by their source, no such write comes before a barrier of the cluster.  (A block that
does not run yet has no shared memory to write to; a run does not show it, since blocks of a cluster mostly begin together.)"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-serve_b200", "csrc")


def closing(text, at):
    """The place behind the bracket that closes the one at `at`."""
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return i + 1
    raise AssertionError("no closing bracket")


def body_of(source, kernel):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, source)).read())
    at = re.search(r"\b%s\([^;{]*\{" % kernel, text)
    return text[at.end() - 1:closing(text, at.end() - 1)]


def lambdas_of(body):
    """(the body without its lambdas' bodies, {name: body})."""
    found, out, at = {}, "", 0
    for m in re.finditer(r"\bauto (\w+) = \[&?\][^{;]*\{", body):
        if m.start() < at:
            continue
        end = closing(body, m.end() - 1)
        found[m.group(1)] = body[m.end():end]
        out += body[at:m.start()]
        at = end
    return out + body[at:], found


@pytest.mark.parametrize("source,kernel,remote", [("sample.cu", "sample_kernel", ["put64", "put32", "get32", "add32"])])
def test_no_remote_access_before_the_blocks_have_met(source, kernel, remote):
    body, lambdas = lambdas_of(body_of(source, kernel))
    reach = set(remote)
    while True:                                     # lambdas that reach another block, by themselves or through others
        more = {n for n, b in lambdas.items() if n not in reach and any(re.search(r"\b%s\(" % r, b) for r in reach)}
        if not more:
            break
        reach |= more
    first = min(m.start() for r in reach for m in re.finditer(r"\b%s\(" % r, body))
    arrive, wait = [body.find(f"{n}();") for n in ("cluster_arrive", "cluster_wait")]
    assert 0 <= arrive < wait < first, (arrive, wait, first)
    assert body.count("cluster_arrive();") == body.count("cluster_wait();") == 1
    between = body[arrive:wait]
    assert "return" not in between and "cluster_sync_all" not in between
    # neither stands in a branch, of the kernel or of a block of its own that is one
    for at in (arrive, wait):
        openings = []
        for i, ch in enumerate(body[:at]):
            if ch == "{":
                openings.append(i)
            elif ch == "}":
                openings.pop()
        assert all(re.search(r"(^|[;}])\s*$", body[:i]) for i in openings), "in a branch"
