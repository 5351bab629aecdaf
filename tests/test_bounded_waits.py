"""Bounded waits of the shared-prefix kernels, by reading their source: where a
whole warp waits, every lane has a clock of its own, and lanes that give up
while others go on would meet different full-warp operations.  So the lanes
vote on the outcome before any of them acts on it.  (Nothing on the GPU can
show this without a wait that runs out at just the wrong moment.)"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-diy_b200", "csrc")
VOTE = "__all_sync(0xffffffffu"


@pytest.mark.parametrize("name", ["own_keys.cuh", "shared_prefix.cuh"])
def test_lanes_vote_before_they_act_on_a_wait(name):
    with open(os.path.join(CSRC, name)) as f:
        lines = [line.split("//")[0].strip() for line in f]
    lines = [line for line in lines if line]
    # waits of its own name: lambdas around mbar_wait, `voting` if the vote is in them
    voting, plain = set(), {"mbar_wait"}
    for i, line in enumerate(lines):
        m = re.match(r"auto (\w+) = \[&\]\(.*?\) \{", line)
        if m:
            end = i + next(k for k, x in enumerate(lines[i:]) if x.endswith("};"))
            body = " ".join(lines[i:end + 1])
            if "mbar_wait(" in body:
                (voting if VOTE in body else plain).add(m[1])
    waits = re.compile(r"\bok = (?:.*\W)?(" + "|".join(plain | voting) + r")\(")
    seen = 0
    for line, after in zip(lines, lines[1:]):
        m = waits.search(line)
        if m and m[1] in plain:
            assert VOTE in line or VOTE in after, line
        seen += bool(m)
    assert seen >= 2
