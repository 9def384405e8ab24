"""The token ops without a GPU: what their sources promise, refusals before any launch, fake forms, the C checks."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "smal-memory-llm_b200", "csrc")


def _loops(text):
    """Bodies of the `for (...) {` loops of a source without comments, inner ones among them."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"\bfor \(", text):
        depth, i = 1, m.end()
        while depth:                                                   # the loop's head
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        while text[i].isspace():
            i += 1
        if text[i] != "{":
            continue
        depth, at = 1, i + 1
        i += 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        yield text[at:i - 1]


def test_no_thread_leaves_a_loop_that_holds_a_barrier():
    """A thread whose bounded wait gave up and left such a loop would be waited for at the barrier without a limit."""
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "slotscan_attn*.cu"))):
        for body in _loops(open(path).read()):
            if "sync_group(" in body or "__syncthreads()" in body:
                found += 1
                assert "break;" not in body, (os.path.basename(path), body[:200])
    assert found >= 4
