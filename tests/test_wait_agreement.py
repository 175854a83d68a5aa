"""A wait that gives up in the large tree-attention kernel must not leave another warp at a
barrier that has no limit. The two warps of a row quadrant (one for each half of a block's columns)
meet at a named barrier once in every job: a warp that leaves the loop over jobs early comes to it for
all the jobs that it has not met the other one in. Read from the source; no GPU."""
import os
import re

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voltattn_b200", "csrc", "decode_tree_tc.cuh")


def block(text, at):
    """The braces' block that begins at or after `at`, and where it ends."""
    at = text.index("{", at)
    depth, end = 0, at
    while True:
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        if depth == 0:
            return text[at:end + 1], end + 1
        end += 1


def test_softmax_warps_meet_in_every_job():
    with open(SRC) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    head = "for (int j = w; j < njobs; j += 2)"
    start = text.index(head)
    loop, _ = block(text, start)
    barrier = "named_barrier_sync(2 + w * 4 + quad, 64);"
    assert loop.count("named_barrier") == loop.count(barrier) == 1 and "return" not in loop
    met = loop.index(barrier)
    breaks = [m.start() for m in re.finditer(r"\bbreak\b", loop)]
    assert breaks
    for at in breaks:
        # the job's barrier is still to come before it, and done after it; no lane leaves alone
        call = "give_up(%s);" % ("j" if at < met else "j + 2")
        assert re.search(r"if \(__any_sync\(0xffffffffu, !ok\)\) \{\s*" + re.escape(call) + r"\s*$", loop[:at]), loop[:at][-200:]
    body, _ = block(text, text.index("const auto give_up", text.index("const int w = set;")))
    assert re.search(r"if \(live_quad\)\s*for \(int k = from; k < njobs; k \+= 2\) " + re.escape(barrier), body)
    assert "if (live_quad) {" in loop[:met]  # who meets is who comes in give_up
