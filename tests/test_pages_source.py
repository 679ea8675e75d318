"""Rules of the page attention kernels' sources that no run shows: what
follows an expired wait."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "arkantos-ai-stack-suite_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_tensor_core_kernel_warps_leave_whole():
    """The lanes of a warp can learn of an expired wait at different polls.
    What the roles do next (elect.sync, votes, __syncwarp, tcgen05) asks for
    all 32, so a lane's own outcome never decides a branch: between a wait of
    single lanes and the next use of its outcome stands a vote."""
    text = source("b2_page_tc.cuh")
    text = text[text.index("page_tc_kernel"):]
    body = text[text.index("auto warp_wait"):]
    assert "__all_sync" in body[:body.index("};")]
    # a wait's outcome is only ever kept in ok, or voted on
    waits = re.findall(r"[^;{}]*(?<![_\w])wait\(&[^;]*;", body)
    assert len(waits) >= 5
    for w in waits:
        assert re.match(r"\s*ok = ", w), w
    event = re.compile(r"(?P<set>(?<![=!\w])ok = [^;]*;)|(?P<use>if \(!ok\)|while \(ok\b|for \([^;]*;[^;]*\bok\b[^;]*;)"
                       r"|(?P<end>auto \w+ = \[&\]|else if \(warp|tc_commit\(done\))")
    voted, seen = True, 0
    for m in event.finditer(body):
        if m["set"]:
            voted = "warp_wait(" in m["set"] or "__all_sync" in m["set"] or m["set"].endswith("= true;")
        else:
            assert voted, body[max(0, m.start() - 300):m.end()]
            seen += 1
    assert seen >= 15


def test_tensor_core_kernel_counts_only_copies_it_issued():
    """A copy that was given up on is not waited for at the end."""
    text = source("b2_page_tc.cuh")
    for m in re.finditer(r"\+\+fills\[i\];", text):
        before = text[:m.start()].rstrip()
        assert before.endswith("if (!ok) break;")
