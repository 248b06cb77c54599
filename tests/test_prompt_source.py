"""CPU checks of the prompt path's kernels that no run can show: orders of memory accesses, by reading the source.

An access that a barrier does not order goes wrong once in so many launches that no test would meet it, so what the
order rests on is held here in the source's own words."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "lightdelta_b200" / "csrc"


def without_comments(text):
    return re.sub(r"//[^\n]*", "", text)


def chain_kernel():
    text = without_comments((CSRC / "prefill.cu").read_text())
    start = text.index("gdn_prefill_chain_kernel(const __grid_constant__ PrefillArgs p)")
    return text[start:text.index("gdn_prefill_join_kernel(", start)]


def state_loop():
    """The loop of the threads that carry the state, a chunk a turn."""
    text = chain_kernel()
    text = text[text.index("setmaxnreg.inc"):]
    start = text.index("for (int64_t n = 0;; ++n)")
    depth, at = 0, text.index("{", start)
    for end in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        if depth == 0:
            return text[at:end]
    raise AssertionError("the loop does not end")


def test_the_state_warps_leave_a_stage_before_they_hand_it_back():
    """After the arrival at kBarChunkDone the moving threads may write the stage's next work.  What the store behind it
    uses (the head among it) is copied before, and lambdas, which read when they are called, name only the copy."""
    loop = state_loop()
    before, after = loop.split("bar_arrive(kBarChunkDone)")
    stage_names = r"\bs\.stage\b|\bst\s*\.|\bst\b"
    assert not re.search(stage_names, after), "the stage is read after it was handed back"
    for body in re.findall(r"\[&\]\([^)]*\)\s*\{(.*?)\n?\s*\};", before, re.S):
        assert not re.search(stage_names, body), f"a lambda reads the stage when it is called: {body.strip()}"
    assert len(re.findall(r"s\.stage\[stage\]\.work", before)) == 1 and "const Work work = s.stage[stage].work;" in before


def test_the_state_warps_store_a_state_together_or_not_at_all():
    """A wait may run out while they store, in a warp that they do not wait for.  One warp decides for all, in front of a
    barrier that all pass, so that no slot takes some warps' rows and not the others'."""
    loop = state_loop()
    assert "s.stop" not in loop and "s.keep" in loop.split("bar_arrive(kBarChunkDone)")[1]
    text = without_comments((CSRC / "prefill.cu").read_text())
    wait = text[text.index("void wait_products("):]
    wait = wait[:wait.index("\n}")]
    decided, joined = wait.index("s.keep = s.stop == 0;"), wait.index("bar_state();")
    assert wait.index("if (x.issuer)") < decided < joined
    assert len(re.findall(r"s\.keep\b", text)) == 2, "one place writes it, one reads it"
