"""Bounded waits of the 4-bit decode kernel, by its source: no GPU can be made to time out here on purpose.

A warp whose lanes disagree about a wait would go on to shuffles and matrix products of all 32 lanes without
some of them, which need not end. So a wait's result is used only after the warp has voted on it.
"""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "saga_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_a_warp_votes_on_the_result_of_a_wait():
    text = source("kv4_decode.cu")
    used = [m.start() for m in re.finditer(r"mbar_wait\(", text)
            if not re.search(r"[;{}]\s*$", text[:m.start()])]     # not a statement of its own
    assert used, "the kernel waits for its copies"
    for at in used:
        assert re.search(r"__all_sync\(0xffffffffu,\s*$", text[:at]), text[at - 80:at + 60]


def test_a_warp_without_tiles_leaves_no_stale_numbers_to_the_merge():
    """The merge reads the numerators of the warps below `busy`, so each of those writes them, also one that gave
    up a wait before and has none."""
    text = source("kv4_decode.cu")
    assert text.index("const int busy =") < text.index("float* so =")
    assert re.search(r"if \(warp < busy\) \{", text)
    assert not re.search(r"if \(mine > 0\)", text)
