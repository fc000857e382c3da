"""Rules of the paged operators' sources that no run shows reliably."""
import os
import re

import pytest

from test_kernel_sources import CSRC, ELECTING, _blocks, _code


def test_sums_of_a_row_block_are_read_before_the_next_are_written():
    """The math warps of the few-row attention write sums of weights, meet, and read all warps' sums; a block that falls to one CTA meets no more behind that.  So the next segment has
    a barrier in front of its own sums whether it has tiles (the tile loop's) or none (a sequence with rows and no positions)."""
    text = _code(os.path.join(CSRC, "paged_attention.cu"))
    (math,) = [b for b in _blocks(text, r"while \(segment\(g\)\) \{")]
    at = math.index("sums[warp * ROWS")
    (with_tiles,) = _blocks(math[:at], r"for \(uint32_t t = g\.t0; t < g\.t1; \+\+t, \+\+it\) \{")
    assert "bar_math();" in with_tiles
    (head,) = _blocks(math[:at], r"if \(MT == 1 && g\.t0 < g\.t1\) \{")
    behind = math[math.index(head) + len(head):at].lstrip("} \n")
    assert behind.startswith("else {") and behind[len("else {"):].lstrip().startswith("bar_math();")


@pytest.mark.parametrize("name", ELECTING)
def test_what_waits_for_a_barrier_is_called_so(name):
    """The rule that lanes meet between a wait and an issue looks for waits by their name: a function of an issuing kernel's source that loops on a barrier's phase has no other."""
    text = _code(os.path.join(CSRC, name))
    for m in re.finditer(r"\bbool (\w+)\([^)]*\) \{", text):
        if "try_wait(" in next(_blocks(text[m.start():], r"\) \{")):
            assert m.group(1).startswith("mbar_wait"), m.group(1)
    for m in re.finditer(r"\bbool (\w+)\([^)]*\) \{\s*return (\w+)\(", text):
        assert not m.group(2).startswith("mbar_wait") or m.group(1).startswith("mbar_wait"), m.group(1)


def test_ctas_of_the_few_row_attention_go_by_the_batch():
    """Its shared memory grows with the batch: a launch that counts on two CTAs an SM where one fits runs in two waves of half the work each."""
    (launch,) = _blocks(_code(os.path.join(CSRC, "paged_attention.cu")), r"int launch_mma\(cudaStream_t stream, const PagedAttnArgs &w\) \{")
    assert not re.search(r"Z::bytes\(\d+\)", launch) and "w.r.batch" in launch[launch.index("const uint32_t grid"):]
