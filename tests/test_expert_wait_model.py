"""Model of what the epilogue warps of the grouped products do when a wait runs out, on the CPU.

Warps of an epilogue share staging buffers, two or more to a buffer, and meet at a named barrier for each tile.  The wait for a tile
is bounded; after one that ran out, whether a warp still sees the tile complete or sees the abort flag first is a matter of timing.
All outcomes are explored for a few warps and tiles: a warp that leaves the tile loop alone leaves its partner at the barrier for good;
if nobody leaves, every barrier gets its warps and all of them reach the end.  The second test holds the kernels to that form."""
import itertools
import re
from pathlib import Path

import pytest

import umdk_original_b200

KERNELS = Path(umdk_original_b200.__file__).parent / "csrc" / "kernels"
TILES = 3


def ends(protocol, outcomes):
    """True if every warp reaches the teardown; outcomes[w][t]: would warp w's wait for tile t succeed."""
    visits = []
    for seen in outcomes:
        met = []
        for t, ok in enumerate(seen):
            if protocol == "leave" and not ok:
                break
            met.append(t)
        visits.append(met)
    # a barrier of two warps completes tile by tile: both have to come as often as each other
    return all(len(a) == len(b) for a, b in zip(visits[0::2], visits[1::2]))


def outcomes(warps):
    one = list(itertools.product((True, False), repeat=TILES))
    return itertools.product(one, repeat=warps)


def test_leaving_the_loop_alone_hangs_and_staying_does_not():
    assert not all(ends("leave", o) for o in outcomes(4))
    assert all(ends("stay", o) for o in outcomes(4))


def epilogues(name):
    """Source of every epilogue of a file: from its heading to the kernel's teardown."""
    text = (KERNELS / name).read_text()
    found = re.findall(r"-{8,} epilogue.*?-{8,} teardown", text, re.S)
    assert found
    return found


@pytest.mark.parametrize("name,count", [("grouped_gemm_fp4.cu", 1), ("grouped_mlp.cu", 2), ("expert_gemm_narrow.cu", 1)])
def test_no_warp_decides_alone(name, count):
    """In the kernels on CTA pairs no epilogue warp leaves the tile loop; in the other form they leave together, on an answer that a
    barrier over all of them has given."""
    found = epilogues(name)
    assert len(found) == count
    for text in found:
        code = re.sub(r"//[^\n]*", "", text)
        for line in code.splitlines():
            if re.search(r"\bbreak\b", line):
                assert "named_bar_and(1, kNwEpiThreads, got)" in line
        assert "named_bar_and" in code or re.search(r"for \(int tile = pair_id; (w\.)?locate\(", code)


@pytest.mark.parametrize("name", ["grouped_gemm.cu", "grouped_gemm_mx.cu", "grouped_gemm_mx2.cu", "grouped_gemm_i8.cu",
                                  "grouped_gemm_rows_n.cuh", "fused_moe_mx.cu"])
def test_warps_of_the_8_bit_products_leave_together(name):
    """All epilogue warps of a CTA agree on the answer of a wait before the first barrier that would need them all; inside a sum over
    K-blocks, which has no barrier, the lanes of a warp agree."""
    for text in epilogues(name):
        code = re.sub(r"//[^\n]*", "", text)
        first = code.index("named_bar_and(1, k")
        assert first < code.index("named_bar_sync(")
        for line in code.splitlines():
            if re.search(r"\bbreak\b", line):
                assert "named_bar_and(1, k" in line or ("__all_sync(" in line and code.index(line) < first)
