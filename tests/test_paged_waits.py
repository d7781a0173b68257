"""What the kernels over a paged cache must keep so that each of their waits ends, read from their source: a wait that runs out is not to be caused on a device."""
import re
from pathlib import Path

CSRC = Path(__file__).parent.parent / "blockwise_int8_linear_b200" / "csrc"


def _results():
    """The part of the kernel for many queries that a tile's four warps run when their last product is done, without comments."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "paged_attention_tc.cu").read_text())
    begin = text.index("mbar_wait(bar(Z::kProductDone + t)")
    return text[:begin], text[begin:text.index("__syncthreads();", begin)]


def test_barriers_without_a_limit_stand_behind_a_vote():
    """A barrier of some of a block's warps waits for all of them, for ever.  Each has to stand behind a vote of the same warps on whether all came with their
    waits' success: otherwise one whose wait ran out leaves the others waiting."""
    before, results = _results()
    barrier = r"role_barrier\(|bar\.sync|barrier\.sync|__barrier_sync"
    assert not re.search(barrier, before)
    vote = re.search(r"if \(role_barrier_all\(t \+ 1, 128, ok\)\) \{", results)
    assert vote, "no vote"
    barriers = [m.start() for m in re.finditer(barrier, results)]
    assert barriers and all(m > vote.end() for m in barriers)
    # nothing between the last bounded wait and the vote leaves, so that every warp comes to it
    assert not re.search(r"return|break|else", results[:vote.start()])

