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



def test_the_kernel_that_begins_without_a_wait_reads_from_the_l2():
    """Beside the kernel for many queries the one for few has no wait that shows it what earlier kernels wrote, so no load of its own may find something older
    in the SM's cache.  (The branch of a lone call and its search for the tile come behind a wait.)"""
    text = re.sub(r"//[^\n]*", "", (CSRC / "paged_attention.cu").read_text())
    kernel = text[text.index("paged_few_kernel(const PagedAttnArgs a)"):text.index("paged_join_kernel(")]
    beside = kernel[kernel.index("if (a.by_length) {"):kernel.index("} else {")]
    assert beside.count("first_token<true>(") == 2 and "wait" not in beside
    rest = kernel[kernel.index("if (qt.rows == 0)"):]
    assert not re.search(r"ld_nc|first_token\(|first_position\(|start\(|not_finite<T, false>", rest)
    assert re.findall(r"a\.by_length \? ld_l2\(p\) : \*p;", rest) and "__ldg" not in rest
    assert "cp.async.cg" in re.search(r"void copy16\(uint32_t dst, const void\* src, int bytes\).*?\n}", (CSRC / "int4_common.cuh").read_text(), re.S).group()
