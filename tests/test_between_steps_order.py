"""What eviction's source promises about memory order, where no run can show it (a weaker form gave the same bytes in every test)."""
import os
import re

SEQ = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "blazr_b200", "csrc", "seq")


def test_rows_have_been_read_before_another_block_writes_over_them():
    """A relaxed arrival at a cluster's barrier orders nothing.  Where threads arrive so, a warp that they have met at a barrier of the block (bar.arrive 2, bar.sync 2) releases for them;
    who stores has waited with acquire."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(SEQ, "seq_evict.cu")).read())
    body = text[text.index("evict_move_kernel("):]
    body = body[:body.index("cudaError_t move_as")]
    read = re.search(r"cp\.async\.wait_group.*?\n\s*store\(", body, re.S).group(0)
    clustered = read[read.index("else"):]
    order = re.findall(r"bar\.arrive 2|barrier\.cluster\.\w+\.\w+", clustered)
    assert order == ["bar.arrive 2", "barrier.cluster.arrive.relaxed", "barrier.cluster.wait.acquire"] or order[0] == "barrier.cluster.arrive.release"
    if order[0] == "bar.arrive 2":
        warp = re.search(r"bar\.sync 2.*?return;", body, re.S).group(0)
        assert re.findall(r"barrier\.cluster\.\w+\.\w+", warp) == ["barrier.cluster.arrive.release", "barrier.cluster.wait.acquire"]
