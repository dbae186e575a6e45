"""CPU: rules of the experts' tensor-core kernels that no run can be relied on to show, read from their source."""
import re

from test_kernel_source import body, code

ACCESS = re.compile(r"MB_TMEM_(?:LD16|ST8)\(")


def accesses(text):
    """Places where a warp reads or writes tensor memory, without the macros' definitions."""
    return [m.start() for m in ACCESS.finditer(text) if not text[:m.start()].rstrip().endswith("#define")]


def test_warps_are_whole_where_they_reach_tensor_memory():
    """The accesses want all lanes of the warp together.  After a wait, whose outcome is each lane's own, a vote or a barrier of the
    warp comes first."""
    text = code("experts.cuh")
    found = accesses(text)
    assert len(found) == 9
    for at in found:
        wait = text.rfind("mbar_wait(", 0, at)
        assert re.search(r"__all_sync\(|__syncwarp\(\)", text[wait:at]), text[wait:at]


def test_lanes_that_leave_a_row_out_come_back_before_the_next_access():
    """A loop over column groups that reads tensor memory and then works on the rows that are there: a barrier of the warp stands ahead of
    the next group's read."""
    text = code("experts.cuh")
    loops = [body(text, m.start()) for m in re.finditer(r"for \(int cg = 0;", text)]
    assert len(loops) == 2
    for loop in loops:
        if "valid" in loop:
            assert "__syncwarp();" in loop[:accesses(loop)[0]], loop
