"""The window's dK/dV kernel gets its units by number, through shared memory, behind waits that are bounded.  A wait that ran out is followed
by a read all the same: what it finds has to be a unit, or a number that ends the loop, and never what the memory held before."""
import re

from test_dependent_launch_cpu import functions, read


def test_unit_numbers_are_set_before_anybody_reads_one():
    (_, body), = functions(read("window_sm100.cu"))[0]["window_dkv_sm100_kernel"]
    setup = body[:body.index("__syncthreads()")]
    loop = re.search(r"for \(int s = 0; s < kDealt; \+\+s\) \{(.*?)\n    \}", setup, re.S)
    assert loop and re.search(r"sm->dealt\[s\] = INT32_MAX;", loop.group(1))
    # the loops end at a number that is no unit
    assert body.count("w < n_units") >= 3
