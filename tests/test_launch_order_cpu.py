"""Three kernels read inputs, and one other reads lengths, ahead of their own griddepcontrol.wait.  That is sound as long as whatever runs in
front of them lets them start only behind a wait of its own: everything older is complete then, and only the kernel directly in front
may still be running.  So every kernel triggers behind its wait, the exceptions are the ones named here, and what the kernel
directly in front writes is read behind the wait.  Read off the sources, since a line that moves brings a race that nobody sees."""
import re

import pytest

from test_dependent_launch_cpu import WAITING, functions, read

# touch global memory ahead of their wait: the kernel -> the kernel in front of it
EARLY = {"window_dq_sm100_kernel": "window_delta_kernel", "window_dkv_sm100_kernel": "window_dq_sm100_kernel",
         "sm100_bwd_dkv_kernel": "sm100_bwd_dq_kernel", "paged_finish_kernel": "paged_attend_kernel"}
TOUCH = re.compile(r"\btma_load_|\bld_behind_wait\(|\bunit_of\(w|\bpg\.length\(|\batomicAdd\(|\bload_queries")


def kernel(source, name):
    (_, body), = functions(read(source))[0][name]
    return body


@pytest.mark.parametrize("source", WAITING)
def test_kernels_let_others_start_only_behind_their_own_wait(source):
    found = 0
    for name, forms in functions(read(source))[0].items():
        for _, body in forms:
            if "grid_dep_launch()" in body:
                found += 1
                assert 0 <= body.index("grid_dep_wait()") < body.index("grid_dep_launch()"), name
    assert found


def test_the_chain_in_front_of_the_early_readers():
    for front in set(EARLY.values()):
        source = {"window": "window_sm100.cu", "sm100_": "attn_sm100.cu", "paged_": "paged.cu"}[front[:6]]
        body = kernel(source, front)
        # its trigger comes behind its own wait; without a trigger the next kernel starts behind its end
        assert body.index("grid_dep_wait()") < body.index("grid_dep_launch()")
    # the delta kernel does nothing ahead of its wait
    body = kernel("window_sm100.cu", "window_delta_kernel")
    assert not TOUCH.search(body[:body.index("grid_dep_wait()")])
    assert body.index("*p.next = 0") > body.index("grid_dep_wait()")


def test_dq_reads_delta_and_writes_behind_its_wait():
    body = kernel("window_sm100.cu", "window_dq_sm100_kernel")
    wait = body.index("grid_dep_wait()")
    assert body.index("fetch_rows(unit_at(0))") > wait               # lse and delta
    definitions = [m.start() for m in re.finditer(r"p\.delta|p\.dq\b|p\.dk\b|p\.dv\b", body)]
    drain = body.index("auto drain = ["), body.index("auto fetch_rows = [")
    for at in definitions:                                           # in the lambdas that are called behind it, or behind it themselves
        assert at > wait or drain[0] < at < drain[1] or body.rindex("auto fetch_rows", 0, at) > drain[0]
    assert body.index("if (warp_uniform(drain_row >= 0)) drain();") > wait


def test_dkv_ends_behind_the_kernel_in_front_and_lets_nothing_start():
    body = kernel("window_sm100.cu", "window_dkv_sm100_kernel")
    assert "grid_dep_launch" not in body and body.count("grid_dep_wait()") == 1
    assert body.index("grid_dep_wait()") < body.rindex("__syncthreads()")
    assert "grid_dep_launch" not in kernel("attn_sm100.cu", "sm100_bwd_dkv_kernel")


def test_no_other_kernel_touches_memory_ahead_of_its_wait():
    for source in WAITING:
        for name, forms in functions(read(source))[0].items():
            for _, body in forms:
                if "grid_dep_wait()" in body and name not in EARLY:
                    # lambdas defined above the wait are called below it; stores and loads proper come behind
                    ahead = re.sub(r"auto \w+ = \[&\][^;]*?\{.*?\n  \};", "", body[:body.index("grid_dep_wait()")], flags=re.S)
                    ahead = re.sub(r"auto \w+ = \[&\]\([^)]*\) \{ return [^\n]*", "", ahead)
                    assert not TOUCH.search(ahead), name
