"""The refusal flag of the step tables kernel (no GPU): thread 0 clears it, any thread may set it, so a block barrier stands
between the two. Which of them comes first is a matter of timing that no run shows for certain."""
import os

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-sglang-cpp_b200", "csrc", "batch.cu")


def test_a_barrier_between_clearing_and_setting():
    text = open(SRC).read()
    kernel = text[text.index("step_tables_kernel(const StepArgs a) {"):]
    clear, first_set = kernel.index("bad = 0;"), kernel.index("atomicOr(&bad")
    assert clear < first_set and "__syncthreads();" in kernel[clear:first_set]
