"""CPU: rules of the cache kernels' sources that no run can show to be kept."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse_b200", "csrc")


def _block(text, start):
    """The braces' content behind `start`."""
    open_brace = text.index("{", start)
    depth, end = 1, open_brace + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        end += 1
    return text[open_brace + 1:end - 1]


def test_a_wait_that_gives_up_leaves_no_result_as_it_was():
    """Where a wait of the prefix kernel ran out, its partial rows hold whatever the workspace held: the kernel
    makes all of them NaN, behind a barrier of the CTA and whether or not a status word was given."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "attn_prefix.cu")).read())
    kernel = _block(text, text.index("attn_prefix_kernel(const __grid_constant__"))
    at = kernel.index("if (*abort_flag) {")
    assert kernel[:at].rstrip().endswith("__syncthreads();")
    marks = re.search(r"for \(int i = threadIdx\.x; i < rows; i \+= L::kThreads\) part_lse\[slot_row \+ i\] = __uint_as_float\(0x7fc00000u\);",
                      _block(kernel, at))
    assert marks
    # (no condition of its own in front of it but the status word's, which ends with its statement)
    before = _block(kernel, at)[:marks.start()]
    assert before.count("if (") == 1 and before.count("{") == 0


def test_tensor_memory_is_taken_behind_the_wait_for_the_launches_before():
    """A CTA that started early and holds tensor memory could keep it from one that it waits for."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "attn_prefix.cu")).read())
    kernel = _block(text, text.index("attn_prefix_kernel(const __grid_constant__"))
    assert kernel.count("tcgen05.alloc") == 1 and kernel.index("pdl_wait();") < kernel.index("tcgen05.alloc")
