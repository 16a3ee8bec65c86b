"""The CTAs of a PageSelectAttention cluster meet equally often whatever lengths they read.

A caller that writes the lengths while the kernel reads them breaks the rules and gets wrong
results, but CTAs of one cluster that take different ways must not leave while another one still
reads their shared memory: on the GPU that is a fault, so it is shown on the source here."""

import re
from pathlib import Path

SRC = (Path(__file__).parents[1] / "iron_b200" / "csrc" / "page_select.cu").read_text()
KERNEL = SRC[SRC.index("select_kernel(SelectArgs a)") : SRC.index("// Pieces: `per` blocks per unit")]


def meetings(text):
    return len(re.findall(r"\bmeet\(\);", text))


def test_both_ways_through_the_kernel_meet_equally_often():
    # one decision, the same for all threads of the CTA
    assert "const bool choose = __syncthreads_or(n > a.top);" in KERNEL
    start, other = KERNEL.index("if (choose) {"), KERNEL.index("  } else {\n    for (int i = threadIdx.x; i < a.top;")
    end = KERNEL.index("if constexpr (!kAttend) return;")
    assert meetings(KERNEL[:start]) == 0 and meetings(KERNEL[other:end]) == 0
    late = KERNEL.index("if (ranks > 1 && !choose && a.M > a.top) {")
    assert meetings(KERNEL[start:other]) == meetings(KERNEL[late:]) == 2
    # what reads other CTAs' memory lies between meetings that both ways have
    assert "map_shared_rank" not in KERNEL[:start] and "map_shared_rank" not in KERNEL[late:]


def test_a_place_read_back_lies_in_the_sequence():
    assert "at >= 0 && at < n ? make_int2(at, ld_act_i32(table + at))" in SRC
