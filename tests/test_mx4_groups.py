"""The grouped tiles of the 4-bit Linear by their source: what orders the wavefronts' use of LDS."""

import os
import re

import sparseflow_amd

CSRC = os.path.join(os.path.dirname(sparseflow_amd.__file__), "csrc")


def test_sums_are_read_before_rows_lie_over_them():
    """The groups' sums (4096 bytes a tile and wavefront) and the rows on their way out (32 of 272 bytes a wavefront) share
    LDS: wavefront 0's rows are bytes 0 to 8703, where wavefront 1's and 2's sums are.  Between the last read of sums and
    the rows stands a barrier of the workgroup, and no wavefront has left before it."""
    with open(os.path.join(CSRC, "sf_mx4_gemm.hip")) as f:
        text = f.read()
    kernel = text[text.index("void k_mx4_gemm_any"):]
    kernel = kernel[:kernel.index("\ntemplate <auto K")]
    code = re.sub(r"//[^\n]*", "", kernel)
    joined = code[code.index("float* sums"):]
    after = joined[joined.rindex("sums["):joined.index("gemm_store(")]
    barrier = after.find("__syncthreads()")
    assert barrier >= 0
    assert "return" not in joined[:joined.rindex("sums[")] and "return" not in after[:barrier]
