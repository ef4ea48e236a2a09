"""What a kernel does when a bounded wait runs out, by reading its source (no test makes one run out on a device)."""
import re

from flambeau_b200.kernels.build import CSRC


def test_the_product_with_four_bit_weights_lets_what_is_under_way_end():
    """Copies and MMAs of a block that gives up still use its shared and tensor memory.  The epilogue is the last to be told: it
    either has had the sums of every unit, and so every copy, or it waits, with a limit, ahead of the block's last barrier, behind
    which the columns are freed."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "gemm_mxfp4.cu").read_text())
    kernel = text[text.index("gemm_mxfp4_kernel("):]
    assert len(re.findall(r"\*bail = 1", kernel)) >= 6, "every role says when it gives up"
    stop, settled, freed = kernel.index("stop = *flag == 2;"), kernel.index("let_end();"), kernel.index("tmem_dealloc(")
    assert re.search(r"if \(stop\) \{\s*let_end\(\);\s*break;", kernel)
    assert stop < settled < kernel.rindex("__syncthreads();", 0, freed) < freed
    assert "void let_end() { fb_settle(); }" in text
    assert re.search(r"global_ns\(\) - t0 < FB_SETTLE_NS", (CSRC / "async_copy.cuh").read_text())
