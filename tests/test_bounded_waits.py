"""What a kernel does when a bounded wait runs out, by reading its source (no test makes one run out on a device)."""
import re

from flambeau_b200.kernels.build import CSRC


def test_the_product_with_four_bit_weights_lets_what_is_under_way_end():
    """Copies and MMAs of a block that gives up still use its shared and tensor memory: it waits for them, with a limit, before it
    frees the columns; the warp that frees them is the block's last to return."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "gemm_mxfp4.cu").read_text())
    end = text[text.rindex("__syncthreads();", 0, text.index("tmem_dealloc(")):]
    assert re.search(r"if \(bailed\(\)\) fb_settle\(\);.*?tmem_dealloc\(", end, re.S)
    waits = text[text.index("gemm_mxfp4_kernel("):]
    assert len(re.findall(r"\*bail = 1", waits)) >= 6, "every role says when it gives up"
    settle = (CSRC / "async_copy.cuh").read_text()
    assert re.search(r"global_ns\(\) - t0 < FB_SETTLE_NS", settle)
