"""mncclSumBlocks takes what mncclQuantizeFp8 makes and refuses larger sizes, whose indices would pass 2^31, before anything is launched."""
import ctypes as C

import mini_nccl_b200 as mn


def test_sizes_that_no_quantisation_makes_are_refused():
    L = mn.lib()
    p = C.c_void_p(4096)   # never looked at
    for blocks, K in ((1, 65535 * 128 + 1), (1, 2**31 - 1), (2**24, 8), (2**31 - 1, 8)):
        for dtype in (6, 7, 9):
            assert L.mncclSumBlocks(p, blocks, K, p, dtype, None) == -2, (blocks, K)
