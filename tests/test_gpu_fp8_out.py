"""The result of gemm_fp8 written into a tensor of the caller's: autograd learns of it."""
import pytest
import torch

import mini_nccl_b200 as mn
from mini_nccl_b200 import _lib
from mini_nccl_b200._ctypes_calls import Calls
from mini_nccl_b200.ops import gemm_fp8, quantize_fp8


@pytest.mark.gpu
def test_a_kept_operand_that_is_overwritten_is_noticed():
    q, s = quantize_fp8(torch.randn(8, 256, device="cuda"))
    w, ws = quantize_fp8(torch.randn(24, 256, device="cuda"), block_rows=128)
    want = gemm_fp8(q, s, w, ws)
    for c in (_lib.ext(), Calls(mn.lib())):
        buffer = torch.ones(8, 24, device="cuda", dtype=torch.bfloat16)
        leaf = torch.ones_like(buffer).requires_grad_()
        y = (leaf * buffer).sum()   # keeps the buffer
        before = buffer._version
        assert c.gemm_fp8(q, s, w, ws, buffer, None, None, None) is buffer and torch.equal(buffer, want) and buffer._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        c.gemm_fp8(q, s, w, ws, buffer[:, :], None, None, None)   # a view's count is its base's
        assert buffer._version > before + 1
        with torch.inference_mode():
            inside = torch.empty(8, 24, device="cuda", dtype=torch.bfloat16)
            c.gemm_fp8(q, s, w, ws, inside, None, None, None)
        assert torch.equal(inside, want)
        c.gemm_fp8(q, s, w, ws, inside, None, None, None)   # keeps no count, in and out of the mode
        assert torch.equal(inside, want)
