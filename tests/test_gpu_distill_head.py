"""The gradients of the output projection in lm_head_distillation: products of the library's own GEMM, whatever the number of classes."""
from pathlib import Path

import pytest
import torch

import mini_nccl_b200.ops.distill as distill
from mini_nccl_b200.ops import distillation_loss, gemm_bf16
from mini_nccl_b200.ops.distill import _LmHeadDistillation


def test_no_product_is_left_to_a_library():
    text = Path(distill.__file__).read_text()
    assert text.count("gemm_bf16(") == 3 and not any(call in text for call in ("torch.mm", "matmul", " @ "))


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,d", [(1, 9, 8), (15, 65, 16), (130, 512, 72), (256, 2049, 128), (300, 8191, 264), (666, 50257, 128), (64, 50257, 1024)])
def test_gradients_are_rounded_once(T, V, d):
    """Logits that bf16 holds exactly, so the gradient of the logits that the node works on is that of the loss alone, bit for bit.  Against its products in 64 bits: one rounding to
    bf16 is off by half a step, at most 2^-8 of a value and in random places within it, 2^-8 / sqrt(3) as a root mean square, and the fp32 sums (of
    random signs, each addition off by 2^-24 of a sum that stays near the result's size) 1e-5; sums rounded in slices come out at 2^-8."""
    g = torch.Generator().manual_seed(V + T)
    x = (torch.randint(-2, 3, (T, d), generator=g).to(torch.bfloat16) * 0.5).cuda().requires_grad_()
    w = (torch.randint(-1, 2, (V, d), generator=g).to(torch.bfloat16) * 0.25).cuda().requires_grad_()
    ids = torch.randint(0, V, (T, 5), generator=g).cuda()
    top = torch.randn(T, 5, generator=g).cuda()
    loss = _LmHeadDistillation.apply(x, w, ids, top, 2.0)
    dx, dw = torch.autograd.grad(loss * 3.0, [x, w])
    logits = torch.empty(T, (V + 7) // 8 * 8, device="cuda", dtype=torch.bfloat16)
    gemm_bf16(x.detach(), w.detach(), out=logits[:, :V])
    assert torch.equal(logits[:, :V].double(), x.detach().double() @ w.detach().double().t())
    z = logits[:, :V].detach().requires_grad_()
    dz, = torch.autograd.grad(distillation_loss(z, ids, top, 2.0) * 3.0, [z])
    for got, want in ((dx, dz.double() @ w.detach().double()), (dw, dz.double().t() @ x.detach().double())):
        assert float((got.double() - want).norm()) <= (2.0 ** -8 / 3 ** 0.5 + 1e-5) * float(want.norm())
    only, = torch.autograd.grad(_LmHeadDistillation.apply(x, w.detach(), ids, top, 2.0) * 3.0, [x])
    assert torch.equal(only, dx)
