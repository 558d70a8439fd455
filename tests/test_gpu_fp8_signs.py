"""Views of numbers with the other sign: PyTorch hands the imaginary part of a conjugate on as a view of the number with a mark, to forward calls and to backward
passes.  The kernels read memory, so the operators resolve the mark or refuse the tensor."""
import pytest
import torch

import mini_nccl_b200 as mn
from mini_nccl_b200 import _lib
from mini_nccl_b200._ctypes_calls import Calls
from mini_nccl_b200.ops import distillation_loss, gemm_fp8, quantize_fp8
from mini_nccl_b200.ops.distill import _gradient_again


def _calls():
    return _lib.ext(), Calls(mn.lib())


def _opposite(t):
    """-t as a view of t's memory with the mark."""
    v = torch._neg_view(t)
    assert v.is_neg() and v.data_ptr() == t.data_ptr()
    return v


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_gradients_that_come_through_a_conjugate(n):
    """With one output feature such a gradient needs no copy for its strides."""
    g = torch.Generator(device="cuda").manual_seed(n)
    w, b, x = (torch.randn(*shape, generator=g, device="cuda") for shape in ((n, 256), (n,), (6, 256)))
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    seen = []
    for c in _calls():
        results = []
        for conjugate in (True, False):
            y = c.linear_fp8(x, w, b)
            if conjugate:
                y.register_hook(lambda d: seen.append(d.is_neg()))
            z = torch.complex(torch.zeros_like(y), y)
            z = z.conj() if conjugate else torch.view_as_complex(torch.view_as_real(z) * torch.tensor([1.0, -1.0], device="cuda"))
            results.append(torch.autograd.grad(z, [x, w, b], torch.full_like(z, 1 + 2j)))
        assert all(torch.equal(p, q) for p, q in zip(*results)) and all(bool(p.any()) for p in results[0])
    assert seen == [True, True]


@pytest.mark.gpu
def test_forward_calls():
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w, b = (torch.randn(*shape, generator=g, device="cuda") for shape in ((6, 256), (130, 256), (130,)))
    for c in _calls():
        want = c.linear_fp8(-x, -w, -b)
        assert torch.equal(c.linear_fp8(_opposite(x), _opposite(w), _opposite(b)), want)
        z, ids = torch.randn(5, 300, generator=g, device="cuda"), torch.randint(0, 300, (5, 3), generator=g, device="cuda")
        top = torch.randn(5, 3, generator=g, device="cuda")
        got, want = (c.distillation(t, ids, top, 1.0, 2, _gradient_again) for t in (_opposite(z), -z))
        assert torch.equal(got, want)
        leaf = z.clone().requires_grad_()
        loss = c.distillation(leaf, ids, top, 1.0, 2, _gradient_again)
        got, want = (torch.autograd.grad(loss, [leaf], d, retain_graph=True)[0] for d in (_opposite(torch.ones((), device="cuda")), -torch.ones((), device="cuda")))
        assert torch.equal(got, want) and bool(got.any())
    assert torch.equal(distillation_loss(z, ids, _opposite(top)), distillation_loss(z, ids, -top))


@pytest.mark.gpu
def test_refusals():
    x, w, b = torch.ones(4, 128, device="cuda"), torch.ones(8, 128, device="cuda"), torch.ones(8, device="cuda", dtype=torch.bfloat16)
    q, s, wq, ws = *quantize_fp8(x), *quantize_fp8(w, block_rows=128)
    for c in _calls():
        with pytest.raises(ValueError, match="other sign"):
            c.quantize_fp8(_opposite(x), 1, False, None)
        for at in (1, 3):
            args = [q, s, wq, ws]
            args[at] = _opposite(args[at])
            with pytest.raises(ValueError, match="other sign"):
                c.gemm_fp8(*args, None, None, None, None)
        with pytest.raises(ValueError, match="other sign"):
            c.gemm_fp8(q, s, wq, ws, _opposite(torch.zeros(4, 8, device="cuda")), None, None, None)
        with pytest.raises(ValueError, match="bias"):
            c.gemm_fp8(q, s, wq, ws, None, None, _opposite(b), None)
    with pytest.raises(ValueError, match="other sign"):
        quantize_fp8(_opposite(x))
    with pytest.raises(ValueError, match="other sign"):
        gemm_fp8(q, _opposite(s), wq, ws)
