"""A student decoder in 8 bits that learns from a teacher's top logits: the operators as a training step uses them together."""
import pytest
import torch

import mini_nccl_b200 as mn
from mini_nccl_b200.models import GPT2Config, GPT2Model


def _models(**more):
    cfg = dict(n_layer=2, d_model=128, n_head=4, vocab_size=515, seq_len=70)
    torch.manual_seed(0)
    plain = GPT2Model(GPT2Config(**cfg))
    fp8 = GPT2Model(GPT2Config(**cfg, linear="fp8"))
    fp8.load_state_dict(plain.state_dict())
    return plain, fp8


def test_configuration():
    plain, fp8 = _models()
    assert [n for n, _ in plain.named_parameters()] == [n for n, _ in fp8.named_parameters()]
    with pytest.raises(ValueError, match="linear"):
        GPT2Model(GPT2Config(n_layer=1, d_model=64, n_head=1, vocab_size=8, seq_len=4, linear="int3"))
    ids = torch.zeros(1, 4, dtype=torch.int64)
    teacher = torch.zeros(1, 4, 2, dtype=torch.int64), torch.zeros(1, 4, 2)
    with pytest.raises(ValueError, match="not both"):
        plain(ids, targets=ids, teacher=teacher)
    assert torch.isfinite(plain(ids, teacher=(*teacher, 2.0)))


@pytest.mark.gpu
def test_student_step_under_data_parallel():
    """Loss and gradients of the 8-bit student are those of the plain decoder up to the quantisation: each product's operands are off by
    2^-4 of a value at most, by 2^-4 / sqrt(3) of it as a root mean square, in random directions; five products deep in both passes that
    stays well below half of a gradient's norm (a wrong scale or a missing product does not)."""
    from mini_nccl_b200.parallel import DistributedDataParallel

    plain, fp8 = (m.cuda().to(torch.bfloat16) for m in _models())
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 515, (3, 70), generator=g, device="cuda")
    with torch.no_grad():
        torch.manual_seed(5)
        teacher = GPT2Model(GPT2Config(n_layer=1, d_model=64, n_head=1, vocab_size=515, seq_len=70)).cuda()
        for p in teacher.parameters():
            p.mul_(3.0)
        top, top_ids = teacher(ids).topk(20, dim=-1)
    top_ids[:, :9] = -1     # the prompt
    entries = (top_ids, top, 2.0)
    want = plain(ids, teacher=entries)
    want.backward()
    comm = mn.Communicator(1, 0)
    try:
        ddp = DistributedDataParallel(fp8, comm, bucket_mb=0.25)
        losses = []
        for _ in range(2):
            ddp.zero_grad()
            loss = ddp(ids, teacher=entries)
            loss.backward()
            losses.append(loss.detach())
        assert torch.equal(*losses)
        assert abs(float(losses[0]) - float(want.detach())) <= 0.05 * abs(float(want.detach()))
        for (name, p), q in zip(plain.named_parameters(), fp8.parameters()):
            assert q.grad is not None and torch.isfinite(q.grad).all(), name
            assert float((q.grad.float() - p.grad.float()).norm()) <= 0.5 * float(p.grad.float().norm()), name
    finally:
        comm.destroy()


@pytest.mark.gpu
def test_step_is_the_operators_one_after_the_other():
    """One Fp8Linear, the head and the loss against the same calls made by hand."""
    from mini_nccl_b200.models.gpt2 import Fp8Linear
    from mini_nccl_b200.ops import distillation_loss, gemm_fp8, linear_fp8, quantize_fp8

    torch.manual_seed(2)
    layer = Fp8Linear(256, 384).cuda().to(torch.bfloat16)
    head = (torch.randn(1000, 384, device="cuda") * 0.05).to(torch.bfloat16)
    x = torch.randn(77, 256, device="cuda").to(torch.bfloat16)
    top, top_ids = torch.randn(77, 1000, device="cuda").topk(10)
    y = layer(x)
    q, s = quantize_fp8(x)
    wq, ws = quantize_fp8(layer.weight.detach(), block_rows=128)
    assert torch.equal(y, gemm_fp8(q, s, wq, ws, bias=layer.bias.detach()))
    loss = distillation_loss(torch.nn.functional.linear(y, head), top_ids, top)
    loss.backward()
    z = torch.nn.functional.linear(y.detach(), head).requires_grad_()
    dz, = torch.autograd.grad(distillation_loss(z, top_ids, top), [z])
    dy = dz @ head
    w = layer.weight.detach().requires_grad_()
    dw, = torch.autograd.grad(linear_fp8(x, w, layer.bias.detach()), [w], dy)
    assert torch.equal(layer.weight.grad, dw)
    g, gs, gt, gts = quantize_fp8(dy, transposed=True)
    _, _, xt, xts = quantize_fp8(x, transposed=True)
    assert torch.equal(dw, gemm_fp8(gt, gts, xt, xts))
