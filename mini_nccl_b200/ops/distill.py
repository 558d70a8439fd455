"""Distillation from a teacher's top logits: the loss of a student's logits against K entries (token id, logit) of a teacher for every
token, on the kernels of csrc/kernels/distill.cu, and the same fused with the output projection of a language model.

Logits are read once forward and once backward, where their gradient is written; elementary operators move them more than
ten times and hold several copies in fp32."""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from .fp8 import _FLOATS, _call, no_tangent
from .gemm import gemm_bf16
from .lm_loss import _MAX_ROWS, _eight, _pays, _plain, _transposed
from .lm_loss import _rows as _dense_rows

_MAX_ENTRIES, _MOST = 1024, 2**31 - 2**12   # mncclDistillForward
_REDUCTIONS = ("none", "sum", "mean")


def _reference(logits, ids, top, tau, reduction):
    """The plain operators, in fp32 (fp64 for fp64 logits)."""
    V = logits.shape[-1]
    z = logits if logits.dtype == torch.float64 else logits.float()
    there = (ids >= 0) & (top != -math.inf)
    counts = there.any(-1)
    t = torch.where(there, top.to(z.dtype), -math.inf) / tau
    log_p = torch.log_softmax(torch.where(counts.unsqueeze(-1), t, 0.0), -1)
    p = torch.where(there, log_p.exp(), 0.0)
    # tokens that count for nothing are taken out before the softmax, so that nothing of theirs reaches a gradient
    log_q = torch.log_softmax(torch.where(counts.unsqueeze(-1), z, 0.0) / tau, -1)
    inside = ids < V
    log_q = torch.where(inside, log_q.gather(-1, torch.where(there & inside, ids, 0)), math.nan)
    rows = tau * tau * torch.where(p != 0, p * (log_p - log_q), 0.0).sum(-1)
    if reduction == "none":
        return rows
    return rows.sum() if reduction == "sum" else rows.sum() / counts.sum()


def _forward(logits, ids, top, tau, reduction):
    """(loss, p, stats, counts, tokens): all but the first for the backward pass."""
    return _call("distill_forward", "mncclDistillForward", "csrc/kernels/distill.cu")(logits, ids, top, tau, _REDUCTIONS.index(reduction))


def _backward(logits, ids, p, stats, counts, tokens, tau, reduction, grad):
    return _call("distill_backward", "mncclDistillBackward", "csrc/kernels/distill.cu")(logits, ids, p, stats, counts, tokens if reduction == "mean" else None,
                                                                                        tau, grad)


def _again(ctx, inputs, f, grad):
    """create_graph: the gradient itself is differentiated, by the plain operators."""
    fresh = [t.view_as(t) for t in inputs]
    picks = [i for i in range(len(inputs)) if ctx.needs_input_grad[i]]
    got = torch.autograd.grad(f(*fresh), [fresh[i] for i in picks], grad, create_graph=True)
    out = dict(zip(picks, got))
    return [out.get(i) for i in range(len(inputs))]


def _gradient_again(logits, ids, top, tau, reduction, grad):
    """The gradient of the logits by operators that can be differentiated."""
    at = ids.view(*logits.shape[:-1], -1), top.view(*logits.shape[:-1], -1)
    with torch.enable_grad():
        z = logits.view_as(logits)
        return torch.autograd.grad(_reference(z, *at, tau, _REDUCTIONS[reduction]), [z], grad, create_graph=True)[0]


class _LmHeadDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, ids, top, tau):
        V = weight.shape[0]
        rows, w = _dense_rows(x.detach()).view(-1, x.shape[-1]), _dense_rows(weight.detach())
        logits = torch.empty((rows.shape[0], _eight(V)), dtype=x.dtype, device=x.device)
        gemm_bf16(rows, w, out=logits[:, :V])
        loss, *kept = _forward(logits[:, :V], ids, top, tau, "mean")
        ctx.save_for_backward(x, weight, ids, top, logits, *kept)
        ctx.tau = tau
        return loss

    @staticmethod
    def backward(ctx, grad):
        x, weight, ids, top, logits, *kept = ctx.saved_tensors
        want_x, want_w = ctx.needs_input_grad[:2]
        if torch.is_grad_enabled():
            at = ids.view(*x.shape[:-1], -1), top.view(*x.shape[:-1], -1)
            return (*_again(ctx, [x, weight], lambda a, b: _reference(F.linear(a, b), *at, ctx.tau, "mean"), grad), None, None, None)
        stream = torch.cuda.current_stream().cuda_stream
        V = weight.shape[0]
        rows, logits = _dense_rows(x).view(-1, x.shape[-1]), _dense_rows(logits)
        d = _backward(logits[:, :V], ids, *kept, ctx.tau, "mean", grad)   # in padded rows, as the logits
        dx = gemm_bf16(d, _transposed(_dense_rows(weight), stream)).view(x.shape) if want_x else None
        dw = gemm_bf16(_transposed(d, stream), _transposed(rows, stream)) if want_w else None
        return dx, dw, None, None, None


def _plain_call():
    """Nothing is active that looks at or transforms the single operators."""
    return not (torch.jit.is_tracing() or torch.compiler.is_compiling() or torch._C._are_functorch_transforms_active()
                or torch._C._len_torch_function_stack() or torch._C._len_torch_dispatch_stack())


def _native(logits, ids, top):
    """Whether the kernels take the call; the plain operators take the others."""
    if not (logits.is_cuda and _plain(logits) and _plain(ids) and _plain(top) and logits.dtype in _FLOATS):
        return False
    if not (0 < ids.shape[-1] <= _MAX_ENTRIES and 0 < ids.numel() // ids.shape[-1] <= _MOST and 0 < logits.shape[-1] <= _MOST) or not _plain_call():
        return False
    return no_tangent(logits)


def _arguments(shape, device, ids, top, temperature, reduction="mean"):
    """The teacher's entries as the kernels read them, and the temperature."""
    lead = tuple(shape[:-1])
    for t, name in ((ids, "top_ids"), (top, "top_logits")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor")
        if t.dim() != len(lead) + 1 or t.shape[:-1] != lead or t.shape[-1] == 0 or t.device != device:
            raise ValueError(f"{name} must be {[*lead, 'K']} on {device}")
    if ids.shape != top.shape:
        raise ValueError("top_ids and top_logits must have one shape")
    if ids.dtype is not torch.int64:
        if ids.dtype is not torch.int32:
            raise TypeError("top_ids must be int64 or int32")
        ids = ids.long()
    if not top.dtype.is_floating_point:
        raise TypeError("top_logits must be floating point")
    temperature = float(temperature)
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError("the temperature must be between 1e-3 and 1e3")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}")
    return ids, top.detach() if top.requires_grad else top, temperature


def _rows_of_entries(t, dtype):
    """[T, K], dense, with its own signs."""
    if t.is_neg():
        t = t.resolve_neg()
    if t.dtype is not dtype:
        t = t.to(dtype)
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.is_contiguous() else t.contiguous()


def distillation_loss(logits, top_ids, top_logits, temperature=1.0, reduction="mean"):
    """Distillation of a student's ``logits [..., V]`` (bf16, fp16 or fp32; loss in fp32) from a teacher's entries ``top_ids [..., K]`` and
    ``top_logits [..., K]``, differentiable in ``logits``.

    With ``p`` the softmax of ``top_logits / temperature`` over a token's entries and ``q`` that of ``logits / temperature`` over all
    classes, a token's loss is ``temperature ** 2 * sum(p * (log p - log q[id]))``.  A negative id or a logit of -inf marks an
    entry that is not there.  Tokens without entries count for nothing, whatever their logits are: no loss, no gradient, left
    out of the mean (which is NaN if no token counts).  Ids may repeat; one of V or more makes its token's loss and gradient NaN.
    ``reduction``: ``"mean"`` over the tokens that count, ``"sum"``, or ``"none"`` for a loss ``[...]`` per token."""
    if not isinstance(logits, torch.Tensor) or not logits.dtype.is_floating_point or logits.dim() < 1:
        raise TypeError("logits must be a floating-point tensor [..., V]")
    if logits.shape[-1] == 0:
        raise ValueError("logits without classes")
    ids, top, tau = _arguments(logits.shape, logits.device, top_ids, top_logits, temperature, reduction)
    if not _native(logits, ids, top):
        return _reference(logits, ids, top, tau, reduction)
    return _call("distillation", "mncclDistillForward", "csrc/kernels/distill.cu")(
        logits, _rows_of_entries(ids, torch.int64), _rows_of_entries(top, torch.float32), tau, _REDUCTIONS.index(reduction), _gradient_again)


def lm_head_distillation(x, weight, top_ids, top_logits, temperature=1.0):
    """Mean :func:`distillation_loss` of ``F.linear(x, weight)`` (logits rounded to x's type) as one node: ``x [..., d]``, ``weight
    [V, d]``; differentiable in both.  The teacher's entries as there."""
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.shape[0] == 0:
        raise ValueError("shapes: x [..., d], weight [V, d]")
    ids, top, tau = _arguments((*x.shape[:-1], weight.shape[0]), x.device, top_ids, top_logits, temperature)
    V, d = weight.shape
    T = math.prod(x.shape[:-1])
    native = (x.dim() >= 2 and x.dtype == weight.dtype == torch.bfloat16 and x.device == weight.device and _plain(x) and _plain(weight)
              and x.is_cuda and x.device.index == torch.cuda.current_device() and V >= 8 and d >= 8 and d % 8 == 0 and 0 < T
              and max(T, V) <= _MAX_ROWS and not torch.is_autocast_enabled() and _native(x, ids, top)
              and no_tangent(weight))
    if not native or not _pays(T, V, d):
        return distillation_loss(F.linear(x, weight), ids, top, tau)
    return _LmHeadDistillation.apply(x, weight, _rows_of_entries(ids, torch.int64), _rows_of_entries(top, torch.float32), tau)
