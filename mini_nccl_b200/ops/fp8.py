"""8-bit floating point (e4m3) with a scale for each block of 128: quantisation, products on the Blackwell tensor cores,
and a linear layer whose three products of a training step run in 8 bits.

Activations and gradients have a scale for each 128 elements of a row, weights for each 128 x 128 elements.  The scales that
:func:`quantize_fp8` chooses are powers of two (csrc/kernels/fp8_quantize.cu says why); :func:`gemm_fp8` takes any fp32
scales, such as a checkpoint's.  Like :func:`gemm_bf16` these fail loudly where the native kernels are missing."""
from __future__ import annotations

import torch

from .._lib import ext, lib

BLOCK = 128
_MOST_ROWS, _MOST_COLUMNS = 2**31 - 1 - 2**16, 65535 * BLOCK   # mncclQuantizeFp8
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_RECORDING = tuple(getattr(torch._C._TorchDispatchModeKey, name) for name in ("FAKE", "PROXY", "FUNCTIONAL"))
_calls = {}   # the extension's entry points, looked up on the first call


def _call(name, symbol, source):
    call = _calls.get(name)
    if call is None:
        if not hasattr(lib(), symbol):
            raise RuntimeError(f"libmini_nccl.so was built without {source}")
        call = _calls[name] = getattr(ext(), name)
    return call


def plain_calls_only(name, *tensors):
    """What is active may record or replace the single operators: a tracer would keep the allocation of a result and not the kernel that fills it, so
    that what it recorded returns memory as it was found.  Modes that only look on (FLOP counters, selective checkpointing) do no harm.  The
    extension asks here for quantize_fp8 and gemm_fp8, where one of these may be the case: asked every time it would cost those a microsecond."""
    if torch.jit.is_tracing() or torch._C._are_functorch_transforms_active() or (
            torch._C._len_torch_dispatch_stack() and any(torch._C._get_dispatch_mode(mode) is not None for mode in _RECORDING)):
        raise RuntimeError(f"{name} has no rule for tracing, functional transforms and fake tensors")
    for t in tensors:
        if isinstance(t, torch.Tensor) and type(t) not in _PLAIN and (
                type(t).__torch_function__ is not torch._C._disabled_torch_function_impl or torch._C._dispatch_keys(t).has(torch._C.DispatchKey.Python)):
            raise TypeError(f"{name} has no rule for {type(t).__name__}, only for plain tensors")


def quantize_fp8(x, block_rows=1, transposed=False, stream=None):
    """``(q, scale)`` of a matrix ``x [M, K]`` (bf16, fp16 or fp32, unit inner stride): ``q [M, K]`` in e4m3 and fp32 scales
    such that ``x`` is about ``q * scale`` of its block.  ``block_rows=1``: blocks of 128 along a row, ``scale
    [M, ceil(K / 128)]``; ``block_rows=128``: blocks of 128 x 128, ``scale [ceil(M / 128), ceil(K / 128)]``.

    A scale is the smallest power of two (from 2^-126 on) for which the block's largest magnitude is at most 448 times it.  A
    block with an infinity or a NaN becomes NaN throughout.

    ``transposed=True``: ``(q, scale, qt, scale_t)``, with the transpose ``qt [K, M]`` as well, from one reading of ``x``; with
    ``block_rows=1`` it is quantised anew, in blocks of 128 along M (``scale_t [K, ceil(M / 128)]``).  K is at most 65535 * 128.
    Not differentiable."""
    return _call("quantize_fp8", "mncclQuantizeFp8", "csrc/kernels/fp8_quantize.cu")(x, block_rows, transposed, stream)


def gemm_fp8(a, a_scale, b, b_scale, out=None, out_dtype=None, bias=None, stream=None):
    """``out[M, N] = a[M, K] @ b[N, K].T (+ bias[N])`` of e4m3 operands with a scale for each block of 128 along K; a scale covers one
    row or 128 rows: ``a_scale [M or ceil(M / 128), ceil(K / 128)]``, ``b_scale`` likewise, any fp32 values and strides.

    A block's products are summed in fp32, multiplied by the fp32 product of its two scales (which has to stay in fp32's range: beyond it the block
    counts as infinite or NaN, below it as 0) and added up in fp32; with the bias added, one rounding to ``out``'s type (bf16 by
    default, fp16 or fp32).  ``bias`` has that type.  Operands have rows that start on 16 bytes.  Not differentiable."""
    return _call("gemm_fp8", "mncclGemmFp8", "csrc/kernels/gemm_fp8.cu")(a, a_scale, b, b_scale, out, out_dtype, bias, stream)


def no_tangent(t):
    """Whether a tensor carries no forward-mode tangent."""
    return torch.autograd.forward_ad._current_level < 0 or torch.autograd.forward_ad.unpack_dual(t).tangent is None


def linear_fp8(x, weight, bias=None):
    """``F.linear(x, weight, bias)`` with 8-bit products: ``x [..., K]`` is quantised in blocks of 128 along K, ``weight [N, K]`` in
    blocks of 128 x 128, the result has their type (bf16, fp16 or fp32, one for all; under autocast, its type).

    Differentiable once, straight through the roundings: with ``Q`` for quantisation along the summed dimension, the gradients
    are ``dx = Q(dy) Q(weight)`` (the forward pass's 8-bit weight), ``dweight = Q(dy).T Q(x)`` with blocks along the tokens, and
    ``dbias`` the fp32 sum of ``dy``.  What is kept for the backward pass is in 8 bits.

    All three refuse to be traced or transformed, and tensor subclasses with rules of their own."""
    plain_calls_only("linear_fp8", x, weight, bias)
    if torch.is_autocast_enabled("cuda"):
        to = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(to), weight.to(to), None if bias is None else bias.to(to)
    for t, name in ((x, "x"), (weight, "weight"), (bias, "bias")):
        if t is None and name == "bias":
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _FLOATS:
            raise TypeError(f"{name} must be a CUDA tensor in bf16, fp16 or fp32")
        if t.dtype != x.dtype or t.device != x.device:
            raise TypeError(f"{name} must have x's type and be on its GPU")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or (bias is not None and tuple(bias.shape) != (weight.shape[0],)):
        raise ValueError("shapes: x [..., K], weight [N, K], bias [N]")
    if weight.shape[1] == 0:
        raise ValueError("a layer without input features")
    if x.numel() // x.shape[-1] > _MOST_ROWS or max(weight.shape) > _MOST_COLUMNS:
        raise ValueError(f"at most {_MOST_ROWS} tokens and {_MOST_COLUMNS} features")
    if not all(no_tangent(t) for t in (x, weight, bias) if t is not None):
        raise RuntimeError("linear_fp8 has no rule for forward-mode differentiation")
    return _call("linear_fp8", "mncclGemmFp8", "csrc/kernels/gemm_fp8.cu")(x, weight, bias)
