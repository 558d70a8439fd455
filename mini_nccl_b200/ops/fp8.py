"""8-bit floating point (e4m3) with a scale for each block of 128: quantisation, products on the Blackwell tensor cores,
and a linear layer whose three products of a training step run in 8 bits.

Activations and gradients have a scale for each 128 elements of a row, weights for each 128 x 128 elements.  The scales that
:func:`quantize_fp8` chooses are powers of two (csrc/kernels/fp8_quantize.cu says why); :func:`gemm_fp8` takes any fp32
scales, such as a checkpoint's.  Like :func:`gemm_bf16` these fail loudly where the native kernels are missing."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .._lib import lib

BLOCK = 128
E4M3 = torch.float8_e4m3fn
_CODES = {torch.float16: 6, torch.float32: 7, torch.bfloat16: 9}
_MOST = 2**31 - 2**16   # rows and columns of a matrix: indices are 32-bit, elements are addressed with 64


def _blocks(n):
    return -(-n // BLOCK)


def _padded(n):
    return -(-n // 16) * 16


def _check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} failed with code {rc}")


class _on:
    """The GPU and the stream that a call runs on: the tensors' GPU, and `stream` or that GPU's current one.  What is
    allocated inside belongs to that stream."""

    def __init__(self, device, stream):
        if stream is not None and stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the tensors are on {device}")
        self.with_ = []
        if device.index != torch.cuda.current_device():
            self.with_.append(torch.cuda.device(device))
        if stream is not None:
            self.with_.append(torch.cuda.stream(stream))

    def __enter__(self):
        for w in self.with_:
            w.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *what):
        for w in reversed(self.with_):
            w.__exit__(*what)


def _matrix(t, name, dtypes):
    """(rows, columns, row stride) of a matrix the kernels can read."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {', '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if t.dim() != 2 or max(t.shape) > _MOST:
        raise ValueError(f"{name} must be a matrix of at most {_MOST} rows and columns")
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} needs a unit inner stride")
    ld = t.stride(0) if rows > 1 else _padded(cols)
    if ld < cols:
        raise ValueError(f"{name}'s rows overlap")
    return rows, cols, ld


def _quantize(x, block_rows, transposed, stream=None):
    """Buffers with padded rows, [M, padded K] and [K, padded M], and scales as the kernels write them."""
    M, K, ld = _matrix(x, "x", _CODES)
    if block_rows not in (1, BLOCK):
        raise ValueError("block_rows must be 1 or 128")
    L = lib()
    if not hasattr(L, "mncclQuantizeFp8"):
        raise RuntimeError("libmini_nccl.so was built without csrc/kernels/fp8_quantize.cu")
    with _on(x.device, stream) as s:
        q = torch.empty((M, _padded(K)), dtype=E4M3, device=x.device)
        scale = torch.empty((_blocks(K), M) if block_rows == 1 else (_blocks(M), _blocks(K)), dtype=torch.float32, device=x.device)
        qt = scale_t = None
        if transposed:
            qt = torch.empty((K, _padded(M)), dtype=E4M3, device=x.device)
            if block_rows == 1:
                scale_t = torch.empty((_blocks(M), K), dtype=torch.float32, device=x.device)
        if M and K:
            _check(L.mncclQuantizeFp8(x.data_ptr(), _CODES[x.dtype], ld, M, K, block_rows, q.data_ptr(), q.shape[1], scale.data_ptr(),
                                      qt.data_ptr() if transposed else None, qt.shape[1] if transposed else 0,
                                      scale_t.data_ptr() if scale_t is not None else None, s), "mncclQuantizeFp8")
    return q, scale, qt, scale_t


def quantize_fp8(x, block_rows=1, transposed=False, stream=None):
    """``(q, scale)`` of a matrix ``x [M, K]`` (bf16, fp16 or fp32, unit inner stride): ``q [M, K]`` in e4m3 and fp32 scales
    such that ``x`` is about ``q * scale`` of its block.  ``block_rows=1``: blocks of 128 along a row, ``scale
    [M, ceil(K / 128)]``; ``block_rows=128``: blocks of 128 x 128, ``scale [ceil(M / 128), ceil(K / 128)]``.

    A scale is the smallest power of two (from 2^-126 on) for which the block's largest magnitude is at most 448 times it.  A
    block with an infinity or a NaN becomes NaN throughout.

    ``transposed=True``: ``(q, scale, qt, scale_t)``, with the transpose ``qt [K, M]`` as well, from one reading of ``x``; with
    ``block_rows=1`` it is quantised anew, in blocks of 128 along M (``scale_t [K, ceil(M / 128)]``).  Not differentiable."""
    q, scale, qt, scale_t = _quantize(x, block_rows, transposed, stream)
    M, K = x.shape
    out = (q[:, :K], scale.t() if block_rows == 1 else scale)
    return out if not transposed else (*out, qt[:, :M], scale_t.t() if block_rows == 1 else scale.t())


def _scale(t, name, rows, K, device):
    """(row stride, block stride, rows of a scale) of the scales of an operand [rows, K]."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != device:
        raise TypeError(f"{name} must be an fp32 tensor on {device}")
    if t.dim() != 2 or t.shape[1] != _blocks(K) or t.shape[0] not in (rows, _blocks(rows)):
        raise ValueError(f"{name} must be [{rows} or {_blocks(rows)}, {_blocks(K)}], not {list(t.shape)}")
    return t.stride(0), t.stride(1), 1 if t.shape[0] == rows else BLOCK


def _operand(t, name):
    rows, cols, ld = _matrix(t, name, (E4M3,))
    if t.numel() and (t.data_ptr() % 16 or ld % 16):
        raise ValueError(f"{name}'s rows must start on 16 bytes (quantize_fp8 lays them out so)")
    return rows, cols, ld


def gemm_fp8(a, a_scale, b, b_scale, out=None, out_dtype=None, bias=None, stream=None):
    """``out[M, N] = a[M, K] @ b[N, K].T (+ bias[N])`` of e4m3 operands with a scale for each block of 128 along K; a scale covers one
    row or 128 rows: ``a_scale [M or ceil(M / 128), ceil(K / 128)]``, ``b_scale`` likewise, any fp32 values and strides.

    A block's products are summed in fp32, scaled and added up in fp32; with the bias added, one rounding to ``out``'s type (bf16 by
    default, fp16 or fp32).  ``bias`` has that type.  Operands have rows that start on 16 bytes.  Not differentiable."""
    M, K, lda = _operand(a, "a")
    N, Kb, ldb = _operand(b, "b")
    if K != Kb or b.device != a.device:
        raise ValueError("shapes: a [M, K], b [N, K], on one GPU")
    sa = _scale(a_scale, "a_scale", M, K, a.device)
    sb = _scale(b_scale, "b_scale", N, K, a.device)
    L = lib()
    if not hasattr(L, "mncclGemmFp8"):
        raise RuntimeError("libmini_nccl.so was built without csrc/kernels/gemm_fp8.cu")
    if out is not None and out_dtype not in (None, out.dtype):
        raise ValueError("out has another type than out_dtype")
    with _on(a.device, stream) as s:
        if out is None:
            out = torch.empty((M, N), dtype=torch.bfloat16 if out_dtype is None else out_dtype, device=a.device)
        if tuple(out.shape) != (M, N) or out.device != a.device:
            raise ValueError("out must be [M, N] on the operands' GPU")
        ldc = _matrix(out, "out", _CODES)[2]
        if bias is not None and (bias.dtype != out.dtype or bias.device != a.device or tuple(bias.shape) != (N,) or (N > 1 and bias.stride(0) != 1)):
            raise ValueError("bias must be [N], dense, of out's type and on its GPU")
        if K == 0:
            return out.zero_() if bias is None else out.copy_(bias.detach().expand(M, N))
        if M and N:
            _check(L.mncclGemmFp8(a.data_ptr(), lda, a_scale.data_ptr(), *sa, b.data_ptr(), ldb, b_scale.data_ptr(), *sb, out.data_ptr(), ldc,
                                  _CODES[out.dtype], bias.data_ptr() if bias is not None else None, M, N, K, s), "mncclGemmFp8")
    return out


def _rows(t, cols):
    """``t [..., cols]`` as a matrix that the quantisation reads (a copy only where the strides need one)."""
    t = t.detach().reshape(-1, cols)
    return t if (cols <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= cols) else t.contiguous()


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        N, K = weight.shape
        want_x, want_w = ctx.needs_input_grad[:2]
        rows = _rows(x, K)
        q, scale, qt, scale_t = _quantize(rows, 1, want_w)
        w, w_scale, wt, _ = _quantize(_rows(weight, K), BLOCK, want_x)
        y = gemm_fp8(q[:, :K], scale.t(), w[:, :K], w_scale, out_dtype=x.dtype, bias=None if bias is None else bias.detach().contiguous())
        # the padded buffers: a saved-tensor hook may hand back a dense copy of what it is given
        ctx.save_for_backward(qt, scale_t, wt, w_scale if want_x else None)
        ctx.shape, ctx.sizes = x.shape, (rows.shape[0], N, K)
        return y.view(*x.shape[:-1], N)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        xt, xt_scale, wt, w_scale = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad
        T, N, K = ctx.sizes
        g = _rows(grad, N)
        dx = dw = None
        if want_x or want_w:
            q, scale, qt, scale_t = _quantize(g, 1, want_w)
        if want_x:
            dx = gemm_fp8(q[:, :N], scale.t(), wt[:, :N], w_scale.t(), out_dtype=grad.dtype).view(ctx.shape)
        if want_w:
            dw = gemm_fp8(qt[:, :T], scale_t.t(), xt[:, :T], xt_scale.t(), out_dtype=grad.dtype)
        return dx, dw, g.float().sum(0).to(grad.dtype) if want_b else None


def linear_fp8(x, weight, bias=None):
    """``F.linear(x, weight, bias)`` with 8-bit products: ``x [..., K]`` is quantised in blocks of 128 along K, ``weight [N, K]`` in
    blocks of 128 x 128, the result has their type (bf16, fp16 or fp32, one for all; under autocast, its type).

    Differentiable once, straight through the roundings: with ``Q`` for quantisation along the summed dimension, the gradients
    are ``dx = Q(dy) Q(weight)`` (the forward pass's 8-bit weight), ``dweight = Q(dy).T Q(x)`` with blocks along the tokens, and
    ``dbias`` the fp32 sum of ``dy``.  What is kept for the backward pass is in 8 bits."""
    if torch.is_autocast_enabled("cuda"):
        to = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(to), weight.to(to), None if bias is None else bias.to(to)
    for t, name in ((x, "x"), (weight, "weight"), (bias, "bias")):
        if t is None and name == "bias":
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _CODES:
            raise TypeError(f"{name} must be a CUDA tensor in bf16, fp16 or fp32")
        if t.dtype != x.dtype or t.device != x.device:
            raise TypeError(f"{name} must have x's type and be on its GPU")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or (bias is not None and tuple(bias.shape) != (weight.shape[0],)):
        raise ValueError("shapes: x [..., K], weight [N, K], bias [N]")
    if weight.shape[1] == 0:
        raise ValueError("a layer without input features")
    return _LinearFp8.apply(x, weight, bias)
