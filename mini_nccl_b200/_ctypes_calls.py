"""The calls of the PyTorch extension (csrc/torch/ext.cpp) through ctypes, with the same arguments, results and
errors: for a PyTorch without CUDA, against which the extension cannot be built, and wherever else it is missing.
About 8 us slower per call."""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

_CODES = {torch.int8: 0, torch.uint8: 1, torch.int32: 2, torch.int64: 4, torch.float16: 6, torch.float32: 7, torch.float64: 8,
          torch.bfloat16: 9}
_CODES.update({getattr(torch, name): code for name, code in (("uint32", 3), ("uint64", 5)) if hasattr(torch, name)})


def _stream(stream) -> int:
    if stream is None:
        return torch.cuda.current_stream().cuda_stream if torch.cuda.is_available() else 0
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _tensor(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    return t


def _bf16(*tensors):
    return all(t.dtype == torch.bfloat16 for t in tensors)


def all_reduce(lib, comm, tensor, out, wire_dtype, op, scale, algo, stream):
    out = _tensor(tensor, "tensor") if out is None else _tensor(out, "out")
    if not tensor.is_contiguous() or not out.is_contiguous():
        raise ValueError("all_reduce needs contiguous tensors")
    if out.numel() != tensor.numel():
        raise ValueError("size mismatch")
    if wire_dtype is not None and not isinstance(wire_dtype, torch.dtype):
        raise TypeError("wire_dtype must be a torch dtype")
    wire = wire_dtype if wire_dtype is not None else (out.dtype if tensor.dtype == out.dtype else torch.bfloat16)
    if not {tensor.dtype, out.dtype, wire} <= _CODES.keys():
        raise TypeError("unsupported dtype")
    return lib.mncclAllReduceEx(tensor.data_ptr(), _CODES[tensor.dtype], out.data_ptr(), _CODES[out.dtype], _CODES[wire], tensor.numel(),
                                op, float(scale), algo, comm, _stream(stream))


def gemm(lib, a, b, out, out_dtype, stream):
    if not _bf16(_tensor(a, "a"), _tensor(b, "b")):
        raise TypeError("gemm_bf16 needs bf16 operands")
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1]:
        raise ValueError("shapes: a [M, K], b [N, K]")
    if a.stride(1) != 1 or b.stride(1) != 1:
        raise ValueError("operands need a unit inner stride")
    (M, K), N = a.shape, b.shape[0]
    if out is None:
        if out_dtype is not None and not isinstance(out_dtype, torch.dtype):
            raise TypeError("out_dtype must be a torch dtype")
        out = torch.empty((M, N), dtype=out_dtype or torch.bfloat16, device=a.device)
    if _tensor(out, "out").dtype not in (torch.bfloat16, torch.float32) or tuple(out.shape) != (M, N) or out.stride(1) != 1:
        raise ValueError("out must be [M, N] bf16 or fp32 with a unit inner stride")
    rc = lib.mncclGemmBf16(a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, a.stride(0), b.stride(0), out.stride(0),
                           1 if out.dtype == torch.float32 else 0, _stream(stream))
    if rc != 0:
        raise RuntimeError(f"mncclGemmBf16 failed with code {rc}")
    return out


def _error(lib, comm) -> int:
    e = C.c_int()
    rc = lib.mncclCommGetAsyncError(comm, C.byref(e))
    return rc if rc != 0 else e.value


def _pointers(address):
    return C.cast(C.c_void_p(address), C.POINTER(C.c_void_p))


def _bytes(address):
    return C.cast(C.c_void_p(address), C.c_char_p)


def gemm_rs(lib, comm, a, b, out, stream, workspace):
    M, N, rank, ranks, stage, flags, state, handle, handle_bytes = workspace
    _tensor(a, "a"), _tensor(b, "b")
    if a.dim() != 2 or b.dim() != 2 or a.shape[0] != M or b.shape[0] != N or a.shape[1] != b.shape[1]:
        raise ValueError("shape mismatch")
    if not _bf16(a, b) or a.stride(1) != 1 or b.stride(1) != 1:
        raise TypeError("bf16 operands with a unit inner stride")
    if out is None:
        out = torch.empty((M // ranks, N), dtype=torch.bfloat16, device=a.device)
    s, e = _stream(stream), _error(lib, comm)
    if e != 0:
        return e
    rc = lib.mncclGemmReduceScatterBf16Comm(a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, a.shape[1], a.stride(0), b.stride(0),
                                            out.stride(0), rank, ranks, _pointers(stage), _pointers(flags), state,
                                            _bytes(handle), handle_bytes, s)
    if rc != 0:
        raise RuntimeError(f"mncclGemmReduceScatterBf16 failed with code {rc}")
    return out


def ag_gemm(lib, comm, n_comm_ctas, b, out, stream, swiglu, workspace):
    M, K, rank, ranks, xg, ready, bar, state, handle, handle_bytes = workspace
    if not _bf16(_tensor(b, "b")) or b.dim() != 2 or b.shape[1] != K or b.stride(1) != 1:
        raise TypeError("b must be bf16 [N, K] with a unit inner stride")
    N = b.shape[0]
    if swiglu and N % 32:
        raise ValueError("SwiGLU in the epilogue needs N a multiple of 32")
    n_out = N // 2 if swiglu else N
    if out is None:
        out = torch.empty((M, n_out), dtype=torch.bfloat16, device=b.device)
    if tuple(_tensor(out, "out").shape) != (M, n_out) or out.dtype != torch.bfloat16 or out.stride(1) != 1:
        raise ValueError(f"out must be bf16 [{M}, {n_out}] with a unit inner stride")
    s, e = _stream(stream), _error(lib, comm)
    if e != 0:
        return e
    rc = lib.mncclAllGatherGemmBf16Comm(_pointers(xg), b.data_ptr(), out.data_ptr(), M, N, K, K, b.stride(0), out.stride(0), rank, ranks,
                                        _pointers(ready), _pointers(bar), state, n_comm_ctas, 1 if swiglu else 0, _bytes(handle),
                                        handle_bytes, s)
    if rc != 0:
        raise RuntimeError(f"all-gather->GEMM kernel failed with code {rc}")
    return out


# ---- 8-bit operators and distillation

_BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_FLOATS = {torch.float16: 6, torch.float32: 7, torch.bfloat16: 9}
_MOST = 2**31 - 1 - 2**16   # rows and columns of a matrix: indices are 32-bit, elements are addressed with 64
_MOST_COLUMNS = 65535 * _BLOCK   # of what mncclQuantizeFp8 takes


def _blocks(n):
    return -(-n // _BLOCK)


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
        self.with_ = [torch.cuda.device(device)] if stream is None else [torch.cuda.device(device), torch.cuda.stream(stream)]

    def __enter__(self):
        for w in self.with_:
            w.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *what):
        for w in reversed(self.with_):
            w.__exit__(*what)


def _matrix(t, name, dtypes):
    """(rows, columns, row stride) of a matrix the kernels can read."""
    if not _tensor(t, name).is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} is of a type that this call does not take: {t.dtype}")
    if t.dim() != 2 or max(t.shape) > _MOST:
        raise ValueError(f"{name} must be a matrix of at most {_MOST} rows and columns")
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} needs a unit inner stride")
    if t.is_neg():
        raise ValueError(f"{name} is a view of numbers with the other sign (resolve_neg() makes them its own)")
    ld = t.stride(0) if rows > 1 else _padded(cols)
    if ld < cols:
        raise ValueError(f"{name}'s rows overlap")
    return rows, cols, ld


def _quantize(lib, x, block_rows, transposed, sums, s):
    M, K, ld = _matrix(x, "x", _FLOATS)
    q = torch.empty((M, _padded(K)), dtype=_E4M3, device=x.device)
    scale = torch.empty((_blocks(K), M) if block_rows == 1 else (_blocks(M), _blocks(K)), dtype=torch.float32, device=x.device)
    qt = torch.empty((K, _padded(M)), dtype=_E4M3, device=x.device) if transposed else None
    scale_t, sums = (torch.empty((_blocks(M), K), dtype=torch.float32, device=x.device) if want else None
                     for want in (transposed and block_rows == 1, transposed and sums))
    if M and K:
        _check(lib.mncclQuantizeFp8(x.data_ptr(), _FLOATS[x.dtype], ld, M, K, block_rows, q.data_ptr(), q.shape[1], scale.data_ptr(),
                                    qt.data_ptr() if transposed else None, qt.shape[1] if transposed else 0,
                                    *(t.data_ptr() if t is not None else None for t in (scale_t, sums)), s), "mncclQuantizeFp8")
    return q, scale, qt, scale_t, sums


def _plain_calls(name, *tensors):
    from .ops.fp8 import plain_calls_only

    plain_calls_only(name, *tensors)


def quantize_fp8(lib, x, block_rows, transposed, stream):
    _plain_calls("quantize_fp8", x)
    _matrix(x, "x", _FLOATS)
    if block_rows not in (1, _BLOCK):
        raise ValueError("block_rows must be 1 or 128")
    if x.shape[1] > _MOST_COLUMNS:
        raise ValueError(f"x must have at most {_MOST_COLUMNS} columns")
    with _on(x.device, stream) as s:
        q, scale, qt, scale_t, _ = _quantize(lib, x, block_rows, transposed, False, s)
    M, K = x.shape
    out = (q[:, :K], scale.t() if block_rows == 1 else scale)
    return out if not transposed else (*out, qt[:, :M], scale_t.t() if block_rows == 1 else scale.t())


def _operand(t, name):
    rows, cols, ld = _matrix(t, name, (_E4M3,))
    if t.numel() and (t.data_ptr() % 16 or ld % 16):
        raise ValueError(f"{name}'s rows must start on 16 bytes (quantize_fp8 lays them out so)")
    return rows, cols, ld


def _scales(t, name, rows, K, device):
    """(row stride, block stride, rows of a scale) of the scales of an operand [rows, K]."""
    if _tensor(t, name).dtype != torch.float32 or t.device != device:
        raise TypeError(f"{name} must be an fp32 tensor on the operands' GPU")
    if t.is_neg():
        raise ValueError(f"{name} is a view of numbers with the other sign (resolve_neg() makes them its own)")
    if t.dim() != 2 or t.shape[1] != _blocks(K) or t.shape[0] not in (rows, _blocks(rows)):
        raise ValueError(f"{name} must be [{rows} or {_blocks(rows)}, {_blocks(K)}]")
    return t.stride(0), t.stride(1), 1 if t.shape[0] == rows else _BLOCK


def gemm_fp8(lib, a, a_scale, b, b_scale, out, out_dtype, bias, stream):
    _plain_calls("gemm_fp8", a, a_scale, b, b_scale, out, bias)
    M, K, lda = _operand(a, "a")
    N, Kb, ldb = _operand(b, "b")
    if K != Kb or b.device != a.device:
        raise ValueError("shapes: a [M, K], b [N, K], on one GPU")
    sa = _scales(a_scale, "a_scale", M, K, a.device)
    sb = _scales(b_scale, "b_scale", N, K, a.device)
    if out_dtype is not None and not isinstance(out_dtype, torch.dtype):
        raise TypeError("out_dtype must be a torch dtype")
    given = out is not None
    with _on(a.device, stream) as s:
        if not given:
            out = torch.empty((M, N), dtype=out_dtype or torch.bfloat16, device=a.device)
        elif out_dtype not in (None, _tensor(out, "out").dtype):
            raise ValueError("out has another type than out_dtype")
        if tuple(out.shape) != (M, N) or out.device != a.device:
            raise ValueError("out must be [M, N] on the operands' GPU")
        ldc = _matrix(out, "out", _FLOATS)[2]
        if bias is not None and (_tensor(bias, "bias").dtype != out.dtype or bias.device != a.device or tuple(bias.shape) != (N,)
                                 or (N > 1 and bias.stride(0) != 1) or bias.is_neg()):
            raise ValueError("bias must be [N], dense, of out's type and on its GPU")
        if K == 0:
            with torch.no_grad():
                return out.zero_() if bias is None else out.copy_(bias.expand(M, N))
        if M and N:
            _check(lib.mncclGemmFp8(a.data_ptr(), lda, a_scale.data_ptr(), *sa, b.data_ptr(), ldb, b_scale.data_ptr(), *sb, out.data_ptr(), ldc,
                                    _FLOATS[out.dtype], bias.data_ptr() if bias is not None else None, M, N, K, s), "mncclGemmFp8")
            if given and not out.is_inference():
                torch.autograd.graph.increment_version(out)
    return out


def _rows(t, cols):
    """``t [..., cols]`` as a matrix that the kernels can read (a copy only where the strides need one, or where ``t`` is a view of numbers with the other sign)."""
    t = t.detach().resolve_neg()
    t = t if t.dim() == 2 else t.reshape(t.numel() // cols if cols else 0, cols)
    return t if (cols <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= cols) else t.contiguous()


def _linear_forward(lib, x, weight, bias, want_x, want_w):
    """y, and for the backward pass x^T and its scales, weight^T and the weight's scales, each None where it is not wanted."""
    N, K = weight.shape
    rows, w = _rows(x, K), _rows(weight, K)
    with _on(x.device, None) as s:
        q, scale, qt, scale_t, _ = _quantize(lib, rows, 1, want_w, False, s)
        wq, w_scale, wt, _, _ = _quantize(lib, w, _BLOCK, want_x, False, s)
    y = gemm_fp8(lib, q[:, :K], scale.t(), wq[:, :K], w_scale, None, x.dtype, None if bias is None else bias.detach().resolve_neg().contiguous(), None)
    return y.view(*x.shape[:-1], N), qt, scale_t, wt, w_scale if want_x else None


def _linear_backward(lib, grad, xt, xt_scale, wt, w_scale, K, want_bias):
    N = grad.shape[-1]
    g = _rows(grad, N)
    T = g.shape[0]
    dx = dw = db = None
    with _on(g.device, None) as s:
        q, scale, qt, scale_t, sums = _quantize(lib, g, 1, xt is not None or want_bias, want_bias, s)
        if want_bias:
            db = torch.zeros(N, dtype=g.dtype, device=g.device)
            if T:
                _check(lib.mncclSumBlocks(sums.data_ptr(), sums.shape[0], N, db.data_ptr(), _FLOATS[db.dtype], s), "mncclSumBlocks")
    if wt is not None:
        dx = gemm_fp8(lib, q[:, :N], scale.t(), wt[:, :N], w_scale.t(), None, g.dtype, None, None)
    if xt is not None:
        dw = gemm_fp8(lib, qt[:, :T], scale_t.t(), xt[:, :T], xt_scale.t(), None, g.dtype, None, None)
    return dx, dw, db


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lib, x, weight, bias, grad):
        want_x, want_w = (grad and want for want in ctx.needs_input_grad[1:3])
        y, *kept = _linear_forward(lib, x, weight, bias, want_x, want_w)
        ctx.save_for_backward(*kept)
        ctx.lib, ctx.shape = lib, x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad.shape[-1] == 0:   # a layer without output features
            shapes = (ctx.shape, (0, ctx.shape[-1]), (0,))
            return (None, *(grad.new_zeros(shape) if want else None for shape, want in zip(shapes, ctx.needs_input_grad[1:4])), None)
        dx, dw, db = _linear_backward(ctx.lib, grad, *ctx.saved_tensors, ctx.shape[-1], ctx.needs_input_grad[3])
        return None, None if dx is None else dx.view(ctx.shape), dw, db, None


def linear_fp8(lib, x, weight, bias):
    return _LinearFp8.apply(lib, x, weight, bias, torch.is_grad_enabled())


def distill_forward(lib, logits, ids, top, tau, reduction):
    rows = _rows(logits, logits.shape[-1])
    (T, V), K = rows.shape, ids.shape[1]
    with _on(rows.device, None) as s:
        empty = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=rows.device)  # noqa: E731
        p, stats, counts, row_loss, loss, tokens = empty(T, K), empty(T, 2), empty(T, dtype=torch.int32), empty(*logits.shape[:-1]), empty(), empty()
        _check(lib.mncclDistillForward(rows.data_ptr(), _FLOATS[rows.dtype], rows.stride(0) if T > 1 else _padded(V), T, V, ids.data_ptr(), top.data_ptr(), K, tau,
                                       p.data_ptr(), stats.data_ptr(), row_loss.data_ptr(), counts.data_ptr(), *(loss.data_ptr() if reduction == r else None for r in (1, 2)), tokens.data_ptr(), s),
               "mncclDistillForward")
    return row_loss if reduction == 0 else loss, p, stats, counts, tokens


def distill_backward(lib, logits, ids, p, stats, counts, tokens, tau, grad):
    rows, grad = _rows(logits, logits.shape[-1]), grad.resolve_neg().contiguous()
    T, V = rows.shape
    per = 16 // rows.element_size()
    with _on(rows.device, None) as s:
        d = torch.empty((T, -(-V // per) * per if rows.stride(0) != V else V), dtype=rows.dtype, device=rows.device)
        _check(lib.mncclDistillBackward(rows.data_ptr(), _FLOATS[rows.dtype], rows.stride(0) if T > 1 else _padded(V), T, V, ids.data_ptr(), p.data_ptr(), ids.shape[1],
                                        tau, stats.data_ptr(), counts.data_ptr(), grad.data_ptr(), 1 if grad.dim() else 0,
                                        tokens.data_ptr() if tokens is not None else None, d.data_ptr(), d.shape[1], s), "mncclDistillBackward")
    return d[:, :V].view(logits.shape)


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lib, logits, ids, top, tau, reduction, again):
        loss, *kept = distill_forward(lib, logits, ids, top, tau, reduction)
        ctx.save_for_backward(logits, ids, top, *kept)
        ctx.rest = lib, tau, reduction, again
        return loss

    @staticmethod
    def backward(ctx, grad):
        logits, ids, top, p, stats, counts, tokens = ctx.saved_tensors
        lib, tau, reduction, again = ctx.rest
        if torch.is_grad_enabled():
            d = again(logits, ids, top, tau, reduction, grad)
        else:
            d = distill_backward(lib, logits, ids, p, stats, counts, tokens if reduction == 2 else None, tau, grad)
        return None, d, None, None, None, None, None


def distillation(lib, logits, ids, top, tau, reduction, again):
    return _Distillation.apply(lib, logits, ids, top, tau, reduction, again)


class Calls:
    """The extension's functions, bound to a loaded library."""

    def __init__(self, lib):
        from functools import partial

        for f in (all_reduce, gemm, gemm_rs, ag_gemm, quantize_fp8, gemm_fp8, linear_fp8, distill_forward, distill_backward, distillation):
            setattr(self, f.__name__, partial(f, lib))
