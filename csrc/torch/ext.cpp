// The calls of the Python binding that are made often enough for their own cost to matter, as a CPython
// extension on PyTorch's C++ API.
//
// Measured per call (8 KiB AllReduce on one GPU, host time): 12.8 us through ctypes, of which 3.4 us were
// torch.cuda.current_stream(), 1.3 us the conversion of twelve ctypes arguments, 2 us attribute reads of
// the tensors and 5 us the library and the launch.  Here a tensor is unpacked in place and the library is
// called through the address that the ctypes binding has already loaded (bind()), so MINI_NCCL_LIB selects
// the library as before and nothing links against it.  Arguments that can be wrong are still checked here,
// with the messages and exception types of the Python layer they come from.
//
// The GIL is released around every library call: the network plane's AllReduce blocks, and the ranks of a
// program may be threads of one process.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <initializer_list>
#include <optional>

#include "mini_nccl_api.h"
#include "mini_nccl_ops.h"

namespace {

struct Library {
  decltype(&mncclAllReduceEx) all_reduce_ex = nullptr;
  decltype(&mncclCommGetAsyncError) async_error = nullptr;
  int (*gemm)(const void*, const void*, void*, int, int, int, int, int, int, int, cudaStream_t) = nullptr;
  int (*gemm_rs)(const void*, const void*, void*, int, int, int, int, int, int, int, int, void* const*, void* const*, uint32_t*,
                 const void*, size_t, cudaStream_t) = nullptr;
  int (*ag_gemm)(void* const*, const void*, void*, int, int, int, int, int, int, int, int, void* const*, void* const*, uint32_t*, int,
                 int, const void*, size_t, cudaStream_t) = nullptr;
  decltype(&mncclQuantizeFp8) quantize_fp8 = nullptr;
  decltype(&mncclSumBlocks) sum_blocks = nullptr;
  decltype(&mncclGemmFp8) gemm_fp8 = nullptr;
  decltype(&mncclDistillForward) distill_forward = nullptr;
  decltype(&mncclDistillBackward) distill_backward = nullptr;
} lib;

// ncclDataType_t of a tensor's scalar type, -1 for a type the library does not have.
int type_code(at::ScalarType t) {
  switch (t) {
    case at::kChar: return ncclInt8;
    case at::kByte: return ncclUint8;
    case at::kInt: return ncclInt32;
    case at::kUInt32: return ncclUint32;
    case at::kLong: return ncclInt64;
    case at::kUInt64: return ncclUint64;
    case at::kHalf: return ncclFloat16;
    case at::kFloat: return ncclFloat;
    case at::kDouble: return ncclDouble;
    case at::kBFloat16: return ncclBfloat16;
    default: return -1;
  }
}

bool have_gpu() {
  static const bool have = c10::cuda::device_count() > 0;
  return have;
}

// None: the current stream (0 without a GPU); a stream object; or a raw handle.
bool stream_arg(PyObject* o, cudaStream_t* out) {
  if (o == Py_None) {
    *out = have_gpu() ? c10::cuda::getCurrentCUDAStream().stream() : nullptr;
    return true;
  }
  PyObject* raw = PyLong_Check(o) ? Py_NewRef(o) : PyObject_GetAttrString(o, "cuda_stream");
  if (!raw) {
    PyErr_Clear();
    raw = PyNumber_Long(o);
    if (!raw) return false;
  }
  *out = reinterpret_cast<cudaStream_t>(PyLong_AsUnsignedLongLongMask(raw));
  Py_DECREF(raw);
  return !PyErr_Occurred();
}

const at::Tensor* tensor_arg(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a torch tensor", name);
    return nullptr;
  }
  return &THPVariable_Unpack(o);
}

bool arg_count(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
  return n == want;
}

// bind(all_reduce_ex, async_error, gemm, gemm_rs, ag_gemm, quantize_fp8, sum_blocks, gemm_fp8, distill_forward,
// distill_backward): addresses in the library that ctypes has loaded (all but the first two may be 0)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arg_count(n, 10)) return nullptr;
  lib.all_reduce_ex = reinterpret_cast<decltype(lib.all_reduce_ex)>(PyLong_AsVoidPtr(args[0]));
  lib.async_error = reinterpret_cast<decltype(lib.async_error)>(PyLong_AsVoidPtr(args[1]));
  lib.gemm = reinterpret_cast<decltype(lib.gemm)>(PyLong_AsVoidPtr(args[2]));
  lib.gemm_rs = reinterpret_cast<decltype(lib.gemm_rs)>(PyLong_AsVoidPtr(args[3]));
  lib.ag_gemm = reinterpret_cast<decltype(lib.ag_gemm)>(PyLong_AsVoidPtr(args[4]));
  lib.quantize_fp8 = reinterpret_cast<decltype(lib.quantize_fp8)>(PyLong_AsVoidPtr(args[5]));
  lib.sum_blocks = reinterpret_cast<decltype(lib.sum_blocks)>(PyLong_AsVoidPtr(args[6]));
  lib.gemm_fp8 = reinterpret_cast<decltype(lib.gemm_fp8)>(PyLong_AsVoidPtr(args[7]));
  lib.distill_forward = reinterpret_cast<decltype(lib.distill_forward)>(PyLong_AsVoidPtr(args[8]));
  lib.distill_backward = reinterpret_cast<decltype(lib.distill_backward)>(PyLong_AsVoidPtr(args[9]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// all_reduce(comm, tensor, out | None, wire_dtype | None, op, scale, algo, stream | None) -> ncclResult_t
PyObject* all_reduce(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arg_count(n, 8)) return nullptr;
  void* comm = PyLong_AsVoidPtr(args[0]);
  const at::Tensor* in = tensor_arg(args[1], "tensor");
  const at::Tensor* out = args[2] == Py_None ? in : tensor_arg(args[2], "out");
  if (!in || !out) return nullptr;
  if (!in->is_contiguous() || !out->is_contiguous()) {
    PyErr_SetString(PyExc_ValueError, "all_reduce needs contiguous tensors");
    return nullptr;
  }
  const int64_t count = in->numel();
  if (out->numel() != count) {
    PyErr_SetString(PyExc_ValueError, "size mismatch");
    return nullptr;
  }
  const int send_type = type_code(in->scalar_type()), recv_type = type_code(out->scalar_type());
  int wire_type = send_type == recv_type ? recv_type : static_cast<int>(ncclBfloat16);
  if (args[3] != Py_None) {
    if (!THPDtype_Check(args[3])) {
      PyErr_SetString(PyExc_TypeError, "wire_dtype must be a torch dtype");
      return nullptr;
    }
    wire_type = type_code(reinterpret_cast<THPDtype*>(args[3])->scalar_type);
  }
  if (send_type < 0 || recv_type < 0 || wire_type < 0) {
    PyErr_SetString(PyExc_TypeError, "unsupported dtype");
    return nullptr;
  }
  const long op = PyLong_AsLong(args[4]);
  const double scale = PyFloat_AsDouble(args[5]);
  const long algo = PyLong_AsLong(args[6]);
  cudaStream_t stream = nullptr;
  if (PyErr_Occurred() || !stream_arg(args[7], &stream)) return nullptr;
  const void* send = in->data_ptr();
  void* recv = out->data_ptr();
  ncclResult_t rc;
  Py_BEGIN_ALLOW_THREADS
  rc = lib.all_reduce_ex(send, static_cast<ncclDataType_t>(send_type), recv, static_cast<ncclDataType_t>(recv_type),
                         static_cast<ncclDataType_t>(wire_type), static_cast<size_t>(count), static_cast<ncclRedOp_t>(op), scale,
                         static_cast<mncclAlgo_t>(algo), static_cast<ncclComm_t>(comm), stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// gemm(a, b, out | None, out_dtype | None, stream | None) -> out; see ops/gemm.py
PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arg_count(n, 5)) return nullptr;
  const at::Tensor* a = tensor_arg(args[0], "a");
  const at::Tensor* b = tensor_arg(args[1], "b");
  if (!a || !b) return nullptr;
  if (a->scalar_type() != at::kBFloat16 || b->scalar_type() != at::kBFloat16) {
    PyErr_SetString(PyExc_TypeError, "gemm_bf16 needs bf16 operands");
    return nullptr;
  }
  if (a->dim() != 2 || b->dim() != 2 || a->size(1) != b->size(1)) {
    PyErr_SetString(PyExc_ValueError, "shapes: a [M, K], b [N, K]");
    return nullptr;
  }
  if (a->stride(1) != 1 || b->stride(1) != 1) {
    PyErr_SetString(PyExc_ValueError, "operands need a unit inner stride");
    return nullptr;
  }
  const int64_t M = a->size(0), K = a->size(1), N = b->size(0);
  at::Tensor fresh;
  const at::Tensor* out = nullptr;
  if (args[2] != Py_None) {
    out = tensor_arg(args[2], "out");
    if (!out) return nullptr;
  } else {
    at::ScalarType t = at::kBFloat16;
    if (args[3] != Py_None) {
      if (!THPDtype_Check(args[3])) {
        PyErr_SetString(PyExc_TypeError, "out_dtype must be a torch dtype");
        return nullptr;
      }
      t = reinterpret_cast<THPDtype*>(args[3])->scalar_type;
    }
    fresh = at::empty({M, N}, a->options().dtype(t));
    out = &fresh;
  }
  const at::ScalarType ot = out->scalar_type();
  if ((ot != at::kBFloat16 && ot != at::kFloat) || out->dim() != 2 || out->size(0) != M || out->size(1) != N || out->stride(1) != 1) {
    PyErr_SetString(PyExc_ValueError, "out must be [M, N] bf16 or fp32 with a unit inner stride");
    return nullptr;
  }
  cudaStream_t stream = nullptr;
  if (!stream_arg(args[4], &stream)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = lib.gemm(a->data_ptr(), b->data_ptr(), out->data_ptr(), static_cast<int>(M), static_cast<int>(N), static_cast<int>(K),
                static_cast<int>(a->stride(0)), static_cast<int>(b->stride(0)), static_cast<int>(out->stride(0)),
                ot == at::kFloat ? 1 : 0, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) {
    PyErr_Format(PyExc_RuntimeError, "mncclGemmBf16 failed with code %d", rc);
    return nullptr;
  }
  return fresh.defined() ? THPVariable_Wrap(fresh) : Py_NewRef(args[2]);
  END_HANDLE_TH_ERRORS
}

// What a fused kernel's Python object keeps for its calls, as a tuple of integers: (M, N or K, rank, ranks, address of
// the first and of the second array of peers' buffers, of the state words, address and length of the
// communicator's device handle, ...)
bool workspace_arg(PyObject* t, Py_ssize_t want, uintptr_t (&v)[10]) {
  if (!PyTuple_Check(t) || PyTuple_GET_SIZE(t) != want) {
    PyErr_SetString(PyExc_TypeError, "bad workspace tuple");
    return false;
  }
  for (Py_ssize_t i = 0; i < want; ++i) v[i] = PyLong_AsUnsignedLongLongMask(PyTuple_GET_ITEM(t, i));
  return !PyErr_Occurred();
}

// A communicator that has failed takes no more work: its error code, 0 when it is usable.
int comm_error(PyObject* comm) {
  ncclResult_t e = ncclSuccess;
  const ncclResult_t rc = lib.async_error(static_cast<ncclComm_t>(PyLong_AsVoidPtr(comm)), &e);
  return rc != ncclSuccess ? rc : e;
}

// gemm_rs(comm, a, b, out | None, stream | None, workspace) -> out, or the communicator's error code; see ops/fused.py
PyObject* gemm_rs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  uintptr_t w[10];
  if (!arg_count(n, 6) || !workspace_arg(args[5], 9, w)) return nullptr;
  const at::Tensor* a = tensor_arg(args[1], "a");
  const at::Tensor* b = tensor_arg(args[2], "b");
  if (!a || !b) return nullptr;
  const int64_t M = static_cast<int64_t>(w[0]), N = static_cast<int64_t>(w[1]), ranks = static_cast<int64_t>(w[3]);
  if (a->dim() != 2 || b->dim() != 2 || a->size(0) != M || b->size(0) != N || a->size(1) != b->size(1)) {
    PyErr_SetString(PyExc_ValueError, "shape mismatch");
    return nullptr;
  }
  if (a->scalar_type() != at::kBFloat16 || b->scalar_type() != at::kBFloat16 || a->stride(1) != 1 || b->stride(1) != 1) {
    PyErr_SetString(PyExc_TypeError, "bf16 operands with a unit inner stride");
    return nullptr;
  }
  at::Tensor fresh;
  if (args[3] == Py_None) fresh = at::empty({M / ranks, N}, a->options());
  const at::Tensor* out = args[3] == Py_None ? &fresh : tensor_arg(args[3], "out");
  cudaStream_t stream = nullptr;
  if (!out || !stream_arg(args[4], &stream)) return nullptr;
  if (const int e = comm_error(args[0])) return PyLong_FromLong(e);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = lib.gemm_rs(a->data_ptr(), b->data_ptr(), out->data_ptr(), static_cast<int>(M), static_cast<int>(N), static_cast<int>(a->size(1)),
                   static_cast<int>(a->stride(0)), static_cast<int>(b->stride(0)), static_cast<int>(out->stride(0)), static_cast<int>(w[2]),
                   static_cast<int>(ranks), reinterpret_cast<void* const*>(w[4]), reinterpret_cast<void* const*>(w[5]),
                   reinterpret_cast<uint32_t*>(w[6]), reinterpret_cast<const void*>(w[7]), w[8], stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) {
    PyErr_Format(PyExc_RuntimeError, "mncclGemmReduceScatterBf16 failed with code %d", rc);
    return nullptr;
  }
  return fresh.defined() ? THPVariable_Wrap(fresh) : Py_NewRef(args[3]);
  END_HANDLE_TH_ERRORS
}

// ag_gemm(comm, n_comm_ctas, b, out | None, stream | None, swiglu, workspace) -> out, or the communicator's error code
PyObject* ag_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  uintptr_t w[10];
  if (!arg_count(n, 7) || !workspace_arg(args[6], 10, w)) return nullptr;
  const at::Tensor* b = tensor_arg(args[2], "b");
  if (!b) return nullptr;
  const int64_t M = static_cast<int64_t>(w[0]), K = static_cast<int64_t>(w[1]);
  if (b->scalar_type() != at::kBFloat16 || b->dim() != 2 || b->size(1) != K || b->stride(1) != 1) {
    PyErr_SetString(PyExc_TypeError, "b must be bf16 [N, K] with a unit inner stride");
    return nullptr;
  }
  const int64_t N = b->size(0);
  const int swiglu = PyObject_IsTrue(args[5]), n_comm_ctas = static_cast<int>(PyLong_AsLong(args[1]));
  if (swiglu < 0 || PyErr_Occurred()) return nullptr;
  if (swiglu && N % 32 != 0) {
    PyErr_SetString(PyExc_ValueError, "SwiGLU in the epilogue needs N a multiple of 32");
    return nullptr;
  }
  const int64_t n_out = swiglu ? N / 2 : N;
  at::Tensor fresh;
  if (args[3] == Py_None) fresh = at::empty({M, n_out}, b->options());
  const at::Tensor* out = args[3] == Py_None ? &fresh : tensor_arg(args[3], "out");
  if (!out) return nullptr;
  if (out->dim() != 2 || out->size(0) != M || out->size(1) != n_out || out->scalar_type() != at::kBFloat16 || out->stride(1) != 1) {
    PyErr_Format(PyExc_ValueError, "out must be bf16 [%lld, %lld] with a unit inner stride", static_cast<long long>(M), static_cast<long long>(n_out));
    return nullptr;
  }
  cudaStream_t stream = nullptr;
  if (!stream_arg(args[4], &stream)) return nullptr;
  if (const int e = comm_error(args[0])) return PyLong_FromLong(e);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = lib.ag_gemm(reinterpret_cast<void* const*>(w[4]), b->data_ptr(), out->data_ptr(), static_cast<int>(M), static_cast<int>(N),
                   static_cast<int>(K), static_cast<int>(K), static_cast<int>(b->stride(0)), static_cast<int>(out->stride(0)),
                   static_cast<int>(w[2]), static_cast<int>(w[3]), reinterpret_cast<void* const*>(w[5]),
                   reinterpret_cast<void* const*>(w[6]), reinterpret_cast<uint32_t*>(w[7]), n_comm_ctas, swiglu,
                   reinterpret_cast<const void*>(w[8]), w[9], stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) {
    PyErr_Format(PyExc_RuntimeError, "all-gather->GEMM kernel failed with code %d", rc);
    return nullptr;
  }
  return fresh.defined() ? THPVariable_Wrap(fresh) : Py_NewRef(args[3]);
  END_HANDLE_TH_ERRORS
}

// ---- 8-bit operators and distillation (ops/fp8.py, ops/distill.py).  They run on their tensors' GPU, whichever is current, and on the given
// stream or that GPU's current one; what they allocate belongs to that stream.

constexpr int64_t kBlock = 128, kMost = 2147483647 - 65536, kMostColumns = 65535 * kBlock;   // kMostColumns: of what mncclQuantizeFp8 takes
int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }
int64_t padded(int64_t n) { return (n + 15) / 16 * 16; }

struct On {
  c10::cuda::OptionalCUDAGuard device;
  c10::cuda::OptionalCUDAStreamGuard stream;
  cudaStream_t raw = nullptr;
};
bool on(const at::Tensor& t, PyObject* stream, On* o) {
  if (stream == Py_None) {
    o->device.set_index(t.get_device());
    o->raw = c10::cuda::getCurrentCUDAStream().stream();
    return true;
  }
  int64_t v[3];
  const char* names[3] = {"stream_id", "device_index", "device_type"};
  for (int i = 0; i < 3; ++i) {
    PyObject* x = PyObject_GetAttrString(stream, names[i]);
    if (!x) return false;
    v[i] = PyLong_AsLongLong(x);
    Py_DECREF(x);
    if (PyErr_Occurred()) return false;
  }
  if (v[1] != t.get_device()) {
    PyErr_Format(PyExc_ValueError, "the stream is on cuda:%lld, the tensors are on cuda:%d", static_cast<long long>(v[1]), static_cast<int>(t.get_device()));
    return false;
  }
  o->stream.reset_stream(c10::Stream::unpack3(v[0], static_cast<c10::DeviceIndex>(v[1]), static_cast<c10::DeviceType>(v[2])));
  o->raw = c10::cuda::getCurrentCUDAStream().stream();
  return true;
}

// Whether nothing is active that may record or replace the single operators, and the arguments (None: left out) are plain tensors.  Where something is,
// ops/fp8.py says whether the call is refused.
bool plain_calls(const char* name, std::initializer_list<PyObject*> tensors) {
  bool plain = !torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
               !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
  for (PyObject* t : tensors) plain = plain && (t == Py_None || THPVariable_CheckExact(t));
  if (plain) return true;
  PyObject* rules = PyImport_ImportModule("mini_nccl_b200.ops.fp8");
  PyObject* rule = rules ? PyObject_GetAttrString(rules, "plain_calls_only") : nullptr;
  PyObject* args = rule ? PyTuple_New(static_cast<Py_ssize_t>(tensors.size()) + 1) : nullptr;
  PyObject* said = nullptr;
  if (args) {
    PyObject* who = PyUnicode_FromString(name);
    PyTuple_SET_ITEM(args, 0, who);
    Py_ssize_t i = 1;
    for (PyObject* t : tensors) PyTuple_SET_ITEM(args, i++, Py_NewRef(t));
    said = who ? PyObject_CallObject(rule, args) : nullptr;
  }
  for (PyObject* o : {rules, rule, args, said}) Py_XDECREF(o);
  return said != nullptr;
}

// fp16, fp32 and bf16, by the library's codes; -1 for another type
int float_code(const at::Tensor& t) {
  const int c = type_code(t.scalar_type());
  return c == ncclFloat16 || c == ncclFloat || c == ncclBfloat16 ? c : -1;
}

// Whether `t` is a matrix the kernels can read, and its row stride.
bool matrix(const at::Tensor& t, const char* name, bool right_type, int64_t* ld) {
  if (!t.is_cuda()) {
    PyErr_Format(PyExc_TypeError, "%s must be a CUDA tensor", name);
  } else if (!right_type) {
    PyErr_Format(PyExc_TypeError, "%s is of a type that this call does not take: %s", name, c10::toString(t.scalar_type()));
  } else if (t.dim() != 2 || t.size(0) > kMost || t.size(1) > kMost) {
    PyErr_Format(PyExc_ValueError, "%s must be a matrix of at most %lld rows and columns", name, static_cast<long long>(kMost));
  } else if (t.size(1) > 1 && t.stride(1) != 1) {
    PyErr_Format(PyExc_ValueError, "%s needs a unit inner stride", name);
  } else if (t.is_neg()) {
    PyErr_Format(PyExc_ValueError, "%s is a view of numbers with the other sign (resolve_neg() makes them its own)", name);
  } else {
    *ld = t.size(0) > 1 ? t.stride(0) : padded(t.size(1));
    if (*ld >= t.size(1)) return true;
    PyErr_Format(PyExc_ValueError, "%s's rows overlap", name);
  }
  return false;
}

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed with code ", rc); }
// The GIL is not held while one of these lives; what it covers may throw.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};
PyObject* wrap(const at::Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); }

// A matrix in 8 bits as the kernels write it: rows padded to 16 bytes, scales [K blocks, M] (block_rows 1) or [M blocks, K blocks]; the
// transpose and the sums of the columns over blocks of rows where they are asked for.
struct Quantized {
  at::Tensor q, scale, qt, scale_t, sums;
};
void quantize(const at::Tensor& x, int64_t ld, bool row, bool transposed, bool sums, cudaStream_t stream, Quantized* out) {
  const int64_t M = x.size(0), K = x.size(1);
  const auto e4m3 = x.options().dtype(at::kFloat8_e4m3fn).requires_grad(false), f32 = x.options().dtype(at::kFloat).requires_grad(false);
  out->q = at::empty({M, padded(K)}, e4m3);
  out->scale = row ? at::empty({blocks(K), M}, f32) : at::empty({blocks(M), blocks(K)}, f32);
  if (transposed) {
    out->qt = at::empty({K, padded(M)}, e4m3);
    if (row) out->scale_t = at::empty({blocks(M), K}, f32);
    if (sums) out->sums = at::empty({blocks(M), K}, f32);
  }
  if (M == 0 || K == 0) return;
  const auto floats = [](const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
  check(lib.quantize_fp8(x.data_ptr(), float_code(x), ld, static_cast<int>(M), static_cast<int>(K), row ? 1 : static_cast<int>(kBlock), out->q.data_ptr(),
                         out->q.size(1), floats(out->scale), transposed ? out->qt.data_ptr() : nullptr, transposed ? out->qt.size(1) : 0, floats(out->scale_t),
                         floats(out->sums), stream),
        "mncclQuantizeFp8");
}

// quantize_fp8(x, block_rows, transposed, stream | None) -> (q, scale) or (q, scale, qt, scale_t); see ops/fp8.py
PyObject* quantize_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arg_count(n, 4) || !plain_calls("quantize_fp8", {args[0]})) return nullptr;
  const at::Tensor* x = tensor_arg(args[0], "x");
  if (!x) return nullptr;
  const long block_rows = PyLong_AsLong(args[1]);
  const int transposed = PyObject_IsTrue(args[2]);
  if (transposed < 0 || PyErr_Occurred()) return nullptr;
  int64_t ld = 0;
  if (!matrix(*x, "x", float_code(*x) >= 0, &ld)) return nullptr;
  if (block_rows != 1 && block_rows != kBlock) {
    PyErr_SetString(PyExc_ValueError, "block_rows must be 1 or 128");
    return nullptr;
  }
  if (x->size(1) > kMostColumns) {
    PyErr_Format(PyExc_ValueError, "x must have at most %lld columns", static_cast<long long>(kMostColumns));
    return nullptr;
  }
  On o;
  if (!on(*x, args[3], &o)) return nullptr;
  const int64_t M = x->size(0), K = x->size(1);
  const bool row = block_rows == 1;
  Quantized q;
  {
    NoGil free;
    c10::AutoGradMode no_grad(false);
    quantize(*x, ld, row, transposed != 0, false, o.raw, &q);
    if (q.q.size(1) != K) q.q = q.q.slice(1, 0, K);
    if (transposed) {
      if (q.qt.size(1) != M) q.qt = q.qt.slice(1, 0, M);
      q.scale_t = row ? q.scale_t.t() : q.scale.t();
    }
    if (row) q.scale = q.scale.t();
  }
  if (!transposed) return Py_BuildValue("(NN)", wrap(q.q), wrap(q.scale));
  return Py_BuildValue("(NNNN)", wrap(q.q), wrap(q.scale), wrap(q.qt), wrap(q.scale_t));
  END_HANDLE_TH_ERRORS
}

bool operand(const at::Tensor& t, const char* name, int64_t* ld) {
  if (!matrix(t, name, t.scalar_type() == at::kFloat8_e4m3fn, ld)) return false;
  if (t.numel() == 0 || (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && *ld % 16 == 0)) return true;
  PyErr_Format(PyExc_ValueError, "%s's rows must start on 16 bytes (quantize_fp8 lays them out so)", name);
  return false;
}
// Whether `t` holds the scales of an operand [rows, K]; *per: rows of a scale.
bool scales(const at::Tensor& t, const char* name, int64_t rows, int64_t K, const at::Tensor& like, int* per) {
  if (t.scalar_type() != at::kFloat || t.device() != like.device()) {
    PyErr_Format(PyExc_TypeError, "%s must be an fp32 tensor on the operands' GPU", name);
    return false;
  }
  if (t.is_neg()) {
    PyErr_Format(PyExc_ValueError, "%s is a view of numbers with the other sign (resolve_neg() makes them its own)", name);
    return false;
  }
  if (t.dim() != 2 || t.size(1) != blocks(K) || (t.size(0) != rows && t.size(0) != blocks(rows))) {
    PyErr_Format(PyExc_ValueError, "%s must be [%lld or %lld, %lld]", name, static_cast<long long>(rows), static_cast<long long>(blocks(rows)),
                 static_cast<long long>(blocks(K)));
    return false;
  }
  *per = t.size(0) == rows ? 1 : static_cast<int>(kBlock);
  return true;
}

// gemm_fp8(a, a_scale, b, b_scale, out | None, out_dtype | None, bias | None, stream | None) -> out; see ops/fp8.py
PyObject* gemm_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arg_count(n, 8) || !plain_calls("gemm_fp8", {args[0], args[1], args[2], args[3], args[4], args[6]})) return nullptr;
  const at::Tensor *a = tensor_arg(args[0], "a"), *sa = a ? tensor_arg(args[1], "a_scale") : nullptr, *b = sa ? tensor_arg(args[2], "b") : nullptr,
                   *sb = b ? tensor_arg(args[3], "b_scale") : nullptr;
  if (!sb) return nullptr;
  int64_t lda = 0, ldb = 0, ldc = 0;
  if (!operand(*a, "a", &lda) || !operand(*b, "b", &ldb)) return nullptr;
  const int64_t M = a->size(0), K = a->size(1), N = b->size(0);
  if (b->size(1) != K || b->device() != a->device()) {
    PyErr_SetString(PyExc_ValueError, "shapes: a [M, K], b [N, K], on one GPU");
    return nullptr;
  }
  int pa = 1, pb = 1;
  if (!scales(*sa, "a_scale", M, K, *a, &pa) || !scales(*sb, "b_scale", N, K, *a, &pb)) return nullptr;
  std::optional<at::ScalarType> type;
  if (args[5] != Py_None) {
    if (!THPDtype_Check(args[5])) {
      PyErr_SetString(PyExc_TypeError, "out_dtype must be a torch dtype");
      return nullptr;
    }
    type = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
  }
  On o;
  if (!on(*a, args[7], &o)) return nullptr;
  at::Tensor fresh;
  const at::Tensor* out = nullptr;
  if (args[4] != Py_None) {
    out = tensor_arg(args[4], "out");
    if (!out) return nullptr;
    if (type && *type != out->scalar_type()) {
      PyErr_SetString(PyExc_ValueError, "out has another type than out_dtype");
      return nullptr;
    }
  } else {
    fresh = at::empty({M, N}, a->options().dtype(type.value_or(at::kBFloat16)).requires_grad(false));
    out = &fresh;
  }
  const int code = float_code(*out);
  if (out->dim() != 2 || out->size(0) != M || out->size(1) != N || out->device() != a->device()) {
    PyErr_SetString(PyExc_ValueError, "out must be [M, N] on the operands' GPU");
    return nullptr;
  }
  if (!matrix(*out, "out", code >= 0, &ldc)) return nullptr;
  const at::Tensor* bias = nullptr;
  if (args[6] != Py_None) {
    bias = tensor_arg(args[6], "bias");
    if (!bias) return nullptr;
    if (bias->scalar_type() != out->scalar_type() || bias->device() != a->device() || bias->dim() != 1 || bias->size(0) != N || (N > 1 && bias->stride(0) != 1) || bias->is_neg()) {
      PyErr_SetString(PyExc_ValueError, "bias must be [N], dense, of out's type and on its GPU");
      return nullptr;
    }
  }
  if (K == 0) {
    c10::AutoGradMode no_grad(false);
    if (bias) out->copy_(bias->expand({M, N}));
    else out->zero_();
  } else if (M > 0 && N > 0) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = lib.gemm_fp8(a->data_ptr(), lda, sa->data_ptr<float>(), sa->stride(0), sa->stride(1), pa, b->data_ptr(), ldb, sb->data_ptr<float>(), sb->stride(0),
                      sb->stride(1), pb, out->data_ptr(), ldc, code, bias ? bias->data_ptr() : nullptr, static_cast<int>(M), static_cast<int>(N),
                      static_cast<int>(K), o.raw);
    Py_END_ALLOW_THREADS
    check(rc, "mncclGemmFp8");
    // autograd notices that an operand it has kept was written, as for PyTorch's own calls with out=
    if (!fresh.defined() && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
  }
  return fresh.defined() ? THPVariable_Wrap(fresh) : Py_NewRef(args[4]);
  END_HANDLE_TH_ERRORS
}

// `t [..., cols]` as a matrix that the kernels can read (a copy only where the strides need one, or where `t` is a view of numbers with the other sign, as
// the imaginary part of a conjugate is), and its row stride.
at::Tensor rows_of(const at::Tensor& t, int64_t cols, int64_t* ld) {
  c10::AutoGradMode no_grad(false);
  at::Tensor r = (t.dim() == 2 ? t : t.reshape({cols > 0 ? t.numel() / cols : 0, cols})).resolve_neg();
  if ((cols > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < cols)) r = r.contiguous();
  *ld = r.size(0) > 1 ? r.stride(0) : padded(cols);
  return r;
}

// out [M, N] = a * b^T (+ bias) of padded buffers: a [M, padded K] with scales [K blocks, M], b [N, padded K] with scales that have these strides.
void product(const at::Tensor& a, const at::Tensor& sa, const at::Tensor& b, const at::Tensor& sb, int64_t sb_row, int64_t sb_blk, int sb_rows, int64_t M, int64_t N,
             int64_t K, const at::Tensor& out, const at::Tensor& bias, cudaStream_t stream) {
  if (M == 0 || N == 0) return;
  if (K == 0) {
    c10::AutoGradMode no_grad(false);
    out.zero_();
    return;
  }
  check(lib.gemm_fp8(a.data_ptr(), a.size(1), sa.data_ptr<float>(), 1, M, 1, b.data_ptr(), b.size(1), sb.data_ptr<float>(), sb_row, sb_blk, sb_rows, out.data_ptr(),
                     N, float_code(out), bias.defined() ? bias.data_ptr() : nullptr, static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), stream),
        "mncclGemmFp8");
}

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// The backward pass of linear_fp8: x^T and its scales, weight^T and the weight's scales, each undefined where it is not wanted.
struct LinearFp8Backward final : torch::autograd::Node {
  SavedVariable xt, xt_scale, wt, w_scale;
  std::vector<int64_t> x_sizes;
  bool want_x = false, want_w = false;

  std::string name() const override { return "LinearFp8Backward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&xt, &xt_scale, &wt, &w_scale}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);   // dx, dweight, dbias
    if (!grads[0].defined()) return out;
    const bool once = c10::GradMode::is_enabled();   // create_graph
    {
      c10::AutoGradMode no_grad(false);
      const bool to_x = want_x && task_should_compute_output(0), to_w = want_w && task_should_compute_output(1), to_b = task_should_compute_output(2);
      const at::Tensor grad = grads[0];
      const c10::cuda::CUDAGuard device(grad.device());
      const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
      const int64_t N = grad.size(-1), K = x_sizes.back();
      int64_t ld = 0;
      const at::Tensor g = rows_of(grad, N, &ld);
      const int64_t T = g.size(0);
      const auto like = g.options().requires_grad(false);
      if (N == 0) {   // a layer without output features
        if (to_x) out[0] = at::zeros(x_sizes, like);
        if (to_w) out[1] = at::zeros({N, K}, like);
        if (to_b) out[2] = at::zeros({N}, like);
        return out;
      }
      Quantized q;
      quantize(g, ld, true, to_w || to_b, to_b, stream, &q);
      if (to_x) {   // rows of weight^T are columns of the weight
        const at::Tensor t = wt.unpack().contiguous(), s = w_scale.unpack().contiguous();
        out[0] = at::empty(x_sizes, like);
        product(q.q, q.scale, t, s, 1, s.size(1), static_cast<int>(kBlock), T, K, N, out[0], at::Tensor(), stream);
      }
      if (to_w) {
        const at::Tensor t = xt.unpack().contiguous(), s = xt_scale.unpack().contiguous();
        out[1] = at::empty({N, K}, like);
        product(q.qt, q.scale_t, t, s, 1, K, 1, N, K, T, out[1], at::Tensor(), stream);
      }
      if (to_b) {
        out[2] = T > 0 ? at::empty({N}, like) : at::zeros({N}, like);
        if (T > 0)
          check(lib.sum_blocks(q.sums.data_ptr<float>(), static_cast<int>(q.sums.size(0)), static_cast<int>(N), out[2].data_ptr(), float_code(out[2]), stream),
                "mncclSumBlocks");
      }
    }
    if (!once) return out;
    // differentiable once: what is made of these gradients may not be differentiated
    for (at::Tensor& t : out)
      if (t.defined()) t = t.detach().requires_grad_(true);
    return torch::autograd::DelayedError("trying to differentiate linear_fp8 twice", static_cast<int64_t>(out.size())).apply(std::move(out));
  }
};

// linear_fp8(x [..., K], weight [N, K], bias [N] | None) -> y [..., N]; ops/fp8.py has checked the arguments
PyObject* linear_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arg_count(n, 3)) return nullptr;
  const at::Tensor *x = tensor_arg(args[0], "x"), *weight = x ? tensor_arg(args[1], "weight") : nullptr, *bias = nullptr;
  if (!weight || (args[2] != Py_None && !(bias = tensor_arg(args[2], "bias")))) return nullptr;
  On o;
  if (!on(*x, Py_None, &o)) return nullptr;
  at::Tensor y;
  {
    NoGil free;
    const at::Tensor b = bias ? *bias : at::Tensor();
    const bool grad = c10::GradMode::is_enabled(), want_x = grad && x->requires_grad(), want_w = grad && weight->requires_grad();
    const bool any = want_x || want_w || (grad && b.defined() && b.requires_grad());
    Quantized qx, qw;
    {
      c10::AutoGradMode no_grad(false);
      const int64_t N = weight->size(0), K = weight->size(1);
      int64_t ldx = 0, ldw = 0;
      const at::Tensor rows = rows_of(*x, K, &ldx), w = rows_of(*weight, K, &ldw), dense = b.defined() ? b.resolve_neg().contiguous() : b;
      quantize(rows, ldx, true, want_w, false, o.raw, &qx);
      quantize(w, ldw, false, want_x, false, o.raw, &qw);
      auto shape = x->sizes().vec();
      shape.back() = N;
      y = at::empty(shape, x->options().requires_grad(false));
      product(qx.q, qx.scale, qw.q, qw.scale, qw.scale.size(1), 1, static_cast<int>(kBlock), rows.size(0), N, K, y, dense, o.raw);
    }
    if (any) {
      std::shared_ptr<LinearFp8Backward> node(new LinearFp8Backward(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(*x, *weight, b));
      node->want_x = want_x;
      node->want_w = want_w;
      node->x_sizes = x->sizes().vec();
      if (want_w) {
        node->xt = SavedVariable(qx.qt, false);
        node->xt_scale = SavedVariable(qx.scale_t, false);
      }
      if (want_x) {
        node->wt = SavedVariable(qw.qt, false);
        node->w_scale = SavedVariable(qw.scale, false);
      }
      torch::autograd::set_history(y, node);
    }
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// A loss and what its backward pass needs.
struct Distilled {
  at::Tensor loss, p, stats, counts, tokens;
};
// reduction: 0 a loss for each row, 1 their sum, 2 their mean
Distilled distill(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& top, double tau, long reduction, cudaStream_t stream) {
  const int64_t V = logits.size(-1);
  int64_t ld = 0;
  const at::Tensor rows = rows_of(logits, V, &ld);
  const int64_t T = rows.size(0), K = ids.size(1);
  const auto f32 = rows.options().dtype(at::kFloat).requires_grad(false);
  Distilled d{at::empty({}, f32), at::empty({T, K}, f32), at::empty({T, 2}, f32), at::empty({T}, f32.dtype(at::kInt)), at::empty({}, f32)};
  const at::Tensor row_loss = at::empty(logits.sizes().slice(0, logits.dim() - 1), f32);
  check(lib.distill_forward(rows.data_ptr(), float_code(rows), ld, static_cast<int>(T), static_cast<int>(V), ids.data_ptr<int64_t>(), top.data_ptr<float>(),
                            static_cast<int>(K), static_cast<float>(tau), d.p.data_ptr<float>(), d.stats.data_ptr<float>(), row_loss.data_ptr<float>(),
                            d.counts.data_ptr<int>(), reduction == 1 ? d.loss.data_ptr<float>() : nullptr, reduction == 2 ? d.loss.data_ptr<float>() : nullptr,
                            d.tokens.data_ptr<float>(), stream),
        "mncclDistillForward");
  if (reduction == 0) d.loss = row_loss;
  return d;
}
// The gradient of the logits, for a gradient of each row's loss or of their sum; tokens: what it is divided by, if defined.
at::Tensor distill_gradient(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& p, const at::Tensor& stats, const at::Tensor& counts,
                            const at::Tensor& tokens, double tau, const at::Tensor& of_loss, cudaStream_t stream) {
  const int64_t V = logits.size(-1);
  int64_t ld = 0;
  const at::Tensor rows = rows_of(logits, V, &ld), grad = of_loss.resolve_neg().contiguous();
  // the gradient's rows lie to 16 bytes as the logits' do: padded where those are
  const int64_t T = rows.size(0), per = 16 / rows.element_size(), ldd = rows.stride(0) != V ? (V + per - 1) / per * per : V;
  at::Tensor d = at::empty({T, ldd}, rows.options().requires_grad(false));
  check(lib.distill_backward(rows.data_ptr(), float_code(rows), ld, static_cast<int>(T), static_cast<int>(V), ids.data_ptr<int64_t>(), p.data_ptr<float>(),
                             static_cast<int>(ids.size(1)), static_cast<float>(tau), stats.data_ptr<float>(), counts.data_ptr<int>(), grad.data_ptr<float>(),
                             grad.dim() > 0 ? 1 : 0, tokens.defined() ? tokens.data_ptr<float>() : nullptr, d.data_ptr(), ldd, stream),
        "mncclDistillBackward");
  if (ldd != V) d = d.slice(1, 0, V);
  return logits.dim() == 2 ? d : d.view(logits.sizes());
}

// distill_forward(logits [..., V], ids [T, K], top [T, K], tau, reduction) -> (loss, p, stats, counts, tokens); ops/distill.py has checked the arguments
PyObject* distill_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arg_count(n, 5)) return nullptr;
  const at::Tensor *logits = tensor_arg(args[0], "logits"), *ids = logits ? tensor_arg(args[1], "ids") : nullptr, *top = ids ? tensor_arg(args[2], "top") : nullptr;
  if (!top) return nullptr;
  const double tau = PyFloat_AsDouble(args[3]);
  const long reduction = PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  On o;
  if (!on(*logits, Py_None, &o)) return nullptr;
  Distilled d;
  {
    NoGil free;
    d = distill(*logits, *ids, *top, tau, reduction, o.raw);
  }
  return Py_BuildValue("(NNNNN)", wrap(d.loss), wrap(d.p), wrap(d.stats), wrap(d.counts), wrap(d.tokens));
  END_HANDLE_TH_ERRORS
}

// distill_backward(logits [..., V], ids, p, stats, counts, tokens | None, tau, grad) -> gradient of the logits
PyObject* distill_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arg_count(n, 8)) return nullptr;
  at::Tensor t[8];
  for (int i = 0; i < 8; ++i) {
    if (i == 6 || (i == 5 && args[i] == Py_None)) continue;
    const at::Tensor* given = tensor_arg(args[i], "argument");
    if (!given) return nullptr;
    t[i] = *given;
  }
  const double tau = PyFloat_AsDouble(args[6]);
  if (PyErr_Occurred()) return nullptr;
  On o;
  if (!on(t[0], Py_None, &o)) return nullptr;
  at::Tensor d;
  {
    NoGil free;
    d = distill_gradient(t[0], t[1], t[2], t[3], t[4], t[5], tau, t[7], o.raw);
  }
  return wrap(d);
  END_HANDLE_TH_ERRORS
}

// What takes over where the gradient itself is to be differentiated (create_graph): f(logits, ids, top, tau, reduction, grad) -> gradient.  Held for
// the life of the process.
PyObject* distill_again = nullptr;

struct DistillationBackward final : torch::autograd::Node {
  SavedVariable logits, ids, top, p, stats, counts, tokens;
  double tau = 1.0;
  long reduction = 0;

  std::string name() const override { return "DistillationBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&logits, &ids, &top, &p, &stats, &counts, &tokens}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined() || !task_should_compute_output(0)) return variable_list(1);
    const at::Tensor z = logits.unpack();
    if (c10::GradMode::is_enabled()) {
      const at::Tensor i = ids.unpack(), t = top.unpack();
      const PyGILState_STATE gil = PyGILState_Ensure();
      at::Tensor got;
      PyObject* r = distill_again ? PyObject_CallFunction(distill_again, "NNNdlN", wrap(z), wrap(i), wrap(t), tau, reduction, wrap(grads[0])) : nullptr;
      if (r && THPVariable_Check(r)) got = THPVariable_Unpack(r);
      Py_XDECREF(r);
      if (!got.defined()) {
        python_error e;
        if (PyErr_Occurred()) e.persist();
        PyGILState_Release(gil);
        throw e;
      }
      PyGILState_Release(gil);
      return {got};
    }
    const c10::cuda::CUDAGuard device(z.device());
    return {distill_gradient(z, ids.unpack(), p.unpack(), stats.unpack(), counts.unpack(), reduction == 2 ? tokens.unpack() : at::Tensor(), tau, grads[0],
                             c10::cuda::getCurrentCUDAStream().stream())};
  }
};

// distillation(logits [..., V], ids [T, K], top [T, K], tau, reduction, again) -> loss, differentiable in the logits; again: see distill_again
PyObject* distillation(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arg_count(n, 6)) return nullptr;
  const at::Tensor *logits = tensor_arg(args[0], "logits"), *ids = logits ? tensor_arg(args[1], "ids") : nullptr, *top = ids ? tensor_arg(args[2], "top") : nullptr;
  if (!top) return nullptr;
  const double tau = PyFloat_AsDouble(args[3]);
  const long reduction = PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  if (!distill_again) distill_again = Py_NewRef(args[5]);
  On o;
  if (!on(*logits, Py_None, &o)) return nullptr;
  Distilled d;
  {
    NoGil free;
    d = distill(*logits, *ids, *top, tau, reduction, o.raw);
    if (c10::GradMode::is_enabled() && logits->requires_grad()) {
      std::shared_ptr<DistillationBackward> node(new DistillationBackward(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(*logits));
      node->tau = tau;
      node->reduction = reduction;
      node->logits = SavedVariable(*logits, false);
      node->ids = SavedVariable(*ids, false);
      node->top = SavedVariable(*top, false);
      node->p = SavedVariable(d.p, false);
      node->stats = SavedVariable(d.stats, false);
      node->counts = SavedVariable(d.counts, false);
      node->tokens = SavedVariable(d.tokens, false);
      torch::autograd::set_history(d.loss, node);
    }
  }
  return wrap(d.loss);
  END_HANDLE_TH_ERRORS
}

// async_error(comm) -> ncclResult_t
PyObject* async_error(PyObject*, PyObject* comm) {
  const int e = comm_error(comm);
  return PyErr_Occurred() ? nullptr : PyLong_FromLong(e);
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {"all_reduce", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(all_reduce)), METH_FASTCALL, nullptr},
    {"gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gemm)), METH_FASTCALL, nullptr},
    {"gemm_rs", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gemm_rs)), METH_FASTCALL, nullptr},
    {"ag_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(ag_gemm)), METH_FASTCALL, nullptr},
    {"quantize_fp8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(quantize_fp8)), METH_FASTCALL, nullptr},
    {"gemm_fp8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gemm_fp8)), METH_FASTCALL, nullptr},
    {"linear_fp8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear_fp8)), METH_FASTCALL, nullptr},
    {"distillation", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(distillation)), METH_FASTCALL, nullptr},
    {"distill_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(distill_forward)), METH_FASTCALL, nullptr},
    {"distill_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(distill_backward)), METH_FASTCALL, nullptr},
    {"async_error", async_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ext", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ext(void) { return PyModule_Create(&module); }
