// Distillation from a teacher's top logits: for each of T tokens, student logits z [V] and K teacher entries (id, logit).
//
//   p   = softmax(top / tau) over the entries that are there: id >= 0 and a logit above -infinity
//   L_t = tau^2 * sum_k p_k (log p_k - log softmax(z / tau)[id_k])
//   dL_t / dz_v = tau * (softmax(z / tau)_v - sum of p_k over the entries with id_k = v)
//
// A token without entries counts for nothing: it is left out of the mean, its loss and its gradient are 0 and its logits
// are not looked at.  Ids may repeat; an id of V or more makes its token's loss and gradient NaN.
//
// What bounds it is memory: the logits are read once forward, and once more backward, where the gradient is written.
// Softmax statistics are {max z, sum of 2^((z - max z) * log2(e) / tau)} in fp32: the difference is taken before it is
// scaled, so that large logits lose nothing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

namespace {

constexpr int kThreads = 256;
constexpr int kMaxEntries = 1024;
constexpr int kMaxParts = 8;   // blocks that share a row of logits
constexpr int kMostIndex = 0x7ffff000;   // tokens, classes: counters pass the last one by up to four blocks' worth of threads before they are compared
constexpr float kLog2e = 1.4426950408889634f;

// 2^x to 2^-22 of the value, 0 below 2^-126; exp2 of -infinity is 0, of a NaN a NaN.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ float as_float(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

// A row of V elements that may start anywhere: elements before the first 16-byte boundary, whole vectors, the rest.
template <typename T>
struct RowSplit {
  static constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  int head, vectors;
  __device__ __forceinline__ RowSplit(const T* row, int V) {
    const int before = static_cast<int>((16u - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / static_cast<int>(sizeof(T));
    head = min(before, V);
    vectors = (V - head) / kPer;
  }
  // the i-th of the elements outside the vectors, or V
  __device__ __forceinline__ int loose(int i, int V) const { return i < head ? i : min(i + vectors * kPer, V); }
};

// The running maximum and sum of a softmax.  With nothing or only -infinity seen what is subtracted is 0, so that
// 2^(-infinity - 0) = 0 instead of a NaN.
struct Running {
  float m, s;
  static __device__ __forceinline__ float base(float m) { return m == -INFINITY ? 0.0f : m; }
  __device__ __forceinline__ void raise(float top, float c) {
    s *= exp2_fast((m - base(top)) * c);
    m = top;
  }
  __device__ __forceinline__ void merge(float m2, float s2, float c) {
    const float top = fmaxf(m, m2), b = base(top);
    s = s * exp2_fast((m - b) * c) + s2 * exp2_fast((m2 - b) * c);
    m = top;
  }
};

// The largest of N elements and `highest`; 16-bit types two at a time.
template <typename T, int N>
__device__ __forceinline__ float highest_of(const T (&x)[N], float highest) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < N; ++j) highest = fmaxf(highest, x[j]);
    return highest;
  } else {
    using Two = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const Two* two = reinterpret_cast<const Two*>(x);
    Two top = two[0];
#pragma unroll
    for (int j = 1; j < N / 2; ++j) top = __hmax2(top, two[j]);
    return fmaxf(highest, fmaxf(as_float(top.x), as_float(top.y)));
  }
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
  return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
// The same over the block, in a fixed order; `box` holds a word for each warp and may be used again after a barrier.
__device__ __forceinline__ float block_max(float x, float* box) {
  x = warp_max(x);
  if ((threadIdx.x & 31) == 0) box[threadIdx.x >> 5] = x;
  __syncthreads();
  x = box[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) x = fmaxf(x, box[w]);
  __syncthreads();
  return x;
}
__device__ __forceinline__ float block_sum(float x, float* box) {
  x = warp_sum(x);
  if ((threadIdx.x & 31) == 0) box[threadIdx.x >> 5] = x;
  __syncthreads();
  x = box[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) x += box[w];
  __syncthreads();
  return x;
}

// A cluster of blocks per token (one where there are many), which meet in the first block's shared memory.  Writes p [T, K], stats[t] =
// {max, sum}, row_loss[t] and counts[t].  PER: teacher's entries a thread holds.  They and the student's logits at their ids are fetched before
// the row is read, so that the end of a block does not wait for memory again.
template <typename T, int PER>
__global__ void __launch_bounds__(kThreads, PER == 1 ? 5 : 3)
distill_rows_kernel(const T* __restrict__ logits, size_t ld, int V, const int64_t* __restrict__ ids, const float* __restrict__ top, int K,
                    float tau, int parts, float* __restrict__ p, float2* __restrict__ stats, float* __restrict__ row_loss, int* __restrict__ counts) {
  __shared__ float box[2][kThreads / 32];
  __shared__ float2 of_part[kMaxParts];
  const size_t t = blockIdx.x / static_cast<unsigned>(parts);
  const int part = static_cast<int>(blockIdx.x % static_cast<unsigned>(parts));
  const T* row = logits + t * ld;
  const float inv_tau = 1.0f / tau, c = kLog2e / tau;

  float teacher[PER], student[PER];
  float high = -INFINITY;
  bool any = false, bad = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int k = static_cast<int>(threadIdx.x) + i * kThreads;
    const int64_t id = k < K ? ids[t * K + k] : -1;
    const float logit = k < K ? top[t * K + k] : -INFINITY;
    teacher[i] = id >= 0 ? logit : -INFINITY;
    const bool there = teacher[i] != -INFINITY;
    any = any || there;
    bad = bad || (there && id >= V);
    student[i] = there && id < V && part == 0 ? as_float(row[id]) : 0.0f;
    high = fmaxf(high, teacher[i]);
  }
  if (__syncthreads_or(any) == 0) {   // the same in all blocks of the cluster
    if (part != 0) return;
    for (int k = threadIdx.x; k < K; k += kThreads) p[t * K + k] = 0.0f;
    if (threadIdx.x == 0) {
      stats[t] = make_float2(0.0f, 1.0f);
      row_loss[t] = 0.0f;
      counts[t] = 0;
    }
    return;
  }

  Running r{-INFINITY, 0.0f};
  const RowSplit<T> split(row, V);
  constexpr int kVec = RowSplit<T>::kPer, kBatch = 4;
  const uint4* body = reinterpret_cast<const uint4*>(row + split.head);
  const int per_part = (split.vectors + parts - 1) / parts;
  const int last = min(split.vectors, (part + 1) * per_part);
  int v = part * per_part + static_cast<int>(threadIdx.x);
  for (; v + (kBatch - 1) * kThreads < last; v += kBatch * kThreads) {
    union { uint4 raw; T x[kVec]; } u[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) u[b].raw = __ldg(body + v + b * kThreads);
    float highest = r.m;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) highest = highest_of(u[b].x, highest);
    r.raise(highest, c);
    const float base = Running::base(r.m);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int j = 0; j < kVec; ++j) r.s += exp2_fast((as_float(u[b].x[j]) - base) * c);
  }
  for (; v < last; v += kThreads) {
    union { uint4 raw; T x[kVec]; } u;
    u.raw = __ldg(body + v);
    r.raise(highest_of(u.x, r.m), c);
    const float base = Running::base(r.m);
#pragma unroll
    for (int j = 0; j < kVec; ++j) r.s += exp2_fast((as_float(u.x[j]) - base) * c);
  }
  const int loose = part == 0 ? split.loose(threadIdx.x, V) : V;
  if (loose < V) {
    const float x = as_float(row[loose]), highest = fmaxf(r.m, x);
    r.raise(highest, c);
    r.s += exp2_fast((x - Running::base(highest)) * c);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) r.merge(__shfl_xor_sync(0xffffffffu, r.m, d), __shfl_xor_sync(0xffffffffu, r.s, d), c);
  if ((threadIdx.x & 31) == 0) {
    box[0][threadIdx.x >> 5] = r.m;
    box[1][threadIdx.x >> 5] = r.s;
  }
  __syncthreads();
  r = Running{box[0][0], box[1][0]};
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) r.merge(box[0][w], box[1][w], c);
  __syncthreads();
  if (parts > 1) {
    const auto cluster = cooperative_groups::this_cluster();
    cluster.sync();   // the first block runs
    if (threadIdx.x == 0) *cluster.map_shared_rank(of_part + part, 0) = make_float2(r.m, r.s);
    cluster.sync();
    if (part != 0) return;
    r = Running{of_part[0].x, of_part[0].y};
    for (int i = 1; i < parts; ++i) r.merge(of_part[i].x, of_part[i].y, c);
  }

  high = Running::base(block_max(high, box[0]));
  float total = 0.0f, e[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    e[i] = teacher[i] == -INFINITY ? 0.0f : exp2_fast((teacher[i] - high) * c);
    total += e[i];
  }
  total = block_sum(total, box[0]);
  const float log_total = logf(total), log_s = logf(r.s);
  float loss = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int k = static_cast<int>(threadIdx.x) + i * kThreads;
    if (k >= K) break;
    const float pk = e[i] / total;
    p[t * K + k] = pk;
    // (a weight of 0 counts for nothing, even where the student's logit is -infinity)
    if (teacher[i] != -INFINITY && pk != 0.0f) loss += pk * (((teacher[i] - high) * inv_tau - log_total) - ((student[i] - r.m) * inv_tau - log_s));
  }
  bad = __syncthreads_or(bad) != 0;
  loss = block_sum(loss, box[0]);
  if (threadIdx.x == 0) {
    stats[t] = bad ? make_float2(__int_as_float(0x7fffffff), 1.0f) : make_float2(r.m, r.s);
    row_loss[t] = bad ? __int_as_float(0x7fffffff) : tau * tau * loss;
    counts[t] = 1;
  }
}

// sum = the rows' losses' sum, mean = that over the number of tokens that count (either may be null), tokens = that number; in one block and a fixed
// order.
__global__ void __launch_bounds__(1024)
distill_mean_kernel(const float* __restrict__ row_loss, const int* __restrict__ counts, int T, float* __restrict__ sum, float* __restrict__ mean,
                    float* __restrict__ tokens) {
  __shared__ float box[2][32];
  float s = 0.0f, n = 0.0f;   // n: whole numbers, exact up to 2^24
  for (int t = threadIdx.x; t < T; t += 1024) {
    s += row_loss[t];
    n += static_cast<float>(counts[t]);
  }
  s = warp_sum(s);
  n = warp_sum(n);
  if ((threadIdx.x & 31) == 0) {
    box[0][threadIdx.x >> 5] = s;
    box[1][threadIdx.x >> 5] = n;
  }
  __syncthreads();
  s = warp_sum(box[0][threadIdx.x & 31]);
  n = warp_sum(box[1][threadIdx.x & 31]);
  if (threadIdx.x == 0) {
    if (sum != nullptr) *sum = s;
    if (mean != nullptr) *mean = s / n;
    *tokens = n;
  }
}

// The gradient of one token: (softmax - p) * tau * grad [/ tokens that count].  The dense part first, then the entries' elements
// once more with all entries of their id taken off before the one rounding.  `parts` blocks share a row.
template <typename T>
__global__ void __launch_bounds__(kThreads)
distill_grad_kernel(const T* __restrict__ logits, size_t ld, int V, const int64_t* __restrict__ ids, const float* __restrict__ p, int K, float tau,
                    const float2* __restrict__ stats, const int* __restrict__ counts, const float* __restrict__ grad, int grad_per_row,
                    const float* __restrict__ tokens, int parts, T* __restrict__ d, size_t ldd) {
  __shared__ int s_id[kMaxEntries];
  __shared__ float s_p[kMaxEntries];
  const size_t t = blockIdx.x / static_cast<unsigned>(parts);
  const int part = static_cast<int>(blockIdx.x % static_cast<unsigned>(parts));
  const T* row = logits + t * ld;
  T* out = d + t * ldd;
  constexpr int kVec = RowSplit<T>::kPer;
  const bool vec = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  const RowSplit<T> split(out, V);
  uint4* out_body = reinterpret_cast<uint4*>(out + split.head);
  // This block's share: vectors [v0, v1) of the gradient's row, the first block the loose elements as well; or elements [x0, x1) where the two
  // rows do not lie alike.
  const int loose = part == 0 ? split.loose(threadIdx.x, V) : V;
  const int per_part = (split.vectors + parts - 1) / parts, v0 = min(part * per_part, split.vectors), v1 = min(v0 + per_part, split.vectors);
  if (counts[t] == 0) {
    for (int v = v0 + threadIdx.x; v < v1; v += kThreads) out_body[v] = make_uint4(0, 0, 0, 0);
    if (loose < V) out[loose] = from_float<T>(0.0f);
    return;
  }
  const int x_per = (V + parts - 1) / parts, x0 = min(part * x_per, V), x1 = min(x0 + x_per, V);
  for (int k = threadIdx.x; k < K; k += kThreads) {
    const int64_t id = ids[t * K + k];
    s_id[k] = id >= 0 && id < V ? static_cast<int>(id) : -1;
    s_p[k] = p[t * K + k];
  }
  const float c = kLog2e / tau, m = stats[t].x;
  const float factor = grad[grad_per_row ? t : 0] * tau / (tokens != nullptr ? *tokens : 1.0f);
  const float inverse = 1.0f / stats[t].y;
  const auto dense = [&](float x) { return exp2_fast((x - m) * c) * inverse * factor; };
  if (vec) {
    const uint4* body = reinterpret_cast<const uint4*>(row + split.head);
    for (int v = v0 + threadIdx.x; v < v1; v += kThreads) {
      union { uint4 raw; T x[kVec]; } u;
      u.raw = __ldg(body + v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) u.x[j] = from_float<T>(dense(as_float(u.x[j])));
      out_body[v] = u.raw;
    }
    if (loose < V) out[loose] = from_float<T>(dense(as_float(row[loose])));
  } else {
    for (int x = x0 + threadIdx.x; x < x1; x += kThreads) out[x] = from_float<T>(dense(as_float(row[x])));
  }
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += kThreads) {
    const int id = s_id[k];
    if (id < 0) continue;
    if (vec) {
      const int at = (id - split.head) / kVec;
      const bool in_vectors = id >= split.head && at < split.vectors;
      if (in_vectors ? at < v0 || at >= v1 : part != 0) continue;   // another block wrote it
    } else if (id < x0 || id >= x1) {
      continue;
    }
    float total = 0.0f;
    for (int j = 0; j < K; ++j) total += s_id[j] == id ? s_p[j] : 0.0f;
    out[id] = from_float<T>((exp2_fast((as_float(row[id]) - m) * c) * inverse - total) * factor);
  }
}

int status() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : static_cast<int>(e) + 1000;
}

template <typename T>
bool aligned(const void* p, int64_t ld, int V) {
  return reinterpret_cast<uintptr_t>(p) % sizeof(T) == 0 && ld >= V;
}

bool good_tau(float tau) { return tau >= 1e-3f && tau <= 1e3f; }

// Blocks that share a row: as many as leave every thread two vectors, up to eight, while there are too few rows to fill the GPU (four blocks an
// SM).  64 x 50257 bf16: 9.1 us forward and 7.5 backward with one.
int parts_of(int T, int V, int size) {
  int parts = 1;
  while (parts < kMaxParts && static_cast<int64_t>(T) * parts * 2 <= 148 * 4 && static_cast<int64_t>(V) * size >= 16LL * kThreads * parts * 4) parts *= 2;
  return parts;
}

template <typename T>
int forward(const void* logits, int64_t ld, int T_, int V, const int64_t* ids, const float* top, int K, float tau, float* p, float* stats,
            float* row_loss, int* counts, float* sum, float* mean, float* tokens, cudaStream_t stream) {
  if (!aligned<T>(logits, ld, V)) return -2;
  const int parts = parts_of(T_, V, sizeof(T));
  if (static_cast<int64_t>(T_) * parts > 0x7fffffff) return -2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(T_) * static_cast<unsigned>(parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(parts);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const auto go = [&](auto kernel) {
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(logits), static_cast<size_t>(ld), V, ids, top, K, tau, parts, p, reinterpret_cast<float2*>(stats),
                              row_loss, counts);
  };
  const cudaError_t e = K <= kThreads ? go(distill_rows_kernel<T, 1>) : go(distill_rows_kernel<T, kMaxEntries / kThreads>);
  if (e != cudaSuccess) return static_cast<int>(e) + 1000;
  distill_mean_kernel<<<1, 1024, 0, stream>>>(row_loss, counts, T_, sum, mean, tokens);
  return status();
}

template <typename T>
int backward(const void* logits, int64_t ld, int T_, int V, const int64_t* ids, const float* p, int K, float tau, const float* stats, const int* counts,
             const float* grad, int grad_per_row, const float* tokens, void* d, int64_t ldd, cudaStream_t stream) {
  if (!aligned<T>(logits, ld, V) || !aligned<T>(d, ldd, V)) return -2;
  const int parts = parts_of(T_, V, sizeof(T));
  distill_grad_kernel<T><<<static_cast<unsigned>(T_) * static_cast<unsigned>(parts), kThreads, 0, stream>>>(
      static_cast<const T*>(logits), static_cast<size_t>(ld), V, ids, p, K, tau, reinterpret_cast<const float2*>(stats), counts, grad, grad_per_row, tokens, parts,
      static_cast<T*>(d), static_cast<size_t>(ldd));
  return status();
}

}  // namespace

extern "C" {
#define MNCCL_EXPORT __attribute__((visibility("default")))

// logits [T, V] (type 6 fp16, 7 fp32, 9 bf16; row stride ld elements; T and V at most 2^31 - 2^12), ids and top [T, K], K at most 1024, tau in [1e-3, 1e3].  Writes for
// the backward pass p [T, K], stats [T, 2] (8-byte aligned), counts [T] and tokens[1] (how many count); row_loss [T], sum and mean (either may be null).
// Returns 0, -1 null or empty, -2 shape, type or alignment, or a cudaError_t + 1000.
MNCCL_EXPORT int mncclDistillForward(const void* logits, int type, int64_t ld, int T, int V, const int64_t* ids, const float* top, int K,
                                     float tau, float* p, float* stats, float* row_loss, int* counts, float* sum, float* mean, float* tokens,
                                     cudaStream_t stream) {
  if (!logits || !ids || !top || !p || !stats || !row_loss || !counts || !tokens || T <= 0 || V <= 0 || K <= 0) return -1;
  if (std::max(T, V) > kMostIndex || K > kMaxEntries || !good_tau(tau) || (reinterpret_cast<uintptr_t>(stats) & 7u) != 0) return -2;
  switch (type) {
    case 6: return forward<__half>(logits, ld, T, V, ids, top, K, tau, p, stats, row_loss, counts, sum, mean, tokens, stream);
    case 7: return forward<float>(logits, ld, T, V, ids, top, K, tau, p, stats, row_loss, counts, sum, mean, tokens, stream);
    case 9: return forward<__nv_bfloat16>(logits, ld, T, V, ids, top, K, tau, p, stats, row_loss, counts, sum, mean, tokens, stream);
  }
  return -2;
}

// Gradient with respect to the logits, d [T, V] of their type (row stride ldd): of each token's loss times grad[t] (grad_per_row) or
// grad[0], over tokens[0] if that is not null (the mean).
MNCCL_EXPORT int mncclDistillBackward(const void* logits, int type, int64_t ld, int T, int V, const int64_t* ids, const float* p, int K, float tau,
                                      const float* stats, const int* counts, const float* grad, int grad_per_row, const float* tokens,
                                      void* d, int64_t ldd, cudaStream_t stream) {
  if (!logits || !ids || !p || !stats || !counts || !grad || !d || T <= 0 || V <= 0 || K <= 0) return -1;
  if (std::max(T, V) > kMostIndex || K > kMaxEntries || !good_tau(tau) || (reinterpret_cast<uintptr_t>(stats) & 7u) != 0) return -2;
  switch (type) {
    case 6: return backward<__half>(logits, ld, T, V, ids, p, K, tau, stats, counts, grad, grad_per_row, tokens, d, ldd, stream);
    case 7: return backward<float>(logits, ld, T, V, ids, p, K, tau, stats, counts, grad, grad_per_row, tokens, d, ldd, stream);
    case 9: return backward<__nv_bfloat16>(logits, ld, T, V, ids, p, K, tau, stats, counts, grad, grad_per_row, tokens, d, ldd, stream);
  }
  return -2;
}

}  // extern "C"
