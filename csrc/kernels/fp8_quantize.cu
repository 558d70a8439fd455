// Quantisation to e4m3 with one scale for each block of 128 elements of a row, or of 128 x 128 elements.
//
//   a = max |x| over the block,  s = 2^e with the smallest e >= -126 for which 448 * 2^e >= a,  q = e4m3(x / s)
//
// 448 is e4m3's largest value.  The scale is a power of two: x / s is then exact, so the only rounding is the one
// to e4m3 (to nearest, ties to even, at most 2^-4 of the value, or 2^-10 * s below e4m3's normal numbers), and the
// result does not depend on how a quotient is rounded.  It costs nothing else, since e4m3 has the same relative step
// everywhere.  A block that holds an infinity or a NaN has the scale NaN and NaN for its values: it cannot be
// represented, and every product that touches it says so.
//
// What bounds it is memory: 2 bytes read and 1 written an element (bf16), 4 read for fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace {

constexpr int kBlock = 128;
constexpr int kThreads = 256;

// Bits of |x| as an fp32 number: their order is that of the magnitudes, with infinity and NaN above all else.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct Scale {
  float scale, inverse;
};
__device__ __forceinline__ Scale scale_of(uint32_t top) {
  if (top >= 0x7f800000u) {
    const float nan = __uint_as_float(0x7fffffffu);
    return {nan, nan};
  }
  // top = 1.m * 2^E and 448 = 1.75 * 2^8
  const int biased = max(static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), 1);
  return {__uint_as_float(static_cast<uint32_t>(biased) << 23), __uint_as_float(static_cast<uint32_t>(254 - biased) << 23)};
}

template <typename T>
__device__ __forceinline__ float as_float(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(x);
  else return __bfloat162float(x);
}

// Elements [c, c + 8) of a row of K, zeros beyond its end.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int c, int K, bool vec, float (&f)[8]) {
  if (vec && c + 8 <= K) {
    T v[8];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(row + c) + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = as_float(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = c + j < K ? as_float(row[c + j]) : 0.0f;
  }
}

__device__ __forceinline__ uint2 quantise8(const float (&f)[8], float inverse) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i] * inverse, f[4 * i + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2] * inverse, f[4 * i + 3] * inverse), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// 1 x 128 blocks.  16 lanes hold a block, 8 elements each; a thread block takes one block of 16 neighbouring rows, whose
// scales are 64 contiguous bytes: scales are stored [K blocks][M].
template <typename T>
__global__ void __launch_bounds__(kThreads)
quantise_rows_kernel(const T* __restrict__ x, size_t ldx, int M, int K, uint8_t* __restrict__ q, size_t ldq, float* __restrict__ scale, bool vec) {
  const int m = static_cast<int>(blockIdx.x) * 16 + static_cast<int>(threadIdx.x >> 4);
  const int c = static_cast<int>(blockIdx.y) * kBlock + static_cast<int>(threadIdx.x & 15) * 8;
  if (m >= M) return;   // all 16 lanes of a block
  float f[8];
  load8(x + m * ldx, c, K, vec, f);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, magnitude(f[j]));
  const uint32_t lanes = 0xffffu << (threadIdx.x & 16);
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(lanes, top, d));
  const Scale s = scale_of(top);
  // (q's rows are padded to 16 bytes)
  if (c < K) *reinterpret_cast<uint2*>(q + m * ldq + c) = quantise8(f, s.inverse);
  if ((threadIdx.x & 15) == 0) scale[static_cast<size_t>(blockIdx.y) * M + m] = s.scale;
}

// A tile of 128 x 128 elements, which holds whole blocks of either kind along both dimensions: x is read once for q and
// the transpose qt.  A thread holds 4 neighbouring rows of 2 x 8 columns, so that 4 elements of a column are one word of
// the transposed tile in shared memory, [column][32 words + 1].
constexpr int kPitch = 33;

template <typename T, bool SQUARE>
__global__ void __launch_bounds__(kThreads)
quantise_tile_kernel(const T* __restrict__ x, size_t ldx, int M, int K, uint8_t* __restrict__ q, size_t ldq, float* __restrict__ scale,
                     uint8_t* __restrict__ qt, size_t ldt, float* __restrict__ scale_t, bool vec) {
  __shared__ uint32_t tile[kBlock * kPitch];
  __shared__ uint32_t part[8][kBlock];   // a warp's largest magnitude of each column
  __shared__ float inverse[kBlock];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = static_cast<int>(blockIdx.x) * kBlock, k0 = static_cast<int>(blockIdx.y) * kBlock;
  const int r0 = warp * 16 + (lane >> 3) * 4, c0 = (lane & 7) * 8;   // columns c0 .. and c0 + 64 ..
  float f[4][2][8];
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + r0 + i;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (m < M) load8(x + m * ldx, k0 + c0 + h * 64, K, vec, f[i][h]);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][h][j] = 0.0f;
    }
  }
  Scale s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, magnitude(f[i][h][j]));
    if constexpr (SQUARE) {
      all = max(all, top);
    } else {
#pragma unroll
      for (int d = 4; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
      s[i] = scale_of(top);
      if ((lane & 7) == 0 && m0 + r0 + i < M) scale[static_cast<size_t>(blockIdx.y) * M + m0 + r0 + i] = s[i].scale;
    }
  }
  if constexpr (SQUARE) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) all = max(all, __shfl_xor_sync(0xffffffffu, all, d));
    if (lane == 0) part[0][warp] = all;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) all = max(all, part[0][w]);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = scale_of(all);
    if (threadIdx.x == 0) scale[static_cast<size_t>(blockIdx.x) * gridDim.y + blockIdx.y] = s[0].scale;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = k0 + c0 + h * 64;
      if (m0 + r0 + i < M && c < K)
        *reinterpret_cast<uint2*>(q + static_cast<size_t>(m0 + r0 + i) * ldq + c) = quantise8(f[i][h], s[i].inverse);
    }
  if (qt == nullptr) return;
  if constexpr (!SQUARE) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, magnitude(f[i][h][j]));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
        if (lane < 8) part[warp][c0 + h * 64 + j] = top;
      }
    __syncthreads();
    if (threadIdx.x < kBlock) {
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) top = max(top, part[w][threadIdx.x]);
      const Scale t = scale_of(top);
      inverse[threadIdx.x] = t.inverse;
      if (k0 + static_cast<int>(threadIdx.x) < K) scale_t[static_cast<size_t>(blockIdx.x) * K + k0 + threadIdx.x] = t.scale;
    }
    __syncthreads();
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = c0 + h * 64 + j;
      const float v = SQUARE ? s[0].inverse : inverse[c];
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0][h][j] * v, f[1][h][j] * v), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2][h][j] * v, f[3][h][j] * v), __NV_SATFINITE, __NV_E4M3);
      tile[c * kPitch + r0 / 4] = lo | (hi << 16);
    }
  __syncthreads();
#pragma unroll 4
  for (int c = warp; c < kBlock; c += 8)   // a column leaves as 128 bytes; rows of qt are padded to 16
    if (k0 + c < K && m0 + lane * 4 < static_cast<int>(ldt))
      *reinterpret_cast<uint32_t*>(qt + static_cast<size_t>(k0 + c) * ldt + m0 + lane * 4) = tile[c * kPitch + lane];
}

template <typename T>
int quantise(const T* x, int64_t ldx, int M, int K, int block_rows, uint8_t* q, int64_t ldq, float* scale, uint8_t* qt, int64_t ldt, float* scale_t,
             cudaStream_t stream) {
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (ldx * static_cast<int64_t>(sizeof(T))) % 16 == 0;
  const int blocks_k = (K + kBlock - 1) / kBlock;
  if (block_rows == 1 && qt == nullptr) {
    quantise_rows_kernel<T><<<dim3((M + 15) / 16, blocks_k), kThreads, 0, stream>>>(x, ldx, M, K, q, ldq, scale, vec);
  } else {
    const dim3 grid((M + kBlock - 1) / kBlock, blocks_k);
    if (block_rows == 1) quantise_tile_kernel<T, false><<<grid, kThreads, 0, stream>>>(x, ldx, M, K, q, ldq, scale, qt, ldt, scale_t, vec);
    else quantise_tile_kernel<T, true><<<grid, kThreads, 0, stream>>>(x, ldx, M, K, q, ldq, scale, qt, ldt, scale_t, vec);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : static_cast<int>(e) + 1000;
}

constexpr int kMaxK = 65535 * kBlock;   // gridDim.y

}  // namespace

extern "C" {
#define MNCCL_EXPORT __attribute__((visibility("default")))

// x [M, K] (type 6 fp16, 7 fp32, 9 bf16; row stride ldx elements) -> q [M, K] e4m3 (row stride ldq, a multiple of 16 that holds K
// rounded up to one; 16-byte aligned; the padding is written) and its scales: block_rows 1: scale[K blocks][M]; block_rows 128:
// scale[M blocks][K blocks].  qt, if not null: the transpose [K, M] (ldt like ldq), for block_rows 1 quantised anew in blocks along M
// with scale_t[M blocks][K].  Returns 0, -1 null or empty, -2 shape or alignment, or a cudaError_t + 1000.
MNCCL_EXPORT int mncclQuantizeFp8(const void* x, int type, int64_t ldx, int M, int K, int block_rows, void* q, int64_t ldq, float* scale,
                                  void* qt, int64_t ldt, float* scale_t, cudaStream_t stream) {
  if (!x || !q || !scale || M <= 0 || K <= 0 || (qt && block_rows == 1 && !scale_t)) return -1;
  const auto padded = [](const void* p, int64_t ld, int64_t n) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 16 == 0 && ld >= (n + 15) / 16 * 16;
  };
  if ((block_rows != 1 && block_rows != kBlock) || ldx < K || K > kMaxK || M > 0x7fffff00 || !padded(q, ldq, K) || (qt && !padded(qt, ldt, M)))
    return -2;
  uint8_t* qb = static_cast<uint8_t*>(q);
  uint8_t* tb = static_cast<uint8_t*>(qt);
  switch (type) {
    case 6: return quantise(static_cast<const __half*>(x), ldx, M, K, block_rows, qb, ldq, scale, tb, ldt, scale_t, stream);
    case 7: return quantise(static_cast<const float*>(x), ldx, M, K, block_rows, qb, ldq, scale, tb, ldt, scale_t, stream);
    case 9: return quantise(static_cast<const __nv_bfloat16*>(x), ldx, M, K, block_rows, qb, ldq, scale, tb, ldt, scale_t, stream);
  }
  return -2;
}

}  // extern "C"
