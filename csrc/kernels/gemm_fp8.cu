// C[M, N] = A[M, K] * B[N, K]^T (+ bias) for e4m3 operands with a scale for each block of 128 along K:
//
//   C[m, n] = sum over blocks b of  sa[m / ra, b] * sb[n / rb, b] * sum over k in b of  a[m, k] * b[n, k]
//
// ra and rb (rows of a scale) are 1 or 128.  Products of e4m3 numbers and a block's sum are taken in fp32, scaled and added
// in fp32; one rounding to C's type, behind the bias.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace {

constexpr int kBlock = 128;

struct Args {
  const uint8_t *a, *b;
  int64_t lda, ldb, ldc;
  int M, N, K;
  const float *sa, *sb;
  int64_t sa_row, sa_blk, sb_row, sb_blk;
  int a_shift, b_shift;   // rows of a scale: 2^shift
  void* c;
  const void* bias;
};

__device__ __forceinline__ float e4m3(uint8_t v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
}

// 64 x 64 outputs a block, 4 x 4 a thread.
template <typename T>
__global__ void __launch_bounds__(256) gemm_fp8_kernel(const Args g) {
  __shared__ float as[32][65], bs[32][65];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int m0 = static_cast<int>(blockIdx.x) * 64, n0 = static_cast<int>(blockIdx.y) * 64;
  float acc[4][4] = {};
  for (int b = 0; b * kBlock < g.K; ++b) {
    float sum[4][4] = {};
    for (int k0 = b * kBlock; k0 < min(g.K, (b + 1) * kBlock); k0 += 32) {
      for (int i = threadIdx.x; i < 64 * 32; i += 256) {
        const int r = i >> 5, k = i & 31;
        as[k][r] = m0 + r < g.M && k0 + k < g.K ? e4m3(g.a[(m0 + r) * g.lda + k0 + k]) : 0.0f;
        bs[k][r] = n0 + r < g.N && k0 + k < g.K ? e4m3(g.b[(n0 + r) * g.ldb + k0 + k]) : 0.0f;
      }
      __syncthreads();
      for (int k = 0; k < 32; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[i][j] += as[k][ty * 4 + i] * bs[k][tx * 4 + j];
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = min(m0 + ty * 4 + i, g.M - 1), n = min(n0 + tx * 4 + j, g.N - 1);
        acc[i][j] += g.sa[(m >> g.a_shift) * g.sa_row + b * g.sa_blk] * g.sb[(n >> g.b_shift) * g.sb_row + b * g.sb_blk] * sum[i][j];
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= g.M || n >= g.N) continue;
      const float v = acc[i][j] + (g.bias ? static_cast<float>(static_cast<const T*>(g.bias)[n]) : 0.0f);
      static_cast<T*>(g.c)[m * g.ldc + n] = static_cast<T>(v);
    }
}

}  // namespace

extern "C" {
#define MNCCL_EXPORT __attribute__((visibility("default")))

// a [M, K], b [N, K] e4m3, 16-byte aligned, row strides multiples of 16; scales with their strides (row of scales, block along K) and rows
// of a scale (1 or 128); C and bias (null: none) of type 6 fp16, 7 fp32 or 9 bf16.
// Returns 0, -1 null or empty, -2 shape or alignment, -3 tensor map, or a cudaError_t + 1000.
MNCCL_EXPORT int mncclGemmFp8(const void* a, int64_t lda, const float* sa, int64_t sa_row, int64_t sa_blk, int sa_rows, const void* b,
                              int64_t ldb, const float* sb, int64_t sb_row, int64_t sb_blk, int sb_rows, void* c, int64_t ldc, int type,
                              const void* bias, int M, int N, int K, cudaStream_t stream) {
  if (!a || !b || !c || !sa || !sb || M <= 0 || N <= 0 || K <= 0) return -1;
  const auto operand = [K](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 16 == 0 && ld >= K; };
  if (!operand(a, lda) || !operand(b, ldb) || ldc < N) return -2;
  if ((sa_rows != 1 && sa_rows != kBlock) || (sb_rows != 1 && sb_rows != kBlock)) return -2;
  const Args g{static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(b), lda, ldb, ldc, M, N, K, sa, sb, sa_row, sa_blk, sb_row, sb_blk,
               sa_rows == 1 ? 0 : 7, sb_rows == 1 ? 0 : 7, c, bias};
  const dim3 grid((M + 63) / 64, (N + 63) / 64);
  switch (type) {
    case 6: gemm_fp8_kernel<__half><<<grid, 256, 0, stream>>>(g); break;
    case 7: gemm_fp8_kernel<float><<<grid, 256, 0, stream>>>(g); break;
    case 9: gemm_fp8_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(g); break;
    default: return -2;
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : static_cast<int>(e) + 1000;
}

}  // extern "C"
