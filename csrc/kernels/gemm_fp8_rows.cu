// The 8-bit product with block scales for up to four tokens and a small weight, without tensor cores: the weight goes from memory through registers,
// once, with nothing staged.
//
// A CTA takes eight rows of B and all of K, its warps 512 bytes of K each: a lane has eight 16-byte loads in flight, one for each row, widens A's
// bytes once for all rows to fp16, which holds every e4m3 value, and multiplies and adds in fp32 (fma.rn.f32.f16: the products are exact).
// Eight lanes hold a block of 128: their sums are reduced and dealt out over them together, seven shuffles for the eight rows, so
// that each lane ends with one whole block's sum, which it scales.  The warps meet in shared memory and are added in order.
//
// The tensor-core kernel for few rows spends more than a microsecond more on descriptors, barriers, tensor memory and the meeting of its slices, which
// this one saves; then this one runs at 4.6 TB/s for one token, bound by its instructions (two for three bytes), at 4 for two and at 2.3 for
// four, and that one at up to 5.5.  Measured in graphs, calls that follow one another (and overlap at their ends, dependent_launch.cuh), weights not in the L2
// (this kernel / that one, us): 1 x 1024 x 1024 2.1 / 3.5, 1 x 4096 x 1024 3.0 / 4.1, 1 x 4096 x 4096 5.5 / 6.7, 1 x 14336 x 4096 14.7 / 12.3; 2 x 4096 x 4096
// 6.5 / 7.0; 4 x 1024 x 1024 2.5 / 4.0, 4 x 4096 x 4096 9.7 / 7.4.  The same weight over and over, which then lies in the L2, 1 x 4096 x 4096: 3.9.  rows_ns is
// fitted to a kernel by itself and a weight from memory (5.8 there).  64 registers and 1024 threads an SM matter: with 80, 1 x 4096 x 4096 took 7.1 us by
// itself.  (Widening to fp32 took 7.8, mma.sync m16n8k32 of the same bytes 7.5 for 8 tokens and 20.1 at 14336.)
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "kernels/dependent_launch.cuh"
#include "kernels/gemm_fp8.cuh"

namespace mnccl {
namespace gemm {
namespace fp8 {

namespace {

constexpr int kRows = 8, kSpan = 512, kMostWarps = 8;   // rows of B a CTA, bytes of K a warp at a time

// 16 bytes of a row from column k on; columns from K on read as zero.
__device__ __forceinline__ uint4 load16(const uint8_t* row, int64_t k, int K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k + 16 <= K) {
    v = load_vector(row + k);
  } else if (k < K) {
    uint32_t w[4] = {};
    for (int i = 0; k + i < K; ++i) w[i >> 2] |= static_cast<uint32_t>(row[k + i]) << (i & 3) * 8;
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
__device__ __forceinline__ void widen(const uint4& v, __half2_raw (&h)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (i & 1) * 16), __NV_E4M3);
}
__device__ __forceinline__ void fma_f16(float& d, unsigned short x, unsigned short y) {
  asm("fma.rn.f32.f16 %0, %1, %2, %0;" : "+f"(d) : "h"(x), "h"(y));
}

template <int TM>
__global__ void __launch_bounds__(32 * kMostWarps, TM <= 2 ? 4 : 2)
    gemm_fp8_rows_kernel(const uint8_t* a, int64_t lda, const uint8_t* b, int64_t ldb, const __grid_constant__ Args g) {
  __shared__ float part[kMostWarps][kRows][TM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int n0 = blockIdx.x * kRows, num_kb = (g.K + kBlockK - 1) / kBlockK;
  const int own = n0 + (lane & 7) * kRows / 8;   // the row of B whose blocks this lane scales
  float acc[TM] = {};
  wait_for_previous();
  let_next_start();
  a = since_wait(a);
  b = since_wait(b);
  for (int64_t k0 = static_cast<int64_t>(warp) * kSpan; k0 < g.K; k0 += static_cast<int64_t>(warps) * kSpan) {
    uint4 w[kRows], x[TM];
#pragma unroll
    for (int r = 0; r < kRows; ++r) w[r] = load16(b + static_cast<int64_t>(min(n0 + r, g.N - 1)) * ldb, k0 + lane * 16, g.K);
#pragma unroll
    for (int m = 0; m < TM; ++m) x[m] = load16(a + static_cast<int64_t>(min(m, g.M - 1)) * lda, k0 + lane * 16, g.K);
    const int64_t kb = k0 / kBlockK + (lane >> 3);
    float sb = 0.0f, sa[TM] = {};
    if (kb < num_kb) {
      sb = g.b.at(min(own, g.N - 1))[kb * g.b.blk];
#pragma unroll
      for (int m = 0; m < TM; ++m) sa[m] = g.a.at(min(m, g.M - 1))[kb * g.a.blk];
    }
    float s[TM][kRows];   // sums of 16 products
    __half2_raw xh[TM][8];
#pragma unroll
    for (int m = 0; m < TM; ++m) widen(x[m], xh[m]);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      __half2_raw wh[8];
      widen(w[r], wh);
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        float even = 0.0f, odd = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          fma_f16(even, wh[i].x, xh[m][i].x);
          fma_f16(odd, wh[i].y, xh[m][i].y);
        }
        s[m][r] = even + odd;
      }
    }
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      // eight lanes hold a block: in each step half of the rows left go to the lane that keeps them
      int left = kRows;
#pragma unroll
      for (int d = 4; d > 0; d >>= 1) {
        const bool upper = (lane & d) != 0;
        if (left > 1) {
          left /= 2;
#pragma unroll
          for (int j = 0; j < left; ++j) {
            const float give = upper ? s[m][j] : s[m][j + left];
            s[m][j] = (upper ? s[m][j + left] : s[m][j]) + __shfl_xor_sync(0xffffffffu, give, d);
          }
        } else {
          s[m][0] += __shfl_xor_sync(0xffffffffu, s[m][0], d);
        }
      }
      if (kb < num_kb) acc[m] += s[m][0] * (sa[m] * sb);
    }
  }
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], 8);
    acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], 16);
    if (lane < 8 && lane % (8 / kRows) == 0) part[warp][lane * kRows / 8][m] = acc[m];
  }
  __syncthreads();
  const int r = threadIdx.x / TM, m = threadIdx.x % TM, n = n0 + r;
  if (r < kRows && m < g.M && n < g.N) {
    float v = part[0][r][m];
    for (int i = 1; i < warps; ++i) v += part[i][r][m];
    store(g, m, n, v + bias_of(g, n));
  }
}

}  // namespace

long rows_ns(int M, int N, int K) {
  if (M > 4) return 1L << 62;
  const double bytes = static_cast<double>(N) * K;
  return M == 1 ? 2300 + static_cast<long>(bytes * 0.207e-3) : M == 2 ? 2300 + static_cast<long>(bytes * 0.255e-3) : 2500 + static_cast<long>(bytes * 0.43e-3);
}

cudaError_t launch_rows(const void* a, int64_t lda, const void* b, int64_t ldb, const Args& g, cudaStream_t stream) {
  const int spans = (g.K + kSpan - 1) / kSpan;
  const dim3 grid((g.N + kRows - 1) / kRows), block(32 * std::min(spans, kMostWarps));
  const auto* pa = static_cast<const uint8_t*>(a);
  const auto* pb = static_cast<const uint8_t*>(b);
  if (g.M == 1) return launch_early(gemm_fp8_rows_kernel<1>, grid, block, stream, pa, lda, pb, ldb, g);
  if (g.M == 2) return launch_early(gemm_fp8_rows_kernel<2>, grid, block, stream, pa, lda, pb, ldb, g);
  return launch_early(gemm_fp8_rows_kernel<4>, grid, block, stream, pa, lda, pb, ldb, g);
}

}  // namespace fp8
}  // namespace gemm
}  // namespace mnccl
