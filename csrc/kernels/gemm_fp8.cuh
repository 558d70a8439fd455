// What the kernels of the 8-bit product with block scales share (gemm_fp8.cu, gemm_fp8_small.cu).
//
//   C[m, n] = sum over blocks b of 128 along K of  sa[m / ra, b] * sb[n / rb, b] * P_b[m, n]  (+ bias[n])
//   P_b[m, n] = sum over k in b of a[m, k] * b[n, k]
//
// The tensor cores compute one block's P_b into an accumulator of its own (four tcgen05.mma of kind f8f6f4, K = 32 each);
// "promotion" warps read it from tensor memory, multiply by the scales and add it to sums that they hold in registers.
// So scales are any fp32 numbers, and between blocks everything is added in fp32.  Accumulators alternate: one block is
// promoted while the next ones are multiplied.  The control flow (bounded waits, one elected lane that issues for its
// warp, a producer that stays until its loads have landed) is that of the bf16 kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <string>

#include "kernels/gemm_kernel.cuh"

namespace mnccl {
namespace gemm {
namespace fp8 {

constexpr int kBlockK = 128;                  // elements, and bytes: a 128-byte swizzle row
constexpr int kTileBytes = 128 * kBlockK;     // 128 rows of an operand: 16 KB
constexpr int kMmaK = 32;

// Scales of one operand: element (row >> shift, block) with strides.
struct Scales {
  const float* s;
  int64_t row, blk;
  int shift;
  __device__ __forceinline__ const float* at(int r) const { return s + static_cast<int64_t>(r >> shift) * row; }
};

struct Args {
  int M, N, K;
  Scales a, b;
  void* c;
  int64_t ldc;
  int type;            // of C and bias: 6 fp16, 7 fp32, 9 bf16
  const void* bias;    // null: none
  uint32_t* err;
  uint64_t wait_budget_ns;
};

// kind::f8f6f4, both operands e4m3 and K-major, fp32 accumulation: c_format F32 (1) in bits [4,6), a and b format E4M3 (0),
// N >> 3 in [17,23), M >> 4 in [24,29).
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void umma_e4m3(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_e4m3_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The wait for this thread's tensor-memory loads, tied to the registers they fill: no use of them can move above it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// This lane's row of a block's accumulator, NC columns from `taddr` on, 16 at a time: use(c, values) for each piece while the next one
// is on its way, released() once the last has been read.
template <int NC, typename Use, typename Released>
__device__ __forceinline__ void promote(uint32_t taddr, Use use, Released released) {
  static_assert(NC % 16 == 0, "whole pieces");
  uint32_t r[2][16];
  tmem_ld_32x16(taddr, r[0]);
  tmem_ld_wait(r[0]);
#pragma unroll
  for (int c = 0; c < NC / 16; ++c) {
    if (c + 1 < NC / 16) tmem_ld_32x16(taddr + (c + 1) * 16, r[(c + 1) & 1]);
    else released();
    use(c, r[c & 1]);
    if (c + 1 < NC / 16) tmem_ld_wait(r[(c + 1) & 1]);
  }
}

template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T round_to(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

// A matrix of bytes [rows, cols], boxes of box_rows x 128, 128-byte swizzle, zeros outside.
bool make_tensor_map_e4m3(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t row_stride, uint32_t box_rows, std::string* why);

struct SmallPlan {
  int tn = 0;            // rows of A per tile: 16, 32, 64 or 128
  int slices = 1;        // CTAs of a cluster that share a tile's K
  int kb_per_slice = 0;
  int tiles = 0;
};
bool plan_small(int M, int N, int K, int sms, SmallPlan* p, long* ns);
cudaError_t launch_small(const void* a, int64_t lda, const void* b, int64_t ldb, const Args& g, const SmallPlan& p, cudaStream_t stream, std::string* why);

}  // namespace fp8
}  // namespace gemm
}  // namespace mnccl
