// What the kernels of the 8-bit product with block scales share (gemm_fp8.cu, gemm_fp8_small.cu, gemm_fp8_rows.cu).
//
//   C[m, n] = sum over blocks b of 128 along K of  (sa[m / ra, b] * sb[n / rb, b]) * P_b[m, n]  (+ bias[n])
//   P_b[m, n] = sum over k in b of a[m, k] * b[n, k]
//
// The tensor cores compute one block's P_b into an accumulator of its own (four tcgen05.mma of kind f8f6f4, K = 32 each);
// "promotion" warps read it from tensor memory, multiply by the scales and add it to sums that they hold in registers.
// So scales are any fp32 numbers, and between blocks everything is added in fp32.  All kernels multiply the two scales first, in fp32, and the
// block's sum by that: where the scales' product leaves fp32's range it is infinite or 0 (an infinite one makes a sum of 0 NaN), whatever the sizes of
// the call.  Either order has scales that it loses; this one costs nothing where a scale of B holds for many columns.  Accumulators alternate: one
// block is promoted while the next ones are multiplied.
//
// The control flow (bounded waits, one elected lane that issues for its
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
// A warp of its own brings the scales into shared memory, for this many blocks at a time and a group ahead: a promotion warp that fetched its
// own spent more time on that than on its sums, and a plain load in flight holds up the thread's next arrival on a barrier (which
// releases what came before it): with scales loaded a block ahead the persistent kernel took 1000 cycles a block.
constexpr int kGroup = 8;

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

// 32 lanes x 16, 32 or 64 columns of tensor memory, read and waited for in one statement, so that no use of the registers can come before the
// wait.  (A wait apart that names the registers it covers costs a move for each of them: half of the promotion warps' instructions.)
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}

// This lane's row of a block's accumulator, NC columns from `taddr` on, at most MOST at a time: use(first column, values) for each piece,
// released() once the last has been read.
template <int NC, int MOST, int C = 0, typename Use, typename Released>
__device__ __forceinline__ void promote(uint32_t taddr, Use use, Released released) {
  constexpr int kPiece = MOST >= 64 && NC - C >= 64 ? 64 : NC - C >= 32 ? 32 : 16;
  uint32_t r[kPiece];
  tmem_read(taddr + C, r);
  if constexpr (C + kPiece == NC) released();
  use(C, r);
  if constexpr (C + kPiece < NC) promote<NC, MOST, C + kPiece>(taddr, use, released);
}

// A row's scale times four columns' scales, two at a time (each product rounded for itself): 4096 x 4096 x 4096 on CTA pairs 97 us,
// 104 one at a time.
__device__ __forceinline__ void times_four(const float4& v, float r, float (&x)[4]) {
  asm("{\n\t"
      ".reg .b64 a, b, c;\n\t"
      "mov.b64 c, {%8, %8};\n\t"
      "mov.b64 a, {%4, %5};\n\t"
      "mov.b64 b, {%6, %7};\n\t"
      "mul.rn.f32x2 a, a, c;\n\t"
      "mul.rn.f32x2 b, b, c;\n\t"
      "mov.b64 {%0, %1}, a;\n\t"
      "mov.b64 {%2, %3}, b;\n\t"
      "}\n"
      : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
      : "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "f"(r));
}

// Whether a barrier's phase is over, without waiting.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// Four bytes, global -> shared, without the thread waiting for them; an arrival on `bar` (counted among those it expects) when all of this
// thread's copies so far have landed.
__device__ __forceinline__ void copy4_async(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Two waits that take one trip where both phases are over already.
__device__ __forceinline__ bool mbar_wait_both(uint32_t bar, uint32_t parity, uint32_t bar2, uint32_t parity2, volatile uint32_t* abort_flag, uint64_t budget_ns) {
  const bool first = mbar_try_wait(bar, parity), second = mbar_try_wait(bar2, parity2);
  if (__all_sync(0xffffffffu, first && second)) return true;
  return mbar_wait_warp(bar, parity, abort_flag, budget_ns) && mbar_wait_warp(bar2, parity2, abort_flag, budget_ns);
}

// Tiled store shared -> global, tracked by bulk async-groups; what lies outside the tensor is not written, but for the rest of the 16 bytes in which a row
// of it ends (seen on a B200: columns behind the last, up to a multiple of 16 bytes, came out overwritten).
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t smem_src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem_src), "r"(c0),
               "r"(c1)
               : "memory");
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

// One result, and its column's bias.
__device__ __forceinline__ void store(const Args& g, int m, int n, float v) {
  if (m >= g.M || n >= g.N) return;
  const size_t at = static_cast<size_t>(m) * g.ldc + n;
  switch (g.type) {
    case 6: static_cast<__half*>(g.c)[at] = __float2half_rn(v); break;
    case 7: static_cast<float*>(g.c)[at] = v; break;
    default: static_cast<__nv_bfloat16*>(g.c)[at] = __float2bfloat16_rn(v);
  }
}
__device__ __forceinline__ float bias_of(const Args& g, int n) {
  if (g.bias == nullptr || n >= g.N) return 0.0f;
  switch (g.type) {
    case 6: return __half2float(static_cast<const __half*>(g.bias)[n]);
    case 7: return static_cast<const float*>(g.bias)[n];
    default: return __bfloat162float(static_cast<const __nv_bfloat16*>(g.bias)[n]);
  }
}

// A matrix of bytes [rows, cols], boxes of box_rows x 128, 128-byte swizzle, zeros outside.
bool make_tensor_map_e4m3(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t row_stride, uint32_t box_rows, std::string* why);

struct SmallPlan {
  int tn = 0;            // rows of A per tile: 16, 32 or 64
  int slices = 1;        // CTAs of a cluster that share a tile's K
  int kb_per_slice = 0;
  int tiles = 0;
  bool deep = false;     // one CTA per SM with the whole shared memory as its ring, or two
};
bool plan_small(int M, int N, int K, int sms, SmallPlan* p, long* ns);
// The kernel for up to four rows of A, and its estimated time.
long rows_ns(int M, int N, int K);
cudaError_t launch_rows(const void* a, int64_t lda, const void* b, int64_t ldb, const Args& g, cudaStream_t stream);
cudaError_t launch_small(const void* a, int64_t lda, const void* b, int64_t ldb, const Args& g, const SmallPlan& p, cudaStream_t stream, std::string* why);

}  // namespace fp8
}  // namespace gemm
}  // namespace mnccl
