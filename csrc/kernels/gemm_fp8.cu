// C[M, N] = A[M, K] * B[N, K]^T (+ bias) for e4m3 operands with a scale for each block of 128 along K (gemm_fp8.cuh has the
// formula and the division of labour), for products that fill the GPU; gemm_fp8_small.cu has the others.
//
// Persistent clusters of two CTAs: tcgen05.mma.cta_group::2 computes the P_b of a 256 x BN tile on two SMs, each CTA loads 128 rows of A and
// half of the tile's rows of B (32 KB a block of K for BN = 256, which is what lets L2 keep up) and holds the sums of its 128 rows:
//
//   both CTAs   warp 0      TMA producer; bytes are counted on the leader's barriers
//   leader      warps 1, 2  for half of the tile's columns each, one lane issues the four MMAs of a block into one of two accumulators (four
//                           for tiles of up to 128 columns) and commits:
//                           the ring stage and the half's accumulator.  Halves are handed over by themselves, so that the tensor cores
//                           work on one while the other is being read
//   both CTAs   warp 3      brings the scales
//   both CTAs   warps 4-11  promotion: two warps for each quarter of tensor memory's lanes, half of the columns each; a lane holds the sums
//                           of its row and BN / 2 columns in registers, then adds the bias, rounds and stores them
//
// The tensor cores take 512 cycles for a block of 128 x 256 x 128 an SM; reading it (64 KB from tensor memory) and 256 fused multiply-adds
// a scheduler overlap with the next block.  Where B has a scale for every row (the gradient of a weight) every column has a product of scales of
// its own, which costs a read of shared memory and half an instruction a warp and column: 4096 x 4096 x 4096 takes 97 us against 69.
//
// What bounds it: the hand-over of accumulators at short clocks, and power in long runs.  4096 x 14336 x 4096 (481 GFLOP) takes 227 us in short bursts,
// 2.1 PFLOP/s, and 275 repeated for seconds; 8192 x 4096 x 1024 41 us, where each tile's first block and its 128 KB of results count most.
#include <algorithm>
#include <cstdio>

#include "kernels/dependent_launch.cuh"
#include "kernels/gemm_fp8.cuh"
#include "mem/cuda_driver.h"

namespace mnccl {
namespace gemm {
namespace fp8 {

bool make_tensor_map_e4m3(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t row_stride, uint32_t box_rows, std::string* why) {
  const CudaDriver* d = CudaDriver::get();
  if (!d || !d->TensorMapEncodeTiled) {
    *why = "cuTensorMapEncodeTiled unavailable";
    return false;
  }
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {row_stride};
  cuuint32_t box[2] = {kBlockK, box_rows};
  cuuint32_t estr[2] = {1, 1};
  const auto encode = [&] {
    return d->TensorMapEncodeTiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  int dev = 0;
  // a thread's first call: the runtime binds its device's context when it is told the device
  if (r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
  if (r != CUDA_SUCCESS) {
    *why = "cuTensorMapEncodeTiled: " + d->error_string(r);
    return false;
  }
  return true;
}

namespace {

constexpr int kPromoters = 8;                                  // warps
constexpr int kFirst = 4;                                      // first promotion warp: register counts are set for four warps at a time
constexpr int kPairThreads = 32 * (kFirst + kPromoters);
// 384 threads start with 168 registers each; what the control warps give back (128 * 96) is what the promotion warps take (256 * 48).
constexpr int kControlRegs = 72, kPromoterRegs = 216;
static_assert(128 * kControlRegs + 32 * kPromoters * kPromoterRegs <= kPairThreads * 168, "registers the block was launched with");
constexpr int kOutRow = 64;                                    // bytes of a row of a piece of the result on its way out
constexpr int kPieceBytes = 32 * kOutRow;
constexpr int kScratchBytes = 2 * kPieceBytes;                 // per promotion warp: two pieces
constexpr int kBiasFloats = 128;                               // per promotion warp: of its columns
template <int BN>
constexpr int kPairStage = kTileBytes + BN / 2 * kBlockK;      // this CTA's 128 rows of A and BN / 2 rows of B

constexpr int kStages = 5;                                     // (seven for the narrow tiles, which shared memory would hold, changed nothing)
template <int BN, bool B_ROWS>
constexpr int kCols = B_ROWS ? BN : 4;                         // scales of B a block: of the tile's columns, or of the two blocks of rows that a half touches
template <int BN, bool B_ROWS>
constexpr int kSlot = kGroup * (128 + kCols<BN, B_ROWS>);      // floats: a group's scales

template <int BN>
constexpr uint32_t kBuffers = BN <= 128 ? 4 : 2;               // accumulators in tensor memory (256 x 4096 x 4096 with 128 columns: 16.2 -> 15.4 us)

struct __align__(16) PairCtl {
  uint64_t full[kStages];        // used in the leader: 2 arrivals (one per producer) and both CTAs' bytes
  uint64_t empty[kStages];       // one per CTA, released by the leader's two commits
  uint64_t acc_full[4][2];       // [accumulator][half of the tile's columns], one per CTA
  uint64_t acc_empty[4][2];      // used in the leader: the half's four promotion warps of both CTAs
  uint64_t scales_full[2];       // 32 arrivals: the lanes of the warp that brings them
  uint64_t scales_empty[2];      // the promotion warps
  uint32_t tmem_base;
  volatile uint32_t abort;
};

// 256 x BN tiles, in groups of four rows of tiles that share B's tiles in L2.
struct Tiles {
  int m, n;
  __device__ __forceinline__ void at(int t, int* tm, int* tn) const {
    constexpr int kGroup = 4;
    const int group = t / (kGroup * n), first = group * kGroup, rows = min(m - first, kGroup), in = t - group * kGroup * n;
    *tm = first + in % rows;
    *tn = in / rows;
  }
};

// The bias of a warp's NC columns, into its shared memory before a tile's first block is there.
template <typename T, int NC>
__device__ __forceinline__ void load_bias(const Args& g, int col, float* bias, int lane) {
  const T* b = static_cast<const T*>(g.bias);
  __syncwarp();   // the tile before has been stored
#pragma unroll
  for (int j = 0; j < NC / 32; ++j) bias[j * 32 + lane] = to_float(b[min(col + j * 32 + lane, g.N - 1)]);
  __syncwarp();
}

// A lane's NC sums of row `row`, columns [col, col + NC): bias, one rounding, out.  With a tensor map of C a warp's 32 rows leave as pieces of 64
// bytes a row that it lays out in shared memory (64-byte swizzle: no bank conflicts) and the TMA unit writes while the next tile is
// begun.  (Each lane storing its own row, 32 bytes at a time, held the tensor cores up for a fifth of the time at K = 4096 and for two fifths
// at K = 1024.)  `pieces` counts them over all of the warp's tiles: the two places in shared memory alternate, so a place is free once all stores
// but the latest have been read, and a tile may have an odd number of them (192 or 64 columns of a 16-bit type; a ragged right edge).
template <typename T, int NC>
__device__ __forceinline__ void store_rows(const Args& g, const CUtensorMap* map, bool mapped, int row, int col, float (&acc)[NC], uint8_t* scratch, uint32_t& pieces, const float* bias, int lane) {
  const int row_base = row - lane;
  if (row_base >= g.M) return;   // the same for the whole warp
  if (g.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < NC; j += 4) {
      const float4 v = *reinterpret_cast<const float4*>(bias + j);
      acc[j] += v.x;
      acc[j + 1] += v.y;
      acc[j + 2] += v.z;
      acc[j + 3] += v.w;
    }
  }
  if (mapped) {
    constexpr int kPer = kOutRow / static_cast<int>(sizeof(T)), kChunk = 16 / static_cast<int>(sizeof(T));
    // The TMA unit cuts a row off behind the 16 bytes that hold the tensor's last column: where these hold columns behind the result as well, the warp
    // stores the last piece by itself.
    const bool ragged = g.N % kChunk != 0;
    uint8_t* piece = scratch;
#pragma unroll
    for (int p = 0; p < NC / kPer; ++p) {
      if (col + p * kPer >= g.N) break;
      piece = scratch + (pieces++ & 1u) * kPieceBytes;
      if (lane == 0) bulk_wait_read<1>();   // the piece before the last has been read
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        union { T x[kChunk]; uint4 w; } u;
#pragma unroll
        for (int k = 0; k < kChunk; ++k) u.x[k] = round_to<T>(acc[p * kPer + c * kChunk + k]);
        *reinterpret_cast<uint4*>(piece + lane * kOutRow + ((c ^ (lane >> 1)) & 3) * 16) = u.w;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {   // (a group of nothing for a piece that does not go out so: groups are counted as pieces are)
        if (!ragged || col + (p + 1) * kPer <= g.N) tma_store_2d(map, smem_u32(piece), col + p * kPer, row_base);
        bulk_commit();
      }
    }
    if (ragged && g.N - col < NC) {
      const int n = g.N / kPer * kPer;   // the last piece's first column
      T* c = static_cast<T*>(g.c) + static_cast<size_t>(row_base) * g.ldc + n;
      for (int i = lane; i < 32 * kPer; i += 32) {
        const int r = i / kPer, k = i % kPer;
        if (row_base + r < g.M && n + k < g.N)
          c[static_cast<size_t>(r) * g.ldc + k] = reinterpret_cast<const T*>(piece + r * kOutRow + ((k / kChunk ^ (r >> 1)) & 3) * 16)[k % kChunk];
      }
    }
    return;
  }
  // Rows that start anywhere: 32 rows of 32 columns at a time through shared memory (column j of row r at j ^ r: no bank conflicts either way), a row
  // per instruction.
  T* c = static_cast<T*>(g.c) + static_cast<size_t>(row_base) * g.ldc;
  float* square = reinterpret_cast<float*>(scratch);
  const int rows = min(32, g.M - row_base);
#pragma unroll
  for (int p = 0; p < NC / 32; ++p) {
#pragma unroll
    for (int j = 0; j < 32; ++j) square[lane * 32 + (j ^ lane)] = acc[p * 32 + j];
    __syncwarp();
    const int n = col + p * 32 + lane;
    if (n < g.N) {
#pragma unroll 8
      for (int r = 0; r < rows; ++r) c[static_cast<size_t>(r) * g.ldc + n] = round_to<T>(square[r * 32 + (lane ^ r)]);
    }
    __syncwarp();
  }
}

// B_ROWS: B has a scale for every row instead of for 128.
template <int BN, bool B_ROWS>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, const __grid_constant__ CUtensorMap tma_c,
                     const __grid_constant__ Args g, bool mapped) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int NS = kStages, NC = BN / 2;
  constexpr uint32_t NB = kBuffers<BN>;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  uint8_t* scratch_all = smem + NS * kPairStage<BN>;      // per promotion warp
  PairCtl* ctl = reinterpret_cast<PairCtl*>(scratch_all + kPromoters * kScratchBytes);
  float* slots = reinterpret_cast<float*>(ctl + 1);      // [2][kGroup][128 rows], then [kGroup][kCols], each
  float* bias_all = slots + 2 * kSlot<BN, B_ROWS>;      // per promotion warp

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();   // 0: leader
  const int pair = static_cast<int>(blockIdx.x) >> 1, n_pairs = static_cast<int>(gridDim.x) >> 1;
  const Tiles tiles{(g.M + 255) / 256, (g.N + BN - 1) / BN};
  const int num_tiles = tiles.m * tiles.n;
  const int num_kb = (g.K + kBlockK - 1) / kBlockK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(smem_u32(&ctl->full[s]), 2);
      mbar_init(smem_u32(&ctl->empty[s]), 2);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&ctl->scales_full[b]), 32);
      mbar_init(smem_u32(&ctl->scales_empty[b]), kPromoters);
    }
    for (int b = 0; b < 2 * static_cast<int>(NB); ++b) {
      mbar_init(smem_u32(&ctl->acc_full[b >> 1][b & 1]), 1);
      mbar_init(smem_u32(&ctl->acc_empty[b >> 1][b & 1]), kPromoters);
    }
    ctl->abort = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tma_a);
    prefetch_tensormap(&tma_b);
    if (mapped) prefetch_tensormap(&tma_c);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&ctl->tmem_base), kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();   // the partner's barriers exist before anything arrives on them
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  wait_for_previous();
  let_next_start();
  const uint64_t budget = g.wait_budget_ns;
  const bool leader = elect_one();   // the lane that issues for its warp

  if (warp < kFirst) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
    if (warp == 0) {
      uint32_t it = 0, s = 0, ph = 1;   // ring position: count, stage, parity to wait for
      bool ok = true;
      const uint32_t leader_full = map_to_cta(smem_u32(&ctl->full[0]), 0);
      for (int t = pair; t < num_tiles && ok; t += n_pairs) {
        int tm, tn;
        tiles.at(t, &tm, &tn);
        const int row_a = tm * 256 + static_cast<int>(cta) * 128, row_b = tn * BN + static_cast<int>(cta) * (BN / 4);
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          if (!mbar_wait_warp(smem_u32(&ctl->empty[0]) + s * 8u, ph, &ctl->abort, budget)) { ok = false; break; }
          if (leader) {
            const uint32_t full = leader_full + s * 8u, dst = base + s * kPairStage<BN>;
            mbar_arrive_expect_tx_cluster(full, kPairStage<BN>);
            tma_load_2d_pair(dst, &tma_a, full, kb * kBlockK, row_a);
            tma_load_2d_pair(dst + kTileBytes, &tma_b, full, kb * kBlockK, row_b);   // a quarter of the tile's rows of B for each half
            tma_load_2d_pair(dst + kTileBytes + BN / 4 * kBlockK, &tma_b, full, kb * kBlockK, row_b + NC);
          }
          if (++s == NS) { s = 0; ph ^= 1u; }
        }
      }
      // Both CTAs' loads count on the leader's barriers, and its partner stays until the cluster barrier at the end.  Where
      // this producer gave up, the partner may be up to a ring ahead.
      if (cta == 0) {
        loads_land(&ctl->full[0], NS, it, budget);
        if (!ok) loads_land(&ctl->full[0], NS, it + NS, budget);
      }
    } else if (warp < 3) {
      if (cta == 0) {
        constexpr uint32_t idesc = make_idesc_e4m3(256, NC);
        const uint32_t half = static_cast<uint32_t>(warp) - 1u;
        const uint64_t da0 = make_smem_desc_sw128(base), db0 = make_smem_desc_sw128(base + kTileBytes + half * (BN / 4 * kBlockK));
        const uint32_t full = smem_u32(&ctl->full[0]), empty = smem_u32(&ctl->empty[0]);
        const uint32_t acc_full = smem_u32(&ctl->acc_full[0][half]), acc_empty = smem_u32(&ctl->acc_empty[0][half]);
        uint32_t s = 0, ph = 0, it = 0;
        bool ok = true;
        for (int t = pair; t < num_tiles && ok; t += n_pairs) {
          for (int kb = 0; kb < num_kb; ++kb, ++it) {
            const uint32_t buf = it % NB, acc_ph = it / NB & 1u;
            ok = mbar_wait_both(full + s * 8u, ph, acc_empty + buf * 16u, acc_ph ^ 1u, &ctl->abort, budget);
            if (!ok) break;
            tc_fence_after_sync();
            const uint64_t da = da0 + static_cast<uint64_t>(s * (kPairStage<BN> >> 4)), db = db0 + static_cast<uint64_t>(s * (kPairStage<BN> >> 4));
            if (leader) {
#pragma unroll
              for (int k = 0; k < kBlockK / kMmaK; ++k)   // 32 bytes on inside a 128-byte swizzle row: +2 in the address field
                umma_e4m3_pair(tmem_base + buf * (kTmemCols / NB) + half * NC, da + static_cast<uint64_t>(k * 2), db + static_cast<uint64_t>(k * 2), idesc, k != 0 ? 1u : 0u);
              umma_commit_pair(acc_full + buf * 16u, 3);
              umma_commit_pair(empty + s * 8u, 3);   // with the other half's: the stage is free in both CTAs
            }
            if (++s == NS) { s = 0; ph ^= 1u; }
          }
        }
      }
    } else {
      // Scales: of this CTA's 128 rows, and of B the tile's columns or, for each half of them, the two blocks of 128 rows that it may touch.
      uint32_t group = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += n_pairs) {
        int tm, tn;
        tiles.at(t, &tm, &tn);
        constexpr int kOwn = B_ROWS ? BN / 32 : 1;
        const float *rows[4], *cols[kOwn];
#pragma unroll
        for (int j = 0; j < 4; ++j) rows[j] = g.a.at(min(tm * 256 + static_cast<int>(cta) * 128 + lane + j * 32, g.M - 1));
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
          const int n = B_ROWS ? tn * BN + lane + j * 32 : ((tn * BN + (lane >> 1 & 1) * NC) & ~127) + (lane & 1) * 128;
          cols[j] = g.b.at(min(n, g.N - 1)) + (B_ROWS ? 0 : (lane >> 2) * g.b.blk);   // lanes 4i .. 4i + 3 fetch the group's i-th block
        }
        for (int kb = 0; kb < num_kb; kb += kGroup, ++group) {
          ok = mbar_wait_warp(smem_u32(&ctl->scales_empty[group & 1u]), (group >> 1 & 1u) ^ 1u, &ctl->abort, budget);
          if (!ok) break;
          float* slot = slots + (group & 1u) * kSlot<BN, B_ROWS>;
          for (int i = 0; i < kGroup && kb + i < num_kb; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              copy4_async(slot + i * 128 + lane + j * 32, rows[j]);
              rows[j] += g.a.blk;
            }
            if constexpr (B_ROWS) {
#pragma unroll
              for (int j = 0; j < kOwn; ++j) {
                copy4_async(slot + kGroup * 128 + i * BN + lane + j * 32, cols[j]);
                cols[j] += g.b.blk;
              }
            }
          }
          if constexpr (!B_ROWS) {
            if (lane < 4 * kGroup && kb + (lane >> 2) < num_kb) copy4_async(slot + kGroup * 128 + lane, cols[0]);
            static_assert(4 * kGroup <= 32, "a lane for each of a group's scales");
            cols[0] += kGroup * g.b.blk;
          }
          copies_arrive(smem_u32(&ctl->scales_full[group & 1u]));
        }
      }
      copies_wait();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPromoterRegs));
    const int q = warp & 3, half = (warp - kFirst) >> 2, first_col = half * NC;
    uint8_t* scratch = scratch_all + (warp - kFirst) * kScratchBytes;
    float* bias = bias_all + (warp - kFirst) * kBiasFloats;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + first_col;
    const uint32_t acc_full = smem_u32(&ctl->acc_full[0][half]), acc_empty = map_to_cta(smem_u32(&ctl->acc_empty[0][half]), 0);
    uint32_t group = 0;
    uint32_t it = 0;
    uint32_t pieces = 0;   // of results that have been sent out
    bool ok = true, ready = false;
    for (int t = pair; t < num_tiles && ok; t += n_pairs) {
      int tm, tn;
      tiles.at(t, &tm, &tn);
      const int row = tm * 256 + static_cast<int>(cta) * 128 + q * 32 + lane, col = tn * BN + first_col;
      if (g.bias != nullptr) {
        switch (g.type) {
          case 6: load_bias<__half, NC>(g, col, bias, lane); break;
          case 7: load_bias<float, NC>(g, col, bias, lane); break;
          default: load_bias<__nv_bfloat16, NC>(g, col, bias, lane);
        }
      }
      float acc[NC];
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[j] = 0.0f;
      // One rolled loop: unrolled by groups, with their scales in registers, it ran into instruction-cache misses.
#pragma unroll 1
      for (int kb = 0; kb < num_kb; ++kb) {
        const int i = kb % kGroup;
        if (i == 0) {
          ok = mbar_wait_warp(smem_u32(&ctl->scales_full[group & 1u]), group >> 1 & 1u, &ctl->abort, budget);
          if (!ok) break;
        }
        const float* slot = slots + (group & 1u) * kSlot<BN, B_ROWS>;
        const float* cols = slot + kGroup * 128 + (B_ROWS ? i * BN + first_col : i * 4 + half * 2);
        const float r = slot[i * 128 + q * 32 + lane];
        float x[2];   // its products with the scales of the two blocks of B's rows
        // A narrow tile's scales of columns are on their way before the block is there, and multiplied one at a time (256 x 4096 x 4096: 13.6 us; fetched
        // behind the block 14.2, two at a time 14.0).
        float4 ahead[8];
        if constexpr (B_ROWS && NC == 32) {
#pragma unroll
          for (int j = 0; j < 8; ++j) ahead[j] = *reinterpret_cast<const float4*>(cols + 4 * j);
        }
        if constexpr (!B_ROWS) {
          x[0] = r * cols[0];
          x[1] = r * cols[1];
        }
        const uint32_t buf = it % NB, acc_ph = it / NB & 1u;
        ++it;
        ok = __all_sync(0xffffffffu, ready) || mbar_wait_warp(acc_full + buf * 16u, acc_ph, &ctl->abort, budget);
        if (!ok) break;
        tc_fence_after_sync();
        promote<NC, B_ROWS ? 32 : 64>(
            taddr + buf * (kTmemCols / NB),
            [&](int c, const auto& v) {
              constexpr int kPiece = sizeof(v) / 4;
              if constexpr (B_ROWS) {
#pragma unroll
                for (int j = 0; j < kPiece; j += 4) {
                  float y[4];   // the products of the two scales
                  if constexpr (NC == 32) {
                    const float4& b = ahead[j / 4];
                    y[0] = r * b.x;
                    y[1] = r * b.y;
                    y[2] = r * b.z;
                    y[3] = r * b.w;
                  } else {
                    times_four(*reinterpret_cast<const float4*>(cols + c + j), r, y);
                  }
#pragma unroll
                  for (int k = 0; k < 4; ++k) acc[c + j + k] += __uint_as_float(v[j + k]) * y[k];
                }
              } else {
#pragma unroll
                for (int h = 0; h < kPiece; h += 32) {
                  const float y = BN != 192 || (col & 127) + c + h < 128 ? x[0] : x[1];   // 32 columns lie in one block: col is a multiple of 32
#pragma unroll
                  for (int j = 0; j < 32; ++j) acc[c + h + j] += __uint_as_float(v[h + j]) * y;
                }
              }
            },
            [&] {
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster(acc_empty + buf * 16u);
              ready = mbar_test(acc_full + it % NB * 16u, it / NB & 1u);   // the next block: its answer is there when the sums are done
            });
        if (i == kGroup - 1 || kb + 1 == num_kb) {   // this group's scales have been read
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&ctl->scales_empty[group & 1u]));
          ++group;
        }
      }
      if (!ok) break;
      if (col < g.N) {
        switch (g.type) {
          case 6: store_rows<__half>(g, &tma_c, mapped, row, col, acc, scratch, pieces, bias, lane); break;
          case 7: store_rows<float>(g, &tma_c, mapped, row, col, acc, scratch, pieces, bias, lane); break;
          default: store_rows<__nv_bfloat16>(g, &tma_c, mapped, row, col, acc, scratch, pieces, bias, lane);
        }
      }
    }
    if (lane == 0) bulk_wait_all();   // what is on its way out lies in this CTA's shared memory
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();   // neither CTA leaves (or frees tensor memory) while its partner may still signal it
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
  if (threadIdx.x == 0 && ctl->abort != 0u && g.err != nullptr) atomicCAS(g.err, 0u, ctl->abort);
}

template <int BN, bool B_ROWS>
cudaError_t fire(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, bool mapped, const Args& g, int tiles, cudaStream_t stream) {
  auto kernel = gemm_fp8_pair_kernel<BN, B_ROWS>;
  constexpr int smem_bytes = kStages * kPairStage<BN> + 1024 /*alignment slack*/ + static_cast<int>(sizeof(PairCtl)) + 2 * kSlot<BN, B_ROWS> * 4 +
                             kPromoters * (kScratchBytes + kBiasFloats * 4);
  static_assert(kPairStage<BN> % 1024 == 0 && 32 * 32 * 4 <= kScratchBytes, "layout of shared memory");
  static_assert(smem_bytes <= 227 * 1024, "shared memory");
  static int most_dev[kMaxDevices] = {};   // pairs that the device holds at once, which a persistent kernel must not exceed
  int& most = most_dev[current_device_slot()];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * 74);
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {{}, early_start()};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;   // the question below is about clusters alone
  if (most == 0) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
    if (e != cudaSuccess) return e;
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    if (e != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = 64;
    }
    most = n;
  }
  cfg.numAttrs = 2;
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min(tiles, most)));
  return cudaLaunchKernelEx(&cfg, kernel, ta, tb, tc, g, mapped);
}

// Whether the TMA unit can write C: rows that start on 16 bytes.
bool can_map_out(const Args& g) {
  const uint64_t size = g.type == 7 ? 4 : 2;
  return (reinterpret_cast<uintptr_t>(g.c) & 15u) == 0 && g.ldc * size % 16 == 0 && g.ldc * size < (1ull << 40);
}
// C for stores of 32 rows of 64 bytes.
bool make_tensor_map_out(CUtensorMap* map, const Args& g) {
  const CudaDriver* d = CudaDriver::get();
  const cuuint64_t size = g.type == 7 ? 4 : 2;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(g.N), static_cast<cuuint64_t>(g.M)};
  cuuint64_t strides[1] = {g.ldc * size};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(kOutRow / size), 32};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType type = g.type == 7 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  return d->TensorMapEncodeTiled(map, type, 2, g.c, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                                 CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The tile width with the least estimated time (ns): a wave of tiles takes about two microseconds and so much a block of K, more with a scale for
// every row of B.  The constants describe a kernel by itself; calls that follow one another overlap and take about a microsecond less each, whatever the
// width.  Measured so, operands not in the L2 (us without / with a scale for every row): 256 x 4096 x 4096, one wave of 64, 12.2 / 13.3, and of 128, 13.6
// / 17.4; 1001 x 1288 x 5000, one of 128, 17.2 / 21.5; 1001 x 5000 x 1288, two of 192, 15.5 / 19.1; 4096 x 4096 x 4096, four of 256, 69 / 96, and
// five of 192, 73 / 95; 8192 x 4096 x 1024, seven of 256, 42 / 55: in these and seven others the width chosen is the fastest of the four.  Rows of C that the TMA unit cannot write
// cost a wave of 128 columns one more (8192 x 4095 x 1024: 57).  A narrower tile pays where it saves a wave or leaves fewer SMs idle; 64 columns on
// all SMs read 10 TB/s from the L2.
int pick_width(int M, int N, int K, bool b_rows, bool mapped, int pairs, long* ns) {
  struct Width {
    int bn;
    long per_block, per_block_rows;
  };
  constexpr Width kWidths[] = {{256, 430, 720}, {192, 390, 560}, {128, 330, 400}, {64, 245, 280}};
  const long num_kb = (K + kBlockK - 1) / kBlockK;
  int best = 256;
  *ns = -1;
  for (const Width& w : kWidths) {
    const long tiles = static_cast<long>((M + 255) / 256) * ((N + w.bn - 1) / w.bn), waves = (tiles + pairs - 1) / pairs;
    const long t = 3100 + waves * (2000 + (mapped ? 0 : 1000 * w.bn / 128) + num_kb * (b_rows ? w.per_block_rows : w.per_block));
    if (*ns < 0 || t < *ns) {
      *ns = t;
      best = w.bn;
    }
  }
  return best;
}

struct Plan {
  bool rows;   // up to four tokens and a small weight: the kernel without tensor cores
  bool small;
  SmallPlan p;
  int bn;   // pairs: tile width
};
Plan make_plan(int M, int N, int K, bool b_rows, bool mapped, int sms) {
  Plan plan{};
  long pair_ns = 0, small_ns = 0;
  plan.bn = pick_width(M, N, K, b_rows, mapped, sms / 2, &pair_ns);
  plan.small = plan_small(M, N, K, sms, &plan.p, &small_ns) && small_ns < pair_ns;
  plan.rows = rows_ns(M, N, K) < std::min(small_ns, pair_ns);
  return plan;
}

int run(const void* a, int64_t lda, const void* b, int64_t ldb, Args g, cudaStream_t stream) {
  std::string why;
  g.err = error_word();
  g.wait_budget_ns = 2000000000ull;
  const Plan plan = make_plan(g.M, g.N, g.K, g.b.shift == 0, can_map_out(g), sm_count());
  const int bn = plan.bn;
  cudaError_t e;
  if (plan.rows) {
    e = launch_rows(a, lda, b, ldb, g, stream);
  } else if (plan.small) {
    e = launch_small(a, lda, b, ldb, g, plan.p, stream, &why);
  } else {
    const long tiles = static_cast<long>((g.M + 255) / 256) * ((g.N + bn - 1) / bn);
    if (tiles > 0x7fffffff / 2) return -2;
    CUtensorMap ta, tb, tc = {};
    bool mapped = false;
    if (!make_tensor_map_e4m3(&ta, a, g.M, g.K, lda, 128, &why) || !make_tensor_map_e4m3(&tb, b, g.N, g.K, ldb, bn / 4, &why)) {
      e = cudaErrorInvalidValue;
    } else {
      mapped = can_map_out(g) && make_tensor_map_out(&tc, g);
      const auto go = [&](auto rows) {
        constexpr bool R = decltype(rows)::value;
        switch (bn) {
          case 256: return fire<256, R>(ta, tb, tc, mapped, g, static_cast<int>(tiles), stream);
          case 192: return fire<192, R>(ta, tb, tc, mapped, g, static_cast<int>(tiles), stream);
          case 128: return fire<128, R>(ta, tb, tc, mapped, g, static_cast<int>(tiles), stream);
          default: return fire<64, R>(ta, tb, tc, mapped, g, static_cast<int>(tiles), stream);
        }
      };
      e = g.b.shift == 0 ? go(std::true_type{}) : go(std::false_type{});
    }
  }
  if (!why.empty()) {
    fprintf(stderr, "[Mini-NCCL] 8-bit GEMM: %s\n", why.c_str());
    return -3;
  }
  return e == cudaSuccess ? 0 : static_cast<int>(e) + 1000;
}

}  // namespace
}  // namespace fp8
}  // namespace gemm
}  // namespace mnccl

extern "C" {
#define MNCCL_EXPORT __attribute__((visibility("default")))

// a [M, K], b [N, K] e4m3, 16-byte aligned, row strides multiples of 16; scales with their strides (row of scales, block along K) and rows
// of a scale (1 or 128); C and bias (null: none) of type 6 fp16, 7 fp32 or 9 bf16.
// Returns 0, -1 null or empty, -2 shape or alignment, -3 tensor map, or a cudaError_t + 1000.
MNCCL_EXPORT int mncclGemmFp8(const void* a, int64_t lda, const float* sa, int64_t sa_row, int64_t sa_blk, int sa_rows, const void* b,
                              int64_t ldb, const float* sb, int64_t sb_row, int64_t sb_blk, int sb_rows, void* c, int64_t ldc, int type,
                              const void* bias, int M, int N, int K, cudaStream_t stream) {
  using namespace mnccl::gemm::fp8;
  if (!a || !b || !c || !sa || !sb || M <= 0 || N <= 0 || K <= 0) return -1;
  const auto operand = [K](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 16 == 0 && ld >= K; };
  if (!operand(a, lda) || !operand(b, ldb) || ldc < N || (type != 6 && type != 7 && type != 9)) return -2;
  if ((sa_rows != 1 && sa_rows != 128) || (sb_rows != 1 && sb_rows != 128) || std::max({M, N, K}) > 0x7fffff00) return -2;
  Args g{};
  g.M = M;
  g.N = N;
  g.K = K;
  g.a = Scales{sa, sa_row, sa_blk, sa_rows == 1 ? 0 : 7};
  g.b = Scales{sb, sb_row, sb_blk, sb_rows == 1 ? 0 : 7};
  g.c = c;
  g.ldc = ldc;
  g.type = type;
  g.bias = bias;
  try {
    return run(a, lda, b, ldb, g, stream);
  } catch (...) {   // out of host memory for a message
    return -3;
  }
}

// The kernel that an M x N x K product takes on `sms` SMs: returns 2 for the one without tensor cores, 1 for the one for few rows or tiles (tile = rows of
// A per tile, slices = CTAs that share a tile's K), 0 for CTA pairs (tile = columns, slices = 1).  b_rows: rows of a scale of B; aligned: whether C's rows start on 16 bytes.
// Host arithmetic only (needs no GPU).
MNCCL_EXPORT int mncclGemmFp8Plan(int M, int N, int K, int b_rows, int aligned, int sms, int* tile, int* slices) {
  using namespace mnccl::gemm::fp8;
  if (M <= 0 || N <= 0 || K <= 0 || sms < 2 || (b_rows != 1 && b_rows != 128)) return -1;
  const Plan plan = make_plan(M, N, K, b_rows == 1, aligned != 0, sms);
  if (tile) *tile = plan.rows ? 8 : plan.small ? plan.p.tn : plan.bn;
  if (slices) *slices = !plan.rows && plan.small ? plan.p.slices : 1;
  return plan.rows ? 2 : plan.small ? 1 : 0;
}

}  // extern "C"
