// The 8-bit product with block scales for few rows of A, or too few tiles for the persistent kernel.
//
// Operands are swapped: the 128 rows of the MMA are rows of B (a weight), its TN columns rows of A, so a tile of 16 tokens costs 2 KB of
// shared memory a block instead of 16, and a column of the result is 128 consecutive elements of a row of C.  K is split over the CTAs of a
// cluster where the tiles alone leave SMs idle; the slices meet in distributed shared memory and are added in slice order.  One tile per CTA.
//
// What bounds it is bytes in flight and handshakes.  A hand-over between the MMA warp and the promotion warps costs both about 300 cycles,
// as much as the MMAs of a block themselves, so accumulators are handed over in units of up to four blocks (each block has its own columns), and
// ring stages hold two blocks where tiles are narrow.
#include <algorithm>

#include "kernels/dependent_launch.cuh"
#include "kernels/gemm_fp8.cuh"

namespace mnccl {
namespace gemm {
namespace fp8 {

namespace {

template <int TN>
constexpr int kPerStage = TN <= 32 ? 2 : 1;       // blocks of K a ring stage holds: 128-row tiles of B, then TN-row tiles of A
template <int TN>
constexpr int kStage = kPerStage<TN> * (kTileBytes + TN * kBlockK);
template <int TN>
constexpr int kUnit = TN <= 16 ? 4 : 2;           // blocks that are handed over together
template <int TN>
constexpr int kWarps = TN >= 64 ? 8 : 4;          // promotion warps: one or two for each quarter of tensor memory's lanes
template <int TN>
constexpr int kCols = TN / (kWarps<TN> / 4);      // columns a promotion warp holds
template <int TN>
constexpr int kBuffers = 2;                       // units in tensor memory
template <int TN>
constexpr int kSlot = kGroup * (128 + TN);         // floats: a group's scales
template <int TN>
constexpr int kThreads = 32 * (3 + kWarps<TN>);    // a producer, an MMA issuer, the promotion warps, one that brings their scales
constexpr int kMostStages = 8;

struct __align__(16) Ctl {
  uint64_t full[kMostStages], empty[kMostStages];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t scales_full[2], scales_empty[2];
  uint32_t tmem_base;
  volatile uint32_t abort;
};

struct SmallArgs {
  Args g;
  int tiles_n, kb_per_slice;
};

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

template <int TN, int NS>
__global__ void __launch_bounds__(kThreads<TN>)
gemm_fp8_small_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x, const __grid_constant__ SmallArgs args) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int NB = kBuffers<TN>, W = kWarps<TN>, NC = kCols<TN>;
  constexpr int KPS = kPerStage<TN>, U = kUnit<TN>;
  constexpr uint32_t kTmem = NB * U * TN;   // 128, 128, 256 columns
  static_assert(U % KPS == 0 && kGroup % U == 0, "a unit is whole stages, a group of scales whole units");
  static_assert(NS <= kMostStages && (NB & (NB - 1)) == 0, "ring depth");
  const Args& g = args.g;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  Ctl* ctl = reinterpret_cast<Ctl*>(smem + NS * kStage<TN>);
  float* slots = reinterpret_cast<float*>(ctl + 1);   // [2][kGroup][128 rows of B], then [kGroup][TN rows of A], each

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slices = static_cast<int>(cluster_size());
  const int slice = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / slices;
  const int n0 = (tile % args.tiles_n) * 128, m0 = (tile / args.tiles_n) * TN;
  const int num_kb = (g.K + kBlockK - 1) / kBlockK;
  const int kb0 = slice * args.kb_per_slice;
  const int nkb = min(num_kb, kb0 + args.kb_per_slice) - kb0;   // at least 1: the plan leaves no slice empty
  const int stages = (nkb + KPS - 1) / KPS;

  const bool leader = elect_one();
  auto load = [&](int i, uint32_t s) {
    const uint32_t full = smem_u32(&ctl->full[0]) + s * 8u, dst = base + s * kStage<TN>;
    mbar_arrive_expect_tx(full, kStage<TN>);
#pragma unroll
    for (int p = 0; p < KPS; ++p) {   // (what lies beyond K is loaded as zeros)
      const int k = (kb0 + i * KPS + p) * kBlockK;
      tma_load_2d(dst + p * kTileBytes, &tma_w, full, k, n0);
      tma_load_2d(dst + KPS * kTileBytes + p * (TN * kBlockK), &tma_x, full, k, m0);
    }
  };
  if (warp == 0) {
    if (leader) {
      prefetch_tensormap(&tma_w);
      prefetch_tensormap(&tma_x);
      for (int s = 0; s < NS; ++s) {
        mbar_init(smem_u32(&ctl->full[s]), 1);
        mbar_init(smem_u32(&ctl->empty[s]), 1);
      }
      for (int b = 0; b < NB; ++b) {
        mbar_init(smem_u32(&ctl->acc_full[b]), 1);
        mbar_init(smem_u32(&ctl->acc_empty[b]), W);
      }
      for (int b = 0; b < 2; ++b) {
        mbar_init(smem_u32(&ctl->scales_full[b]), 32);
        mbar_init(smem_u32(&ctl->scales_empty[b]), W);
      }
      ctl->abort = 0;
      fence_barrier_init();
      fence_proxy_async();
    }
    __syncwarp();
    wait_for_previous();
    for (int i = 0; i < NS && i < stages; ++i)
      if (leader) load(i, i);
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(smem_u32(&ctl->tmem_base), kTmem);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = ctl->tmem_base;
  wait_for_previous();
  let_next_start();

  // promotion warps: warp's quarter of the lanes, its columns of the tile, this lane's row of B
  const int q = warp & 3, first_col = ((warp - 2) >> 2) * NC;
  const int n = n0 + q * 32 + lane;
  const bool promoter = warp >= 2 && warp < 2 + W;
  float acc[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) acc[j] = 0.0f;
  bool ok = true;
  const bool one = g.b.shift != 0;   // a scale of B holds for the whole tile
  const float bias = promoter ? bias_of(g, n) : 0.0f;

  if (warp == 0) {
    uint32_t s = 0, ph = 0;
    int i = NS;
    for (; i < stages; ++i) {
      if (!mbar_wait_warp(smem_u32(&ctl->empty[0]) + s * 8u, ph, &ctl->abort, g.wait_budget_ns)) break;
      if (leader) load(i, s);
      if (++s == NS) { s = 0; ph ^= 1u; }
    }
    loads_land(&ctl->full[0], NS, static_cast<uint32_t>(min(i, stages)), g.wait_budget_ns);
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_e4m3(128, TN);
    const uint64_t dw0 = make_smem_desc_sw128(base), dx0 = make_smem_desc_sw128(base + KPS * kTileBytes);
    uint32_t s = 0, ph = 0, unit = 0;
    for (int i0 = 0; i0 < nkb && ok; i0 += U, ++unit) {
      const uint32_t buf = unit & 1u;
      ok = mbar_wait_warp(smem_u32(&ctl->acc_empty[0]) + buf * 8u, (unit >> 1 & 1u) ^ 1u, &ctl->abort, g.wait_budget_ns);
      if (!ok) break;
#pragma unroll
      for (int st = 0; st < U; st += KPS) {
        if (i0 + st >= nkb) break;
        ok = mbar_wait_warp(smem_u32(&ctl->full[0]) + s * 8u, ph, &ctl->abort, g.wait_budget_ns);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t dw = dw0 + static_cast<uint64_t>(s * (kStage<TN> >> 4)), dx = dx0 + static_cast<uint64_t>(s * (kStage<TN> >> 4));
        if (leader) {
#pragma unroll
          for (int p = 0; p < KPS; ++p) {
            if (p != 0 && i0 + st + p >= nkb) break;
#pragma unroll
            for (int k = 0; k < kBlockK / kMmaK; ++k)   // 32 bytes on inside a 128-byte swizzle row: +2 in the address field
              umma_e4m3(tmem + buf * (U * TN) + (st + p) * TN, dw + static_cast<uint64_t>(p * (kTileBytes >> 4) + k * 2),
                        dx + static_cast<uint64_t>(p * (TN * kBlockK >> 4) + k * 2), idesc, k != 0 ? 1u : 0u);
          }
          umma_commit(smem_u32(&ctl->empty[0]) + s * 8u);
        }
        if (++s == NS) { s = 0; ph ^= 1u; }
      }
      if (ok && leader) umma_commit(smem_u32(&ctl->acc_full[0]) + buf * 8u);
    }
  } else if (warp == 2 + W) {
    const float *rows[4], *cols[(TN + 31) / 32];
#pragma unroll
    for (int j = 0; j < 4; ++j) rows[j] = g.b.at(min(n0 + (one ? 0 : lane + j * 32), g.N - 1)) + (kb0 + (one ? lane : 0)) * g.b.blk;
#pragma unroll
    for (int j = 0; j < (TN + 31) / 32; ++j) cols[j] = g.a.at(min(m0 + lane + j * 32, g.M - 1)) + kb0 * g.a.blk;
    uint32_t group = 0;
    for (int i0 = 0; i0 < nkb; i0 += kGroup, ++group) {
      if (!mbar_wait_warp(smem_u32(&ctl->scales_empty[group & 1u]), (group >> 1 & 1u) ^ 1u, &ctl->abort, g.wait_budget_ns)) break;
      float* slot = slots + (group & 1u) * kSlot<TN>;
      if (one) {   // lane i fetches the group's i-th block
        if (lane < kGroup && i0 + lane < nkb) copy4_async(slot + lane * 128, rows[0]);
        rows[0] += kGroup * g.b.blk;
      }
      for (int i = 0; i < kGroup && i0 + i < nkb; ++i) {
        if (!one) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            copy4_async(slot + i * 128 + lane + j * 32, rows[j]);
            rows[j] += g.b.blk;
          }
        }
#pragma unroll
        for (int j = 0; j < (TN + 31) / 32; ++j) {
          if (lane + j * 32 < TN) copy4_async(slot + kGroup * 128 + i * TN + lane + j * 32, cols[j]);
          cols[j] += g.a.blk;
        }
      }
      copies_arrive(smem_u32(&ctl->scales_full[group & 1u]));
    }
    copies_wait();
  } else {
    const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + first_col;
    const uint32_t acc_full = smem_u32(&ctl->acc_full[0]), acc_empty = smem_u32(&ctl->acc_empty[0]);
    uint32_t group = 0;
    uint32_t unit = 0;
    bool ready = false;
#pragma unroll 1
    for (int i0 = 0; i0 < nkb; i0 += U, ++unit) {
      if (i0 % kGroup == 0) {
        ok = mbar_wait_warp(smem_u32(&ctl->scales_full[group & 1u]), group >> 1 & 1u, &ctl->abort, g.wait_budget_ns);
        if (!ok) break;
      }
      const float* slot = slots + (group & 1u) * kSlot<TN>;
      const uint32_t buf = unit & 1u;
      ok = __all_sync(0xffffffffu, ready) || mbar_wait_warp(acc_full + buf * 8u, unit >> 1 & 1u, &ctl->abort, g.wait_budget_ns);
      if (!ok) break;
      tc_fence_after_sync();
      const int blocks = min(U, nkb - i0);
#pragma unroll
      for (int p = 0; p < U; ++p) {
        if (p >= blocks) break;
        const int in = i0 % kGroup + p;
        const float* cols = slot + kGroup * 128 + in * TN + first_col;
        const float r = slot[in * 128 + (one ? 0 : q * 32 + lane)];
        uint32_t v[NC];
        tmem_read(taddr + buf * (U * TN) + p * TN, v);
        if (p == blocks - 1) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty + buf * 8u);
          ready = mbar_test(acc_full + (buf ^ 1u) * 8u, (unit + 1u) >> 1 & 1u);   // the next unit: its answer is there when the sums are done
        }
#pragma unroll
        for (int j = 0; j < NC; j += 4) {
          float x[4];
          times_four(*reinterpret_cast<const float4*>(cols + j), r, x);
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[j + k] += __uint_as_float(v[j + k]) * x[k];
        }
      }
      if ((i0 + U) % kGroup == 0 || i0 + U >= nkb) {   // this group's scales have been read
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl->scales_empty[group & 1u]));
        ++group;
      }
    }
  }
  __syncwarp();

  if (slices == 1) {
    if (promoter && ok) {
#pragma unroll
      for (int j = 0; j < NC; ++j) store(g, m0 + first_col + j, n, acc[j] + bias);
    }
  } else {
    // Every CTA of the cluster has left its main loop: its ring may be overwritten.
    cluster_sync_all();
    const int own = TN / slices, own_log2 = 31 - __clz(own);   // columns this slice finishes (a power of two)
    float* recv = reinterpret_cast<float*>(smem);               // [source slice][own columns][128 rows]
    if (promoter && ok) {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int col = first_col + j;
        const uint32_t dst = map_to_cta(smem_u32(recv + (slice * own + (col & (own - 1))) * 128 + q * 32 + lane), static_cast<uint32_t>(col >> own_log2));
        st_cluster_f32(dst, acc[j]);
      }
    }
    cluster_sync_all();
    if (promoter && ok) {
      for (int c = (warp - 2) >> 2; c < own; c += W / 4) {
        const int m = m0 + slice * own + c;
        if (m >= g.M) break;
        float v = recv[c * 128 + q * 32 + lane];
        for (int s = 1; s < slices; ++s) v += recv[(s * own + c) * 128 + q * 32 + lane];
        store(g, m, n, v + bias);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kTmem);
  }
  if (threadIdx.x == 0 && ctl->abort != 0u && g.err != nullptr) atomicCAS(g.err, 0u, ctl->abort);
}

template <int TN, int NS>
cudaError_t fire(const CUtensorMap& tw, const CUtensorMap& tx, const SmallArgs& a, const SmallPlan& p, cudaStream_t stream) {
  auto kernel = gemm_fp8_small_kernel<TN, NS>;
  constexpr int smem_bytes = NS * kStage<TN> + 1024 /*alignment slack*/ + static_cast<int>(sizeof(Ctl)) + 2 * kSlot<TN> * 4;
  static_assert(smem_bytes <= 227 * 1024, "shared memory");
  static_assert(TN * 128 * 4 <= NS * kStage<TN>, "the slices' partial sums fit the ring");
  static bool configured[kMaxDevices] = {};
  const int dev = current_device_slot();
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.tiles) * p.slices);
  cfg.blockDim = dim3(kThreads<TN>);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {{}, early_start()};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.slices);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, tw, tx, a);
}

}  // namespace

// Blocks of K a slice takes: whole ring stages.
int per_slice(int num_kb, int slices, int tn) {
  const int per_stage = tn <= 32 ? 2 : 1, stages = (num_kb + per_stage - 1) / per_stage;
  return (stages + slices - 1) / slices * per_stage;
}

// The plan with the least estimated time (ns).  The constants describe a kernel by itself.  Measured on 148 SMs, calls that follow one another and
// overlap (about a microsecond less each), operands not in L2 (M x N x K, tile's rows of A / slices):
//   1 x 4096 x 4096      16 / 4: 6.7 us, 16 / 8: 6.8, 16 / 2: 8.3          64 x 14336 x 4096   64 / 1: 16.7 us, 32 / 1: 19.1, pairs: 19.8
//   16 x 4096 x 14336    16 / 8: 13.3 us, 16 / 4: 15.0, 16 / 2: 21.5       64 x 4096 x 4096    64 / 4: 9.7 us, 32 / 4: 10.2, pairs: 11.9
//   256 x 1024 x 1024    16 / 1: 5.4 us, 64 / 4: 6.7, pairs: 5.2           128 x 4096 x 4096   64 / 2: 12.5 us, 32 / 1: 13.8, pairs: 12.1
//   512 x 1024 x 1024    16 / 1: 6.4 us, pairs: 5.6                        777 x 1003 x 1544   64 / 1: 10.6 us, pairs: 7.8
// The choice is the fastest of all in 28 of 32 products tried so, within 4 % in three more, and 13 % off for 16 x 4096 x 14336 (it takes 16 / 4).
// So a tile takes a fixed time and one per block of K that grows with its width; two narrow tiles on an SM overlap by a third, two wide
// ones hardly; and nothing is faster than the operands come from memory.  Tiles of 128 rows of A never won (128 x 4096 x 4096 by itself: 16.4 us).  A
// tile that has its K and its SM to itself takes all of the shared memory as its ring (16 x 14336 x 4096 by itself: 16.9 -> 15.5 us);
// slices do better with half, which lets the next wave's CTAs in early (1 x 4096 x 4096 by itself: 9.0 -> 8.2 us).
bool plan_small(int M, int N, int K, int sms, SmallPlan* p, long* ns) {
  struct Cost {
    int tn;
    long fixed, per_block, split;   // a tile; a block of K; the meeting of the slices
  };
  constexpr Cost kCost[] = {{16, 1800, 260, 1300}, {32, 3300, 330, 1400}, {64, 5500, 320, 1500}};
  constexpr long kLaunch = 3000;
  const int num_kb = (K + kBlockK - 1) / kBlockK;
  const long tiles_n = (N + 127) / 128, floor_ns = 4000 + static_cast<long>((static_cast<double>(K) * (static_cast<double>(M) + N) + 2.0 * M * N) / 6300.0);
  *ns = -1;
  for (const Cost& c : kCost) {
    const long tiles = tiles_n * ((M + c.tn - 1) / c.tn);
    if (tiles > (1 << 20)) continue;
    for (int slices = 1; slices <= 8; slices *= 2) {
      const int per = per_slice(num_kb, slices, c.tn);
      const long items = tiles * slices, rounds = (items + sms - 1) / sms;
      if ((slices - 1) * per >= num_kb || (slices > 1 && items > 2L * sms)) break;   // a slice would be empty, or CTAs wait for others
      const long each = c.fixed + std::min(per, num_kb) * c.per_block + (slices > 1 ? c.split : 0);
      const long t = std::max(kLaunch + (rounds > 1 && c.tn <= 32 ? rounds * each * 7 / 10 : rounds * each), floor_ns + (rounds > 1 ? 300 : 0));
      if (*ns < 0 || t < *ns) {
        *ns = t;
        *p = SmallPlan{c.tn, slices, per, static_cast<int>(tiles), slices == 1 && items <= sms};
      }
    }
  }
  return *ns > 0;
}

cudaError_t launch_small(const void* a, int64_t lda, const void* b, int64_t ldb, const Args& g, const SmallPlan& p, cudaStream_t stream, std::string* why) {
  CUtensorMap tw, tx;
  if (!make_tensor_map_e4m3(&tw, b, g.N, g.K, ldb, 128, why) || !make_tensor_map_e4m3(&tx, a, g.M, g.K, lda, p.tn, why)) return cudaErrorInvalidValue;
  const SmallArgs s{g, (g.N + 127) / 128, p.kb_per_slice};
  // ring depths: all of an SM's shared memory, or half of it
  switch (p.tn) {
    case 16: return p.deep ? fire<16, 5>(tw, tx, s, p, stream) : fire<16, 2>(tw, tx, s, p, stream);
    case 32: return p.deep ? fire<32, 5>(tw, tx, s, p, stream) : fire<32, 2>(tw, tx, s, p, stream);
    case 64: return p.deep ? fire<64, 8>(tw, tx, s, p, stream) : fire<64, 4>(tw, tx, s, p, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace fp8
}  // namespace gemm
}  // namespace mnccl
