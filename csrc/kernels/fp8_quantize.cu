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
// What bounds it is memory: 2 bytes read and 1 written an element (bf16), 4 read for fp32.  8192 x 4096 bf16 in rows 18.7 us (5.4 TB/s), 14336 x
// 4096 fp32 in squares 49.5 (5.9); with the transpose 28.2 (4.8), where the instructions for two quantisations count as well.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <type_traits>

#include "kernels/dependent_launch.cuh"

namespace {

constexpr int kBlock = 128;
constexpr int kThreads = 256;

// The scale of a block whose largest magnitude has these fp32 bits, and its inverse.
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

// Eight elements of a row as they lie in memory, and what is asked of them.
template <typename T>
struct Eight {
  static constexpr int kWords = 2 * sizeof(T);   // 32-bit
  uint32_t w[kWords];

  // Elements [c, c + 8) of a row of K, zeros beyond its end.
  __device__ __forceinline__ void load(const T* row, int c, int K, bool vec) {
    if (vec && c + 8 <= K) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 v = mnccl::load_vector(reinterpret_cast<const uint4*>(row + c) + i);
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = c + j < K ? __float_as_uint(row[c + j]) : 0u;
    } else {
      const uint16_t* bits = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = (c + 2 * j < K ? bits[c + 2 * j] : 0u) | (c + 2 * j + 1 < K ? static_cast<uint32_t>(bits[c + 2 * j + 1]) << 16 : 0u);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    else if constexpr (std::is_same_v<T, __half>) return __half2float(__ushort_as_half(static_cast<uint16_t>(w[j / 2] >> (j % 2 * 16))));
    else return __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
};

// Magnitudes as bits, whose order is that of the numbers, with infinity and NaN above all else: one fp32 a word, or two 16-bit numbers.
template <typename T>
struct Bits {
  static __device__ __forceinline__ uint32_t of(uint32_t w) { return w & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu); }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) return max(a, b);
    else return __vmaxu2(a, b);
  }
  // the larger of a word's two numbers (or its one), as the bits of an fp32 number
  static __device__ __forceinline__ uint32_t as_fp32(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
      return w;
    } else {
      const uint32_t top = max(w & 0xffffu, w >> 16);
      if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(top))));
      else return top << 16;
    }
  }
};
template <typename T>
__device__ __forceinline__ uint32_t largest(const Eight<T>& v) {
  uint32_t top = Bits<T>::of(v.w[0]);
#pragma unroll
  for (int i = 1; i < Eight<T>::kWords; ++i) top = Bits<T>::most(top, Bits<T>::of(v.w[i]));
  return top;
}

__device__ __forceinline__ uint32_t quantise4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// The product of a word's two bf16 numbers with two scales' inverses.  Powers of two: it is exact, or so small that e4m3 makes it zero.
__device__ __forceinline__ uint32_t times(uint32_t w, uint32_t inverses) {
  __nv_bfloat162 a, b;
  memcpy(&a, &w, 4);
  memcpy(&b, &inverses, 4);
  a = __hmul2(a, b);
  memcpy(&w, &a, 4);
  return w;
}
__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t twice(float inverse) { return __byte_perm(__float_as_uint(inverse), 0u, 0x3232); }   // as two bf16 numbers

template <typename T>
__device__ __forceinline__ uint2 quantise8(const Eight<T>& v, float inverse) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const uint32_t s = twice(inverse), a = times(v.w[0], s), b = times(v.w[1], s), c = times(v.w[2], s), d = times(v.w[3], s);
    return make_uint2(quantise4(low(a), high(a), low(b), high(b)), quantise4(low(c), high(c), low(d), high(d)));
  }
  return make_uint2(quantise4(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse),
                    quantise4(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse));
}

// 1 x 128 blocks.  16 lanes hold a block, 8 elements each; a thread block takes N blocks of 16 neighbouring rows, all loaded before the first is
// looked at, and a block's scales of 16 rows are 64 contiguous bytes: scales are stored [K blocks][M].
template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
quantise_rows_kernel(const T* x, size_t ldx, int M, int K, uint8_t* __restrict__ q, size_t ldq, float* __restrict__ scale, bool vec) {
  mnccl::wait_for_previous();
  mnccl::let_next_start();
  x = mnccl::since_wait(x);
  const int m = static_cast<int>(blockIdx.x) * 16 + static_cast<int>(threadIdx.x >> 4);
  const int first = static_cast<int>(blockIdx.y) * N, c = first * kBlock + static_cast<int>(threadIdx.x & 15) * 8;
  if (m >= M) return;   // all 16 lanes of a block
  Eight<T> v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i].load(x + m * ldx, c + i * kBlock, K, vec);
  const uint32_t lanes = 0xffffu << (threadIdx.x & 16);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if ((first + i) * kBlock >= K) break;
    uint32_t top = largest(v[i]);
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) top = Bits<T>::most(top, __shfl_xor_sync(lanes, top, d));
    const Scale s = scale_of(Bits<T>::as_fp32(top));
    // (q's rows are padded to 16 bytes)
    if (c + i * kBlock < K) *reinterpret_cast<uint2*>(q + m * ldq + c + i * kBlock) = quantise8(v[i], s.inverse);
    if ((threadIdx.x & 15) == 0) scale[static_cast<size_t>(first + i) * M + m] = s.scale;
  }
}

// A tile of 128 x 128 elements, which holds whole blocks of either kind along both dimensions: x is read once for q, the transpose qt and the sums
// of the tile's columns.  A thread holds 4 neighbouring rows of 2 x 8 columns, as they lie in memory (as fp32 numbers 16-bit types took 128
// registers, and half of the memory's rate: 64 us for 8192 x 4096), so that 4 elements of a column are one word of the transposed tile in shared
// memory: [column][8 units of 16 bytes], unit u of column c at u ^ (c / 8 mod 8), which keeps the banks apart both for the words that come in
// and for the units that go out.

template <typename T, bool SQUARE>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : 3)
quantise_tile_kernel(const T* x, size_t ldx, int M, int K, uint8_t* __restrict__ q, size_t ldq, float* __restrict__ scale,
                     uint8_t* __restrict__ qt, size_t ldt, float* __restrict__ scale_t, float* __restrict__ sums, bool vec) {
  __shared__ __align__(16) uint32_t tile[kBlock * 32];
  __shared__ uint32_t part[8][kBlock];   // a warp's largest magnitude of each column, then its sum
  __shared__ __align__(16) float inverse[kBlock];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = static_cast<int>(blockIdx.x) * kBlock, k0 = static_cast<int>(blockIdx.y) * kBlock;
  const int r0 = warp * 16 + (lane >> 3) * 4, c0 = (lane & 7) * 8;   // columns c0 .. and c0 + 64 ..
  mnccl::wait_for_previous();
  mnccl::let_next_start();
  x = mnccl::since_wait(x);
  Eight<T> v[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + r0 + i;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (m < M) v[i][h].load(x + m * ldx, k0 + c0 + h * 64, K, vec);
      else v[i][h].clear();
    }
  }
  float row_inverse[4];
  if constexpr (SQUARE) {
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) all = Bits<T>::most(all, Bits<T>::most(largest(v[i][0]), largest(v[i][1])));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) all = Bits<T>::most(all, __shfl_xor_sync(0xffffffffu, all, d));
    if (lane == 0) part[0][warp] = all;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) all = Bits<T>::most(all, part[0][w]);
    const Scale s = scale_of(Bits<T>::as_fp32(all));
#pragma unroll
    for (int i = 0; i < 4; ++i) row_inverse[i] = s.inverse;
    if (threadIdx.x == 0) scale[static_cast<size_t>(blockIdx.x) * gridDim.y + blockIdx.y] = s.scale;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t top = Bits<T>::most(largest(v[i][0]), largest(v[i][1]));
#pragma unroll
      for (int d = 4; d > 0; d >>= 1) top = Bits<T>::most(top, __shfl_xor_sync(0xffffffffu, top, d));
      const Scale s = scale_of(Bits<T>::as_fp32(top));
      row_inverse[i] = s.inverse;
      if ((lane & 7) == 0 && m0 + r0 + i < M) scale[static_cast<size_t>(blockIdx.y) * M + m0 + r0 + i] = s.scale;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = k0 + c0 + h * 64;
      if (m0 + r0 + i < M && c < K)
        *reinterpret_cast<uint2*>(q + static_cast<size_t>(m0 + r0 + i) * ldq + c) = quantise8(v[i][h], row_inverse[i]);
    }
  if (qt == nullptr) return;
  if constexpr (!SQUARE) {
    // Largest magnitude of each column: of the thread's four rows, of the warp's 16, of the tile.  A word holds the columns that lie next to one
    // another in memory.
    constexpr int kPer = 4 / static_cast<int>(sizeof(T));   // columns a word holds
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < Eight<T>::kWords; ++j) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = Bits<T>::most(top, Bits<T>::of(v[i][h].w[j]));
        top = Bits<T>::most(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = Bits<T>::most(top, __shfl_xor_sync(0xffffffffu, top, 16));
        if (lane < 8) part[warp][(c0 + h * 64) / kPer + j] = top;
      }
    __syncthreads();
    if (threadIdx.x < kBlock) {
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) top = Bits<T>::most(top, part[w][threadIdx.x / kPer]);
      if constexpr (kPer == 2) top = threadIdx.x & 1 ? top >> 16 : top & 0xffffu;
      const Scale t = scale_of(Bits<T>::as_fp32(top));
      inverse[threadIdx.x] = t.inverse;
      if (k0 + static_cast<int>(threadIdx.x) < K) scale_t[static_cast<size_t>(blockIdx.x) * K + k0 + threadIdx.x] = t.scale;
    }
    __syncthreads();
    if (sums != nullptr) {   // in a fixed order: rows of a thread, of a warp, warps; the caller's blocks of rows
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float s = (v[0][h][j] + v[1][h][j]) + (v[2][h][j] + v[3][h][j]);
          s += __shfl_xor_sync(0xffffffffu, s, 8);
          s += __shfl_xor_sync(0xffffffffu, s, 16);
          if (lane < 8) part[warp][c0 + h * 64 + j] = __float_as_uint(s);
        }
    }
  }
  uint32_t* out = tile + ((warp ^ (lane & 7)) * 4 + (lane >> 3));   // c / 8 mod 8 is lane mod 8
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const int c = c0 + h * 64 + j;
      const float2 s = SQUARE ? make_float2(row_inverse[0], row_inverse[0]) : *reinterpret_cast<const float2*>(inverse + c);
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        const uint32_t both = __byte_perm(__float_as_uint(s.x), __float_as_uint(s.y), 0x7632);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = times(v[i][h].w[j / 2], both);
        out[c * 32] = quantise4(low(w[0]), low(w[1]), low(w[2]), low(w[3]));
        out[(c + 1) * 32] = quantise4(high(w[0]), high(w[1]), high(w[2]), high(w[3]));
      } else {
        out[c * 32] = quantise4(v[0][h][j] * s.x, v[1][h][j] * s.x, v[2][h][j] * s.x, v[3][h][j] * s.x);
        out[(c + 1) * 32] = quantise4(v[0][h][j + 1] * s.y, v[1][h][j + 1] * s.y, v[2][h][j + 1] * s.y, v[3][h][j + 1] * s.y);
      }
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {   // a column leaves as 128 bytes, the last as M rounded up to 16
    const int c = i * 32 + warp * 4 + (lane >> 3), u = lane & 7;
    if (k0 + c < K && m0 + u * 16 < M)
      *reinterpret_cast<uint4*>(qt + static_cast<size_t>(k0 + c) * ldt + m0 + u * 16) = *reinterpret_cast<const uint4*>(tile + c * 32 + (u ^ (c >> 3 & 7)) * 4);
  }
  if (!SQUARE && sums != nullptr && threadIdx.x < kBlock && k0 + static_cast<int>(threadIdx.x) < K) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += __uint_as_float(part[w][threadIdx.x]);
    sums[static_cast<size_t>(blockIdx.x) * K + k0 + threadIdx.x] = s;
  }
}

// out[k] = the sum over the tiles' sums [tiles][K], in their order.  32 columns a block, eight threads a column.
template <typename T>
__global__ void __launch_bounds__(256) sum_tiles_kernel(const float* sums, int tiles, int K, T* __restrict__ out) {
  __shared__ float part[8][32];
  const int k = static_cast<int>(blockIdx.x) * 32 + static_cast<int>(threadIdx.x & 31), y = threadIdx.x >> 5;
  const int per = (tiles + 7) / 8;
  mnccl::wait_for_previous();
  mnccl::let_next_start();
  float s = 0.0f;
  if (k < K)
    for (int t = y * per; t < min(tiles, (y + 1) * per); ++t) s += sums[static_cast<size_t>(t) * K + k];
  part[y][threadIdx.x & 31] = s;
  __syncthreads();
  if (y != 0 || k >= K) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
  if constexpr (sizeof(T) == 4) out[k] = s;
  else if constexpr (std::is_same_v<T, __half>) out[k] = __float2half_rn(s);
  else out[k] = __float2bfloat16_rn(s);
}

int status(cudaError_t e) {
  return e == cudaSuccess ? 0 : static_cast<int>(e) + 1000;
}

template <typename T>
int quantise(const T* x, int64_t ldx, int M, int K, int block_rows, uint8_t* q, int64_t ldq, float* scale, uint8_t* qt, int64_t ldt, float* scale_t,
             float* sums, cudaStream_t stream) {
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (ldx * static_cast<int64_t>(sizeof(T))) % 16 == 0;
  const int blocks_k = (K + kBlock - 1) / kBlock, rows16 = (M + 15) / 16;
  const dim3 grid((M + kBlock - 1) / kBlock, blocks_k);
  if (block_rows == 128)
    return status(mnccl::launch_early(quantise_tile_kernel<T, true>, grid, dim3(kThreads), stream, x, ldx, M, K, q, ldq, scale, qt, ldt, scale_t, nullptr, vec));
  if (qt != nullptr)
    return status(mnccl::launch_early(quantise_tile_kernel<T, false>, grid, dim3(kThreads), stream, x, ldx, M, K, q, ldq, scale, qt, ldt, scale_t, sums, vec));
  // Enough for every SM several times over: four blocks a thread in flight (8192 x 4096 bf16: 24.7 us with one).
  if (static_cast<int64_t>(rows16) * blocks_k >= 4 * 2048)
    return status(mnccl::launch_early(quantise_rows_kernel<T, 4>, dim3(rows16, (blocks_k + 3) / 4), dim3(kThreads), stream, x, ldx, M, K, q, ldq, scale, vec));
  return status(mnccl::launch_early(quantise_rows_kernel<T, 1>, dim3(rows16, blocks_k), dim3(kThreads), stream, x, ldx, M, K, q, ldq, scale, vec));
}

constexpr int kMaxK = 65535 * kBlock;   // gridDim.y

}  // namespace

extern "C" {
#define MNCCL_EXPORT __attribute__((visibility("default")))

// x [M, K] (type 6 fp16, 7 fp32, 9 bf16; row stride ldx elements) -> q [M, K] e4m3 (row stride ldq, a multiple of 16 that holds K
// rounded up to one; 16-byte aligned; bytes up to that may be written, none behind it) and its scales: block_rows 1: scale[K blocks][M]; block_rows 128:
// scale[M blocks][K blocks].  qt, if not null: the transpose [K, M] (ldt like ldq), for block_rows 1 quantised anew in blocks along M
// with scale_t[M blocks][K].  sums, if not null (only with qt and block_rows 1): [M blocks][K], the columns' sums over each 128 rows.
// Returns 0, -1 null or empty, -2 shape or alignment, or a cudaError_t + 1000.
MNCCL_EXPORT int mncclQuantizeFp8(const void* x, int type, int64_t ldx, int M, int K, int block_rows, void* q, int64_t ldq, float* scale,
                                  void* qt, int64_t ldt, float* scale_t, float* sums, cudaStream_t stream) {
  if (!x || !q || !scale || M <= 0 || K <= 0 || (qt && block_rows == 1 && !scale_t)) return -1;
  const auto padded = [](const void* p, int64_t ld, int64_t n) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 16 == 0 && ld >= (n + 15) / 16 * 16;
  };
  if ((block_rows != 1 && block_rows != kBlock) || ldx < K || K > kMaxK || M > 0x7fffff00 || !padded(q, ldq, K) || (qt && !padded(qt, ldt, M)) ||
      (sums && (!qt || block_rows != 1)))
    return -2;
  uint8_t* qb = static_cast<uint8_t*>(q);
  uint8_t* tb = static_cast<uint8_t*>(qt);
  switch (type) {
    case 6: return quantise(static_cast<const __half*>(x), ldx, M, K, block_rows, qb, ldq, scale, tb, ldt, scale_t, sums, stream);
    case 7: return quantise(static_cast<const float*>(x), ldx, M, K, block_rows, qb, ldq, scale, tb, ldt, scale_t, sums, stream);
    case 9: return quantise(static_cast<const __nv_bfloat16*>(x), ldx, M, K, block_rows, qb, ldq, scale, tb, ldt, scale_t, sums, stream);
  }
  return -2;
}

// out[K] (type as above) = the columns' sums of mncclQuantizeFp8 over all `blocks` blocks of rows.  Returns as that.
MNCCL_EXPORT int mncclSumBlocks(const float* sums, int blocks, int K, void* out, int type, cudaStream_t stream) {
  if (!sums || !out || blocks <= 0 || K <= 0) return -1;
  if (K > kMaxK || blocks > 0x7fffff00 / kBlock) return -2;   // of what mncclQuantizeFp8 takes
  const dim3 grid(static_cast<unsigned>((K + 31) / 32));
  switch (type) {
    case 6: return status(mnccl::launch_early(sum_tiles_kernel<__half>, grid, dim3(256), stream, sums, blocks, K, out));
    case 7: return status(mnccl::launch_early(sum_tiles_kernel<float>, grid, dim3(256), stream, sums, blocks, K, out));
    case 9: return status(mnccl::launch_early(sum_tiles_kernel<__nv_bfloat16>, grid, dim3(256), stream, sums, blocks, K, out));
  }
  return -2;
}

}  // extern "C"
