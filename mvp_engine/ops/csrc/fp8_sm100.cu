// 8-bit floating point matrices with one power-of-two scale per block of 128, and their product.
//
// Format.  A block is 128 consecutive values of a row along the reduction, or (weights) a 128 x 128 tile.
//   e    = the least integer with amax <= MAX 2^e, at least -127         (MAX: 448 for e4m3, 57344 for e5m2)
//   code = value 2^-e rounded to the nearest 8-bit value, ties to even   (exact scaling, one rounding)
// A block holding a value that is not finite becomes NaN codes with e = 0.  Power-of-two scales are what the tensor
// core's block-scaled form takes (one unsigned exponent byte per 32 values of a row): a block of 128 is four such
// groups with the same byte, so the product needs no rescaling of partial sums outside the MMA.
//
// Layout.  codes [rows, blocks * 128], zero padded; scale bytes e + 127 in 512-byte atoms of 128 rows x 4 blocks,
// [rows / 128][blocks / 4][row % 32][row / 32 % 4][block % 4], zero padded: one atom is the image that tcgen05.cp
// spreads over the 4 x 32 lanes of tensor memory, so the product loads scales with plain 512-byte copies.
//
// Quantisation reads a matrix once and writes the codes of its rows, of its columns (the transposed matrix, blocks
// along the former rows), or both.  Its floor is memory: 2 bytes read and 1 or 2 written per bf16 value.  Measured, row blocks,
// both orientations: 8192 x 4096 in 29 us (4.6 TB/s; fp32 values 42 us, 4.8), 8192 x 12288 in 74 us (5.4 TB/s; fp32 114 us, 5.3);
// 128 x 128 tiles 27 and 68 us; e5m2 as e4m3.  Below some tens of millions of values the few waves of CTAs, whose load, reduction
// and store follow one another, keep it off the copy rate (6.45).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "pair_sm100.cuh"
#include "tma_host.h"

namespace mvp {
namespace fp8 {

constexpr int BLOCK = 128;
constexpr int ATOM = 512;  // scale bytes of 128 rows x 4 blocks

// ---------------------------------------------------------------------------------------- quantisation
constexpr int QT = 256;  // threads: 16 row groups of 8 rows x 16 lanes of 8 columns

struct QuantParams {
  const void* x;
  int64_t ld;            // row stride in elements (unit column stride)
  int rows, cols;
  int tile_cols;         // 128-column tiles per row of tiles
  uint8_t* q;            // codes of the rows [rows, col_blocks * 128], or null
  uint8_t* s;            // their scale atoms
  uint8_t* qt;           // codes of the columns [cols, row_blocks * 128], or null
  uint8_t* st;
  bool vec;              // rows are 16-byte aligned
};

// Scale byte of a block from the bits of its largest magnitude: 127 + e, or -1 if it is not finite.
// amax = 1.m 2^(E-127); MAX = 1.75 2^p, so e = E - 127 - p, one more if 1.m > 1.75: adding a quarter less one unit to the
// fraction carries into the exponent exactly then.
template <bool E5M2>
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
  constexpr int p = E5M2 ? 15 : 8;
  const int b = max(0, static_cast<int>((amax_bits + 0x1FFFFFu) >> 23) - p);
  return amax_bits >= 0x7F800000u ? -1 : b;
}
// 2^-e for scale byte b (b <= 247, so the exponent field stays in 7..254).
__device__ __forceinline__ float inverse_scale(int b) { return __uint_as_float(static_cast<uint32_t>(254 - b) << 23); }

// NaN codes in the first n of 8 places, zeros behind.
__device__ __forceinline__ uint2 nan_codes(int n) {
  return make_uint2(n >= 4 ? 0x7F7F7F7Fu : n <= 0 ? 0u : 0x7F7F7F7Fu >> (8 * (4 - n)),
                    n >= 8 ? 0x7F7F7F7Fu : n <= 4 ? 0u : 0x7F7F7F7Fu >> (8 * (8 - n)));
}

// 2^-e as a pair of bf16 (a power of two, so products with it are exact and subnormal ones end as zero codes either way).
__device__ __forceinline__ __nv_bfloat162 bf16_pair(float lo, float hi) { return __floats2bfloat162_rn(lo, hi); }
__device__ __forceinline__ uint32_t scaled2(uint32_t two, __nv_bfloat162 f) {
  const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&two), f);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Two codes, `lo` in the low byte.
template <bool E5M2>
__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}

// 8 values of a row as fp32 bits (bf16 values keep 16 bits each until used).
template <typename T>
struct Eight;
template <>
struct Eight<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int n, bool vec) {
    if (vec && n >= 8) {
      u = *reinterpret_cast<const uint4*>(p);
      return;
    }
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) w[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[j]) << (16 * (j & 1));
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ uint32_t bits(int j) const {
    const uint32_t w = j < 2 ? u.x : j < 4 ? u.y : j < 6 ? u.z : u.w;
    return (j & 1) ? (w & 0xFFFF0000u) : (w << 16);
  }
};
template <>
struct Eight<float> {
  uint4 a, b;
  __device__ __forceinline__ void load(const float* p, int n, bool vec) {
    if (vec && n >= 8) {
      a = reinterpret_cast<const uint4*>(p)[0];
      b = reinterpret_cast<const uint4*>(p)[1];
      return;
    }
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = j < n ? __float_as_uint(p[j]) : 0u;
    a = make_uint4(w[0], w[1], w[2], w[3]);
    b = make_uint4(w[4], w[5], w[6], w[7]);
  }
  __device__ __forceinline__ uint32_t bits(int j) const {
    return j == 0 ? a.x : j == 1 ? a.y : j == 2 ? a.z : j == 3 ? a.w : j == 4 ? b.x : j == 5 ? b.y : j == 6 ? b.z : b.w;
  }
};

// One CTA per 128 x 128 tile.  Thread (g, l) holds rows 8 g .. 8 g + 7 of columns 8 l .. 8 l + 7: a row's 128 columns are
// 16 lanes (its largest magnitude is four shuffles), and the 8 rows make 8-byte pieces of the transposed codes, which
// go through shared memory (16-byte pieces swizzled by column group, free of bank conflicts) to leave as whole rows.
// bf16 magnitudes are compared two at a time as 16-bit integers; that and four resident CTAs per SM (64 registers)
// keep the kernel near memory speed.
template <typename T, bool E5M2, bool TILE>
__global__ void __launch_bounds__(QT, sizeof(T) == 2 ? 4 : 2) quantize_kernel(const QuantParams p) {
  constexpr bool BF16 = sizeof(T) == 2;
  __shared__ __align__(16) uint8_t turned[BLOCK * BLOCK];
  __shared__ uint32_t col_max[QT / 32][BLOCK];
  __shared__ __align__(16) float col_inv[BLOCK];  // 2^-e of each column's block; 0: it is not finite
  __shared__ uint8_t col_byte[BLOCK];
  __shared__ __align__(8) uint8_t row_byte[BLOCK];
  const int tile_r = blockIdx.x / p.tile_cols, tile_c = blockIdx.x - tile_r * p.tile_cols;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int l = threadIdx.x % 16, g = threadIdx.x / 16;
  const int r0 = tile_r * BLOCK + g * 8, c0 = tile_c * BLOCK + l * 8;
  pdl_launch();
  Eight<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = (r0 + i < p.rows) ? p.cols - c0 : 0;
    v[i].load(static_cast<const T*>(p.x) + static_cast<int64_t>(n > 0 ? r0 + i : 0) * p.ld + (n > 0 ? c0 : 0), n, p.vec);
  }
  auto publish = [&](int col, uint32_t amax_bits) {
    const int b = scale_byte<E5M2>(amax_bits);
    col_inv[col] = b < 0 ? 0.f : inverse_scale(b);
    col_byte[col] = static_cast<uint8_t>(b < 0 ? 127 : b);
  };
  int row_b[8];
  if constexpr (TILE) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (BF16) {
        m = __vmaxu2(m, __vmaxu2(__vmaxu2(v[i].u.x & 0x7FFF7FFFu, v[i].u.y & 0x7FFF7FFFu),
                                 __vmaxu2(v[i].u.z & 0x7FFF7FFFu, v[i].u.w & 0x7FFF7FFFu)));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, v[i].bits(j) & 0x7FFFFFFFu);
      }
    }
    if constexpr (BF16) m = max(m & 0xFFFF0000u, m << 16);
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) col_max[warp][0] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < QT / 32; ++w) m = max(m, col_max[w][0]);
    const int b = scale_byte<E5M2>(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) row_b[i] = b;
    if (threadIdx.x < BLOCK) publish(threadIdx.x, m);
    __syncthreads();
  } else {
    if (p.q != nullptr) {
      if constexpr (BF16) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // rows 2 k (low half) and 2 k + 1 (high half)
          uint32_t m[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 u = v[2 * k + h].u;
            m[h] = __vmaxu2(__vmaxu2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu), __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
          }
          uint32_t both = __vmaxu2(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
          row_b[2 * k] = scale_byte<E5M2>(both << 16);
          row_b[2 * k + 1] = scale_byte<E5M2>(both & 0xFFFF0000u);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t m = 0u;
#pragma unroll
          for (int j = 0; j < 8; ++j) m = max(m, v[i].bits(j) & 0x7FFFFFFFu);
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          row_b[i] = scale_byte<E5M2>(m);
        }
      }
    }
    if (p.qt != nullptr) {
      if constexpr (BF16) {
        uint32_t m[4] = {0u, 0u, 0u, 0u};  // columns 8 l + 2 k (low half) and 8 l + 2 k + 1
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          m[0] = __vmaxu2(m[0], v[i].u.x & 0x7FFF7FFFu);
          m[1] = __vmaxu2(m[1], v[i].u.y & 0x7FFF7FFFu);
          m[2] = __vmaxu2(m[2], v[i].u.z & 0x7FFF7FFFu);
          m[3] = __vmaxu2(m[3], v[i].u.w & 0x7FFF7FFFu);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = __vmaxu2(m[k], __shfl_xor_sync(0xffffffffu, m[k], 16));
        if (lane < 16) *reinterpret_cast<uint4*>(&col_max[warp][l * 4]) = make_uint4(m[0], m[1], m[2], m[3]);
        __syncthreads();
        if (threadIdx.x < BLOCK / 2) {
          uint32_t t = 0u;
#pragma unroll
          for (int w = 0; w < QT / 32; ++w) t = __vmaxu2(t, col_max[w][threadIdx.x]);
          publish(2 * threadIdx.x, t << 16);
          publish(2 * threadIdx.x + 1, t & 0xFFFF0000u);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t m = 0u;
#pragma unroll
          for (int i = 0; i < 8; ++i) m = max(m, v[i].bits(j) & 0x7FFFFFFFu);
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
          if (lane < 16) col_max[warp][l * 8 + j] = m;
        }
        __syncthreads();
        if (threadIdx.x < BLOCK) {
          uint32_t m = 0u;
#pragma unroll
          for (int w = 0; w < QT / 32; ++w) m = max(m, col_max[w][threadIdx.x]);
          publish(threadIdx.x, m);
        }
      }
      __syncthreads();
    }
  }
  const int row_blocks = (p.rows + BLOCK - 1) / BLOCK;
  if (p.q != nullptr) {
    const int64_t ldq = static_cast<int64_t>(p.tile_cols) * BLOCK;
    const int groups = (p.tile_cols + 3) / 4;
    uint8_t* atom = p.s + (static_cast<int64_t>(tile_r) * groups + tile_c / 4) * ATOM;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = inverse_scale(max(row_b[i], 0));
      uint32_t w[4];
      if constexpr (BF16) {
        const __nv_bfloat162 ff = bf16_pair(f, f);
        const uint32_t u[4] = {scaled2(v[i].u.x, ff), scaled2(v[i].u.y, ff), scaled2(v[i].u.z, ff), scaled2(v[i].u.w, ff)};
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = codes2<E5M2>(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xFFFF0000u));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = codes2<E5M2>(__uint_as_float(v[i].bits(2 * j)) * f, __uint_as_float(v[i].bits(2 * j + 1)) * f);
      }
      uint2 out = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
      if (row_b[i] < 0) out = nan_codes(p.cols - c0);
      if (r0 + i < p.rows) *reinterpret_cast<uint2*>(p.q + (r0 + i) * ldq + c0) = out;
    }
    // the scale bytes of the tile's rows, one row per thread, from the lanes that hold them
    if (l == 0) {
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i / 4] |= static_cast<uint32_t>(r0 + i < p.rows ? (row_b[i] < 0 ? 127 : row_b[i]) : 0) << (8 * (i & 3));
      *reinterpret_cast<uint2*>(&row_byte[g * 8]) = make_uint2(w[0], w[1]);
    }
    __syncthreads();
    if (threadIdx.x < BLOCK) {
      uint8_t* a = atom + (threadIdx.x % 32) * 16 + (threadIdx.x / 32) * 4;
      a[tile_c % 4] = row_byte[threadIdx.x];
      if (tile_c == p.tile_cols - 1)  // blocks the atom has beyond the matrix
        for (int b = tile_c % 4 + 1; b < 4; ++b) a[b] = 0;
    }
  }
  if (p.qt != nullptr) {
    const int groups = (row_blocks + 3) / 4;
    const float4 inv0 = *reinterpret_cast<const float4*>(col_inv + l * 8);
    const float4 inv1 = *reinterpret_cast<const float4*>(col_inv + l * 8 + 4);
    const float inv[8] = {inv0.x, inv0.y, inv0.z, inv0.w, inv1.x, inv1.y, inv1.z, inv1.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // columns 8 l + 2 k and the next
      uint32_t w[2][4];
      if constexpr (BF16) {
        const __nv_bfloat162 ff = bf16_pair(inv[2 * k], inv[2 * k + 1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 e = v[2 * i].u, o = v[2 * i + 1].u;
          const uint32_t u0 = scaled2(k == 0 ? e.x : k == 1 ? e.y : k == 2 ? e.z : e.w, ff);
          const uint32_t u1 = scaled2(k == 0 ? o.x : k == 1 ? o.y : k == 2 ? o.z : o.w, ff);
          w[0][i] = codes2<E5M2>(__uint_as_float(u0 << 16), __uint_as_float(u1 << 16));
          w[1][i] = codes2<E5M2>(__uint_as_float(u0 & 0xFFFF0000u), __uint_as_float(u1 & 0xFFFF0000u));
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[h][i] = codes2<E5M2>(__uint_as_float(v[2 * i].bits(2 * k + h)) * inv[2 * k + h],
                                   __uint_as_float(v[2 * i + 1].bits(2 * k + h)) * inv[2 * k + h]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint2 out = make_uint2(w[h][0] | (w[h][1] << 16), w[h][2] | (w[h][3] << 16));
        if (inv[2 * k + h] == 0.f) out = nan_codes(p.rows - r0);
        *reinterpret_cast<uint2*>(turned + (l * 8 + 2 * k + h) * BLOCK + (g ^ l) * 8) = out;
      }
    }
    if (threadIdx.x < BLOCK) {
      const int col = tile_c * BLOCK + threadIdx.x;
      uint8_t* a = p.st + (static_cast<int64_t>(tile_c) * groups + tile_r / 4) * ATOM + (threadIdx.x % 32) * 16 +
                   (threadIdx.x / 32) * 4;
      a[tile_r % 4] = col < p.cols ? col_byte[threadIdx.x] : 0;
      if (tile_r == row_blocks - 1)
        for (int k = tile_r % 4 + 1; k < 4; ++k) a[k] = 0;
    }
    __syncthreads();
    const int64_t ldt = static_cast<int64_t>(row_blocks) * BLOCK;
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
      const int col = pass * 32 + threadIdx.x / 8, k = threadIdx.x % 8;
      const int sw = col / 8;  // the swizzle of this column's 8-byte pieces
      uint4 u = *reinterpret_cast<const uint4*>(turned + col * BLOCK + (k ^ (sw >> 1)) * 16);
      if (sw & 1) u = make_uint4(u.z, u.w, u.x, u.y);
      if (tile_c * BLOCK + col < p.cols)
        *reinterpret_cast<uint4*>(p.qt + (static_cast<int64_t>(tile_c) * BLOCK + col) * ldt + tile_r * BLOCK + k * 16) = u;
    }
  }
  // Where this kernel may start before the one in front of it has ended (the second quantisation of a linear layer, which
  // shares nothing with the first), it ends after it: what waits for this kernel may then rely on both.
  pdl_wait();
}

template <typename T>
void quantize(const QuantParams& p, bool e5m2, bool tile, int ctas, bool early, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(QT);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  auto kern = tile ? (e5m2 ? quantize_kernel<T, true, true> : quantize_kernel<T, false, true>)
                   : (e5m2 ? quantize_kernel<T, true, false> : quantize_kernel<T, false, false>);
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
}

}  // namespace fp8

// ------------------------------------------------------------------------------------------------ product
//   C[M, N] (+)= A[M, K] B[N, K]^T of two such matrices, fp32 accumulation
//
// The pair-of-SMs GEMM (roles as in gemm2sm_sm100.cu) with tcgen05.mma kind::mxf8f6f4.block_scale: per 128-deep
// k-block each CTA loads 128 rows of A and half a tile's rows of B and every fourth k-block the scale atoms (its 128 rows
// of A; all rows of B, which both SMs of a pair need), which tcgen05.cp moves to tensor memory; the
// k-block's byte of a scale word is picked by the instruction descriptor.
//
// Tiles are 256 x TN, TN = 256, 192 or 128, whichever gives the shortest schedule (choose_tile).
// Tensor memory: the last 64 of 512 columns hold four sets of scales (16 columns each); the accumulators start at
// columns 0 and 192.  For TN = 256 they share 64 columns: the epilogue reads those first and hands them back at
// once, and the next tile's MMAs wait for that.  For smaller tiles they wait only for the tile two before.
// A set of scales is used again four groups (of four k-blocks) later.  At most one tile boundary lies in between (the
// tile two before has been read out), so at least 10 k-blocks do, more than the ring's stages: the full
// stage that the new group waits for was emptied after the old group's MMAs.
//
// Bound by the tensor core, and for long runs by the power limit: 8192 x 4096 -> 24576 in 560 to 585 us in short runs (2.8 to
// 2.9 PFLOP/s, 0.87 of twice the bf16 rate measured on the same GPU) and 660 to 690 us in long ones (2.4 to 2.5),
// 8192 x 12288 -> 4096 in 270 to 280 and 325 us.  Adding into an fp32 C costs 9 to 25 % more: its rows are read behind the
// accumulator, and the ring is one stage shorter.
namespace fp8gemm {

using namespace gemm2;
using fp8::ATOM;

constexpr int BK = 128;
constexpr int TM = 256;
constexpr int HALF = 128;
constexpr int A_BYTES = HALF * BK;
constexpr int TMEM_COLS = 512;
constexpr int ACC1_COL = 192;
constexpr int SF_COL = 448;
constexpr int EPI_WARPS = 8;  // two for each quarter of the accumulator's lanes, half of the columns each
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int CHUNK = 32;     // columns the epilogue handles at a time

enum Epilogue : int { kStoreBf16 = 0, kStoreF32 = 1, kAccumF32 = 2 };

template <int TN, int EPI>
struct Plan {
  static constexpr int B_BYTES = TN / 2 * BK;
  static constexpr int SFB = TN == 128 ? 1 : 2;  // atoms that TN columns touch (192: 64 columns off every other tile)
  static constexpr int SF_BYTES = (1 + SFB) * ATOM;
  static constexpr int STAGES = EPI == kStoreBf16 ? 6 : 5;
  static constexpr int EPI_BUF = 32 * CHUNK * (EPI == kStoreBf16 ? 2 : 4);
  static constexpr int SMEM = STAGES * (A_BYTES + B_BYTES + SF_BYTES) + EPI_WARPS * EPI_BUF + 1024 + 256;
  static constexpr bool SHARED_COLS = TN > ACC1_COL;
  static constexpr int CHUNKS = TN / 2 / CHUNK;  // per epilogue warp
};

struct Params {
  int M, N;
  int num_kb;   // 128-deep k-blocks
  int sf_groups;  // scale atoms per 128 rows
  void* C;
  int64_t ldc;
  bool vec;     // rows of C are 16-byte aligned
  uint32_t idesc;
  int* status;
};

__device__ __forceinline__ void mma_scaled_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 32 rows x 16 bytes of shared memory to the 4 columns at `taddr`, repeated in the four 32-lane quarters, in both CTAs.
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t smem_addr) {
  // no swizzle, 8-row groups 128 bytes apart
  const uint64_t desc = static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128 >> 4) << 32) |
                        (1ull << 46);
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// kind::mxf8f6f4: types (0 e4m3, 1 e5m2) at bits 7 and 10, N / 8 at 17, unsigned-exponent scales at 23, M / 16 at 24;
// the scale byte of the k-block goes to bits 29 (A) and 4 (B).
inline uint32_t make_idesc(bool a_e5m2, bool b_e5m2, int tn) {
  return ((a_e5m2 ? 1u : 0u) << 7) | ((b_e5m2 ? 1u : 0u) << 10) | ((static_cast<uint32_t>(tn) >> 3) << 17) |
         (1u << 23) | ((static_cast<uint32_t>(TM) >> 4) << 24);
}

template <int TN>
__device__ __forceinline__ void tile_coords(const Params& p, int t, int& tm, int& tn) {
  constexpr int kGroup = 8;
  const int num_m = (p.M + TM - 1) / TM, num_n = (p.N + TN - 1) / TN;
  const int per_group = kGroup * num_n;
  const int g = t / per_group, first = g * kGroup;
  const int gm = min(kGroup, num_m - first);
  const int r = t - g * per_group;
  tm = first + r % gm;
  tn = r / gm;
}

// A warp's 32 rows x 32 columns from one row per lane to C: through the warp's shared memory in 16-byte pieces swizzled by
// row, so that 4 (bf16) or 8 (fp32) consecutive lanes write each row.
template <int EPI>
__device__ __forceinline__ void store_chunk(const Params& p, uint8_t* buf, int m0, int n, const uint32_t (&r)[32]) {
  if (m0 >= p.M || n >= p.N) return;  // same for all lanes
  const int lane = threadIdx.x % 32;
  if constexpr (EPI == kStoreBf16) {
    auto piece = [](int row, int j) { return row * 64 + ((j ^ ((row >> 1) & 3)) << 4); };
#pragma unroll
    for (int v = 0; v < 4; ++v)
      *reinterpret_cast<uint4*>(buf + piece(lane, v)) =
          make_uint4(pack_bf16x2(__uint_as_float(r[8 * v]), __uint_as_float(r[8 * v + 1])),
                     pack_bf16x2(__uint_as_float(r[8 * v + 2]), __uint_as_float(r[8 * v + 3])),
                     pack_bf16x2(__uint_as_float(r[8 * v + 4]), __uint_as_float(r[8 * v + 5])),
                     pack_bf16x2(__uint_as_float(r[8 * v + 6]), __uint_as_float(r[8 * v + 7])));
    __syncwarp();
    __nv_bfloat16* C = static_cast<__nv_bfloat16*>(p.C) + static_cast<int64_t>(m0) * p.ldc + n;
    if (p.vec && n + CHUNK <= p.N) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + lane / 4, j = lane & 3;
        if (m0 + row < p.M)
          *reinterpret_cast<uint4*>(C + row * p.ldc + j * 8) = *reinterpret_cast<const uint4*>(buf + piece(row, j));
      }
    } else {
#pragma unroll 8
      for (int row = 0; row < 32; ++row)
        if (m0 + row < p.M && n + lane < p.N)
          C[row * p.ldc + lane] = *reinterpret_cast<const __nv_bfloat16*>(buf + piece(row, lane / 8) + (lane & 7) * 2);
    }
  } else {
    auto piece = [](int row, int j) { return row * 128 + ((j ^ (row & 7)) << 4); };
    float* C = static_cast<float*>(p.C) + static_cast<int64_t>(m0) * p.ldc + n;
#pragma unroll
    for (int v = 0; v < 8; ++v)
      *reinterpret_cast<uint4*>(buf + piece(lane, v)) = make_uint4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
    __syncwarp();
    if (p.vec && n + CHUNK <= p.N) {
      const int j = lane & 7;
#pragma unroll
      for (int i0 = 0; i0 < 8; i0 += 4) {
        float4 o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (EPI == kAccumF32 && m0 + (i0 + i) * 4 + lane / 8 < p.M)
            o[i] = *reinterpret_cast<const float4*>(C + ((i0 + i) * 4 + lane / 8) * p.ldc + j * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (i0 + i) * 4 + lane / 8;
          if (m0 + row >= p.M) continue;
          float4 q = *reinterpret_cast<const float4*>(buf + piece(row, j));
          if constexpr (EPI == kAccumF32) {
            q.x += o[i].x;
            q.y += o[i].y;
            q.z += o[i].z;
            q.w += o[i].w;
          }
          *reinterpret_cast<float4*>(C + row * p.ldc + j * 4) = q;
        }
      }
    } else {
#pragma unroll 4
      for (int row = 0; row < 32; ++row)
        if (m0 + row < p.M && n + lane < p.N) {
          float q = *reinterpret_cast<const float*>(buf + piece(row, lane / 4) + (lane & 3) * 4);
          if constexpr (EPI == kAccumF32) q += C[row * p.ldc + lane];
          C[row * p.ldc + lane] = q;
        }
    }
  }
  __syncwarp();  // the buffer may be written again
}

template <int TN, int EPI>
__global__ void __launch_bounds__(THREADS, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const Params p) {
  using P = Plan<TN, EPI>;
  constexpr int STAGES = P::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint8_t* sS = sB + STAGES * P::B_BYTES;
  uint8_t* sE = sS + STAGES * P::SF_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sE + EPI_WARPS * P::EPI_BUF);  // used in the leader
  uint64_t* empty_bar = full_bar + STAGES;                                        // both CTAs
  uint64_t* tfull_bar = empty_bar + STAGES;                                       // [2] both CTAs
  uint64_t* handed_bar = tfull_bar + 2;  // [2] used in the leader: an accumulator (or its shared columns) has been read
  uint64_t* done_bar = handed_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const uint32_t crank = cluster_ctarank();  // 0 = leader
  const int cluster_id = blockIdx.x >> 1;
  const int clusters = gridDim.x >> 1;
  const int total = ((p.M + TM - 1) / TM) * ((p.N + TN - 1) / TN);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&handed_bar[a], 2 * 32 * EPI_WARPS);  // epilogue threads of both CTAs
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // barriers of both CTAs initialised before any remote arrive / copy
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch();
  pdl_wait();  // every thread: the operands are written by the kernels before this one

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (elect_one_sync()) {
      const uint32_t leader_full0 = mapa_shared(smem_u32(&full_bar[0]), 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, issued = false;
      for (int t = cluster_id; ok && t < total; t += clusters) {
        int tm, tn;
        tile_coords<TN>(p, t, tm, tn);
        const int m0 = tm * TM + crank * HALF, n0 = tn * TN + crank * (TN / 2);
        const int sa = (tm * 2 + static_cast<int>(crank)) * p.sf_groups, sb = (tn * TN / HALF) * p.sf_groups;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, abort_flag, p.status, kTimeoutProducer)) {
            ok = false;
            break;
          }
          const bool scales = (kb & 3) == 0;
          if (crank == 0)
            mbar_arrive_expect_tx(&full_bar[stage], 2 * (A_BYTES + P::B_BYTES + (scales ? P::SF_BYTES : 0)));
          issued = true;
          const uint32_t bar = leader_full0 + stage * 8;
          tma_load_2d_pair(sA + stage * A_BYTES, &tmA, bar, kb * BK, m0);
          tma_load_2d_pair(sB + stage * P::B_BYTES, &tmB, bar, kb * BK, n0);
          if (scales) {
            uint8_t* dst = sS + stage * P::SF_BYTES;
            tma_load_2d_pair(dst, &tmSA, bar, 0, sa + kb / 4);
#pragma unroll
            for (int a = 0; a < P::SFB; ++a)
              tma_load_2d_pair(dst + (1 + a) * ATOM, &tmSB, bar, 0, sb + a * p.sf_groups + kb / 4);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // After an abort, let copies already issued into this CTA's ring land (bounded) before exit.
      if ((!ok || *abort_flag) && issued) {
        const uint64_t t0 = globaltimer();
        while (globaltimer() - t0 < 200000000ull) {
        }
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA (leader only)
    if (crank == 0 && elect_one_sync()) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0, group = 0;
      bool ok = true;
      for (int t = cluster_id; ok && t < total; t += clusters, ++local) {
        const int before = local - (P::SHARED_COLS ? 1 : 2);  // the tile whose read-out this one waits for
        if (before >= 0 &&
            !mbar_wait_bounded(&handed_bar[before & 1], (before >> 1) & 1, abort_flag, p.status, kTimeoutMma))
          break;
        tc_fence_after();
        int tm, tn;
        tile_coords<TN>(p, t, tm, tn);
        const uint32_t d_tmem = tmem_base + (local & 1) * ACC1_COL;
        const uint32_t shift = (tn * TN % HALF) / 32;  // TN = 192: an odd tile starts at row 64 of its first atom
        uint32_t sf = 0;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait_bounded(&full_bar[stage], phase, abort_flag, p.status, kTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if ((kb & 3) == 0) {
            sf = tmem_base + SF_COL + (group++ & 3) * 16;
            const uint32_t src = smem_u32(sS + stage * P::SF_BYTES);
            scales_to_tmem(sf, src);
#pragma unroll
            for (int a = 0; a < P::SFB; ++a) scales_to_tmem(sf + 8 + 4 * a, src + (1 + a) * ATOM);
          }
          const uint32_t idesc = p.idesc | (static_cast<uint32_t>(kb & 3) << 29) | (static_cast<uint32_t>(kb & 3) << 4);
          const uint32_t a_base = smem_u32(sA + stage * A_BYTES);
          const uint32_t b_base = smem_u32(sB + stage * P::B_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_scaled_pair(d_tmem, make_smem_desc_sw128(a_base + k * 32, 16, 1024),
                            make_smem_desc_sw128(b_base + k * 32, 16, 1024), idesc, sf, sf + 8 + shift,
                            (kb != 0 || k != 0) ? 1u : 0u);
          mma_commit_pair(&empty_bar[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit_pair(&tfull_bar[local & 1]);
      }
      mma_commit_pair_local(done_bar);
      mbar_wait_bounded(done_bar, 0, abort_flag, p.status, kTimeoutDrain);
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int sub = warp & 3, ew = warp - 2, half = ew / 4;
    uint8_t* const buf = sE + ew * P::EPI_BUF;
    const uint32_t leader_handed = mapa_shared(smem_u32(&handed_bar[0]), 0);
    const uint32_t lanes = static_cast<uint32_t>(sub * 32) << 16;
    int local = 0;
    for (int t = cluster_id; t < total; t += clusters, ++local) {
      int tm, tn;
      tile_coords<TN>(p, t, tm, tn);
      const int acc = local & 1;
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tfull_bar[acc], (local >> 1) & 1, abort_flag, p.status,
                                                     kTimeoutEpilogue)))
        break;
      tc_fence_after();
      const int m0 = tm * TM + static_cast<int>(crank) * HALF + sub * 32;
      const int n0 = tn * TN + half * (TN / 2);
      const uint32_t base = tmem_base + lanes + acc * ACC1_COL + half * (TN / 2);
      int first = 0, count = P::CHUNKS;  // chunks still to be read after the shared columns
      if constexpr (P::SHARED_COLS) {
        // columns shared with the other accumulator: the last 64 of accumulator 0, the first 64 of accumulator 1
        const bool mine = half == 1 - acc;
        if (mine) {
          const int c = acc == 0 ? P::CHUNKS - 2 : 0;
          uint32_t r0[32], r1[32];
          tmem_ld_32x32b_x32(base + c * CHUNK, r0);
          tmem_ld_32x32b_x32(base + c * CHUNK + CHUNK, r1);
          tmem_wait_ld();
          tc_fence_before();
          remote_arrive_relaxed(leader_handed + acc * 8);
          store_chunk<EPI>(p, buf, m0, n0 + c * CHUNK, r0);
          store_chunk<EPI>(p, buf, m0, n0 + c * CHUNK + CHUNK, r1);
          first = acc == 0 ? 0 : 2;
          count = P::CHUNKS - 2;
        } else {
          tc_fence_before();
          remote_arrive_relaxed(leader_handed + acc * 8);  // this warp's part of the tile before has been read
        }
      }
#pragma unroll 1
      for (int i = 0; i < count; ++i) {
        const int c = first + i;
        uint32_t r[32];
        tmem_ld_32x32b_x32(base + c * CHUNK, r);
        tmem_wait_ld();
        if (!P::SHARED_COLS && i == count - 1) {
          tc_fence_before();
          remote_arrive_relaxed(leader_handed + acc * 8);
        }
        store_chunk<EPI>(p, buf, m0, n0 + c * CHUNK, r);
      }
    }
  }

  // Both CTAs: every role is done (the leader's MMAs have retired); then free the pair's TMEM.
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

inline void encode(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t inner, int64_t outer,
                   int64_t row_bytes, uint32_t box0, uint32_t box1, CUtensorMapSwizzle swizzle) {
  ensure_thread_context();
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
  cuuint32_t box[2] = {box0, box1};
  cuuint32_t es[2] = {1, 1};
  const CUresult r = encode_tiled_fn()(map, type, 2, const_cast<void*>(base), dims, strides, box, es,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "gemm_fp8: cuTensorMapEncodeTiled failed with code ", static_cast<int>(r));
}

// Tile width with the shortest schedule: waves x (cycles of a tile: its k-blocks, plus what it costs besides), and the last
// tile's read-out.  A k-block of 128 takes 2 TN cycles at the tensor core's rate and a little more where A's share of the
// shared-memory traffic grows.  Measured with each width in turn (us at 256 / 192 / 128 columns, bf16 result):
//   256 x 4096 -> 4096   15.9 / 13.1 / 11.6     8192 x 4096 -> 4096    106 / 109 / 128
//   777 x 2560 -> 9728   25.4 / 20.5 / 25.3     8192 x 4096 -> 24576   694 / 665 / 836  (256: hand-over of the shared columns)
//   4096 x 4096 -> 4096  66.7 / 61.9 / 70.5     8192 x 12288 -> 4096   328 / 349 / 402
// Over 14 such shapes the choice is within 1 % of the best, and within 8 % where C is added to in fp32 (8192 x 4096 -> 12288:
// 388 at 256 columns, 408 at the chosen 192), whose longer read-out it does not weigh.
inline int choose_tile(int64_t M, int64_t N, int num_kb, int sms) {
  const int64_t clusters = std::max(1, sms / 2);
  struct Width {
    int tn, block, besides;
  };
  int best = 256;
  int64_t best_cost = -1;
  for (const Width w : {Width{256, 512, 700}, Width{192, 390, 150}, Width{128, 350, 150}}) {
    const int64_t tiles = (M + TM - 1) / TM * ((N + w.tn - 1) / w.tn);
    const int64_t waves = (tiles + clusters - 1) / clusters;
    const int64_t cost = waves * (static_cast<int64_t>(w.block) * num_kb + w.besides) + 8 * w.tn;
    if (best_cost < 0 || cost < best_cost) {
      best = w.tn;
      best_cost = cost;
    }
  }
  return best;
}

template <int TN, int EPI>
void launch(const CUtensorMap (&t)[4], const Params& p, int sms, cudaStream_t stream) {
  auto kern = fp8_gemm_kernel<TN, EPI>;
  static std::atomic<uint64_t> configured{0};
  allow_smem(kern, Plan<TN, EPI>::SMEM, configured);
  const int64_t tiles = static_cast<int64_t>((p.M + TM - 1) / TM) * ((p.N + TN - 1) / TN);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min<int64_t>(tiles, std::max(1, sms / 2))));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Plan<TN, EPI>::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, t[0], t[1], t[2], t[3], p));
}

template <int TN>
void launch_tile(int epi, const CUtensorMap (&t)[4], const Params& p, int sms, cudaStream_t stream) {
  if (epi == kStoreBf16) launch<TN, kStoreBf16>(t, p, sms, stream);
  else if (epi == kStoreF32) launch<TN, kStoreF32>(t, p, sms, stream);
  else launch<TN, kAccumF32>(t, p, sms, stream);
}

}  // namespace fp8gemm
}  // namespace mvp

namespace {

using mvp::fp8::ATOM;
using mvp::fp8::BLOCK;

bool is_e5m2(const torch::Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kFloat8_e5m2, what,
              ": codes are float8_e4m3fn or float8_e5m2");
  return t.scalar_type() == at::kFloat8_e5m2;
}

int64_t blocks_of(int64_t n) { return (n + BLOCK - 1) / BLOCK; }
int64_t code_bytes(int64_t rows, int64_t cols) { return rows * blocks_of(cols) * BLOCK; }
int64_t scale_bytes(int64_t rows, int64_t cols) { return blocks_of(rows) * ((blocks_of(cols) + 3) / 4) * ATOM; }

// A quantised matrix [rows, cols] (or none: data == nullptr).
struct Matrix {
  uint8_t* data = nullptr;
  uint8_t* scale = nullptr;
  int64_t rows = 0, cols = 0;
  bool e5m2 = false;
};

// The matrix of an Fp8Matrix's two tensors, checked.
Matrix as_matrix(const torch::Tensor& data, const torch::Tensor& scale, int64_t cols, const torch::Device& dev,
                 const char* what) {
  Matrix m;
  m.e5m2 = is_e5m2(data, what);
  m.rows = data.size(0);
  m.cols = cols;
  TORCH_CHECK(data.device() == dev && data.dim() == 2 && data.is_contiguous() && data.size(0) > 0 && cols > 0 &&
                  data.size(1) == blocks_of(cols) * BLOCK,
              what, ": contiguous codes [rows, whole blocks of 128] on the operands' device");
  TORCH_CHECK(scale.device() == dev && scale.scalar_type() == at::kByte && scale.is_contiguous() &&
                  scale.numel() == scale_bytes(m.rows, cols),
              what, ": scale bytes");
  m.data = static_cast<uint8_t*>(data.data_ptr());
  m.scale = scale.data_ptr<uint8_t>();
  TORCH_CHECK((reinterpret_cast<uintptr_t>(m.data) & 15) == 0 && (reinterpret_cast<uintptr_t>(m.scale) & 15) == 0, what,
              ": 16-byte aligned codes and scales");
  return m;
}

// New tensors for a quantised matrix.
Matrix new_matrix(int64_t rows, int64_t cols, bool e5m2, const torch::Tensor& like, torch::Tensor& data,
                  torch::Tensor& scale) {
  data = torch::empty({rows, blocks_of(cols) * BLOCK}, like.options().dtype(e5m2 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn));
  scale = torch::empty({blocks_of(rows), (blocks_of(cols) + 3) / 4, 32, 4, 4}, like.options().dtype(at::kByte));
  Matrix m;
  m.data = static_cast<uint8_t*>(data.data_ptr());
  m.scale = scale.data_ptr<uint8_t>();
  m.rows = rows;
  m.cols = cols;
  m.e5m2 = e5m2;
  return m;
}

// Space in a call's own buffer for a matrix that does not outlive the call; `used` grows by it.
void place(Matrix& m, int64_t rows, int64_t cols, bool e5m2, uint8_t* base, int64_t& used) {
  auto up = [](int64_t n) { return (n + 511) / 512 * 512; };
  m.rows = rows;
  m.cols = cols;
  m.e5m2 = e5m2;
  m.data = base + used;
  m.scale = m.data + up(code_bytes(rows, cols));
  used += up(code_bytes(rows, cols)) + up(scale_bytes(rows, cols));
}

// x (checked: a CUDA matrix with unit column stride, bf16 or fp32) into q and / or, transposed, t.
void quantize_into(const torch::Tensor& x, bool tile, const Matrix& q, const Matrix& t, bool early, cudaStream_t stream) {
  using namespace mvp::fp8;
  const int64_t rb = blocks_of(x.size(0)), cb = blocks_of(x.size(1));
  TORCH_CHECK(x.size(0) < (int64_t(1) << 31) - 256 && x.size(1) < (int64_t(1) << 31) - 256 &&
                  rb * cb < (int64_t(1) << 31),
              "quantize_fp8: too many blocks");
  QuantParams p{};
  p.x = x.data_ptr();
  p.ld = x.stride(0);
  p.rows = static_cast<int>(x.size(0));
  p.cols = static_cast<int>(x.size(1));
  p.tile_cols = static_cast<int>(cb);
  p.vec = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && (p.ld * x.element_size()) % 16 == 0;
  p.q = q.data;
  p.s = q.scale;
  p.qt = t.data;
  p.st = t.scale;
  const bool e5m2 = q.data != nullptr ? q.e5m2 : t.e5m2;
  const int ctas = static_cast<int>(rb * cb);
  if (x.scalar_type() == at::kBFloat16) quantize<__nv_bfloat16>(p, e5m2, tile, ctas, early, stream);
  else quantize<float>(p, e5m2, tile, ctas, early, stream);
}

void check_input(const torch::Tensor& x, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(0) > 0 && x.size(1) > 0 && (x.stride(1) == 1 || x.size(1) == 1), what,
              ": CUDA matrix with unit column stride");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat, what, ": bf16 or fp32 input");
}

// c (+)= a b^T; c checked against a and b here.
void gemm_into(const Matrix& a, const Matrix& b, torch::Tensor& c, bool accumulate, int64_t status_ptr,
               cudaStream_t stream) {
  using namespace mvp::fp8gemm;
  TORCH_CHECK(a.cols == b.cols, "gemm_fp8: reduction sizes differ");
  constexpr int64_t kMost = (int64_t(1) << 31) - 512;
  const int64_t kb = blocks_of(a.cols), groups = (kb + 3) / 4, ra = blocks_of(a.rows), rb = blocks_of(b.rows);
  TORCH_CHECK(a.rows < kMost && b.rows < kMost && kb * BLOCK < kMost && (ra + 2) * groups < kMost &&
                  (rb + 2) * groups < kMost && ((ra + 1) / 2) * rb < kMost,
              "gemm_fp8: sizes");
  TORCH_CHECK(c.dim() == 2 && c.size(0) == a.rows && c.size(1) == b.rows && (c.stride(1) == 1 || c.size(1) == 1) &&
                  (c.size(0) == 1 || c.stride(0) >= c.size(1)),
              "gemm_fp8: output [M, N] with unit column stride");
  TORCH_CHECK(c.scalar_type() == at::kFloat || (c.scalar_type() == at::kBFloat16 && !accumulate),
              "gemm_fp8: bf16 or fp32 output, fp32 to accumulate");
  const int sms = mvp::num_sms(c.get_device());
  const int tn = choose_tile(a.rows, b.rows, static_cast<int>(kb), sms);
  CUtensorMap t[4];
  const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  encode(&t[0], u8, a.data, kb * BLOCK, a.rows, kb * BLOCK, BK, HALF, CU_TENSOR_MAP_SWIZZLE_128B);
  encode(&t[1], u8, b.data, kb * BLOCK, b.rows, kb * BLOCK, BK, tn / 2, CU_TENSOR_MAP_SWIZZLE_128B);
  const auto u32 = CU_TENSOR_MAP_DATA_TYPE_UINT32;
  encode(&t[2], u32, a.scale, ATOM / 4, ra * groups, ATOM, ATOM / 4, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
  encode(&t[3], u32, b.scale, ATOM / 4, rb * groups, ATOM, ATOM / 4, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
  Params p{};
  p.M = static_cast<int>(a.rows);
  p.N = static_cast<int>(b.rows);
  p.num_kb = static_cast<int>(kb);
  p.sf_groups = static_cast<int>(groups);
  p.C = c.data_ptr();
  p.ldc = c.stride(0);
  p.idesc = make_idesc(a.e5m2, b.e5m2, tn);
  p.vec = (reinterpret_cast<uintptr_t>(p.C) & 15) == 0 && (p.ldc * c.element_size()) % 16 == 0;
  p.status = reinterpret_cast<int*>(status_ptr);
  const int epi = c.scalar_type() == at::kBFloat16 ? kStoreBf16 : accumulate ? kAccumF32 : kStoreF32;
  if (tn == 256) launch_tile<256>(epi, t, p, sms, stream);
  else if (tn == 192) launch_tile<192>(epi, t, p, sms, stream);
  else launch_tile<128>(epi, t, p, sms, stream);
}

}  // namespace

// {codes, scales} of x's rows and {codes, scales} of its columns (undefined where not asked for); tile: 128 x 128 blocks
// instead of 1 x 128.
std::vector<torch::Tensor> quantize_fp8(const torch::Tensor& x, bool tile, bool rows, bool columns, bool e5m2) {
  check_input(x, "quantize_fp8");
  TORCH_CHECK(rows || columns, "quantize_fp8: nothing to write");
  const at::cuda::CUDAGuard guard(x.device());
  std::vector<torch::Tensor> out(4);
  Matrix q, t;
  if (rows) q = new_matrix(x.size(0), x.size(1), e5m2, x, out[0], out[1]);
  if (columns) t = new_matrix(x.size(1), x.size(0), e5m2, x, out[2], out[3]);
  quantize_into(x, tile, q, t, false, at::cuda::getCurrentCUDAStream());
  return out;
}

// c (+)= a b^T of quantised matrices with `cols` values per row.
void gemm_fp8(const torch::Tensor& a, const torch::Tensor& sa, const torch::Tensor& b, const torch::Tensor& sb,
              int64_t cols, torch::Tensor& c, bool accumulate, int64_t status_ptr) {
  TORCH_CHECK(a.is_cuda() && c.device() == a.device(), "gemm_fp8: CUDA operands and output on one device");
  const Matrix ma = as_matrix(a, sa, cols, a.device(), "gemm_fp8"), mb = as_matrix(b, sb, cols, a.device(), "gemm_fp8");
  const at::cuda::CUDAGuard guard(a.device());
  gemm_into(ma, mb, c, accumulate, status_ptr, at::cuda::getCurrentCUDAStream());
}

// Forward of ops.linear_fp8: {y, x^T codes, scales, w^T codes, scales} (the last four where asked for).  w8 / sw8: w's codes
// kept by the caller.
std::vector<torch::Tensor> linear_fp8_fwd(const torch::Tensor& x, const torch::Tensor& w,
                                          const c10::optional<torch::Tensor>& w8, const c10::optional<torch::Tensor>& sw8,
                                          bool need_xt, bool need_wt, int64_t status_ptr) {
  check_input(x, "linear_fp8");
  check_input(w, "linear_fp8");
  TORCH_CHECK(x.device() == w.device() && x.size(1) == w.size(1), "linear_fp8: x [T, K] and w [N, K] on one device");
  const at::cuda::CUDAGuard guard(x.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int64_t T = x.size(0), K = x.size(1), N = w.size(0);
  const bool own_w = !w8.has_value();
  int64_t bytes = 0;
  Matrix mx, mw, mxt, mwt;
  place(mx, T, K, false, nullptr, bytes);
  if (own_w) place(mw, N, K, false, nullptr, bytes);
  auto buf = torch::empty({bytes}, x.options().dtype(at::kByte));
  bytes = 0;
  place(mx, T, K, false, buf.data_ptr<uint8_t>(), bytes);
  if (own_w) place(mw, N, K, false, buf.data_ptr<uint8_t>(), bytes);
  else {
    TORCH_CHECK(sw8.has_value(), "linear_fp8: scales of the kept weight");
    mw = as_matrix(*w8, *sw8, K, x.device(), "linear_fp8");
    TORCH_CHECK(mw.rows == N, "linear_fp8: the kept weight has another shape");
  }
  std::vector<torch::Tensor> out(5);
  if (need_xt) mxt = new_matrix(K, T, false, x, out[1], out[2]);
  if (need_wt && own_w) mwt = new_matrix(K, N, false, x, out[3], out[4]);
  out[0] = torch::empty({T, N}, x.options().dtype(at::kBFloat16));
  quantize_into(x, false, mx, mxt, false, stream);
  if (own_w) quantize_into(w, true, mw, mwt, true, stream);
  gemm_into(mx, mw, out[0], false, status_ptr, stream);
  return out;
}

// Backward of ops.linear_fp8: {dx, dw} (undefined where not asked for; dw goes into acc when that is given).
std::vector<torch::Tensor> linear_fp8_bwd(const torch::Tensor& dy, const c10::optional<torch::Tensor>& xt,
                                          const c10::optional<torch::Tensor>& sxt,
                                          const c10::optional<torch::Tensor>& wt,
                                          const c10::optional<torch::Tensor>& swt, bool e5m2,
                                          c10::optional<torch::Tensor> acc, int64_t status_ptr) {
  check_input(dy, "linear_fp8");
  const at::cuda::CUDAGuard guard(dy.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int64_t T = dy.size(0), N = dy.size(1);
  const bool need_dw = xt.has_value(), need_dx = wt.has_value();
  TORCH_CHECK((need_dw || need_dx) && need_dw == sxt.has_value() && need_dx == swt.has_value(), "linear_fp8: operands");
  Matrix mxt, mwt, md, mdt;
  if (need_dw) mxt = as_matrix(*xt, *sxt, T, dy.device(), "linear_fp8");
  if (need_dx) mwt = as_matrix(*wt, *swt, N, dy.device(), "linear_fp8");
  int64_t bytes = 0;
  if (need_dx) place(md, T, N, e5m2, nullptr, bytes);
  if (need_dw) place(mdt, N, T, e5m2, nullptr, bytes);
  auto buf = torch::empty({bytes}, dy.options().dtype(at::kByte));
  bytes = 0;
  if (need_dx) place(md, T, N, e5m2, buf.data_ptr<uint8_t>(), bytes);
  if (need_dw) place(mdt, N, T, e5m2, buf.data_ptr<uint8_t>(), bytes);
  std::vector<torch::Tensor> out(2);
  if (need_dx) out[0] = torch::empty({T, mwt.rows}, dy.options().dtype(at::kBFloat16));
  if (need_dw && !acc.has_value()) out[1] = torch::empty({N, mxt.rows}, dy.options().dtype(at::kBFloat16));
  if (need_dw && acc.has_value())
    TORCH_CHECK(acc->device() == dy.device() && acc->scalar_type() == at::kFloat,
                "linear_fp8: fp32 accumulator on the gradient's device");
  quantize_into(dy, false, md, mdt, false, stream);
  if (need_dx) gemm_into(md, mwt, out[0], false, status_ptr, stream);
  if (need_dw) gemm_into(mdt, mxt, acc.has_value() ? *acc : out[1], acc.has_value(), status_ptr, stream);
  return out;
}
