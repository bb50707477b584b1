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
// along the former rows), or both.  It is bound by memory: 2 bytes read and 1 or 2 written per bf16 value.
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
// amax = 1.m 2^(E-127); MAX = 1.75 2^p, so e = E - 127 - p, one more if 1.m > 1.75.
template <bool E5M2>
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
  const int E = static_cast<int>(amax_bits >> 23);
  if (E == 255) return -1;
  constexpr int p = E5M2 ? 15 : 8;
  return max(0, E - p + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0));
}
// 2^-e for scale byte b (b <= 247, so the exponent field stays in 7..254).
__device__ __forceinline__ float inverse_scale(int b) { return __uint_as_float(static_cast<uint32_t>(254 - b) << 23); }

// NaN codes in the first n of 8 places, zeros behind.
__device__ __forceinline__ uint2 nan_codes(int n) {
  return make_uint2(n >= 4 ? 0x7F7F7F7Fu : n <= 0 ? 0u : 0x7F7F7F7Fu >> (8 * (4 - n)),
                    n >= 8 ? 0x7F7F7F7Fu : n <= 4 ? 0u : 0x7F7F7F7Fu >> (8 * (8 - n)));
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
  const int tile_r = blockIdx.x / p.tile_cols, tile_c = blockIdx.x - tile_r * p.tile_cols;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int l = threadIdx.x % 16, g = threadIdx.x / 16;
  const int r0 = tile_r * BLOCK + g * 8, c0 = tile_c * BLOCK + l * 8;
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
      uint2 out;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = codes2<E5M2>(__uint_as_float(v[i].bits(2 * j)) * f, __uint_as_float(v[i].bits(2 * j + 1)) * f);
      out = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
      if (row_b[i] < 0) out = nan_codes(p.cols - c0);
      if (r0 + i < p.rows) *reinterpret_cast<uint2*>(p.q + (r0 + i) * ldq + c0) = out;
      if (l == 0) {
        const int rr = g * 8 + i;
        uint8_t* a = atom + (rr % 32) * 16 + (rr / 32) * 4;
        a[tile_c % 4] = r0 + i < p.rows ? static_cast<uint8_t>(row_b[i] < 0 ? 127 : row_b[i]) : 0;
        if (tile_c == p.tile_cols - 1)  // blocks the atom has beyond the matrix
          for (int b = tile_c % 4 + 1; b < 4; ++b) a[b] = 0;
      }
    }
  }
  if (p.qt != nullptr) {
    const int groups = (row_blocks + 3) / 4;
    const float4 inv0 = *reinterpret_cast<const float4*>(col_inv + l * 8);
    const float4 inv1 = *reinterpret_cast<const float4*>(col_inv + l * 8 + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = j == 0 ? inv0.x : j == 1 ? inv0.y : j == 2 ? inv0.z : j == 3 ? inv0.w
                    : j == 4 ? inv1.x : j == 5 ? inv1.y : j == 6 ? inv1.z : inv1.w;
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = codes2<E5M2>(__uint_as_float(v[2 * i].bits(j)) * f, __uint_as_float(v[2 * i + 1].bits(j)) * f);
      uint2 out = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
      if (f == 0.f) out = nan_codes(p.rows - r0);
      *reinterpret_cast<uint2*>(turned + (l * 8 + j) * BLOCK + (g ^ l) * 8) = out;
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
}

template <typename T>
void quantize(const QuantParams& p, bool e5m2, bool tile, int ctas, cudaStream_t stream) {
  if (tile) {
    if (e5m2) quantize_kernel<T, true, true><<<ctas, QT, 0, stream>>>(p);
    else quantize_kernel<T, false, true><<<ctas, QT, 0, stream>>>(p);
  } else {
    if (e5m2) quantize_kernel<T, true, false><<<ctas, QT, 0, stream>>>(p);
    else quantize_kernel<T, false, false><<<ctas, QT, 0, stream>>>(p);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace fp8

// ------------------------------------------------------------------------------------------------ product
//   C[M, N] (+)= A[M, K] B[N, K]^T of two such matrices, fp32 accumulation
//
// The pair-of-SMs GEMM (roles as in gemm2sm_sm100.cu) with tcgen05.mma kind::mxf8f6f4.block_scale: per 128-deep
// k-block each CTA loads 128 rows of A and of B (16 KB each) and every fourth k-block three scale atoms (its 128 rows
// of A; all 256 rows of B, which both SMs of a pair need), which tcgen05.cp moves to tensor memory; the
// k-block's byte of a scale word is picked by the instruction descriptor.
// Tensor memory: two 256-column accumulators at columns 0 and 192 share 64 columns, because the last 64 hold four
// sets of scales (16 columns each).  The epilogue reads the shared columns of a tile first and hands them back at
// once, so the next tile's MMAs wait only for that.  A set is reused four groups (16 k-blocks) later; the ring has 6
// stages, so a full stage there means that the group's MMAs are done, and a tile starts only after the last one's.
namespace fp8gemm {

using namespace gemm2;
using fp8::ATOM;

constexpr int BK = 128;
constexpr int TILE = 256;
constexpr int HALF = 128;
constexpr int STAGES = 6;
constexpr int OP_BYTES = HALF * BK;
constexpr int SF_BYTES = 3 * ATOM;
constexpr int STAGE_BYTES = 2 * OP_BYTES;
constexpr int TMEM_COLS = 512;
constexpr int ACC1_COL = 192;  // accumulator 0: columns 0..255, accumulator 1: 192..447
constexpr int SF_COL = 448;
constexpr int THREADS = 192;
constexpr int SMEM_BYTES = STAGES * (STAGE_BYTES + SF_BYTES) + 1024 + 256;

enum Epilogue : int { kStoreBf16 = 0, kStoreF32 = 1, kAccumF32 = 2 };

struct Params {
  int M, N;
  int num_kb;   // 128-deep k-blocks
  int sf_groups;  // scale atoms per 128 rows
  void* C;
  int64_t ldc;
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
inline uint32_t make_idesc(bool a_e5m2, bool b_e5m2) {
  return ((a_e5m2 ? 1u : 0u) << 7) | ((b_e5m2 ? 1u : 0u) << 10) | ((static_cast<uint32_t>(TILE) >> 3) << 17) |
         (1u << 23) | ((static_cast<uint32_t>(TILE) >> 4) << 24);
}

__device__ __forceinline__ void tile_coords(const Params& p, int t, int& tm, int& tn) {
  constexpr int kGroup = 8;
  const int num_m = (p.M + TILE - 1) / TILE, num_n = (p.N + TILE - 1) / TILE;
  const int per_group = kGroup * num_n;
  const int g = t / per_group, first = g * kGroup;
  const int gm = min(kGroup, num_m - first);
  const int r = t - g * per_group;
  tm = first + r % gm;
  tn = r / gm;
}

template <int EPI>
__device__ __forceinline__ void store_chunk(const Params& p, int m, int n, const uint32_t (&r)[32]) {
  if (m >= p.M || n >= p.N) return;
  const bool full = n + 32 <= p.N;
  if constexpr (EPI == kStoreBf16) {
    __nv_bfloat16* C = static_cast<__nv_bfloat16*>(p.C) + static_cast<int64_t>(m) * p.ldc + n;
    if (full && (reinterpret_cast<uintptr_t>(C) & 15) == 0) {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        reinterpret_cast<uint4*>(C)[v] =
            make_uint4(pack_bf16x2(__uint_as_float(r[8 * v]), __uint_as_float(r[8 * v + 1])),
                       pack_bf16x2(__uint_as_float(r[8 * v + 2]), __uint_as_float(r[8 * v + 3])),
                       pack_bf16x2(__uint_as_float(r[8 * v + 4]), __uint_as_float(r[8 * v + 5])),
                       pack_bf16x2(__uint_as_float(r[8 * v + 6]), __uint_as_float(r[8 * v + 7])));
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (n + j < p.N) C[j] = __float2bfloat16_rn(__uint_as_float(r[j]));
    }
  } else {
    float* C = static_cast<float*>(p.C) + static_cast<int64_t>(m) * p.ldc + n;
    if (full && (reinterpret_cast<uintptr_t>(C) & 15) == 0) {
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        float4 q = make_float4(__uint_as_float(r[4 * v]), __uint_as_float(r[4 * v + 1]), __uint_as_float(r[4 * v + 2]),
                               __uint_as_float(r[4 * v + 3]));
        if constexpr (EPI == kAccumF32) {
          const float4 o = reinterpret_cast<const float4*>(C)[v];
          q.x += o.x;
          q.y += o.y;
          q.z += o.z;
          q.w += o.w;
        }
        reinterpret_cast<float4*>(C)[v] = q;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (n + j < p.N) C[j] = __uint_as_float(r[j]) + (EPI == kAccumF32 ? C[j] : 0.f);
    }
  }
}

template <int EPI>
__global__ void __launch_bounds__(THREADS, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * OP_BYTES;
  uint8_t* sS = smem + STAGES * STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sS + STAGES * SF_BYTES);  // used in the leader
  uint64_t* empty_bar = full_bar + STAGES;                                   // both CTAs
  uint64_t* tfull_bar = empty_bar + STAGES;                                  // [2] both CTAs
  uint64_t* handed_bar = tfull_bar + 2;                                      // used in the leader: shared columns read
  uint64_t* done_bar = handed_bar + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const uint32_t crank = cluster_ctarank();  // 0 = leader
  const int cluster_id = blockIdx.x >> 1;
  const int clusters = gridDim.x >> 1;
  const int total = ((p.M + TILE - 1) / TILE) * ((p.N + TILE - 1) / TILE);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) mbar_init(&tfull_bar[a], 1);
    mbar_init(handed_bar, 2 * 128);  // epilogue threads of both CTAs
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

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (elect_one_sync()) {
      const uint32_t leader_full0 = mapa_shared(smem_u32(&full_bar[0]), 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, issued = false;
      for (int t = cluster_id; ok && t < total; t += clusters) {
        int tm, tn;
        tile_coords(p, t, tm, tn);
        const int m0 = tm * TILE + crank * HALF, n0 = tn * TILE + crank * HALF;
        const int sa = (tm * 2 + static_cast<int>(crank)) * p.sf_groups, sb = tn * 2 * p.sf_groups;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, abort_flag, p.status, kTimeoutProducer)) {
            ok = false;
            break;
          }
          const bool scales = (kb & 3) == 0;
          if (crank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * (STAGE_BYTES + (scales ? SF_BYTES : 0)));
          issued = true;
          const uint32_t bar = leader_full0 + stage * 8;
          tma_load_2d_pair(sA + stage * OP_BYTES, &tmA, bar, kb * BK, m0);
          tma_load_2d_pair(sB + stage * OP_BYTES, &tmB, bar, kb * BK, n0);
          if (scales) {
            uint8_t* dst = sS + stage * SF_BYTES;
            tma_load_2d_pair(dst, &tmSA, bar, 0, sa + kb / 4);
            tma_load_2d_pair(dst + ATOM, &tmSB, bar, 0, sb + kb / 4);
            tma_load_2d_pair(dst + 2 * ATOM, &tmSB, bar, 0, sb + p.sf_groups + kb / 4);
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
        // the columns this tile shares with the one before have been read (completion number `local`)
        if (local > 0 &&
            !mbar_wait_bounded(handed_bar, (local - 1) & 1, abort_flag, p.status, kTimeoutMma))
          break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (local & 1) * ACC1_COL;
        uint32_t sf = 0;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait_bounded(&full_bar[stage], phase, abort_flag, p.status, kTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if ((kb & 3) == 0) {
            sf = tmem_base + SF_COL + (group++ & 3) * 16;
            const uint32_t src = smem_u32(sS + stage * SF_BYTES);
            scales_to_tmem(sf, src);
            scales_to_tmem(sf + 8, src + ATOM);
            scales_to_tmem(sf + 12, src + 2 * ATOM);
          }
          const uint32_t idesc = p.idesc | (static_cast<uint32_t>(kb & 3) << 29) | (static_cast<uint32_t>(kb & 3) << 4);
          const uint32_t a_base = smem_u32(sA + stage * OP_BYTES);
          const uint32_t b_base = smem_u32(sB + stage * OP_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_scaled_pair(d_tmem, make_smem_desc_sw128(a_base + k * 32, 16, 1024),
                            make_smem_desc_sw128(b_base + k * 32, 16, 1024), idesc, sf, sf + 8,
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
    const int sub = warp & 3;
    const int row_in_tile = crank * HALF + sub * 32 + lane;
    const uint32_t leader_handed = mapa_shared(smem_u32(handed_bar), 0);
    const uint32_t lanes = static_cast<uint32_t>(sub * 32) << 16;
    int local = 0;
    for (int t = cluster_id; t < total; t += clusters, ++local) {
      int tm, tn;
      tile_coords(p, t, tm, tn);
      const int acc = local & 1;
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tfull_bar[acc], (local >> 1) & 1, abort_flag, p.status,
                                                     kTimeoutEpilogue)))
        break;
      tc_fence_after();
      const int m = tm * TILE + row_in_tile;
      const uint32_t base = tmem_base + lanes + acc * ACC1_COL;
      // columns shared with the other accumulator: the last 64 of accumulator 0, the first 64 of accumulator 1
      const int c_first = acc == 0 ? 6 : 0;
      {
        uint32_t r0[32], r1[32];
        tmem_ld_32x32b_x32(base + c_first * 32, r0);
        tmem_ld_32x32b_x32(base + c_first * 32 + 32, r1);
        tmem_wait_ld();
        tc_fence_before();
        remote_arrive(leader_handed);
        store_chunk<EPI>(p, m, tn * TILE + c_first * 32, r0);
        store_chunk<EPI>(p, m, tn * TILE + c_first * 32 + 32, r1);
      }
#pragma unroll 1
      for (int i = 0; i < 6; ++i) {
        const int c = acc == 0 ? i : i + 2;
        uint32_t r[32];
        tmem_ld_32x32b_x32(base + c * 32, r);
        tmem_wait_ld();
        store_chunk<EPI>(p, m, tn * TILE + c * 32, r);
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

template <int EPI>
void launch(const CUtensorMap (&t)[4], const Params& p, int sms, cudaStream_t stream) {
  auto kern = fp8_gemm_kernel<EPI>;
  static std::atomic<uint64_t> configured{0};
  allow_smem(kern, SMEM_BYTES, configured);
  const int64_t tiles = static_cast<int64_t>((p.M + TILE - 1) / TILE) * ((p.N + TILE - 1) / TILE);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min<int64_t>(tiles, std::max(1, sms / 2))));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, t[0], t[1], t[2], t[3], p));
}

}  // namespace fp8gemm
}  // namespace mvp

static bool is_e5m2(const torch::Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kFloat8_e5m2, what,
              ": codes are float8_e4m3fn or float8_e5m2");
  return t.scalar_type() == at::kFloat8_e5m2;
}

// Codes and scale atoms of x's rows (q, s) and / or columns (qt, st); tile: 128 x 128 blocks instead of 1 x 128.
void quantize_fp8(const torch::Tensor& x, bool tile, const c10::optional<torch::Tensor>& q,
                  const c10::optional<torch::Tensor>& s, const c10::optional<torch::Tensor>& qt,
                  const c10::optional<torch::Tensor>& st) {
  using namespace mvp::fp8;
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(0) > 0 && x.size(1) > 0 && (x.stride(1) == 1 || x.size(1) == 1),
              "quantize_fp8: CUDA matrix with unit column stride");
  TORCH_CHECK(x.size(0) < (int64_t(1) << 31) - 256 && x.size(1) < (int64_t(1) << 31) - 256, "quantize_fp8: sizes");
  const int64_t rb = (x.size(0) + BLOCK - 1) / BLOCK, cb = (x.size(1) + BLOCK - 1) / BLOCK;
  TORCH_CHECK(rb * cb < (int64_t(1) << 31), "quantize_fp8: too many blocks");
  bool e5m2 = false;
  auto check = [&](const c10::optional<torch::Tensor>& d, const c10::optional<torch::Tensor>& a, int64_t rows,
                   int64_t blocks, int64_t row_blocks) {
    if (!d.has_value()) return;
    e5m2 = is_e5m2(*d, "quantize_fp8");
    TORCH_CHECK(d->device() == x.device() && d->is_contiguous() && d->dim() == 2 && d->size(0) == rows &&
                    d->size(1) == blocks * BLOCK && a.has_value() && a->device() == x.device() && a->is_contiguous() &&
                    a->scalar_type() == at::kByte && a->numel() == row_blocks * ((blocks + 3) / 4) * ATOM,
                "quantize_fp8: outputs");
  };
  check(q, s, x.size(0), cb, rb);
  check(qt, st, x.size(1), rb, cb);
  TORCH_CHECK(q.has_value() || qt.has_value(), "quantize_fp8: nothing to write");
  TORCH_CHECK(!q.has_value() || !qt.has_value() || q->scalar_type() == qt->scalar_type(), "quantize_fp8: one type");
  const at::cuda::CUDAGuard guard(x.device());
  QuantParams p{};
  p.x = x.data_ptr();
  p.ld = x.stride(0);
  p.rows = static_cast<int>(x.size(0));
  p.cols = static_cast<int>(x.size(1));
  p.tile_cols = static_cast<int>(cb);
  p.vec = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && (p.ld * x.element_size()) % 16 == 0;
  if (q.has_value()) {
    p.q = static_cast<uint8_t*>(q->data_ptr());
    p.s = s->data_ptr<uint8_t>();
  }
  if (qt.has_value()) {
    p.qt = static_cast<uint8_t*>(qt->data_ptr());
    p.st = st->data_ptr<uint8_t>();
  }
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int ctas = static_cast<int>(rb * cb);
  if (x.scalar_type() == at::kBFloat16) quantize<__nv_bfloat16>(p, e5m2, tile, ctas, stream);
  else if (x.scalar_type() == at::kFloat) quantize<float>(p, e5m2, tile, ctas, stream);
  else TORCH_CHECK(false, "quantize_fp8: bf16 or fp32 input");
}

// c (+)= a b^T of quantised matrices: a [M, K'], b [N, K'] codes with their scale atoms.
void gemm_fp8(const torch::Tensor& a, const torch::Tensor& sa, const torch::Tensor& b, const torch::Tensor& sb,
              torch::Tensor& c, bool accumulate, int64_t status_ptr) {
  using namespace mvp::fp8gemm;
  const bool a5 = is_e5m2(a, "gemm_fp8"), b5 = is_e5m2(b, "gemm_fp8");
  TORCH_CHECK(a.is_cuda() && a.dim() == 2 && b.dim() == 2 && a.is_contiguous() && b.is_contiguous() &&
                  a.size(1) == b.size(1) && a.size(1) % BK == 0 && a.size(0) > 0 && b.size(0) > 0 && a.size(1) > 0,
              "gemm_fp8: contiguous codes with the same whole blocks of 128");
  TORCH_CHECK(a.size(0) < (int64_t(1) << 31) - 512 && b.size(0) < (int64_t(1) << 31) - 512 &&
                  a.size(1) < (int64_t(1) << 31) - 512,
              "gemm_fp8: sizes");
  const int64_t kb = a.size(1) / BK, groups = (kb + 3) / 4;
  const int64_t ra = (a.size(0) + HALF - 1) / HALF, rb = (b.size(0) + HALF - 1) / HALF;
  TORCH_CHECK((ra + 2) * groups < (int64_t(1) << 31) && (rb + 2) * groups < (int64_t(1) << 31) &&
                  ((ra + 1) / 2) * ((rb + 1) / 2) < (int64_t(1) << 31) - 1024,
              "gemm_fp8: sizes");
  auto scales = [&](const torch::Tensor& s, int64_t blocks) {
    TORCH_CHECK(s.device() == a.device() && s.scalar_type() == at::kByte && s.is_contiguous() &&
                    s.numel() == blocks * groups * ATOM,
                "gemm_fp8: scale bytes");
  };
  scales(sa, ra);
  scales(sb, rb);
  TORCH_CHECK(b.device() == a.device() && c.device() == a.device() && c.dim() == 2 && c.size(0) == a.size(0) &&
                  c.size(1) == b.size(0) && (c.stride(1) == 1 || c.size(1) == 1) &&
                  (c.size(0) == 1 || c.stride(0) >= c.size(1)),
              "gemm_fp8: output [M, N] with unit column stride on the operands' device");
  TORCH_CHECK(c.scalar_type() == at::kFloat || (c.scalar_type() == at::kBFloat16 && !accumulate),
              "gemm_fp8: bf16 or fp32 output, fp32 to accumulate");
  for (const torch::Tensor* t : {&a, &b, &sa, &sb})
    TORCH_CHECK((reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0, "gemm_fp8: 16-byte aligned operands");
  const at::cuda::CUDAGuard guard(a.device());
  CUtensorMap t[4];
  const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  encode(&t[0], u8, a.data_ptr(), a.size(1), a.size(0), a.size(1), BK, HALF, CU_TENSOR_MAP_SWIZZLE_128B);
  encode(&t[1], u8, b.data_ptr(), b.size(1), b.size(0), b.size(1), BK, HALF, CU_TENSOR_MAP_SWIZZLE_128B);
  const auto u32 = CU_TENSOR_MAP_DATA_TYPE_UINT32;
  encode(&t[2], u32, sa.data_ptr(), ATOM / 4, ra * groups, ATOM, ATOM / 4, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
  encode(&t[3], u32, sb.data_ptr(), ATOM / 4, rb * groups, ATOM, ATOM / 4, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
  Params p{};
  p.M = static_cast<int>(a.size(0));
  p.N = static_cast<int>(b.size(0));
  p.num_kb = static_cast<int>(kb);
  p.sf_groups = static_cast<int>(groups);
  p.C = c.data_ptr();
  p.ldc = c.stride(0);
  p.idesc = make_idesc(a5, b5);
  p.status = reinterpret_cast<int*>(status_ptr);
  const int sms = mvp::num_sms(a.get_device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (c.scalar_type() == at::kBFloat16) launch<kStoreBf16>(t, p, sms, stream);
  else if (!accumulate) launch<kStoreF32>(t, p, sms, stream);
  else launch<kAccumF32>(t, p, sms, stream);
}
