// Orthogonalisation of update matrices by Newton-Schulz products, and the optimizer step built on it.
//
//   X <- u / max(|u|_F, eps)
//   repeat `steps` times, over the short side s = min(m, n):
//     A = X X^T (m <= n) or X^T X (m > n)          [s, s], symmetric
//     B = b A + c A A                              [s, s], symmetric
//     X <- a X + B X (or a X + X B)                [m, n]
//   O = X;   step: p <- p (1 - lr wd) - lr adj O
//
// Numbers.  The products run on the tensor core in fp16 with fp32 accumulation.  Rounding X to 16 bits would
// put white noise of relative size r into every singular direction, and the linear term multiplies what lies in
// the weak ones by a = 3.44 per iteration, 485 times in five: for a matrix with a fast decaying spectrum bf16
// (r = 2^-9 on average) ends 10 to 20 % off and fp16 1 to 3 %.  So the linear term a X is exact to 22 bits: X is kept as
// the sum of two fp16 values (hi + lo), the epilogue adds a (hi + lo) to the fp32 accumulator, and only hi goes
// into the products, whose part of the result is small while a weak direction is.  All spectra tried then end
// within 1.5e-3 of 64-bit arithmetic before the final rounding.  A matrix with |u|_F below eps starts with entries of X that much
// below 1, down among fp16's subnormal values, whose step is 2^-24: sqrt(2) 2^-25 of |X|_F = 1 is lost in each X, at most 3e-5 of
// the result in five steps (a + a^2 + .. + a^5 times it), which is 0.3 % of a result that began at 2e-5 eps.
// fp16's range is met by fixed powers of two: |X|_F <= 1 at the start makes the mean square of X sigma = 2^k,
// k = round(log2(m n) / 2), equal to about 1, and A, B (trace <= 1 at first) are stored times tau = 2^round(log2 s).
// A and B are close to multiples of the identity once X is nearly orthogonal, so their diagonals are kept in fp32 and
// only what is off them is rounded to fp16: with A = D + A~, A A = A~ A~ + (D_i + D_j) A~ + D^2 element by element, and
// B's diagonal joins the linear term, (a + B_ii) (hi + lo).  That halves the error of well conditioned matrices
// (simulated against 64 bits at 512 x 2048: 1.7e-3 -> 0.5e-3) and bounds it for tiny ones.
// A result that keeps more than 16 bits (the fp32 step or output) shows more of that error, small matrices most, whose roundings
// average less.  There X's low part enters the products as well, (hi + lo)(hi + lo)^T without lo lo^T and B (hi + lo), as more
// passes over the reduction (Shape::split), and A and B off their diagonals are kept as hi + lo too (Shape::split_s).
// Entries then stay below 1.9 sigma and 3.9 tau (the caller checks the coefficients for it), within 65504, and
// what underflows is 2^-24 of an average entry.
//
// Work.  A and A A are symmetric: only tiles on and below the diagonal are computed, and the epilogue writes a
// tile and its mirror, which makes an iteration s^2 l + s^3 + 2 s^2 l operations instead of 4 s^2 l + 2 s^3.
// One launch per product handles a whole stack of same-shaped matrices.  The kernel is the pair-of-SMs GEMM
// (256 x 256 or 256 x 128 tile per cluster, see gemm2sm_sm100.cu for the roles) over 3-D tensor maps.
// Measured, five iterations: 4 x 4096 x 4096 in 4.5 ms in short runs and 5.1 ms in long ones under the power limit (1.2 and 1.1
// PFLOP/s; the bf16 GEMM settles at 1.4), 12 x 1024 x 4096 in 1.2 ms, bound by what X's update moves through L2 (4 bytes read
// and 4 written per value beside the operands), 1 x 256 x 512 in 104 us, bound by 17 dependent launches.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>

#include "common.cuh"
#include "pair_sm100.cuh"
#include "tma_host.h"

namespace mvp {
namespace muon {

using namespace gemm2;

constexpr int BK = 64;
constexpr int TM = 256;                  // tiles are 256 x TN, TN = 256 or 128 (choose_tile)
constexpr int HALF = 128;
constexpr int STAGES = 5;
constexpr int A_BYTES = HALF * BK * 2;   // per stage and CTA; of B half a tile's columns
template <int TN>
constexpr int kStageBytes = A_BYTES + TN / 2 * BK * 2;
constexpr int CHUNK = 32;                 // columns the epilogue handles at a time
constexpr int HALF_BUF = 32 * CHUNK * 2;  // a warp's 32 rows of a chunk in fp16
constexpr int EPI_BUF = 2 * HALF_BUF;     // hi and lo, or fp32
constexpr int EPI_BYTES = 8 * 2 * EPI_BUF;  // two buffers for each warp
constexpr int TMEM_COLS = 512;
constexpr int EPI_WARPS = 8;             // two for each quarter of the accumulator's lanes, half of the columns each
constexpr int THREADS = 64 + 32 * EPI_WARPS;
template <int TN>
constexpr int kSmemBytes = STAGES * kStageBytes<TN> + EPI_BYTES + 1024 + 256;
constexpr int kMaxStack = 64;  // matrices per launch (their pointers travel as kernel parameters)

// What the epilogue does with the fp32 accumulator `acc` of a tile.
enum Epi : int {
  kGram = 0,   // A: D = alpha acc, tile and mirror of a symmetric product; its diagonal goes to diag, in fp32
  kPoly = 1,   // B: D = alpha acc + (beta + gamma (a_m + a_n)) C with A's diagonal a; as above
  kNext = 2,   // X: D_hi + D_lo = alpha acc + (beta + diag) (C_hi + C_lo)
  kOut = 3,    // out[b] = alpha acc + (beta + diag) (C_hi + C_lo), in the output's type
  kStep = 4,   // p[b] = decay p[b] - rate (alpha acc + (beta + diag) (C_hi + C_lo)), and its bf16 copy
};

struct Outs {
  void* out[kMaxStack];               // kOut: the results; kStep: fp32 master weights
  __nv_bfloat16* shadow[kMaxStack];   // kStep: bf16 copies, or null
};

struct Params {
  int M, N, K, count;   // per matrix: D [M, N], reduction K; matrices in the stack
  int tiles;            // tiles per matrix
  float alpha, beta;
  const __half* C_hi;   // element-wise term, row stride ld, matrix stride ld * M
  const __half* C_lo;
  __half* D_hi;
  __half* D_lo;         // null: A and B have no low parts
  int ld;               // of C and D (a multiple of 8, at least N)
  float* diag;          // [count, ld_s] diagonal of D (kGram, kPoly: written, and zeroed in D) or of B (others: added
  int ld_s;             // to beta, times diag_scale, for row m where X is short by rows, else for column n)
  float diag_scale;
  const float* diag_a;  // kPoly: A's diagonal
  float gamma, tau;
  float decay, rate;
  int passes;           // over the reduction; in pass i an operand is the low part of X where bit i of its mask is set
  uint32_t low_a, low_b;
  int* status;
};

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const void* tmap, uint32_t bar, int c0, int c1,
                                                 int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// Instruction descriptor of kind::f16 with fp16 operands (A and B format 0) and fp32 accumulate.
__host__ __device__ constexpr uint32_t make_idesc_f16(int M, int N, bool a_mn_major, bool b_mn_major) {
  return (1u << 4) | ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) |
         ((static_cast<uint32_t>(N) >> 3) << 17) | ((static_cast<uint32_t>(M) >> 4) << 24);
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Tile t of a matrix: symmetric products take the 256-row blocks on and below the diagonal, row by row (the block on the
// diagonal whole, so that only blocks below it are mirrored), others 8-row groups.
template <bool SYM, int TN>
__device__ __forceinline__ void tile_of(const Params& p, int t, int& tm, int& tn) {
  if constexpr (SYM) {
    constexpr int R = TM / TN;  // tiles per block
    const int block = t / R;
    tm = static_cast<int>((sqrtf(8.f * block + 1.f) - 1.f) * 0.5f);
    while (tm * (tm + 1) / 2 > block) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= block) ++tm;
    tn = (block - tm * (tm + 1) / 2) * R + t % R;
  } else {
    const int num_m = (p.M + TM - 1) / TM, num_n = (p.N + TN - 1) / TN;
    constexpr int kGroup = 8;
    const int per_group = kGroup * num_n;
    const int g = t / per_group, first = g * kGroup;
    const int gm = min(kGroup, num_m - first);
    const int r = t - g * per_group;
    tm = first + r % gm;
    tn = r / gm;
  }
}

__device__ __forceinline__ float2 h2f(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ uint32_t f2h(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// LOW: C and D have low parts (always so for X; for A and B where Shape::split_s is set).
template <bool A_MN, bool B_MN, int EPI, typename OUT, int TN, bool LOW>
__global__ void __launch_bounds__(THREADS, 1)
    ns_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                      const __grid_constant__ CUtensorMap tmA_low, const __grid_constant__ CUtensorMap tmB_low,
                      const Params p, const __grid_constant__ Outs outs) {
  constexpr bool SYM = EPI == kGram || EPI == kPoly;
  static_assert(SYM || LOW, "X has a low part");
  constexpr int B_BYTES = kStageBytes<TN> - A_BYTES;
  constexpr int CHUNKS = TN / 2 / CHUNK;  // per epilogue warp and tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint8_t* sE = smem + STAGES * kStageBytes<TN>;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sE + EPI_BYTES);               // used in the leader
  uint64_t* empty_bar = full_bar + STAGES;                                        // both CTAs
  uint64_t* tfull_bar = empty_bar + STAGES;                                       // [2] both CTAs
  uint64_t* tempty_bar = tfull_bar + 2;                                           // [2] used in the leader
  uint64_t* done_bar = tempty_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const uint32_t crank = cluster_ctarank();  // 0 = leader
  const int cluster_id = blockIdx.x >> 1;
  const int clusters = gridDim.x >> 1;
  const int num_kb = (p.K + BK - 1) / BK;
  const int total = p.tiles * p.count;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 2 * 32 * EPI_WARPS);  // epilogue threads of both CTAs
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
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
  pdl_wait();  // every thread: what follows reads the product before this one, and writes what it may still read

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (elect_one_sync()) {
      const uint32_t leader_full0 = mapa_shared(smem_u32(&full_bar[0]), 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, issued = false;
      for (int t = cluster_id; ok && t < total; t += clusters) {
        const int b = t / p.tiles;
        int tm, tn;
        tile_of<SYM, TN>(p, t - b * p.tiles, tm, tn);
        const int m0 = tm * TM + crank * HALF, n0 = tn * TN + crank * (TN / 2);
        for (int i = 0; i < num_kb * p.passes; ++i) {
          const int pass = i / num_kb, kb = i - pass * num_kb;
          const CUtensorMap* ta = (p.low_a >> pass) & 1u ? &tmA_low : &tmA;
          const CUtensorMap* tb = (p.low_b >> pass) & 1u ? &tmB_low : &tmB;
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, abort_flag, p.status, kTimeoutProducer)) {
            ok = false;
            break;
          }
          if (crank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * kStageBytes<TN>);
          issued = true;
          const uint32_t bar = leader_full0 + stage * 8;
          uint8_t* a_dst = sA + stage * A_BYTES;
          uint8_t* b_dst = sB + stage * B_BYTES;
          const int k0 = kb * BK;
          if constexpr (!A_MN) {
            tma_load_3d_pair(a_dst, ta, bar, k0, m0, b);
          } else {
            tma_load_3d_pair(a_dst, ta, bar, m0, k0, b);
            tma_load_3d_pair(a_dst + 64 * BK * 2, ta, bar, m0 + 64, k0, b);
          }
          if constexpr (!B_MN) {
            tma_load_3d_pair(b_dst, tb, bar, k0, n0, b);
          } else {
            tma_load_3d_pair(b_dst, tb, bar, n0, k0, b);
            if constexpr (TN == 256) tma_load_3d_pair(b_dst + 64 * BK * 2, tb, bar, n0 + 64, k0, b);
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
      constexpr uint32_t idesc = make_idesc_f16(TM, TN, A_MN, B_MN);
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int t = cluster_id; ok && t < total; t += clusters, ++local) {
        const int acc = local & 1;
        const uint32_t acc_phase = (local >> 1) & 1;
        if (!mbar_wait_bounded(&tempty_bar[acc], acc_phase ^ 1, abort_flag, p.status, kTimeoutMma)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * TN;
        for (int kb = 0; kb < num_kb * p.passes; ++kb) {
          if (!mbar_wait_bounded(&full_bar[stage], phase, abort_flag, p.status, kTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_base = smem_u32(sA + stage * A_BYTES);
          const uint32_t b_base = smem_u32(sB + stage * B_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            uint64_t adesc, bdesc;
            if constexpr (!A_MN) adesc = make_smem_desc_sw128(a_base + k * 32, 16, 1024);
            else adesc = make_smem_desc_sw128(a_base + k * 2048, 64 * BK * 2, 1024);
            if constexpr (!B_MN) bdesc = make_smem_desc_sw128(b_base + k * 32, 16, 1024);
            else bdesc = make_smem_desc_sw128(b_base + k * 2048, 64 * BK * 2, 1024);
            mma_pair(d_tmem, adesc, bdesc, idesc, (kb != 0 || k != 0) ? 1u : 0u);
          }
          mma_commit_pair(&empty_bar[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit_pair(&tfull_bar[acc]);
      }
      mma_commit_pair_local(done_bar);
      mbar_wait_bounded(done_bar, 0, abort_flag, p.status, kTimeoutDrain);
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    // A warp takes its 32 rows in chunks of 32 columns.  tcgen05.ld gives a lane one row; global memory wants rows of
    // consecutive lanes.  So both directions pass through a warp's own shared-memory buffer, in 16-byte pieces swizzled
    // by row: the element-wise terms arrive by cp.async two chunks ahead (the first during the tile's MMAs), a lane
    // combines its row, and 4 (fp16) or 8 (fp32) lanes write each row.
    const int sub = warp & 3, ew = warp - 2;
    uint8_t* const bufs = sE + ew * 2 * EPI_BUF;
    const uint32_t leader_tempty0 = mapa_shared(smem_u32(&tempty_bar[0]), 0);
    const int row_in_tile = static_cast<int>(crank) * HALF + sub * 32;
    const int col_in_tile = (ew / 4) * (TN / 2);
    // byte offset of 16-byte piece j of row r: 64-byte rows (fp16) and 128-byte rows (fp32), both free of conflicts for
    // lanes that read or write the same piece of 8 rows
    auto piece16 = [](int r, int j) { return r * 64 + ((j ^ ((r >> 1) & 3)) << 4); };
    auto piece32 = [](int r, int j) { return r * 128 + ((j ^ (r & 7)) << 4); };
    auto fetch = [&](int seq) {  // element-wise terms of chunk `seq` of this warp's sequence
      if constexpr (EPI != kGram) {
        const int t = cluster_id + (seq / CHUNKS) * clusters;
        if (t < total) {
          const int b = t / p.tiles;
          int tm, tn;
          tile_of<SYM, TN>(p, t - b * p.tiles, tm, tn);
          const int n = tn * TN + col_in_tile + (seq % CHUNKS) * CHUNK + (lane & 3) * 8;
          const int64_t mat = static_cast<int64_t>(b) * p.M * p.ld;
          const uint32_t dst = smem_u32(bufs + (seq & 1) * EPI_BUF);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + lane / 4, m = tm * TM + row_in_tile + r;
            const bool ok = m < p.M && n < p.ld;  // the columns between N and ld are never used
            const int64_t at = ok ? mat + static_cast<int64_t>(m) * p.ld + n : 0;
            const uint32_t d = dst + piece16(r, lane & 3);
            cp_async_16(d, p.C_hi + at, ok ? 16 : 0);
            if constexpr (LOW) cp_async_16(d + HALF_BUF, p.C_lo + at, ok ? 16 : 0);
          }
        }
        cp_async_commit();
      }
    };
    fetch(0);
    fetch(1);
    int local = 0;
    for (int t = cluster_id; t < total; t += clusters, ++local) {
      const int b = t / p.tiles;
      int tm, tn;
      tile_of<SYM, TN>(p, t - b * p.tiles, tm, tn);
      const int acc = local & 1;
      const int m_warp = tm * TM + row_in_tile;  // the warp's first row
      const int m = m_warp + lane;
      const bool row_ok = m < p.M;
      const int64_t mat = static_cast<int64_t>(b) * p.M * p.ld;
      constexpr bool kDiagByColumn = !SYM && !B_MN;  // X B: the diagonal belongs to X's columns
      constexpr bool kByColumn = kDiagByColumn || EPI == kPoly;
      const float* col_term = EPI == kPoly ? p.diag_a : p.diag;
      const float col_scale = EPI == kPoly ? p.gamma : p.diag_scale;
      float beta = p.beta, a_row = 0.f;
      if constexpr (!SYM && !kDiagByColumn)
        if (row_ok) beta += p.diag_scale * p.diag[static_cast<int64_t>(b) * p.ld_s + m];
      if constexpr (EPI == kPoly) {
        if (row_ok) a_row = p.diag_a[static_cast<int64_t>(b) * p.ld_s + m];
        beta += p.gamma * a_row;
      }
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tfull_bar[acc], (local >> 1) & 1, abort_flag, p.status,
                                                     kTimeoutEpilogue)))
        break;
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < CHUNKS; ++c) {
        const int seq = local * CHUNKS + c;
        const int n = tn * TN + col_in_tile + c * CHUNK;
        uint8_t* const buf = bufs + (seq & 1) * EPI_BUF;
        const bool live = n < p.N && m_warp < p.M;  // same for all lanes
        float x[CHUNK];
        if (live) {
          uint32_t r[CHUNK];
          tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(sub * 32) << 16) + acc * TN + col_in_tile + c * CHUNK,
                             r);
          if constexpr (EPI != kGram) {
            float by_col = 0.f;  // lane j: what column n + j adds to beta
            if constexpr (kByColumn)
              if (n + lane < p.N) by_col = col_scale * col_term[static_cast<int64_t>(b) * p.ld_s + n + lane];
            cp_async_wait_but_one();
            __syncwarp();
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const uint8_t* at = buf + piece16(lane, v);
              const uint4 hi = *reinterpret_cast<const uint4*>(at);
              uint4 lo = make_uint4(0u, 0u, 0u, 0u);
              if constexpr (LOW) lo = *reinterpret_cast<const uint4*>(at + HALF_BUF);
              const uint32_t* hw = &hi.x;
              const uint32_t* lw = &lo.x;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float2 e = h2f(hw[q]);
                if constexpr (LOW) {
                  const float2 f = h2f(lw[q]);
                  e.x += f.x;
                  e.y += f.y;
                }
                const int j = 8 * v + 2 * q;
                x[j] = (kByColumn ? beta + __shfl_sync(0xffffffffu, by_col, j) : beta) * e.x;
                x[j + 1] = (kByColumn ? beta + __shfl_sync(0xffffffffu, by_col, j + 1) : beta) * e.y;
              }
            }
            __syncwarp();  // all rows of the buffer have been read
          }
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < CHUNK; ++j)
            x[j] = EPI == kGram ? p.alpha * __uint_as_float(r[j]) : fmaf(p.alpha, __uint_as_float(r[j]), x[j]);
        }
        if (c == CHUNKS - 1) {  // the accumulator has been read
          tc_fence_before();
          remote_arrive_relaxed(leader_tempty0 + acc * 8);
        }
        if (live) {
          if constexpr (SYM) {
            if (n == m_warp) {  // the chunk on the diagonal: element j of lane j
              float d = 0.f;
#pragma unroll
              for (int j = 0; j < CHUNK; ++j)
                if (j == lane) {
                  d = x[j];
                  x[j] = 0.f;
                }
              // tau times the diagonal element: A's comes out of the sum, B's adds b a + c a^2 (C is zero there)
              if constexpr (EPI == kPoly) d = fmaf(p.tau * a_row, p.beta + p.gamma * a_row, d);
              if (row_ok) p.diag[static_cast<int64_t>(b) * p.ld_s + m] = d / p.tau;
            }
          }
          if constexpr (SYM || EPI == kNext) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t h[4], l[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float u0 = x[8 * v + 2 * q], u1 = x[8 * v + 2 * q + 1];
                h[q] = f2h(u0, u1);
                const float2 back = h2f(h[q]);
                l[q] = f2h(u0 - back.x, u1 - back.y);
              }
              uint8_t* at = buf + piece16(lane, v);
              *reinterpret_cast<uint4*>(at) = make_uint4(h[0], h[1], h[2], h[3]);
              if constexpr (LOW) *reinterpret_cast<uint4*>(at + HALF_BUF) = make_uint4(l[0], l[1], l[2], l[3]);
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = i * 8 + lane / 4, col = n + (lane & 3) * 8;
              const uint8_t* at = buf + piece16(r, lane & 3);
              if (m_warp + r < p.M && col < p.ld) {
                const int64_t d = mat + static_cast<int64_t>(m_warp + r) * p.ld + col;
                *reinterpret_cast<uint4*>(p.D_hi + d) = *reinterpret_cast<const uint4*>(at);
                if constexpr (LOW)
                  *reinterpret_cast<uint4*>(p.D_lo + d) = *reinterpret_cast<const uint4*>(at + HALF_BUF);
              }
            }
            if constexpr (SYM) {
              if (tn * TN + TN <= tm * TM && row_ok) {  // mirror: a warp's 32 rows are 64 contiguous bytes of each mirrored row
                // (low parts are kept of matrices that are one block only, and no block is below the diagonal there)
                __half* d = p.D_hi + mat + static_cast<int64_t>(n) * p.ld + m;
#pragma unroll
                for (int j = 0; j < CHUNK; ++j)
                  if (n + j < p.N) d[static_cast<int64_t>(j) * p.ld] = __float2half_rn(x[j]);
              }
            }
          } else if constexpr (EPI == kOut && sizeof(OUT) == 2) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              __align__(16) OUT e[8];
#pragma unroll
              for (int q = 0; q < 8; ++q) e[q] = from_f32<OUT>(x[8 * v + q]);
              *reinterpret_cast<uint4*>(buf + piece16(lane, v)) = *reinterpret_cast<const uint4*>(e);
            }
            __syncwarp();
            OUT* out = static_cast<OUT*>(outs.out[b]);
            if (p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + lane / 4, col = n + (lane & 3) * 8;
                if (m_warp + r < p.M && col < p.N)
                  *reinterpret_cast<uint4*>(out + static_cast<int64_t>(m_warp + r) * p.N + col) =
                      *reinterpret_cast<const uint4*>(buf + piece16(r, lane & 3));
              }
            } else {
#pragma unroll 4
              for (int r = 0; r < 32; ++r)
                if (m_warp + r < p.M && n + lane < p.N)
                  out[static_cast<int64_t>(m_warp + r) * p.N + n + lane] =
                      *reinterpret_cast<const OUT*>(buf + piece16(r, lane / 8) + (lane & 7) * 2);
            }
          } else {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<float4*>(buf + piece32(lane, v)) =
                  make_float4(x[4 * v], x[4 * v + 1], x[4 * v + 2], x[4 * v + 3]);
            __syncwarp();
            float* w = static_cast<float*>(outs.out[b]);
            __nv_bfloat16* s = EPI == kStep ? outs.shadow[b] : nullptr;
            if (p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0 && (reinterpret_cast<uintptr_t>(s) & 7) == 0) {
              float4 o[8];
              const int col = n + (lane & 7) * 4;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + lane / 8;
                if (EPI == kStep && m_warp + r < p.M && col < p.N)
                  o[i] = *reinterpret_cast<const float4*>(w + static_cast<int64_t>(m_warp + r) * p.N + col);
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + lane / 8;
                if (m_warp + r >= p.M || col >= p.N) continue;
                float4 u = *reinterpret_cast<const float4*>(buf + piece32(r, lane & 7));
                const int64_t at = static_cast<int64_t>(m_warp + r) * p.N + col;
                if constexpr (EPI == kStep) {
                  u.x = fmaf(-p.rate, u.x, p.decay * o[i].x);
                  u.y = fmaf(-p.rate, u.y, p.decay * o[i].y);
                  u.z = fmaf(-p.rate, u.z, p.decay * o[i].z);
                  u.w = fmaf(-p.rate, u.w, p.decay * o[i].w);
                  if (s != nullptr)
                    *reinterpret_cast<uint2*>(s + at) = make_uint2(pack_bf16x2(u.x, u.y), pack_bf16x2(u.z, u.w));
                }
                *reinterpret_cast<float4*>(w + at) = u;
              }
            } else {
#pragma unroll 1
              for (int r0 = 0; r0 < 32; r0 += 8) {
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  if (EPI == kStep && m_warp + r0 + i < p.M && n + lane < p.N)
                    o[i] = w[static_cast<int64_t>(m_warp + r0 + i) * p.N + n + lane];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const int r = r0 + i;
                  if (m_warp + r >= p.M || n + lane >= p.N) continue;
                  float u = *reinterpret_cast<const float*>(buf + piece32(r, lane / 4) + (lane & 3) * 4);
                  const int64_t at = static_cast<int64_t>(m_warp + r) * p.N + n + lane;
                  if constexpr (EPI == kStep) {
                    u = fmaf(-p.rate, u, p.decay * o[i]);
                    if (s != nullptr) s[at] = __float2bfloat16_rn(u);
                  }
                  w[at] = u;
                }
              }
            }
          }
        } else if constexpr (EPI != kGram) {
          cp_async_wait_but_one();
        }
        __syncwarp();  // the buffer has been written out
        fetch(seq + 2);
      }
    }
    if constexpr (EPI != kGram) cp_async_wait_all();
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

// ------------------------------------------------------------------ norm and first X
struct Ins {
  const void* u[kMaxStack];  // the matrix (orthogonalize) or the gradient (step)
  float* mom[kMaxStack];     // momentum buffers (step)
};

struct StartParams {
  int rows, cols, ld;
  int parts;           // partial sums per matrix
  double* partial;     // [count, parts] sums of squares, added in index order by every reader
  __half* hi;
  __half* lo;
  float sigma;
  double eps;
  float momentum, one_minus;  // one_minus: 1 - momentum, taken in 64 bits
  int nesterov;
  float grad_scale;
  const float* norm_sq;
  float max_norm;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// The gradient's factor: its scale times the global-norm clip coefficient (as in the AdamW kernel, NaN norms included).
__device__ __forceinline__ float grad_factor(const StartParams& p) {
  float scale = p.grad_scale;
  if (p.norm_sq != nullptr) {
    const float total = sqrtf(*p.norm_sq) * p.grad_scale;
    const float coef = p.max_norm / (total + 1e-6f);
    scale *= (coef > 1.f) ? 1.f : coef;  // a NaN norm stays NaN
  }
  return scale;
}

// Block sum of doubles in a fixed order; the result is valid in thread 0.
template <int THREADS_>
__device__ __forceinline__ double block_sum(double s) {
  __shared__ double red[THREADS_ / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < THREADS_ / 32; ++w) s += red[w];
  }
  return s;
}

constexpr int kStartThreads = 256;

__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 u = *reinterpret_cast<const float4*>(p);
  v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
}
template <typename H>
__device__ __forceinline__ void load4(const H* p, float (&v)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const H* h = reinterpret_cast<const H*>(&u);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = to_f32(h[j]);
}
// Whether a matrix (and its momentum) can be read four values at a time from its start.
template <typename T, bool STEP>
__device__ __forceinline__ bool aligned_for(const T* g, const float* mom) {
  return reinterpret_cast<uintptr_t>(g) % (4 * sizeof(T)) == 0 && (!STEP || reinterpret_cast<uintptr_t>(mom) % 16 == 0);
}

// Partial sums of squares of u (squares in 64 bits: the norm of values near the ends of fp32's range is right).
// STEP: u is built here from the gradient and the momentum, which is updated.
template <typename T, bool STEP>
__global__ void __launch_bounds__(kStartThreads) ns_norm_kernel(const __grid_constant__ Ins ins, const StartParams p) {
  const int b = blockIdx.y;
  pdl_launch();  // launched without the attribute itself: the stream's earlier work is complete
  const int64_t n = static_cast<int64_t>(p.rows) * p.cols;
  const T* g = static_cast<const T*>(ins.u[b]);
  float* mom = STEP ? ins.mom[b] : nullptr;
  const float scale = STEP ? grad_factor(p) : 1.f;
  double s = 0.0;
  auto one = [&](float gi, float& mi) {  // a value's square joins s; mi: momentum, updated
    float u = gi;
    if constexpr (STEP) {
      gi *= scale;
      mi = mi + p.one_minus * (gi - mi);
      u = p.nesterov ? gi + p.momentum * (mi - gi) : mi;
    }
    s += static_cast<double>(u) * u;
  };
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kStartThreads;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kStartThreads + threadIdx.x;
  int64_t done = 0;
  if (aligned_for<T, STEP>(g, mom)) {  // four values at a time, two such loads under way
    done = n & ~int64_t(3);
    for (int64_t i = first; i < done / 4; i += 2 * stride) {
      float v[2][4];
      float4 o[2];
      const bool two = i + stride < done / 4;
      load4(g + 4 * i, v[0]);
      if (two) load4(g + 4 * (i + stride), v[1]);
      if constexpr (STEP) {
        o[0] = reinterpret_cast<const float4*>(mom)[i];
        if (two) o[1] = reinterpret_cast<const float4*>(mom)[i + stride];
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (k == 1 && !two) break;
        one(v[k][0], o[k].x);
        one(v[k][1], o[k].y);
        one(v[k][2], o[k].z);
        one(v[k][3], o[k].w);
        if constexpr (STEP) reinterpret_cast<float4*>(mom)[i + k * stride] = o[k];
      }
    }
  }
  for (int64_t i = done + first; i < n; i += stride) {
    float mi = STEP ? mom[i] : 0.f;
    one(to_f32(g[i]), mi);
    if constexpr (STEP) mom[i] = mi;
  }
  s = block_sum<kStartThreads>(s);
  if (threadIdx.x == 0) p.partial[b * p.parts + blockIdx.x] = s;
}

// X = sigma u / max(|u|_F, eps) as hi + lo, rows padded with zeros to ld.
template <typename T, bool STEP>
__global__ void __launch_bounds__(kStartThreads) ns_first_kernel(const __grid_constant__ Ins ins, const StartParams p) {
  __shared__ double factor_s;
  const int b = blockIdx.y;
  pdl_launch();
  pdl_wait();
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < p.parts; i += 32) s += p.partial[b * p.parts + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const double norm = sqrt(s);
    // a norm that is not a number stays one
    if (threadIdx.x == 0) factor_s = static_cast<double>(p.sigma) / (norm < p.eps ? p.eps : norm);
  }
  __syncthreads();
  const double factor = factor_s;
  const T* g = static_cast<const T*>(ins.u[b]);
  const float* mom = STEP ? ins.mom[b] : nullptr;
  const float scale = STEP ? grad_factor(p) : 1.f;
  const bool vec = p.cols % 4 == 0 && aligned_for<T, STEP>(g, mom);
  const int groups = p.ld / 8;
  const int64_t total = static_cast<int64_t>(p.rows) * groups;
  const int64_t base = static_cast<int64_t>(b) * p.rows * p.ld;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kStartThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kStartThreads) {
    const int64_t r = i / groups;
    const int c = static_cast<int>(i - r * groups) * 8;
    float x[8];
    auto value = [&](float u, float mi) {
      if constexpr (STEP) {
        u *= scale;
        u = p.nesterov ? u + p.momentum * (mi - u) : mi;
      }
      return static_cast<float>(u * factor);
    };
    if (vec && c + 8 <= p.cols) {
      const int64_t at = r * p.cols + c;
      float v[2][4];
      float4 o[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        load4(g + at + 4 * k, v[k]);
        if constexpr (STEP) o[k] = *reinterpret_cast<const float4*>(mom + at + 4 * k);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        x[4 * k] = value(v[k][0], o[k].x);
        x[4 * k + 1] = value(v[k][1], o[k].y);
        x[4 * k + 2] = value(v[k][2], o[k].z);
        x[4 * k + 3] = value(v[k][3], o[k].w);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t at = r * p.cols + c + j;
        x[j] = c + j < p.cols ? value(to_f32(g[at]), STEP ? mom[at] : 0.f) : 0.f;
      }
    }
    uint32_t h[4], l[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      h[q] = f2h(x[2 * q], x[2 * q + 1]);
      const float2 back = h2f(h[q]);
      l[q] = f2h(x[2 * q] - back.x, x[2 * q + 1] - back.y);
    }
    *reinterpret_cast<uint4*>(p.hi + base + r * p.ld + c) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(p.lo + base + r * p.ld + c) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// ------------------------------------------------------------------------- host side
// A product's operand: a stack [count, rows, cols] of fp16 matrices with row stride ld.
struct Operand {
  const __half* base;
  int cols, rows, ld;
  const __half* low = nullptr;  // its low part, where products read it
};

// Its tensor map; mn_major: boxes of 64 columns x BK rows, else of 64 columns (the reduction) x box_rows rows.
inline void make_map(CUtensorMap* map, const Operand& o, bool low, int count, bool mn_major, int box_rows) {
  ensure_thread_context();
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(o.cols), static_cast<cuuint64_t>(o.rows), static_cast<cuuint64_t>(count)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(o.ld) * 2, static_cast<cuuint64_t>(o.ld) * 2 * o.rows};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(mn_major ? BK : box_rows), 1};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = encode_tiled_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(low ? o.low : o.base), dims,
                                       strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "orthogonalize: cuTensorMapEncodeTiled failed with code ", static_cast<int>(r));
}

// Tiles of one matrix.
inline int64_t tiles_of(bool sym, int M, int N, int tn) {
  const int64_t m = (M + TM - 1) / TM;
  return sym ? m * (m + 1) / 2 * (TM / tn) : m * ((N + tn - 1) / tn);
}

// Tile width with the shorter schedule.  A tile's MMAs take 512 cycles per k-block at TN = 256 and about 350 at 128 (A's share
// of the shared-memory traffic grows); its read-out, which overlaps the next tile's MMAs, about 5500 cycles (A),
// 9500 (B) and 12500 (X) at 256 and half of that at 128 (both from time stamps of single tiles).  Beyond two waves of the
// narrow tiles memory sets the pace and the wide ones win.  Measured, whole iterations (us, wide / narrow / chosen per product):
//   1 x 256 x 512    139 / 103 / 103     2 x 1024 x 4096    352 / 303 / 289      2 x 2048 x 2048   435 / 497 / 436
//   1 x 1024 x 1024  225 / 159 / 159     4 x 1024 x 4096    480 / 549 / 473      1 x 4096 x 4096  1352 / 1720 / 1350
//   3 x 1001 x 777   249 / 201 / 201     12 x 1024 x 4096  1223 / 1551 / 1220    12 x 512 x 2048   324 / 280 / 273
// The worst of 16 such stacks is 6 x 1001 x 777: 283 chosen, 268 with narrow tiles throughout.
inline int choose_tile(bool sym, bool reads, int M, int N, int K, int count, int sms) {
  const int64_t clusters = std::max(1, sms / 2), kb = (K + BK - 1) / BK;
  int64_t cost[2], waves = 0;
  for (int i = 0; i < 2; ++i) {
    const int tn = i == 0 ? 256 : 128;
    waves = (tiles_of(sym, M, N, tn) * count + clusters - 1) / clusters;
    const int64_t mma = kb * (i == 0 ? 512 : 350), out = (sym ? (reads ? 9500 : 5500) : 12500) >> i;
    cost[i] = waves * std::max(mma, out) + std::min(mma, out);
  }
  return waves <= 2 && cost[1] < cost[0] ? 128 : 256;
}

template <bool A_MN, bool B_MN, int EPI, typename OUT, int TN, bool LOW>
void launch(const Operand& a, const Operand& b, Params p, const Outs& outs, int sms, cudaStream_t stream) {
  CUtensorMap ta, tb;
  make_map(&ta, a, false, p.count, A_MN, HALF);
  make_map(&tb, b, false, p.count, B_MN, TN / 2);
  CUtensorMap ta_low = ta, tb_low = tb;
  p.passes = 1;
  p.low_a = p.low_b = 0;
  if (a.low != nullptr && b.low != nullptr) {  // X X^T, A A, B X: hi hi, hi lo, lo hi
    p.passes = 3;
    p.low_a = 0b100;
    p.low_b = 0b010;
  } else if (a.low != nullptr || b.low != nullptr) {  // B X with one of them split: hi, lo
    p.passes = 2;
    p.low_a = p.low_b = 0b10;
  }
  if (a.low != nullptr) make_map(&ta_low, a, true, p.count, A_MN, HALF);
  if (b.low != nullptr) make_map(&tb_low, b, true, p.count, B_MN, TN / 2);
  p.tiles = static_cast<int>(tiles_of(EPI == kGram || EPI == kPoly, p.M, p.N, TN));
  auto kern = ns_product_kernel<A_MN, B_MN, EPI, OUT, TN, LOW>;
  static std::atomic<uint64_t> configured{0};
  allow_smem(kern, kSmemBytes<TN>, configured);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * std::min(p.tiles * p.count, std::max(1, sms / 2)));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = kSmemBytes<TN>;
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
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, ta, tb, ta_low, tb_low, p, outs));
}

template <bool A_MN, bool B_MN, int EPI, typename OUT = float>
void product(const Operand& a, const Operand& b, const Params& p, const Outs& outs, int sms, cudaStream_t stream) {
  constexpr bool SYM = EPI == kGram || EPI == kPoly;
  const int passes = a.low != nullptr && b.low != nullptr ? 3 : a.low != nullptr || b.low != nullptr ? 2 : 1;
  const bool wide = choose_tile(SYM, EPI != kGram, p.M, p.N, passes * p.K, p.count, sms) == 256;
  if (!SYM || p.D_lo != nullptr) {
    if (wide) launch<A_MN, B_MN, EPI, OUT, 256, true>(a, b, p, outs, sms, stream);
    else launch<A_MN, B_MN, EPI, OUT, 128, true>(a, b, p, outs, sms, stream);
  } else if constexpr (SYM) {
    if (wide) launch<A_MN, B_MN, EPI, OUT, 256, false>(a, b, p, outs, sms, stream);
    else launch<A_MN, B_MN, EPI, OUT, 128, false>(a, b, p, outs, sms, stream);
  }
}

struct Shape {
  int rows, cols, count;
  int short_side, ldx, lds;
  bool tall;
  bool split;    // X's low part takes part in the products
  bool split_s;  // A's and B's low parts are kept and take part in the products
  float sigma, tau;
  // `fine`: the result keeps more than 16 bits.  The error of the update falls with both sides, while the extra passes cost
  // least where a product is mostly start and end, and those of A and B next to nothing where they are one k-block.  Measured on
  // stacks of three, error against 64 bits and time, without low parts / X's / A's and B's / both (* what is taken):
  //   8 x 16      1.1e-3  8.1e-4  1.0e-3  8e-7*     69   72   73   77 us
  //   64 x 64     7.5e-4  4.5e-4  5.7e-4  1e-6*     82   86   90   93 us
  //   64 x 512    4.9e-4  4.1e-4  2.7e-4* 4e-6      94  112  101  119 us
  //   8 x 4096    5.0e-4  5.2e-4  2.1e-4* 7e-5     151  284  158  291 us
  //   128 x 512   4.7e-4  3.5e-4* 3.1e-4  4e-6     104  121  119  137 us
  //   256 x 256   6.1e-4  3.8e-4* 4.7e-4  2e-6     105  117  125  138 us
  //   128 x 4096  3.8e-4* 3.4e-4  1.8e-4  4e-5     175  306  190  323 us
  // Larger matrices end at 2e-4 to 5e-4 without any of it.
  Shape(int64_t m, int64_t n, int64_t L, bool fine)
      : rows(static_cast<int>(m)), cols(static_cast<int>(n)), count(static_cast<int>(L)) {
    tall = m > n;
    short_side = tall ? cols : rows;
    split_s = fine && short_side <= BK;
    split = fine && std::max(m, n) <= (split_s ? 256 : 768);
    ldx = (cols + 7) / 8 * 8;
    lds = (short_side + 7) / 8 * 8;
    sigma = std::ldexp(1.f, static_cast<int>(std::min(15.0, std::round(0.5 * std::log2(static_cast<double>(m) * n)))));
    tau = std::ldexp(1.f, static_cast<int>(std::min(14.0, std::round(std::log2(static_cast<double>(short_side))))));
  }
  // fp16 elements of the workspace: X hi twice (a product reads one while its epilogue writes the other), X lo (twice too
  // where products read it), A and B (and their low parts)
  int64_t x_elems() const { return static_cast<int64_t>(count) * rows * ldx; }
  int64_t s_elems() const { return static_cast<int64_t>(count) * short_side * lds; }
  int64_t elems() const { return (split ? 4 : 3) * x_elems() + (split_s ? 4 : 2) * s_elems(); }
};

struct Workspace {
  torch::Tensor buf;
  __half *hi[2], *lo[2], *A, *B, *A_lo, *B_lo;
  float *diag_a, *diag_b;
  Workspace(const Shape& s, const torch::Device& dev) {
    const int64_t diag_elems = 4 * static_cast<int64_t>(s.count) * s.lds;  // two vectors of fp32
    buf = torch::empty({s.elems() + diag_elems}, torch::TensorOptions().dtype(at::kHalf).device(dev));
    hi[0] = reinterpret_cast<__half*>(buf.data_ptr());
    hi[1] = hi[0] + s.x_elems();
    lo[0] = hi[1] + s.x_elems();
    lo[1] = s.split ? lo[0] + s.x_elems() : lo[0];
    A = lo[1] + s.x_elems();
    B = A + s.s_elems();
    A_lo = s.split_s ? B + s.s_elems() : nullptr;
    B_lo = s.split_s ? A_lo + s.s_elems() : nullptr;
    diag_a = reinterpret_cast<float*>((s.split_s ? B_lo : B) + s.s_elems());
    diag_b = diag_a + static_cast<int64_t>(s.count) * s.lds;
  }
};

// The iterations on a workspace whose hi[0] / lo hold the first X; `last` launches the final product.
template <typename Last>
void iterate(const Shape& s, Workspace& w, int steps, double a, double b, double c, int* status, int sms,
             cudaStream_t stream, Last last) {
  const Outs none{};
  const Operand A{w.A, s.short_side, s.short_side, s.lds, w.A_lo}, B{w.B, s.short_side, s.short_side, s.lds, w.B_lo};
  for (int it = 0; it < steps; ++it) {
    const int cur = it & 1;
    const Operand X{w.hi[cur], s.cols, s.rows, s.ldx, s.split ? w.lo[cur] : nullptr};
    Params p{};
    p.count = s.count;
    p.status = status;
    p.ld_s = s.lds;
    p.tau = s.tau;
    // A' = tau A = (tau / sigma^2) X' X'^T
    p.M = p.N = s.short_side;
    p.K = s.tall ? s.rows : s.cols;
    p.ld = s.lds;
    p.alpha = s.tau / s.sigma / s.sigma;
    p.beta = 0.f;
    p.D_hi = w.A;
    p.D_lo = w.A_lo;
    p.diag = w.diag_a;
    if (s.tall) product<true, true, kGram>(X, X, p, none, sms, stream);
    else product<false, false, kGram>(X, X, p, none, sms, stream);
    // B' = tau (b A + c A A), off the diagonal (b + c (a_i + a_j)) A' + (c / tau) A' A' with A' zero on it
    p.K = s.short_side;
    p.alpha = static_cast<float>(c / s.tau);
    p.beta = static_cast<float>(b);
    p.C_hi = w.A;
    p.C_lo = w.A_lo;
    p.D_hi = w.B;
    p.D_lo = w.B_lo;
    p.gamma = static_cast<float>(c);
    p.diag_a = w.diag_a;
    p.diag = w.diag_b;
    product<false, false, kPoly>(A, A, p, none, sms, stream);
    // X' <- a X' + (1 / tau) B' X'   (or X' B')
    p.M = s.rows;
    p.N = s.cols;
    p.K = s.short_side;
    p.ld = s.ldx;
    p.alpha = 1.f / s.tau;
    p.beta = static_cast<float>(a);
    p.diag_scale = 1.f;
    p.C_hi = w.hi[cur];
    p.C_lo = w.lo[cur];
    if (it + 1 < steps) {
      p.D_hi = w.hi[cur ^ 1];
      p.D_lo = w.lo[cur ^ 1];  // in place where no product reads it: each element is read and written by one thread
      if (s.tall) product<false, false, kNext>(X, B, p, none, sms, stream);
      else product<false, true, kNext>(B, X, p, none, sms, stream);
    } else {
      p.alpha /= s.sigma;
      p.beta /= s.sigma;
      p.diag_scale /= s.sigma;
      last(s.tall ? X : B, s.tall ? B : X, p);
    }
  }
}

// Matrices per group: bounded by the pointer table and by 2 GiB of workspace.
inline int64_t group_size(int64_t rows, int64_t cols, int64_t count) {
  const Shape one(rows, cols, 1, true);
  const int64_t fit = std::max<int64_t>(1, (int64_t(1) << 30) / std::max<int64_t>(1, one.elems()));
  return std::min<int64_t>(count, std::min<int64_t>(kMaxStack, fit));
}

// Norm, first X and three products an iteration.
inline int64_t kernels_per_group(int64_t steps) { return 2 + 3 * steps; }

inline StartParams start_params(const Shape& s, Workspace& w, torch::Tensor& partial, double eps) {
  StartParams q{};
  q.rows = s.rows;
  q.cols = s.cols;
  q.ld = s.ldx;
  q.parts = static_cast<int>(partial.size(1));
  q.partial = partial.data_ptr<double>();
  q.hi = w.hi[0];
  q.lo = w.lo[0];
  q.sigma = s.sigma;
  q.eps = eps;
  q.grad_scale = 1.f;
  return q;
}

// CTAs per matrix of the two start kernels: enough to fill the GPU eight times over the stack, at least 2048 values each.
inline int start_ctas(const Shape& s, int sms) {
  const int64_t n = static_cast<int64_t>(s.rows) * s.ldx;
  const int64_t want = std::max<int64_t>(1, 8ll * sms / s.count);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, n / 2048)));
}

template <typename T, bool STEP>
void start(const Ins& ins, const StartParams& q, const Shape& s, int ctas, cudaStream_t stream) {
  ns_norm_kernel<T, STEP><<<dim3(q.parts, s.count), kStartThreads, 0, stream>>>(ins, q);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, s.count);
  cfg.blockDim = dim3(kStartThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, ns_first_kernel<T, STEP>, ins, q));
}

void check_sizes(int64_t rows, int64_t cols, int64_t steps, const std::vector<double>& coefficients) {
  TORCH_CHECK(rows > 0 && cols > 0 && rows < (1 << 30) && cols < (1 << 30), "orthogonalize: matrix sizes");
  TORCH_CHECK(steps >= 1 && coefficients.size() == 3, "orthogonalize: at least one step, three coefficients");
}

template <typename OUT>
void last_out(const Operand& ta, const Operand& tb, const Params& p, const Outs& o, bool tall, int sms,
              cudaStream_t stream) {
  if (tall) product<false, false, kOut, OUT>(ta, tb, p, o, sms, stream);
  else product<false, true, kOut, OUT>(ta, tb, p, o, sms, stream);
}

}  // namespace muon
}  // namespace mvp

// O [count, m, n] of x [count, m, n] (contiguous fp32 / bf16 / fp16), in `out`'s type.  Returns the kernels launched.
int64_t orthogonalize(const torch::Tensor& x, torch::Tensor& out, int64_t steps, const std::vector<double>& coefficients,
                   double eps, int64_t status_ptr) {
  using namespace mvp::muon;
  TORCH_CHECK(x.is_cuda() && x.dim() == 3 && x.is_contiguous(), "orthogonalize: contiguous CUDA [count, m, n]");
  TORCH_CHECK(out.is_cuda() && out.device() == x.device() && out.is_contiguous() && out.sizes() == x.sizes(),
              "orthogonalize: contiguous output of the input's shape and device");
  check_sizes(x.size(1), x.size(2), steps, coefficients);
  const at::cuda::CUDAGuard guard(x.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int sms = mvp::num_sms(x.get_device());
  const int64_t size = x.size(1) * x.size(2);
  const int64_t group = group_size(x.size(1), x.size(2), x.size(0));
  int64_t launched = 0;
  for (int64_t first = 0; first < x.size(0); first += group) {
    const Shape s(x.size(1), x.size(2), std::min<int64_t>(group, x.size(0) - first), out.scalar_type() == at::kFloat);
    Workspace w(s, x.device());
    const int ctas = start_ctas(s, sms);
    auto partial = torch::empty({s.count, ctas}, x.options().dtype(at::kDouble));
    StartParams q = start_params(s, w, partial, eps);
    Ins ins{};
    Outs outs{};
    for (int i = 0; i < s.count; ++i) {
      ins.u[i] = static_cast<const char*>(x.data_ptr()) + (first + i) * size * x.element_size();
      outs.out[i] = static_cast<char*>(out.data_ptr()) + (first + i) * size * out.element_size();
    }
    if (x.scalar_type() == at::kFloat) start<float, false>(ins, q, s, ctas, stream);
    else if (x.scalar_type() == at::kBFloat16) start<__nv_bfloat16, false>(ins, q, s, ctas, stream);
    else if (x.scalar_type() == at::kHalf) start<__half, false>(ins, q, s, ctas, stream);
    else TORCH_CHECK(false, "orthogonalize: fp32, bf16 or fp16 input");
    iterate(s, w, static_cast<int>(steps), coefficients[0], coefficients[1], coefficients[2],
            reinterpret_cast<int*>(status_ptr), sms, stream,
            [&](const Operand& ta, const Operand& tb, const Params& p) {
              if (out.scalar_type() == at::kFloat) last_out<float>(ta, tb, p, outs, s.tall, sms, stream);
              else if (out.scalar_type() == at::kBFloat16) last_out<__nv_bfloat16>(ta, tb, p, outs, s.tall, sms, stream);
              else if (out.scalar_type() == at::kHalf) last_out<__half>(ta, tb, p, outs, s.tall, sms, stream);
              else TORCH_CHECK(false, "orthogonalize: fp32, bf16 or fp16 output");
            });
    launched += kernels_per_group(steps);
  }
  return launched;
}

// One step on same-shaped fp32 matrices p (master), g (gradient), mom (momentum); see ops.muon_step_.  Returns the kernels
// launched.
int64_t muon_step_(const std::vector<torch::Tensor>& p, const std::vector<torch::Tensor>& g,
                const std::vector<torch::Tensor>& mom, const std::vector<torch::Tensor>& p_bf16, double rate,
                double decay, double momentum, bool nesterov, int64_t steps, const std::vector<double>& coefficients,
                double eps, double grad_scale, const c10::optional<torch::Tensor>& norm_sq, double max_norm,
                int64_t status_ptr) {
  using namespace mvp::muon;
  if (p.empty()) return 0;
  const size_t count = p.size();
  TORCH_CHECK(g.size() == count && mom.size() == count && (p_bf16.empty() || p_bf16.size() == count),
              "muon_step_: one gradient, momentum (and bf16 copy) per weight");
  const auto dev = p[0].device();
  const auto sizes = p[0].sizes();
  TORCH_CHECK(p[0].is_cuda() && p[0].dim() == 2, "muon_step_: CUDA matrices");
  auto check = [&](const torch::Tensor& t, at::ScalarType type, const char* what) {
    TORCH_CHECK(t.device() == dev && t.scalar_type() == type && t.sizes() == sizes && t.is_contiguous(), "muon_step_: ",
                what, " must be contiguous, of one shape, type and device");
  };
  for (size_t i = 0; i < count; ++i) {
    check(p[i], at::kFloat, "fp32 weights");
    check(g[i], at::kFloat, "fp32 gradients");
    check(mom[i], at::kFloat, "fp32 momenta");
    if (!p_bf16.empty()) check(p_bf16[i], at::kBFloat16, "bf16 copies");
  }
  TORCH_CHECK(!norm_sq.has_value() || (norm_sq->device() == dev && norm_sq->scalar_type() == at::kFloat &&
                                       norm_sq->numel() == 1),
              "muon_step_: norm_sq must be one fp32 value on the weights' device");
  check_sizes(sizes[0], sizes[1], steps, coefficients);
  const at::cuda::CUDAGuard guard(dev);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int sms = mvp::num_sms(dev.index());
  const int64_t group = group_size(sizes[0], sizes[1], static_cast<int64_t>(count));
  int64_t launched = 0;
  for (int64_t first = 0; first < static_cast<int64_t>(count); first += group) {
    const Shape s(sizes[0], sizes[1], std::min<int64_t>(group, static_cast<int64_t>(count) - first), true);
    Workspace w(s, dev);
    const int ctas = start_ctas(s, sms);
    auto partial = torch::empty({s.count, ctas}, p[0].options().dtype(at::kDouble));
    StartParams q = start_params(s, w, partial, eps);
    q.momentum = static_cast<float>(momentum);
    q.one_minus = static_cast<float>(1.0 - momentum);
    q.nesterov = nesterov ? 1 : 0;
    q.grad_scale = static_cast<float>(grad_scale);
    q.norm_sq = norm_sq.has_value() ? norm_sq->data_ptr<float>() : nullptr;
    q.max_norm = static_cast<float>(max_norm);
    Ins ins{};
    Outs outs{};
    for (int i = 0; i < s.count; ++i) {
      ins.u[i] = g[first + i].data_ptr();
      ins.mom[i] = mom[first + i].data_ptr<float>();
      outs.out[i] = p[first + i].data_ptr();
      outs.shadow[i] = p_bf16.empty() ? nullptr : reinterpret_cast<__nv_bfloat16*>(p_bf16[first + i].data_ptr());
    }
    start<float, true>(ins, q, s, ctas, stream);
    iterate(s, w, static_cast<int>(steps), coefficients[0], coefficients[1], coefficients[2],
            reinterpret_cast<int*>(status_ptr), sms, stream,
            [&](const Operand& ta, const Operand& tb, Params l) {
              l.rate = static_cast<float>(rate);
              l.decay = static_cast<float>(decay);
              if (s.tall) product<false, false, kStep>(ta, tb, l, outs, sms, stream);
              else product<false, true, kStep>(ta, tb, l, outs, sms, stream);
            });
    launched += kernels_per_group(steps);
  }
  return launched;
}
