// Product of two microscaled 4-bit matrices on the block-scaled tensor cores of sm_100a, and the
// gated product of one with two (see include/gemmzoo/microscale.h for the operators):
//
//   D = act(alpha * row_scale * col_scale * A B^T + beta * C + bias)
//   H = act(alpha * A G^T) * (alpha_up * A U^T)          (optionally quantised along its rows)
//
// The machinery is that of sm100_gemm.cuh (TMA producers, one MMA issuer, epilogue warps, bounded
// waits) with a fourth ring operand: the scales.  A stage holds 256 elements of K: 128-byte-swizzled
// rows of codes and, per 128 rows, 512-byte tiles of scales, which the MMA warp copies to tensor
// memory (tcgen05.cp, four columns per tile, repeated for the four lane quadrants) right before the
// tcgen05.mma that reads them.  Copies and MMAs of one thread execute in order, so the four scale slots
// in tensor memory need no barrier of their own.
//
// Two tile families:
//   row tiles  256 x 256 or 256 x 128 on a CTA pair (cta_group::2), 128 x 256 or 128 x 128 on one CTA: A's
//              rows on the 128-lane side.  In a pair each CTA loads its own 128 rows of A and its own 128 rows of B, and the
//              scales of all 256 rows of B.  The gated product takes 128 rows of the gate and 128 of the
//              up projection as its 256 (in a pair CTA 0 loads the gate's, CTA 1 the up projection's):
//              one MMA computes both halves and no operand is loaded twice.  Two fp32 accumulators of
//              256 columns would fill tensor memory and leave no room for scales, so they overlap in 64
//              columns: [0, 256) and [192, 448).  The epilogue reads the shared 64 columns first and
//              the next tile's main loop starts while it works on the other 192.  The tensor pipe idles
//              for about 1,500 clocks per tile (two signals and the first MMA's way through the pipe);
//              running ahead with the half that overlaps nothing needs MMAs of 128 columns, which lose
//              more than that (8192^3: 187 -> 206 us).  A sixth stage in place of half of the output
//              staging, the epilogue's parameters held in registers, or one store per 64 columns
//              change nothing or cost a little.
//   swapped    few rows of A: B's rows on the 128-lane side (128 features per tile), 16, 32 or 64 rows of
//              A on the narrow side, so every byte a stage loads is a useful byte of B.  The gated
//              product keeps two row blocks per stage (gate and up).  One tile per CTA and shared memory
//              for two CTAs per SM: one streams while the other starts or finishes.  The accumulator
//              is the transpose of the output; it goes through shared memory, after which a warp takes
//              one output row at a time, a lane four neighbouring columns.
// Where tiles are fewer than SMs, the CTAs (pairs) of a cluster share a tile's K range.  Their partial
// sums meet in shared memory; each CTA adds and finishes a share of the tile, in rank order, so there
// is no workspace, nothing to clear and one order of summation.  The partial sums lie in the ring that
// the main loop no longer needs, and the CTA that finishes a share fetches it from its peers 16 bytes a
// lane.  (Storing each row into the CTA that finishes it instead saves a barrier but measured 0.3 us
// slower at 16 rows and 2.4 us at 64: remote stores of a word per lane are slow.)
#ifndef GZ_MX_GEMM_CUH
#define GZ_MX_GEMM_CUH

#include <type_traits>

#include "mx_format.cuh"
#include "sm100_gemm.cuh"

namespace gz {

// Output of a gated product: a gz_dtype, or one of these.
constexpr uint32_t MX_OUT_FP4 = 16, MX_OUT_NVFP4 = 17;

struct MxMaps {
  CUtensorMap wide, wide_scales;      // the operand on the 128-lane side
  CUtensorMap narrow, narrow_scales;  // the other one
  CUtensorMap up, up_scales;          // gated: the up projection (the gate is `wide` of a swapped tile, `narrow` of a row tile)
  CUtensorMap d;
};

struct MxParams {
  TileGrid grid;  // tiles_m along the 128-lane side
  uint32_t m, n;  // rows and columns of the output
  uint32_t k_blocks;
  uint32_t split;  // CTAs or CTA pairs (one cluster) that share a tile's K range
  uint32_t prefetch;  // swapped tiles: K blocks brought into L2 ahead of the launch's dependencies (at most 32)
  uint32_t idesc;
  uint32_t out_type;
  uint32_t out_tma, c_vec_ok;
  uint32_t d_vec_ok;  // swapped tiles: four columns of C and of D may be accessed at once
  uint32_t test_flags;
  uint32_t epi_flags, act;  // bit 0 bias, 1 row_scale, 2 col_scale
  float alpha, alpha_up, beta, out_multiplier;
  const float* bias;
  const float* row_scale;
  const float* col_scale;
  const void* c;
  void* d;
  uint8_t* d_scales;
  int64_t ldc, ldd;   // elements (a quantised output: bytes)
  int64_t d_groups;   // quantised output: scale tiles per 128 rows
  uint32_t* status;
  uint64_t wait_limit_ns;
};

template <bool NV_, int BN_, int CTAS_, bool GATED_>
struct MxCfg {
  static constexpr bool NV = NV_, GATED = GATED_;
  static constexpr int BN = BN_, CTAS = CTAS_;
  static constexpr bool SWAP = BN <= 64;
  static constexpr int MB = (GATED && SWAP) ? 2 : 1;  // 128-row blocks on the wide side per CTA
  static constexpr int TILES_K = NV ? 4 : 2;          // scale tiles per stage and 128 rows
  static constexpr int NRB = BN > 128 ? 2 : 1;        // scale row groups of the narrow side
  static constexpr int W_BYTES = MB * 128 * 128;
  static constexpr int N_BYTES = (BN / CTAS) * 128;
  static constexpr int WS_BYTES = MB * TILES_K * 512;
  static constexpr int NS_BYTES = NRB * TILES_K * 512;
  static constexpr int STAGE_BYTES = W_BYTES + N_BYTES + WS_BYTES + NS_BYTES;
  static constexpr int EPI_WARPS = SWAP ? 4 : 8;
  static constexpr int STAGING_BYTES = SWAP ? 0 : EPI_WARPS * 4096;
  static constexpr int BAR_BYTES = 512;
  // 227 KB per block; two blocks per SM share 228 KB of which each costs 1 KB more than it asks for
  static constexpr int PER_SM = SWAP ? 2 : 1;
  static constexpr int SMEM_LIMIT = PER_SM == 2 ? 115712 : 232448;
  static constexpr int STAGES = (SMEM_LIMIT - 1024 - STAGING_BYTES - BAR_BYTES) / STAGE_BYTES;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int SMEM_BYTES = 1024 + RING_BYTES + STAGING_BYTES + BAR_BYTES;
  static constexpr int THREADS = 96 + 32 * EPI_WARPS;
  // Tensor memory: accumulators, then four 16-column scale slots.  (Swapped tiles: at most half of it, so
  // that a second block's allocation never has to wait for the first block.)
  static constexpr int ACC_STRIDE = BN == 256 ? 192 : BN;  // row tiles: from one accumulator to the next
  static constexpr int ACC_COLS = SWAP ? MB * BN : ACC_STRIDE + BN;
  static constexpr int SLOT_COLS = 16;
  static constexpr int TMEM_COLS = ACC_COLS + 64 <= 128 ? 128 : ACC_COLS + 64 <= 256 ? 256 : 512;
  static_assert(ACC_COLS % 16 == 0 && ACC_COLS + 64 <= TMEM_COLS && (!SWAP || TMEM_COLS <= 256), "tensor memory");
  // (a row tile's B scales have to start at a whole scale tile: 128 rows)
  static_assert(SWAP ? (BN % 16 == 0 && CTAS == 1) : (BN == 256 || (BN == 128 && !GATED)), "tile shapes");
  static_assert(STAGE_BYTES % 1024 == 0 && STAGES >= 2, "ring");
  static_assert(MB * BN * 128 * 4 <= RING_BYTES, "partial sums meet in the ring");
  static_assert(8 * (2 * STAGES + 3) + 16 <= BAR_BYTES, "barriers");
};

namespace detail {

#if defined(GZ_BOUNDS_CHECK)
static __device__ __noinline__ bool mx_store_in_bounds(const MxParams& p, uint32_t row, uint32_t col, uint32_t ncols,
                                                       uint32_t rows, uint32_t cols) {
  if (row < rows && col < cols && ncols <= cols - col) return true;
  if (atomicCAS(p.status, 0u, STORE_OUT_OF_BOUNDS) == 0u) {
    p.status[1] = blockIdx.x;
    p.status[2] = row;
    p.status[3] = col;
    __threadfence();
  }
  return false;
}
#define GZ_MX_STORE_OK(p, row, col, ncols, rows, cols) detail::mx_store_in_bounds(p, row, col, ncols, rows, cols)
#else
#define GZ_MX_STORE_OK(p, row, col, ncols, rows, cols) true
#endif
// The same for `blocks` scales of one row from `block` on: the scale array holds whole tiles of 128 rows x 4 blocks.
#define GZ_MX_SCALE_OK(p, row, block, blocks) \
  GZ_MX_STORE_OK(p, row, static_cast<uint32_t>(block), blocks, ((p).m + 127u) & ~127u, static_cast<uint32_t>(4 * (p).d_groups))

// The activations, within 5e-7 |x| of the exact ones.  Both GELUs are taken from the complement that is small where x is
// negative (1 + erf and 1 + tanh would cancel there: at x = -6 nothing is left in fp32): erfc by the factors of erf_fast,
// 1 + tanh u as 2 / (1 + e^(-2u)).
__device__ __forceinline__ float mx_activate(float x, uint32_t act) {
  if (act == 2u) {
    float poly_t, e;
    erfc_factors(fabsf(x * 0.70710678118654752f), poly_t, e);
    const float c = poly_t * e;
    return 0.5f * x * (x < 0.0f ? c : 2.0f - c);
  }
  if (act == 3u) {
    const float u = 0.7978845608028654f * (x + 0.044715f * x * x * x);
    return x * rcp_approx(1.0f + __expf(-2.0f * u));
  }
  return activate(x, act);
}

// One activation's code per pass.
template <int N>
__device__ __forceinline__ void activate_all(float (&f)[N], uint32_t act) {
  switch (act) {
    case 1:
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = mx_activate(f[i], 1);
      break;
    case 2:
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = mx_activate(f[i], 2);
      break;
    case 3:
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = mx_activate(f[i], 3);
      break;
    case 4:
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = mx_activate(f[i], 4);
      break;
    default: break;
  }
}

__device__ __forceinline__ float mx_load_c(const MxParams& p, int64_t at) {
  switch (p.out_type) {
    case 0: return __half2float(static_cast<const __half*>(p.c)[at]);
    case 1: return __bfloat162float(static_cast<const __nv_bfloat16*>(p.c)[at]);
    default: return static_cast<const float*>(p.c)[at];
  }
}

// 32 columns of one row of C as raw words, where they can be read 16 bytes at a time.  A row tile reads
// them ahead of the sums they are added to: a lane's row is 64 or 128 bytes at an address of its
// own, so the loads are all latency.
__device__ __forceinline__ bool mx_c_vectors(const MxParams& p, uint32_t row, uint32_t col0) {
  return p.beta != 0.0f && p.c_vec_ok && row < p.m && col0 + 32u <= p.n;
}
__device__ __forceinline__ void mx_load_c_words(const MxParams& p, uint32_t row, uint32_t col0, uint32_t (&w)[32]) {
  if (!mx_c_vectors(p, row, col0)) return;
  const int64_t at = static_cast<int64_t>(row) * p.ldc + col0;
  const uint4* c4 = p.out_type == 2u ? reinterpret_cast<const uint4*>(static_cast<const float*>(p.c) + at)
                                     : reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.c) + at);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    if (q < 4 || p.out_type == 2u) {
      const uint4 c = c4[q];
      w[4 * q] = c.x;
      w[4 * q + 1] = c.y;
      w[4 * q + 2] = c.z;
      w[4 * q + 3] = c.w;
    }
  }
}

// The same for a C whose rows cannot be read 16 bytes at a time: the warp takes one row after the other, a lane one
// column, and mx_row_terms turns the box (a lane's own row in single values measured 1265 us for 8192 x 16383 fp16 at
// k = 64, this 419).
__device__ __forceinline__ void mx_load_c_rows(const MxParams& p, uint32_t row0, uint32_t col0, uint32_t lane, uint32_t (&w)[32]) {
  if (row0 >= p.m || col0 >= p.n) return;
  const uint32_t rows = col0 + lane < p.n ? p.m - row0 : 0u;  // that this lane has a column of
  const int64_t at = static_cast<int64_t>(row0) * p.ldc + col0 + lane;
  if (p.out_type == 2u) {
    const uint32_t* c = static_cast<const uint32_t*>(p.c) + at;
#pragma unroll
    for (int r = 0; r < 32; ++r) w[r] = static_cast<uint32_t>(r) < rows ? c[r * p.ldc] : 0u;
  } else {
    const uint16_t* c = static_cast<const uint16_t*>(p.c) + at;
#pragma unroll
    for (int r = 0; r < 32; ++r) w[r] = static_cast<uint32_t>(r) < rows ? c[r * p.ldc] : 0u;
  }
}
template <bool BY_ROWS>
__device__ __forceinline__ void mx_load_c_box(const MxParams& p, uint32_t row0, uint32_t col0, uint32_t lane, uint32_t (&w)[32]) {
  if constexpr (BY_ROWS) mx_load_c_rows(p, row0, col0, lane, w);
  else mx_load_c_words(p, row0 + lane, col0, w);
}

// The optional terms on 32 columns of one row (row tiles); w: the words that mx_load_c_box read.
template <bool BY_ROWS>
__device__ __forceinline__ void mx_row_terms(const MxParams& p, float (&f)[32], const uint32_t (&w)[32], uint32_t stg,
                                             uint32_t row, uint32_t col0, uint32_t lane) {
  const bool row_ok = row < p.m;
  const uint32_t ncols = p.n - col0 < 32u ? p.n - col0 : 32u;
  const bool col_ok = lane < ncols;
  if (p.epi_flags & 2u) {
    const float rs = row_ok ? p.row_scale[row] : 1.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] *= rs;
  }
  if (p.epi_flags & 4u) {
    const float mine = col_ok ? p.col_scale[col0 + lane] : 1.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] *= __shfl_sync(0xFFFFFFFFu, mine, i);
  }
  if constexpr (BY_ROWS) {
    // turned in the staging, whose rows are rotated so that neither side meets a bank twice
    if (p.out_tma && lane == 0) ptx::bulk_wait_group_read<0>();
    __syncwarp();
#pragma unroll
    for (uint32_t r = 0; r < 32; ++r) {
      const float c = p.out_type == 2u   ? __uint_as_float(w[r])
                      : p.out_type == 0u ? unpack2<__half>(w[r]).x
                                         : unpack2<__nv_bfloat16>(w[r]).x;
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(stg + r * 128u + (((lane + r) & 31u) << 2)), "f"(c) : "memory");
    }
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < 32; ++i) {
      float c;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(c) : "r"(stg + lane * 128u + (((i + lane) & 31u) << 2)) : "memory");
      f[i] = fmaf(p.beta, c, f[i]);
    }
  } else if (p.beta != 0.0f && row_ok) {
    if (mx_c_vectors(p, row, col0)) {
      if (p.out_type == 2u) {
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = fmaf(p.beta, __uint_as_float(w[i]), f[i]);
      } else {
        const bool half_in = p.out_type == 0u;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 c = half_in ? unpack2<__half>(w[i]) : unpack2<__nv_bfloat16>(w[i]);
          f[2 * i] = fmaf(p.beta, c.x, f[2 * i]);
          f[2 * i + 1] = fmaf(p.beta, c.y, f[2 * i + 1]);
        }
      }
    } else {
      const int64_t at = static_cast<int64_t>(row) * p.ldc + col0;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (static_cast<uint32_t>(i) < ncols) f[i] = fmaf(p.beta, mx_load_c(p, at + i), f[i]);
    }
  }
  if (p.epi_flags & 1u) {
    const float mine = col_ok ? p.bias[col0 + lane] : 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] += __shfl_sync(0xFFFFFFFFu, mine, i);
  }
  activate_all(f, p.act);
}

// 32 rows x 32 columns (lane = row) to the output through the warp's 4 KB of staging: a TMA store of a
// swizzled box, or, where TMA cannot describe D, whole row pieces with plain stores.  The latter also for a last
// box whose rows end inside 16 bytes: a TMA store ends there at the next multiple of 16 bytes and would write to
// what lies beside D.  `turn` alternates the two halves of the staging for 16-bit outputs.
__device__ __forceinline__ void mx_store_box(const MxParams& p, const void* tm_d, uint32_t stg, uint32_t lane,
                                             const float (&f)[32], uint32_t row0, uint32_t col0, uint32_t& turn) {
  const bool wide = p.out_type == 2u;
  const uint32_t box = wide ? stg : stg + (turn & 1u) * 2048u;
  const bool tma = p.out_tma && (col0 + 32u <= p.n || (p.n & (wide ? 3u : 7u)) == 0u);
  if (p.out_tma) {
    if (lane == 0) {
      if (wide || !tma) ptx::bulk_wait_group_read<0>();  // (a box without a group of its own: the next may wait for one only)
      else ptx::bulk_wait_group_read<1>();
    }
  }
  __syncwarp();
  if (wide) {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + lane * 128u + ((j ^ (lane & 7u)) << 4)),
                   "f"(f[4 * j]), "f"(f[4 * j + 1]), "f"(f[4 * j + 2]), "f"(f[4 * j + 3])
                   : "memory");
  } else {
    uint32_t w[16];
    if (p.out_type == 0u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pack2<__half>(f[2 * i], f[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pack2<__nv_bfloat16>(f[2 * i], f[2 * i + 1]);
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + lane * 64u + ((j ^ ((lane >> 1) & 3u)) << 4)),
                   "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                   : "memory");
  }
  if (tma) {
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      ptx::tma_store_3d(tm_d, box, static_cast<int32_t>(col0), static_cast<int32_t>(row0), 0);
      ptx::bulk_commit_group();
    }
  } else {
    __syncwarp();
    const uint32_t rows = lane < p.n - col0 ? p.m - row0 : 0u;  // that this lane has a column of
    // Four values out of shared memory, then four stores: one after the other costs a latency per row.  8192 x 16383 fp16
    // at k = 64: 1 / 4 / 8 at a time 248 / 214 / 192 us, but with 8 the aligned form with C, short of registers,
    // goes from 58 to 66 us (2048 x 14336 x 4096 fp16).
#pragma unroll 1
    for (uint32_t r0 = 0; r0 < 32u; r0 += 4u) {
      const int64_t at = static_cast<int64_t>(row0 + r0) * p.ldd + col0 + lane;
      uint32_t v[4];
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t r = r0 + e;
        if (wide) {
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[e]) : "r"(box + r * 128u + (((lane >> 2) ^ (r & 7u)) << 4) + (lane & 3u) * 4u) : "memory");
        } else {
          uint16_t h;
          asm volatile("ld.shared.b16 %0, [%1];" : "=h"(h) : "r"(box + r * 64u + (((lane >> 3) ^ ((r >> 1) & 3u)) << 4) + (lane & 7u) * 2u) : "memory");
          v[e] = h;
        }
      }
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        if (r0 + e >= rows || !GZ_MX_STORE_OK(p, row0 + r0 + e, col0 + lane, 1u, p.m, p.n)) continue;
        if (wide) static_cast<uint32_t*>(p.d)[at + e * p.ldd] = v[e];
        else static_cast<uint16_t*>(p.d)[at + e * p.ldd] = static_cast<uint16_t>(v[e]);
      }
    }
    __syncwarp();
  }
  ++turn;
}

// 32 columns of one row, quantised: the codes and the one or two scales (pair tile; lane = row).
template <bool NV>
__device__ __forceinline__ void mx_store_quantized(const MxParams& p, const float (&f)[32], uint32_t row, uint32_t col0) {
  constexpr int BLOCK = mx::Format<NV>::BLOCK;
  const bool row_ok = row < p.m;
  uint32_t codes[4];
#pragma unroll
  for (int b = 0; b < 32 / BLOCK; ++b) {
    float v[BLOCK];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) {
      v[i] = col0 + b * BLOCK + i < p.n ? f[b * BLOCK + i] * p.out_multiplier : 0.0f;
      amax = mx::amax_nan(amax, v[i]);
    }
    const mx::Scale s = mx::block_scale<NV>(amax);
#pragma unroll
    for (int i = 0; i < BLOCK / 8; ++i) {
      float* x = &v[i * 8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = mx::in_code_units<NV>(x[j], s);
      const uint32_t c = mx::pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
      codes[b * (BLOCK / 8) + i] = s.byte == mx::Format<NV>::NAN_SCALE ? 0u : c;
    }
    const int64_t block = static_cast<int64_t>(col0) / BLOCK + b;
    if (block < 4 * p.d_groups && GZ_MX_SCALE_OK(p, row, block, 1u))  // rows up to the next multiple of 128 exist in the scale array
      p.d_scales[mx::scale_word(row, block >> 2, p.d_groups) + (block & 3)] = static_cast<uint8_t>(row_ok ? s.byte : 0u);
  }
  if (row_ok && col0 < p.n && GZ_MX_STORE_OK(p, row, col0, 1u, p.m, p.n))
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.d) + static_cast<int64_t>(row) * p.ldd + col0 / 2) =
        make_uint4(codes[0], codes[1], codes[2], codes[3]);
}

// One output row of a swapped tile, quantised: the warp's lanes hold four neighbouring columns each, so
// eight lanes share an e8m0 block and four an e4m3 block.
template <bool NV>
__device__ __forceinline__ void mx_store_quantized_row(const MxParams& p, const float (&f)[4], uint32_t row, uint32_t col,
                                                       uint32_t lane, bool live) {
  constexpr int LANES = mx::Format<NV>::BLOCK / 4;
  float v[4];
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = col + i < p.n ? f[i] * p.out_multiplier : 0.0f;
    amax = mx::amax_nan(amax, v[i]);
  }
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) amax = mx::amax_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
  const mx::Scale s = mx::block_scale<NV>(amax);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mx::in_code_units<NV>(v[i], s);
  uint32_t codes = mx::pack8(v[0], v[1], v[2], v[3], 0.0f, 0.0f, 0.0f, 0.0f);
  if (s.byte == mx::Format<NV>::NAN_SCALE) codes = 0u;
  if (live && (col & ~31u) < p.n && GZ_MX_STORE_OK(p, row, col & ~31u, 1u, p.m, p.n))  // the codes of a row fill up whole 32s
    *reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(p.d) + static_cast<int64_t>(row) * p.ldd + col / 2) =
        static_cast<uint16_t>(codes);
  const int64_t block = col / mx::Format<NV>::BLOCK;
  if (live && lane % LANES == 0u && block < 4 * p.d_groups && GZ_MX_SCALE_OK(p, row, block, 1u))
    p.d_scales[mx::scale_word(row, block >> 2, p.d_groups) + (block & 3)] = static_cast<uint8_t>(s.byte);
}

// Up to four columns of a row as fp32, and back (`n` of them exist).
__device__ __forceinline__ void mx_load4(const float* v, uint32_t n, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = static_cast<uint32_t>(i) < n ? v[i] : 0.0f;
}

}  // namespace detail

// Finish one output row of a swapped tile: the warp's lanes hold the sums of four neighbouring columns each.
// live == false does everything but the stores: the epilogue runs this once while it waits for its
// accumulator, because code that runs cold runs at the speed instructions can be fetched.
template <class Cfg>
__device__ __forceinline__ void mx_finish_row(const MxParams& p, float (&f)[4], const float (&u)[4], uint32_t row,
                                              uint32_t col, uint32_t lane, bool live) {
  const uint32_t have = col >= p.n ? 0u : p.n - col < 4u ? p.n - col : 4u;  // columns that exist
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] *= p.alpha;
  if constexpr (Cfg::GATED) {
    detail::activate_all(f, p.act);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= p.alpha_up * u[i];
    if (p.out_type == MX_OUT_FP4) return detail::mx_store_quantized_row<false>(p, f, row, col, lane, live);
    if (p.out_type == MX_OUT_NVFP4) return detail::mx_store_quantized_row<true>(p, f, row, col, lane, live);
  }
  if (have == 0u || !GZ_MX_STORE_OK(p, row, col, have, p.m, p.n)) return;
  const bool vec = have == 4u && p.d_vec_ok;
  if constexpr (!Cfg::GATED) {
    float t[4];
    if (p.epi_flags & 2u) {
      const float rs = p.row_scale[row];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] *= rs;
    }
    if (p.epi_flags & 4u) {
      detail::mx_load4(p.col_scale + col, have, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] *= t[i];
    }
    if (p.beta != 0.0f) {
      const int64_t at = static_cast<int64_t>(row) * p.ldc + col;
      if (vec && p.out_type != 2u) {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.c) + at);
        const float2 lo = p.out_type == 0u ? detail::unpack2<__half>(w.x) : detail::unpack2<__nv_bfloat16>(w.x);
        const float2 hi = p.out_type == 0u ? detail::unpack2<__half>(w.y) : detail::unpack2<__nv_bfloat16>(w.y);
        t[0] = lo.x;
        t[1] = lo.y;
        t[2] = hi.x;
        t[3] = hi.y;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = static_cast<uint32_t>(i) < have ? detail::mx_load_c(p, at + i) : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = fmaf(p.beta, t[i], f[i]);
    }
    if (p.epi_flags & 1u) {
      detail::mx_load4(p.bias + col, have, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] += t[i];
    }
    detail::activate_all(f, p.act);
  }
  if (!live) return;
  const int64_t at = static_cast<int64_t>(row) * p.ldd + col;
  if (p.out_type == 2u) {
    float* d = static_cast<float*>(p.d) + at;
    if (vec) {
      *reinterpret_cast<float4*>(d) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (static_cast<uint32_t>(i) < have) d[i] = f[i];
    }
  } else {
    uint2 w;
    w.x = p.out_type == 0u ? detail::pack2<__half>(f[0], f[1]) : detail::pack2<__nv_bfloat16>(f[0], f[1]);
    w.y = p.out_type == 0u ? detail::pack2<__half>(f[2], f[3]) : detail::pack2<__nv_bfloat16>(f[2], f[3]);
    uint16_t* d = static_cast<uint16_t*>(p.d) + at;
    if (vec) {
      *reinterpret_cast<uint2*>(d) = w;
    } else {
      const uint32_t h[2] = {w.x, w.y};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (static_cast<uint32_t>(i) < have) d[i] = static_cast<uint16_t>(h[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// Quantised output of a swapped tile: the scale rows from m up to the next multiple of 128 are zero.
// `row` is one of the tile's 128 in its one (e8m0) or two (e4m3) scale tiles.
__device__ __forceinline__ void mx_clear_scale_row(const MxParams& p, uint32_t tm, uint32_t row) {
  if (p.out_type < MX_OUT_FP4 || row < p.m) return;
  const uint32_t words = p.out_type == MX_OUT_NVFP4 ? 2u : 1u;
  for (uint32_t w = 0; w < words; ++w) {
    const int64_t g = static_cast<int64_t>(tm) * words + w;
    if (g < p.d_groups && GZ_MX_SCALE_OK(p, row, 4 * g, 4u)) *reinterpret_cast<uint32_t*>(p.d_scales + mx::scale_word(row, g, p.d_groups)) = 0u;
  }
}

// 32 columns of one row (lane = row) of a row tile, from the sums x (gated: and y) to the output.  c holds
// the words of C for these columns on entry and those for next_col0 on return (C_ROWS: see mx_load_c_rows).
template <class Cfg, bool C_ROWS>
__device__ __forceinline__ void mx_finish_slice(const MxParams& p, const void* tm_d, uint32_t stg, uint32_t lane,
                                                const uint32_t (&x)[32], const uint32_t (&y)[32], uint32_t (&c)[32],
                                                uint32_t row0, uint32_t col0, uint32_t next_col0, uint32_t& turn) {
  float f[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) f[i] = p.alpha * __uint_as_float(x[i]);
  if constexpr (Cfg::GATED) {
    detail::activate_all(f, p.act);
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] *= p.alpha_up * __uint_as_float(y[i]);
    if (p.out_type >= MX_OUT_FP4) {
      if (row0 < ((p.m + 127u) & ~127u)) {  // rows up to the next multiple of 128 have scales
        if (p.out_type == MX_OUT_FP4) detail::mx_store_quantized<false>(p, f, row0 + lane, col0);
        else detail::mx_store_quantized<true>(p, f, row0 + lane, col0);
      }
      return;
    }
    if (row0 >= p.m || col0 >= p.n) return;
  } else {
    if (row0 >= p.m || col0 >= p.n) {
      detail::mx_load_c_box<C_ROWS>(p, row0, next_col0, lane, c);  // the first group of an even tile may lie outside
      return;
    }
    if (p.epi_flags != 0u || p.beta != 0.0f || p.act != 0u) {
      detail::mx_row_terms<C_ROWS>(p, f, c, stg, row0 + lane, col0, lane);
      detail::mx_load_c_box<C_ROWS>(p, row0, next_col0, lane, c);
    }
  }
  detail::mx_store_box(p, tm_d, stg, lane, f, row0, col0, turn);
}

// What it measured (CUDA-graph replays over rotating operands, one B200): 8192^3, e8m0, bf16 out: 188 to 195 us, 5.6 to
// 5.8 PFLOP/s, the tensor pipe busy 81 % of the cycles at a clock that the power limit holds at 1.3 to 1.55 GHz.  Two thousand
// rows x 14336 x 4096, e4m3: product 51, + C 58, gated 93 us: tensor-bound, with the last wave of tiles partly empty.
// One row x 14336 x 4096: product 9.5 us, gated 13.5 us: B at the copy rate (5.0, 9.5) and about 4 us of a launch's two ends.
template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, Cfg::PER_SM)
mx_gemm_kernel(const __grid_constant__ MxMaps maps, const MxParams p) {
  constexpr int CTAS = Cfg::CTAS, STAGES = Cfg::STAGES, BN = Cfg::BN, MB = Cfg::MB;
  constexpr bool NV = Cfg::NV, SWAP = Cfg::SWAP, GATED = Cfg::GATED;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - raw_addr);
  const uint32_t staging_base = base + Cfg::RING_BYTES;
  const uint32_t bars = staging_base + Cfg::STAGING_BYTES;
  auto full_bar = [&](uint32_t s) { return bars + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bars + 8u * (STAGES + s); };
  const uint32_t acc_full_bar = bars + 8u * (2 * STAGES), acc_empty_bar = acc_full_bar + 8u;
  const uint32_t drain_bar = acc_full_bar + 16u;
  uint32_t* const tmem_slot =
      reinterpret_cast<uint32_t*>(smem + Cfg::RING_BYTES + Cfg::STAGING_BYTES + 8 * (2 * STAGES + 3));
  uint32_t* const abort_flag = tmem_slot + 1;

  const uint32_t warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t crank = ptx::cluster_ctarank();
  const uint32_t rank = CTAS == 2 ? (crank & 1u) : 0u;  // within the pair
  const uint32_t part = CTAS == 2 ? crank >> 1 : crank;  // which share of a tile's K range
  const uint32_t leader = CTAS == 2 ? (crank & ~1u) : crank;
  const uint32_t cluster = ptx::cluster_id_x(), num_clusters = ptx::num_clusters_x();
  const detail::Abort ab{abort_flag, p.status, p.wait_limit_ns};

  // ------------------------------------------------------------ set-up (as in sm100_gemm.cuh)
  if (warp == 0) {
    if (lane == 31u) ptx::prefetch_tensormap(&maps.wide);
    if (lane == 30u) ptx::prefetch_tensormap(&maps.wide_scales);
    if (lane == 29u && p.out_tma) ptx::prefetch_tensormap(&maps.d);
    for (uint32_t s = lane; s < STAGES; s += 32u) {
      ptx::mbar_init(full_bar(s), 2);
      ptx::mbar_init(empty_bar(s), 1);
    }
    if (lane == 0u) {
      ptx::mbar_init(acc_full_bar, 1);
      ptx::mbar_init(acc_empty_bar, Cfg::EPI_WARPS * CTAS);
      ptx::mbar_init(drain_bar, 1);
      *abort_flag = 0u;
    }
    ptx::fence_mbar_init_cluster();
    __syncwarp();
    ptx::named_barrier_arrive(2, 64);
    ptx::named_barrier_arrive(3, Cfg::THREADS - 32);
    if constexpr (CTAS == 2) ptx::cluster_arrive_release();
  } else if (warp == 6) {
    if (lane == 0) ptx::prefetch_tensormap(&maps.narrow);
    if (lane == 1) ptx::prefetch_tensormap(&maps.narrow_scales);
    if (GATED && lane == 2) ptx::prefetch_tensormap(&maps.up);
    if (GATED && lane == 3) ptx::prefetch_tensormap(&maps.up_scales);
    if constexpr (CTAS == 2) ptx::cluster_arrive_release();
    ptx::named_barrier_sync(2, 64);
  } else {
    if constexpr (CTAS == 2) ptx::cluster_arrive_release();
    if (warp == 1) {
      ptx::tmem_alloc<CTAS>(ptx::smem_u32(tmem_slot), Cfg::TMEM_COLS);
      ptx::tmem_relinquish<CTAS>();
    }
    ptx::tc_fence_before_sync();
    ptx::named_barrier_sync(3, Cfg::THREADS - 32);
    ptx::tc_fence_after_sync();
  }
  if constexpr (CTAS == 2) ptx::cluster_wait_acquire();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  ptx::grid_launch_dependents();

  // The K blocks that are this CTA's (pair's).  The tiles: a swapped CTA has one; a row-tile cluster that
  // shares K ranges has one; otherwise a cluster is a CTA (pair) that walks tiles in steps of the grid.
  uint32_t kb_lo = 0, kb_hi = p.k_blocks;
  if (p.split > 1u) {
    kb_lo = static_cast<uint32_t>(static_cast<uint64_t>(part) * p.k_blocks / p.split);
    kb_hi = static_cast<uint32_t>(static_cast<uint64_t>(part + 1u) * p.k_blocks / p.split);
  }

  if (warp == 0 || warp == 6) {
    // ---------------------------------------------------------- TMA producers
    // Warp 0: the wide operand and its scales; warp 6: the narrow one.
    const bool is_narrow = warp == 6;
    const uint32_t my_bytes = is_narrow ? Cfg::N_BYTES + Cfg::NS_BYTES : Cfg::W_BYTES + Cfg::WS_BYTES;
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    // A swapped tile's first K blocks are brought into L2 while the kernel before this one finishes.  Nothing
    // is read yet: whatever that kernel still writes to these lines is written to them in L2.
    if constexpr (SWAP) {
      const uint32_t nkb = kb_hi - kb_lo;
      if (lane < (nkb < p.prefetch ? nkb : p.prefetch) && cluster < p.grid.num_tiles) {
        const uint32_t at = kb_lo + (lane + cluster * 5u) % nkb;
        const int32_t kx = static_cast<int32_t>(at * 128u), kt = static_cast<int32_t>(at * Cfg::TILES_K);
        const int32_t rb = static_cast<int32_t>(cluster);
        if (is_narrow) {
          ptx::tma_prefetch_3d(&maps.narrow, kx, 0, 0);
          ptx::tma_prefetch_3d(&maps.narrow_scales, 0, kt, 0);
        } else {
          ptx::tma_prefetch_3d(&maps.wide, kx, rb * 128, 0);
          ptx::tma_prefetch_3d(&maps.wide_scales, 0, kt, rb);
          if constexpr (MB == 2) {
            ptx::tma_prefetch_3d(&maps.up, kx, rb * 128, 0);
            ptx::tma_prefetch_3d(&maps.up_scales, 0, kt, rb);
          }
        }
      }
      __syncwarp();
    }
    ptx::grid_dependency_wait();
    for (uint32_t t = cluster; ok && t < p.grid.num_tiles; t += num_clusters) {
      uint32_t tm, tn;
      tile_coords(p.grid, t, tm, tn);
      const int32_t wide_rb = static_cast<int32_t>(tm * CTAS + rank);
      // Swapped tiles stream B once: they start at different K blocks, or all CTAs would read addresses a
      // multiple of the row pitch apart, which load the HBM channels unevenly.
      const uint32_t rot = SWAP ? (t * 5u) % (kb_hi - kb_lo) : 0u;
      for (uint32_t kb = kb_lo; kb < kb_hi; ++kb) {
        ok = __all_sync(0xFFFFFFFFu, detail::wait(empty_bar(stage), phase ^ 1u, ab, WAIT_PRODUCER_EMPTY, t, kb));
        if (!ok) break;
        if (ptx::elect_one()) {
          const uint32_t dst = base + stage * Cfg::STAGE_BYTES;
          uint32_t at = kb + rot;  // K block fetched in this step
          if (at >= kb_hi) at -= kb_hi - kb_lo;
          const int32_t kx = static_cast<int32_t>(at * 128u);
          const int32_t kt = static_cast<int32_t>(at * Cfg::TILES_K);
          uint32_t fb = full_bar(stage);
          if constexpr (CTAS == 1) {
            ptx::mbar_arrive_expect_tx(fb, my_bytes);
          } else {
            if (rank == 0) ptx::mbar_arrive_expect_tx(fb, 2u * my_bytes);
            fb = ptx::mapa(fb, leader);
          }
          auto load = [&](uint32_t to, const void* map, int32_t c0, int32_t c1, int32_t c2) {
            if constexpr (CTAS == 1) ptx::tma_load_3d(to, map, c0, c1, c2, fb);
            else ptx::tma_load_3d_pair(to, map, c0, c1, c2, fb);
          };
          const uint32_t ws = dst + Cfg::W_BYTES + Cfg::N_BYTES, ns = ws + Cfg::WS_BYTES;
          if (!is_narrow) {
            load(dst, &maps.wide, kx, wide_rb * 128, 0);
            load(ws, &maps.wide_scales, 0, kt, wide_rb);
            if constexpr (MB == 2) {
              load(dst + 128u * 128u, &maps.up, kx, wide_rb * 128, 0);
              load(ws + Cfg::TILES_K * 512u, &maps.up_scales, 0, kt, wide_rb);
            }
          } else if constexpr (!SWAP) {
            const uint32_t nd = dst + Cfg::W_BYTES;
            if constexpr (BN == 256) {
              // 256 rows as two groups of 128: rows of B, or the gate's and the up projection's
              const int32_t rb0 = static_cast<int32_t>(GATED ? tn : tn * 2u), rb1 = GATED ? rb0 : rb0 + 1;
              const CUtensorMap* const second = GATED ? &maps.up : &maps.narrow;
              const CUtensorMap* const second_scales = GATED ? &maps.up_scales : &maps.narrow_scales;
              if (CTAS == 1 || rank == 0u) load(nd, &maps.narrow, kx, rb0 * 128, 0);
              if (CTAS == 1) load(nd + 128u * 128u, second, kx, rb1 * 128, 0);
              else if (rank == 1u) load(nd, second, kx, rb1 * 128, 0);
              load(ns, &maps.narrow_scales, 0, kt, rb0);
              load(ns + Cfg::TILES_K * 512u, second_scales, 0, kt, rb1);
            } else {
              load(nd, &maps.narrow, kx, static_cast<int32_t>(tn * BN + rank * (BN / CTAS)), 0);
              load(ns, &maps.narrow_scales, 0, kt, static_cast<int32_t>(tn * BN / 128u));
            }
          } else {
            load(dst + Cfg::W_BYTES, &maps.narrow, kx, 0, 0);
            load(ns, &maps.narrow_scales, 0, kt, 0);
          }
        }
        __syncwarp();
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok && rank == 0 && lane == 0) {
      // Aborting: give loads already issued a bounded chance to land (see sm100_gemm.cuh).
      const uint64_t t0 = ptx::globaltimer_ns();
      for (uint32_t i = 0; i < STAGES; ++i) {
        const uint32_t s = (stage + STAGES - 1u - i) % STAGES;
        const uint32_t ph = (s < stage) ? phase : (phase ^ 1u);
        while (!ptx::mbar_try_wait(full_bar(s), ph)) {
          if (ptx::globaltimer_ns() - t0 > 2000000ull) break;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    ptx::grid_dependency_wait();
    if (rank == 0) {
      uint32_t stage = 0, phase = 0, it = 0, slot = 0;
      bool ok = true, issued = false;
      // Shared-memory descriptors: codes in 128-byte-swizzled rows (8 rows = 1024 bytes); scales as
      // 32 rows of 16 bytes, 8 rows = 128 bytes, unswizzled.
      const uint64_t code_hi = static_cast<uint64_t>((1024u >> 4) | (1u << 14) | (2u << 29)) << 32 | (1u << 16);
      const uint64_t scale_hi = static_cast<uint64_t>((128u >> 4) | (1u << 14)) << 32 | ((128u >> 4) << 16);
      for (uint32_t t = cluster; ok && t < p.grid.num_tiles; t += num_clusters, ++it) {
        ok = __all_sync(0xFFFFFFFFu, detail::wait(acc_empty_bar, (it & 1u) ^ 1u, ab, WAIT_MMA_TMEM_EMPTY, t, 0));
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + (SWAP ? 0u : (it & 1u) * Cfg::ACC_STRIDE);
        for (uint32_t kb = kb_lo; kb < kb_hi; ++kb) {
          ok = __all_sync(0xFFFFFFFFu, detail::wait(full_bar(stage), phase, ab, WAIT_MMA_FULL, t, kb));
          if (!ok) break;
          ptx::tc_fence_after_sync();
          if (ptx::elect_one()) {
            const uint32_t st = base + stage * Cfg::STAGE_BYTES;
            const uint32_t ws = st + Cfg::W_BYTES + Cfg::N_BYTES, ns = ws + Cfg::WS_BYTES;
            const uint64_t wd = code_hi | ((st >> 4) & 0x3FFFu), nd = code_hi | (((st + Cfg::W_BYTES) >> 4) & 0x3FFFu);
#pragma unroll
            for (uint32_t a = 0; a < static_cast<uint32_t>(Cfg::TILES_K); ++a) {
              const uint32_t sf = tmem_base + Cfg::ACC_COLS + ((slot + a) & 3u) * Cfg::SLOT_COLS;
#pragma unroll
              for (uint32_t mb = 0; mb < static_cast<uint32_t>(MB); ++mb)
                ptx::tmem_copy_scales<CTAS>(sf + mb * 4u, scale_hi | (((ws + (mb * Cfg::TILES_K + a) * 512u) >> 4) & 0x3FFFu));
#pragma unroll
              for (uint32_t rb = 0; rb < static_cast<uint32_t>(Cfg::NRB); ++rb)
                ptx::tmem_copy_scales<CTAS>(sf + 8u + rb * 4u, scale_hi | (((ns + (rb * Cfg::TILES_K + a) * 512u) >> 4) & 0x3FFFu));
              constexpr uint32_t STEPS = 4 / Cfg::TILES_K;  // MMAs per scale tile
#pragma unroll
              for (uint32_t j = 0; j < STEPS; ++j) {
                // which of the four scales of a row this step starts at (two per step for e8m0)
                const uint32_t idesc = p.idesc | (j * 2u) << 4 | (j * 2u) << 29;
                const uint32_t step = a * STEPS + j;
#pragma unroll
                for (uint32_t mb = 0; mb < static_cast<uint32_t>(MB); ++mb)
                  ptx::umma_mx<NV, CTAS>(d_tmem + mb * BN, wd + step * 2u + mb * ((128u * 128u) >> 4), nd + step * 2u,
                                         idesc, sf + mb * 4u, sf + 8u, (kb != kb_lo || step != 0u) ? 1u : 0u);
              }
            }
            ptx::tc_commit<CTAS>(empty_bar(stage));
            if constexpr (CTAS == 2) ptx::tc_commit<CTAS>(ptx::mapa(empty_bar(stage), crank | 1u));
          }
          __syncwarp();
          issued = true;
          slot = (slot + Cfg::TILES_K) & 3u;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (!(p.test_flags & 1u) && ptx::elect_one()) {
          ptx::tc_commit<CTAS>(acc_full_bar);
          if constexpr (CTAS == 2) ptx::tc_commit<CTAS>(ptx::mapa(acc_full_bar, crank | 1u));
        }
        __syncwarp();
      }
      if ((!ok || (p.test_flags & 1u)) && issued && lane == 0) {
        ptx::tc_commit<CTAS>(drain_bar);
        const uint64_t t0 = ptx::globaltimer_ns();
        while (!ptx::mbar_try_wait(drain_bar, 0)) {
          if (ptx::globaltimer_ns() - t0 > 2000000ull) break;
        }
      }
    }
  } else {
    // ---------------------------------------------------------- epilogue
    ptx::grid_dependency_wait();
    const uint32_t quad = warp & 3u;
    const uint32_t lanes = tmem_base + ((quad * 32u) << 16);
    if constexpr (SWAP) {
      // The accumulator's columns are output rows, its lanes output columns: [operand][row][128 columns].
      const uint32_t park = base + (quad * 32u + lane) * 4u;
      const uint32_t mine = base + lane * 16u;
      uint32_t tm, tn;
      tile_coords(p.grid, cluster, tm, tn);
      const uint32_t col = tm * 128u + lane * 4u;
      bool live = false;  // the first round is the dry one
      for (uint32_t r = part + p.split * quad;;) {
        float f[4] = {}, u[4] = {};
        if (live) {
          if (r >= p.m) break;
          if (p.split == 1u) {
            ptx::ld_shared_f32x4(mine + r * 512u, f);
            if constexpr (GATED) ptx::ld_shared_f32x4(mine + (BN + r) * 512u, u);
          } else {
            // up to four peers' loads in flight; the sums are taken in rank order
            for (uint32_t q = 0; q < p.split; q += 4u) {
              float x[4][4], y[4][4];
#pragma unroll
              for (uint32_t e = 0; e < 4; ++e) {
                if (q + e < p.split) {
                  const uint32_t at = ptx::mapa(mine, q + e) + r * 512u;
                  ptx::ld_cluster_f32x4(at, x[e]);
                  if constexpr (GATED) ptx::ld_cluster_f32x4(at + BN * 512u, y[e]);
                }
              }
#pragma unroll
              for (uint32_t e = 0; e < 4; ++e) {
                if (q + e < p.split) {
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    f[i] = q + e == 0u ? x[e][i] : f[i] + x[e][i];
                    if constexpr (GATED) u[i] = q + e == 0u ? y[e][i] : u[i] + y[e][i];
                  }
                }
              }
            }
          }
        }
        if (r < p.m) mx_finish_row<Cfg>(p, f, u, r, col, lane, live);
        if (live) {
          r += p.split * 4u;
          continue;
        }
        live = true;
        const bool ok = __all_sync(0xFFFFFFFFu, detail::wait(acc_full_bar, 0, ab, WAIT_EPILOGUE_TMEM_FULL, cluster, 0));
        if (ok) {
          ptx::tc_fence_after_sync();
#pragma unroll 1
          for (uint32_t sl = 0; sl * 16u < p.m; ++sl) {
            uint32_t x[MB][16];
#pragma unroll
            for (uint32_t mb = 0; mb < static_cast<uint32_t>(MB); ++mb) ptx::tmem_ld_32x16(lanes + mb * BN + sl * 16u, x[mb]);
            ptx::tmem_wait_ld();
#pragma unroll
            for (uint32_t mb = 0; mb < static_cast<uint32_t>(MB); ++mb) {
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i)
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(park + (mb * BN + sl * 16u + i) * 512u), "r"(x[mb][i]) : "memory");
            }
          }
          ptx::tc_fence_before_sync();
        }
        if (p.split > 1u) {
          __syncwarp();
          ptx::cluster_arrive_release();
          ptx::cluster_wait_acquire();
        } else {
          ptx::named_barrier_sync(1, 128);
        }
        if (!ok || detail::aborted(ab)) break;
      }
      if constexpr (GATED) {
        if (part == 0u && !detail::aborted(ab)) mx_clear_scale_row(p, tm, quad * 32u + lane);
      }
    } else {
      const uint32_t half = warp >= 7u ? 1u : 0u;
      const uint32_t stg = staging_base + (half * 4u + quad) * 4096u;
      constexpr uint32_t TILE_COLS = GATED ? BN / 2u : BN;  // output columns
      constexpr uint32_t GROUPS = TILE_COLS / 64u;          // of 64; this warp's half of each is 32 wide
      uint32_t turn = 0;
      // One of two copies runs: one loop for both ways of reading C costs the aligned one (2048 x 14336 x 4096 fp16: 57 -> 62 us).
      auto finish_tiles = [&](auto by_rows) {
      constexpr bool C_ROWS = decltype(by_rows)::value;
      if (p.split <= 1u) {
        const uint32_t release = ptx::mapa(acc_empty_bar, leader);
        uint32_t it = 0;
        for (uint32_t t = cluster; t < p.grid.num_tiles; t += num_clusters, ++it) {
          uint32_t tm, tn;
          tile_coords(p.grid, t, tm, tn);
          const uint32_t row0 = (tm * CTAS + rank) * 128u + quad * 32u;
          const uint32_t tile_col = tn * TILE_COLS + half * 32u;
          // the group that the next tile's accumulator overlaps comes first
          auto group_col = [&](uint32_t s) { return tile_col + ((it & 1u) ? s : (s + GROUPS - 1u) % GROUPS) * 64u; };
          uint32_t c[32];
          if constexpr (!GATED) detail::mx_load_c_box<C_ROWS>(p, row0, group_col(0), lane, c);
          if (!__all_sync(0xFFFFFFFFu, detail::wait(acc_full_bar, it & 1u, ab, WAIT_EPILOGUE_TMEM_FULL, t, 0))) break;
          ptx::tc_fence_after_sync();
          const uint32_t acc = lanes + (it & 1u) * Cfg::ACC_STRIDE;
#pragma unroll 1
          for (uint32_t s = 0; s < GROUPS; ++s) {
            const uint32_t col0 = group_col(s), off = col0 - tile_col + half * 32u;
            uint32_t x[32], y[32];
            ptx::tmem_ld_32x32(acc + off, x);
            if constexpr (GATED) ptx::tmem_ld_32x32(acc + BN / 2u + off, y);
            ptx::tmem_wait_ld();
            if (s == 0) {
              ptx::tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive_cluster(release);
            }
            mx_finish_slice<Cfg, C_ROWS>(p, &maps.d, stg, lane, x, y, c, row0, col0, s + 1u < GROUPS ? group_col(s + 1u) : p.n, turn);
          }
          // one release per tile, made above; the rest of this tile's columns are read before the next
          // tile's release, which is what the tile after that waits for
          ptx::tc_fence_before_sync();
        }
      } else {
        // The cluster's one tile.  Partial sums lie as [four columns][128 rows][4]: a lane writes or reads 16
        // bytes, a warp 512 in a row.
        uint32_t tm, tn;
        tile_coords(p.grid, cluster, tm, tn);
        const uint32_t row0 = (tm * CTAS + rank) * 128u + quad * 32u;
        const uint32_t mine = base + (quad * 32u + lane) * 16u;
        const bool ok = __all_sync(0xFFFFFFFFu, detail::wait(acc_full_bar, 0, ab, WAIT_EPILOGUE_TMEM_FULL, cluster, 0));
        if (ok) {
          ptx::tc_fence_after_sync();
#pragma unroll 1
          for (uint32_t g = 0; g < BN / 64u; ++g) {
            const uint32_t off = g * 64u + half * 32u;
            uint32_t x[32];
            ptx::tmem_ld_32x32(lanes + off, x);
            ptx::tmem_wait_ld();
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + (off / 4u + i) * 2048u), "r"(x[4 * i]),
                           "r"(x[4 * i + 1]), "r"(x[4 * i + 2]), "r"(x[4 * i + 3])
                           : "memory");
          }
          ptx::tc_fence_before_sync();
        }
        __syncwarp();
        ptx::cluster_arrive_release();
        ptx::cluster_wait_acquire();
        if (ok && !detail::aborted(ab)) {
          // The tile's 32-column slices are dealt to the parts in order; a slice is finished by the warps of
          // one half, as without a shared K range.
          constexpr uint32_t SLICES = TILE_COLS / 32u;
          for (uint32_t sl = part * SLICES / p.split; sl < (part + 1u) * SLICES / p.split; ++sl) {
            if ((sl & 1u) != half) continue;
            const uint32_t col0 = tn * TILE_COLS + sl * 32u;
            uint32_t x[32], y[32], c[32];
            if constexpr (!GATED) detail::mx_load_c_box<C_ROWS>(p, row0, col0, lane, c);
            for (uint32_t q = 0; q < p.split; ++q) {
              const uint32_t peer = ptx::mapa(mine, CTAS == 2 ? q * 2u + rank : q) + sl * (8u * 2048u);
#pragma unroll
              for (uint32_t mb = 0; mb < (GATED ? 2u : 1u); ++mb) {
                float v[8][4];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) ptx::ld_cluster_f32x4(peer + (mb * (BN / 8u) + i) * 2048u, v[i]);
                uint32_t(&sum)[32] = mb == 0u ? x : y;
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  sum[i] = __float_as_uint(q == 0u ? v[i / 4][i % 4] : __uint_as_float(sum[i]) + v[i / 4][i % 4]);
              }
            }
            mx_finish_slice<Cfg, C_ROWS>(p, &maps.d, stg, lane, x, y, c, row0, col0, p.n, turn);
          }
        }
      }
      };
      if (!GATED && p.beta != 0.0f && !p.c_vec_ok) finish_tiles(std::integral_constant<bool, !GATED>{});
      else finish_tiles(std::false_type{});
      if (p.out_tma && lane == 0) ptx::bulk_wait_group_read<0>();
    }
  }
  if (p.split > 1u) {
    // The epilogue warps have met their peers once, when the partial sums were in place.
    __syncwarp();
    if (warp < 2u || warp == 6u) {
      ptx::cluster_arrive_release();
      ptx::cluster_wait_acquire();
    }
    ptx::cluster_arrive_release();  // nobody leaves while a peer may still read its partial sums
    ptx::cluster_wait_acquire();
  }

  // -------------------------------------------------------------- teardown (as in sm100_gemm.cuh)
  __syncwarp();
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::grid_dependency_wait();
  if (detail::aborted(ab)) {
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 100000ull) __nanosleep(1000);
  }
  if constexpr (CTAS == 2) {
    ptx::cluster_arrive_release();
    ptx::cluster_wait_acquire();
  }
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<CTAS>(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace gz
#endif
