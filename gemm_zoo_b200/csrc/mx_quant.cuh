// Quantisation to the microscaled 4-bit formats and its inverse (include/gemmzoo/microscale.h).
//
// Both are one pass over memory: a block's scale needs its largest magnitude, which a thread (or
// two neighbouring ones) holds in registers, so a value is read once and its code written once.  HBM bounds
// them from some 10 MB on.  Measured as CUDA-graph replays (quantise, decode; share of the measured copy rate):
//   16384 x 4096 bf16, e8m0                28.7 us (90 %), 28.4 us (91 %)
//   14336 x 4096 fp32, e4m3, K contiguous  41.7 us (98 %), 40.6 us (100 %)
//   14336 x 4096 fp32, e4m3, K strided     46.3 us (88 %), 45.6 us (90 %)
//   14336 x 4096 bf16, e4m3, K strided     34.3 us (67 %), 29.8 us (77 %): 76 % of the quantiser's issue slots are taken
#ifndef GZ_MX_QUANT_CUH
#define GZ_MX_QUANT_CUH

#include <cuda_bf16.h>

#include <type_traits>

#include "mx_format.cuh"
#include "ptx.cuh"

namespace gz {
namespace mx {

struct QuantParams {
  const void* in;  // quantise: the values; dequantise: unused
  void* out;       // dequantise: the values
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows, k, ld, pitch;
  int64_t code_bytes;  // of a row: round_up(k, 32) / 2
  int64_t groups;      // scale tiles per 128 rows
  // Row layout: a block takes `block_rows` rows x `row_threads` 16-element chunks (a whole number of
  // scale words); inv_threads = ceil(65536 / row_threads) divides a thread index by row_threads.
  uint32_t row_threads, inv_threads, block_rows;
  uint32_t vec;   // bytes that an access to the values may have: 32, 16, or 0 (single values)
  uint32_t unit;  // multiplier == 1
  float multiplier;
  float pre;  // decode: a power of two that the scale is multiplied by first (`multiplier` has been divided by it)
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 32 bytes at a 32-byte aligned address.  What is quantised is read once and what is decoded written once, so
// both may leave the L2 first: quantise and decode in turn 16384 x 4096 bf16 57.7 -> 53.4 us; 14336 x 4096 fp32
// with K strided 113 -> 96 (16-byte accesses with the same hint: 101).
__device__ __forceinline__ void load32(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.L1::no_allocate.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.L1::no_allocate.L2::evict_first.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Largest magnitude among 16 values held as raw bits, as raw bits (of one value): without their signs
// the numbers order like integers, NaN above infinity.
template <typename T>
__device__ __forceinline__ float amax_raw(const uint32_t* w) {
  uint32_t m = 0;
  if constexpr (sizeof(T) == 2) {
    uint32_t a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = w[i] & 0x7FFF7FFFu;
    m = __vimax3_u16x2(__vimax3_u16x2(a[0], a[1], a[2]), __vimax3_u16x2(a[3], a[4], a[5]), __vimax3_u16x2(a[6], a[7], 0u));
    m = max(m & 0xFFFFu, m >> 16);
    const uint16_t h = static_cast<uint16_t>(m);
    return to_float<T>(*reinterpret_cast<const T*>(&h));
  } else {
#pragma unroll
    for (int i = 0; i < 16; i += 2) m = __vimax3_u32(m, w[i] & 0x7FFFFFFFu, w[i + 1] & 0x7FFFFFFFu);
    return __uint_as_float(m);
  }
}

// Value i of a row of raw words.
template <typename T>
__device__ __forceinline__ float value_of(const uint32_t* w, int i) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float((i & 1) ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  else {
    const uint16_t h = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
    return __half2float(*reinterpret_cast<const __half*>(&h));
  }
}

// 16 raw values of one row -> their 8 bytes of codes; `scale` receives the byte of their block.  An e8m0
// block is shared with the neighbouring lane (`mask`: the lanes that call).  The largest magnitude is
// taken before the multiplier, which rounding, being monotone, allows.
template <typename T, bool NV>
__device__ __forceinline__ uint2 encode16(const uint32_t* w, const QuantParams& p, uint32_t mask, uint32_t& scale) {
  float amax = amax_raw<T>(w) * fabsf(p.multiplier);
  if constexpr (!NV) amax = amax_nan(amax, __shfl_xor_sync(mask, amax, 1));
  const Scale s = block_scale<NV>(amax);
  float v[16];
  if (p.unit) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = in_code_units<NV>(value_of<T>(w, i), s);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = in_code_units<NV>(value_of<T>(w, i) * p.multiplier, s);
  }
  uint2 codes;
  codes.x = pack8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
  codes.y = pack8(v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]);
  if (s.byte == Format<NV>::NAN_SCALE) codes = make_uint2(0u, 0u);
  scale = s.byte;
  return codes;
}

// The four scales of a word, put together among the lanes that hold them; valid in all of them.
// `in_word` counts the lanes from the word's first one.
template <bool NV>
__device__ __forceinline__ uint32_t gather_word(uint32_t byte, uint32_t in_word, uint32_t mask) {
  constexpr int PER_WORD = NV ? 4 : 8;
  uint32_t word = byte << (8 * (NV ? in_word : in_word / 2));
#pragma unroll
  for (int d = PER_WORD / 4; d < PER_WORD; d *= 2) word |= __shfl_xor_sync(mask, word, d);
  return word;
}

// A block's part of the row layout: piece of the row's chunks, first row.
__device__ __forceinline__ bool row_item(const QuantParams& p, int64_t& row, int64_t& chunk, int rows_per_thread) {
  const uint32_t in = (threadIdx.x * p.inv_threads) >> 16;  // row of the block; exact for indexes below 256
  const int64_t piece = static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y;
  row = static_cast<int64_t>(blockIdx.x) * p.block_rows * rows_per_thread + in;
  chunk = piece * p.row_threads + (threadIdx.x - in * p.row_threads);
  return in < p.block_rows;
}

// Rows with K contiguous.  A thread takes 16 consecutive elements (32 bytes of a 16-bit type in one
// load) of two rows, both loads before any arithmetic; 16 elements are one e4m3 block or half of an e8m0
// block.  The lanes that share a 4-byte word of scales are neighbours, so amax and the word are put
// together with shuffles.  Rows beyond the last up to the next multiple of 128 exist in the scale array
// only and get zero bytes.
constexpr int ROWS_PER_THREAD = 2;
template <typename T, bool NV>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p) {
  constexpr int PER_WORD = NV ? 4 : 8;  // lanes whose blocks share a word of scales
  constexpr int WORDS = 4 * sizeof(T);  // of 16 values
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  int64_t row0, chunk;
  const bool mine = row_item(p, row0, chunk, ROWS_PER_THREAD) && chunk / PER_WORD < p.groups;
  // Every thread of the block gets here.  The lanes that go on are whole words of scales: row_threads is a multiple of PER_WORD.
  const uint32_t mask = __ballot_sync(0xFFFFFFFFu, mine);
  if (!mine) return;
  const int64_t k0 = chunk * 16;
  uint32_t w[ROWS_PER_THREAD][WORDS];
#pragma unroll
  for (int r = 0; r < ROWS_PER_THREAD; ++r) {
    const int64_t row = row0 + r * p.block_rows;
    const T* src = static_cast<const T*>(p.in) + row * p.ld + k0;
    if (row < p.rows && k0 + 16 <= p.k && p.vec == 32u) {
#pragma unroll
      for (int l = 0; l < WORDS / 8; ++l) load32(src + l * (32 / sizeof(T)), *reinterpret_cast<uint32_t(*)[8]>(&w[r][8 * l]));
    } else if (row < p.rows && k0 + 16 <= p.k && p.vec == 16u) {
#pragma unroll
      for (int l = 0; l < WORDS / 4; ++l)
        *reinterpret_cast<uint4*>(&w[r][4 * l]) = *reinterpret_cast<const uint4*>(src + l * (16 / sizeof(T)));
    } else {
      T e[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = (row < p.rows && k0 + i < p.k) ? src[i] : from_float<T>(0.0f);
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[r][i] = reinterpret_cast<const uint32_t*>(e)[i];
    }
  }
  const int64_t rows_padded = (p.rows + 127) & ~static_cast<int64_t>(127);
#pragma unroll
  for (int r = 0; r < ROWS_PER_THREAD; ++r) {
    const int64_t row = row0 + r * p.block_rows;
    uint32_t byte;
    const uint2 codes = encode16<T, NV>(w[r], p, mask, byte);
    if (row < p.rows && k0 / 2 < p.code_bytes) *reinterpret_cast<uint2*>(p.codes + row * p.pitch + k0 / 2) = codes;
    const uint32_t in_word = static_cast<uint32_t>(chunk) % PER_WORD;
    const uint32_t word = gather_word<NV>(row < p.rows ? byte : 0u, in_word, mask);
    if (in_word == 0 && row < rows_padded)
      *reinterpret_cast<uint32_t*>(p.scales + scale_word(row, chunk / PER_WORD, p.groups)) = word;
  }
}

// K strided: element k of row i at in[k * ld + i].  A block takes ROWS rows x 128 k through shared
// memory: filled along the rows (128 bytes per k), read along k.  A thread takes 16 k of two neighbouring
// rows (one 32- or 64-bit word of shared memory per k); eight threads side by side hold a row's 128 k, so
// that its 64 bytes of codes are written together.  The eight extra elements per 16 k put the
// eight threads' words in different banks.
constexpr int COL_K = 128;
template <typename T>
struct ColTile {
  static constexpr int ROWS = 128 / sizeof(T);
  static constexpr int THREADS = ROWS * 4;
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr int PER_LINE = ROWS / VEC;  // 16-byte pieces of a line
  static constexpr int PITCH = ROWS;
  static constexpr int ELEMS = ROWS * COL_K + 8 * 8;
  static __device__ __forceinline__ int at(int k, int row) { return k * PITCH + (k >> 4) * 8 + row; }
};

// WIDE: every line is 32-byte aligned, and whole tiles are read 32 bytes at a time.  A kernel of its own, because
// all three ways of reading in one need more registers (14340 x 4096 fp32, e4m3 blocks: 53 -> 61 us).
template <typename T, bool NV, bool WIDE>
__global__ void __launch_bounds__(ColTile<T>::THREADS) quantize_cols_kernel(const QuantParams p) {
  using Tile = ColTile<T>;
  __shared__ __align__(16) T tile[Tile::ELEMS];
  constexpr int LINES = COL_K * Tile::PER_LINE / Tile::THREADS;  // 16-byte pieces per thread
  constexpr int VEC = Tile::VEC;
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * Tile::ROWS;
  const int64_t k0 = (static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * COL_K;
  if (k0 >= p.k) return;
  const T* const src = static_cast<const T*>(p.in) + k0 * p.ld + row0;
  const int line = threadIdx.x / Tile::PER_LINE, piece = (threadIdx.x % Tile::PER_LINE) * VEC;
  constexpr int STEP = Tile::THREADS / Tile::PER_LINE;  // lines per pass
  uint4 w[LINES];
  const bool inside = k0 + COL_K <= p.k && row0 + Tile::ROWS <= p.rows;
  const int line2 = threadIdx.x / (Tile::PER_LINE / 2), piece2 = (threadIdx.x % (Tile::PER_LINE / 2)) * 2 * VEC;
  if (WIDE && inside) {
#pragma unroll
    for (int l = 0; l < LINES / 2; ++l)
      load32(src + static_cast<int64_t>(l * 2 * STEP + line2) * p.ld + piece2, *reinterpret_cast<uint32_t(*)[8]>(&w[2 * l]));
  } else if (!WIDE && p.vec && inside) {
#pragma unroll
    for (int l = 0; l < LINES; ++l)
      w[l] = __ldcs(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(l * STEP + line) * p.ld + piece));
  } else {
#pragma unroll
    for (int l = 0; l < LINES; ++l) {
      w[l] = make_uint4(0u, 0u, 0u, 0u);
      const int kk = l * STEP + line;
      if ((WIDE || p.vec) && k0 + kk < p.k) {
        const T* s = src + static_cast<int64_t>(kk) * p.ld + piece;
        if (row0 + piece + VEC <= p.rows) {
          w[l] = *reinterpret_cast<const uint4*>(s);
        } else {
          T* e = reinterpret_cast<T*>(&w[l]);
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (row0 + piece + i < p.rows) e[i] = s[i];
        }
      }
    }
  }
  if (WIDE && inside) {
    const bool swap = (threadIdx.x & 4u) != 0u;  // every other four lanes begin with their second piece: other banks
#pragma unroll
    for (int l = 0; l < LINES / 2; ++l) {
      T* const to = &tile[Tile::at(l * 2 * STEP + line2, piece2)];
      *reinterpret_cast<uint4*>(to + (swap ? VEC : 0)) = swap ? w[2 * l + 1] : w[2 * l];
      *reinterpret_cast<uint4*>(to + (swap ? 0 : VEC)) = swap ? w[2 * l] : w[2 * l + 1];
    }
  } else if (WIDE || p.vec) {
#pragma unroll
    for (int l = 0; l < LINES; ++l) *reinterpret_cast<uint4*>(&tile[Tile::at(l * STEP + line, piece)]) = w[l];
  } else {
    // single values, neighbouring lanes on neighbouring rows
    for (int i = threadIdx.x; i < Tile::ROWS * COL_K; i += Tile::THREADS) {
      const int kk = i / Tile::ROWS, r = i % Tile::ROWS;
      tile[Tile::at(kk, r)] = (k0 + kk < p.k && row0 + r < p.rows) ? src[static_cast<int64_t>(kk) * p.ld + r] : from_float<T>(0.0f);
    }
  }
  __syncthreads();
  const uint32_t c = threadIdx.x & 7u;                 // chunk of 16 k
  const int pair = static_cast<int>(threadIdx.x >> 3) * 2;  // first of the two rows
  uint32_t v[2][4 * sizeof(T)];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = *reinterpret_cast<const uint32_t*>(&tile[Tile::at(c * 16 + 2 * i, pair)]);
      const uint32_t b = *reinterpret_cast<const uint32_t*>(&tile[Tile::at(c * 16 + 2 * i + 1, pair)]);
      v[0][i] = __byte_perm(a, b, 0x5410);
      v[1][i] = __byte_perm(a, b, 0x7632);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint2 a = *reinterpret_cast<const uint2*>(&tile[Tile::at(c * 16 + i, pair)]);
      v[0][i] = a.x;
      v[1][i] = a.y;
    }
  }
  const int64_t rows_padded = (p.rows + 127) & ~static_cast<int64_t>(127);
  const int64_t at = k0 / 2 + c * 8;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t row = row0 + pair + r;
    uint32_t byte;
    const uint2 codes = encode16<T, NV>(v[r], p, 0xFFFFFFFFu, byte);
    if (row < p.rows && at < p.code_bytes) *reinterpret_cast<uint2*>(p.codes + row * p.pitch + at) = codes;
    constexpr uint32_t PER_WORD = NV ? 4 : 8;
    const uint32_t word = gather_word<NV>(row < p.rows ? byte : 0u, c % PER_WORD, 0xFFFFFFFFu);
    const int64_t g = NV ? k0 / 64 + c / 4 : k0 / 128;
    if (c % PER_WORD == 0 && row < rows_padded && g < p.groups)
      *reinterpret_cast<uint32_t*>(p.scales + scale_word(row, g, p.groups)) = word;
  }
}

// Dequantising: code * scale is exact in fp32; the product with the multiplier is rounded once there and
// once to T.  (6 * 2^127 is beyond fp32, though not what a small multiplier makes of it: `pre` takes such scales down by
// an exact 1/4.)
template <typename T, bool NV>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(const QuantParams p) {
  extern __shared__ __align__(16) uint8_t row_buffer[];  // 256 x 16 values where single values are stored, else none
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  int64_t row0, chunk;
  const bool mine = row_item(p, row0, chunk, ROWS_PER_THREAD) && chunk * 16 < p.k;
  if (!mine && p.vec) return;
  const int64_t k0 = chunk * 16;
  uint2 codes[ROWS_PER_THREAD] = {};
  uint32_t bytes[ROWS_PER_THREAD] = {};
  constexpr int BLOCK = Format<NV>::BLOCK;
#pragma unroll
  for (int r = 0; r < ROWS_PER_THREAD; ++r) {
    const int64_t row = row0 + r * p.block_rows;
    if (mine && row < p.rows) {
      codes[r] = *reinterpret_cast<const uint2*>(p.codes + row * p.pitch + k0 / 2);
      const int64_t block = k0 / BLOCK;
      bytes[r] = p.scales[scale_word(row, block >> 2, p.groups) + (block & 3)];
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS_PER_THREAD; ++r) {
    const int64_t row = row0 + r * p.block_rows;
    const float s = scale_value<NV>(bytes[r]) * p.pre;
    float v[16];
    unpack8(codes[r].x, *reinterpret_cast<float(*)[8]>(&v[0]));
    unpack8(codes[r].y, *reinterpret_cast<float(*)[8]>(&v[8]));
    T e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = from_float<T>(v[i] * s * p.multiplier);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(e);
    if (p.vec) {
      if (row >= p.rows) break;
      T* dst = static_cast<T*>(p.out) + row * p.ld + k0;
      constexpr int WORDS = 4 * sizeof(T);
      if (k0 + 16 <= p.k && p.vec == 32u) {
#pragma unroll
        for (int l = 0; l < WORDS / 8; ++l) store32(dst + l * (32 / sizeof(T)), *reinterpret_cast<const uint32_t(*)[8]>(&w[8 * l]));
      } else if (k0 + 16 <= p.k) {
#pragma unroll
        for (int l = 0; l < WORDS / 4; ++l)
          *reinterpret_cast<uint4*>(dst + l * (16 / sizeof(T))) = make_uint4(w[4 * l], w[4 * l + 1], w[4 * l + 2], w[4 * l + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + i < p.k) dst[i] = e[i];
      }
    } else {
      // Rows that start at any value: through shared memory, neighbouring lanes on neighbouring values (16
      // strided single stores per thread measured 98 us for 16384 x 1000 bf16).
      T* const buffer = reinterpret_cast<T*>(row_buffer);
      __syncthreads();  // the previous row has been read out
#pragma unroll
      for (int i = 0; i < 4 * static_cast<int>(sizeof(T)) / 4; ++i)
        *reinterpret_cast<uint4*>(buffer + threadIdx.x * 16 + i * (16 / sizeof(T))) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      __syncthreads();
      const int64_t first = (static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * p.row_threads * 16;  // of the piece
      const int64_t left = p.k - first;
      const uint32_t run = static_cast<uint32_t>(left < 0 ? 0 : left < p.row_threads * 16 ? left : p.row_threads * 16);
      for (uint32_t in = 0; in < p.block_rows; ++in) {
        const int64_t out_row = static_cast<int64_t>(blockIdx.x) * p.block_rows * ROWS_PER_THREAD + r * p.block_rows + in;
        if (out_row >= p.rows) break;
        T* dst = static_cast<T*>(p.out) + out_row * p.ld + first;
        for (uint32_t i = threadIdx.x; i < run; i += blockDim.x) dst[i] = buffer[in * p.row_threads * 16 + i];
      }
    }
  }
}

// The inverse of quantize_cols_kernel, with the same tile and the same division of work.
template <typename T, bool NV>
__global__ void __launch_bounds__(ColTile<T>::THREADS) dequantize_cols_kernel(const QuantParams p) {
  using Tile = ColTile<T>;
  __shared__ __align__(16) T tile[Tile::ELEMS];
  constexpr int VEC = Tile::VEC;
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * Tile::ROWS;
  const int64_t k0 = (static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * COL_K;
  if (k0 >= p.k) return;
  const int c = static_cast<int>(threadIdx.x & 7u), pair = static_cast<int>(threadIdx.x >> 3) * 2;
  const int64_t kc = k0 + c * 16;
  uint2 codes[2] = {};
  uint32_t bytes[2] = {};
  constexpr int BLOCK = Format<NV>::BLOCK;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t row = row0 + pair + r;
    if (row < p.rows && kc < p.k) {
      codes[r] = *reinterpret_cast<const uint2*>(p.codes + row * p.pitch + kc / 2);
      const int64_t block = kc / BLOCK;
      bytes[r] = p.scales[scale_word(row, block >> 2, p.groups) + (block & 3)];
    }
  }
  float v[2][16];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float s = scale_value<NV>(bytes[r]) * p.pre;
    unpack8(codes[r].x, *reinterpret_cast<float(*)[8]>(&v[r][0]));
    unpack8(codes[r].y, *reinterpret_cast<float(*)[8]>(&v[r][8]));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[r][i] = v[r][i] * s * p.multiplier;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    T both[2] = {from_float<T>(v[0][i]), from_float<T>(v[1][i])};
    T* const to = &tile[Tile::at(c * 16 + i, pair)];
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(both);
    else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(both);
  }
  __syncthreads();
  T* const dst = static_cast<T*>(p.out) + k0 * p.ld + row0;
  if (!p.vec) {  // single values, neighbouring lanes on neighbouring rows
    for (int i = threadIdx.x; i < Tile::ROWS * COL_K; i += Tile::THREADS) {
      const int kk = i / Tile::ROWS, r = i % Tile::ROWS;
      if (k0 + kk < p.k && row0 + r < p.rows) dst[static_cast<int64_t>(kk) * p.ld + r] = tile[Tile::at(kk, r)];
    }
    return;
  }
  constexpr int STEP = Tile::THREADS / Tile::PER_LINE;
  if (p.vec == 32u && k0 + COL_K <= p.k && row0 + Tile::ROWS <= p.rows) {  // as in quantize_cols_kernel
    const int line2 = threadIdx.x / (Tile::PER_LINE / 2), piece2 = (threadIdx.x % (Tile::PER_LINE / 2)) * 2 * VEC;
    const bool swap = (threadIdx.x & 4u) != 0u;
#pragma unroll
    for (int l = 0; l < COL_K / STEP / 2; ++l) {
      const int kk = l * 2 * STEP + line2;
      const uint4* e = reinterpret_cast<const uint4*>(&tile[Tile::at(kk, piece2)]);
      const uint4 a = e[swap ? 1 : 0], b = e[swap ? 0 : 1];
      const uint4 lo = swap ? b : a, hi = swap ? a : b;
      const uint32_t words[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      store32(dst + static_cast<int64_t>(kk) * p.ld + piece2, words);
    }
    return;
  }
  const int line = threadIdx.x / Tile::PER_LINE, piece = (threadIdx.x % Tile::PER_LINE) * VEC;
#pragma unroll
  for (int l = 0; l < COL_K / STEP; ++l) {
    const int kk = l * STEP + line;
    if (k0 + kk >= p.k) break;
    const T* e = &tile[Tile::at(kk, piece)];
    T* d = dst + static_cast<int64_t>(kk) * p.ld + piece;
    if (row0 + piece + VEC <= p.rows) {
      __stcs(reinterpret_cast<uint4*>(d), *reinterpret_cast<const uint4*>(e));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (row0 + piece + i < p.rows) d[i] = e[i];
    }
  }
}

}  // namespace mx
}  // namespace gz
#endif
