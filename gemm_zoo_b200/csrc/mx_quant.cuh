// Quantisation to the microscaled 4-bit formats and its inverse (include/gemmzoo/microscale.h).
//
// Both are one pass over memory: a block's scale needs its largest magnitude, which a thread (or
// two neighbouring ones) holds in registers, so a value is read once and its code written once.
#ifndef GZ_MX_QUANT_CUH
#define GZ_MX_QUANT_CUH

#include <cuda_bf16.h>

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
  int64_t items;       // work items of the launch (row layout)
  uint32_t per_row;    // 16-element chunks per row, a whole number of scale words
  uint32_t vec;        // vector access to the values is legal
  float multiplier;
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

// 32 bytes at a 32-byte aligned address.
__device__ __forceinline__ void load32(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Which (row, chunk) the thread's item is: the block's first item is divided in 64 bits once, the
// thread's offset from it in 32.
__device__ __forceinline__ void item_coords(const QuantParams& p, int64_t first, uint32_t offset, int64_t& row,
                                            uint32_t& chunk) {
  const int64_t row0 = first / p.per_row;
  const uint32_t rem = static_cast<uint32_t>(first - row0 * p.per_row) + offset;
  const uint32_t add = rem / p.per_row;
  row = row0 + add;
  chunk = rem - add * p.per_row;
}

// Rows with K contiguous.  A thread takes 16 consecutive elements (32 bytes of a 16-bit type in one
// load), which is one e4m3 block or half of an e8m0 block; the lanes that share a 4-byte word of
// scales are neighbours, so amax and the word are put together with shuffles.  Rows beyond the last
// up to the next multiple of 128 exist in the scale array only and get zero bytes.
template <typename T, bool NV>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p) {
  constexpr int PER_WORD = NV ? 4 : 8;  // threads whose blocks share a word of scales
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x;
  const bool mine = first + threadIdx.x < p.items;
  const uint32_t mask = __ballot_sync(0xFFFFFFFFu, mine);  // whole words: items are a multiple of PER_WORD
  if (!mine) return;
  int64_t row;
  uint32_t chunk;
  item_coords(p, first, threadIdx.x, row, chunk);
  const int64_t k0 = static_cast<int64_t>(chunk) * 16;
  float v[16];
  const T* src = static_cast<const T*>(p.in) + row * p.ld + k0;
  if (row < p.rows && k0 + 16 <= p.k && p.vec) {
    constexpr int LOADS = sizeof(T) / 2;
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      uint32_t w[8];
      load32(src + l * (16 / LOADS), w);
      const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int i = 0; i < 16 / LOADS; ++i) v[l * (16 / LOADS) + i] = to_float<T>(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = (row < p.rows && k0 + i < p.k) ? to_float<T>(src[i]) : 0.0f;
  }
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    v[i] *= p.multiplier;
    amax = amax_nan(amax, v[i]);
  }
  if constexpr (!NV) amax = amax_nan(amax, __shfl_xor_sync(mask, amax, 1));
  const Scale s = block_scale<NV>(amax);
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = in_code_units<NV>(v[i], s);
  uint2 codes;
  codes.x = pack8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
  codes.y = pack8(v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]);
  if (s.byte == Format<NV>::NAN_SCALE) codes = make_uint2(0u, 0u);
  if (row < p.rows && k0 / 2 < p.code_bytes)
    *reinterpret_cast<uint2*>(p.codes + row * p.pitch + k0 / 2) = codes;
  const uint32_t in_word = chunk % PER_WORD;
  uint32_t word = (row < p.rows ? s.byte : 0u) << (8 * (NV ? in_word : in_word / 2));
#pragma unroll
  for (int d = PER_WORD / 4; d < PER_WORD; d *= 2) word |= __shfl_xor_sync(mask, word, d);
  if (in_word == 0) *reinterpret_cast<uint32_t*>(p.scales + scale_word(row, chunk / PER_WORD, p.groups)) = word;
}

// K strided: element k of row i at in[k * ld + i].  A block takes 64 rows x 128 k through shared
// memory: it is filled along the rows (128 or 256 bytes per k) and read along k, four threads side by
// side on one row with 32 k each, so that a row's 64 bytes of codes are written together.  The 16
// extra elements per 32 k put the four threads' words in different banks.
constexpr int COL_ROWS = 64, COL_K = 128;
template <typename T>
struct ColTile {
  static constexpr int PAD = 32 / sizeof(T);  // eight words
  static constexpr int ELEMS = COL_ROWS * COL_K + 4 * PAD;
  static __device__ __forceinline__ int at(int k, int row) { return k * COL_ROWS + (k >> 5) * PAD + row; }
};

template <typename T, bool NV>
__global__ void __launch_bounds__(256) quantize_cols_kernel(const QuantParams p) {
  __shared__ __align__(16) T tile[ColTile<T>::ELEMS];
  constexpr int VEC = 16 / sizeof(T);
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int64_t row_tiles = ((p.rows + 127) / 128) * 2;
  const int64_t k0 = (blockIdx.x / row_tiles) * COL_K, row0 = (blockIdx.x % row_tiles) * COL_ROWS;
  const T* const src = static_cast<const T*>(p.in);
  constexpr int PER_LINE = COL_ROWS / VEC;
#pragma unroll
  for (int l = 0; l < COL_K * PER_LINE / 256; ++l) {
    const int at = l * 256 + threadIdx.x;
    const int kk = at / PER_LINE, r = (at % PER_LINE) * VEC;
    const int64_t gk = k0 + kk, gr = row0 + r;
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (gk < p.k) {
      if (gr + VEC <= p.rows && p.vec) {
        w = *reinterpret_cast<const uint4*>(src + gk * p.ld + gr);
      } else {
        T* e = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (gr + i < p.rows) e[i] = src[gk * p.ld + gr + i];
      }
    }
    *reinterpret_cast<uint4*>(&tile[ColTile<T>::at(kk, r)]) = w;
  }
  __syncthreads();
  const int r = threadIdx.x >> 2, quarter = threadIdx.x & 3;
  const int64_t row = row0 + r;
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = to_float<T>(tile[ColTile<T>::at(quarter * 32 + i, r)]) * p.multiplier;
  uint32_t bytes = 0;  // this thread's one or two scales
  constexpr int BLOCK = Format<NV>::BLOCK;
  uint32_t codes[4];
#pragma unroll
  for (int b = 0; b < 32 / BLOCK; ++b) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) amax = amax_nan(amax, v[b * BLOCK + i]);
    const Scale s = block_scale<NV>(amax);
    bytes |= s.byte << (8 * b);
#pragma unroll
    for (int i = 0; i < BLOCK / 8; ++i) {
      float* x = &v[b * BLOCK + i * 8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = in_code_units<NV>(x[j], s);
      const uint32_t c = pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
      codes[b * (BLOCK / 8) + i] = s.byte == Format<NV>::NAN_SCALE ? 0u : c;
    }
  }
  const int64_t at = (k0 + quarter * 32) / 2;
  if (row < p.rows && at < p.code_bytes)
    *reinterpret_cast<uint4*>(p.codes + row * p.pitch + at) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
  if (row >= p.rows) bytes = 0;
  if constexpr (!NV) {
    uint32_t word = bytes << (8 * quarter);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 1);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2);
    if (quarter == 0) *reinterpret_cast<uint32_t*>(p.scales + scale_word(row, k0 / 128, p.groups)) = word;
  } else {
    uint32_t word = bytes << (16 * (quarter & 1));
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 1);
    const int64_t g = k0 / 64 + quarter / 2;
    if ((quarter & 1) == 0 && g < p.groups) *reinterpret_cast<uint32_t*>(p.scales + scale_word(row, g, p.groups)) = word;
  }
}

// code * scale is exact in fp32; the product with the multiplier is rounded once there and once to T.
template <bool NV>
__device__ __forceinline__ float scale_of(const QuantParams& p, int64_t row, int64_t block) {
  return scale_value<NV>(__ldg(p.scales + scale_word(row, block >> 2, p.groups) + (block & 3)));
}

template <typename T, bool NV>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(const QuantParams p) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x;
  if (first + threadIdx.x >= p.items) return;
  int64_t row;
  uint32_t chunk;
  item_coords(p, first, threadIdx.x, row, chunk);
  const int64_t k0 = static_cast<int64_t>(chunk) * 16;
  const uint2 codes = *reinterpret_cast<const uint2*>(p.codes + row * p.pitch + k0 / 2);
  const float s = scale_of<NV>(p, row, k0 / Format<NV>::BLOCK);
  float v[16];
  unpack8(codes.x, *reinterpret_cast<float(*)[8]>(&v[0]));
  unpack8(codes.y, *reinterpret_cast<float(*)[8]>(&v[8]));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = v[i] * s * p.multiplier;
  T* dst = static_cast<T*>(p.out) + row * p.ld + k0;
  if (k0 + 16 <= p.k && p.vec) {
    constexpr int STORES = sizeof(T) / 2;
#pragma unroll
    for (int l = 0; l < STORES; ++l) {
      uint32_t w[8];
      T* e = reinterpret_cast<T*>(w);
#pragma unroll
      for (int i = 0; i < 16 / STORES; ++i) e[i] = from_float<T>(v[l * (16 / STORES) + i]);
      store32(dst + l * (16 / STORES), w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k0 + i < p.k) dst[i] = from_float<T>(v[i]);
  }
}

template <typename T, bool NV>
__global__ void __launch_bounds__(256) dequantize_cols_kernel(const QuantParams p) {
  __shared__ __align__(16) T tile[ColTile<T>::ELEMS];
  constexpr int VEC = 16 / sizeof(T);
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int64_t row_tiles = (p.rows + COL_ROWS - 1) / COL_ROWS;
  const int64_t k0 = (blockIdx.x / row_tiles) * COL_K, row0 = (blockIdx.x % row_tiles) * COL_ROWS;
  const int r = threadIdx.x >> 2, quarter = threadIdx.x & 3;
  const int64_t row = row0 + r, kq = k0 + quarter * 32;
  if (row < p.rows && kq < p.k) {
    const uint4 c = *reinterpret_cast<const uint4*>(p.codes + row * p.pitch + kq / 2);
    const uint32_t words[4] = {c.x, c.y, c.z, c.w};
    constexpr int BLOCK = Format<NV>::BLOCK;
#pragma unroll
    for (int b = 0; b < 32 / BLOCK; ++b) {
      const int64_t block = kq / BLOCK + b;
      const float s = block * BLOCK < p.k ? scale_of<NV>(p, row, block) : 0.0f;
#pragma unroll
      for (int i = 0; i < BLOCK / 8; ++i) {
        float v[8];
        unpack8(words[b * (BLOCK / 8) + i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          tile[ColTile<T>::at(quarter * 32 + b * BLOCK + i * 8 + j, r)] = from_float<T>(v[j] * s * p.multiplier);
      }
    }
  }
  __syncthreads();
  T* const dst = static_cast<T*>(p.out);
  constexpr int PER_LINE = COL_ROWS / VEC;
#pragma unroll
  for (int l = 0; l < COL_K * PER_LINE / 256; ++l) {
    const int at = l * 256 + threadIdx.x;
    const int kk = at / PER_LINE, rr = (at % PER_LINE) * VEC;
    const int64_t gk = k0 + kk, gr = row0 + rr;
    if (gk >= p.k) break;
    const T* e = &tile[ColTile<T>::at(kk, rr)];
    if (gr + VEC <= p.rows && p.vec) {
      *reinterpret_cast<uint4*>(dst + gk * p.ld + gr) = *reinterpret_cast<const uint4*>(e);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (gr + i < p.rows) dst[gk * p.ld + gr + i] = e[i];
    }
  }
}

}  // namespace mx
}  // namespace gz
#endif
