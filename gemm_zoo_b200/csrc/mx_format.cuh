// Arithmetic of the microscaled 4-bit formats, shared by the quantising kernels and by the
// quantising epilogue of the gated product (see include/gemmzoo/microscale.h for the formats).
#ifndef GZ_MX_FORMAT_CUH
#define GZ_MX_FORMAT_CUH

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace gz {
namespace mx {

constexpr uint32_t SCALE_TILE_BYTES = 512;  // 128 rows x 4 blocks

// Elements per scale.
template <bool NV>
struct Format {
  static constexpr int BLOCK = NV ? 16 : 32;
  static constexpr uint32_t NAN_SCALE = NV ? 0x7Fu : 0xFFu;
};

// Byte offset of the 4 scales (blocks 4g .. 4g+3) of row `r` in a scale array with `groups` tiles per
// 128 rows.
__host__ __device__ __forceinline__ int64_t scale_word(int64_t r, int64_t g, int64_t groups) {
  return ((r >> 7) * groups + g) * static_cast<int64_t>(SCALE_TILE_BYTES) + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// max(|a|, |b|) that keeps a NaN.
__device__ __forceinline__ float amax_nan(float a, float b) {
  return ptx::max_nan(fabsf(a), fabsf(b));
}

// A block's scale from the largest magnitude in it, and what turns its values into code units.
struct Scale {
  uint32_t byte;
  float value;  // the scale (only used by the e4m3 form)
  float inv;    // its reciprocal: exact for e8m0, correctly rounded for e4m3; 0 = every code is 0
};

template <bool NV>
__device__ __forceinline__ Scale block_scale(float amax) {
  Scale s;
  const uint32_t bits = __float_as_uint(amax);
  const bool bad = bits >= 0x7F800000u;  // an infinity or a NaN in the block: the whole block is NaN
  if constexpr (!NV) {
    // 2^(floor(log2 amax) - 2): the exponent field less the 2 binades that e2m1 spans above 1
    const uint32_t e = bits >> 23;
    s.byte = (e > 2u ? e : 2u) - 2u;
    s.inv = __uint_as_float((254u - s.byte) << 23);
    s.value = 0.0f;
  } else {
    // amax / 6 and 1 / scale, each correctly rounded by one residual correction (see in_code_units; the
    // scale is one of 126 numbers, all of which the tests go through)
    const float q = amax * (1.0f / 6.0f);
    const __nv_fp8_storage_t b = __nv_cvt_float_to_fp8(fmaf(fmaf(-6.0f, q, amax), 1.0f / 6.0f, q), __NV_SATFINITE, __NV_E4M3);
    s.byte = b;
    s.value = __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s.value));
    s.inv = b != 0 ? fmaf(fmaf(-s.value, r, 1.0f), r, r) : 0.0f;
  }
  if (bad) {
    s.byte = Format<NV>::NAN_SCALE;
    s.inv = 0.0f;
  }
  return s;
}

// x in code units (x / scale), accurate enough that rounding it to e2m1 is the rounding of the exact
// quotient.  e8m0: a multiplication by a power of two.  e4m3: the correctly rounded quotient by one
// residual correction of x * (1/s) (Markstein's theorem: with a correctly rounded reciprocal the
// corrected quotient is correctly rounded).  Correct rounding suffices: the rounding borders of e2m1
// have 3 significant bits and the scale 4, so border * scale is an fp32 number and an x beside it
// differs from it by at least one unit of x, which is more than half a unit of the quotient.  The
// residual is taken as q s - x, so that an exact quotient, -0 among them, comes through unchanged.
template <bool NV>
__device__ __forceinline__ float in_code_units(float x, const Scale& s) {
  if constexpr (!NV) return x * s.inv;
  const float q = x * s.inv;
  return fmaf(-fmaf(q, s.value, -x), s.inv, q);
}

// Eight values in code units -> eight e2m1 codes, the first in the low nibble (ties to even,
// saturating at 6).
__device__ __forceinline__ uint32_t pack8(float v0, float v1, float v2, float v3, float v4, float v5, float v6,
                                          float v7) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t"
      "}"
      : "=r"(r)
      : "f"(v0), "f"(v1), "f"(v2), "f"(v3), "f"(v4), "f"(v5), "f"(v6), "f"(v7));
  return r;
}

// Eight e2m1 codes -> eight fp32 values (exact).
__device__ __forceinline__ void unpack8(uint32_t codes, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
      "}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// The value of a scale byte.
template <bool NV>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  if constexpr (NV) return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
  else return __uint_as_float(byte == 255u ? 0x7FFFFFFFu : byte == 0u ? 0x00400000u : byte << 23);
}

}  // namespace mx
}  // namespace gz
#endif
