/* Microscaled 4-bit matrices on NVIDIA B200 (sm_100a): quantisation and its inverse, the product of
 * two quantised matrices, and the gated feed-forward product.  The reference project has no counterpart;
 * its narrowest type is 8 bits (nvidia/bench/bench_cublaslt_e4m3.cu:6-21).  Conventions (device pointers,
 * status codes, host alpha/beta, streams, no fallback) are those of gemmzoo/gemm.h.
 *
 * A quantised matrix of `rows` x `k` has
 *   codes   e2m1 values (0 0.5 1 1.5 2 3 4 6 and their negatives), two to a byte, the even k in the low
 *           nibble; rows `pitch` bytes apart (a multiple of 16, at least gz_mx_code_pitch(k)).  An odd k
 *           is followed by a zero code.
 *   scales  one byte per block of consecutive k:
 *             GZ_MX_FP4    32 elements, e8m0 (2^(byte - 127); 255 = NaN)
 *             GZ_MX_NVFP4  16 elements, e4m3 (sign 0; 127 = NaN)
 *           in tiles of 128 rows x 4 blocks (512 bytes, what the tensor core reads): the scale of row r,
 *           block b is byte  ((r / 128) * ceil(blocks / 4) + b / 4) * 512 + (r % 32) * 16 +
 *           (r % 128 / 32) * 4 + b % 4.  The array covers whole tiles; bytes of rows and blocks that do
 *           not exist must not be NaN (the functions here write 0).
 * and stands for code * scale (* a multiplier the caller keeps, see below).
 *
 * Codes and scales must be 16-byte aligned.  Extents are positive (an empty matrix is refused, as
 * everywhere in this library).  Outputs must not overlap inputs, the epilogue's vectors among them (D and C may
 * be the same matrix; equal addresses of others are refused).  Calls that overlap on the GPU may share inputs and plans freely: no
 * entry point below keeps a workspace or counters between calls (a plan's status words apart). */
#ifndef GEMMZOO_MICROSCALE_H
#define GEMMZOO_MICROSCALE_H

#include "gemmzoo/gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Numbered apart from gz_dtype, so that gz_mx_desc::out_type can name either. */
typedef enum gz_mx_format {
  GZ_MX_FP4 = 16,
  GZ_MX_NVFP4 = 17
} gz_mx_format;

/* Bytes of one packed row of codes (k rounded up to 32, two to a byte), and of a scale array.  -1 for
 * arguments that are not positive or a format that does not exist. */
GZ_API int64_t gz_mx_code_pitch(int64_t k);
GZ_API int64_t gz_mx_scale_bytes(int32_t format, int64_t rows, int64_t k);

/* Quantises values * multiplier (one rounding to fp32) along k:
 *   GZ_MX_FP4    scale = 2^(floor(log2 amax) - 2), at least 2^-127
 *   GZ_MX_NVFP4  scale = amax / 6 rounded to e4m3 (at most 448); 0 makes the block's codes 0
 *   code = value * multiplier / scale rounded to e2m1, ties to even, saturated at 6
 * with amax the largest magnitude of the block.  A block that holds a NaN or an infinity gets a NaN
 * scale and zero codes, so that it stays NaN.  The result stands for the values times the multiplier:
 * fold 1 / multiplier into alpha (or into the dequantising multiplier).
 *   src_type  GZ_DT_F16, GZ_DT_BF16 or GZ_DT_F32
 *   layout    GZ_ROW_MAJOR: element k of row i at src[i * ld + k];  GZ_COL_MAJOR: at src[k * ld + i]
 *             (a weight stored K x N row-major is a column-major one of N rows)
 *   ld, pitch 0 = packed
 * Writes round_up(k, 32) / 2 bytes of each row of codes and the whole scale array.  Asynchronous on
 * `stream`, which belongs to `device`. */
GZ_API gz_status gz_mx_quantize(const void* src, int32_t src_type, int32_t layout, int64_t ld, int64_t rows, int64_t k,
                                int32_t format, float multiplier, void* codes, int64_t pitch, void* scales,
                                int32_t device, void* stream);

/* code * scale * multiplier (rounded once in fp32 and once to dst_type) into a row- or column-major
 * matrix. */
GZ_API gz_status gz_mx_dequantize(const void* codes, int64_t pitch, const void* scales, int32_t format, int64_t rows,
                                  int64_t k, float multiplier, void* dst, int32_t dst_type, int32_t layout, int64_t ld,
                                  int32_t device, void* stream);

/* Tiles: explicit values pin one for tests and benchmarks. */
typedef enum gz_mx_config {
  GZ_MX_CFG_AUTO = 0,
  GZ_MX_CFG_PAIR = 1,     /* 256 rows x 256 columns (gated: 128 columns) on a CTA pair */
  GZ_MX_CFG_SINGLE = 2,   /* 128 rows x 256 columns (gated: 128 columns) on one CTA */
  GZ_MX_CFG_SWAP_M16 = 3, /* 128 columns x up to 16 / 32 / 64 rows, m <= 16 / 32 / 64 */
  GZ_MX_CFG_SWAP_M32 = 4,
  GZ_MX_CFG_SWAP_M64 = 5,
  GZ_MX_CFG_PAIR_N128 = 6,  /* 256 rows x 128 columns on a CTA pair (not gated) */
  GZ_MX_CFG_SINGLE_N128 = 7 /* 128 rows x 128 columns on one CTA (not gated) */
} gz_mx_config;

/* One product  D[m x n] = A[m x k] * B[n x k]^T  of quantised matrices of one format, or a gated one. */
typedef struct gz_mx_desc {
  uint32_t struct_size; /* sizeof(gz_mx_desc) */
  int32_t format;       /* gz_mx_format of A and B */
  int32_t out_type;     /* GZ_DT_F16, GZ_DT_BF16, GZ_DT_F32; gated also a gz_mx_format: D is quantised */
  int32_t gated;        /* 0: gz_mx_gemm_run, 1: gz_mx_gated_run */
  int32_t device;
  int32_t config;       /* gz_mx_config */
  int32_t split;        /* CTAs (pair tiles: pairs) that share a tile's K range: 1, 2, 4 or 8, at most one
                           per 256 of K and eight CTAs, in row tiles (PAIR, SINGLE and their N128) also at
                           most one per 32 output columns of the tile; 0 = chosen */
  uint32_t flags;       /* 0 or GZ_FLAG_TEST_WITHHOLD_ACC_READY */
  int64_t m, n, k;
  int64_t pitch_a, pitch_b; /* bytes between rows of codes (gated: pitch_b for gate and up); 0 = packed */
  int64_t ldc, ldd;         /* elements between rows; a quantised D: ldd = bytes between rows of codes; 0 = packed */
  uint64_t wait_limit_ns;   /* as gz_gemm_desc */
} gz_mx_desc;

typedef struct gz_mx_plan gz_mx_plan;

typedef struct gz_mx_plan_info {
  int32_t config, split;
  int32_t tile_m, tile_n, tile_k;
  int32_t stages, grid, smem_bytes;
  int32_t out_tma;  /* 1 if D's row pitch lets the tile be stored by TMA */
  int32_t reserved;
  int64_t tiles;
} gz_mx_plan_info;

/* Host-only validation, as gz_gemm_desc_validate. */
GZ_API gz_status gz_mx_desc_validate(const gz_mx_desc* desc, int sm_count, gz_mx_plan_info* info);
GZ_API gz_status gz_mx_plan_create(gz_mx_plan** plan, const gz_mx_desc* desc);
GZ_API gz_status gz_mx_plan_destroy(gz_mx_plan* plan);
GZ_API gz_status gz_mx_plan_info_get(const gz_mx_plan* plan, gz_mx_plan_info* info);

/* D = act(alpha * row_scale[i] * col_scale[j] * (A B^T)[i][j] + beta * C + bias[j]), fp32 accumulation
 * and epilogue.  c may be NULL when *beta == 0 and may be d (then with ldc == ldd); ep may be NULL.  alpha,
 * beta: host floats.
 *
 * Activations are within 5e-7 |x| of their exact value at the fp32 x they are given, at a result of normal
 * size SiLU and the tanh GELU also within (6e-7 + 5e-7 |y|) of the result (e^y is their exponential) and the
 * erf GELU within 1e-4 of it for x >= -3, 1e-3 for x >= -4.5 and 1e-2 for x >= -7.5. */
GZ_API gz_status gz_mx_gemm_run(gz_mx_plan* plan, const void* a, const void* a_scales, const void* b,
                                const void* b_scales, const void* c, void* d, const float* alpha, const float* beta,
                                const gz_epilogue* ep, void* stream);

/* D = act(alpha_gate * A G^T) * (alpha_up * A U^T) with gate and up n x k: both projections, the
 * activation and the product in one launch.  With a quantised output type, d receives the codes and
 * d_scales the scales of D * out_multiplier, as gz_mx_quantize of the unrounded fp32 values would write
 * them (ready for the next product); otherwise d_scales is NULL and out_multiplier is not used. */
GZ_API gz_status gz_mx_gated_run(gz_mx_plan* plan, const void* a, const void* a_scales, const void* gate,
                                 const void* gate_scales, const void* up, const void* up_scales, void* d,
                                 void* d_scales, const float* alpha_gate, const float* alpha_up, int32_t activation,
                                 float out_multiplier, void* stream);

/* As gz_last_device_status. */
GZ_API gz_status gz_mx_last_device_status(gz_mx_plan* plan, void* stream, uint32_t detail[4]);

#ifdef __cplusplus
}
#endif
#endif
