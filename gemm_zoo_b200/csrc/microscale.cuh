// Host layer of the microscaled 4-bit operators (include/gemmzoo/microscale.h): argument checks, tile
// choice, tensor maps and launches.  Included at the end of gemm_api.cu, whose helpers it uses.
#ifndef GZ_MICROSCALE_CUH
#define GZ_MICROSCALE_CUH

#include "gemmzoo/microscale.h"
#include "mx_gemm.cuh"
#include "mx_quant.cuh"
#include "mx_table.h"

namespace {

bool is_mx(int f) { return f == GZ_MX_FP4 || f == GZ_MX_NVFP4; }
int mx_block(int format) { return format == GZ_MX_NVFP4 ? 16 : 32; }
int64_t mx_groups(int format, int64_t k) { return cdiv(cdiv(k, mx_block(format)), 4); }
bool mx_float_type(int t) { return t == GZ_DT_F16 || t == GZ_DT_BF16 || t == GZ_DT_F32; }
bool mx_aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
constexpr int64_t kMxExtent = (int64_t(1) << 31) - 1024;  // 32-bit tile and TMA coordinates

// rows x pitch addressable, without overflow
bool mx_span_ok(int64_t rows, int64_t pitch) {
  int64_t s;
  return !__builtin_mul_overflow(rows, pitch, &s) && s <= (int64_t(1) << 60);
}

gz_status mx_device_ok(int device) {
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev == 0) {
    (void)cudaGetLastError();
    return GZ_ERR_NO_DEVICE;
  }
  return device < ndev ? GZ_OK : GZ_ERR_INVALID_ARG;
}

// What quantisation and its inverse check alike.
gz_status mx_quant_params(gz::mx::QuantParams* p, const void* values, int type, int layout, int64_t ld, int64_t rows,
                          int64_t k, int format, float multiplier, const void* codes, int64_t pitch, const void* scales,
                          int device) {
  if (!values || !codes || !scales || rows <= 0 || k <= 0 || device < 0 || ld < 0 || pitch < 0) return GZ_ERR_INVALID_ARG;
  if (layout != GZ_ROW_MAJOR && layout != GZ_COL_MAJOR) return GZ_ERR_INVALID_ARG;
  if (!is_mx(format) || dtype_size(type) == 0 || !(std::fabs(multiplier) <= 3.4028234e38f) || multiplier == 0.0f)
    return GZ_ERR_INVALID_ARG;
  if (!mx_float_type(type)) return GZ_ERR_UNSUPPORTED;
  if (rows > kMxExtent || k > kMxExtent) return GZ_ERR_TOO_LARGE;
  const bool cols = layout == GZ_COL_MAJOR;
  if (ld == 0) ld = cols ? rows : k;
  if (pitch == 0) pitch = gz_mx_code_pitch(k);
  if (ld < (cols ? rows : k) || pitch < gz_mx_code_pitch(k) || pitch % 16 != 0) return GZ_ERR_INVALID_ARG;
  const int size = dtype_size(type);
  if (!mx_span_ok(cols ? k : rows, ld) || !mx_span_ok(rows, pitch)) return GZ_ERR_TOO_LARGE;
  if (values == codes || values == scales || codes == scales) return GZ_ERR_INVALID_ARG;  // nothing is converted in place
  if (!mx_aligned(values, size) || !mx_aligned(codes, 16) || !mx_aligned(scales, 16)) return GZ_ERR_MISALIGNED;
  std::memset(p, 0, sizeof(*p));
  p->rows = rows;
  p->k = k;
  p->ld = ld;
  p->pitch = pitch;
  p->code_bytes = gz_mx_code_pitch(k);
  p->groups = mx_groups(format, k);
  p->multiplier = multiplier;
  p->unit = multiplier == 1.0f ? 1u : 0u;
  for (const int bytes : {32, 16})  // the widest access that every row allows
    if (p->vec == 0 && mx_aligned(values, bytes) && (ld * size) % bytes == 0) p->vec = (uint32_t)bytes;
  return GZ_OK;
}

struct MxShape {
  int config, bn, ctas;
  bool swap() const { return bn <= 64; }
};
const MxShape kMxShapes[] = {{GZ_MX_CFG_PAIR, 256, 2},
                             {GZ_MX_CFG_SINGLE, 256, 1},
                             {GZ_MX_CFG_SWAP_M16, 16, 1},
                             {GZ_MX_CFG_SWAP_M32, 32, 1},
                             {GZ_MX_CFG_SWAP_M64, 64, 1},
                             {GZ_MX_CFG_PAIR_N128, 128, 2},
                             {GZ_MX_CFG_SINGLE_N128, 128, 1}};
const MxShape* mx_shape_of(int config) {
  for (const auto& s : kMxShapes)
    if (s.config == config) return &s;
  return nullptr;
}

struct MxProblem {
  gz_mx_desc d;
  int out_size;  // 0: quantised
};

gz_status mx_normalise(const gz_mx_desc* desc, MxProblem* pr) {
  if (!desc || desc->struct_size != sizeof(gz_mx_desc)) return GZ_ERR_INVALID_ARG;
  gz_mx_desc d = *desc;
  if (d.m <= 0 || d.n <= 0 || d.k <= 0 || d.device < 0 || !is_mx(d.format)) return GZ_ERR_INVALID_ARG;
  if (d.gated != 0 && d.gated != 1) return GZ_ERR_INVALID_ARG;
  if (dtype_size(d.out_type) == 0 && !is_mx(d.out_type)) return GZ_ERR_INVALID_ARG;
  if (d.flags & ~GZ_FLAG_TEST_WITHHOLD_ACC_READY) return GZ_ERR_INVALID_ARG;
  if (d.config != GZ_MX_CFG_AUTO && !mx_shape_of(d.config)) return GZ_ERR_INVALID_ARG;
  if (d.split != 0 && d.split != 1 && d.split != 2 && d.split != 4 && d.split != 8) return GZ_ERR_INVALID_ARG;
  if (!mx_float_type(d.out_type) && !(is_mx(d.out_type) && d.gated)) return GZ_ERR_UNSUPPORTED;
  if (d.m > kMxExtent || d.n > kMxExtent || d.k > kMxExtent) return GZ_ERR_TOO_LARGE;
  const bool quantised = is_mx(d.out_type);
  const int64_t in_pitch = gz_mx_code_pitch(d.k), out_ld = quantised ? gz_mx_code_pitch(d.n) : d.n;
  if (d.pitch_a < 0 || d.pitch_b < 0 || d.ldc < 0 || d.ldd < 0) return GZ_ERR_INVALID_ARG;
  if (d.pitch_a == 0) d.pitch_a = in_pitch;
  if (d.pitch_b == 0) d.pitch_b = in_pitch;
  if (d.ldc == 0) d.ldc = d.n;
  if (d.ldd == 0) d.ldd = out_ld;
  if (d.pitch_a < in_pitch || d.pitch_b < in_pitch || d.ldc < d.n || d.ldd < out_ld) return GZ_ERR_INVALID_ARG;
  if (d.pitch_a % 16 != 0 || d.pitch_b % 16 != 0 || (quantised && d.ldd % 16 != 0)) return GZ_ERR_MISALIGNED;
  const int64_t stride_lim = int64_t(1) << 39;  // of a tensor map
  if (!mx_span_ok(d.m, d.pitch_a) || !mx_span_ok(d.n, d.pitch_b) || !mx_span_ok(d.m, d.ldc) || !mx_span_ok(d.m, d.ldd) ||
      d.pitch_a > stride_lim || d.pitch_b > stride_lim)
    return GZ_ERR_TOO_LARGE;
  if (cdiv(d.m, 128) * cdiv(d.n, 128) > (int64_t(1) << 31) - 1) return GZ_ERR_TOO_LARGE;
  if (d.wait_limit_ns == 0) d.wait_limit_ns = 2000000000ull;
  pr->d = d;
  pr->out_size = dtype_size(d.out_type);
  return GZ_OK;
}

bool mx_shape_fits(const MxProblem& pr, const MxShape& s) {
  if (s.swap()) return pr.d.m <= s.bn;
  return s.bn == 256 || !pr.d.gated;
}

// Output columns of a tile.
int mx_tile_n(const MxProblem& pr, const MxShape& s) { return s.swap() ? 128 : pr.d.gated ? s.bn / 2 : s.bn; }

int64_t mx_tiles(const MxProblem& pr, const MxShape& s) {
  return (s.swap() ? 1 : cdiv(pr.d.m, 128 * s.ctas)) * cdiv(pr.d.n, mx_tile_n(pr, s));
}

// The largest cluster is eight CTAs, and a row tile has a slice for every 32 columns to deal to the parts.
int mx_max_split(const MxProblem& pr, const MxShape& s) {
  const int slices = s.swap() ? 8 : mx_tile_n(pr, s) / 32, ctas = 8 / s.ctas;
  return slices < ctas ? slices : ctas;
}

// CTAs that can be resident at the same time in clusters of `cluster`.  A cluster lies within one GPC; of 148 SMs in GPCs of
// 16 to 20, 14 clusters of eight or 32 of four, one CTA per SM, are counted on (one part's runtime answers 15 and 33).
// Swapped tiles have two CTAs per SM (1.9 active by the counters at 1 x 37888 x 4096; the runtime's occupancy query says
// one for any of these kernels, so it cannot be asked instead).
int64_t mx_resident(const MxShape& s, int cluster, int sm_count) {
  const int64_t sms = cluster >= 8 ? sm_count * 112 / 148 : cluster == 4 ? sm_count * 128 / 148 : sm_count;
  return s.swap() ? 2 * sms : sms;
}

// Microseconds that a configuration is estimated to take: a fixed part, the K blocks of the longest CTA at
// the pace of its tile, what handing over a shared K range costs, and never less than B takes from HBM
// (of which a swapped CTA, with its ring of 110 KB, draws 43 GB/s under load).  Fitted to graph-timed
// sweeps of every tile and split over 129 shapes, plain and gated, m 1 to 8192; over 100 other random shapes the
// pick lost 1.5 % on the best configuration on average and 15 % at worst.
double mx_cost(const MxProblem& pr, const MxShape& s, int split, int sm_count) {
  const int64_t tiles = mx_tiles(pr, s);
  const bool nv = pr.d.format == GZ_MX_NVFP4, gated = pr.d.gated != 0, quantised = pr.out_size == 0;
  const int64_t slots = mx_resident(s, s.ctas * split, sm_count) / (s.ctas * split);  // clusters at a time
  if (slots <= 0) return 1e30;
  const double waves = double(cdiv(tiles, slots)), blocks = double(cdiv(cdiv(pr.d.k, 256), split));
  const double b_bytes = double(pr.d.n) * double(pr.d.k) * (nv ? 0.5625 : 0.53125) * (gated ? 2 : 1);
  const double m = double(pr.d.m);
  double fixed, per_block, hand_over = 0.0, per_wave, hbm = b_bytes / 6.3e6;
  if (s.swap()) {
    // parking is every CTA's, finishing is shared
    fixed = 3.3 + 0.04 * m * (gated ? 1.5 : 1.0) + 0.04 * m / split * (gated ? 1.5 : 1.0) * (quantised ? 1.5 : 1.0);
    per_block = !gated ? 0.28 : nv ? 0.9 : 0.6;  // a gated ring holds two or three stages
    if (split > 1) hand_over = 0.6;
    per_wave = 0.3;
    const double ctas = double(tiles) * split, drawn = 43e3 * (ctas < 2.0 * sm_count ? ctas : 2.0 * sm_count);
    if (drawn < 6.3e6) hbm = b_bytes / drawn;
  } else if (s.bn == 256) {
    fixed = (s.ctas == 2 ? 5.4 : 4.9) + (quantised ? 3.0 : gated ? 1.0 : 0.0);
    per_block = s.ctas == 2 ? 0.318 : 0.5;
    if (split > 1) hand_over = split == 2 ? 3.2 : 6.0;
    per_wave = 0.8;
  } else {
    fixed = s.ctas == 2 ? 3.9 : 3.5;
    per_block = s.ctas == 2 ? 0.267 : tiles * split * 2 <= sm_count ? 0.29 : 0.38;
    if (split > 1) hand_over = 0.95 * split;
    per_wave = 0.6;
  }
  const double stream = waves * (blocks * per_block + per_wave);
  return fixed + hand_over + (stream > hbm ? stream : hbm);
}

int mx_choose_split(const MxProblem& pr, const MxShape& s, int sm_count, double* cost) {
  const int64_t tiles = mx_tiles(pr, s), k_blocks = cdiv(pr.d.k, 256);
  int best = 1;
  *cost = mx_cost(pr, s, 1, sm_count);
  for (int split = 2; split <= mx_max_split(pr, s); split *= 2) {
    if (k_blocks < split || tiles * s.ctas * split > mx_resident(s, s.ctas * split, sm_count)) break;
    const double c = mx_cost(pr, s, split, sm_count);
    if (c < *cost) {
      *cost = c;
      best = split;
    }
  }
  return best;
}

int mx_choose(const MxProblem& pr, int sm_count) {
  double best = 0;
  int best_cfg = GZ_MX_CFG_SINGLE;
  for (const auto& s : kMxShapes) {
    if (!mx_shape_fits(pr, s) || sm_count < s.ctas) continue;
    double cost;
    if (pr.d.split) {
      if (pr.d.split > mx_max_split(pr, s)) continue;
      cost = mx_cost(pr, s, pr.d.split, sm_count);
    } else {
      mx_choose_split(pr, s, sm_count, &cost);
    }
    if (best == 0 || cost < best) {
      best = cost;
      best_cfg = s.config;
    }
  }
  return best_cfg;
}

gz::MxEntry mx_entry_of(const MxProblem& pr, int config) {
  return pr.d.format == GZ_MX_NVFP4 ? gz::mx_kernels_nvfp4(config, pr.d.gated != 0)
                                    : gz::mx_kernels_fp4(config, pr.d.gated != 0);
}

gz_status mx_resolve(const MxProblem& pr, int sm_count, gz_mx_plan_info* info) {
  const int config = pr.d.config == GZ_MX_CFG_AUTO ? mx_choose(pr, sm_count) : pr.d.config;
  const MxShape& s = *mx_shape_of(config);
  if (!mx_shape_fits(pr, s)) return GZ_ERR_UNSUPPORTED;
  const int64_t tiles = mx_tiles(pr, s);
  double cost;
  const int split = pr.d.split ? pr.d.split : mx_choose_split(pr, s, sm_count, &cost);
  if (split > mx_max_split(pr, s) || sm_count < s.ctas) return GZ_ERR_UNSUPPORTED;
  // a shared K range: every CTA has a part of it, and a row tile's cluster has one tile
  if (split > 1 && cdiv(pr.d.k, 256) < split) return GZ_ERR_UNSUPPORTED;
  const gz::MxEntry e = mx_entry_of(pr, config);
  std::memset(info, 0, sizeof(*info));
  info->config = config;
  info->split = split;
  info->tile_m = s.swap() ? s.bn : 128 * s.ctas;
  info->tile_n = mx_tile_n(pr, s);
  info->tile_k = 256;
  info->stages = e.stages;
  info->smem_bytes = e.smem_bytes;
  const int64_t walkers = sm_count / s.ctas;  // CTAs or pairs that walk the tiles of a persistent launch
  const int64_t clusters = s.swap() || split > 1 || tiles < walkers ? tiles : walkers;
  if (clusters * s.ctas * split > (int64_t(1) << 31) - 1) return GZ_ERR_TOO_LARGE;
  info->grid = (int32_t)(clusters * s.ctas * split);
  info->out_tma = (!s.swap() && pr.out_size != 0 && (pr.d.ldd * pr.out_size) % 16 == 0 &&
                   pr.d.ldd * pr.out_size < (int64_t(1) << 40)) ? 1 : 0;
  info->tiles = tiles;
  return GZ_OK;
}

bool mx_encode(CUtensorMap* tm, CUtensorMapDataType type, const void* base, uint64_t d0, uint64_t d1, uint64_t d2,
               uint64_t stride1, uint64_t stride2, uint32_t b0, uint32_t b1, CUtensorMapSwizzle swizzle, bool promote) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) {
    g_last_cuda_error = "cuTensorMapEncodeTiled entry point not available";
    return false;
  }
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {stride1, stride2};
  cuuint32_t box[3] = {b0, b1, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(tm, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle, promote ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_NONE,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    char buf[96];
    std::snprintf(buf, sizeof(buf), "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    g_last_cuda_error = buf;
    return false;
  }
  return true;
}

}  // namespace

struct gz_mx_plan {
  MxProblem pr;
  gz_mx_plan_info info;
  gz::MxEntry entry;
  gz::MxParams base;  // everything that does not depend on the operands of a call
  uint32_t* status_dev;
};

namespace {

// Tensor maps of one operand: codes in boxes of `box_rows` rows x 128 bytes, scales in boxes of one row
// group x one stage's tiles.  Bytes behind ceil(k / 2) and tiles behind the last are read as zero.
bool mx_encode_operand(const gz_mx_plan* pl, CUtensorMap* codes_map, CUtensorMap* scales_map, const void* codes,
                       const void* scales, int64_t rows, int64_t pitch, uint32_t box_rows) {
  const gz_mx_desc& d = pl->pr.d;
  const uint64_t groups = (uint64_t)mx_groups(d.format, d.k);
  return mx_encode(codes_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, (uint64_t)cdiv(d.k, 2), (uint64_t)rows, 1, (uint64_t)pitch,
                   (uint64_t)pitch * (uint64_t)rows, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B, true) &&
         mx_encode(scales_map, CU_TENSOR_MAP_DATA_TYPE_INT32, scales, 128, groups, (uint64_t)cdiv(rows, 128), 512,
                   512 * groups, 128, d.format == GZ_MX_NVFP4 ? 4 : 2, CU_TENSOR_MAP_SWIZZLE_NONE, true);
}

// a x b (and, gated, a x up) into p->d; the caller has filled the epilogue's part of *p.
gz_status mx_launch(gz_mx_plan* pl, gz::MxParams* p, const void* a, const void* a_scales, const void* b,
                    const void* b_scales, const void* up, const void* up_scales, cudaStream_t stream) {
  const gz_mx_desc& d = pl->pr.d;
  const MxShape& s = *mx_shape_of(pl->info.config);
  gz::MxMaps maps;
  bool ok;
  if (!s.swap())
    ok = mx_encode_operand(pl, &maps.wide, &maps.wide_scales, a, a_scales, d.m, d.pitch_a, 128) &&
         mx_encode_operand(pl, &maps.narrow, &maps.narrow_scales, b, b_scales, d.n, d.pitch_b,
                           s.bn == 256 ? 128u : (uint32_t)(s.bn / s.ctas));
  else
    ok = mx_encode_operand(pl, &maps.wide, &maps.wide_scales, b, b_scales, d.n, d.pitch_b, 128) &&
         mx_encode_operand(pl, &maps.narrow, &maps.narrow_scales, a, a_scales, d.m, d.pitch_a, (uint32_t)s.bn);
  if (ok && up) ok = mx_encode_operand(pl, &maps.up, &maps.up_scales, up, up_scales, d.n, d.pitch_b, 128);
  if (!ok) return GZ_ERR_CUDA;
  if (!up) {  // unused by the kernel
    maps.up = maps.narrow;
    maps.up_scales = maps.narrow_scales;
  }
  // four columns at a time in the swapped tiles' epilogue
  const int64_t quad = 4 * pl->pr.out_size;
  p->d_vec_ok = (quad != 0 && mx_aligned(p->d, quad) && d.ldd % 4 == 0 && (!p->c || (mx_aligned(p->c, quad) && d.ldc % 4 == 0))) ? 1u : 0u;
  p->out_tma = (pl->info.out_tma && mx_aligned(p->d, 16)) ? 1u : 0u;
  if (p->out_tma) {
    const bool f32 = d.out_type == GZ_DT_F32;
    if (!mx_encode(&maps.d, tmap_type(d.out_type), p->d, (uint64_t)d.n, (uint64_t)d.m, 1, (uint64_t)(d.ldd * pl->pr.out_size),
                   (uint64_t)(d.ldd * pl->pr.out_size) * (uint64_t)d.m, 32, 32,
                   f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, false))
      return GZ_ERR_CUDA;
  } else {
    maps.d = maps.wide;  // unused by the kernel
  }
  if (!cuda_ok(pl->entry.launch(maps, *p, pl->info.grid, s.ctas * pl->info.split, stream), "kernel launch"))
    return GZ_ERR_CUDA;
  return GZ_OK;
}

}  // namespace

extern "C" {

GZ_API int64_t gz_mx_code_pitch(int64_t k) { return k <= 0 || k > kMxExtent ? -1 : cdiv(k, 32) * 16; }

GZ_API int64_t gz_mx_scale_bytes(int32_t format, int64_t rows, int64_t k) {
  if (!is_mx(format) || rows <= 0 || k <= 0 || rows > kMxExtent || k > kMxExtent) return -1;
  return cdiv(rows, 128) * mx_groups(format, k) * 512;
}

GZ_API gz_status gz_mx_quantize(const void* src, int32_t src_type, int32_t layout, int64_t ld, int64_t rows, int64_t k,
                                int32_t format, float multiplier, void* codes, int64_t pitch, void* scales,
                                int32_t device, void* stream) {
  gz::mx::QuantParams p;
  gz_status st = mx_quant_params(&p, src, src_type, layout, ld, rows, k, format, multiplier, codes, pitch, scales, device);
  if (st != GZ_OK) return st;
  const bool nv = format == GZ_MX_NVFP4, cols = layout == GZ_COL_MAJOR;
  DeviceGuard guard(device);
  if (!guard.ok()) return (st = mx_device_ok(device)) != GZ_OK ? st : GZ_ERR_CUDA;
  p.in = src;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint8_t*>(scales);
  if (!cuda_ok(gz::mx_launch_quantize(src_type, nv, cols, p, static_cast<cudaStream_t>(stream)), "kernel launch"))
    return GZ_ERR_CUDA;
  return GZ_OK;
}

GZ_API gz_status gz_mx_dequantize(const void* codes, int64_t pitch, const void* scales, int32_t format, int64_t rows,
                                  int64_t k, float multiplier, void* dst, int32_t dst_type, int32_t layout, int64_t ld,
                                  int32_t device, void* stream) {
  gz::mx::QuantParams p;
  gz_status st = mx_quant_params(&p, dst, dst_type, layout, ld, rows, k, format, multiplier, codes, pitch, scales, device);
  if (st != GZ_OK) return st;
  const bool nv = format == GZ_MX_NVFP4, cols = layout == GZ_COL_MAJOR;
  DeviceGuard guard(device);
  if (!guard.ok()) return (st = mx_device_ok(device)) != GZ_OK ? st : GZ_ERR_CUDA;
  p.out = dst;
  p.pre = !nv && std::fabs(multiplier) < 1.0f ? 0.25f : 1.0f;
  p.multiplier = multiplier / p.pre;
  p.codes = const_cast<uint8_t*>(static_cast<const uint8_t*>(codes));
  p.scales = const_cast<uint8_t*>(static_cast<const uint8_t*>(scales));
  if (!cuda_ok(gz::mx_launch_dequantize(dst_type, nv, cols, p, static_cast<cudaStream_t>(stream)), "kernel launch"))
    return GZ_ERR_CUDA;
  return GZ_OK;
}

GZ_API gz_status gz_mx_desc_validate(const gz_mx_desc* desc, int sm_count, gz_mx_plan_info* info) {
  MxProblem pr;
  gz_status st = mx_normalise(desc, &pr);
  if (st != GZ_OK) return st;
  gz_mx_plan_info tmp;
  st = mx_resolve(pr, sm_count > 0 ? sm_count : 148, &tmp);
  if (st == GZ_OK && info) *info = tmp;
  return st;
}

GZ_API gz_status gz_mx_plan_create(gz_mx_plan** out, const gz_mx_desc* desc) {
  if (!out) return GZ_ERR_INVALID_ARG;
  *out = nullptr;
  MxProblem pr;
  gz_status st = mx_normalise(desc, &pr);
  if (st != GZ_OK) return st;
  if ((st = mx_device_ok(pr.d.device)) != GZ_OK) return st;
  int major = 0, sms = 0;
  if (!cuda_ok(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, pr.d.device), "device attribute") ||
      !cuda_ok(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, pr.d.device), "device attribute"))
    return GZ_ERR_CUDA;
  if (major != 10) return GZ_ERR_NO_DEVICE;
  gz_mx_plan_info info;
  if ((st = mx_resolve(pr, sms, &info)) != GZ_OK) return st;
  DeviceGuard guard(pr.d.device);
  if (!guard.ok()) return GZ_ERR_CUDA;
  gz_mx_plan* pl = new (std::nothrow) gz_mx_plan();
  if (!pl) return GZ_ERR_OUT_OF_MEMORY;
  pl->pr = pr;
  pl->info = info;
  pl->entry = mx_entry_of(pr, info.config);
  pl->status_dev = nullptr;
  if (!cuda_ok(pl->entry.attr(), "cudaFuncSetAttribute(max dynamic shared memory)") ||
      !cuda_ok(cudaMalloc(&pl->status_dev, 4 * sizeof(uint32_t)), "cudaMalloc(status)") ||
      !cuda_ok(cudaMemset(pl->status_dev, 0, 4 * sizeof(uint32_t)), "cudaMemset(status)")) {
    if (pl->status_dev) cudaFree(pl->status_dev);
    delete pl;
    return GZ_ERR_CUDA;
  }
  const gz_mx_desc& d = pl->pr.d;
  const MxShape& s = *mx_shape_of(info.config);
  gz::MxParams& p = pl->base;
  std::memset(&p, 0, sizeof(p));
  p.grid.tiles_m = (uint32_t)(s.swap() ? cdiv(d.n, 128) : cdiv(d.m, 128 * s.ctas));
  p.grid.tiles_n = (uint32_t)(s.swap() ? 1 : cdiv(d.n, info.tile_n));
  p.grid.group_m = s.ctas == 2 ? 8u : 16u;  // about 2048 rows of output per group, as for the 8- and 16-bit tiles
  p.grid.num_tiles = p.grid.tiles_m * p.grid.tiles_n;
  p.m = (uint32_t)d.m;
  p.n = (uint32_t)d.n;
  p.k_blocks = (uint32_t)cdiv(d.k, 256);
  p.split = (uint32_t)info.split;
  // Over 96 chains (1 to 48 rows, N and K 1000 to 32000, both formats, plain and gated) 0 blocks take 0.3 % longer than 2 on
  // average (-6 to +6 %), 8 blocks 1.8 % (-8 to +18 %).  1 x 14336 x 4096, e4m3: 9.8 / 9.6 / 10.4 us for 0 / 2 / 8.
  p.prefetch = 2;
  // e2m1 operands, N, scale type, M
  p.idesc = (1u << 7) | (1u << 10) | ((uint32_t)(s.bn >> 3) << 17) | ((d.format == GZ_MX_FP4 ? 1u : 0u) << 23) |
            ((uint32_t)(8 * s.ctas) << 24);
  p.out_type = (uint32_t)d.out_type;
  p.test_flags = (d.flags & GZ_FLAG_TEST_WITHHOLD_ACC_READY) ? 1u : 0u;
  p.ldc = d.ldc;
  p.ldd = d.ldd;
  p.d_groups = is_mx(d.out_type) ? mx_groups(d.out_type, d.n) : 0;
  p.status = pl->status_dev;
  p.wait_limit_ns = d.wait_limit_ns;
  *out = pl;
  return GZ_OK;
}

GZ_API gz_status gz_mx_plan_destroy(gz_mx_plan* pl) {
  if (!pl) return GZ_ERR_INVALID_ARG;
  DeviceGuard guard(pl->pr.d.device);
  if (pl->status_dev) cudaFree(pl->status_dev);
  delete pl;
  return GZ_OK;
}

GZ_API gz_status gz_mx_plan_info_get(const gz_mx_plan* pl, gz_mx_plan_info* info) {
  if (!pl || !info) return GZ_ERR_INVALID_ARG;
  *info = pl->info;
  return GZ_OK;
}

GZ_API gz_status gz_mx_gemm_run(gz_mx_plan* pl, const void* a, const void* a_scales, const void* b,
                                const void* b_scales, const void* c, void* d, const float* alpha, const float* beta,
                                const gz_epilogue* ep, void* stream) {
  if (!pl || !a || !a_scales || !b || !b_scales || !d || !alpha || !beta || pl->pr.d.gated) return GZ_ERR_INVALID_ARG;
  if (*beta != 0.0f && !c) return GZ_ERR_INVALID_ARG;
  const gz_mx_desc& ds = pl->pr.d;
  const int size = pl->pr.out_size;
  if (d == a || d == b || d == a_scales || d == b_scales) return GZ_ERR_INVALID_ARG;
  if (*beta != 0.0f && c == d && ds.ldc != ds.ldd && ds.m > 1) return GZ_ERR_INVALID_ARG;  // other CTAs' rows of C
  if (!mx_aligned(a, 16) || !mx_aligned(a_scales, 16) || !mx_aligned(b, 16) || !mx_aligned(b_scales, 16) ||
      !mx_aligned(d, size) || !mx_aligned(c, size))
    return GZ_ERR_MISALIGNED;
  gz::MxParams p = pl->base;
  if (ep) {
    if (ep->struct_size != sizeof(gz_epilogue) || ep->activation < GZ_ACT_NONE || ep->activation > GZ_ACT_SILU)
      return GZ_ERR_INVALID_ARG;
    if (d == ep->bias || d == ep->row_scale || d == ep->col_scale) return GZ_ERR_INVALID_ARG;  // read while others write
    if (!mx_aligned(ep->bias, 4) || !mx_aligned(ep->row_scale, 4) || !mx_aligned(ep->col_scale, 4)) return GZ_ERR_MISALIGNED;
    p.epi_flags = (ep->bias ? 1u : 0u) | (ep->row_scale ? 2u : 0u) | (ep->col_scale ? 4u : 0u);
    p.act = (uint32_t)ep->activation;
    p.bias = ep->bias;
    p.row_scale = ep->row_scale;
    p.col_scale = ep->col_scale;
  }
  p.alpha = *alpha;
  p.beta = *beta;
  p.c = *beta != 0.0f ? c : nullptr;
  p.d = d;
  p.c_vec_ok = (p.c && mx_aligned(c, 16) && (ds.ldc * size) % 16 == 0) ? 1u : 0u;
  DeviceGuard guard(ds.device);
  if (!guard.ok()) return GZ_ERR_CUDA;
  return mx_launch(pl, &p, a, a_scales, b, b_scales, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

GZ_API gz_status gz_mx_gated_run(gz_mx_plan* pl, const void* a, const void* a_scales, const void* gate,
                                 const void* gate_scales, const void* up, const void* up_scales, void* d,
                                 void* d_scales, const float* alpha_gate, const float* alpha_up, int32_t activation,
                                 float out_multiplier, void* stream) {
  if (!pl || !a || !a_scales || !gate || !gate_scales || !up || !up_scales || !d || !alpha_gate || !alpha_up ||
      !pl->pr.d.gated || activation < GZ_ACT_NONE || activation > GZ_ACT_SILU)
    return GZ_ERR_INVALID_ARG;
  const bool quantised = pl->pr.out_size == 0;
  if (quantised != (d_scales != nullptr)) return GZ_ERR_INVALID_ARG;
  for (const void* in : {a, a_scales, gate, gate_scales, up, up_scales})  // read while others write
    if (d == in || (d_scales && d_scales == in)) return GZ_ERR_INVALID_ARG;
  if (d == d_scales) return GZ_ERR_INVALID_ARG;
  if (quantised && (!(std::fabs(out_multiplier) <= 3.4028234e38f) || out_multiplier == 0.0f)) return GZ_ERR_INVALID_ARG;
  if (!mx_aligned(a, 16) || !mx_aligned(a_scales, 16) || !mx_aligned(gate, 16) || !mx_aligned(gate_scales, 16) ||
      !mx_aligned(up, 16) || !mx_aligned(up_scales, 16) || !mx_aligned(d, quantised ? 16 : pl->pr.out_size) ||
      !mx_aligned(d_scales, 16))
    return GZ_ERR_MISALIGNED;
  gz::MxParams p = pl->base;
  p.act = (uint32_t)activation;
  p.alpha = *alpha_gate;
  p.alpha_up = *alpha_up;
  p.out_multiplier = out_multiplier;
  p.d = d;
  p.d_scales = static_cast<uint8_t*>(d_scales);
  DeviceGuard guard(pl->pr.d.device);
  if (!guard.ok()) return GZ_ERR_CUDA;
  return mx_launch(pl, &p, a, a_scales, gate, gate_scales, up, up_scales, static_cast<cudaStream_t>(stream));
}

GZ_API gz_status gz_mx_last_device_status(gz_mx_plan* pl, void* stream_v, uint32_t detail[4]) {
  if (!pl) return GZ_ERR_INVALID_ARG;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  DeviceGuard guard(pl->pr.d.device);
  if (!guard.ok()) return GZ_ERR_CUDA;
  uint32_t h[4] = {0, 0, 0, 0};
  if (!cuda_ok(cudaStreamSynchronize(stream), "cudaStreamSynchronize") ||
      !cuda_ok(cudaMemcpy(h, pl->status_dev, sizeof(h), cudaMemcpyDeviceToHost), "read status"))
    return GZ_ERR_CUDA;
  if (detail) std::memcpy(detail, h, sizeof(h));
  if (h[0] == 0) return GZ_OK;
  (void)cudaMemset(pl->status_dev, 0, sizeof(h));
  return h[0] == gz::STORE_OUT_OF_BOUNDS ? GZ_ERR_DEBUG_CHECK : GZ_ERR_DEVICE_TIMEOUT;
}

}  // extern "C"
#endif
