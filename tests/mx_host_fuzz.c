/* Driver of tests/test_microscale_sanitizers.py: calls every entry point of include/gemmzoo/microscale.h that can be
 * reached without a GPU with many seeded arguments (valid ones, edge sizes, garbage) under AddressSanitizer and
 * UndefinedBehaviorSanitizer.  Calls whose arguments are accepted get addresses that nothing may touch: without a GPU
 * they must answer GZ_ERR_NO_DEVICE. */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "gemmzoo/microscale.h"

static uint64_t state = 0x9E3779B97F4A7C15ull;
static uint64_t rnd(void) {
  state ^= state << 13;
  state ^= state >> 7;
  state ^= state << 17;
  return state;
}

int main(void) {
  static const int64_t sizes[] = {1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 255, 256, 257, 1000, 4096, 8192, 14336, 100000,
                                  (int64_t)1 << 30, 2147482623, 2147482624, 2147483647, (int64_t)1 << 40, INT64_MAX};
  const int nsizes = (int)(sizeof(sizes) / sizeof(sizes[0]));
  static const int sms[] = {0, 1, 2, 3, 74, 132, 148, 160};
  long ok = 0, rejected = 0;
  for (int it = 0; it < 40000; ++it) {
    const int garbage = (it % 4) == 3;
    gz_mx_desc d;
    memset(&d, 0, sizeof d);
    d.struct_size = garbage && rnd() % 8 == 0 ? (uint32_t)(rnd() % 200) : (uint32_t)sizeof d;
    d.format = garbage ? (int)(rnd() % 20) - 1 : 16 + (int)(rnd() % 2);
    d.gated = garbage ? (int)(rnd() % 4) - 1 : (int)(rnd() % 2);
    d.out_type = garbage ? (int)(rnd() % 20) - 1 : (rnd() % 4 == 0 && d.gated) ? 16 + (int)(rnd() % 2) : (int)(rnd() % 3);
    d.config = garbage ? (int)(rnd() % 12) - 2 : (rnd() % 3) ? 0 : (int)(rnd() % 8);
    d.split = garbage ? (int)(rnd() % 12) - 2 : (rnd() % 3) ? 0 : 1 << (rnd() % 4);
    d.device = garbage && rnd() % 8 == 0 ? -1 : 0;
    d.flags = garbage && rnd() % 4 == 0 ? (uint32_t)rnd() : 0;
    d.m = garbage ? (int64_t)rnd() : sizes[rnd() % nsizes];
    d.n = sizes[rnd() % nsizes];
    d.k = sizes[rnd() % nsizes];
    if (rnd() % 4 == 0) d.pitch_a = (int64_t)(rnd() % 65536);
    if (rnd() % 4 == 0) d.pitch_b = garbage ? (int64_t)rnd() : (int64_t)(rnd() % 65536) * 16;
    if (rnd() % 4 == 0) d.ldc = garbage ? (int64_t)rnd() : (int64_t)(rnd() % 65536);
    if (rnd() % 4 == 0) d.ldd = garbage ? (int64_t)rnd() : (int64_t)(rnd() % 65536);
    gz_mx_plan_info info;
    memset(&info, 0, sizeof info);
    const gz_status st = gz_mx_desc_validate(&d, sms[rnd() % 8], rnd() % 8 ? &info : NULL);
    if (st == GZ_OK) ++ok;
    else ++rejected;
    if (gz_status_string(st) == NULL) return 2;
    if (st == GZ_OK && info.tiles != 0 && (info.grid <= 0 || info.split < 1 || info.smem_bytes > 232448)) {
      printf("bad geometry: grid %d split %d\n", info.grid, info.split);
      return 3;
    }
    if (it % 50 == 0) {
      gz_mx_plan* plan = NULL;
      const gz_status pc = gz_mx_plan_create(&plan, &d);
      if (pc == GZ_OK) gz_mx_plan_destroy(plan);
    }
    const int64_t rows = garbage ? (int64_t)rnd() : sizes[rnd() % nsizes], k = sizes[rnd() % nsizes];
    const int64_t bytes = gz_mx_scale_bytes((int)(rnd() % 20), rows, k), pitch = gz_mx_code_pitch(rows);
    if (bytes == 0 || bytes < -1 || pitch == 0 || pitch < -1 || (pitch > 0 && pitch % 16 != 0)) return 4;
    static const float multipliers[] = {1.0f, 0.0f, -2.0f, 1e38f, 1e-45f};
    float mult = multipliers[rnd() % 5];
    if (rnd() % 16 == 0) mult = NAN;
    if (rnd() % 16 == 0) mult = INFINITY;
    char* const base = (char*)(uintptr_t)0x100000;
    const void* src = rnd() % 8 ? base + (rnd() % 4 == 0 ? rnd() % 64 : 0) : NULL;
    void* codes = rnd() % 8 ? base + 4096 + (rnd() % 4 == 0 ? rnd() % 64 : 0) : NULL;
    void* scales = rnd() % 8 ? base + 8192 + (rnd() % 4 == 0 ? rnd() % 64 : 0) : NULL;
    /* a device that does not exist anywhere: accepted arguments must end in an error, not in a launch */
    const int device = 4096;
    const gz_status q = gz_mx_quantize(src, (int)(rnd() % 9) - 1, (int)(rnd() % 3), rnd() % 2 ? 0 : (int64_t)(rnd() % 70000), rows, k,
                                       (int)(rnd() % 20), mult, codes, rnd() % 2 ? 0 : (int64_t)(rnd() % 4096) * 16, scales, device, NULL);
    const gz_status u = gz_mx_dequantize(codes, rnd() % 2 ? 0 : (int64_t)(rnd() % 4096) * 16, scales, (int)(rnd() % 20), rows, k, mult,
                                         (void*)src, (int)(rnd() % 9) - 1, (int)(rnd() % 3), 0, device, NULL);
    if (q == GZ_OK || u == GZ_OK) return 5;
  }
  if (gz_mx_gemm_run(NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL) != GZ_ERR_INVALID_ARG) return 6;
  if (gz_mx_gated_run(NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, 0, 1.0f, NULL) != GZ_ERR_INVALID_ARG) return 7;
  printf("accepted %ld rejected %ld\nMX HOST FUZZ OK\n", ok, rejected);
  return ok > 100 && rejected > 100 ? 0 : 8;
}
