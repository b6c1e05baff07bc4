// Launch table of the microscaled 4-bit kernels (instantiated in csrc/inst/k_mx_*.cu; the host layer
// sees only these functions).
#ifndef GZ_MX_TABLE_H
#define GZ_MX_TABLE_H

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace gz {

struct MxMaps;
struct MxParams;
namespace mx {
struct QuantParams;
}

struct MxEntry {
  // cluster: CTAs per cluster (CTAs of a tile x CTAs or pairs that share its K range)
  cudaError_t (*launch)(const MxMaps&, const MxParams&, int grid, int cluster, cudaStream_t);
  cudaError_t (*attr)();
  int stages, smem_bytes;
};

// config: a gz_mx_config naming a tile family.  All-null entry = no such tile.
MxEntry mx_kernels_fp4(int config, bool gated);
MxEntry mx_kernels_nvfp4(int config, bool gated);

// type: GZ_DT_F16, GZ_DT_BF16 or GZ_DT_F32; cols: the values have K strided.
cudaError_t mx_launch_quantize(int type, bool nv, bool cols, const mx::QuantParams& p, cudaStream_t stream);
cudaError_t mx_launch_dequantize(int type, bool nv, bool cols, const mx::QuantParams& p, cudaStream_t stream);

}  // namespace gz
#endif
