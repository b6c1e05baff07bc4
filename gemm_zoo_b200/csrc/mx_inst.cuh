// Instantiates mx_gemm_kernel for every tile of one format.  Included by csrc/inst/k_mx_fp4.cu and
// k_mx_nvfp4.cu.
#ifndef GZ_MX_INST_CUH
#define GZ_MX_INST_CUH

#include <cstring>

#include "gemmzoo/microscale.h"
#include "mx_gemm.cuh"
#include "mx_table.h"

namespace gz {
namespace inst {

template <class Cfg>
cudaError_t mx_set_attr() {
  return cudaFuncSetAttribute(mx_gemm_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
}

template <class Cfg>
cudaError_t mx_launch(const MxMaps& maps, const MxParams& p, int grid, int cluster, cudaStream_t stream) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(Cfg::THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as in kernel_inst.cuh
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, mx_gemm_kernel<Cfg>, maps, p);
}

template <bool NV, int BN, int CTAS>
MxEntry mx_entry(bool gated) {
  using G = MxCfg<NV, BN, CTAS, true>;
  using P = MxCfg<NV, BN, CTAS, false>;
  if (gated) return {mx_launch<G>, mx_set_attr<G>, G::STAGES, G::SMEM_BYTES};
  return {mx_launch<P>, mx_set_attr<P>, P::STAGES, P::SMEM_BYTES};
}

template <bool NV, int BN, int CTAS>
MxEntry mx_entry_plain(bool gated) {
  using P = MxCfg<NV, BN, CTAS, false>;
  if (gated) return {nullptr, nullptr, 0, 0};
  return {mx_launch<P>, mx_set_attr<P>, P::STAGES, P::SMEM_BYTES};
}

template <bool NV>
MxEntry mx_entry_for(int config, bool gated) {
  switch (config) {
    case GZ_MX_CFG_PAIR_N128: return mx_entry_plain<NV, 128, 2>(gated);
    case GZ_MX_CFG_SINGLE_N128: return mx_entry_plain<NV, 128, 1>(gated);
    case GZ_MX_CFG_PAIR: return mx_entry<NV, 256, 2>(gated);
    case GZ_MX_CFG_SINGLE: return mx_entry<NV, 256, 1>(gated);
    case GZ_MX_CFG_SWAP_M16: return mx_entry<NV, 16, 1>(gated);
    case GZ_MX_CFG_SWAP_M32: return mx_entry<NV, 32, 1>(gated);
    case GZ_MX_CFG_SWAP_M64: return mx_entry<NV, 64, 1>(gated);
  }
  return {nullptr, nullptr, 0, 0};
}

}  // namespace inst
}  // namespace gz
#endif
