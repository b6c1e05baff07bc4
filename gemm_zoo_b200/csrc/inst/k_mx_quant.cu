// Launchers of the quantising and dequantising kernels.
#include <cstring>

#include "gemmzoo/gemm.h"
#include "mx_quant.cuh"
#include "mx_table.h"

namespace {

template <class K>
cudaError_t launch(K kernel, const gz::mx::QuantParams& p, int64_t blocks, cudaStream_t stream) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, bool NV>
cudaError_t quantize(bool cols, const gz::mx::QuantParams& p, int64_t blocks, cudaStream_t stream) {
  return launch(cols ? gz::mx::quantize_cols_kernel<T, NV> : gz::mx::quantize_rows_kernel<T, NV>, p, blocks, stream);
}
template <typename T, bool NV>
cudaError_t dequantize(bool cols, const gz::mx::QuantParams& p, int64_t blocks, cudaStream_t stream) {
  return launch(cols ? gz::mx::dequantize_cols_kernel<T, NV> : gz::mx::dequantize_rows_kernel<T, NV>, p, blocks, stream);
}

}  // namespace

cudaError_t gz::mx_launch_quantize(int type, bool nv, bool cols, const mx::QuantParams& p, int64_t blocks,
                                   cudaStream_t stream) {
  switch (type) {
    case GZ_DT_F16: return nv ? quantize<__half, true>(cols, p, blocks, stream) : quantize<__half, false>(cols, p, blocks, stream);
    case GZ_DT_BF16:
      return nv ? quantize<__nv_bfloat16, true>(cols, p, blocks, stream) : quantize<__nv_bfloat16, false>(cols, p, blocks, stream);
    default: return nv ? quantize<float, true>(cols, p, blocks, stream) : quantize<float, false>(cols, p, blocks, stream);
  }
}

cudaError_t gz::mx_launch_dequantize(int type, bool nv, bool cols, const mx::QuantParams& p, int64_t blocks,
                                     cudaStream_t stream) {
  switch (type) {
    case GZ_DT_F16: return nv ? dequantize<__half, true>(cols, p, blocks, stream) : dequantize<__half, false>(cols, p, blocks, stream);
    case GZ_DT_BF16:
      return nv ? dequantize<__nv_bfloat16, true>(cols, p, blocks, stream) : dequantize<__nv_bfloat16, false>(cols, p, blocks, stream);
    default: return nv ? dequantize<float, true>(cols, p, blocks, stream) : dequantize<float, false>(cols, p, blocks, stream);
  }
}
