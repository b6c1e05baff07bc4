// Launchers of the quantising and dequantising kernels.
#include <cstring>

#include "gemmzoo/gemm.h"
#include "mx_quant.cuh"
#include "mx_table.h"

namespace {

template <class K>
cudaError_t launch(K kernel, const gz::mx::QuantParams& p, dim3 grid, int threads, cudaStream_t stream, int smem = 0) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// `pieces` of K on grid.y (and z beyond 32768), rows on grid.x.
dim3 grid_of(int64_t rows, int64_t pieces) {
  const int64_t y = pieces < 32768 ? pieces : 32768;
  return dim3(static_cast<unsigned>(rows), static_cast<unsigned>(y), static_cast<unsigned>((pieces + y - 1) / y));
}

// Row layout: the 16-element chunks of a row (`chunks`, in whole words of `word`) over equal pieces of
// at most 256 threads, and as many rows as fit a block of 256.
template <class K>
cudaError_t launch_rows(K kernel, gz::mx::QuantParams p, int64_t rows, int64_t chunks, int64_t word, cudaStream_t stream, int smem = 0) {
  const int64_t pieces = (chunks + 255) / 256;
  const int64_t threads = ((chunks + pieces - 1) / pieces + word - 1) / word * word;
  p.row_threads = static_cast<uint32_t>(threads);
  p.inv_threads = static_cast<uint32_t>((65536 + threads - 1) / threads);
  p.block_rows = static_cast<uint32_t>(256 / threads);
  const int64_t per_block = static_cast<int64_t>(p.block_rows) * gz::mx::ROWS_PER_THREAD;
  return launch(kernel, p, grid_of((rows + per_block - 1) / per_block, pieces),
                static_cast<int>((p.block_rows * threads + 31) / 32 * 32), stream, smem);
}

template <typename T, bool NV>
cudaError_t quantize(bool cols, const gz::mx::QuantParams& p, cudaStream_t stream) {
  const int64_t padded = (p.rows + 127) / 128 * 128;  // the scale array's rows
  if (!cols) return launch_rows(gz::mx::quantize_rows_kernel<T, NV>, p, padded, p.groups * (NV ? 4 : 8), NV ? 4 : 8, stream);
  using Tile = gz::mx::ColTile<T>;
  return launch(p.vec == 32u ? gz::mx::quantize_cols_kernel<T, NV, true> : gz::mx::quantize_cols_kernel<T, NV, false>, p,
                grid_of(padded / Tile::ROWS, (p.k + gz::mx::COL_K - 1) / gz::mx::COL_K), Tile::THREADS, stream);
}
template <typename T, bool NV>
cudaError_t dequantize(bool cols, const gz::mx::QuantParams& p, cudaStream_t stream) {
  if (!cols) return launch_rows(gz::mx::dequantize_rows_kernel<T, NV>, p, p.rows, (p.k + 15) / 16, 1, stream,
                                p.vec ? 0 : 256 * 16 * static_cast<int>(sizeof(T)));
  using Tile = gz::mx::ColTile<T>;
  return launch(gz::mx::dequantize_cols_kernel<T, NV>, p,
                grid_of((p.rows + Tile::ROWS - 1) / Tile::ROWS, (p.k + gz::mx::COL_K - 1) / gz::mx::COL_K), Tile::THREADS, stream);
}

}  // namespace

cudaError_t gz::mx_launch_quantize(int type, bool nv, bool cols, const mx::QuantParams& p, cudaStream_t stream) {
  switch (type) {
    case GZ_DT_F16: return nv ? quantize<__half, true>(cols, p, stream) : quantize<__half, false>(cols, p, stream);
    case GZ_DT_BF16:
      return nv ? quantize<__nv_bfloat16, true>(cols, p, stream) : quantize<__nv_bfloat16, false>(cols, p, stream);
    default: return nv ? quantize<float, true>(cols, p, stream) : quantize<float, false>(cols, p, stream);
  }
}

cudaError_t gz::mx_launch_dequantize(int type, bool nv, bool cols, const mx::QuantParams& p, cudaStream_t stream) {
  switch (type) {
    case GZ_DT_F16: return nv ? dequantize<__half, true>(cols, p, stream) : dequantize<__half, false>(cols, p, stream);
    case GZ_DT_BF16:
      return nv ? dequantize<__nv_bfloat16, true>(cols, p, stream) : dequantize<__nv_bfloat16, false>(cols, p, stream);
    default: return nv ? dequantize<float, true>(cols, p, stream) : dequantize<float, false>(cols, p, stream);
  }
}
