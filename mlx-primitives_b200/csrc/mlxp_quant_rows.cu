// mlxp_quant_rows.cu — launches of the many-row kernel of attention over an 8-bit paged cache.

#include <cuda_runtime.h>

#include <atomic>

#include "../../include/mlxp_attn.h"
#include "host_common.h"
#include "quant_attn_rows.cuh"

namespace mlxp {
namespace {

template <typename T, int D, bool INT8>
int launch(const QaParams& p, unsigned grid, cudaStream_t s) {
  auto kernel = quant_attn_rows_kernel<T, D, INT8>;
  static std::atomic<unsigned long long> attr_done{0};  // one bit per device
  int dev;
  if (int rc = current_device(dev)) return rc;
  cudaError_t e;
  if (!(attr_done.load() >> dev & 1ull)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, QrCfg<D>::SMEM);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(quantized paged attention, rows)");
    attr_done.fetch_or(1ull << dev);
  }
  kernel<<<grid, kQrThreads, QrCfg<D>::SMEM, s>>>(p);
  e = cudaGetLastError();
  return e == cudaSuccess ? MLXP_OK : cuda_fail(e, "quantized paged attention launch (rows)");
}

template <typename T>
int launch_t(int64_t D, bool int8, const QaParams& p, unsigned grid, cudaStream_t s) {
  if (D == 128) return int8 ? launch<T, 128, true>(p, grid, s) : launch<T, 128, false>(p, grid, s);
  return int8 ? launch<T, 64, true>(p, grid, s) : launch<T, 64, false>(p, grid, s);
}

}  // namespace

int qa_rows_launch(int64_t dtype, int64_t D, bool int8, const QaParams& p, unsigned grid, cudaStream_t s) {
  return dtype == MLXP_DTYPE_BF16 ? launch_t<__nv_bfloat16>(D, int8, p, grid, s)
                                  : launch_t<__half>(D, int8, p, grid, s);
}

}  // namespace mlxp
