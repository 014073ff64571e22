// paged_attention_launch.cuh -- host launchers of the paged attention kernels for one
// 16-bit type; instantiated by paged_attention_f16.cu and paged_attention_bf16.cu.
#pragma once

#include <algorithm>
#include <atomic>

#include "../runtime/internal.h"
#include "paged_attention_sm100.cuh"
#include "pdl_launch.h"

namespace clove {
namespace rt {
namespace paged {

template <typename T, bool F8, int D, int NT>
int launch(kern::PagedAttnParams& p, int ctas, const DeviceInfo& dev, cudaStream_t stream) {
  using S = kern::PagedShape<F8, D, NT>;
  static std::atomic<uint64_t> attr{0};
  const uint64_t bit = 1ull << (dev.device & 63);
  auto* fn = &kern::paged_attention_kernel<T, F8, D, NT>;
  if ((attr.load(std::memory_order_acquire) & bit) == 0) {
    const int rc = check_cuda(
        cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM),
        "cudaFuncSetAttribute(paged attention smem)");
    if (rc) return rc;
    attr.fetch_or(bit, std::memory_order_acq_rel);
  }
  cudaLaunchAttribute la[1];
  cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(ctas)), S::THREADS, S::SMEM, stream, la);
  const int rc = check_cuda(cudaLaunchKernelEx(&cfg, fn, p), "paged attention launch");
  if (rc || p.key_weights == nullptr) return rc;
  return launch_paged_key_weights(p, stream);
}

template <typename T, bool F8>
int dispatch(kern::PagedAttnParams& p, int head_dim, int heads, int ctas, const DeviceInfo& dev,
             cudaStream_t stream) {
  if (head_dim == 64)
    return heads == 16 ? launch<T, F8, 64, 2>(p, ctas, dev, stream)
                       : launch<T, F8, 64, 1>(p, ctas, dev, stream);
  if (head_dim == 128)
    return heads == 16 ? launch<T, F8, 128, 2>(p, ctas, dev, stream)
                       : launch<T, F8, 128, 1>(p, ctas, dev, stream);
  return launch<T, F8, 256, 1>(p, ctas, dev, stream);
}

}  // namespace paged
}  // namespace rt
}  // namespace clove
