// paged_key_weights.cu -- the weight that each cached key received, from the scores that
// the attention kernel stored.
#include <algorithm>

#include "../runtime/internal.h"
#include "paged_cache.cuh"
#include "pdl_launch.h"

namespace clove {
namespace kern {

// Key weights from the stored scores: w_t = sum over the group of 2^(s_t - LSE2), written
// to (or added to) the key's place in the paged weights. Reads 4 bytes per head and key, and
// is bound by its few dependent loads: with the scores' stores it adds 8 us to 38 us of
// attention (8 sequences of up to 20000 keys, 32 / 8 heads), 2 to 3 us to a small call.
__global__ void __launch_bounds__(256) paged_key_weights_kernel(const PagedAttnParams p) {
  dev::grid_dependency_wait();
  const int page_mask = (1 << p.cache.page_shift) - 1;
  const long long rows = static_cast<long long>(p.batch) * p.cache.kv_heads;
  for (long long bh = blockIdx.y; bh < rows; bh += gridDim.y) {
    const int b = static_cast<int>(bh / p.cache.kv_heads);
    const int h = static_cast<int>(bh - static_cast<long long>(b) * p.cache.kv_heads);
    const PagedSpan s = paged_span<kPagedTile>(p, b);
    const float* lse2 = p.lse2 + static_cast<long long>(b) * p.heads + h * p.group;
    for (int t = s.first + static_cast<int>(blockIdx.x * blockDim.x + threadIdx.x); t < s.len;
         t += static_cast<int>(gridDim.x * blockDim.x)) {
      const float* sc = p.scores + (bh * p.capacity + t) * p.group;
      float w = 0.f;
      if ((p.group & 3) == 0) {
        for (int g = 0; g < p.group; g += 4) {
          const float4 x = *reinterpret_cast<const float4*>(sc + g);
          w += dev::ex2_approx(x.x - lse2[g]) + dev::ex2_approx(x.y - lse2[g + 1]) +
               dev::ex2_approx(x.z - lse2[g + 2]) + dev::ex2_approx(x.w - lse2[g + 3]);
        }
      } else {
        for (int g = 0; g < p.group; ++g) w += dev::ex2_approx(sc[g] - lse2[g]);
      }
      const int pg = p.page_table[b * p.table_stride + (t >> p.cache.page_shift)];
      if (pg < 0 || pg >= p.cache.num_pages) continue;  // reported by the attention kernel
      float* to = p.key_weights +
                  ((static_cast<long long>(pg) * p.cache.kv_heads + h) << p.cache.page_shift) +
                  (t & page_mask);
      *to = p.accumulate ? *to + w : w;
    }
  }
}

// Counters of the attention kernel (PagedAttnParams::counters), zero between calls; handed
// out by the host.
__device__ unsigned g_paged_counters[kPagedCounters];

}  // namespace kern

namespace rt {

int paged_counter_base(unsigned** out) {
  return check_cuda(cudaGetSymbolAddress(reinterpret_cast<void**>(out), kern::g_paged_counters),
                    "cudaGetSymbolAddress(paged counters)");
}

int launch_paged_key_weights(const kern::PagedAttnParams& p, cudaStream_t stream) {
  const long long rows = static_cast<long long>(p.batch) * p.cache.kv_heads;
  const unsigned strips = static_cast<unsigned>(std::max(1, std::min((p.capacity + 255) / 256, 64)));
  cudaLaunchAttribute la[1];
  cudaLaunchConfig_t cfg = pdl_config(
      dim3(strips, static_cast<unsigned>(std::min<long long>(rows, 65535))), 256, 0, stream, la);
  return check_cuda(cudaLaunchKernelEx(&cfg, &kern::paged_key_weights_kernel, p),
                    "paged key weights launch");
}

}  // namespace rt
}  // namespace clove
