// paged_attention_bf16.cu -- the paged attention kernels for bf16 queries.
#include "paged_attention_launch.cuh"

namespace clove {
namespace rt {

CLOVE_DEFINE_ERROR_READER(read_clear_error_paged_bf16)

int launch_paged_attention_bf16(kern::PagedAttnParams& p, int head_dim, int heads, bool e4m3, int ctas,
                               const DeviceInfo& dev, cudaStream_t stream) {
  return e4m3 ? paged::dispatch<__nv_bfloat16, true>(p, head_dim, heads, ctas, dev, stream)
              : paged::dispatch<__nv_bfloat16, false>(p, head_dim, heads, ctas, dev, stream);
}

}  // namespace rt
}  // namespace clove
