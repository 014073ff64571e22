// paged_attention_f16.cu -- the paged attention kernels for f16 queries.
#include "paged_attention_launch.cuh"

namespace clove {
namespace rt {

CLOVE_DEFINE_ERROR_READER(read_clear_error_paged_f16)

int launch_paged_attention_f16(kern::PagedAttnParams& p, int head_dim, int heads, bool e4m3, int ctas,
                               const DeviceInfo& dev, cudaStream_t stream) {
  return e4m3 ? paged::dispatch<__half, true>(p, head_dim, heads, ctas, dev, stream)
              : paged::dispatch<__half, false>(p, head_dim, heads, ctas, dev, stream);
}

namespace {
template <bool F8, int D, int NT>
constexpr int ctas_per_sm() {
  return kern::PagedShape<F8, D, NT>::CTAS_PER_SM;
}
}  // namespace

// CTAs that fit on the device at once.
int paged_attention_max_ctas(int head_dim, int heads, bool f8, const DeviceInfo& dev) {
  int k;
  if (head_dim == 64)
    k = heads == 16 ? (f8 ? ctas_per_sm<true, 64, 2>() : ctas_per_sm<false, 64, 2>())
                    : (f8 ? ctas_per_sm<true, 64, 1>() : ctas_per_sm<false, 64, 1>());
  else if (head_dim == 128)
    k = heads == 16 ? (f8 ? ctas_per_sm<true, 128, 2>() : ctas_per_sm<false, 128, 2>())
                    : (f8 ? ctas_per_sm<true, 128, 1>() : ctas_per_sm<false, 128, 1>());
  else
    k = f8 ? ctas_per_sm<true, 256, 1>() : ctas_per_sm<false, 256, 1>();
  return k * dev.num_sms;
}

}  // namespace rt
}  // namespace clove
