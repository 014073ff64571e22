// evict_cache.cu -- eviction from a paged cache by accumulated key weight.
//
// For each (sequence, key head) with n keys and a budget of B: n <= B keeps everything;
// otherwise the last `recent` keys stay, and of the others the B - recent with the largest
// weights, ties to the lowest index. Kept keys (K, V and weight) are copied in their order
// to the slots of a second page table.
//
// Two kernels. The selection: one cluster per (sequence, key head), each CTA holding a
// contiguous slice of the weights in shared memory as order-preserving integers, so that
// they are read once; a radix select of four 8-bit digits over histograms that the CTAs
// add up through distributed shared memory (one cluster barrier per digit), then an
// ordered compaction by ballots. Integer counts only: the result does not depend on
// timing. The copy: bound by memory, 16 bytes per lane, four rows per lane in flight.
#include <algorithm>
#include <atomic>

#include "../runtime/internal.h"
#include "paged_cache.cuh"
#include "pdl_launch.h"

namespace clove {
namespace kern {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWarps = kEvictThreads / 32;
// Keys of a slice held in shared memory (96 KB: two CTAs per SM); a longer slice reads the
// rest again from memory in every pass.
constexpr int kEvictCached = 24576;

// Larger weight <=> larger integer; -0 equals 0; every NaN above everything.
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint32_t ld_cluster_u32(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  const uint32_t a = dev::map_shared_to_rank(dev::smem_u32(p), rank);
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

__global__ void __launch_bounds__(kEvictThreads, 2) evict_select_kernel(const EvictParams p, int cs) {
  extern __shared__ uint32_t cached[];
  __shared__ uint32_t hist[2][256];
  __shared__ uint32_t sums[256];
  __shared__ uint32_t counts[2];  // this CTA's keys above the threshold, and equal to it
  __shared__ uint32_t warp_eq[2][kEvictWarps], warp_take[2][kEvictWarps];
  __shared__ uint32_t pick[2];  // chosen digit, keys of larger digits
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = blockIdx.x % cs;
  const long long row = blockIdx.x / cs;
  const int b = static_cast<int>(row / p.cache.kv_heads);
  const int h = static_cast<int>(row - static_cast<long long>(b) * p.cache.kv_heads);
  const int page_mask = (1 << p.cache.page_shift) - 1;
  dev::grid_dependency_wait();
  dev::allow_dependent_launch();
  int n = p.seq_lens[b];
  if (n < 0 || n > p.capacity) {
    if (tid == 0) dev::record_error(dev::kDevErrBadIndex);
    n = n < 0 ? 0 : p.capacity;
  }
  int* kept = p.kept + row * p.budget;
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = min(n, p.budget);
  if (n <= p.budget) {
    for (int j = static_cast<int>(rank) * kEvictThreads + tid; j < p.budget; j += cs * kEvictThreads)
      kept[j] = j < n ? j : -1;
    return;  // the whole cluster
  }
  // Candidates [0, m), `want` of them to keep; slice [s0, s1) of this CTA.
  const int m = n - p.recent, want = p.budget - p.recent;
  const int per = (m + cs - 1) / cs;
  const int s0 = min(m, static_cast<int>(rank) * per), s1 = min(m, s0 + per), sn = s1 - s0;
  auto load = [&](int t) {
    const int pg = p.page_table[b * p.table_stride + (t >> p.cache.page_shift)];
    if (pg < 0 || pg >= p.cache.num_pages) {
      dev::record_error(dev::kDevErrBadIndex);
      return weight_order(0.f);
    }
    return weight_order(p.key_weights[((static_cast<long long>(pg) * p.cache.kv_heads + h)
                                       << p.cache.page_shift) +
                                      (t & page_mask)]);
  };
  if (tid < 256) hist[0][tid] = 0;
  const int in_smem = min(sn, kEvictCached);
#pragma unroll 4
  for (int i = tid; i < in_smem; i += kEvictThreads) cached[i] = load(s0 + i);
  __syncthreads();
  auto key = [&](int i) { return i < in_smem ? cached[i] : load(s0 + i); };

  uint32_t prefix = 0;  // digits chosen so far
  uint32_t left = static_cast<uint32_t>(want), above = 0;
  for (int d = 0; d < 4; ++d) {
    const int shift = 24 - 8 * d;
    uint32_t* mine = hist[d & 1];
    for (int i = tid; i < sn; i += kEvictThreads) {
      const uint32_t u = key(i);
      if (d == 0 || (u >> (shift + 8)) == prefix) atomicAdd(&mine[(u >> shift) & 255u], 1u);
    }
    // All CTAs' histograms of this digit are complete, and those of the digit before have
    // been read.
    dev::cluster_sync_all();
    uint32_t sum = 0;
    if (tid < 256) {
      for (int r = 0; r < cs; ++r) sum += ld_cluster_u32(&mine[tid], static_cast<uint32_t>(r));
      sums[tid] = sum;
      hist[(d & 1) ^ 1][tid] = 0;
    }
    __syncthreads();
    // Warp 0: the digit in which the `left`-th largest key lies. Lane l holds digits
    // 255 - 8 l - e, from the largest down.
    if (warp == 0) {
      uint32_t own = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) own += sums[255 - 8 * lane - e];
      uint32_t inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      uint32_t run = inc - own;
      const bool here = run < left && inc >= left;
      if (here) {
        for (int e = 0; e < 8; ++e) {
          const uint32_t c = sums[255 - 8 * lane - e];
          if (run + c >= left) {
            pick[0] = static_cast<uint32_t>(255 - 8 * lane - e);
            pick[1] = run;
            break;
          }
          run += c;
        }
      }
      // left == 0: nothing above the largest digit is wanted.
      if (left == 0 && lane == 0) pick[0] = 255u, pick[1] = 0u;
    }
    __syncthreads();
    const uint32_t digit = pick[0];
    // This CTA's keys above the chosen digit (the others' likewise, in their CTAs).
    if (warp == 0) {
      uint32_t c = 0;
      for (uint32_t x = digit + 1 + lane; x < 256; x += 32) c += mine[x];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
      above += c;
      if (d == 3 && lane == 0) {
        counts[0] = above;
        counts[1] = mine[digit];
      }
    }
    left -= pick[1];
    prefix = (prefix << 8) | digit;
    __syncthreads();
  }
  dev::cluster_sync_all();
  // `left` keys equal to the threshold are kept, the first ones. What the slices before
  // this one keep:
  uint32_t eq_before = 0, out = 0;
  for (uint32_t r = 0; r < rank; ++r) {
    const uint32_t gt = ld_cluster_u32(&counts[0], r), eq = ld_cluster_u32(&counts[1], r);
    out += gt + min(eq, left - min(left, eq_before));
    eq_before += eq;
  }
  dev::cluster_sync_all();  // no CTA leaves while its counts may be read
  for (int base = 0, it = 0; base < sn; base += kEvictThreads, ++it) {
    const int i = base + tid;
    const uint32_t u = i < sn ? key(i) : 0u;
    const bool gt = i < sn && u > prefix, eq = i < sn && u == prefix;
    const unsigned eq_b = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) warp_eq[it & 1][warp] = __popc(eq_b);
    __syncthreads();
    // Equal keys in the warps before this one, and in the strip.
    const uint32_t ew = warp_eq[it & 1][lane];
    uint32_t e_inc = ew;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, e_inc, o);
      if (lane >= o) e_inc += v;
    }
    const uint32_t e_warp = __shfl_sync(0xffffffffu, e_inc - ew, warp);
    const uint32_t e_all = __shfl_sync(0xffffffffu, e_inc, 31);
    const uint32_t e_rank = eq_before + e_warp + __popc(eq_b & ((1u << lane) - 1u));
    const bool take = gt || (eq && e_rank < left);
    const unsigned tk = __ballot_sync(0xffffffffu, take);
    if (lane == 0) warp_take[it & 1][warp] = __popc(tk);
    __syncthreads();
    const uint32_t tw = warp_take[it & 1][lane];
    uint32_t t_inc = tw;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, t_inc, o);
      if (lane >= o) t_inc += v;
    }
    const uint32_t t_warp = __shfl_sync(0xffffffffu, t_inc - tw, warp);
    const uint32_t t_all = __shfl_sync(0xffffffffu, t_inc, 31);
    if (take) kept[out + t_warp + __popc(tk & ((1u << lane) - 1u))] = s0 + i;
    out += t_all;
    eq_before += e_all;
  }
  // The recent keys.
  for (int j = static_cast<int>(rank) * kEvictThreads + tid; j < p.recent; j += cs * kEvictThreads)
    kept[want + j] = m + j;
}

// LPR lanes of 16 bytes per row; ROWS rows of one (sequence, head) per lane.
template <int LPR, int ROWS>
__global__ void __launch_bounds__(256) evict_copy_kernel(const EvictParams p, int strips) {
  constexpr int PER = 256 / LPR;  // rows at a time
  const int piece = static_cast<int>(threadIdx.x) % LPR, slot = static_cast<int>(threadIdx.x) / LPR;
  const long long row = blockIdx.x / strips;
  const int strip = static_cast<int>(blockIdx.x - row * strips);
  const int b = static_cast<int>(row / p.cache.kv_heads);
  const int h = static_cast<int>(row - static_cast<long long>(b) * p.cache.kv_heads);
  const int page_mask = (1 << p.cache.page_shift) - 1;
  dev::grid_dependency_wait();
  const int j0 = strip * (PER * ROWS) + slot;
  const int* kept = p.kept + row * p.budget;
  long long src[ROWS], dst[ROWS];  // element offsets, -1: no row
  long long wsrc[ROWS], wdst[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int j = j0 + i * PER;
    src[i] = -1;
    const int t = j < p.budget ? kept[j] : -1;
    if (t < 0) continue;
    const int sp = p.page_table[b * p.table_stride + (t >> p.cache.page_shift)];
    const int dp = p.dst_table[b * p.dst_stride + (j >> p.cache.page_shift)];
    if (sp < 0 || sp >= p.cache.num_pages || dp < 0 || dp >= p.cache.num_pages) {
      dev::record_error(dev::kDevErrBadIndex);
      continue;
    }
    src[i] = sp * p.cache.page_stride + (t & page_mask) * p.cache.token_stride + h * p.cache.head_stride;
    dst[i] = dp * p.cache.page_stride + (j & page_mask) * p.cache.token_stride + h * p.cache.head_stride;
    wsrc[i] = ((static_cast<long long>(sp) * p.cache.kv_heads + h) << p.cache.page_shift) + (t & page_mask);
    wdst[i] = ((static_cast<long long>(dp) * p.cache.kv_heads + h) << p.cache.page_shift) + (j & page_mask);
  }
  const char* k = static_cast<const char*>(p.cache.K) + piece * 16;
  const char* v = static_cast<const char*>(p.cache.V) + piece * 16;
  uint4 kr[ROWS], vr[ROWS];
  float w[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (src[i] < 0) continue;
    kr[i] = *reinterpret_cast<const uint4*>(k + src[i] * p.elem);
    vr[i] = *reinterpret_cast<const uint4*>(v + src[i] * p.elem);
    w[i] = p.key_weights[wsrc[i]];
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (src[i] < 0) continue;
    *reinterpret_cast<uint4*>(const_cast<char*>(k) + dst[i] * p.elem) = kr[i];
    *reinterpret_cast<uint4*>(const_cast<char*>(v) + dst[i] * p.elem) = vr[i];
    if (piece == 0) p.key_weights[wdst[i]] = w[i];
  }
}

}  // namespace kern

namespace rt {

CLOVE_DEFINE_ERROR_READER(read_clear_error_evict)

namespace {

std::atomic<uint64_t> g_evict_attr{0};

template <int LPR>
int launch_copy(const kern::EvictParams& p, cudaStream_t stream) {
  constexpr int kRows = 4;
  const int per = 256 / LPR * kRows;
  const int strips = (p.budget + per - 1) / per;
  const long long blocks = static_cast<long long>(p.batch) * p.cache.kv_heads * strips;
  if (blocks > 0x7fffffffLL) return fail(CLOVE_ERR_UNSUPPORTED, "evict_cache: too many rows");
  cudaLaunchAttribute la[1];
  cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(blocks)), 256, 0, stream, la);
  return check_cuda(cudaLaunchKernelEx(&cfg, kern::evict_copy_kernel<LPR, kRows>, p, strips),
                    "evict copy launch");
}

}  // namespace

int launch_evict_cache(const kern::EvictParams& p, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kSmem = kern::kEvictCached * 4;
  const uint64_t bit = 1ull << (dev.device & 63);
  if ((g_evict_attr.load(std::memory_order_acquire) & bit) == 0) {
    const int rc = check_cuda(cudaFuncSetAttribute(kern::evict_select_kernel,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
                              "cudaFuncSetAttribute(evict smem)");
    if (rc) return rc;
    g_evict_attr.fetch_or(bit, std::memory_order_acq_rel);
  }
  // CTAs per (sequence, head): up to 8 while all of them fit on the GPU at once (two per
  // SM) and each still has a strip of 1024 keys.
  const long long rows = static_cast<long long>(p.batch) * p.cache.kv_heads;
  int cs = 1;
  while (cs < 8 && rows * cs * 2 <= 2LL * dev.num_sms && p.capacity > cs * kern::kEvictThreads) cs *= 2;
  if (rows * cs > 0x7fffffffLL) return fail(CLOVE_ERR_UNSUPPORTED, "evict_cache: batch x heads exceeds 2^31");
  const int slice = (p.capacity + cs - 1) / cs;
  cudaLaunchAttribute la[2];
  cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>(rows * cs)), kern::kEvictThreads,
                                      std::min(slice, kern::kEvictCached) * 4, stream, la);
  la[1].id = cudaLaunchAttributeClusterDimension;
  la[1].val.clusterDim.x = static_cast<unsigned>(cs);
  la[1].val.clusterDim.y = 1;
  la[1].val.clusterDim.z = 1;
  cfg.numAttrs = 2;
  int rc = check_cuda(cudaLaunchKernelEx(&cfg, kern::evict_select_kernel, p, cs), "evict select launch");
  if (rc) return rc;
  switch (p.row_bytes) {
    case 64: return launch_copy<4>(p, stream);
    case 128: return launch_copy<8>(p, stream);
    case 256: return launch_copy<16>(p, stream);
    default: return launch_copy<32>(p, stream);
  }
}

}  // namespace rt
}  // namespace clove
