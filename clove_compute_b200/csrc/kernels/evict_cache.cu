// evict_cache.cu -- eviction from a paged cache by accumulated key weight.
//
// For each (sequence, key head) with n keys and a budget of B: n <= B keeps everything;
// otherwise the last `recent` keys stay, and of the others the B - recent with the largest
// weights, ties to the lowest index. Kept keys (K, V and weight) are copied in their order
// to the slots of a second page table.
//
// Two kernels. The selection: one cluster per (sequence, key head), each CTA holding a
// contiguous slice of the weights in shared memory as order-preserving integers, so that
// they are read once; a radix select of three digits (11, 11 and 10 bits: an octave of
// weights falls into four first digits) over histograms that the CTAs add up through
// distributed shared memory (one cluster barrier per digit), then an ordered compaction,
// every warp over a contiguous part of its own. Integer counts only: the result does not
// depend on timing. The copy: bound by memory, 16 bytes per lane, four rows of K and V per
// lane in flight while the next rows' places are looked up.
//
// Measured on one B200: 131071 keys, 8 heads, to 16001 (e4m3) 40 us: selection 26 (8 CTAs a
// row: 7 to read the weights, the rest issue and barriers), copy 13. 8 sequences of up to
// 32768 keys, 8 heads, to 8192 (fp16) 82 us: selection 25, copy 54 (300 MB: 0.85 of the copy rate).
// 4096 keys, 8 heads, to 1024: 15 us. Instructions that run once are fetched at about 0.3 us
// per KB, so loops are kept short rather than unrolled.
#include <algorithm>
#include <atomic>

#include "../runtime/internal.h"
#include "paged_cache.cuh"
#include "pdl_launch.h"

namespace clove {
namespace kern {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWarps = kEvictThreads / 32;
// Keys of a slice held in shared memory (160 KB: one CTA per SM); a longer slice reads the
// rest again from memory in every pass.
constexpr int kEvictCached = 40960;
constexpr int kEvictBins = 2048;

// Larger weight <=> larger integer; -0 equals 0; every NaN above everything.
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint2 ld_cluster_v2(const uint32_t* p, uint32_t rank) {
  uint2 v;
  const uint32_t a = dev::map_shared_to_rank(dev::smem_u32(p), rank);
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  const uint32_t a = dev::map_shared_to_rank(dev::smem_u32(p), rank);
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// LONG: slices may exceed kEvictCached keys.
template <bool LONG>
__global__ void __launch_bounds__(kEvictThreads, 1) evict_select_kernel(const EvictParams p, int cs) {
  extern __shared__ uint32_t cached[];
  __shared__ __align__(16) uint32_t hist[2][kEvictBins];
  __shared__ uint32_t coarse[2][kEvictWarps];
  __shared__ uint32_t counts[2];  // this CTA's keys above the threshold, and equal to it
  __shared__ uint32_t warp_a[kEvictWarps], warp_b[kEvictWarps];
  __shared__ uint32_t pick[2];  // chosen digit, keys of larger digits
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = blockIdx.x % cs;
  const int row = static_cast<int>(blockIdx.x) / cs;
  const int b = row / p.cache.kv_heads, h = row - b * p.cache.kv_heads;
  const int page_mask = (1 << p.cache.page_shift) - 1;
  dev::grid_dependency_wait();
  dev::allow_dependent_launch();
  int n = p.seq_lens[b];
  if (n < 0 || n > p.capacity) {
    if (tid == 0) dev::record_error(dev::kDevErrBadIndex);
    n = n < 0 ? 0 : p.capacity;
  }
  int* kept = p.kept + static_cast<long long>(row) * p.budget;
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = min(n, p.budget);
  if (n <= p.budget) {
    for (int j = static_cast<int>(rank) * kEvictThreads + tid; j < p.budget; j += cs * kEvictThreads)
      kept[j] = j < n ? j : -1;
    return;  // the whole cluster
  }
  // Candidates [0, m), `want` of them to keep; slice [s0, s0 + sn) of this CTA.
  const int m = n - p.recent, want = p.budget - p.recent;
  const int per = (m + cs - 1) / cs;
  const int s0 = min(m, static_cast<int>(rank) * per), sn = min(m, s0 + per) - s0;
  for (int i = tid; i < kEvictBins; i += kEvictThreads) hist[0][i] = 0;
  __syncthreads();
  // Every warp keeps to a contiguous part [w0, w1) of the slice.
  const int part = ((sn + kEvictWarps - 1) / kEvictWarps + 31) & ~31;
  const int w0 = min(sn, warp * part), w1 = min(sn, w0 + part);
  auto good = [&](int pg) { return pg >= 0 && pg < p.cache.num_pages; };
  auto page_at = [&](int i) { return p.page_table[b * p.table_stride + ((s0 + i) >> p.cache.page_shift)]; };
  // (A clamped page: the load is unconditional, so that none waits for another.)
  auto weight_at = [&](int i, int pg) {
    return p.key_weights[((static_cast<long long>(good(pg) ? pg : 0) * p.cache.kv_heads + h)
                          << p.cache.page_shift) +
                         ((s0 + i) & page_mask)];
  };
  bool bad = false;
  auto key = [&](int i) {
    if (!LONG || i < kEvictCached) return cached[i];
    const int pg = page_at(i);
    const float w = weight_at(i, pg);
    bad = bad || !good(pg);
    return weight_order(good(pg) ? w : 0.f);  // a bad page counts as weight 0
  };
  // One more key with this digit, for the lanes with `in`. Where many lanes have one, the
  // first lane's digit is counted once for the warp: equal weights (zeros, as a rule) would
  // otherwise queue up at one address.
  auto count = [&](uint32_t* mine, bool in, uint32_t digit) {
    const unsigned act = __ballot_sync(0xffffffffu, in);
    if (__popc(act) > 4) {
      const int lead = __ffs(act) - 1;
      const uint32_t d0 = __shfl_sync(0xffffffffu, digit, lead);
      const unsigned same = __ballot_sync(0xffffffffu, in && digit == d0);
      if (lane == lead) atomicAdd(&mine[d0], static_cast<uint32_t>(__popc(same)));
      in = in && digit != d0;
    }
    if (in) atomicAdd(&mine[digit], 1u);
  };
  // The weights: KEYS at a time, whose pages (of 16 keys or more: fewer than 32) one load of
  // the warp brings, the next KEYS' pages ahead of their use. The first digit is
  // counted as they arrive.
  constexpr int DEEP = 4, KEYS = 32 * DEEP;
  const bool wide = p.cache.page_shift >= 4;
  auto pages_of = [&](int base) {
    const int first = (s0 + base) >> p.cache.page_shift, last = (s0 + min(base + KEYS, w1) - 1) >> p.cache.page_shift;
    return wide && base < w1 ? p.page_table[b * p.table_stride + min(first + lane, last)] : 0;
  };
  int win = pages_of(w0);
#pragma unroll 1
  for (int base = w0; base < w1; base += KEYS) {
    const int now = win, first = (s0 + base) >> p.cache.page_shift;
    win = pages_of(base + KEYS);
    float w[DEEP];
    int pg[DEEP];
    uint32_t ok = 0;
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      const int i = min(base + 32 * k + lane, w1 - 1);
      pg[k] = __shfl_sync(0xffffffffu, now, (((s0 + i) >> p.cache.page_shift) - first) & 31);
      if (!wide) pg[k] = page_at(i);
    }
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      ok |= good(pg[k]) ? 1u << k : 0u;
      w[k] = weight_at(min(base + 32 * k + lane, w1 - 1), pg[k]);
    }
    bad = bad || ok != (1u << DEEP) - 1u;  // (places past the end repeat the last key's)
    const int n8 = min(DEEP, (w1 - base + 31) / 32);
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      const int i = base + 32 * k + lane;
      if (k >= n8) break;
      const uint32_t u = weight_order(ok & (1u << k) ? w[k] : 0.f);
      if (i < w1 && (!LONG || i < kEvictCached)) cached[i] = u;
      count(hist[0], i < w1, u >> 21);
    }
  }
  __syncwarp();

  uint32_t prefix = 0;  // digits chosen so far
  uint32_t left = static_cast<uint32_t>(want);
#pragma unroll 1
  for (int d = 0; d < 3; ++d) {
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d == 2 ? 10 : 11;
    const uint32_t mask = (1u << bits) - 1u;
    uint32_t* mine = hist[d & 1];
    if (d > 0) {
#pragma unroll 2
      for (int base = w0; base < w1; base += 32) {
        const int i = base + lane;
        const uint32_t u = i < w1 ? key(i) : 0u;
        const bool in = i < w1 && (u >> (shift + bits)) == prefix;
        if (__any_sync(0xffffffffu, in)) count(mine, in, (u >> shift) & mask);
      }
    }
    __syncthreads();
    // Sums of 64 bins each, one per warp, from the largest down.
    {
      const int bin = kEvictBins - 64 * (warp + 1) + 2 * lane;
      uint32_t v = mine[bin] + mine[bin + 1];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) coarse[d & 1][warp] = v;
    }
    // All CTAs' histograms of this digit are complete, and those of the digit before have
    // been read by all of them: only now may this one's be cleared, for the next digit.
    dev::cluster_sync_all();
    for (int i = tid; i < kEvictBins; i += kEvictThreads) hist[(d & 1) ^ 1][i] = 0;
    if (warp == 0) {
      // Warp 0 finds the `left`-th largest key's 64 bins, then its bin, adding up the CTAs'
      // counts of those alone.
      auto scan_from_top = [&](uint32_t own) {
        uint32_t inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += v;
        }
        return inc - own;
      };
      uint32_t x[8], own = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) x[r] = r < cs ? ld_cluster_u32(&coarse[d & 1][lane], static_cast<uint32_t>(r)) : 0u;
#pragma unroll
      for (int r = 0; r < 8; ++r) own += x[r];
      uint32_t run = scan_from_top(own);
      unsigned hit = __ballot_sync(0xffffffffu, run < left && run + own >= left);
      const int block = hit ? __ffs(hit) - 1 : 0;  // (left == 0: nothing is wanted, digit `mask`)
      run = __shfl_sync(0xffffffffu, run, block);
      const int low = kEvictBins - 64 * block - 2 * (lane + 1);
      uint2 y[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        y[r] = r < cs ? ld_cluster_v2(&mine[low], static_cast<uint32_t>(r)) : make_uint2(0u, 0u);
      uint32_t c0 = 0, c1 = 0;  // the larger and the smaller of the lane's two bins
#pragma unroll
      for (int r = 0; r < 8; ++r) c0 += y[r].y, c1 += y[r].x;
      run += scan_from_top(c0 + c1);
      if (left == 0) {
        if (lane == 0) pick[0] = mask, pick[1] = 0u;
      } else if (run < left && run + c0 + c1 >= left) {
        const bool first = run + c0 >= left;
        pick[0] = static_cast<uint32_t>(first ? low + 1 : low);
        pick[1] = first ? run : run + c0;
      }
    }
    __syncthreads();
    left -= pick[1];
    prefix = (prefix << bits) | pick[0];
    __syncthreads();
  }
  if (bad) dev::record_error(dev::kDevErrBadIndex);
  // Keys above and equal to the threshold in each warp's part.
  uint32_t gt_n = 0, eq_n = 0;
#pragma unroll 2
  for (int i = w0 + lane; i < w1; i += 32) {
    const uint32_t u = key(i);
    gt_n += u > prefix ? 1u : 0u;
    eq_n += u == prefix ? 1u : 0u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    gt_n += __shfl_xor_sync(0xffffffffu, gt_n, o);
    eq_n += __shfl_xor_sync(0xffffffffu, eq_n, o);
  }
  if (lane == 0) warp_a[warp] = gt_n, warp_b[warp] = eq_n;
  __syncthreads();
  if (warp == 0) {
    uint32_t g = warp_a[lane], q = warp_b[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      g += __shfl_xor_sync(0xffffffffu, g, o);
      q += __shfl_xor_sync(0xffffffffu, q, o);
    }
    if (lane == 0) counts[0] = g, counts[1] = q;
  }
  dev::cluster_sync_all();
  // `left` keys equal to the threshold are kept, the first ones. What the slices, and the
  // warps' parts, before this one keep:
  // (Lanes 0 .. rank - 1 hold the slices', then lanes 0 .. warp - 1 the parts' counts.)
  uint32_t eq_before = 0, out = 0;
  auto skip = [&](uint32_t gt, uint32_t eq) {
    uint32_t inc = eq;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const uint32_t before = eq_before + inc - eq;
    uint32_t kept_n = gt + min(eq, left - min(left, before));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) kept_n += __shfl_xor_sync(0xffffffffu, kept_n, o);
    out += kept_n;
    eq_before += __shfl_sync(0xffffffffu, inc, 31);
  };
  const bool slice_before = lane < static_cast<int>(rank);
  skip(slice_before ? ld_cluster_u32(&counts[0], lane) : 0u, slice_before ? ld_cluster_u32(&counts[1], lane) : 0u);
  skip(lane < warp ? warp_a[lane] : 0u, lane < warp ? warp_b[lane] : 0u);
  dev::cluster_arrive();  // no CTA leaves while its counts may be read
  const unsigned below = (1u << lane) - 1u;
  if (eq_n == 0 || eq_before >= left || eq_before + eq_n <= left) {
    // All of the part's equal keys are kept, or none: one comparison decides.
    const bool with_eq = eq_before < left;
#pragma unroll 2
    for (int base = w0; base < w1; base += 32) {
      const int i = base + lane;
      const uint32_t u = i < w1 ? key(i) : 0u;
      const bool take = i < w1 && (with_eq ? u >= prefix : u > prefix);
      const unsigned tk = __ballot_sync(0xffffffffu, take);
      if (take) kept[out + __popc(tk & below)] = s0 + i;
      out += __popc(tk);
    }
  } else {
#pragma unroll 1
    for (int base = w0; base < w1; base += 32) {
      const int i = base + lane;
      const uint32_t u = i < w1 ? key(i) : 0u;
      const bool eq = i < w1 && u == prefix;
      const unsigned eq_b = __ballot_sync(0xffffffffu, eq);
      const bool take = (i < w1 && u > prefix) || (eq && eq_before + __popc(eq_b & below) < left);
      const unsigned tk = __ballot_sync(0xffffffffu, take);
      if (take) kept[out + __popc(tk & below)] = s0 + i;
      out += __popc(tk);
      eq_before += __popc(eq_b);
    }
  }
  // The recent keys.
  for (int j = static_cast<int>(rank) * kEvictThreads + tid; j < p.recent; j += cs * kEvictThreads)
    kept[want + j] = m + j;
  __syncwarp();
  dev::cluster_wait();
}

// LPR lanes of 16 bytes per row; ROWS rows of one (sequence, head) per lane and step.
template <int LPR, int ROWS>
__global__ void __launch_bounds__(256, 3) evict_copy_kernel(const EvictParams p, int strips, int total) {
  constexpr int PER = 256 / LPR;  // rows at a time
  const int piece = static_cast<int>(threadIdx.x) % LPR, slot = static_cast<int>(threadIdx.x) / LPR;
  const int page_mask = (1 << p.cache.page_shift) - 1;
  const char* k = static_cast<const char*>(p.cache.K) + piece * 16;
  const char* v = static_cast<const char*>(p.cache.V) + piece * 16;
  dev::grid_dependency_wait();
  // Cache slots of a step's rows, source and destination; -1: no row.
  int src[ROWS], dst[ROWS], next_h = 0;
  auto look_up = [&](int step) {
    const int row = step / strips, strip = step - row * strips;
    const int b = row / p.cache.kv_heads;
    next_h = row - b * p.cache.kv_heads;
    const int* kept = p.kept + static_cast<long long>(row) * p.budget;
    // (Unconditional loads at clamped places: none waits for a branch on another.)
    int t[ROWS], sp[ROWS], dp[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int j = min(strip * (PER * ROWS) + i * PER + slot, p.budget - 1);
      t[i] = kept[j];
      dp[i] = p.dst_table[b * p.dst_stride + (j >> p.cache.page_shift)];
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      sp[i] = p.page_table[b * p.table_stride + (max(t[i], 0) >> p.cache.page_shift)];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (strip * (PER * ROWS) + i * PER + slot >= p.budget) t[i] = -1;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int j = strip * (PER * ROWS) + i * PER + slot;
      const bool ok = sp[i] >= 0 && sp[i] < p.cache.num_pages && dp[i] >= 0 && dp[i] < p.cache.num_pages;
      bad = bad || (t[i] >= 0 && !ok);
      src[i] = t[i] >= 0 && ok ? (sp[i] << p.cache.page_shift) + (t[i] & page_mask) : -1;
      dst[i] = (dp[i] << p.cache.page_shift) + (j & page_mask);
    }
    if (bad) dev::record_error(dev::kDevErrBadIndex);
  };
  const long long page_b = p.cache.page_stride * p.elem, tok_b = p.cache.token_stride * p.elem;
  int step = static_cast<int>(blockIdx.x);
  if (step < total) look_up(step);
  for (; step < total; step += static_cast<int>(gridDim.x)) {
    const int h = next_h;
    const long long head = h * p.cache.head_stride * p.elem;
    uint4 kr[ROWS], vr[ROWS];
    float w[ROWS];
    int to[ROWS];
    // Row h of slot s in the paged weights.
    auto weight_at = [&](int s) {
      return ((static_cast<long long>(s >> p.cache.page_shift) * p.cache.kv_heads + h) << p.cache.page_shift) +
             (s & page_mask);
    };
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      to[i] = src[i] < 0 ? -1 : dst[i];
      if (src[i] < 0) continue;
      const long long off = (src[i] >> p.cache.page_shift) * page_b + (src[i] & page_mask) * tok_b + head;
      kr[i] = *reinterpret_cast<const uint4*>(k + off);
      vr[i] = *reinterpret_cast<const uint4*>(v + off);
      w[i] = p.key_weights[weight_at(src[i])];
    }
    if (step + static_cast<int>(gridDim.x) < total) look_up(step + static_cast<int>(gridDim.x));
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (to[i] < 0) continue;
      const long long off = (to[i] >> p.cache.page_shift) * page_b + (to[i] & page_mask) * tok_b + head;
      *reinterpret_cast<uint4*>(const_cast<char*>(k) + off) = kr[i];
      *reinterpret_cast<uint4*>(const_cast<char*>(v) + off) = vr[i];
      if (piece == 0) p.key_weights[weight_at(to[i])] = w[i];
    }
  }
}

}  // namespace kern

namespace rt {

CLOVE_DEFINE_ERROR_READER(read_clear_error_evict)

namespace {

std::atomic<uint64_t> g_evict_attr{0};

template <int LPR>
int launch_copy(const kern::EvictParams& p, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kRows = 4;
  const int per = 256 / LPR * kRows;
  const int strips = (p.budget + per - 1) / per;
  const long long total = static_cast<long long>(p.batch) * p.cache.kv_heads * strips;
  if (total > 0x7fffffffLL - 65536) return fail(CLOVE_ERR_UNSUPPORTED, "evict_cache: too many rows");
  const unsigned blocks = static_cast<unsigned>(std::min<long long>(total, 3LL * dev.num_sms));
  cudaLaunchAttribute la[1];
  cudaLaunchConfig_t cfg = pdl_config(dim3(blocks), 256, 0, stream, la);
  return check_cuda(cudaLaunchKernelEx(&cfg, kern::evict_copy_kernel<LPR, kRows>, p, strips,
                                       static_cast<int>(total)),
                    "evict copy launch");
}

}  // namespace

int launch_evict_cache(const kern::EvictParams& p, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kSmem = kern::kEvictCached * 4;
  const uint64_t bit = 1ull << (dev.device & 63);
  if ((g_evict_attr.load(std::memory_order_acquire) & bit) == 0) {
    int rc = check_cuda(cudaFuncSetAttribute(kern::evict_select_kernel<false>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
                        "cudaFuncSetAttribute(evict smem)");
    if (!rc)
      rc = check_cuda(cudaFuncSetAttribute(kern::evict_select_kernel<true>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
                      "cudaFuncSetAttribute(evict smem)");
    if (rc) return rc;
    g_evict_attr.fetch_or(bit, std::memory_order_acq_rel);
  }
  // CTAs per (sequence, head): up to 8, doubled while all of them fit on the GPU at once (one
  // per SM) and each has more than 4096 keys, four per thread; after the doubling it has more
  // than 2048. That goes by the table's width: shorter rows leave their CTAs less. (Clusters of 16 do not all fit: 131071 keys
  // of 8 heads take 56 us with them, 42 us with 8. Twice as many CTAs as SMs: 8 sequences of
  // 32768 keys, 8 heads, ragged 82 -> 76 us, but of equal lengths 125 -> 134 us.)
  const long long rows = static_cast<long long>(p.batch) * p.cache.kv_heads;
  int cs = 1;
  while (cs < 8 && rows * cs * 2 <= dev.num_sms && p.capacity > cs * 4 * kern::kEvictThreads) cs *= 2;
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
  const int rc = check_cuda(slice > kern::kEvictCached
                                ? cudaLaunchKernelEx(&cfg, kern::evict_select_kernel<true>, p, cs)
                                : cudaLaunchKernelEx(&cfg, kern::evict_select_kernel<false>, p, cs),
                            "evict select launch");
  if (rc || p.capacity == 0) return rc;
  switch (p.row_bytes) {
    case 64: return launch_copy<4>(p, dev, stream);
    case 128: return launch_copy<8>(p, dev, stream);
    case 256: return launch_copy<16>(p, dev, stream);
    default: return launch_copy<32>(p, dev, stream);
  }
}

}  // namespace rt
}  // namespace clove
