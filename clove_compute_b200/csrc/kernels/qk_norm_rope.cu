// qk_norm_rope.cu -- per-head RMS norm of queries and keys, position rotation, and the
// append of new keys and values to a paged cache, in one pass.
//
// For a head row x of D elements, weight w, and the table row (cos, sin) of the token's
// position over the first R elements:
//   y   = x / sqrt(mean(x^2) + eps) * w                 (no weights: y = x)
//   y'_i = y_i cos_p - y_j sin_p,  y'_j = y_j cos_p + y_i sin_p
// for pair p = (p, p + R/2) (halves) or (2p, 2p + 1) (interleaved); elements from R on
// keep y. All of it in fp32, rounded once to the output's type.
//
// Bound by memory: every row is read once and written once. D / 16 lanes hold one row, each
// lane two runs of eight elements that pair with each other: 16-byte accesses, the rotation
// needs no exchange between lanes, only the sum of squares is shuffled; the arithmetic is
// in packed fp32 pairs. Two kernels:
// * qk_norm_rope_kernel: one row per lane, straight from global memory. For decode steps,
//   where latency counts (2 us on the GPU for up to 64 tokens), and tokens of few heads.
// * qk_norm_rope_stream_kernel: for calls that fill the GPU. Loads held in registers keep
//   too few bytes in flight beside this much arithmetic (0.65 to 0.75 of the copy rate, with
//   one to four rows per lane), so here each warp streams whole tokens, rows and table row,
//   into a ring in shared memory with bulk copies and computes from there: 8191 tokens of
//   32 + 8 + 8 heads of 128 take 38.4 us, 5.4 TB/s or 0.82 of the copy rate.
#include <algorithm>
#include <atomic>

#include "../runtime/internal.h"
#include "paged_cache.cuh"
#include "pdl_launch.h"

namespace clove {
namespace kern {

constexpr int kRopeThreads = 256;

// Eight consecutive elements as fp32 pairs and back.
template <typename T>
__device__ __forceinline__ void unpack8(uint4 r, uint64_t (&v)[4]) {
  float f[4];
  Quad<T>::unpack(make_uint2(r.x, r.y), f);
  v[0] = dev::f2_pack(f[0], f[1]), v[1] = dev::f2_pack(f[2], f[3]);
  Quad<T>::unpack(make_uint2(r.z, r.w), f);
  v[2] = dev::f2_pack(f[0], f[1]), v[3] = dev::f2_pack(f[2], f[3]);
}
template <typename C>
__device__ __forceinline__ void store8(C* to, const uint64_t (&v)[4]) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) dev::f2_unpack(v[e], f[2 * e], f[2 * e + 1]);
  const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
  const auto a = Quad<C>::pack(lo), b = Quad<C>::pack(hi);
  if constexpr (sizeof(C) == 2)
    *reinterpret_cast<uint4*>(to) = make_uint4(a.x, a.y, b.x, b.y);
  else
    *reinterpret_cast<uint2*>(to) = make_uint2(a, b);
}
// (e0 e1)(e2 e3).. of 16 consecutive elements x, y <-> first elements of the pairs in x, the
// second ones in y.
__device__ __forceinline__ void deal16(uint64_t (&x)[4], uint64_t (&y)[4]) {
  float f[16];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    dev::f2_unpack(x[e], f[2 * e], f[2 * e + 1]);
    dev::f2_unpack(y[e], f[8 + 2 * e], f[8 + 2 * e + 1]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = dev::f2_pack(f[4 * e], f[4 * e + 2]);
    y[e] = dev::f2_pack(f[4 * e + 1], f[4 * e + 3]);
  }
}
__device__ __forceinline__ void gather16(uint64_t (&x)[4], uint64_t (&y)[4]) {
  float f[16];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    dev::f2_unpack(x[e], f[4 * e], f[4 * e + 2]);
    dev::f2_unpack(y[e], f[4 * e + 1], f[4 * e + 3]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = dev::f2_pack(f[2 * e], f[2 * e + 1]);
    y[e] = dev::f2_pack(f[8 + 2 * e], f[8 + 2 * e + 1]);
  }
}

// What both kernels do with a row: x, y the lane's runs [a, a + 8) and [b, b + 8).
// Weights wa, wb (fp32 pairs, dealt like the elements); c, s the table's row for the lane.
template <int LPR, bool INTER>
__device__ __forceinline__ void norm_rope_row(uint64_t (&x)[4], uint64_t (&y)[4], bool norm,
                                              const uint64_t (&wa)[4], const uint64_t (&wb)[4], float eps,
                                              bool rotated, const uint64_t (&c)[4], const uint64_t (&s)[4]) {
  if (norm) {
    uint64_t s2 = dev::f2_mul(x[0], x[0]), t2 = dev::f2_mul(y[0], y[0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) s2 = dev::f2_fma(x[e], x[e], s2), t2 = dev::f2_fma(y[e], y[e], t2);
    float s0, s1;
    dev::f2_unpack(dev::f2_add(s2, t2), s0, s1);
    float ss = s0 + s1;
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss * (1.f / (LPR * 16)) + eps);
    const uint64_t inv2 = dev::f2_pack(inv, inv);
    if (INTER) deal16(x, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = dev::f2_mul(dev::f2_mul(x[e], inv2), wa[e]);
      y[e] = dev::f2_mul(dev::f2_mul(y[e], inv2), wb[e]);
    }
  } else if (INTER) {
    deal16(x, y);
  }
  if (rotated) {
    const uint64_t minus = dev::f2_pack(-1.f, -1.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t lo = dev::f2_fma(x[e], c[e], dev::f2_mul(dev::f2_mul(y[e], minus), s[e]));
      y[e] = dev::f2_fma(y[e], c[e], dev::f2_mul(x[e], s[e]));
      x[e] = lo;
    }
  }
  if (INTER) gather16(x, y);
}

// The lane's place in a row.
template <int LPR, bool INTER>
struct RopeLane {
  int u, a, b;
  bool rotated;
  __device__ __forceinline__ explicit RopeLane(int rotary) {
    u = static_cast<int>(threadIdx.x) % LPR;
    rotated = u < rotary / 16;
    a = rotated && !INTER ? 8 * u : 16 * u;
    b = rotated && !INTER ? rotary / 2 + 8 * u : 16 * u + 8;
  }
};

__device__ __forceinline__ void load_pairs(const float* t, uint64_t (&v)[4]) {
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    const float4 x = *reinterpret_cast<const float4*>(t + 2 * e);
    v[e] = dev::f2_pack(x.x, x.y), v[e + 1] = dev::f2_pack(x.z, x.w);
  }
}

template <typename T, bool INTER>
__device__ __forceinline__ void load_weights(const void* weight, int a, int b, uint64_t (&wa)[4],
                                             uint64_t (&wb)[4]) {
  const T* w = static_cast<const T*>(weight);
  unpack8<T>(*reinterpret_cast<const uint4*>(w + a), wa);
  unpack8<T>(*reinterpret_cast<const uint4*>(w + b), wb);
  if (INTER) deal16(wa, wb);
}

// Element offset of a slot in the cache, or -1 (reported once, by the lane with `report`).
__device__ __forceinline__ long long slot_offset(const RopeParams& p, int slot, bool report) {
  if (slot < 0) return -1;
  const int page = slot >> p.cache.page_shift;
  if (page >= p.cache.num_pages) {
    if (report) dev::record_error(dev::kDevErrBadIndex);
    return -1;
  }
  return page * p.cache.page_stride + (slot & ((1 << p.cache.page_shift) - 1)) * p.cache.token_stride;
}

// Writes a finished row (kind 0 query, 1 key, 2 value) where it belongs.
template <typename T, typename C>
__device__ __forceinline__ void store_row(const RopeParams& p, int kind, long long tok, int row, int D,
                                          int a, int b, long long slot_off, uint64_t (&x)[4],
                                          uint64_t (&y)[4]) {
  if (kind != 2 && p.part[kind].out != nullptr) {
    T* out = static_cast<T*>(p.part[kind].out) + tok * p.part[kind].out_stride + row * D;
    store8<T>(out + a, x);
    store8<T>(out + b, y);
  }
  if (kind == 0 || slot_off < 0) return;
  C* to = static_cast<C*>(kind == 2 ? p.cache.V : p.cache.K) + slot_off + row * p.cache.head_stride;
  if (sizeof(C) == 1) {
    const float per = kind == 2 ? p.v_per_scale : p.k_per_scale;
    const uint64_t per2 = dev::f2_pack(per, per);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = dev::f2_mul(x[e], per2), y[e] = dev::f2_mul(y[e], per2);
  }
  store8<C>(to + a, x);
  store8<C>(to + b, y);
}

// T: type of Q, K, V and the outputs; C: the cache's. LPR = D / 16 lanes per row. INTER:
// interleaved pairs. Every block works on one kind of row, 2^shift rows of each of its
// tokens side by side.
template <typename T, typename C, int LPR, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const RopeParams p) {
  constexpr int D = LPR * 16, SLOTS = kRopeThreads / LPR;
  const int kind = blockIdx.x < p.part[1].first ? 0 : blockIdx.x < p.part[2].first ? 1 : 2;
  const RopePart& part = p.part[kind];
  unsigned idx = blockIdx.x - part.first, chunk = 0;
  if (part.chunks > 1) {
    chunk = idx % part.chunks;
    idx /= part.chunks;
  }
  const RopeLane<LPR, INTER> ln(p.rotary);
  const int slot = static_cast<int>(threadIdx.x) / LPR;
  const unsigned token = idx * (SLOTS >> part.shift) + (slot >> part.shift);
  const int row = static_cast<int>(chunk << part.shift) + (slot & ((1 << part.shift) - 1));
  const bool inside = token < static_cast<unsigned>(p.tokens);
  const long long tok = token;
  const T* in = static_cast<const T*>(part.in) + tok * part.in_stride + row * D;
  dev::grid_dependency_wait();
  // All of the token's loads at once; only the table's row waits for the position.
  const int pos = inside ? p.positions[token] : -1;
  const int slot_in = inside && kind != 0 && p.slots != nullptr ? p.slots[token] : -1;
  uint4 ra = make_uint4(0u, 0u, 0u, 0u), rb = ra;
  if (inside && row < part.rows) {
    ra = *reinterpret_cast<const uint4*>(in + ln.a);
    rb = *reinterpret_cast<const uint4*>(in + ln.b);
  }
  const bool norm = part.weight != nullptr;
  uint64_t wa[4], wb[4], c[4], s[4];
  if (norm) load_weights<T, INTER>(part.weight, ln.a, ln.b, wa, wb);
  // A negative position marks a padding token; one behind the table is an error. Both
  // leave every output row of the token as it was. (Lanes stay for the shuffles.)
  const bool live = pos >= 0 && pos < p.table_len;
  if (pos >= p.table_len && ln.u == 0) dev::record_error(dev::kDevErrBadIndex);
  if (kind != 2 && live && ln.rotated) {
    const float* t = p.table + static_cast<long long>(pos) * p.rotary + 8 * ln.u;
    load_pairs(t, c);
    load_pairs(t + p.rotary / 2, s);
  }
  uint64_t x[4], y[4];
  unpack8<T>(ra, x);
  unpack8<T>(rb, y);
  if (kind != 2) norm_rope_row<LPR, INTER>(x, y, norm, wa, wb, p.eps, ln.rotated, c, s);
  if (!live || row >= part.rows) return;
  store_row<T, C>(p, kind, tok, row, D, ln.a, ln.b, slot_offset(p, slot_in, ln.u == 0), x, y);
}

// Every warp works by itself on units of up to unit_rows rows of one token (of its query,
// key and value rows in that order), with a ring of its own: a stage holds a unit's rows and
// the table's row.
constexpr int kStreamWarps = 4;
constexpr int kStreamMaxStages = 8;

template <typename T, typename C, int LPR, bool INTER>
__global__ void __launch_bounds__(kStreamWarps * 32, 2)
    qk_norm_rope_stream_kernel(const RopeParams p, int units_per_token, int unit_rows, int stages) {
  constexpr int D = LPR * 16, ROWB = D * 2, SIDE = 32 / LPR;  // rows at a time
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kStreamWarps][kStreamMaxStages];
  __shared__ int2 meta[kStreamWarps][kStreamMaxStages];  // position (-1: nothing to do), slot
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  const int warp = static_cast<int>(dev::warp_idx()), lane = static_cast<int>(dev::lane_idx());
  const int stage_bytes = unit_rows * ROWB + p.rotary * 4;
  uint8_t* ring = smem + static_cast<size_t>(warp) * stages * stage_bytes;
  const int heads = p.part[0].rows, kv = p.part[1].rows, rows = heads + kv + p.part[2].rows;
  const unsigned units = static_cast<unsigned>(p.tokens) * units_per_token;
  const unsigned first = blockIdx.x * kStreamWarps + warp, every = gridDim.x * kStreamWarps;
  const int mine = first < units ? static_cast<int>((units - first + every - 1) / every) : 0;
  if (lane == 0) {
    for (int i = 0; i < stages; ++i) dev::mbar_init(&full[warp][i], 1);
    dev::fence_mbarrier_init();
  }
  if (threadIdx.x == 0) abort_s = 0;
  __syncthreads();
  dev::grid_dependency_wait();
  dev::allow_dependent_launch();

  int pos = -1, slot = -1;  // of the 32 units around the one loaded next, one per lane
  auto issue = [&](int k) {
    if (k >= mine) return;
    if ((k & 31) == 0) {
      pos = slot = -1;
      if (k + lane < mine) {
        const unsigned token = (first + static_cast<unsigned>(k + lane) * every) / units_per_token;
        pos = p.positions[token];
        if (p.slots != nullptr) slot = p.slots[token];
        if (pos >= p.table_len) {
          dev::record_error(dev::kDevErrBadIndex);
          pos = -1;
        }
      }
    }
    const int at = __shfl_sync(0xffffffffu, pos, k & 31), to = __shfl_sync(0xffffffffu, slot, k & 31);
    const unsigned unit = first + static_cast<unsigned>(k) * every;
    const unsigned token = unit / units_per_token;
    const int r0 = static_cast<int>(unit - token * units_per_token) * unit_rows, r1 = min(rows, r0 + unit_rows);
    const int st = k % stages;
    uint64_t* bar = &full[warp][st];
    if (lane == 0) {
      meta[warp][st] = make_int2(at, to);
      dev::mbar_arrive_expect_tx(bar, at < 0 ? 0u : static_cast<uint32_t>((r1 - r0) * ROWB + p.rotary * 4));
    }
    __syncwarp();
    if (at < 0) return;
    uint8_t* dst = ring + static_cast<size_t>(st) * stage_bytes;
    // Lanes 0 to 2: the unit's query, key and value rows; lane 3: the table's row.
    if (lane < 3) {
      const int begin = lane == 0 ? 0 : lane == 1 ? heads : heads + kv;
      const int b = max(r0, begin), e = min(r1, begin + p.part[lane].rows);
      if (b < e)
        dev::bulk_load_1d(dst + (b - r0) * ROWB,
                          static_cast<const T*>(p.part[lane].in) +
                              static_cast<long long>(token) * p.part[lane].in_stride + (b - begin) * D,
                          static_cast<uint32_t>((e - b) * ROWB), bar);
    } else if (lane == 3) {
      dev::bulk_load_1d(dst + unit_rows * ROWB, p.table + static_cast<long long>(at) * p.rotary,
                        static_cast<uint32_t>(p.rotary * 4), bar);
    }
  };

  for (int k = 0; k < stages - 1; ++k) issue(k);
  const RopeLane<LPR, INTER> ln(p.rotary);
  const bool norm = p.part[0].weight != nullptr;
  uint4 raw[2][2] = {};  // the lane's query and key weights
  if (norm)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const T* w = static_cast<const T*>(p.part[k].weight);
      raw[k][0] = *reinterpret_cast<const uint4*>(w + ln.a);
      raw[k][1] = *reinterpret_cast<const uint4*>(w + ln.b);
    }
  for (int k = 0; k < mine; ++k) {
    issue(k + stages - 1);
    const int st = k % stages;
    if (!__all_sync(0xffffffffu, dev::mbar_wait(&full[warp][st], (k / stages) & 1, abort_flag))) {
      // Given up: let the copies still in flight land before the warp leaves.
      volatile int no_abort = 0;
      for (int i = k; i < min(mine, k + stages); ++i)
        dev::mbar_wait(&full[warp][i % stages], (i / stages) & 1, &no_abort);
      return;
    }
    const int2 m = meta[warp][st];
    if (m.x >= 0) {
      const unsigned unit = first + static_cast<unsigned>(k) * every;
      const unsigned token = unit / units_per_token;
      const int r0 = static_cast<int>(unit - token * units_per_token) * unit_rows, n = min(rows - r0, unit_rows);
      const uint8_t* src = ring + static_cast<size_t>(st) * stage_bytes;
      const long long slot_off = slot_offset(p, m.y, lane == 0);
      uint64_t c[4], s[4];
      if (ln.rotated) {
        const float* t = reinterpret_cast<const float*>(src + unit_rows * ROWB) + 8 * ln.u;
        load_pairs(t, c);
        load_pairs(t + p.rotary / 2, s);
      }
      // Query rows, key rows, value rows; every lane stays for the shuffles.
#pragma unroll
      for (int kind = 0; kind < 3; ++kind) {
        const int begin = kind == 0 ? 0 : kind == 1 ? heads : heads + kv;
        const int b = max(r0, begin), e = min(r0 + n, begin + p.part[kind].rows);
        uint64_t wa[4], wb[4];
        if (kind < 2) {
          unpack8<T>(raw[kind][0], wa);
          unpack8<T>(raw[kind][1], wb);
          if (INTER) deal16(wa, wb);
        }
#pragma unroll 2
        for (int i0 = b; i0 < e; i0 += SIDE) {
          const int row = i0 + lane / LPR;
          const T* in = reinterpret_cast<const T*>(src) + (min(row, e - 1) - r0) * D;
          uint64_t x[4], y[4];
          unpack8<T>(*reinterpret_cast<const uint4*>(in + ln.a), x);
          unpack8<T>(*reinterpret_cast<const uint4*>(in + ln.b), y);
          if (kind < 2) norm_rope_row<LPR, INTER>(x, y, norm, wa, wb, p.eps, ln.rotated, c, s);
          if (row < e) store_row<T, C>(p, kind, token, row - begin, D, ln.a, ln.b, slot_off, x, y);
        }
      }
    }
    __syncwarp();
  }
}

}  // namespace kern

namespace rt {

CLOVE_DEFINE_ERROR_READER(read_clear_error_rope)

namespace {

// The streaming kernel takes units of at most 12 KB of rows, and at least two of them per
// warp; two CTAs per SM share its shared memory.
constexpr int kStreamUnit = 12 * 1024, kStreamSmem = 108 * 1024;

template <typename T, typename C, int LPR, bool INTER>
int launch_stream(const kern::RopeParams& p, int rows, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kRowB = LPR * 32;
  static std::atomic<uint64_t> attr{0};
  auto* fn = &kern::qk_norm_rope_stream_kernel<T, C, LPR, INTER>;
  const uint64_t bit = 1ull << (dev.device & 63);
  if ((attr.load(std::memory_order_acquire) & bit) == 0) {
    const int rc = check_cuda(
        cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamSmem),
        "cudaFuncSetAttribute(qk_norm_rope smem)");
    if (rc) return rc;
    attr.fetch_or(bit, std::memory_order_acq_rel);
  }
  const int least = (rows * kRowB + kStreamUnit - 1) / kStreamUnit;
  const int unit_rows = (rows + least - 1) / least;
  const int per_token = (rows + unit_rows - 1) / unit_rows;
  const int stage = unit_rows * kRowB + p.rotary * 4;
  const int stages = std::min(kern::kStreamMaxStages, kStreamSmem / kern::kStreamWarps / stage);
  const long long units = static_cast<long long>(p.tokens) * per_token;
  if (units > 0x7fffffffLL) return fail(CLOVE_ERR_UNSUPPORTED, "qk_norm_rope: too many rows");
  cudaLaunchAttribute la[1];
  cudaLaunchConfig_t cfg =
      pdl_config(dim3(static_cast<unsigned>(std::min<long long>(
                     (units + kern::kStreamWarps - 1) / kern::kStreamWarps, 2LL * dev.num_sms))),
                 kern::kStreamWarps * 32, kern::kStreamWarps * stages * stage, stream, la);
  return check_cuda(cudaLaunchKernelEx(&cfg, fn, p, per_token, unit_rows, stages),
                    "qk_norm_rope stream launch");
}

template <typename T, typename C, int LPR>
int launch_rope_h(kern::RopeParams& p, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kSlots = kern::kRopeThreads / LPR, kRowB = LPR * 32;
  const int rows = p.part[0].rows + p.part[1].rows + p.part[2].rows;
  const int force = get_override().path;  // tests: 1 streaming, 2 direct
  // Streaming pays for its start-up (4 us) from about 40 MB of rows on, and for its work per
  // token from 8 KB a token on. 4096 tokens, streamed and direct: 48 rows of 128 26.0 and
  // 27.8 us, 96 rows of 128 43.1 and 48.6, 48 rows of 256 42.4 and 51.4; but 48 rows of 64
  // 18.5 and 16.4, 12 rows of 128 12.6 and 8.2, and 1024 tokens of 48 rows of 128 9.4 and 8.2.
  const bool streams = static_cast<long long>(rows) * kRowB >= 8192 &&
                       static_cast<long long>(p.tokens) * rows * kRowB >= (40LL << 20);
  if (force == 1 || (force != 2 && streams))
    return p.interleaved ? launch_stream<T, C, LPR, true>(p, rows, dev, stream)
                         : launch_stream<T, C, LPR, false>(p, rows, dev, stream);
  long long blocks = 0;
  for (kern::RopePart& part : p.part) {
    // Rows of a token side by side (2^shift): the fewest idle lanes, then the most rows.
    long long best = -1;
    for (int shift = 0; (1 << shift) <= kSlots; ++shift) {
      const long long n = (part.rows + (1LL << shift) - 1) >> shift;
      const long long cost = (((n << shift) - part.rows) << 4) + (8 - shift);
      if (best < 0 || cost < best) {
        best = cost;
        part.shift = shift;
        part.chunks = static_cast<int>(n);
      }
    }
    part.first = static_cast<unsigned>(blocks);
    const int per_block = kSlots >> part.shift;
    blocks += static_cast<long long>((p.tokens - 1) / per_block + 1) * part.chunks;
    if (blocks > 0x7fffffffLL) return fail(CLOVE_ERR_UNSUPPORTED, "qk_norm_rope: too many rows");
  }
  cudaLaunchAttribute la[1];
  cudaLaunchConfig_t cfg =
      pdl_config(dim3(static_cast<unsigned>(blocks)), kern::kRopeThreads, 0, stream, la);
  return check_cuda(p.interleaved
                        ? cudaLaunchKernelEx(&cfg, kern::qk_norm_rope_kernel<T, C, LPR, true>, p)
                        : cudaLaunchKernelEx(&cfg, kern::qk_norm_rope_kernel<T, C, LPR, false>, p),
                    "qk_norm_rope launch");
}

template <typename T, typename C>
int launch_rope_d(kern::RopeParams& p, int head_dim, const DeviceInfo& dev, cudaStream_t stream) {
  if (head_dim == 64) return launch_rope_h<T, C, 4>(p, dev, stream);
  if (head_dim == 128) return launch_rope_h<T, C, 8>(p, dev, stream);
  return launch_rope_h<T, C, 16>(p, dev, stream);
}

}  // namespace

int launch_qk_norm_rope(kern::RopeParams& p, int head_dim, int dtype, int cache_dtype,
                        const DeviceInfo& dev, cudaStream_t stream) {
  const bool e4m3 = cache_dtype == CLOVE_DTYPE_E4M3;
  if (dtype == CLOVE_DTYPE_F16)
    return e4m3 ? launch_rope_d<__half, kern::fp8_e4m3>(p, head_dim, dev, stream)
                : launch_rope_d<__half, __half>(p, head_dim, dev, stream);
  return e4m3 ? launch_rope_d<__nv_bfloat16, kern::fp8_e4m3>(p, head_dim, dev, stream)
              : launch_rope_d<__nv_bfloat16, __nv_bfloat16>(p, head_dim, dev, stream);
}

}  // namespace rt
}  // namespace clove
