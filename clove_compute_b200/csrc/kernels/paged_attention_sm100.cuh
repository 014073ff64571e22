// paged_attention_sm100.cuh -- attention of one new token per sequence over a paged
// key-value cache (decode), split over the cache's length and joined.
//
//   s_t = scale * q . k_t,   O = sum_t exp(s_t) v_t / sum_t exp(s_t),
//   LSE = log sum_t exp(s_t)   over the sequence's keys t (the last `window` of them)
//
// Each K and V element is used by the query heads of one group only (1 to 16 products per
// element), so the kernel is bound by reading the cache once, and everything serves that:
//
// * Work split. An item is one (sequence, key head, block of up to 8 or 16 of its query
//   heads); its keys are cut into tiles of 64, or of 128 where a row has 128 bytes or less
//   (head_dim 64, and head_dim 128 in e4m3). All tiles of all items, in order, are dealt
//   out evenly: CTA c of W takes tiles [c N / W, (c+1) N / W). So ragged batches, a single
//   long sequence and many short ones all load every SM alike, with at most two unfinished
//   items per CTA. Those are left as partial sums in a workspace; the CTA that finishes an
//   item's last part adds the parts up in their order (results do not depend on timing).
//   Which CTA that is, a wrapping counter says, which is zero again when the item is done.
//   (A second kernel for the join cost 3 us more per call.) Lengths are read on the device:
//   one captured launch serves every step.
// * Loads. Four warps per CTA, each with its own ring of K and V chunks of 16 keys (32 where
//   tiles have 128) filled by 16-byte cp.async (any page size, order and strides), no CTA
//   barrier until an item ends. Two CTAs per SM keep about 128 KB in flight per SM; for
//   head_dim 256 only one fits, with 128 KB in 16 bits but 64 KB in e4m3. The ring runs
//   across items.
// * Products. S^T = K Q^T and O^T = V^T P^T as m16n8k16 matrix instructions with the keys
//   (or head elements) as the 16 rows and 8 query heads as the columns: a group of up to 8
//   heads wastes nothing that costs time. (tcgen05 wants 64 or 128 rows of queries.)
//   K and V reach the instructions by ldmatrix from XOR-swizzled rows; e4m3 elements are
//   widened to fp16 in registers. P is passed as the sum of two 16-bit halves: in bf16 they
//   keep 2^-17 of a weight; in fp16, taken 2^15 times as large, 2^-23 of it, down to 2^-40 of
//   the largest weight, below which weights vanish from the sum of values (unscaled halves
//   lost what is below 2^-25: keys beside one that is 17 nats above them). Scores, maxima,
//   totals and O stay in fp32.
// * Softmax. Running maximum and total per warp; the maximum is reduced over the warp
//   only when some lane's score exceeds it.
//
// Measured, back to back on one B200: 64 sequences of up to 16384 keys, 32 / 8 heads of 128,
// fp16 160 to 167 us (6.2 to 6.4 TB/s, 0.94 to 0.98 of the copy rate); 2 x 131071 keys, 64 / 8
// heads, e4m3 102 to 109 us (0.75 to 0.80; rows of 128 bytes at strides of 1 KB; 96 us with a
// head's rows side by side); 1 x 4096 keys, 32 / 32 heads, fp16 19 us, of which 9 read the
// cache, 4 pass before the first key (length, page and key, three DRAM latencies in a row)
// and 4 in merging and joining.
#pragma once

#include <cuda_runtime.h>

#include <type_traits>

#include "paged_cache.cuh"

namespace clove {
namespace kern {

constexpr int kPagedWarps = 4;

template <bool F8, int D, int NT>
struct PagedShape {
  static constexpr int THREADS = kPagedWarps * 32;
  static constexpr int HEADS = 8 * NT;             // query heads per item
  static constexpr int ROWB = D * (F8 ? 1 : 2);    // bytes of a K (or V) row
  static constexpr int CPR = ROWB / 16;            // 16-byte pieces per row
  // Groups of 16 keys per warp and step: two where rows are short, so that a step's fixed
  // cost (cursors, votes, waits) is paid for 8 KB of keys and values at least.
  static constexpr int M = ROWB <= 128 ? 2 : 1;
  static constexpr int TILE = kPagedWarps * 16 * M;  // keys per CTA step
  static constexpr int CHUNK = 16 * M * ROWB;        // bytes of a warp's K (or V) chunk
  // 24 KB of ring per warp where that holds three chunks, else three chunks (head_dim 256 in
  // 16 bits). Two CTAs fit on an SM but for head_dim 256, whose merge buffer takes 33 KB
  // beside the rings: in e4m3 as well one CTA of 129 KB runs alone there (2 x 65536 keys, 32 /
  // 8 heads: 114 us, 0.72 of the copy rate).
  static constexpr int STAGES = 24576 / (2 * CHUNK) >= 8 ? 8
                                : 24576 / (2 * CHUNK) >= 3 ? 24576 / (2 * CHUNK) : 3;
  static constexpr int RING = STAGES * 2 * CHUNK;  // per warp
  static constexpr int OPITCH = D + 4;             // floats; conflict-free column writes
  static constexpr int MERGE = kPagedWarps * 8 * OPITCH * 4;
  static constexpr int SMEM = kPagedWarps * RING + MERGE + kPagedWarps * HEADS * 2 * 4;
  // 8 rows of a chunk read by one ldmatrix phase fall into different banks.
  __host__ __device__ static constexpr int swizzle(int r) { return CPR >= 8 ? (r & 7) : ((r >> 1) & 3); }
  static constexpr int CTAS_PER_SM = 2 * (SMEM + 1024) <= 228 * 1024 ? 2 : 1;
};

// ---- 16-bit types: pairs, conversion, the matrix instruction
template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  __device__ static __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  __device__ static __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Pair<__nv_bfloat16> {
  __device__ static __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  __device__ static __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Four e4m3 values as fp16 (exact): the two lower ones in lo, the others in hi.
__device__ __forceinline__ void e4m3_to_half(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// 16 bytes global -> shared; src_bytes 0 fills zeros and reads nothing.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Place in the tile order: sequence, key head, head block of the group, tile of the item.
struct PagedCursor {
  int b, h, block, tile;
  PagedSpan s;
};
template <int TILE>
__device__ __forceinline__ void paged_next_item(const PagedAttnParams& p, PagedCursor& c) {
  c.tile = 0;
  if (++c.block < p.blocks) return;
  c.block = 0;
  if (++c.h < p.cache.kv_heads) return;
  c.h = 0;
  do {
    ++c.b;
    if (c.b >= p.batch) {
      c.s = PagedSpan{0, 0, 0, 0};
      return;
    }
    c.s = paged_span<TILE>(p, c.b);
  } while (c.s.tiles == 0);
}

// Inclusive sum over the warp's lanes.
__device__ __forceinline__ int warp_scan(int v) {
  const int lane = static_cast<int>(dev::lane_idx());
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

// Tiles of the sequences [l R, (l+1) R) of lane l, R = per_lane, times items per sequence.
// (The host has checked that all tiles together stay below 2^31.)
template <int TILE>
__device__ __forceinline__ int paged_lane_tiles(const PagedAttnParams& p, int hh_n, int per_lane) {
  const int b0 = static_cast<int>(dev::lane_idx()) * per_lane, b1 = min(p.batch, b0 + per_lane);
  int sum = 0;
  for (int b = b0; b < b1; ++b) sum += paged_span<TILE>(p, b).tiles;
  return sum * hh_n;
}

// The (warp-uniform) cursor of tile `at`; own, upto: this lane's tiles and their inclusive
// sum. The lane that holds the tile names 32 R sequences, which are scanned in strips.
template <int TILE>
__device__ __forceinline__ PagedCursor paged_find(const PagedAttnParams& p, int hh_n, int per_lane,
                                                  int own, int upto, int at) {
  const int lane = static_cast<int>(dev::lane_idx());
  const unsigned above = __ballot_sync(0xffffffffu, upto > at);
  const int owner = above ? __ffs(above) - 1 : 31;
  int before = __shfl_sync(0xffffffffu, upto - own, owner);
  int b = owner;
  if (per_lane > 1) {
    const int b_end = min(p.batch, (owner + 1) * per_lane);
    for (int b0 = owner * per_lane; b0 < b_end; b0 += 32) {
      const int t = b0 + lane < b_end ? paged_span<TILE>(p, b0 + lane).tiles * hh_n : 0;
      const int inc = warp_scan(t);
      const unsigned hit = __ballot_sync(0xffffffffu, before + inc > at);
      if (hit) {
        const int l = __ffs(hit) - 1;
        before += __shfl_sync(0xffffffffu, inc - t, l);
        b = b0 + l;
        break;
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  PagedCursor c;
  c.b = b;
  c.s = paged_span<TILE>(p, b);
  const int hh = (at - before) / c.s.tiles;
  c.tile = at - before - hh * c.s.tiles;
  c.h = hh / p.blocks;
  c.block = hh - c.h * p.blocks;
  return c;
}

// Four elements of a head's result from their sums v, the maximum and the total.
template <typename T, int D>
__device__ __forceinline__ void paged_store(const PagedAttnParams& p, int b, int head, int d, float (&v)[4],
                                            float top, float sum) {
  const float inv = p.v_scale / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] *= inv;
  T* out = static_cast<T*>(p.o) + b * p.o_stride + static_cast<long long>(head) * D + d;
  *reinterpret_cast<uint2*>(out) = Quad<T>::pack(v);
  if (d != 0) return;
  const float l2 = top + log2f(sum);
  const long long at = static_cast<long long>(b) * p.heads + head;
  if (p.lse != nullptr) p.lse[at] = l2 * 0.6931471805599453f;
  if (p.lse2 != nullptr) p.lse2[at] = l2;
}

// Adds up the partial results of CTAs c0 .. c1 (c0's second, the others' first) with a
// running maximum, kPagedJoin parts in flight, and stores the item. (Short code on purpose:
// it runs once or twice per CTA, and fetching its instructions is much of its time.)
constexpr int kPagedJoin = 8;
template <typename T, int D, int HEADS>
__device__ __forceinline__ void paged_join(const PagedAttnParams& p, int c0, int c1, int live_heads, int b,
                                           int head0) {
  const int work = live_heads * (D / 4);  // four elements of a head each
#pragma unroll 1
  for (int idx = static_cast<int>(threadIdx.x); idx < work; idx += kPagedWarps * 32) {
    const int n = idx / (D / 4), d = (idx - n * (D / 4)) * 4;
    float top = __int_as_float(0xff800000), sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int c = c0; c <= c1; c += kPagedJoin) {
      float m[kPagedJoin], l[kPagedJoin];
      float4 x[kPagedJoin];
#pragma unroll
      for (int k = 0; k < kPagedJoin; ++k) {
        // (Past the last part: the last one again, emptied.)
        const int ck = min(c + k, c1), at = (2 * ck + (ck == c0 ? 1 : 0)) * HEADS + n;
        m[k] = __ldcg(p.part_m + at);
        l[k] = __ldcg(p.part_l + at);
        x[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D + d));
        if (c + k > c1) l[k] = 0.f, x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float t = top;
#pragma unroll
      for (int k = 0; k < kPagedJoin; ++k) t = fmaxf(t, m[k]);
      const float f0 = top == t ? 1.f : dev::ex2_approx(top - t);
      top = t;
      sum *= f0;
      v[0] *= f0, v[1] *= f0, v[2] *= f0, v[3] *= f0;
#pragma unroll
      for (int k = 0; k < kPagedJoin; ++k) {
        const float f = m[k] == t ? 1.f : dev::ex2_approx(m[k] - t);
        sum += f * l[k];
        v[0] += f * x[k].x, v[1] += f * x[k].y, v[2] += f * x[k].z, v[3] += f * x[k].w;
      }
    }
    paged_store<T, D>(p, b, head0 + n, d, v, top, sum);
  }
}

template <typename T, bool F8, int D, int NT>
__global__ void __launch_bounds__(PagedShape<F8, D, NT>::THREADS,
                                  PagedShape<F8, D, NT>::CTAS_PER_SM)
    paged_attention_kernel(const PagedAttnParams p) {
  using S = PagedShape<F8, D, NT>;
  // e4m3 elements (and their queries) are multiplied as fp16, whatever the query type.
  using MT = typename std::conditional<F8, __half, T>::type;
  using P2 = Pair<MT>;
  // Weights are multiplied by this before they are halved (at most 32768 in fp16; the sums,
  // at most 2^16 x 2^15 x 2^31 keys, stay far inside fp32), O by its inverse at the end.
  // bf16 has fp32's exponents and needs none.
  constexpr float P_UP = std::is_same<MT, __half>::value ? 32768.f : 1.f;
  constexpr int ROWB = S::ROWB, CPR = S::CPR, KK = D / 16, M = S::M;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem + kPagedWarps * S::RING);
  float* sm_m = merge + S::MERGE / 4;         // [warp][HEADS]
  float* sm_l = sm_m + kPagedWarps * S::HEADS;
  const int lane = static_cast<int>(dev::lane_idx());
  const int warp = static_cast<int>(dev::warp_idx());
  const int cta = static_cast<int>(blockIdx.x);
  const uint32_t ring = dev::smem_u32(smem) + warp * S::RING;
  const int hh_n = p.cache.kv_heads * p.blocks;
  const int row4 = lane >> 2, col4 = lane & 3;

  dev::grid_dependency_wait();
  dev::allow_dependent_launch();

  // Sequences without keys: zeros. Bad lengths are clamped and reported.
  for (int b = cta; b < p.batch; b += static_cast<int>(gridDim.x)) {
    const int n = p.seq_lens[b];
    if ((n < 0 || n > p.capacity) && threadIdx.x == 0) dev::record_error(dev::kDevErrBadIndex);
    if (min(n, p.capacity) > 0) continue;
    T* o = static_cast<T*>(p.o) + b * p.o_stride;
    for (int i = static_cast<int>(threadIdx.x) * 8; i < p.heads * D; i += S::THREADS * 8)
      *reinterpret_cast<uint4*>(o + i) = make_uint4(0u, 0u, 0u, 0u);
    if (p.lse != nullptr)
      for (int i = static_cast<int>(threadIdx.x); i < p.heads; i += S::THREADS)
        p.lse[static_cast<long long>(b) * p.heads + i] = __int_as_float(0xff800000);
  }

  const int per_lane = (p.batch + 31) / 32;
  const int own = paged_lane_tiles<S::TILE>(p, hh_n, per_lane), upto = warp_scan(own);
  const int total = __shfl_sync(0xffffffffu, upto, 31);
  const int workers = min(static_cast<int>(gridDim.x), total);
  if (cta >= workers) return;
  // Every worker takes total / workers tiles, the first total % workers one more.
  const int share = total / workers, more = total - share * workers;
  const int n_tiles = share + (cta < more ? 1 : 0);
  const int t_begin = cta * share + min(cta, more);
  PagedCursor cur = paged_find<S::TILE>(p, hh_n, per_lane, own, upto, t_begin);
  PagedCursor ld = cur;  // the loads' place
  int ld_left = n_tiles;
  const int page_mask = (1 << p.cache.page_shift) - 1;
  const bool whole_pages = p.cache.page_shift >= 4;  // a 16-key chunk lies in one page

  auto chunk_key = [&](const PagedCursor& c) { return c.s.base + c.tile * S::TILE + warp * (16 * M); };
  auto good_page = [&](int pg) { return pg >= 0 && pg < p.cache.num_pages; };
  // Byte strides, and this lane's part of the addresses: a chunk is loaded RPI rows at a
  // time, CPR lanes per row; 16-byte piece c of row r lies at piece c ^ swizzle(r).
  constexpr int EB = F8 ? 1 : 2, RPI = 32 / CPR;
  const long long tok_b = p.cache.token_stride * EB;
  const long long v_minus_k = static_cast<const uint8_t*>(p.cache.V) - static_cast<const uint8_t*>(p.cache.K);
  const int ld_row = lane / CPR, piece = lane % CPR;
  const uint8_t* ld_base = static_cast<const uint8_t*>(p.cache.K) + ld_row * tok_b + piece * 16;
  const uint32_t ld_dst = ring + ld_row * ROWB + ((piece ^ S::swizzle(ld_row)) << 4);
  // Pages of this warp's chunks, where 16 keys lie in one page: lane i holds that of group
  // i % M of tile win_tile + i / M of the item that is being loaded; the next 32, and those
  // of the next item, are read well before they are needed. -1: no keys, or a bad page.
  constexpr int WTILES = 32 / M;
  PagedCursor nx;
  int win = -1, win_tile = 0, win_more = -1, win_next = -1;
  auto window = [&](const PagedCursor& c, int tile) {
    tile += lane / M;
    const int key = c.s.base + tile * S::TILE + warp * (16 * M) + lane % M * 16;
    if (tile >= c.s.tiles || key >= c.s.len) return -1;
    const int pg = p.page_table[c.b * p.table_stride + (key >> p.cache.page_shift)];
    if (good_page(pg)) return pg;
    dev::record_error(dev::kDevErrBadIndex);
    return -1;
  };
  const uint8_t* ld_src = nullptr;  // this lane's address in row 0 of page 0 for the item's head
  auto enter = [&]() {  // `ld` has come to an item; its window is in win
    win_tile = ld.tile;
    ld_src = ld_base + ld.h * p.cache.head_stride * EB;
    if (ld_left > ld.s.tiles - ld.tile) {
      nx = ld;
      paged_next_item<S::TILE>(p, nx);
      if (whole_pages) win_next = window(nx, 0);
    }
  };
  auto issue = [&](int stage) {
    if (ld_left > 0) {
      const int key = chunk_key(ld);
      const int at = ld.tile - win_tile;
      int page[M];
#pragma unroll
      for (int g = 0; g < M; ++g) page[g] = __shfl_sync(0xffffffffu, win, (at * M + g) & 31);
      if (key < ld.s.len) {
        const uint32_t dst = ld_dst + stage * 2 * S::CHUNK;
        bool plain = whole_pages && key >= ld.s.first && key + 16 * M <= ld.s.len;
#pragma unroll
        for (int g = 0; g < M; ++g) plain = plain && page[g] >= 0;
        if (plain) {
#pragma unroll
          for (int g = 0; g < M; ++g) {
            const uint8_t* src =
                ld_src + page[g] * p.cache.page_stride * EB + ((key + 16 * g) & page_mask) * tok_b;
#pragma unroll
            for (int i = g * 16 / RPI; i < (g + 1) * 16 / RPI; ++i) {
              // swizzle(ld_row + i RPI) = swizzle(ld_row) ^ swizzle(i RPI): ld_row < RPI.
              const uint32_t d = (dst ^ (S::swizzle(i * RPI) << 4)) + i * RPI * ROWB;
              cp_async_16(d, src, 16u);
              cp_async_16(d + S::CHUNK, src + v_minus_k, 16u);
              src += RPI * tok_b;
            }
          }
        } else {
          // Keys outside the sequence, bad pages, or pages of less than 16 keys: row by row.
          constexpr int N = 16 * M / RPI;
          int pg[N];
          bool bad = false;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int t = key + ld_row + i * RPI;
            pg[i] = page[i * RPI / 16];
            if (!whole_pages)  // (a clamped key: the loads do not wait for one another)
              pg[i] = p.page_table[ld.b * p.table_stride +
                                   (max(ld.s.first, min(t, ld.s.len - 1)) >> p.cache.page_shift)];
          }
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int t = key + ld_row + i * RPI;
            bool ok = t >= ld.s.first && t < ld.s.len;
            bad = bad || (!whole_pages && ok && !good_page(pg[i]));
            ok = ok && good_page(pg[i]);
            const uint32_t d = (dst ^ (S::swizzle(i * RPI) << 4)) + i * RPI * ROWB;
            const uint8_t* from =
                ok ? ld_src + pg[i] * p.cache.page_stride * EB + ((t & page_mask) - ld_row) * tok_b : ld_src;
            cp_async_16(d, from, ok ? 16u : 0u);
            cp_async_16(d + S::CHUNK, from + v_minus_k, ok ? 16u : 0u);
          }
          if (bad) dev::record_error(dev::kDevErrBadIndex);
        }
      }
      --ld_left;
      if (++ld.tile >= ld.s.tiles) {
        if (ld_left > 0) {
          ld = nx;
          win = win_next;
          enter();
        }
      } else if (whole_pages) {
        if (at == WTILES / 2 - 1) win_more = window(ld, win_tile + WTILES);
        if (at == WTILES - 1) win = win_more, win_tile += WTILES;
      }
    }
    cp_async_commit();
  };
  if (whole_pages) win = window(ld, ld.tile);
  enter();
#pragma unroll 1  // (instructions fetched once)
  for (int i = 0; i < S::STAGES - 1; ++i) issue(i);

  // ldmatrix addresses within a chunk; piece c is reached by an exclusive or with c << 4.
  // K (and e4m3 V): lanes 0-15 name rows 0-15 of an even piece, lanes 16-31 of the odd one
  // behind it. 16-bit V: lanes 0-7, 8-15 rows 0-7 of the even and odd piece, the others
  // rows 8-15.
  const uint32_t k_lane = (lane & 15) * ROWB + (((lane >> 4) ^ S::swizzle(lane & 15)) << 4);
  const int v_row = F8 ? (lane & 15) : (lane & 7) + ((lane >> 4) << 3);
  const uint32_t v_lane =
      v_row * ROWB + (((F8 ? lane >> 4 : (lane >> 3) & 1) ^ S::swizzle(v_row)) << 4);

  constexpr bool SCALED_Q = F8 && !std::is_same<T, MT>::value;
  float q_scale[NT][2];
  if (!SCALED_Q)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) q_scale[nt][0] = q_scale[nt][1] = p.scale_log2;
  uint32_t qf[NT][KK][2];
  float o[NT][KK][4], m[NT][2], l[NT][2];
  // The item's queries, as B fragments. The k order within 16 elements follows the K
  // fragments (below).
  auto load_q = [&](const PagedCursor& c) {
    const int live = min(S::HEADS, p.group - c.block * S::HEADS);
    const T* q = static_cast<const T*>(p.q) + c.b * p.q_stride +
                 static_cast<long long>(c.h * p.group + c.block * S::HEADS) * D + (F8 ? 4 : 2) * col4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = nt * 8 + row4;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        qf[nt][kk][0] = qf[nt][kk][1] = 0u;
        if (n < live) {
          const T* x = q + n * D + kk * 16;
          qf[nt][kk][0] = *reinterpret_cast<const uint32_t*>(x);
          qf[nt][kk][1] = *reinterpret_cast<const uint32_t*>(x + (F8 ? 2 : 8));
        }
      }
    }
  };
  auto scale_q = [&]() {
    // bf16 queries as fp16: each head's row is first multiplied by the power of two that
    // brings its largest element to [2^15, 2^16), its scores by the inverse. Elements down to
    // 2^-32 of the largest keep all their bits, smaller ones end at 2^-40 of it. (Products
    // with e4m3 stay below 2^25, far inside the fp32 sum.)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t big = 0u;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          big = max(big, max(qf[nt][kk][e] & 0x7fff0000u, (qf[nt][kk][e] << 16) & 0x7fff0000u));
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // Biased exponent; rows below 2^-111 are multiplied by 2^126, those with an infinity or
      // NaN by 1.
      uint32_t ex = big >> 23;
      ex = ex == 255u ? 142u : max(ex, 16u);
      const float scale_up = __uint_as_float((269u - ex) << 23);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 f = Pair<__nv_bfloat16>::unpack(qf[nt][kk][e]);
          qf[nt][kk][e] = P2::pack(f.x * scale_up, f.y * scale_up);
        }
      const float up = __uint_as_float((ex - 15u) << 23) * p.scale_log2;
      q_scale[nt][0] = __shfl_sync(0xffffffffu, up, col4 * 8);
      q_scale[nt][1] = __shfl_sync(0xffffffffu, up, col4 * 8 + 4);
    }
  };
  auto reset = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][kk][e] = 0.f;
      m[nt][0] = m[nt][1] = __int_as_float(0xff800000);
      l[nt][0] = l[nt][1] = 0.f;
    }
  };
  int stage = 0;
  int seg_begin = cur.tile;  // first tile of the current item in this CTA
  load_q(cur);
  if (SCALED_Q) scale_q();
  reset();
  for (int i = 0; i < n_tiles; ++i) {
    cp_async_wait<S::STAGES - 2>();
    __syncwarp();
    issue(stage == 0 ? S::STAGES - 1 : stage - 1);

    const int key = chunk_key(cur);
    if (key < cur.s.len) {
      const uint32_t ks = ring + stage * 2 * S::CHUNK, vs = ks + S::CHUNK;
      float sc[M][NT][4];
#pragma unroll
      for (int g = 0; g < M; ++g)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[g][nt][e] = 0.f;
      // S^T: rows = keys, columns = heads.
#pragma unroll
      for (int c = 0; c < CPR; c += 2)
#pragma unroll
        for (int g = 0; g < M; ++g) {
          uint32_t a[4];
          ldsm_x4(a, ((ks + k_lane) ^ (c << 4)) + g * 16 * ROWB);
          if constexpr (!F8) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) P2::mma(sc[g][nt], a, qf[nt][c / 2][0], qf[nt][c / 2][1]);
          } else {
            // A lane holds four consecutive elements of a row: the first two stand in for
            // k = 2c, 2c+1 and the others for k = 2c+8, 2c+9, in Q's fragments alike.
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              uint32_t x[4];
              e4m3_to_half(a[2 * w], x[0], x[2]);
              e4m3_to_half(a[2 * w + 1], x[1], x[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) P2::mma(sc[g][nt], x, qf[nt][c + w][0], qf[nt][c + w][1]);
            }
          }
        }
      const float none = __int_as_float(0xff800000);
      const bool full = key >= cur.s.first && key + 16 * M <= cur.s.len;
#pragma unroll
      for (int g = 0; g < M; ++g)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[g][nt][e] *= q_scale[nt][e & 1];
      if (!full) {
#pragma unroll
        for (int g = 0; g < M; ++g) {
          const int t0 = key + 16 * g + row4, t1 = t0 + 8;
          const bool ok0 = t0 >= cur.s.first && t0 < cur.s.len, ok1 = t1 >= cur.s.first && t1 < cur.s.len;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(e < 2 ? ok0 : ok1)) sc[g][nt][e] = none;
        }
      }
      float top[NT][2];  // largest of this lane's scores, per head
      bool up = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = fmaxf(sc[0][nt][e], sc[0][nt][e + 2]);
#pragma unroll
          for (int g = 1; g < M; ++g) top[nt][e] = fmaxf(top[nt][e], fmaxf(sc[g][nt][e], sc[g][nt][e + 2]));
          up = up || top[nt][e] > m[nt][e];
        }
      if (p.scores != nullptr) {
        const int g0 = cur.block * S::HEADS, live_heads = min(S::HEADS, p.group - g0);
        float* out = p.scores +
                     ((static_cast<long long>(cur.b) * p.cache.kv_heads + cur.h) * p.capacity) * p.group + g0;
#pragma unroll
        for (int g = 0; g < M; ++g)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int n = nt * 8 + col4 * 2 + (e & 1);
              const int t = key + 16 * g + row4 + (e < 2 ? 0 : 8);
              if (n < live_heads && t >= cur.s.first && t < cur.s.len)
                out[static_cast<long long>(t) * p.group + n] = sc[g][nt][e];
            }
      }
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = fmaxf(m[nt][e], top[nt][e]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
            // All scores -inf so far: nothing to rescale.
            const float alpha = v == m[nt][e] ? 1.f : dev::ex2_approx(m[nt][e] - v);
            m[nt][e] = v;
            l[nt][e] *= alpha;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
              o[nt][kk][e] *= alpha;
              o[nt][kk][e + 2] *= alpha;
            }
          }
      }
      // P^T as the B operand: transposed 8 x 8 blocks of the score fragments, as two 16-bit
      // halves.
      uint32_t ph[M][NT][2], pl[M][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float mm0 = m[nt][0] == none ? 0.f : m[nt][0];
        const float mm1 = m[nt][1] == none ? 0.f : m[nt][1];
#pragma unroll
        for (int g = 0; g < M; ++g)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p0 = dev::ex2_approx(sc[g][nt][2 * e] - mm0);
            const float p1 = dev::ex2_approx(sc[g][nt][2 * e + 1] - mm1);
            l[nt][0] += p0;
            l[nt][1] += p1;
            const float u0 = p0 * P_UP, u1 = p1 * P_UP;
            const uint32_t hi = P2::pack(u0, u1);
            const float2 f = P2::unpack(hi);
            ph[g][nt][e] = transpose_8x8(hi);
            pl[g][nt][e] = transpose_8x8(P2::pack(u0 - f.x, u1 - f.y));
          }
      }
      // O^T += V^T P^T: rows = head elements. 16-bit: tile kk holds elements 16 kk + row.
      // e4m3: ldmatrix moves pairs of elements; tile row j < 8 is element 16 kk + 2 j, row
      // 8 + j element 16 kk + 2 j + 1.
#pragma unroll
      for (int g = 0; g < M; ++g) {
        const uint32_t vg = vs + v_lane;
        if constexpr (!F8) {
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            uint32_t a[4];
            ldsm_x4_t(a, (vg ^ (kk << 5)) + g * 16 * ROWB);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              P2::mma(o[nt][kk], a, ph[g][nt][0], ph[g][nt][1]);
              P2::mma(o[nt][kk], a, pl[g][nt][0], pl[g][nt][1]);
            }
          }
        } else {
#pragma unroll
          for (int k2 = 0; k2 < KK; k2 += 2) {
            uint32_t a[4];
            ldsm_x4_t(a, (vg ^ (k2 << 4)) + g * 16 * ROWB);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              uint32_t x[4];
              e4m3_to_half(__byte_perm(a[2 * w], 0u, 0x3120), x[0], x[1]);
              e4m3_to_half(__byte_perm(a[2 * w + 1], 0u, 0x3120), x[2], x[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                P2::mma(o[nt][k2 + w], x, ph[g][nt][0], ph[g][nt][1]);
                P2::mma(o[nt][k2 + w], x, pl[g][nt][0], pl[g][nt][1]);
              }
            }
          }
        }
      }
    }
    stage = stage + 1 == S::STAGES ? 0 : stage + 1;

    const bool item_ends = cur.tile + 1 == cur.s.tiles;
    if (!item_ends && i + 1 < n_tiles) {
      ++cur.tile;
      continue;
    }
    // The item (or this CTA's part of it) is done. The next one's queries are on their way
    // while the four warps' results are joined.
    const PagedCursor done = cur;
    const bool whole = seg_begin == 0 && item_ends;
    const int item_tile = t_begin + i - done.tile;  // the item's first tile in the tile order
    const int live_heads = min(S::HEADS, p.group - done.block * S::HEADS);
    const int head0 = done.h * p.group + done.block * S::HEADS;
    const int slot = 2 * cta + (seg_begin == 0 ? 1 : 0);
    if (i + 1 < n_tiles) {
      paged_next_item<S::TILE>(p, cur);
      load_q(cur);
      seg_begin = 0;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = l[nt][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
        if (row4 == 0) {
          sm_m[warp * S::HEADS + nt * 8 + col4 * 2 + e] = m[nt][e];
          sm_l[warp * S::HEADS + nt * 8 + col4 * 2 + e] = v;
        }
      }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float* mine = merge + warp * 8 * S::OPITCH;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int n = nt * 8 + col4 * 2 + e;
        float top = sm_m[n];
#pragma unroll
        for (int w = 1; w < kPagedWarps; ++w) top = fmaxf(top, sm_m[w * S::HEADS + n]);
        const float f = (m[nt][e] == top ? 1.f : dev::ex2_approx(m[nt][e] - top)) * (1.f / P_UP);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          const int d0 = kk * 16 + (F8 ? 2 * row4 : row4), d1 = d0 + (F8 ? 1 : 8);
          mine[(col4 * 2 + e) * S::OPITCH + d0] = o[nt][kk][e] * f;
          mine[(col4 * 2 + e) * S::OPITCH + d1] = o[nt][kk][e + 2] * f;
        }
      }
      __syncthreads();
      const int heads_here = min(8, live_heads - nt * 8);
      for (int idx = static_cast<int>(threadIdx.x); idx < heads_here * (D / 4); idx += S::THREADS) {
        const int j = idx / (D / 4), d = (idx - j * (D / 4)) * 4, n = nt * 8 + j;
        float top = sm_m[n];
#pragma unroll
        for (int w = 1; w < kPagedWarps; ++w) top = fmaxf(top, sm_m[w * S::HEADS + n]);
        float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) {
          const float mw = sm_m[w * S::HEADS + n];
          sum += sm_l[w * S::HEADS + n] * (mw == top ? 1.f : dev::ex2_approx(mw - top));
          const float4 x = *reinterpret_cast<const float4*>(merge + (w * 8 + j) * S::OPITCH + d);
          v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        }
        if (whole) {
          paged_store<T, D>(p, done.b, head0 + n, d, v, top, sum);
        } else {
          const long long at = static_cast<long long>(slot) * S::HEADS + n;
          *reinterpret_cast<float4*>(p.part_o + at * D + d) = make_float4(v[0], v[1], v[2], v[3]);
          if (d == 0) {
            p.part_m[at] = top;
            p.part_l[at] = sum;
          }
        }
      }
      __syncthreads();
    }
    if (!whole) {
      // Its parts lie with the CTAs c0 .. c1, in that order; the last one to get here joins
      // them. Each CTA opens one unfinished item at most: c0's counter is the item's.
      const int item_end = item_tile + done.s.tiles - 1;
      const int edge = more * (share + 1);
      const int c0 = item_tile < edge ? item_tile / (share + 1) : more + (item_tile - edge) / share;
      const int c1 = item_end < edge ? item_end / (share + 1) : more + (item_end - edge) / share;
      int* last = reinterpret_cast<int*>(sm_m);
      __threadfence();  // the partial results, before the count
      __syncthreads();
      if (threadIdx.x == 0) *last = atomicInc(p.counters + c0, c1 - c0) == static_cast<unsigned>(c1 - c0);
      __syncthreads();
      const bool join = *last != 0;
      __syncthreads();
      if (join) {
        __threadfence();
        paged_join<T, D, S::HEADS>(p, c0, c1, live_heads, done.b, head0);
      }
    }
    if (SCALED_Q) scale_q();
    reset();
  }
  cp_async_wait<0>();
}

}  // namespace kern
}  // namespace clove
