// paged_api.cpp -- extern "C" entry points of the paged key-value cache operators
// (include/clove/capi.h): argument checks, workspace, dispatch.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "../kernels/paged_params.h"
#include "internal.h"

namespace clove {
namespace rt {
namespace {

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// While it lives, this thread's allocations outside a capture neither fail because another
// thread captures (in the default, global mode) nor spoil its capture.
struct OutsideCaptures {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  OutsideCaptures() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~OutsideCaptures() { cudaThreadExchangeStreamCaptureMode(&mode); }
  OutsideCaptures(const OutsideCaptures&) = delete;
  OutsideCaptures& operator=(const OutsideCaptures&) = delete;
};

// Stream-ordered scratch, one pool per device; under stream capture an allocation of the
// graph's own. Between calls the pool holds kPoolHolds, the kept workspaces among them; what
// is above goes back to the device when the program next waits for it.
constexpr uint64_t kPoolHolds = 512u << 20;
std::mutex g_pool_mu;
cudaMemPool_t g_pool[64];

int scratch_alloc(void** out, size_t bytes, int device, bool capturing, cudaStream_t s) {
  if (capturing) return check_cuda(cudaMallocAsync(out, bytes, s), "cudaMallocAsync(paged attention)");
  const OutsideCaptures outside;
  cudaMemPool_t pool;
  {
    std::lock_guard<std::mutex> lock(g_pool_mu);
    if (g_pool[device & 63] == nullptr) {
      cudaMemPoolProps props = {};
      props.allocType = cudaMemAllocationTypePinned;
      props.location.type = cudaMemLocationTypeDevice;
      props.location.id = device;
      int rc = check_cuda(cudaMemPoolCreate(&pool, &props), "cudaMemPoolCreate(paged attention)");
      if (rc) return rc;
      uint64_t keep = kPoolHolds;
      rc = check_cuda(cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep),
                      "cudaMemPoolSetAttribute(paged attention)");
      if (rc) {
        cudaMemPoolDestroy(pool);
        return rc;
      }
      g_pool[device & 63] = pool;
    }
    pool = g_pool[device & 63];
  }
  return check_cuda(cudaMallocFromPoolAsync(out, bytes, pool, s), "cudaMallocFromPoolAsync(paged attention)");
}

int scratch_free(void* p, bool capturing, cudaStream_t s) {
  if (capturing) return check_cuda(cudaFreeAsync(p, s), "cudaFreeAsync(paged attention)");
  const OutsideCaptures outside;
  return check_cuda(cudaFreeAsync(p, s), "cudaFreeAsync(paged attention)");
}

// Workspace of the attention kernel: per-CTA counters, zero between calls, and partial
// results. Calls that can overlap on the GPU must not share one:
// * each stream keeps its own (by the stream's id: a destroyed stream's handle may return
//   as another stream's, and every thread's default stream has the same handle). There are
//   kMaxKept of them; a further stream takes over the least recently used one if that one's
//   last call is over (its event says so; nothing waits for another stream), or brings one
//   for the call alone;
// * a captured call's graph may be replayed beside anything: it gets partial results from the
//   graph's memory and counters that no call outside its graph ever gets. Calls of one graph
//   share them where the graph itself orders them (find_counters). (Its memory also keeps a
//   graph from having two instances at a time.)
// Counters come from an array in the library, 1 MB per device: two per SM for each stream
// and each chain of captured calls, enough for about 800. When it is used up, or its address
// is not known yet under capture, a call brings its own and clears them first.
constexpr size_t kKeptParts = 8u << 20;
constexpr int kMaxKept = 16;
struct KeptWorkspace {
  unsigned long long stream_id = 0;
  unsigned* counters = nullptr;
  float* parts = nullptr;
  cudaEvent_t event = nullptr;
  bool recorded = false;        // the event stands behind the latest call
  int users = 0;                // calls between take_workspace and drop_workspace
  unsigned long long used = 0;  // when, in calls
};
// Counters of captured calls, and the node that ends the last call that took them (null: one
// is being captured). The latest kMaxCaptures are found again.
constexpr int kMaxCaptures = 64;
struct CaptureCounters {
  unsigned long long capture_id;
  cudaGraphNode_t last;
  unsigned* counters;
};
struct DeviceWorkspaces {
  unsigned* base = nullptr;  // the device's counters
  int used = 0;
  int kept_count = 0;
  unsigned long long calls = 0;
  KeptWorkspace kept[kMaxKept];
  CaptureCounters captures[kMaxCaptures] = {};
  unsigned next_capture = 0;
};
std::mutex g_ws_mu;
DeviceWorkspaces g_ws[64];

struct Workspace {
  unsigned* counters = nullptr;
  float* parts = nullptr;
  void* own = nullptr;  // to be released after the call
  bool capturing = false;
  unsigned long long capture_id = 0;
  KeptWorkspace* kept = nullptr;  // the stream's
};

// `count` counters that nobody else has, or null.
unsigned* reserve_counters(DeviceWorkspaces& d, int count) {
  if (d.base == nullptr || d.used + count > kern::kPagedCounters) return nullptr;
  unsigned* c = d.base + d.used;
  d.used += count;
  return c;
}

// Counters of an earlier call of this capture that is over, in every replay, before the work
// that is captured on `s` next: one whose last node is reached from the stream's
// dependencies. (The last node frees the partial results and so follows the kernels in full;
// what starts after it, programmatically overlapped or not, starts after them.) The search
// ends after kMaxVisited nodes: a model's layer has a few dozen between two calls.
constexpr int kMaxVisited = 512, kMaxEdges = 16;
unsigned* find_counters(DeviceWorkspaces& d, unsigned long long capture_id, const cudaGraphNode_t* deps, size_t n) {
  cudaGraphNode_t seen[kMaxVisited];
  int count = 0;
  auto visit = [&](cudaGraphNode_t node) {
    for (int i = 0; i < count; ++i)
      if (seen[i] == node) return;
    if (count < kMaxVisited) seen[count++] = node;
  };
  for (size_t i = 0; i < n; ++i) visit(deps[i]);
  for (int at = 0; at < count; ++at) {
    for (CaptureCounters& c : d.captures)
      if (c.capture_id == capture_id && c.last == seen[at]) {
        c.last = nullptr;
        return c.counters;
      }
    cudaGraphNode_t before[kMaxEdges];
    cudaGraphEdgeData edges[kMaxEdges];
    size_t m = kMaxEdges;
    if (cudaGraphNodeGetDependencies_v2(seen[at], before, edges, &m) != cudaSuccess) return nullptr;
    for (size_t i = 0; i < m && i < kMaxEdges; ++i)
      if (before[i] != nullptr) visit(before[i]);
  }
  return nullptr;
}

// A workspace for a stream that has none: null where all are in use.
int new_workspace(DeviceWorkspaces& d, unsigned long long id, int counters, int device, cudaStream_t s,
                  KeptWorkspace** out) {
  const OutsideCaptures outside;
  if (d.base == nullptr) {
    const int rc = paged_counter_base(&d.base);
    if (rc) return rc;
  }
  if (d.kept_count < kMaxKept) {
    KeptWorkspace& k = d.kept[d.kept_count];
    if (k.event == nullptr) {
      const int rc = check_cuda(cudaEventCreateWithFlags(&k.event, cudaEventDisableTiming), "cudaEventCreate");
      if (rc) return rc;
    }
    if (k.counters == nullptr) k.counters = reserve_counters(d, counters);
    if (k.counters == nullptr) return CLOVE_OK;
    void* parts = nullptr;
    const int rc = scratch_alloc(&parts, kKeptParts, device, false, s);
    if (rc) return rc;
    k.parts = static_cast<float*>(parts);
    k.stream_id = id;
    ++d.kept_count;
    *out = &k;
    return CLOVE_OK;
  }
  KeptWorkspace* oldest = nullptr;
  for (KeptWorkspace& k : d.kept)
    if (k.users == 0 && k.recorded && (oldest == nullptr || k.used < oldest->used)) oldest = &k;
  if (oldest == nullptr) return CLOVE_OK;
  if (cudaEventQuery(oldest->event) != cudaSuccess) {
    (void)cudaGetLastError();  // (not ready is no error)
    return CLOVE_OK;
  }
  oldest->stream_id = id;
  *out = oldest;
  return CLOVE_OK;
}

// (ctas is at most the device's `most`, two per SM.)
int take_workspace(Workspace* w, int ctas, size_t part_bytes, const DeviceInfo& dev, cudaStream_t s) {
  const int device = dev.device, most = (2 * dev.num_sms + 31) & ~31;
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  const cudaGraphNode_t* deps = nullptr;
  const cudaGraphEdgeData* edges = nullptr;
  size_t num_deps = 0;
  int rc = check_cuda(cudaStreamGetCaptureInfo_v3(s, &cap, &w->capture_id, nullptr, &deps, &edges, &num_deps),
                      "cudaStreamGetCaptureInfo");
  if (rc) return rc;
  w->capturing = cap != cudaStreamCaptureStatusNone;
  if (!w->capturing) {  // (the id of a capturing stream cannot be asked for)
    rc = check_cuda(cudaStreamGetId(s, &id), "cudaStreamGetId");
    if (rc) return rc;
  }
  if (ctas > most || part_bytes > kKeptParts)
    return fail(CLOVE_ERR_UNSUPPORTED, "paged_attention: workspace of %d CTAs", ctas);
  {
    std::lock_guard<std::mutex> lock(g_ws_mu);
    DeviceWorkspaces& d = g_ws[device & 63];
    if (w->capturing) {
      w->counters = find_counters(d, w->capture_id, deps, num_deps);
      if (w->counters == nullptr && (w->counters = reserve_counters(d, most)) != nullptr)
        d.captures[d.next_capture++ % kMaxCaptures] = CaptureCounters{w->capture_id, nullptr, w->counters};
    } else {
      KeptWorkspace* k = nullptr;
      for (int i = 0; i < d.kept_count && k == nullptr; ++i)
        if (d.kept[i].stream_id == id) k = &d.kept[i];
      if (k == nullptr) {
        rc = new_workspace(d, id, most, device, s, &k);
        if (rc) return rc;
      }
      if (k != nullptr) {
        ++k->users;
        k->used = ++d.calls;
        w->kept = k;
        w->counters = k->counters;
        w->parts = k->parts;
        return CLOVE_OK;
      }
    }
  }
  // Partial results, and counters where none were left, for this call alone.
  const size_t head = w->counters == nullptr ? static_cast<size_t>(most) * sizeof(unsigned) : 0;
  rc = scratch_alloc(&w->own, head + part_bytes, device, w->capturing, s);
  if (rc) return rc;
  w->parts = reinterpret_cast<float*>(static_cast<char*>(w->own) + head);
  if (head != 0) {
    w->counters = static_cast<unsigned*>(w->own);
    rc = check_cuda(cudaMemsetAsync(w->own, 0, head, s), "cudaMemsetAsync(paged attention)");
    if (rc) scratch_free(w->own, w->capturing, s);
  }
  return rc;
}

int drop_workspace(Workspace* w, int device, cudaStream_t s) {
  if (w->kept != nullptr) {
    std::lock_guard<std::mutex> lock(g_ws_mu);
    KeptWorkspace& k = *w->kept;
    --k.users;
    // (One stream alone, as a rule, needs no event: nobody takes over from it.)
    k.recorded = false;
    if (g_ws[device & 63].kept_count == 1) return CLOVE_OK;
    const int rc = check_cuda(cudaEventRecord(k.event, s), "cudaEventRecord(paged attention)");
    k.recorded = rc == CLOVE_OK;
    return rc;
  }
  if (w->own == nullptr) return CLOVE_OK;
  const int rc = scratch_free(w->own, w->capturing, s);
  if (rc || !w->capturing) return rc;
  // The node that a later call has to follow to take the same counters.
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  const cudaGraphNode_t* deps = nullptr;
  const cudaGraphEdgeData* edges = nullptr;
  size_t num_deps = 0;
  if (cudaStreamGetCaptureInfo_v3(s, &cap, &id, nullptr, &deps, &edges, &num_deps) != cudaSuccess ||
      id != w->capture_id || num_deps != 1)
    return CLOVE_OK;
  std::lock_guard<std::mutex> lock(g_ws_mu);
  for (CaptureCounters& c : g_ws[device & 63].captures)
    if (c.capture_id == id && c.counters == w->counters) c.last = deps[0];
  return CLOVE_OK;
}

// Checks a cache description and converts it; `dtype` is the 16-bit type it is used with.
int take_cache(const clove_paged_cache* c, int dtype, kern::PagedCache* out) {
  if (c == nullptr) return fail(CLOVE_ERR_INVALID_ARG, "cache is NULL");
  if (c->K == nullptr || c->V == nullptr) return fail(CLOVE_ERR_INVALID_ARG, "cache: null K or V");
  if (c->num_pages <= 0 || c->num_kv_heads <= 0)
    return fail(CLOVE_ERR_INVALID_ARG, "cache: num_pages and num_kv_heads must be positive");
  if (c->page_size <= 0 || (c->page_size & (c->page_size - 1)) != 0)
    return fail(CLOVE_ERR_UNSUPPORTED, "cache: page_size %d is not a power of two", c->page_size);
  if (static_cast<long long>(c->num_pages) * c->page_size > INT_MAX)
    return fail(CLOVE_ERR_UNSUPPORTED, "cache: more than 2^31 - 1 slots");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(CLOVE_ERR_UNSUPPORTED, "cache: head_dim %d (64, 128 and 256 are supported)", c->head_dim);
  if (c->dtype != CLOVE_DTYPE_F16 && c->dtype != CLOVE_DTYPE_BF16 && c->dtype != CLOVE_DTYPE_E4M3)
    return fail(CLOVE_ERR_INVALID_ARG, "cache: unknown dtype %d", c->dtype);
  if (dtype >= 0 && c->dtype != dtype && c->dtype != CLOVE_DTYPE_E4M3)
    return fail(CLOVE_ERR_UNSUPPORTED, "cache: its type must be the operands' or e4m3");
  const int eb = c->dtype == CLOVE_DTYPE_E4M3 ? 1 : 2;
  if (!aligned(c->K, 16) || !aligned(c->V, 16) || (c->page_stride * eb) % 16 != 0 ||
      (c->token_stride * eb) % 16 != 0 || (c->head_stride * eb) % 16 != 0)
    return fail(CLOVE_ERR_UNSUPPORTED, "cache: K, V and the strides must be multiples of 16 bytes");
  if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0)
    return fail(CLOVE_ERR_INVALID_ARG, "cache: negative stride");
  if (!(c->k_scale > 0.f) || !(c->v_scale > 0.f) || !std::isfinite(c->k_scale) || !std::isfinite(c->v_scale))
    return fail(CLOVE_ERR_INVALID_ARG, "cache: scales must be positive and finite");
  if (eb == 2 && (c->k_scale != 1.f || c->v_scale != 1.f))
    return fail(CLOVE_ERR_INVALID_ARG, "cache: only an e4m3 cache has scales");
  out->K = c->K;
  out->V = c->V;
  out->num_pages = c->num_pages;
  out->page_shift = 0;
  while ((1 << out->page_shift) < c->page_size) ++out->page_shift;
  out->kv_heads = c->num_kv_heads;
  out->page_stride = c->page_stride;
  out->token_stride = c->token_stride;
  out->head_stride = c->head_stride;
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  return CLOVE_OK;
}

}  // namespace
}  // namespace rt
}  // namespace clove

using namespace clove;
using namespace clove::rt;

extern "C" {

int clove_qk_norm_rope(const void* Q, const void* K, const void* V, long long q_stride,
                       long long k_stride, long long v_stride, const void* q_weight,
                       const void* k_weight, float eps, const float* rope_table, int table_len,
                       int rotary_dim, int interleaved, const int* positions,
                       const clove_paged_cache* cache, const int* slots, void* Q_out,
                       long long q_out_stride, void* K_out, long long k_out_stride, int num_tokens,
                       int num_heads, int num_kv_heads, int head_dim, int dtype, void* stream) {
  if (num_tokens < 0) return fail(CLOVE_ERR_INVALID_ARG, "negative num_tokens");
  if (num_heads <= 0 || num_kv_heads <= 0)
    return fail(CLOVE_ERR_INVALID_ARG, "num_heads and num_kv_heads must be positive");
  if (dtype != CLOVE_DTYPE_F16 && dtype != CLOVE_DTYPE_BF16)
    return fail(CLOVE_ERR_INVALID_ARG, "dtype must be CLOVE_DTYPE_F16 or CLOVE_DTYPE_BF16");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(CLOVE_ERR_UNSUPPORTED, "head_dim %d (64, 128 and 256 are supported)", head_dim);
  if (rotary_dim <= 0 || rotary_dim % 16 != 0 || rotary_dim > head_dim)
    return fail(CLOVE_ERR_UNSUPPORTED, "rotary_dim %d must be a multiple of 16 up to head_dim", rotary_dim);
  if (table_len <= 0) return fail(CLOVE_ERR_INVALID_ARG, "the rotation table is empty");
  if ((q_weight == nullptr) != (k_weight == nullptr))
    return fail(CLOVE_ERR_INVALID_ARG, "q_weight and k_weight: both or neither");
  if (!(eps >= 0.f) || !std::isfinite(eps))
    return fail(CLOVE_ERR_INVALID_ARG, "eps must be finite and not negative");
  kern::RopeParams p = {};
  int cache_dtype = dtype;
  if (cache != nullptr) {
    const int rc = take_cache(cache, dtype, &p.cache);
    if (rc) return rc;
    if (cache->num_kv_heads != num_kv_heads || cache->head_dim != head_dim)
      return fail(CLOVE_ERR_INVALID_ARG, "the cache has %d heads of %d, K has %d of %d", cache->num_kv_heads,
                  cache->head_dim, num_kv_heads, head_dim);
    if (!std::isfinite(1.f / cache->k_scale) || !std::isfinite(1.f / cache->v_scale))
      return fail(CLOVE_ERR_INVALID_ARG, "cache: a scale's inverse exceeds fp32");
    if (num_tokens > 0 && (V == nullptr || slots == nullptr))
      return fail(CLOVE_ERR_INVALID_ARG, "a cache needs V and slots");
    cache_dtype = cache->dtype;
  } else if (V != nullptr || slots != nullptr) {
    return fail(CLOVE_ERR_INVALID_ARG, "V and slots need a cache");
  }
  if (num_tokens == 0) return CLOVE_OK;
  if (Q == nullptr || K == nullptr || Q_out == nullptr || rope_table == nullptr || positions == nullptr ||
      (K_out == nullptr && cache == nullptr))
    return fail(CLOVE_ERR_INVALID_ARG, "null pointer");
  if (!aligned(Q, 16) || !aligned(K, 16) || !aligned(V, 16) || !aligned(Q_out, 16) || !aligned(K_out, 16) ||
      !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(rope_table, 16))
    return fail(CLOVE_ERR_UNSUPPORTED, "qk_norm_rope needs 16-byte aligned tensors");
  if (!aligned(positions, 4) || !aligned(slots, 4))
    return fail(CLOVE_ERR_INVALID_ARG, "positions and slots must be 4-byte aligned");
  const long long qn = static_cast<long long>(num_heads) * head_dim, kn = static_cast<long long>(num_kv_heads) * head_dim;
  if (num_tokens > 1 && (q_stride < qn || k_stride < kn || q_out_stride < qn || (K_out && k_out_stride < kn) ||
                         (V && v_stride < kn)))
    return fail(CLOVE_ERR_INVALID_ARG, "a token stride is smaller than the token's heads");
  if (q_stride % 8 || k_stride % 8 || (V && v_stride % 8) || q_out_stride % 8 || (K_out && k_out_stride % 8))
    return fail(CLOVE_ERR_UNSUPPORTED, "token strides must be multiples of 8 elements");
  if (static_cast<long long>(num_heads) + 2LL * num_kv_heads > 65535)
    return fail(CLOVE_ERR_UNSUPPORTED, "over 65535 head rows per token");
  DeviceInfo dev;
  const int rc = current_device(&dev);
  if (rc) return rc;
  p.part[0] = kern::RopePart{Q, Q_out, q_weight, q_stride, q_out_stride, num_heads, 0u, 0, 0};
  p.part[1] = kern::RopePart{K, K_out, k_weight, k_stride, k_out_stride, num_kv_heads, 0u, 0, 0};
  p.part[2] = kern::RopePart{V, nullptr, nullptr, v_stride, 0, cache != nullptr ? num_kv_heads : 0, 0u, 0, 0};
  p.table = rope_table;
  p.positions = positions;
  p.slots = slots;
  p.tokens = num_tokens;
  p.table_len = table_len;
  p.rotary = rotary_dim;
  p.interleaved = interleaved != 0;
  p.eps = eps;
  p.k_per_scale = cache != nullptr ? 1.f / p.cache.k_scale : 1.f;
  p.v_per_scale = cache != nullptr ? 1.f / p.cache.v_scale : 1.f;
  return launch_qk_norm_rope(p, head_dim, dtype, cache_dtype, dev, static_cast<cudaStream_t>(stream));
}

int clove_paged_attention(const void* Q, long long q_stride, const clove_paged_cache* cache,
                          const int* page_table, long long table_stride, int max_pages,
                          const int* seq_lens, void* O, long long o_stride, float* lse,
                          float* key_weights, int accumulate, int batch, int num_heads, float scale,
                          int window, int dtype, void* stream) {
  if (batch < 0) return fail(CLOVE_ERR_INVALID_ARG, "negative batch");
  if (num_heads <= 0) return fail(CLOVE_ERR_INVALID_ARG, "num_heads must be positive");
  if (dtype != CLOVE_DTYPE_F16 && dtype != CLOVE_DTYPE_BF16)
    return fail(CLOVE_ERR_INVALID_ARG, "dtype must be CLOVE_DTYPE_F16 or CLOVE_DTYPE_BF16");
  kern::PagedAttnParams p = {};
  int rc = take_cache(cache, dtype, &p.cache);
  if (rc) return rc;
  if (num_heads % cache->num_kv_heads != 0)
    return fail(CLOVE_ERR_INVALID_ARG, "num_heads (%d) is not a multiple of num_kv_heads (%d)", num_heads,
                cache->num_kv_heads);
  if (!(scale > 0.f) || !std::isfinite(scale))
    return fail(CLOVE_ERR_INVALID_ARG, "scale must be positive and finite");
  // Scores are multiplied by this. Subnormal, it would have lost its digits.
  p.scale_log2 = scale * p.cache.k_scale * 1.4426950408889634f;
  if (!std::isnormal(p.scale_log2))
    return fail(CLOVE_ERR_INVALID_ARG, "scale * k_scale leaves the range of fp32");
  if (window < 0) return fail(CLOVE_ERR_INVALID_ARG, "negative window");
  if (max_pages < 0) return fail(CLOVE_ERR_INVALID_ARG, "negative max_pages");
  if (batch == 0) return CLOVE_OK;
  if (Q == nullptr || O == nullptr || seq_lens == nullptr || (page_table == nullptr && max_pages > 0))
    return fail(CLOVE_ERR_INVALID_ARG, "null pointer");
  if (!aligned(Q, 16) || !aligned(O, 16) || q_stride % 8 || o_stride % 8)
    return fail(CLOVE_ERR_UNSUPPORTED, "paged_attention: Q and O 16-byte aligned, strides multiples of 8 elements");
  if (!aligned(page_table, 4) || !aligned(seq_lens, 4) || !aligned(lse, 4) || !aligned(key_weights, 4))
    return fail(CLOVE_ERR_INVALID_ARG, "int and float arrays must be 4-byte aligned");
  const int D = cache->head_dim;
  if (batch > 1 && (q_stride < static_cast<long long>(num_heads) * D ||
                    o_stride < static_cast<long long>(num_heads) * D || table_stride < max_pages))
    return fail(CLOVE_ERR_INVALID_ARG, "a row stride is smaller than the row");
  const long long capacity = static_cast<long long>(max_pages) * cache->page_size;
  if (capacity > INT_MAX - 65536) return fail(CLOVE_ERR_UNSUPPORTED, "page table rows name over 2^31 tokens");
  DeviceInfo dev;
  rc = current_device(&dev);
  if (rc) return rc;
  const bool e4m3 = cache->dtype == CLOVE_DTYPE_E4M3;
  p.q = Q;
  p.o = O;
  p.lse = lse;
  p.q_stride = q_stride;
  p.o_stride = o_stride;
  p.page_table = page_table;
  p.seq_lens = seq_lens;
  p.table_stride = table_stride;
  p.capacity = static_cast<int>(capacity);
  p.batch = batch;
  p.heads = num_heads;
  p.group = num_heads / cache->num_kv_heads;
  // Blocks of 16 heads once a group has more than 8 (one pass over the keys instead of
  // two); head_dim 256 keeps 8, whose accumulators already take half the registers.
  const int hb = D <= 128 && p.group > 8 ? 16 : 8;
  p.blocks = (p.group + hb - 1) / hb;
  p.window = window;
  p.v_scale = p.cache.v_scale;
  p.key_weights = key_weights;
  p.accumulate = accumulate != 0;
  // As many CTAs as fit at once, or as there can be tiles. The batch's empty rows need one.
  const double most = static_cast<double>(batch) * p.cache.kv_heads * p.blocks *
                      static_cast<double>(capacity / kern::kPagedTile + 2);
  if (most > INT_MAX) return fail(CLOVE_ERR_UNSUPPORTED, "paged_attention: batch x heads x table exceeds 2^31 tiles");
  const long long tiles = static_cast<long long>(most);
  const int ctas = static_cast<int>(std::min<long long>(paged_attention_max_ctas(D, hb, e4m3, dev), tiles));
  const size_t heads = (static_cast<size_t>(batch) * num_heads * 4 + 255) & ~size_t(255);
  const size_t scores = static_cast<size_t>(batch) * num_heads * static_cast<size_t>(capacity) * 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Workspace ws;
  rc = take_workspace(&ws, ctas, static_cast<size_t>(ctas) * 2 * hb * (D + 2) * 4, dev, s);
  if (rc) return rc;
  p.counters = ws.counters;
  p.part_o = ws.parts;
  p.part_m = p.part_o + static_cast<size_t>(ctas) * 2 * hb * D;
  p.part_l = p.part_m + static_cast<size_t>(ctas) * 2 * hb;
  char* sc = nullptr;
  if (key_weights != nullptr) {
    rc = scratch_alloc(reinterpret_cast<void**>(&sc), heads + scores, dev.device, ws.capturing, s);
    if (!rc) {
      p.lse2 = reinterpret_cast<float*>(sc);
      p.scores = reinterpret_cast<float*>(sc + heads);
    }
  }
  if (!rc)
    rc = dtype == CLOVE_DTYPE_F16 ? launch_paged_attention_f16(p, D, hb, e4m3, ctas, dev, s)
                                  : launch_paged_attention_bf16(p, D, hb, e4m3, ctas, dev, s);
  if (sc != nullptr) {
    const int rc2 = scratch_free(sc, ws.capturing, s);
    if (!rc) rc = rc2;
  }
  const int rc2 = drop_workspace(&ws, dev.device, s);
  return rc ? rc : rc2;
}

int clove_evict_cache(const clove_paged_cache* cache, float* key_weights, const int* page_table,
                      long long table_stride, int max_pages, const int* seq_lens, const int* dst_table,
                      long long dst_stride, int dst_pages, int* kept, int* new_lens, int batch, int budget,
                      int recent, void* stream) {
  if (batch < 0) return fail(CLOVE_ERR_INVALID_ARG, "negative batch");
  kern::EvictParams p = {};
  int rc = take_cache(cache, -1, &p.cache);
  if (rc) return rc;
  if (budget <= 0) return fail(CLOVE_ERR_INVALID_ARG, "budget must be positive");
  if (budget > (1 << 30)) return fail(CLOVE_ERR_UNSUPPORTED, "budget beyond 2^30 tokens");
  if (recent < 0 || recent > budget) return fail(CLOVE_ERR_INVALID_ARG, "recent must be in [0, budget]");
  if (max_pages < 0 || dst_pages < 0) return fail(CLOVE_ERR_INVALID_ARG, "negative table width");
  if (static_cast<long long>(dst_pages) * cache->page_size < budget)
    return fail(CLOVE_ERR_INVALID_ARG, "dst_table rows name %lld tokens, the budget is %d",
                static_cast<long long>(dst_pages) * cache->page_size, budget);
  if (batch == 0) return CLOVE_OK;
  if (key_weights == nullptr || seq_lens == nullptr || dst_table == nullptr || kept == nullptr ||
      new_lens == nullptr || (page_table == nullptr && max_pages > 0))
    return fail(CLOVE_ERR_INVALID_ARG, "null pointer");
  if (!aligned(key_weights, 4) || !aligned(seq_lens, 4) || !aligned(dst_table, 4) || !aligned(kept, 4) ||
      !aligned(new_lens, 4) || !aligned(page_table, 4))
    return fail(CLOVE_ERR_INVALID_ARG, "int and float arrays must be 4-byte aligned");
  if (batch > 1 && (table_stride < max_pages || dst_stride < dst_pages))
    return fail(CLOVE_ERR_INVALID_ARG, "a row stride is smaller than the row");
  const long long capacity = static_cast<long long>(max_pages) * cache->page_size;
  if (capacity > INT_MAX - 16384) return fail(CLOVE_ERR_UNSUPPORTED, "page table rows name over 2^31 tokens");
  DeviceInfo dev;
  rc = current_device(&dev);
  if (rc) return rc;
  p.page_table = page_table;
  p.seq_lens = seq_lens;
  p.dst_table = dst_table;
  p.table_stride = table_stride;
  p.dst_stride = dst_stride;
  p.capacity = static_cast<int>(capacity);
  p.batch = batch;
  p.budget = budget;
  p.recent = recent;
  p.key_weights = key_weights;
  p.kept = kept;
  p.new_lens = new_lens;
  p.elem = cache->dtype == CLOVE_DTYPE_E4M3 ? 1 : 2;
  p.row_bytes = cache->head_dim * p.elem;
  return launch_evict_cache(p, dev, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
