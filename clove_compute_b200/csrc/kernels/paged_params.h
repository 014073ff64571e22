// paged_params.h -- launch parameters of the paged-cache kernels, shared by the host
// entry points and the kernel translation units.
#pragma once

#include <cstdint>

namespace clove {
namespace kern {

// A paged key-value cache. Strides in elements, the same for K and V; the innermost
// (head_dim) one is 1. page_size is a power of two (page_shift = log2).
struct PagedCache {
  void* K;
  void* V;
  int num_pages;
  int page_shift;
  int kv_heads;
  long long page_stride;
  long long token_stride;
  long long head_stride;
  float k_scale;
  float v_scale;
};

// qk_norm_rope.cu. One kind of row (queries, keys, values) of every token.
struct RopePart {
  const void* in;
  void* out;           // null: not wanted (keys with a cache; values)
  const void* weight;  // null: no norm
  long long in_stride, out_stride;
  int rows;  // per token; 0: none
  // Filled by the launcher: the kind's first block, log2 of the rows of a token side by
  // side, blocks per group of tokens.
  unsigned first;
  int shift, chunks;
};
struct RopeParams {
  RopePart part[3];
  const float* table;
  const int* positions;
  const int* slots;  // null: no cache
  int tokens, table_len, rotary, interleaved;
  float eps;
  float k_per_scale, v_per_scale;  // 1 / the cache's scales
  PagedCache cache;
};

// paged_attention_sm100.cuh
constexpr int kPagedTile = 64;  // keys per CTA step, at least (64 or 128)
constexpr int kPagedCounters = 1 << 18;
struct PagedAttnParams {
  const void* q;
  void* o;
  float* lse;  // may be null
  long long q_stride, o_stride;
  const int* page_table;  // [batch, max_pages], rows table_stride apart
  const int* seq_lens;
  long long table_stride;
  int capacity;  // max_pages * page_size: tokens a table row can name
  int batch, heads;
  int group;   // query heads per key head
  int blocks;  // head blocks per key head: ceil(group / heads in a block)
  int window;  // 0: all keys
  float scale_log2;  // scale * k_scale * log2(e)
  float v_scale;
  // Workspace: per CTA two partial results (heads in a block x D sums, maxima, totals) and
  // one counter, zero before and after the call. Calls that run one after the other may
  // share them.
  float* part_o;
  float* part_m;
  float* part_l;
  unsigned* counters;
  // Key weights (null: not asked for): the scores of every key and head, times log2(e),
  // [batch, kv_heads, capacity, group], and each head's log2-sum-exp2 [batch, heads].
  float* scores;
  float* lse2;
  float* key_weights;  // [num_pages, kv_heads, page_size]
  int accumulate;
  PagedCache cache;
};

// evict_cache.cu
struct EvictParams {
  const int* page_table;
  const int* seq_lens;
  const int* dst_table;
  long long table_stride, dst_stride;
  int capacity;      // tokens a page_table row can name
  int batch;
  int budget, recent;
  float* key_weights;  // [num_pages, kv_heads, page_size]
  int* kept;           // [batch, kv_heads, budget]
  int* new_lens;       // [batch]
  int row_bytes;       // one head's K (or V) row
  int elem;            // bytes per cache element
  PagedCache cache;
};

}  // namespace kern
}  // namespace clove
