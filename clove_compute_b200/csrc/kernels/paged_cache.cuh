// paged_cache.cuh -- what the paged-cache kernels share: the 16-bit / 8-bit element types
// and their conversions to fp32 in quads.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "paged_params.h"
#include "sm100_ptx.cuh"

namespace clove {
namespace kern {

using fp8_e4m3 = __nv_fp8_e4m3;

// Four consecutive elements as fp32 and back (8-byte accesses for 16-bit types, 4-byte
// for e4m3). Stores round to nearest even; e4m3 saturates at +-448 and keeps NaN.
template <typename T>
struct Quad;

template <>
struct Quad<__half> {
  using Raw = uint2;
  __device__ static __forceinline__ void unpack(Raw r, float (&v)[4]) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
  __device__ static __forceinline__ Raw pack(const float (&v)[4]) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
};

template <>
struct Quad<__nv_bfloat16> {
  using Raw = uint2;
  __device__ static __forceinline__ void unpack(Raw r, float (&v)[4]) {
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
  __device__ static __forceinline__ Raw pack(const float (&v)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
};

template <>
struct Quad<fp8_e4m3> {
  using Raw = uint32_t;
  __device__ static __forceinline__ Raw pack(const float (&v)[4]) {
    const uint32_t lo =
        __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi =
        __nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
};

// A sequence's keys: [first, len), cut into tiles of TILE from `base` (first rounded down to
// 16).
struct PagedSpan {
  int len, first, base, tiles;
};
template <int TILE>
__device__ __forceinline__ PagedSpan paged_span(const PagedAttnParams& p, int b) {
  PagedSpan s;
  int n = p.seq_lens[b];
  n = n < 0 ? 0 : (n > p.capacity ? p.capacity : n);
  s.len = n;
  s.first = p.window > 0 && n > p.window ? n - p.window : 0;
  s.base = s.first & ~15;
  s.tiles = n > 0 ? (n - s.base + TILE - 1) / TILE : 0;
  return s;
}

}  // namespace kern
}  // namespace clove
