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
// Bound by memory: every row is read once and written once. D / 8 lanes hold one row,
// each lane the two quads (four elements) whose elements pair with each other, so that
// the rotation needs no exchange between lanes and only the sum of squares is shuffled.
// A lane handles HPT rows of one token, all loaded before the first is used: one row
// where the call is small (a decode step: latency counts), four where it fills the GPU.
#include <algorithm>

#include "../runtime/internal.h"
#include "paged_cache.cuh"
#include "pdl_launch.h"

namespace clove {
namespace kern {

constexpr int kRopeThreads = 256;

// T: type of Q, K, V and the outputs; C: the cache's. LPR = D / 8 lanes per row.
template <typename T, typename C, int LPR, int HPT>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const RopeParams p) {
  using QT = Quad<T>;
  constexpr int D = LPR * 8;
  const int u = static_cast<int>(threadIdx.x) % LPR;
  const long long task =
      static_cast<long long>(blockIdx.x) * (kRopeThreads / LPR) + threadIdx.x / LPR;
  const long long token = task / p.chunks;
  const int chunk = static_cast<int>(task - token * p.chunks);
  dev::grid_dependency_wait();
  int pos = -1;
  if (token < p.tokens) pos = p.positions[token];
  // A negative position marks a padding token; one behind the table is an error. Both
  // leave every output row of the token as it was. (Lanes stay for the shuffles.)
  if (pos >= p.table_len) {
    if (u == 0) dev::record_error(dev::kDevErrBadIndex);
    pos = -1;
  }
  const bool live = pos >= 0;

  // This lane's quads [a, a + 4) and [b, b + 4) of the row: both rotated, or both kept.
  const int units = p.rotary / 8;
  const bool rotated = u < units;
  int a, b;
  if (rotated && !p.interleaved) {
    a = 4 * u;
    b = p.rotary / 2 + 4 * u;
  } else {
    a = 8 * u;
    b = a + 4;
  }
  const T* src[HPT];
  typename QT::Raw ra[HPT], rb[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int row = chunk + i * p.chunks;  // neighbouring lanes' rows are neighbours
    src[i] = nullptr;
    if (live && row < p.rows) {
      if (row < p.heads)
        src[i] = static_cast<const T*>(p.q) + token * p.q_stride + static_cast<long long>(row) * D;
      else if (row < p.heads + p.kv_heads)
        src[i] = static_cast<const T*>(p.k) + token * p.k_stride +
                 static_cast<long long>(row - p.heads) * D;
      else
        src[i] = static_cast<const T*>(p.v) + token * p.v_stride +
                 static_cast<long long>(row - p.heads - p.kv_heads) * D;
      ra[i] = *reinterpret_cast<const typename QT::Raw*>(src[i] + a);
      rb[i] = *reinterpret_cast<const typename QT::Raw*>(src[i] + b);
    }
  }
  float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live && rotated) {
    const float* t = p.table + static_cast<long long>(pos) * p.rotary + 4 * u;
    cs = *reinterpret_cast<const float4*>(t);
    sn = *reinterpret_cast<const float4*>(t + p.rotary / 2);
  }
  const float c[4] = {cs.x, cs.y, cs.z, cs.w}, s[4] = {sn.x, sn.y, sn.z, sn.w};
  long long slot_off = -1;  // element offset of the token's slot, head 0
  if (live && p.slots != nullptr) {
    const int slot = p.slots[token];
    const int page = slot >> p.cache.page_shift;
    if (slot >= 0 && page < p.cache.num_pages)
      slot_off = page * p.cache.page_stride +
                 (slot & ((1 << p.cache.page_shift) - 1)) * p.cache.token_stride;
    else if (slot >= 0 && u == 0)
      dev::record_error(dev::kDevErrBadIndex);
  }

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int row = chunk + i * p.chunks;
    const bool have = src[i] != nullptr;
    const bool is_v = row >= p.heads + p.kv_heads;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
    if (have) {
      QT::unpack(ra[i], x);
      QT::unpack(rb[i], y);
    }
    if (p.q_weight != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (have && !is_v) {
        const T* w = static_cast<const T*>(row < p.heads ? p.q_weight : p.k_weight);
        float wa[4], wb[4];
        QT::unpack(*reinterpret_cast<const typename QT::Raw*>(w + a), wa);
        QT::unpack(*reinterpret_cast<const typename QT::Raw*>(w + b), wb);
        const float inv = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = x[e] * inv * wa[e];
          y[e] = y[e] * inv * wb[e];
        }
      }
    }
    if (!have) continue;
    if (!is_v && rotated) {
      if (p.interleaved) {
        const float z[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        float r[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          r[2 * e] = z[2 * e] * c[e] - z[2 * e + 1] * s[e];
          r[2 * e + 1] = z[2 * e + 1] * c[e] + z[2 * e] * s[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = r[e], y[e] = r[4 + e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float lo = x[e] * c[e] - y[e] * s[e];
          y[e] = y[e] * c[e] + x[e] * s[e];
          x[e] = lo;
        }
      }
    }
    T* out = nullptr;
    if (row < p.heads)
      out = static_cast<T*>(p.q_out) + token * p.q_out_stride + static_cast<long long>(row) * D;
    else if (!is_v && p.k_out != nullptr)
      out = static_cast<T*>(p.k_out) + token * p.k_out_stride +
            static_cast<long long>(row - p.heads) * D;
    if (out != nullptr) {
      *reinterpret_cast<typename QT::Raw*>(out + a) = QT::pack(x);
      *reinterpret_cast<typename QT::Raw*>(out + b) = QT::pack(y);
    }
    if (row >= p.heads && slot_off >= 0) {
      const int h = is_v ? row - p.heads - p.kv_heads : row - p.heads;
      C* to = static_cast<C*>(is_v ? p.cache.V : p.cache.K) + slot_off + h * p.cache.head_stride;
      if (sizeof(C) == 1) {
        const float sc = is_v ? p.cache.v_scale : p.cache.k_scale;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] /= sc, y[e] /= sc;
      }
      *reinterpret_cast<typename Quad<C>::Raw*>(to + a) = Quad<C>::pack(x);
      *reinterpret_cast<typename Quad<C>::Raw*>(to + b) = Quad<C>::pack(y);
    }
  }
}

}  // namespace kern

namespace rt {

CLOVE_DEFINE_ERROR_READER(read_clear_error_rope)

namespace {

template <typename T, typename C, int LPR, int HPT>
int launch_rope_t(kern::RopeParams& p, cudaStream_t stream) {
  p.chunks = (p.rows + HPT - 1) / HPT;
  const int per_block = kern::kRopeThreads / LPR;
  const long long blocks = (static_cast<long long>(p.tokens) * p.chunks + per_block - 1) / per_block;
  if (blocks > 0x7fffffffLL) return fail(CLOVE_ERR_UNSUPPORTED, "qk_norm_rope: too many rows");
  cudaLaunchAttribute la[1];
  cudaLaunchConfig_t cfg =
      pdl_config(dim3(static_cast<unsigned>(blocks)), kern::kRopeThreads, 0, stream, la);
  return check_cuda(cudaLaunchKernelEx(&cfg, kern::qk_norm_rope_kernel<T, C, LPR, HPT>, p),
                    "qk_norm_rope launch");
}

template <typename T, typename C, int LPR>
int launch_rope_h(kern::RopeParams& p, const DeviceInfo& dev, cudaStream_t stream) {
  // Four rows per lane once that still gives every SM its 2048 threads.
  const long long threads = static_cast<long long>(p.tokens) * p.rows * LPR;
  if (threads >= 4LL * 2048 * dev.num_sms) return launch_rope_t<T, C, LPR, 4>(p, stream);
  return launch_rope_t<T, C, LPR, 1>(p, stream);
}

template <typename T, typename C>
int launch_rope_d(kern::RopeParams& p, int head_dim, const DeviceInfo& dev, cudaStream_t stream) {
  if (head_dim == 64) return launch_rope_h<T, C, 8>(p, dev, stream);
  if (head_dim == 128) return launch_rope_h<T, C, 16>(p, dev, stream);
  return launch_rope_h<T, C, 32>(p, dev, stream);
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
