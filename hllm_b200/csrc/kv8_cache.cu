// kv8_cache.cu -- writing the 8-bit paged KV cache (q/k RMSNorm, rotary
// positions, quantisation) and reading it back.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "kv8.cuh"

namespace hb {
namespace {

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) {
  return *reinterpret_cast<const float4*>(p);
}
template <>
__device__ __forceinline__ float4 load4<__half>(const __half* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u),
                     __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
}

// ---------------------------------------------------------------- write
// Per token t and head h of qkv: y = x * (1 / sqrt(mean x^2 + eps)) * w for q
// and k where weights are given; then for i < rotary / 2 the pair (i, i +
// rotary/2), or (2i, 2i + 1) interleaved, turns by a = 2 pi * position *
// turns[i]:  y0' = y0 c - y1 s, y1' = y1 c + y0 s, c = factor cos a, s =
// factor sin a.  q goes out as F16; K and V rows are quantised (kv8.cuh) into
// page slot / 16, row slot % 16.  Memory-bound: every element is read once and
// written once.
//
// The angle is reduced to a fraction of a turn in 64 bits (position * turns
// minus its nearest integer), so a position of 10^6 is as exact as 0; F32
// angles would be off by 0.03 rad there.  The CTA's heads share one token's
// cosines through shared memory: 64 pairs of 64-bit products a token, not a
// head.
constexpr int kWriteThreads = 256;

template <typename T, int LANES, int GROUPS>  // LANES threads a head, GROUPS x 4 elements each
__global__ void __launch_bounds__(kWriteThreads) kv8_write_kernel(const Kv8WriteArgs a) {
  constexpr int kUnits = kWriteThreads / LANES;
  __shared__ float2 cs[kKv8MaxDim / 2];
  __shared__ __align__(16) float buf[kUnits][4 * LANES * GROUPS];
  griddep_enter();
  const int t = blockIdx.x;
  const int d = a.cache.dim, hkv = a.cache.hkv, hq = a.hq;
  const int heads = hq + 2 * hkv;
  const int unit = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const int step = gridDim.y * kUnits;
  const int h0 = blockIdx.y * kUnits + unit;
  const T* row = static_cast<const T*>(a.qkv) + static_cast<size_t>(t) * heads * d;
  const int slot = a.slots[t];
  const int pos = a.positions[t];
  float4 x[GROUPS];
  auto fetch = [&](int h) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int i = (g * LANES + lane) * 4;
      x[g] = h < heads && i < d ? load4<T>(row + static_cast<size_t>(h) * d + i)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  fetch(h0);
  const int half = a.rotary >> 1;
  for (int i = threadIdx.x; i < half; i += kWriteThreads) {
    const double turns = static_cast<double>(pos) * a.turns[i];
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c * a.factor, s * a.factor);
  }
  const bool stored = slot >= 0 && slot < a.cache.blocks * kKv8Page;
  if (threadIdx.x == 0 && slot >= 0 && !stored) atomicOr(a.status, kDevBadIndex);
  __syncthreads();

  auto sum_lanes = [&](float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto max_lanes = [&](float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  for (int base = blockIdx.y * kUnits; base < heads; base += step) {  // uniform over the CTA
    const int h = base + unit;
    const bool live = h < heads;
    const bool is_q = h < hq, is_v = h >= hq + hkv;
    const float* w = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
    float y[GROUPS][4];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      y[g][0] = x[g].x;
      y[g][1] = x[g].y;
      y[g][2] = x[g].z;
      y[g][3] = x[g].w;
    }
    fetch(h + step);  // the next head's loads run under this head's arithmetic
    // Shuffles take part in whole warps: a warp may hold two heads of different kinds.
    float ss = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      ss += y[g][0] * y[g][0] + y[g][1] * y[g][1] + y[g][2] * y[g][2] + y[g][3] * y[g][3];
    ss = sum_lanes(ss);
    if (w && live) {
      const float inv = 1.0f / sqrtf(ss / static_cast<float>(d) + a.eps);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int i = (g * LANES + lane) * 4;
        if (i < d) {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[g][e] = y[g][e] * inv * w[i + e];
        }
      }
    }
    if (a.interleaved) {
      if (!is_v) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const int i = (g * LANES + lane) * 4;
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            if (i + e < a.rotary) {
              const float2 r = cs[(i + e) >> 1];
              const float y0 = y[g][e], y1 = y[g][e + 1];
              y[g][e] = y0 * r.x - y1 * r.y;
              y[g][e + 1] = y1 * r.x + y0 * r.y;
            }
          }
        }
      }
    } else {
      // The other half of a pair lies in another lane: through shared memory.
      float* b = buf[unit];
      __syncwarp();
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        *reinterpret_cast<float4*>(b + (g * LANES + lane) * 4) =
            make_float4(y[g][0], y[g][1], y[g][2], y[g][3]);
      __syncwarp();
      if (!is_v) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const int i = (g * LANES + lane) * 4;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = i + e;
            if (j < a.rotary) {
              const bool lo = j < half;
              const float2 r = cs[lo ? j : j - half];
              const float other = b[lo ? j + half : j - half];
              y[g][e] = lo ? y[g][e] * r.x - other * r.y : y[g][e] * r.x + other * r.y;
            }
          }
        }
      }
    }
    if (is_q) {
      if (live) {
        __half* dst = a.q_out + (static_cast<size_t>(t) * hq + h) * d;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const int i = (g * LANES + lane) * 4;
          if (i < d) {
            __half2 p[2] = {__floats2half2_rn(y[g][0], y[g][1]), __floats2half2_rn(y[g][2], y[g][3])};
            *reinterpret_cast<uint2*>(dst + i) = *reinterpret_cast<uint2*>(p);
          }
        }
      }
    }
    float top = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float m = fabsf(y[g][e]);
        if (m <= kKv8Limit) top = fmaxf(top, m);
        else y[g][e] = __uint_as_float(0x7fffffffu);  // not finite, or past the format
      }
    top = max_lanes(top);
    if (!is_q && live && stored) {
      const int e = kv8_exponent(top);
      const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      const int kvh = is_v ? h - hq - hkv : h - hq;
      const size_t at = (static_cast<size_t>(slot / kKv8Page) * hkv + kvh) * kKv8Page + slot % kKv8Page;
      uint8_t* dst = (is_v ? a.cache.v : a.cache.k) + at * d;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int i = (g * LANES + lane) * 4;
        if (i < d)
          *reinterpret_cast<uint32_t*>(dst + i) =
              kv8_codes(y[g][0] * inv, y[g][1] * inv) | (kv8_codes(y[g][2] * inv, y[g][3] * inv) << 16);
      }
      if (lane == 0) (is_v ? a.cache.v_scale : a.cache.k_scale)[at] = static_cast<uint8_t>(e + 127);
    }
  }
}

template <typename T, int LANES, int GROUPS>
cudaError_t launch_write(const Kv8WriteArgs& a, cudaStream_t stream) {
  constexpr int kUnits = kWriteThreads / LANES;
  const int heads = a.hq + 2 * a.cache.hkv;
  // Few tokens: a head a unit, so that the whole call is one round of loads.
  // Many tokens: one CTA walks a token's heads and computes its angles once.
  const int slices = (heads + kUnits - 1) / kUnits;
  const int y = a.tokens >= 592 ? 1 : slices;
  return launch_dependent(kv8_write_kernel<T, LANES, GROUPS>, dim3(a.tokens, y),
                          dim3(kWriteThreads), 0, stream, a);
}

template <typename T>
cudaError_t dispatch_write(const Kv8WriteArgs& a, cudaStream_t stream) {
  if (a.cache.dim <= 64) return launch_write<T, 16, 1>(a, stream);
  if (a.cache.dim <= 128) return launch_write<T, 32, 1>(a, stream);
  return launch_write<T, 32, 2>(a, stream);
}

// ---------------------------------------------------------------- read
// value = code * 2^e, rounded once to the output type.  Memory-bound.  A CTA
// takes kReadTokens consecutive output rows: one warp finds their pages, then
// every thread converts 16 codes at a time (one 16-byte load).
constexpr int kReadThreads = 256;
constexpr int kReadTokens = 16;

template <typename T>
__device__ __forceinline__ void store16(T* dst, const uint4& w, float s);
template <>
__device__ __forceinline__ void store16<float>(float* dst, const uint4& w, float s) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = kv8_half2_lo(v[j]), hi = kv8_half2_hi(v[j]);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    reinterpret_cast<float4*>(dst)[j] = make_float4(a.x * s, a.y * s, b.x * s, b.y * s);
  }
}
template <>
__device__ __forceinline__ void store16<__half>(__half* dst, const uint4& w, float s) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  uint32_t o[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = kv8_half2_lo(v[j]), hi = kv8_half2_hi(v[j]);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    const __half2 p = __floats2half2_rn(a.x * s, a.y * s), q = __floats2half2_rn(b.x * s, b.y * s);
    o[2 * j] = *reinterpret_cast<const uint32_t*>(&p);
    o[2 * j + 1] = *reinterpret_cast<const uint32_t*>(&q);
  }
  reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
  reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
}
template <>
__device__ __forceinline__ void store16<__nv_bfloat16>(__nv_bfloat16* dst, const uint4& w, float s) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  uint32_t o[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = kv8_half2_lo(v[j]), hi = kv8_half2_hi(v[j]);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    const __nv_bfloat162 p = __floats2bfloat162_rn(a.x * s, a.y * s);
    const __nv_bfloat162 q = __floats2bfloat162_rn(b.x * s, b.y * s);
    o[2 * j] = *reinterpret_cast<const uint32_t*>(&p);
    o[2 * j + 1] = *reinterpret_cast<const uint32_t*>(&q);
  }
  reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
  reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

template <typename T>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(const Kv8ReadArgs a) {
  __shared__ long long source[kReadTokens];  // row of (kv head 0) in the pool, -1: none, -2: no output
  griddep_enter();
  const int t0 = blockIdx.x * kReadTokens;
  const int hkv = a.cache.hkv, d = a.cache.dim;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    // Row of each token: the number of rows that end at or before it.
    const int t = t0 + lane;
    int r = 0;
    for (int base = 0; base < a.rows; base += 32) {
      const int end = base + lane < a.rows ? a.offsets[base + lane + 1] : 0x7fffffff;
      const int n = min(32, a.rows - base);
      for (int k = 0; k < n; ++k) r += __shfl_sync(0xffffffffu, end, k) <= t ? 1 : 0;
    }
    if (lane < kReadTokens) {
      long long src = -2;
      const int begin = a.offsets[0];
      if (r < a.rows && t < a.tokens && t >= begin) {
        const int first = a.first ? a.first[r] : 0;
        const long long p = static_cast<long long>(first) + (t - a.offsets[r]);
        src = -1;
        if (p >= 0 && p < a.lengths[r] && p < static_cast<long long>(a.max_blocks) * kKv8Page) {
          const int b = a.tables[static_cast<size_t>(r) * a.max_blocks + p / kKv8Page];
          if (b >= 0 && b < a.cache.blocks)
            src = static_cast<long long>(b) * hkv * kKv8Page + p % kKv8Page;
        }
        if (src < 0) atomicOr(a.status, kDevBadIndex);
      }
      source[lane] = src;
    }
  }
  __syncthreads();
  const int chunks = d >> 4;
  const int per = hkv * chunks;
  for (int i = threadIdx.x; i < 2 * kReadTokens * per; i += kReadThreads) {
    const int which = i / (kReadTokens * per), rest = i % (kReadTokens * per);
    const int tl = rest / per, u = rest % per;
    const int kvh = u / chunks, c = u % chunks;
    const long long src = source[tl];
    if (src == -2) continue;
    T* dst = static_cast<T*>(which ? a.v_out : a.k_out) +
             (static_cast<size_t>(t0 + tl) * hkv + kvh) * d + c * 16;
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    float s = 0.f;
    if (src >= 0) {
      const size_t at = static_cast<size_t>(src) + static_cast<size_t>(kvh) * kKv8Page;
      w = __ldg(reinterpret_cast<const uint4*>((which ? a.cache.v : a.cache.k) + at * d + c * 16));
      s = kv8_scale(__ldg((which ? a.cache.v_scale : a.cache.k_scale) + at));
    }
    store16<T>(dst, w, s);
  }
}

}  // namespace

cudaError_t kv8_write_launch(const Kv8WriteArgs& a, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  switch (a.type) {
    case kKv8F32: return dispatch_write<float>(a, stream);
    case kKv8F16: return dispatch_write<__half>(a, stream);
    default: return dispatch_write<__nv_bfloat16>(a, stream);
  }
}

cudaError_t kv8_read_launch(const Kv8ReadArgs& a, cudaStream_t stream) {
  if (a.tokens == 0 || a.rows == 0) return cudaSuccess;
  const dim3 grid((a.tokens + kReadTokens - 1) / kReadTokens);
  switch (a.type) {
    case kKv8F32:
      return launch_dependent(kv8_read_kernel<float>, grid, dim3(kReadThreads), 0, stream, a);
    case kKv8F16:
      return launch_dependent(kv8_read_kernel<__half>, grid, dim3(kReadThreads), 0, stream, a);
    default:
      return launch_dependent(kv8_read_kernel<__nv_bfloat16>, grid, dim3(kReadThreads), 0, stream, a);
  }
}

}  // namespace hb
