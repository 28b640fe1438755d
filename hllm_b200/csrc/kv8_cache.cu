// kv8_cache.cu -- writing the 8-bit paged KV cache (q/k RMSNorm, rotary
// positions, quantisation) and reading it back.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kv8.cuh"

namespace hb {
namespace {

// Eight consecutive elements of a row as they lie in memory, and as F32.
template <typename T>
struct Eight {
  uint4 w;
  __device__ __forceinline__ void load(const T* p, bool live) {
    w = live ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ static float2 pair(uint32_t v) {
    if constexpr (std::is_same<T, __half>::value) {
      return __half22float2(*reinterpret_cast<const __half2*>(&v));
    } else {
      return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
  }
  __device__ __forceinline__ void values(float* y) const {
    const float2 a = pair(w.x), b = pair(w.y), c = pair(w.z), d = pair(w.w);
    y[0] = a.x, y[1] = a.y, y[2] = b.x, y[3] = b.y, y[4] = c.x, y[5] = c.y, y[6] = d.x, y[7] = d.y;
  }
};
template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, bool live) {
    a = b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
      a = __ldg(reinterpret_cast<const float4*>(p));
      b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
  }
  __device__ __forceinline__ void values(float* y) const {
    y[0] = a.x, y[1] = a.y, y[2] = a.z, y[3] = a.w, y[4] = b.x, y[5] = b.y, y[6] = b.z, y[7] = b.w;
  }
};

// ---------------------------------------------------------------- write
// Per token t and head h of qkv: y = x * (1 / sqrt(mean x^2 + eps)) * w for q
// and k where weights are given; then for i < rotary / 2 the pair (i, i +
// rotary/2), or (2i, 2i + 1) interleaved, turns by a = 2 pi * position *
// turns[i]:  y0' = y0 c - y1 s, y1' = y1 c + y0 s, c = factor cos a, s =
// factor sin a.  q goes out as F16; K and V rows are quantised (kv8.cuh) into
// page slot / 16, row slot % 16.  Memory-bound: every element is read once and
// written once.
//
// A warp takes one token and 32 / LANES of its heads at a time, the next
// heads' loads in flight under this step's arithmetic.  A lane holds both
// members of eight pairs: elements 8 j .. and rotary/2 + 8 j .. of a head (past
// `rotary`, and where pairs are neighbours: of halves of that), so pairs meet in
// registers; the pairs' cosines serve all the token's heads.
// Where rotary / 2 is not a multiple of 8 (kExchange) chunks of eight would
// cross a border, and a lane takes 16 consecutive elements and fetches the
// other members through shared memory.
//
// The angle is reduced to a fraction of a turn in 64 bits (position * turns
// minus its nearest integer), so a position of 10^6 is as exact as 0; F32
// angles would be off by 0.03 rad there.  The fraction's own rounding to F32 is
// kept and put back to first order: cos(a + r) = cos a - r sin a.
constexpr int kWriteThreads = 128;
constexpr int kWriteWarps = kWriteThreads / 32;
// Warps that a call should have (three rounds of a B200's 148 SMs at 24 warps): below it a token's
// heads are spread over several warps, each with the token's cosines to
// compute.  8192 tokens of 32 + 8 + 8 heads of 128 in F16: 40.5 us (4.6 TB/s) so,
// 48 at one round; the cosines in registers (80 of them a thread) 45, the loads
// of two steps ahead 44.
constexpr int kWarpsWanted = 148 * 24 * 3;
enum { kHalves, kNeighbours, kExchange };

// y0, y1 of a pair turned by r = (cos, sin).
__device__ __forceinline__ void turn(float& y0, float& y1, float2 r) {
  const float a = y0, b = y1;
  y0 = a * r.x - b * r.y;
  y1 = b * r.x + a * r.y;
}

template <typename T, int LANES, int FORM>  // LANES threads a head, 16 elements each
__global__ void __launch_bounds__(kWriteThreads, FORM == kExchange ? 4 : 6)
    kv8_write_kernel(const __grid_constant__ Kv8WriteArgs a, int slices) {
  constexpr int kHeads = 32 / LANES;
  __shared__ __align__(16) float2 turns_of[kWriteWarps][kKv8MaxDim / 2];
  __shared__ float other_of[FORM == kExchange ? kWriteWarps : 1][FORM == kExchange ? kHeads : 1]
                           [FORM == kExchange ? LANES * 16 + 1 : 1];
  griddep_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = lane / LANES, j = lane % LANES;
  const long long at_warp = static_cast<long long>(blockIdx.x) * kWriteWarps + warp;
  const int t = static_cast<int>(at_warp / slices), slice = static_cast<int>(at_warp % slices);
  if (t >= a.tokens) return;  // whole warps; nothing below spans warps
  const int d = a.cache.dim, hkv = a.cache.hkv, hq = a.hq;
  const int heads = hq + 2 * hkv, half = a.rotary >> 1;
  // Where the lane's two chunks of eight begin: lanes side by side read and
  // write 16 bytes side by side (a 32-byte stride doubled the load wavefronts).
  const bool used = j * 16 < d;
  const bool turns = j * 8 < half;  // in halves: whether the lane's chunks turn
  const int i0 = FORM == kExchange ? j * 16
                 : FORM == kNeighbours || turns ? j * 8
                                                : a.rotary + j * 8 - half;
  const int i1 = FORM == kExchange      ? i0 + 8
                 : FORM == kNeighbours ? (d >> 1) + j * 8
                 : turns                ? half + j * 8
                                        : i0 + ((d - a.rotary) >> 1);

  const int slot = __ldg(a.slots + t);
  const int pos = __ldg(a.positions + t);
  const T* row = static_cast<const T*>(a.qkv) + static_cast<size_t>(t) * heads * d;
  Eight<T> x0, x1;
  auto fetch = [&](int h) {
    const bool live = used && h < heads;
    const T* p = row + static_cast<size_t>(live ? h : 0) * d;
    x0.load(p + i0, live);
    x1.load(p + i1, live);
  };
  int h = slice * kHeads + unit;
  fetch(h);
  float2* cs = turns_of[warp];
  // Where pair i lies: a lane's pairs LANES apart, so that lanes read side by side.
  auto place = [&](int i) {
    if (FORM == kExchange) return i;
    if (FORM == kHalves) return (i & 7) * LANES + (i >> 3);
    const int q = d >> 2, hi = i >= q ? 1 : 0, k = i - hi * q;
    return (hi * 4 + (k & 3)) * LANES + (k >> 2);
  };
  for (int i = lane; i < half; i += 32) {
    const double all = static_cast<double>(pos) * a.turns[i];
    const double part = 2.0 * (all - rint(all));  // half turns, -1 .. 1
    const float f = static_cast<float>(part);
    const float r = static_cast<float>(part - f) * 3.14159265f;
    float s, c;
    sincospif(f, &s, &c);
    cs[place(i)] = make_float2((c - r * s) * a.factor, (s + r * c) * a.factor);
  }
  const bool stored = slot >= 0 && slot < a.cache.blocks * kKv8Page;
  if (slice == 0 && lane == 0 && slot >= 0 && !stored) atomicOr(a.status, kDevBadIndex);
  __syncwarp();
  auto r = [&](int e) { return cs[e * LANES + j]; };
  const size_t page = static_cast<size_t>(stored ? slot / kKv8Page : 0) * hkv;
  const int in_page = slot % kKv8Page;

  for (int base = slice * kHeads; base < heads; base += slices * kHeads, h += slices * kHeads) {
    const bool live = used && h < heads;
    const bool is_q = h < hq, is_v = h >= hq + hkv;
    const float* w = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
    float y[16];
    x0.values(y);
    x1.values(y + 8);
    fetch(h + slices * kHeads);
    // Shuffles take part in whole warps: a warp may hold heads of different kinds.
    if (a.q_norm != nullptr || a.k_norm != nullptr) {
      Eight<float> w0, w1;
      w0.load(w + i0, w != nullptr && live);
      w1.load(w + i1, w != nullptr && live);
      float2 squares = make_float2(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float2 v = make_float2(y[e], y[e + 1]);
        squares = fma2(v, v, squares);
      }
      float ss = squares.x + squares.y;
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (w != nullptr) {
        const float inv = 1.0f / sqrtf(ss / static_cast<float>(d) + a.eps);
        float m[16];
        w0.values(m);
        w1.values(m + 8);
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float2 v = mul2f(mul2f(make_float2(y[e], y[e + 1]), make_float2(inv, inv)),
                                 make_float2(m[e], m[e + 1]));
          y[e] = v.x;
          y[e + 1] = v.y;
        }
      }
    }
    if constexpr (FORM == kHalves) {
      if (turns && !is_v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) turn(y[e], y[8 + e], r(e));
      }
    } else if constexpr (FORM == kNeighbours) {
      if (!is_v) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (((e < 4 ? i0 : i1) >> 1) + (e & 3) < half) turn(y[2 * e], y[2 * e + 1], r(e));
      }
    } else {
      float* b = other_of[warp][unit];
      __syncwarp();
#pragma unroll
      for (int e = 0; e < 16; ++e) b[j * 16 + e] = y[e];
      __syncwarp();
      if (!is_v) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int i = j * 16 + e;
          if (i < a.rotary) {
            const bool lo = i < half;
            const float2 q = cs[lo ? i : i - half];
            const float other = b[lo ? i + half : i - half];
            y[e] = lo ? y[e] * q.x - other * q.y : y[e] * q.x + other * q.y;
          }
        }
      }
    }
    if (is_q && live) {
      __half* dst = a.q_out + (static_cast<size_t>(t) * hq + h) * d;
      *reinterpret_cast<uint4*>(dst + i0) = make_uint4(half2_bits(y[0], y[1]), half2_bits(y[2], y[3]),
                                                       half2_bits(y[4], y[5]), half2_bits(y[6], y[7]));
      *reinterpret_cast<uint4*>(dst + i1) =
          make_uint4(half2_bits(y[8], y[9]), half2_bits(y[10], y[11]), half2_bits(y[12], y[13]),
                     half2_bits(y[14], y[15]));
    }
    if (base + kHeads <= hq) continue;  // q only: the same for the whole warp
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e)
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(y[e])));
    if (!(top <= kKv8Limit)) {  // values that are not finite, or past the format
      top = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float m = fabsf(y[e]);
        if (m <= kKv8Limit) top = fmaxf(top, m);
        else y[e] = __uint_as_float(0x7fffffffu);
      }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!is_q && live && stored) {
      const int e = kv8_exponent(top);
      const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      const size_t at = (page + (is_v ? h - hq - hkv : h - hq)) * kKv8Page + in_page;
      uint8_t* dst = (is_v ? a.cache.v : a.cache.k) + at * d;
      uint32_t c[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 lo = mul2f(make_float2(y[4 * k], y[4 * k + 1]), make_float2(inv, inv));
        const float2 hi = mul2f(make_float2(y[4 * k + 2], y[4 * k + 3]), make_float2(inv, inv));
        c[k] = kv8_codes(lo.x, lo.y, hi.x, hi.y);
      }
      *reinterpret_cast<uint2*>(dst + i0) = make_uint2(c[0], c[1]);
      *reinterpret_cast<uint2*>(dst + i1) = make_uint2(c[2], c[3]);
      if (j == 0) (is_v ? a.cache.v_scale : a.cache.k_scale)[at] = static_cast<uint8_t>(e + 127);
    }
  }
}

template <typename T, int LANES, int FORM>
cudaError_t launch_write(const Kv8WriteArgs& a, cudaStream_t stream) {
  constexpr int kHeads = 32 / LANES;
  const long long steps = (a.hq + 2LL * a.cache.hkv + kHeads - 1) / kHeads;
  const int slices = static_cast<int>(
      std::min(steps, (kWarpsWanted + a.tokens - 1LL) / a.tokens));
  const long long warps = static_cast<long long>(a.tokens) * slices;
  return launch_dependent(kv8_write_kernel<T, LANES, FORM>,
                          dim3(static_cast<unsigned>((warps + kWriteWarps - 1) / kWriteWarps)),
                          dim3(kWriteThreads), 0, stream, a, slices);
}

template <typename T, int FORM>
cudaError_t size_write(const Kv8WriteArgs& a, cudaStream_t stream) {
  if (a.cache.dim <= 64) return launch_write<T, 4, FORM>(a, stream);
  if (a.cache.dim <= 128) return launch_write<T, 8, FORM>(a, stream);
  return launch_write<T, 16, FORM>(a, stream);
}

template <typename T>
cudaError_t dispatch_write(const Kv8WriteArgs& a, cudaStream_t stream) {
  if (a.interleaved) return size_write<T, kNeighbours>(a, stream);
  return a.rotary % 16 == 0 ? size_write<T, kHalves>(a, stream) : size_write<T, kExchange>(a, stream);
}

// ---------------------------------------------------------------- read
// value = code * 2^e, rounded once to the output type.  Memory-bound.  A CTA
// takes kReadTokens consecutive output rows: its threads find the rows' pages
// together, then a warp takes K or V of a token at a time, each lane as many
// codes as fill 16 bytes of output, kReadBatch loads in flight a lane.
constexpr int kReadThreads = 256;
constexpr int kReadTokens = 16;
constexpr int kReadBatch = 4;

template <typename T>
struct Sixteen {  // 16 bytes of output
  static constexpr int kCodes = 8;
  using Codes = uint2;
  __device__ __forceinline__ static uint32_t two(uint32_t h, float s) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
    if constexpr (std::is_same<T, __half>::value) {
      return half2_bits(v.x * s, v.y * s);
    } else {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v.x * s, v.y * s);
      return *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  __device__ __forceinline__ static uint4 of(uint2 w, float s) {
    return make_uint4(two(kv8_half2_lo(w.x), s), two(kv8_half2_hi(w.x), s),
                      two(kv8_half2_lo(w.y), s), two(kv8_half2_hi(w.y), s));
  }
};
template <>
struct Sixteen<float> {
  static constexpr int kCodes = 4;
  using Codes = uint32_t;
  __device__ __forceinline__ static uint4 of(uint32_t w, float s) {
    const uint32_t lo = kv8_half2_lo(w), hi = kv8_half2_hi(w);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return make_uint4(__float_as_uint(a.x * s), __float_as_uint(a.y * s), __float_as_uint(b.x * s),
                      __float_as_uint(b.y * s));
  }
};

template <typename T>
__global__ void __launch_bounds__(kReadThreads)
    kv8_read_kernel(const __grid_constant__ Kv8ReadArgs a, uint32_t inverse) {
  using Out = Sixteen<T>;
  using Codes = typename Out::Codes;
  __shared__ long long source[kReadTokens];  // row of (kv head 0) in the pool, -1: none, -2: no output
  __shared__ int ends[kReadTokens];          // rows that end at a token of the CTA (the first: or before it)
  griddep_enter();
  const int t0 = blockIdx.x * kReadTokens;
  const int hkv = a.cache.hkv, d = a.cache.dim;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < kReadTokens) ends[threadIdx.x] = 0;
  __syncthreads();
  for (int base = warp * 32; base < a.rows; base += kReadThreads) {
    int k = kReadTokens;
    if (base + lane < a.rows) {
      const int end = __ldg(a.offsets + base + lane + 1);
      k = max(end, t0) - t0;
      if (blockIdx.x == 0) {  // one CTA reports rows that end past the output, or before they begin
        const int begin = __ldg(a.offsets + base + lane);
        if (begin < 0 || end < begin || end > a.tokens) atomicOr(a.status, kDevBadIndex);
      }
    }
    const unsigned before = __ballot_sync(0xffffffffu, k == 0);
    if (lane == 0 && before) atomicAdd(&ends[0], __popc(before));
    if (k > 0 && k < kReadTokens) atomicAdd(&ends[k], 1);
  }
  __syncthreads();
  if (threadIdx.x < kReadTokens) {
    const int t = t0 + lane;
    int r = 0;  // row of the token: the number of rows that end at or before it
    for (int k = 0; k <= lane; ++k) r += ends[k];
    long long src = -2;
    if (r < a.rows && t < a.tokens && t >= a.offsets[0]) {
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
  __syncthreads();
  const uint32_t chunks = static_cast<uint32_t>(d) / Out::kCodes;
  const uint32_t per = static_cast<uint32_t>(hkv) * chunks;
  for (int item = warp; item < 2 * kReadTokens; item += kReadThreads / 32) {
    const int tl = item >> 1, which = item & 1;
    const long long src = source[tl];
    if (src == -2) continue;
    const uint8_t* codes = which ? a.cache.v : a.cache.k;
    const uint8_t* scales = which ? a.cache.v_scale : a.cache.k_scale;
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(which ? a.v_out : a.k_out) +
                                          static_cast<size_t>(t0 + tl) * hkv * d);
    for (uint32_t u0 = lane; u0 < per; u0 += 32 * kReadBatch) {
      Codes w[kReadBatch];
      uint32_t s[kReadBatch];
#pragma unroll
      for (int k = 0; k < kReadBatch; ++k) {
        const uint32_t u = u0 + 32 * k;
        w[k] = Codes{};
        s[k] = 127u;
        if (src >= 0 && u < per) {
          const uint32_t kvh = __umulhi(u, inverse);  // u / chunks
          const size_t at = static_cast<size_t>(src) + static_cast<size_t>(kvh) * kKv8Page;
          w[k] = __ldg(reinterpret_cast<const Codes*>(codes + at * d) + (u - kvh * chunks));
          s[k] = __ldg(scales + at);
        }
      }
#pragma unroll
      for (int k = 0; k < kReadBatch; ++k)
        if (u0 + 32 * k < per) dst[u0 + 32 * k] = Out::of(w[k], kv8_scale(s[k]));
    }
  }
}

template <typename T>
cudaError_t launch_read(const Kv8ReadArgs& a, cudaStream_t stream) {
  const dim3 grid((a.tokens + kReadTokens - 1) / kReadTokens);
  // ceil(2^32 / chunks): u * inverse >> 32 is u / chunks for u * chunks < 2^32.
  const uint32_t chunks = static_cast<uint32_t>(a.cache.dim) / Sixteen<T>::kCodes;
  const uint32_t inverse = static_cast<uint32_t>((0x100000000ull + chunks - 1) / chunks);
  return launch_dependent(kv8_read_kernel<T>, grid, dim3(kReadThreads), 0, stream, a, inverse);
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
  switch (a.type) {
    case kKv8F32: return launch_read<float>(a, stream);
    case kKv8F16: return launch_read<__half>(a, stream);
    default: return launch_read<__nv_bfloat16>(a, stream);
  }
}

}  // namespace hb
