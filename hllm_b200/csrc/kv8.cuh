// kv8.cuh -- the 8-bit paged KV cache: host launchers of its write, its
// read-back and its attention, and the number format they share.
//
// Format.  A (token, kv head) row of K or of V is d e4m3 codes and one scale
// 2^e, e the least integer in [-24, 39] with max |x| <= 448 * 2^e, kept as the
// byte e + 127.  Powers of two lose nothing that e4m3 has: a code's relative
// rounding error is 2^-4 at most whatever the scale's mantissa, and code * 2^e
// is exact in F32 (and in F16 where F16 has the range), so the attention can
// put the scales into its scores' and weights' exponents without a rounding.
// The clamp at -24 only coarsens rows below 448 * 2^-24 = 2.7e-5, whose steps
// are then 2^-33, finer than the F16 cache's 2^-24; the clamp at 39 lets every
// sum of 2^63 ratios stay in F32.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "common.cuh"

namespace hb {

constexpr int kKv8Page = 16;     // tokens of a page, as in the F16 pool
constexpr int kKv8MaxDim = 256;  // head sizes: multiples of 32 up to this
constexpr int kKv8ExpMin = -24, kKv8ExpMax = 39;
constexpr float kKv8Limit = 448.0f * 549755813888.0f;  // 448 * 2^39: larger values are stored as NaN

// Codes [blocks][Hkv][16][d], scale bytes [blocks][Hkv][16].
struct Kv8Cache {
  uint8_t *k, *k_scale, *v, *v_scale;
  long long blocks;
  int hkv, dim;
};

// Element types of the write's input and the read's output (hllm_b200_dtype).
enum Kv8Type : int { kKv8F32 = 0, kKv8F16 = 1, kKv8BF16 = 2 };

struct Kv8WriteArgs {
  Kv8Cache cache;
  const void* qkv;           // [T][(Hq + 2 Hkv) d]
  int type;                  // Kv8Type
  int tokens, hq;
  const int32_t* positions;  // [T]
  const int32_t* slots;      // [T], -1: the token is not stored
  const float *q_norm, *k_norm;  // [d] or null
  float eps;
  const double* turns;       // [rotary / 2] turns per position
  int rotary, interleaved;
  float factor;              // on cos and sin
  __half* q_out;             // [T][Hq d]
  uint32_t* status;
};
cudaError_t kv8_write_launch(const Kv8WriteArgs& a, cudaStream_t stream);

struct Kv8ReadArgs {
  Kv8Cache cache;
  const int32_t* tables;   // [rows][max_blocks]
  const int32_t* first;    // [rows] or null: 0
  const int32_t* lengths;  // [rows] end positions
  const int32_t* offsets;  // [rows + 1] output rows
  int rows, max_blocks, tokens, type;
  void *k_out, *v_out;     // [tokens][Hkv][d]
  uint32_t* status;
};
cudaError_t kv8_read_launch(const Kv8ReadArgs& a, cudaStream_t stream);

struct Kv8AttnArgs {
  Kv8Cache cache;
  const __half* q;            // [T][ld_q]
  long long ld_q;
  const int32_t* cu_seqlens;  // [rows + 1]
  const int32_t* lengths;     // [rows] keys of a row, its new tokens included
  const int32_t* tables;      // [rows][max_blocks]
  int rows, tokens, max_row_tokens, hq, max_blocks;
  float scale;
  __half* out;                // [T][ld_out]
  long long ld_out;
  float* workspace;
  uint32_t* status;
  int sm_count;
};
// Whether the tile pass (kv8_tile.cu: prompt chunks on tcgen05) takes a head
// size, its share of the workspace, and its launches: tiles, then, once the
// stream pass is launched, the join of their key splits.
bool kv8_tile_supported(int dim);
size_t kv8_tile_workspace(int dim, int sm_count);
cudaError_t kv8_tile_launch(const Kv8AttnArgs& a, int tile_from, float* partial, cudaStream_t stream);
cudaError_t kv8_tile_join_launch(const Kv8AttnArgs& a, int tile_from, const float* partial,
                                 cudaStream_t stream);

size_t kv8_attention_workspace(int max_row_tokens, int hq, int hkv, int dim, int sm_count);
cudaError_t kv8_attention_launch(const Kv8AttnArgs& a, cudaStream_t stream);

#ifdef __CUDACC__
// A kernel's dynamic shared memory limit, raised once a device.
struct Kv8Configured {
  std::atomic<bool> done[64] = {};
  template <typename K>
  cudaError_t once(K kernel, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done[dev].store(true, std::memory_order_relaxed);
    return e;
  }
};

// ---------------------------------------------------------------- device side
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoReference = -1e30f;  // below every finite score
// A softmax reference moves when a weight (with its value row's scale) would pass
// 2^kMost, and then so that the largest is 2^kTop: F16 keeps weights down to
// 2^-24, so 2^-31 of the largest at least, and a long tail of small ones counts.
// (With the largest at 1 a flat tail 2^-25 below one key went missing from the
// sums, 2^-8 of the output at 131071 keys.)  2^kMost leaves F16 a factor of 4 for
// what large scores round.
constexpr float kTop = 7.f, kMost = 14.f;
constexpr float kMostWeight = 16384.f;  // 2^kMost

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two F32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)),
        "l"(reinterpret_cast<const unsigned long long&>(b)),
        "l"(reinterpret_cast<const unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2f(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)),
        "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2f(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)),
        "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}
// The scale exponent of a row whose largest magnitude is `top` (finite, at
// most kKv8Limit): the least e in [-24, 39] with top <= 448 * 2^e.  With
// top = 1.f * 2^k, 448 = 1.75 * 2^8: e = k - 8, one more where 1.f > 1.75.
__device__ __forceinline__ int kv8_exponent(float top) {
  const uint32_t b = __float_as_uint(top);
  const int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kKv8ExpMin), kKv8ExpMax);
}
// The value of a scale byte.
__device__ __forceinline__ float kv8_scale(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}
// Two codes as F16: the low or the high half of a word of four.
__device__ __forceinline__ uint32_t kv8_half2_lo(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
      : "=r"(h)
      : "r"(w));
  return h;
}
__device__ __forceinline__ uint32_t kv8_half2_hi(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}"
      : "=r"(h)
      : "r"(w));
  return h;
}
// 0xff in the bytes of four codes that are NaN.
__device__ __forceinline__ uint32_t kv8_nan_codes(uint32_t w) {
  return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 255u;
}
// Four values as codes (the first in the low byte), ties to even.
__device__ __forceinline__ uint32_t kv8_codes(float a, float b, float c, float d) {
  uint32_t w;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
      : "=r"(w)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return w;
}

// A row's place in the packed batch and its streams: groups of `cols` columns,
// a column being one query head of the kv head's group at one new token.
struct Kv8Row {
  int count, len, t0;  // new tokens, keys, first packed token
  int pages;           // at least 1, so that a row without keys is answered too
  int chunks;          // column groups per kv head
};

__device__ __forceinline__ int kv8_pages(int len) { return len > 0 ? (len - 1) / kKv8Page + 1 : 1; }

// Row r as the stream pass (tiles false: rows under tile_from columns) or the
// tile pass (the others) sees it: rows of the other pass, and rows out of the
// batch's bounds (reported), have count 0.
__device__ __forceinline__ Kv8Row kv8_row(const Kv8AttnArgs& a, int r, int group, int cols,
                                          int tile_from, bool report, bool tiles = false) {
  Kv8Row x;
  x.t0 = __ldg(a.cu_seqlens + r);
  const int end = __ldg(a.cu_seqlens + r + 1);
  x.len = __ldg(a.lengths + r);
  const long long count = static_cast<long long>(end) - x.t0;
  const bool bad = x.t0 < 0 || count < 0 || end > a.tokens || count > a.max_row_tokens ||
                   x.len < 0 || x.len > a.max_blocks * static_cast<long long>(kKv8Page);
  if (bad && report) atomicOr(a.status, kDevBadIndex);
  x.count = bad || (count * group >= tile_from) != tiles ? 0 : static_cast<int>(count);
  if (bad) x.len = 0;
  x.pages = kv8_pages(x.len);
  x.chunks = static_cast<int>((static_cast<long long>(x.count) * group + cols - 1) / cols);
  return x;
}
#endif

}  // namespace hb
