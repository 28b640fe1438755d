// kv8_tile.cu -- prompt chunks over the 8-bit paged KV cache on the
// 5th-generation tensor cores (head sizes 64 and 128).
//
// The rows of a tile are 128 columns (token, query head of the kv head's
// group) of one batch row; S = Q K^T and O += P V run as tcgen05 products of
// F16 operands into TMEM, 128 keys at a time.  Tensor-bound: 4 x 128 x 128 x D
// operations a tile, next to which the codes are few bytes, so the work is to
// keep the tensor pipe fed while codes become F16 and scores become weights:
//
//   warps 8-11  converters of K, warps 12-15 of V: a tile's codes from their
//               pages into shared memory as swizzled F16 operands, the next
//               tile's loads going out as the registers become free.  K rows
//               are code * 2^(e - E) with E the tile's largest exponent, which
//               goes into the score scale of the tile, and V rows likewise, where
//               the tile's exponents lie within 2^15 and 2^8 of their largest:
//               nothing is rounded then (a code's lowest bit is 2^-9, F16's 2^-24).
//               Else both are the codes, and each key's scales go into its score
//               and its weights: no key, seen or hidden, coarsens another.
//   warp 16     one thread issues the products.
//   warps 0-7   two softmax groups of 128 threads, one row (TMEM lane) a
//               thread.  The weights go back into TMEM over the scores they
//               came from, as F16, and are the A operand of P V from there.
//
// The two groups keep the tensor pipe busy for one another: while one group's
// scores become weights, the other's products run.  With many tiles (SHARED) a
// CTA holds two tiles of queries and both groups use each key tile that the
// converters make.  With few, both groups work on one tile of queries and take
// the key tiles in turn, the two halves being joined at the end; and the keys
// of a tile are split over CTAs, joined by a second launch.
//
// With s_j the score in log2 and ev_j the exponent of value row j, a row keeps
// one reference m for  l = sum 2^(s_j - m)  and  O = sum (2^(s_j - m) 2^ev_j) d_j,
// d_j the codes: the weights in brackets are what F16 has to hold, so m follows
// max (s_j + ev_j), lazily, and o = O / l.  (2^(s_j - m + E') 2^(ev_j - E') d_j
// where E' is taken out: the weights are then the exponentials themselves.)
// Every wait is bounded (common.cuh).
//
// Measured, 32 heads on 8 of 128: 2048 tokens behind 8192 keys 369 us (838
// TFLOP/s of the causal products, 50 % of what cuBLAS reaches), 512 behind 1024
// 29.7 us (362).  A step with two query tiles is 4.7k cycles, of which the products
// are 2.8k: the rest is a group's chain, scores, maximum and exponentials (3.0k),
// products, next scores, for which TMEM has no second buffer beside two results of
// 128 dimensions.  With one query tile a step is 2.5k, and the codes' conversion
// (2.7k a tile, K and V side by side) is as long.  Unrolling the passes over the
// scores, or keeping 64 of them in registers, was slower by a third.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kv8.cuh"

namespace hb {
namespace {

constexpr int kKeys = 128;       // keys of a tile
constexpr int kRows = 128;       // columns of a query tile
constexpr int kSoftmax = 256;    // threads of the softmax groups
constexpr int kThreads = kSoftmax + 256 + 32;
constexpr int kSpread = 8;        // V exponents this near their tile's largest are taken out of the weights,
constexpr int kSpreadK = 15;      // and K exponents this near out of the scores, exactly
constexpr int kApart = 1000;      // others

// The products' instructions, by the lane for which `on` holds, in code that a
// whole warp runs: its addresses then stay in uniform registers (one thread's
// branch took 85 cycles an instruction, more than the product).  Descriptors
// are two words, of which only the low one moves.
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(on));
  return on != 0u;
}
// D[tmem] (+)= A[smem] * B[smem]:
__device__ __forceinline__ void mma_ss(bool on, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 a, {%2, %4};\n\tmov.b64 b, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %5, p;\n\t}\n" ::"r"(static_cast<uint32_t>(on)),
      "r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], A being F16 pairs, a row per lane:
__device__ __forceinline__ void mma_ts(bool on, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t hi,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], b, %5, p;\n\t}\n" ::"r"(static_cast<uint32_t>(on)),
      "r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// `bar` is arrived at once the lane's products so far are done.
__device__ __forceinline__ void mma_commit(bool on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}\n" ::"r"(
          static_cast<uint32_t>(on)),
      "r"(smem_u32(bar))
      : "memory");
}

// 2^y of two numbers on the FMA pipes, beside the exponentials of the special
// function unit, which bounds a softmax: y = n + r with n the nearest integer
// (found in the low bits of y + 1.5 2^23), 2^r by a polynomial of degree 5 fitted
// to a small largest relative error on [-1/2, 1/2] (Remez, then rounded: 1.6e-7 with
// these coefficients, 2.2e-7 in F32 arithmetic), times 2^n.
// Numbers below -120 count as that; NaN stays NaN.
__device__ __forceinline__ float2 exp2_fma(float2 y) {
  float2 t;
  asm("max.NaN.f32 %0, %1, 0fC2F00000;" : "=f"(y.x) : "f"(y.x));
  asm("max.NaN.f32 %0, %1, 0fC2F00000;" : "=f"(y.y) : "f"(y.y));
  t = add2f(y, make_float2(12582912.f, 12582912.f));
  const float2 n = add2f(t, make_float2(-12582912.f, -12582912.f));
  const float2 r = fma2(n, make_float2(-1.f, -1.f), y);
  auto both = [](float c) { return make_float2(c, c); };
  float2 p = both(0.0013276472454890609f);
  p = fma2(p, r, both(0.009675540961325169f));
  p = fma2(p, r, both(0.05550713092088699f));
  p = fma2(p, r, both(0.24022120237350464f));
  p = fma2(p, r, both(0.6931469440460205f));
  p = fma2(p, r, both(1.0000001192092896f));
  return mul2f(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                              __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}

// Consecutive columns of a thread's lane: 16 read without the wait, 8 written.
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32"
      " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <int D, bool SHARED>
struct Tile {
  static constexpr int kQueries = SHARED ? 2 : 1;           // query tiles of a CTA
  static constexpr uint32_t kAtom = 128 * 128;              // 128 rows x 64 F16: one swizzle column
  static constexpr uint32_t kOperand = 128 * D * 2;         // Q, K or V of 128 rows
  static constexpr uint32_t kQ = 0, kK = kQueries * kOperand, kV = kK + 2 * kOperand;
  static constexpr uint32_t kEnd = kV + 2 * kOperand;
  static constexpr uint32_t kSmem = kEnd + 1024;            // 1024-byte alignment slack
  static constexpr uint32_t kTmemS = 0, kTmemO = 256;       // per group: + 128 g
  // A partial result: D / 4 x 128 rows x 4 sums, then 128 x (m, l).
  static constexpr int kPiece = 128 * (D + 2);              // floats
};

// Loads that leave zeros where !live, without a branch, so that a run of them
// is in flight together.
__device__ __forceinline__ uint4 load16_if(const void* p, bool live) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"(static_cast<uint32_t>(live)));
  return v;
}
__device__ __forceinline__ uint32_t load_byte_if(const uint8_t* p, bool live) {
  uint32_t v;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t"
      "@p ld.global.nc.u8 %0, [%1];\n\t}"
      : "=&r"(v)
      : "l"(p), "r"(static_cast<uint32_t>(live)));
  return v;
}

// 2^(k - 127), at most 1, in both halves of a word (0 where F16 has no such value).
__device__ __forceinline__ uint32_t half_power2(int k) {
  const float f = __uint_as_float(static_cast<uint32_t>(max(k, 0)) << 23);
  return half2_bits(f, f);
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// How the 128 threads of a converter group share a tile: 16 codes of a key a
// thread, kRows keys a pass.  Of eight lanes in a row four hold one key's codes
// and four its neighbour's: their 16-byte chunks of F16, every second one of a
// key, then reach eight different groups of banks under the swizzle.
template <int D>
struct Share {
  static constexpr int kLanes = D / 16;             // threads of a key
  static constexpr int kRows = 128 / kLanes;        // keys of a pass
  static constexpr int kPasses = kKeys / kRows;
  int chunk, row;                                   // codes 16 chunk ..., key row of a pass
  __device__ explicit Share(int tid) {
    const int lane = tid & 31, warp = tid >> 5;
    if (D == 128) {
      chunk = (lane & 3) | (lane >> 1 & 4);
      row = warp * 4 + (lane >> 4) * 2 + (lane >> 2 & 1);
    } else {
      chunk = lane & 3;
      row = warp * 8 + (lane >> 2);
    }
  }
};
// The codes of pass p from `page` (pool page of this kv head, -1: none); zeros
// from key `left` on.
template <int D>
__device__ __forceinline__ uint4 load_codes(const Share<D>& h, const uint8_t* pool, int page, int p,
                                            int left) {
  const uint8_t* at = pool + static_cast<uint64_t>(static_cast<uint32_t>(page)) * (kKv8Page * D);
  return load16_if(at, page >= 0 && p * Share<D>::kRows + h.row < left);
}
// Times 2^k (a factor for both halves of a word) as two swizzled chunks of F16.
template <int D>
__device__ __forceinline__ void store_codes(uint8_t* dst, const Share<D>& h, int p, const uint4& c,
                                            uint32_t factor) {
  const int r = p * Share<D>::kRows + h.row;
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c16 = h.chunk * 2 + k;
    *reinterpret_cast<uint4*>(dst + (c16 >> 3) * (128 * 128) + r * 128 + (((c16 & 7) ^ (r & 7)) << 4)) =
        make_uint4(mul2(kv8_half2_lo(w[2 * k]), factor), mul2(kv8_half2_hi(w[2 * k]), factor),
                   mul2(kv8_half2_lo(w[2 * k + 1]), factor), mul2(kv8_half2_hi(w[2 * k + 1]), factor));
  }
}

// The codes of V at a key of a row, null where its page is missing.
__device__ __forceinline__ const uint8_t* value_row(const Kv8AttnArgs& a, int row, int kvh, int key, int dim) {
  const int id = __ldg(a.tables + static_cast<size_t>(row) * a.max_blocks + key / kKv8Page);
  if (id < 0 || id >= a.cache.blocks) return nullptr;
  return a.cache.v + ((static_cast<size_t>(id) * a.cache.hkv + kvh) * kKv8Page + key % kKv8Page) * dim;
}
// A weight of 0 would not hide a NaN code of V from the columns that do not see
// its key.  So what this thread stored of such codes, in keys from `first` on,
// becomes zeros, and the columns that see them get their NaN with the result.
// (Neither is inlined: hardly a call needs them, and the passes have no registers
// to spare.)
template <int D>
__device__ __noinline__ void hide_nan(uint8_t* dst, Share<D> h, int first) {
  for (int r = h.row; r < kKeys; r += Share<D>::kRows) {
    if (r < first) continue;
    for (int c = h.chunk * 16; c < h.chunk * 16 + 16; ++c) {
      uint16_t* const at = reinterpret_cast<uint16_t*>(
          dst + (c >> 6) * (128 * 128) + r * 128 + (((c >> 3 & 7) ^ (r & 7)) << 4) + (c & 7) * 2);
      if ((*at & 0x7fffu) > 0x7c00u) *at = 0;
    }
  }
}
// `to` is the column's result: F16, or a partial result's sums.
template <int D>
__device__ __noinline__ void put_nan(const Kv8AttnArgs& a, int row, int kvh, int key0, int key1, int c0, int c1,
                                     __half* to, float* piece) {
  for (int key = key0; key < key1; ++key) {
    const uint8_t* codes = value_row(a, row, kvh, key, D);
    for (int c = c0; codes && c < c1; ++c) {
      if ((__ldg(codes + c) & 0x7f) != 0x7f) continue;
      if (piece) piece[c / 4 * (128 * 4) + c % 4] = __uint_as_float(0x7fffffffu);
      else to[c] = __ushort_as_half(0x7fff);
    }
  }
}

// Keys that the last of `columns` columns from x0 on sees.
__device__ __forceinline__ int seen_keys(const Kv8Row& x, int group, int x0, int columns) {
  const int last_token = (min(x0 + columns, x.count * group) - 1) / group;
  return max(0, x.len - x.count + last_token + 1);
}
// The splits that `tiles` key tiles are worth, of those that were launched: a
// piece costs about two tiles to begin and to join.
constexpr int kLeastTiles = 4;
__device__ __forceinline__ int parts_of(int tiles, int splits) {
  return max(1, min(splits, tiles / kLeastTiles));
}

// Tiles of a group of 32 rows up to each lane's, whose own they are.
__device__ __forceinline__ int tiles_upto(int own, int lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, own, off);
    if (lane >= off) own += v;
  }
  return own;
}
// Whether a row's tiles, numbered in the rows' order, are among the `most` that
// were launched and that the workspace has pieces for.  They are unless
// cu_seqlens decreases, so that rows overlap: the rows past that number are
// skipped, in the tile pass and in the join alike.
__device__ __forceinline__ bool fits(int before, int upto, int most) { return before + upto <= most; }

template <int D, bool SHARED>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_tile_kernel(const __grid_constant__ Kv8AttnArgs a, int group, int tile_from, float* partial) {
  using T = Tile<D, SHARED>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_full[2],
      o_done[2], looked;
  __shared__ uint32_t tmem_slot;
  __shared__ float2 group_ml[2][kRows];  // m and l of the groups, where they share a tile
  __shared__ int found[3];             // row, tile of the row, tile of all rows
  // By key tile: E + 127 of its K; E' of its V, or kApart; and then each key's
  // 2^ev (0 where there is no key), ev (-inf) and 2^ek (0).
  __shared__ volatile int exps[4][2];
  __shared__ __align__(16) float value_scale[4][3 * kKeys];
  __shared__ int extremes[2][2][4][4];          // by group, tile and warp: E, E', least ev and ek, all + 127
  __shared__ uint8_t scale_byte[2][2][kKeys];   // by group and tile
  __shared__ volatile int nan_hidden;  // whether V has NaN codes in keys that some columns do not see
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kCta = T::kQueries * kRows;  // columns of a CTA

  griddep_enter();
  if (threadIdx.x == 0) {
    nan_hidden = 0;
    mbar_init(&q_full, kSoftmax);
    mbar_init(&looked, kSoftmax);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 128);
      mbar_init(&v_full[s], 128);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 128);
      mbar_init(&o_done[s], 1);
    }
    fence_mbar_init();
  }
  if (warp == 16) {
    // The row of this CTA's tile: of 32 rows the one with the most keys first,
    // and of a row the late tiles; all kv heads of a tile together; and the CTAs
    // that the grid has too many last.
    const bool reports = blockIdx.x + blockIdx.z == 0;
    const int most = static_cast<int>(gridDim.x) / a.cache.hkv;  // tiles that the grid has
    int w = static_cast<int>(blockIdx.x) / a.cache.hkv;  // tiles before it
    int row = -1, tile = 0, cell = 0, tiles_before = 0;  // cell: its number in the rows' order
    for (int base = 0; base < a.rows && (row < 0 || reports); base += 32) {
      int own = 0, len = -1;
      if (base + lane < a.rows) {
        const Kv8Row x = kv8_row(a, base + lane, group, kCta, tile_from, reports, true);
        own = x.chunks;
        len = x.len;
      }
      const int all = __reduce_add_sync(0xffffffffu, own);
      if (!fits(tiles_before, all, most)) {
        const int upto = tiles_upto(own, lane);  // (of the whole warp)
        const bool skipped = own > 0 && !fits(tiles_before, upto, most);
        if (skipped && reports) atomicOr(a.status, kDevBadIndex);
        if (skipped) own = 0;
      }
      int first = 0, lower = 0;  // tiles of rows that go before this one, and that stand before it
      for (int j = 0; j < min(32, a.rows - base); ++j) {
        const int chunks = __shfl_sync(0xffffffffu, own, j), keys = __shfl_sync(0xffffffffu, len, j);
        if (keys > len || (keys == len && j < lane)) first += chunks;
        if (j < lane) lower += chunks;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, row < 0 && w >= first && w < first + own);
      if (hit) {
        const int src = __ffs(hit) - 1;
        row = base + src;
        tile = __shfl_sync(0xffffffffu, own - 1 - (w - first), src);
        cell = tiles_before + __shfl_sync(0xffffffffu, lower, src) + tile;
      }
      w -= __reduce_add_sync(0xffffffffu, own);
      tiles_before = min(tiles_before + all, most);
    }
    if (lane == 0) {
      found[0] = row;
      found[1] = tile;
      found[2] = cell;
    }
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int row = found[0];
  if (row < 0) {  // the whole CTA: fewer tiles than the grid has room for
    if (warp == 0) tmem_dealloc(tmem, 512);
    return;
  }

  const Kv8Row x = kv8_row(a, row, group, kCta, tile_from, false, true);
  const int hkv = a.cache.hkv, kvh = blockIdx.x % hkv;
  const int x0 = found[1] * kCta, cols = x.count * group;
  const int past = x.len - x.count;  // position of the row's first new token
  // Keys that the CTA's last column sees, and this split's share of their tiles.
  const int keys = seen_keys(x, group, x0, kCta);
  const int all = (keys + kKeys - 1) / kKeys;
  const int parts = parts_of(all, gridDim.z), part = blockIdx.z;
  if (part >= parts) {  // too few keys for this many splits
    if (warp == 0) tmem_dealloc(tmem, 512);
    return;
  }
  const int kt0 = static_cast<int>(static_cast<long long>(all) * part / parts);
  const int n = static_cast<int>(static_cast<long long>(all) * (part + 1) / parts) - kt0;

  // The keys of this split that some columns of the CTA do not see.
  const int hidden0 = max(kt0 * kKeys, past + x0 / group + 1), hidden1 = min(keys, (kt0 + n) * kKeys);

  if (warp == 16) {
    // ---------------------------------------------------------------- products
    constexpr uint32_t idesc_s = umma_idesc(kRows, kKeys, 0);
    constexpr uint32_t idesc_pv = umma_idesc(kRows, D, 0) | (1u << 16);  // V: MN-major
    const bool on = elect_one();
    const uint32_t base = smem_u32(smem);
    const uint64_t desc_k = sw128_desc(base), desc_v = sw128_desc_mn(base, T::kAtom);
    const uint32_t k_lo = static_cast<uint32_t>(desc_k), k_hi = static_cast<uint32_t>(desc_k >> 32);
    const uint32_t v_lo = static_cast<uint32_t>(desc_v), v_hi = static_cast<uint32_t>(desc_v >> 32);
    // (Through shuffles, so that what follows is uniform to the compiler.)
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const int tiles = __shfl_sync(0xffffffffu, n, 0);
    // A descriptor's address field counts 16 bytes: offsets are added to it.
    auto scores = [&](int t, int g) {  // S of group g on key tile t
      const uint32_t qd = k_lo + ((T::kQ + (SHARED ? g * T::kOperand : 0u)) >> 4);
      const uint32_t kd = k_lo + ((T::kK + (t & 1) * T::kOperand) >> 4);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = ((kk >> 2) * T::kAtom + (kk & 3) * 32) >> 4;
        mma_ss(on, tm + T::kTmemS + g * 128, qd + off, kd + off, k_hi, idesc_s, kk > 0 ? 1u : 0u);
      }
      mma_commit(on, &s_full[g]);
    };
    auto sums = [&](int t, int g, bool fresh) {  // O of group g (+)= P V
      const uint32_t vd = v_lo + ((T::kV + (t & 1) * T::kOperand) >> 4);
#pragma unroll
      for (int ks = 0; ks < kKeys / 16; ++ks)
        mma_ts(on, tm + T::kTmemO + g * 128, tm + T::kTmemS + g * 128 + ks * 8, vd + ks * (2048 >> 4), v_hi,
               idesc_pv, !fresh || ks > 0 ? 1u : 0u);
      mma_commit(on, &o_done[g]);
    };
    auto wait = [&](uint64_t* bar, int use) {
      const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, use & 1, a.status));
      tc_fence_after();
      return ok;
    };
    bool ok = tiles > 0 && wait(&q_full, 0);
    if (SHARED) {
      ok = ok && wait(&k_full[0], 0);
      if (ok) {
        scores(0, 0);
        // Half a period behind: one group's weights then run under the
        // other's products, and neither waits for the exponentials of both.
        ok = wait(&p_full[0], 0);
        if (ok) scores(0, 1);
        mma_commit(on, &k_empty[0]);
      }
#pragma unroll 1
      for (int t = 0; ok && t < tiles; ++t) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          ok = ok && wait(&p_full[g], t);
          if (g == 0) ok = ok && wait(&v_full[t & 1], t >> 1);
          if (!ok) break;
          sums(t, g, t == 0);
          if (g == 1) mma_commit(on, &v_empty[t & 1]);
          if (t + 1 < tiles) {
            if (g == 0) ok = wait(&k_full[(t + 1) & 1], (t + 1) >> 1);
            if (!ok) break;
            scores(t + 1, g);
            if (g == 1) mma_commit(on, &k_empty[(t + 1) & 1]);
          }
        }
      }
    } else {
#pragma unroll 1
      for (int t = 0; ok && t < 2 && t < tiles; ++t) {
        ok = wait(&k_full[t], 0);
        if (!ok) break;
        scores(t, t);
        mma_commit(on, &k_empty[t]);
      }
#pragma unroll 1
      for (int t = 0; ok && t < tiles; ++t) {
        const int g = t & 1;
        ok = wait(&p_full[g], t >> 1) && wait(&v_full[g], t >> 1);
        if (!ok) break;
        sums(t, g, t < 2);
        mma_commit(on, &v_empty[g]);
        if (t + 2 < tiles) {
          ok = wait(&k_full[g], (t + 2) >> 1);
          if (!ok) break;
          scores(t + 2, g);
          mma_commit(on, &k_empty[g]);
        }
      }
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- converters
    const bool values = warp >= 12;
    const int tid = (threadIdx.x - kSoftmax) & 127, cw = warp & 3;
    const Share<D> share(tid);
    constexpr int kPasses = Share<D>::kPasses;
    const int32_t* table = a.tables + static_cast<size_t>(row) * a.max_blocks;
    // The tile's pages of this kv head, in the first eight lanes (-1: none).
    auto load_ids = [&](int t) {
      const int key = (kt0 + t) * kKeys + lane * kKv8Page;
      // Below max_blocks: keys is at most the row's length.
      return t < n && lane < 8 && key < keys ? __ldg(table + key / kKv8Page) : -1;
    };
    auto pages_of = [&](int id) { return id >= 0 && id < a.cache.blocks ? id * hkv + kvh : -1; };
    const uint8_t* pool = (values ? a.cache.v : a.cache.k) + (share.row % kKv8Page) * D + share.chunk * 16;
    uint4 c[kPasses];
    int pages = pages_of(load_ids(0));
    auto page_of = [&](int p) {
      return __shfl_sync(0xffffffffu, pages, (p * Share<D>::kRows + share.row) / kKv8Page);
    };
    int ids = load_ids(1);  // a tile ahead, so that no load waits for another
    uint32_t ks = 0u, vs = 0u;        // scale bytes of key `tid` of the tile
    bool have = false, hole = false;  // whether that key is there, or should be
    auto load_scales = [&](int t) {
      const int page = __shfl_sync(0xffffffffu, pages, tid / kKv8Page);
      const bool key = (kt0 + t) * kKeys + tid < keys;
      have = page >= 0 && key;
      hole = page < 0 && key;
      const size_t at = static_cast<size_t>(max(page, 0)) * kKv8Page + tid % kKv8Page;
      ks = load_byte_if(a.cache.k_scale + at, have);
      vs = load_byte_if(a.cache.v_scale + at, have);
    };
    if (n > 0) {
      load_scales(0);
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
        c[p] = load_codes<D>(share, pool, page_of(p), p, keys - kt0 * kKeys);
    }
    const int group_of = values ? 1 : 0;
    uint64_t* const full = values ? v_full : k_full;
    uint64_t* const empty = values ? v_empty : k_empty;
    uint8_t* const operand = smem + (values ? T::kV : T::kK);
    bool ok = true;
#pragma unroll 1
    for (int t = 0; t < n; ++t) {
      // The tile's exponents; bytes are e + 127, and 0 is no key's.
      if (hole && !values) atomicOr(a.status, kDevBadIndex);
      const int mine = static_cast<int>(values ? vs : ks);
      scale_byte[group_of][t & 1][tid] = static_cast<uint8_t>(mine);
      const int ek = __reduce_max_sync(0xffffffffu, have ? static_cast<int>(ks) : 0);
      const int ev = __reduce_max_sync(0xffffffffu, have ? static_cast<int>(vs) : 0);
      // A missing page takes the path that looks at each key.
      const int least = __reduce_min_sync(0xffffffffu, have ? static_cast<int>(vs) : hole ? -1000 : 1000);
      const int least_k = __reduce_min_sync(0xffffffffu, have ? static_cast<int>(ks) : 1000);
      if (lane == 0) {
        extremes[group_of][t & 1][cw][0] = ek;
        extremes[group_of][t & 1][cw][1] = ev;
        extremes[group_of][t & 1][cw][2] = least;
        extremes[group_of][t & 1][cw][3] = least_k;
      }
      const float scale = have ? kv8_scale(vs) : 0.f, k_scale = have ? kv8_scale(ks) : 0.f;
      const float exponent = have ? static_cast<float>(static_cast<int>(vs) - 127) : -INFINITY;
      pages = pages_of(ids);  // -1 everywhere past the last tile
      ids = load_ids(t + 2);
      load_scales(t + 1);
      // All four warps go on, or none: a wait that ran out is known to all here.
      ok = named_bar_all(3 + group_of, 128, ok);
      if (!ok) break;
      int e_k = 0, e_v = 0, low = 1000, low_k = 1000;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        e_k = max(e_k, extremes[group_of][t & 1][w][0]);
        e_v = max(e_v, extremes[group_of][t & 1][w][1]);
        low = min(low, extremes[group_of][t & 1][w][2]);
        low_k = min(low_k, extremes[group_of][t & 1][w][3]);
      }
      // (max (s f) is max (s) f for a scale >= 0 only.)
      const bool apart = e_v - low > kSpread || e_k - low_k > kSpreadK || !(a.scale >= 0.f);
      ok = t < 2 || mbar_wait(&empty[t & 1], ((t - 2) >> 1) & 1, a.status);
      if (!values) {
        // The scores of tile t - 2 followed the sums of tile t - 4, so that
        // tile's entry is read by nobody any more.
        if (tid == 0) {
          exps[t & 3][0] = e_k > 0 && !apart ? e_k : 127;
          exps[t & 3][1] = apart ? kApart : e_v - 127;
        }
        if (apart) {
          value_scale[t & 3][tid] = scale;
          value_scale[t & 3][kKeys + tid] = exponent;
          value_scale[t & 3][2 * kKeys + tid] = k_scale;
        }
      }
      uint8_t* dst = operand + (t & 1) * T::kOperand;
      const int top = values ? e_v : e_k;
      const int left = keys - (kt0 + t + 1) * kKeys;
      // All passes' factors and pages first: nothing then waits between stores.
      uint32_t factor[kPasses];
      int page[kPasses];
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        page[p] = page_of(p);
        const int byte = scale_byte[group_of][t & 1][p * Share<D>::kRows + share.row];
        factor[p] = apart ? 0x3c003c00u : half_power2(byte - top + 127);
      }
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        store_codes<D>(dst, share, p, c[p], factor[p]);
        c[p] = load_codes<D>(share, pool, page[p], p, left);
      }
      if (values && (kt0 + t + 1) * kKeys > hidden0) {
        ok = mbar_wait(&looked, 0, a.status) && ok;
        if (nan_hidden) hide_nan<D>(dst, share, hidden0 - (kt0 + t) * kKeys);
      }
      fence_proxy_async();
      mbar_arrive(&full[t & 1]);
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const int g = warp >> 2, tid = threadIdx.x & 127;  // group, row (TMEM lane)
    // Queries into shared memory: 16-byte chunks, swizzled.
    {
      constexpr int kChunks = D / 8;
      const int who = SHARED ? tid : threadIdx.x, step = SHARED ? 128 : kSoftmax;
      const int c0 = x0 + (SHARED ? g * kRows : 0);
      uint8_t* dst = smem + T::kQ + (SHARED ? g * T::kOperand : 0u);
      const int c = who % kChunks, rows = step / kChunks;
      const __half* from = a.q + static_cast<size_t>(x.t0) * a.ld_q +
                           static_cast<size_t>(kvh) * group * D + c * 8;
#pragma unroll 1
      for (int r0 = who / kChunks; r0 < kRows; r0 += 8 * rows) {  // eight loads in flight
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = r0 + i * rows, col = c0 + r, token = col / group;
          v[i] = load16_if(from + static_cast<size_t>(token) * a.ld_q +
                               static_cast<size_t>(col - token * group) * D,
                           r < kRows && col < cols);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = r0 + i * rows;
          if (r < kRows)
            *reinterpret_cast<uint4*>(dst + (c >> 3) * T::kAtom + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
                v[i];
        }
      }
      fence_proxy_async();
      mbar_arrive(&q_full);
    }
    // While the first scores are on their way: NaN codes in V of those keys.
    constexpr int kPieces = D / 16;
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < (hidden1 - hidden0) * kPieces; i0 += 4 * kSoftmax) {
      const uint8_t* at[4];
      uint32_t nan = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = hidden0 + (i0 + i * kSoftmax) / kPieces;
        at[i] = key < hidden1 ? value_row(a, row, kvh, key, D) : nullptr;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 c = load16_if(at[i] + (i0 + i * kSoftmax) % kPieces * 16, at[i] != nullptr);
        nan |= kv8_nan_codes(c.x) | kv8_nan_codes(c.y) | kv8_nan_codes(c.z) | kv8_nan_codes(c.w);
      }
      if (nan) nan_hidden = 1;
    }
    mbar_arrive(&looked);
    const int col = x0 + (SHARED ? g * kRows : 0) + tid;
    const int lim = col < cols ? min(past + col / group, keys - 1) : -1;  // last key seen
    const float sl2 = a.scale * kLog2e;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t sa = lanes + T::kTmemS + g * 128, oa = lanes + T::kTmemO + g * 128;
    float m = kNoReference, l = 0.f;
    bool ok = true;
    const int mine = SHARED ? n : (n + 1 - g) >> 1;  // key tiles of this group
    for (int j = 0; j < mine; ++j) {
      const int t = SHARED ? j : 2 * j + g;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[g], j & 1, a.status));
      if (!ok) break;
      tc_fence_after();
      const float f = sl2 * __uint_as_float(static_cast<uint32_t>(exps[t & 3][0]) << 23);
      const int e_v = exps[t & 3][1];
      const int seen = lim - (kt0 + t) * kKeys;  // keys 0 .. seen of the tile
      const float4* vs = reinterpret_cast<const float4*>(value_scale[t & 3]);
      const float2 f2 = make_float2(f, f);
      auto pair_of = [](uint32_t lo, uint32_t hi) {
        return make_float2(__uint_as_float(lo), __uint_as_float(hi));
      };
      float alpha = 1.f;
      // Two passes over the scores in rolled loops: the code of all roles has to
      // stay in the instruction cache, or the products wait for their
      // instructions.  16 scores are on their way while 16 are worked on.
      auto pass = [&](auto kind) {
        constexpr bool kMasked = decltype(kind)::value >= 1, kEach = decltype(kind)::value == 2;
        float m0 = -INFINITY, m1 = -INFINITY;
        uint32_t v[2][16];
        auto largest = [&](const uint32_t (&x)[16], int c) {
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            float2 y0 = pair_of(x[i], x[i + 1]), y1 = pair_of(x[i + 2], x[i + 3]);
            if (kEach) {
              const float4 ev = vs[(kKeys + c + i) / 4], ks = vs[(2 * kKeys + c + i) / 4];
              y0 = fma2(mul2f(y0, make_float2(ks.x, ks.y)), f2, make_float2(ev.x, ev.y));
              y1 = fma2(mul2f(y1, make_float2(ks.z, ks.w)), f2, make_float2(ev.z, ev.w));
            }
            if (kMasked) {
              if (c + i > seen) y0.x = -INFINITY;
              if (c + i + 1 > seen) y0.y = -INFINITY;
              if (c + i + 2 > seen) y1.x = -INFINITY;
              if (c + i + 3 > seen) y1.y = -INFINITY;
            }
            m0 = fmaxf(m0, fmaxf(y0.x, y0.y));
            m1 = fmaxf(m1, fmaxf(y1.x, y1.y));
          }
        };
        tmem_ld16_nowait(sa, v[0]);
#pragma unroll 1
        for (int c = 0; c < kKeys; c += 32) {
          tmem_ld_wait();
          tmem_ld16_nowait(sa + c + 16, v[1]);
          largest(v[0], c);
          tmem_ld_wait();
          tmem_ld16_nowait(sa + (c + 32) % kKeys, v[0]);  // at the end: the second pass's first
          largest(v[1], c + 16);
        }
        const float offset = kEach ? 0.f : static_cast<float>(e_v);
        const float mx = kEach ? fmaxf(m0, m1) : fmaf(fmaxf(m0, m1), f, offset);
        // A reference moves only when a weight, rounded as below, would pass 2^14.
        if ((kEach ? mx - m : fmaf(fmaxf(m0, m1), f, offset - m)) > kMost) {
          alpha = ex2(m - (mx - kTop));
          m = mx - kTop;
        }
        float2 sum = make_float2(0.f, 0.f);
        const float2 minus = make_float2(offset - m, offset - m);
        // The weights of 16 keys go over scores that are read already.
        auto weigh = [&](const uint32_t (&x)[16], int c) {
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            float2 y0 = pair_of(x[i], x[i + 1]), y1 = pair_of(x[i + 2], x[i + 3]);
            if (kEach) {
              const float4 ks = vs[(2 * kKeys + c + i) / 4];
              y0 = mul2f(y0, make_float2(ks.x, ks.y));
              y1 = mul2f(y1, make_float2(ks.z, ks.w));
            }
            y0 = fma2(y0, f2, minus);
            y1 = fma2(y1, f2, minus);
            if (kMasked) {
              if (c + i > seen) y0.x = -INFINITY;
              if (c + i + 1 > seen) y0.y = -INFINITY;
              if (c + i + 2 > seen) y1.x = -INFINITY;
              if (c + i + 3 > seen) y1.y = -INFINITY;
            }
            float2 w0, w1;
            if (kEach) {
              const float4 sc = vs[(c + i) / 4];
              w0 = make_float2(sc.x == 0.f ? 0.f : ex2(y0.x), sc.y == 0.f ? 0.f : ex2(y0.y));
              w1 = make_float2(sc.z == 0.f ? 0.f : ex2(y1.x), sc.w == 0.f ? 0.f : ex2(y1.y));
              sum = add2f(sum, add2f(w0, w1));
              w0 = mul2f(w0, make_float2(sc.x, sc.y));
              w1 = mul2f(w1, make_float2(sc.z, sc.w));
            } else {
              w0 = make_float2(ex2(y0.x), ex2(y0.y));
              // Three of eight pairs on the FMA pipes (2048 tokens behind 8192 keys 411 ->
              // 384 us; four 399).  With one query tile the special function unit is
              // not what bounds, and the longer code costs.
              w1 = SHARED && !kMasked && i != 0 ? exp2_fma(y1) : make_float2(ex2(y1.x), ex2(y1.y));
              sum = add2f(sum, add2f(w0, w1));
            }
            pk[i >> 1] = half2_bits(w0.x, w0.y);
            pk[(i >> 1) + 1] = half2_bits(w1.x, w1.y);
          }
          tmem_st8(sa + c / 2, pk);
        };
#pragma unroll 1
        for (int c = 0; c < kKeys; c += 32) {
          tmem_ld_wait();
          tmem_ld16_nowait(sa + c + 16, v[1]);
          weigh(v[0], c);
          tmem_ld_wait();
          if (c + 32 < kKeys) tmem_ld16_nowait(sa + c + 32, v[0]);
          weigh(v[1], c + 16);
        }
        return kEach ? sum.x + sum.y : (sum.x + sum.y) * ex2(-offset);
      };
      const bool full = __all_sync(0xffffffffu, seen >= kKeys - 1);
      const float rs = e_v == kApart ? pass(std::integral_constant<int, 2>{})
                       : full ? pass(std::integral_constant<int, 0>{})
                              : pass(std::integral_constant<int, 1>{});
      l = l * alpha + rs;
      // O was summed to another reference: bring it to the new one.
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        ok = __all_sync(0xffffffffu, mbar_wait(&o_done[g], (j - 1) & 1, a.status));
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t v[32];
          tmem_ld32_nowait(oa + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
          tmem_st32(oa + c, v);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[g]);
    }
    // The last of this group's products; where both groups work on one tile of
    // queries, each waits for its own, and they meet (a group without a key tile
    // has no sums).
    if (mine > 0)
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&o_done[g], (mine - 1) & 1, a.status));
    const bool have0 = n > 0, have1 = !SHARED && n > 1;
    float w0 = 1.f, w1 = 0.f;  // weights of the groups' sums
    if (!SHARED) {
      group_ml[g][tid] = make_float2(m, l);
      tc_fence_before();
      ok = named_bar_all(1, kSoftmax, ok);
      const float2 ml0 = group_ml[0][tid], ml1 = group_ml[1][tid];
      m = fmaxf(ml0.x, ml1.x);
      w0 = ex2(ml0.x - m);
      w1 = ex2(ml1.x - m);
      l = ml0.y * w0 + ml1.y * w1;
    }
    tc_fence_after();
    if (ok) {
      const bool split = !SHARED && parts > 1;
      const size_t cell = (static_cast<size_t>(found[2]) * hkv + kvh) * gridDim.z + blockIdx.z;
      float4* piece = reinterpret_cast<float4*>(partial + cell * T::kPiece);
      const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: no key on a page that is there
      __half* out = col < cols ? a.out + static_cast<size_t>(x.t0 + col / group) * a.ld_out +
                                     static_cast<size_t>(kvh * group + col % group) * D
                               : nullptr;
      // 16 dimensions at a time; groups that share their rows take half each.
      const uint32_t from = SHARED ? oa : lanes + T::kTmemO;
#pragma unroll 1
      for (int c = SHARED ? 0 : g * (D / 2); c < (SHARED ? D : (g + 1) * (D / 2)); c += 16) {
        uint32_t v0[16], v1[16];
        if (have0) tmem_ld16_nowait(from + c, v0);
        if (!SHARED && have1) tmem_ld16_nowait(from + 128 + c, v1);
        tmem_ld_wait();
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          v[i] = have0 ? __uint_as_float(v0[i]) * w0 : 0.f;
          if (!SHARED && have1) v[i] += __uint_as_float(v1[i]) * w1;
        }
        if (split) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            piece[(c / 4 + i) * 128 + tid] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else if (out) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              h[k] = lim < 0 ? 0u : half2_bits(v[8 * i + 2 * k] * inv, v[8 * i + 2 * k + 1] * inv);
            *reinterpret_cast<uint4*>(out + c + 8 * i) = make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
      }
      if (split && g == 0) reinterpret_cast<float2*>(piece + 128 * (D / 4))[tid] = make_float2(m, l);
      if (nan_hidden && col < cols)
        put_nan<D>(a, row, kvh, hidden0, min(lim + 1, hidden1), SHARED ? 0 : g * (D / 2),
                   SHARED ? D : (g + 1) * (D / 2), out,
                   split ? reinterpret_cast<float*>(piece + tid) : nullptr);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// Joins the key splits of a query tile in order: one CTA a tile and kv head.
template <int D>
__global__ void __launch_bounds__(256)
    kv8_tile_join_kernel(const Kv8AttnArgs a, int group, int tile_from, const float* partial, int splits) {
  using T = Tile<D, false>;
  __shared__ int found[2];
  griddep_enter();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    const int want = blockIdx.x, most = gridDim.x;
    int row = -1, before = 0;
    for (int base = 0; base < a.rows && before <= want; base += 32) {
      const int r = base + lane;
      const int own = r < a.rows ? kv8_row(a, r, group, kRows, tile_from, false, true).chunks : 0;
      const int upto = tiles_upto(own, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > want);
      if (hit) {
        const int src = __ffs(hit) - 1;
        row = __shfl_sync(0xffffffffu, fits(before, upto, most) ? r : -1, src);
        before += __shfl_sync(0xffffffffu, upto - own, src);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      found[0] = row;
      found[1] = want - before;
    }
  }
  __syncthreads();
  if (found[0] < 0) return;
  const Kv8Row x = kv8_row(a, found[0], group, kRows, tile_from, false, true);
  const int kvh = blockIdx.y, x0 = found[1] * kRows, cols = x.count * group;
  const int parts = parts_of((seen_keys(x, group, x0, kRows) + kKeys - 1) / kKeys, splits);
  if (parts == 1) return;  // the tile pass wrote the result
  const float4* base = reinterpret_cast<const float4*>(
      partial + (static_cast<size_t>(blockIdx.x) * a.cache.hkv + kvh) * splits * T::kPiece);
  // A thread takes one row's eight dimensions.
  for (int u = threadIdx.x; u < kRows * (D / 8); u += 256) {
    const int r = u % kRows, d8 = u / kRows, col = x0 + r;
    if (col >= cols) continue;
    auto ml_of = [&](int s) {
      return __ldcg(reinterpret_cast<const float2*>(base + static_cast<size_t>(s) * (T::kPiece / 4) +
                                                    128 * (D / 4)) + r);
    };
    float m = kNoReference;
    for (int s = 0; s < parts; ++s) m = fmaxf(m, ml_of(s).x);
    float l = 0.f;
    float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
    for (int s = 0; s < parts; ++s) {
      const float4* piece = base + static_cast<size_t>(s) * (T::kPiece / 4);
      const float2 ml = ml_of(s);
      const float w = ex2(ml.x - m);
      l += ml.y * w;
      const float4 v0 = __ldcg(piece + (d8 * 2) * 128 + r), v1 = __ldcg(piece + (d8 * 2 + 1) * 128 + r);
      lo.x += v0.x * w;
      lo.y += v0.y * w;
      lo.z += v0.z * w;
      lo.w += v0.w * w;
      hi.x += v1.x * w;
      hi.y += v1.y * w;
      hi.z += v1.z * w;
      hi.w += v1.w * w;
    }
    const bool none = x.len - x.count + col / group < 0;
    const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: no key on a page that is there
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (!none)
      o = make_uint4(half2_bits(lo.x * inv, lo.y * inv), half2_bits(lo.z * inv, lo.w * inv),
                     half2_bits(hi.x * inv, hi.y * inv), half2_bits(hi.z * inv, hi.w * inv));
    *reinterpret_cast<uint4*>(a.out + static_cast<size_t>(x.t0 + col / group) * a.ld_out +
                              static_cast<size_t>(kvh * group + col % group) * D + d8 * 8) = o;
  }
}

// The most query tiles of `columns` columns that the batch's rows can have.
long long most_tiles(int rows, int tokens, int group, int columns) {
  return static_cast<long long>(tokens) * group / columns + std::min(rows, tokens);
}

struct Plan {
  bool shared;
  int tiles, splits;
};
constexpr int kMostSplits = 16;
Plan plan_tiles(int rows, int tokens, int hq, int hkv, int sm_count) {
  const int group = hq / hkv;
  // Two query tiles a CTA halve the conversions; worth it from two waves on.
  const long long single = most_tiles(rows, tokens, group, kRows);
  Plan p{};
  p.shared = static_cast<long long>(tokens) * group / kRows * hkv >= 2LL * sm_count;
  p.tiles = static_cast<int>(p.shared ? most_tiles(rows, tokens, group, 2 * kRows) : single);
  // Splits for the CTAs that have work: a row has one tile at least, and most
  // batches about the larger of both counts (eight rows of 64 columns on 8 kv
  // heads behind 4000 keys: 59 -> 43 us at head size 64, 67 -> 56 at 128).
  const long long likely = std::max(static_cast<long long>(tokens) * group / kRows,
                                    static_cast<long long>(std::min(rows, tokens)));
  p.splits = p.shared ? 1
                      : static_cast<int>(std::max(
                            1LL, std::min<long long>(kMostSplits, sm_count / std::max(1LL, likely * hkv))));
  return p;
}

template <int D, bool SHARED>
cudaError_t launch_tile(const Kv8AttnArgs& a, const Plan& p, int tile_from, float* partial,
                        cudaStream_t stream) {
  using T = Tile<D, SHARED>;
  static Kv8Configured configured;
  const cudaError_t e = configured.once(kv8_tile_kernel<D, SHARED>, static_cast<int>(T::kSmem));
  if (e != cudaSuccess) return e;
  return launch_dependent(kv8_tile_kernel<D, SHARED>, dim3(p.tiles * a.cache.hkv, 1, p.splits), dim3(kThreads),
                          T::kSmem, stream, a, a.hq / a.cache.hkv, tile_from, partial);
}

}  // namespace

bool kv8_tile_supported(int dim) { return dim == 64 || dim == 128; }

size_t kv8_tile_workspace(int dim, int sm_count) {
  // Splits are made while the likely CTAs are no more than the SMs, and the grid
  // has at most twice as many.  Fewer tokens can have more splits, so the room is
  // for any count up to these.
  return static_cast<size_t>(sm_count) * 2 * 128 * (dim + 2) * sizeof(float);
}

cudaError_t kv8_tile_launch(const Kv8AttnArgs& a, int tile_from, float* partial, cudaStream_t stream) {
  const Plan p = plan_tiles(a.rows, a.tokens, a.hq, a.cache.hkv, a.sm_count);
  if (a.cache.dim == 64)
    return p.shared ? launch_tile<64, true>(a, p, tile_from, partial, stream)
                    : launch_tile<64, false>(a, p, tile_from, partial, stream);
  return p.shared ? launch_tile<128, true>(a, p, tile_from, partial, stream)
                  : launch_tile<128, false>(a, p, tile_from, partial, stream);
}

cudaError_t kv8_tile_join_launch(const Kv8AttnArgs& a, int tile_from, const float* partial,
                                 cudaStream_t stream) {
  const Plan p = plan_tiles(a.rows, a.tokens, a.hq, a.cache.hkv, a.sm_count);
  if (p.splits == 1) return cudaSuccess;
  const dim3 grid(p.tiles, a.cache.hkv);
  const int group = a.hq / a.cache.hkv;
  return a.cache.dim == 64 ? launch_dependent(kv8_tile_join_kernel<64>, grid, dim3(256), 0, stream, a,
                                              group, tile_from, partial, p.splits)
                           : launch_dependent(kv8_tile_join_kernel<128>, grid, dim3(256), 0, stream, a,
                                              group, tile_from, partial, p.splits);
}

}  // namespace hb
