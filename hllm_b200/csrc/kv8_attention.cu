// kv8_attention.cu -- attention over the 8-bit paged KV cache: the pass that
// streams pages through registers (new tokens one or a few at a time), and the
// join of what it split.
//
// o = sum_j softmax_j(scale q.k_j) v_j over the keys j <= the query's position.
// With k_j = 2^ek_j c_j and v_j = 2^ev_j d_j (codes c, d) and s_j = scale
// log2(e) 2^ek_j (q.c_j), one reference m serves
//   l = sum 2^(s_j - m),   O = sum (2^(s_j - m) 2^ev_j) d_j,   o = O / l.
// The weights in brackets are what the products round (F16, by 2^-11), so m
// follows max (s_j + ev_j): they keep their precision whatever the sizes of the
// value rows.  It is raised only when a weight passes 2^14, to where the largest is
// 2^7: most pages rescale nothing.
//
// Work.  A row's new tokens and the query heads of one kv head form columns
// (token, head), 8 NT of them a stream; a stream walks the row's pages, one to
// four at a time (a unit).  The batch's units in order are one sequence, cut evenly over
// the CTAs of one wave and, within a CTA, over its warps, whatever the rows'
// lengths.  Everything about the cut follows from the lengths on the device:
// a captured launch serves any lengths.  What a cut leaves of a stream is
// joined first in the CTA (shared memory), then, where a stream spans CTAs, by
// a second small launch, in order: results do not depend on timing.
//
// Per page a warp computes S^T = K Q^T and O^T = V^T P^T with m16n8k16 F16
// products, codes becoming F16 in registers (exactly; a product of e4m3 operands
// would not be faster: mma.sync runs it as F16 products after converting both).
// The 16 keys, then 16 value dimensions, are the M side, so that the columns are
// the 8-wide N side and one decode row wastes half of a
// tile, not three quarters.  The order of the products' inner dimension is
// free, so a lane takes 16 consecutive bytes of a key for four steps of QK, and
// for PV the bytes of four keys, paired by byte permutes.  Pages arrive by TMA,
// one lane of a warp asking for its warp's, in boxes whose swizzle spreads each
// read over all banks (rows and the order of reads are chosen for that).
//
// Bound by memory where rows are long: 64 rows of 1024 to 16384 keys, 32 heads on
// 8 of 128, 141 us for 768 MB, 5.4 TB/s.  There a warp's unit of two pages is 2600
// cycles, 1050 of them for asking for the next one.  Short calls are latency: one
// row of 1000 keys 9.7 us, of which the way from the lengths over the table to the
// first page is about 4, the joins 4.  The same rows with 16 query heads on a kv
// head: 186 us (as two streams of 8 columns each, 265).
#include <cudaTypedefs.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kv8.cuh"

namespace hb {
namespace {

// Units of a CTA, where there are so many: one a warp.  One row of 1000 keys, 8 kv
// heads: 9.7 us at 4 or 8, 10.5 at 2 (more pieces to join), 11.2 at 16.
constexpr int kLeast = 8;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t o;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(o) : "r"(v));
  return o;
}

// Words (4 codes) of a lane's own slot of the ring.
template <int W>
__device__ __forceinline__ void read_words(uint32_t (&w)[W], const uint8_t* p) {
  if constexpr (W == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  } else if constexpr (W == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
// How a page of 16 keys x D codes lies in shared memory: boxes of BOX bytes of
// every key, 16-byte chunks swizzled within 128 bytes by the key's line, and who
// reads what.  K: four lanes (t) share a key row, KW words of four codes each,
// KS steps.  V: eight lanes (g) share a value row, VW words each, VS steps.
template <int D>
struct Layout {
  static constexpr int BOX = D % 128 == 0 ? 128 : D % 64 == 0 ? 64 : 32;
  static constexpr int KW = D % 64 == 0 ? 4 : 2, KS = D / (16 * KW);
  static constexpr int VW = D % 128 == 0 ? 4 : D % 64 == 0 ? 2 : 1, VS = D / (32 * VW);
  __device__ static int swizzle(int row) {
    return BOX == 128 ? row & 7 : BOX == 64 ? row >> 1 & 3 : row >> 2 & 1;
  }
  // Key of row g of the score product (and + 8 of row g + 8): with 128-byte
  // boxes two neighbouring g take rows whose swizzles differ in bit 2.
  __device__ static int key_of(int g) { return BOX == 128 ? (g >> 1) | (g & 1) << 2 : g; }
  // Byte of lane (g, t)'s words of step s, key row g.
  __device__ static int k_at(int g, int t, int s) {
    const int row = key_of(g), byte = (s * 4 + t) * KW * 4;
    return byte / BOX * (16 * BOX) + row * BOX + ((byte % BOX / 16 ^ swizzle(row)) << 4) + byte % 16;
  }
  // Value rows of lane t: keys value_key(t, 0 .. 3), in the order of the
  // weights' fragment.  Some lanes read the first two, and the last two, in
  // the other order, which makes eight reads reach all banks.
  __device__ static int value_key(int t, int h) {
    return (BOX == 128 ? t + 4 * (h & 1) : 2 * t + (h & 1)) + 8 * (h >> 1);
  }
  __device__ static bool swapped(int g, int t) {
    return BOX == 128 ? g & 1 : BOX == 64 ? g >> 1 & 1 : t >> 1;
  }
  __device__ static int byte_at(int row, int byte) {
    return byte / BOX * (16 * BOX) + row * BOX + ((byte % BOX / 16 ^ swizzle(row)) << 4) + byte % 16;
  }
  __device__ static int v_at(int g, int t, int h, int s) {
    return byte_at(value_key(t, h), (s * 8 + g) * VW * 4);
  }
};

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}
// 4 or 16 bytes from global to shared memory, asynchronously (zeros where
// !live); the arrival on a barrier once a lane's copies have landed; and the
// wait for them.
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void copy4_async(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <int D, int NT>
struct Shape : Layout<D> {
  using Layout<D>::VW;
  static constexpr int kCols = 8 * NT;
  // Enough warps to hide the latency of one unit's chain of products, and
  // enough bytes in flight to hide that of memory (at D = 128 two units of 8 KB a
  // warp beside the one in use, 128 KB an SM).
  // Pages of a unit, which share its waits and copies, and of them at a time in
  // registers.  64 long rows: D = 64, 8 columns 100 us at two pages a unit, 87 at
  // four; 16 columns, D = 64 173 at one, 135 at two; D = 128 215 and 186.
  static constexpr int KP = D > 128 ? 1 : D > 64 || NT > 1 ? 2 : 4;
  static constexpr int MP = D * NT > 128 ? 1 : KP;
  static constexpr int kWarps = D * NT > 64 ? 8 : 12;
  static constexpr int kThreads = kWarps * 32;
  // A piece: D / 16 x NT fragments of 32 lanes x 4 sums, then cols x (m, l).
  static constexpr int kUnits = D / 16 * NT * 32;
  static constexpr int kPiece = kUnits * 4 + kCols * 2;  // floats
  // A warp's shared memory: its ring of units, whose place the piece that it
  // ends with takes; their scales; the ring's barriers; the queries of a stream
  // to come (each lane's own); three pieces of the block table.  Behind the warps' lie
  // kSlots places for pieces that are done earlier (one a stream that ends
  // within a warp's share and began before it; any more go to the workspace).
  static constexpr int kPage = 32 * D;  // codes of K, then of V
  static constexpr int kStage = KP * kPage;
  static constexpr int kPieceBytes = kPiece * static_cast<int>(sizeof(float));
  static constexpr int kQueryBytes = kCols * D * 2;
  static constexpr int kSlots = D * NT <= 64 ? 4 : 1;
  static constexpr int kRoom = (225 * 1024 - kSlots * kPieceBytes) / kWarps / 1024 * 1024;
  __host__ __device__ static constexpr int bytes(int stages) {
    return (stages * (kStage + 32 * KP + 8) + 8 + kQueryBytes + 3 * 128 + 1023) / 1024 * 1024;
  }
  static constexpr int kStages = bytes(4) <= kRoom ? 4 : bytes(3) <= kRoom ? 3 : 2;
  static constexpr int kWarpBytes = bytes(kStages);
  static constexpr int kScalesAt = kStages * kStage, kBarsAt = kScalesAt + kStages * 32 * KP;
  static constexpr int kQueriesAt = (kBarsAt + kStages * 8 + 15) / 16 * 16, kTableAt = kQueriesAt + kQueryBytes;
  static constexpr int kSmem = kWarps * kWarpBytes + kSlots * kPieceBytes + 1024;  // 1024: alignment
  static_assert(kScalesAt >= kPieceBytes && kTableAt + 3 * 128 <= kWarpBytes && kWarpBytes <= kRoom,
                "shared memory of a warp");
  // Value dimension of unit (i, lane): rows g and g + 8 of product i are
  // consecutive dimensions.
  __device__ static int dim_of(int i, int g) {
    const int st = i / (2 * VW), rest = i % (2 * VW);
    return (st * 8 + g) * VW * 4 + rest * 2;
  }
};

// The code pools as boxes of BOX codes x one page: [page of a kv head][16][D].
struct PoolMaps {
  CUtensorMap k, v;
};

// Units of one stream of a row, of KP pages, and of all its streams.
template <int KP>
__device__ __forceinline__ int stream_units(const Kv8Row& x) {
  return (x.pages + KP - 1) / KP;
}
template <int KP>
__device__ __forceinline__ long long row_units(const Kv8Row& x, int hkv) {
  return static_cast<long long>(x.chunks) * hkv * stream_units<KP>(x);
}

// a / b for a >= 0, b > 0: a 64-bit division costs hundreds of cycles, and
// nearly no batch needs one.
__device__ __forceinline__ long long divide(long long a, long long b) {
  if ((a | b) >> 32 == 0)
    return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}
// The even cut of the units over CTAs: the first `more` take one unit more.
struct Cut {
  int ctas;               // CTAs with work
  long long total, each;  // units, and of a CTA at least
  int more;
};
__device__ __forceinline__ Cut make_cut(long long total, int most, int least) {
  Cut c;
  c.total = total;
  c.ctas = static_cast<int>(
      min(static_cast<long long>(most), max(1LL, divide(total + least - 1, least))));
  c.each = divide(total, c.ctas);
  c.more = static_cast<int>(total - c.each * c.ctas);
  return c;
}
__device__ __forceinline__ long long cut_begin(const Cut& c, int i) {
  return c.each * i + min(i, c.more);
}
__device__ __forceinline__ int cut_owner(const Cut& c, long long unit) {
  const long long big = (c.each + 1) * c.more;
  return static_cast<int>(unit < big ? divide(unit, c.each + 1) : c.more + divide(unit - big, c.each));
}

// The workspace: per CTA a record, two pieces (the stream it continues, the
// stream it leaves open), and a piece a warp.  The record is of a stream that earlier CTAs began
// and this one ended: the CTA that began it (-1: there is none), and what its
// output needs.
struct Record {
  int first, kvh, x0;      // the stream's first column
  int count, len, t0;      // of its row
  int pad[2];
};

// Where column `col` of a stream goes (null past the row's columns), and the
// factor that makes its sums the output (0: it has no key, or none on a page
// that is there, and its sums are zeros).
struct Output {
  __half* to;
  float factor;
};
__device__ __forceinline__ Output output_of(const Kv8AttnArgs& a, const Kv8Row& x, int group, int kvh,
                                            int col, float l) {
  if (col >= x.count * group) return Output{nullptr, 0.f};
  const int token = x.count > 1 ? col / group : 0;
  return Output{a.out + static_cast<size_t>(x.t0 + token) * a.ld_out +
                    static_cast<size_t>(kvh * group + col - token * group) * a.cache.dim,
                x.len - x.count + token < 0 || l == 0.f ? 0.f : 1.f / l};
}
// One unit: sums of two columns at dimensions dim, dim + 1.
__device__ __forceinline__ void store_unit(const Output& c0, const Output& c1, int dim, const float4& v) {
  if (c0.to) *reinterpret_cast<__half2*>(c0.to + dim) = __floats2half2_rn(v.x * c0.factor, v.z * c0.factor);
  if (c1.to) *reinterpret_cast<__half2*>(c1.to + dim) = __floats2half2_rn(v.y * c1.factor, v.w * c1.factor);
}

// CHUNKS: rows may have several new tokens, so a stream's columns may see
// different keys (hide_nan).  Batches of one token a row go without that code: 64
// long rows take 141 us so, 144 with it.
template <int D, int NT, bool CHUNKS>
__global__ void __launch_bounds__(Shape<D, NT>::kThreads, 1)
    kv8_stream_kernel(const __grid_constant__ PoolMaps maps, const Kv8AttnArgs a, int group,
                      int tile_from, bool beside) {
  using S = Shape<D, NT>;
  constexpr int kCols = S::kCols, kWarps = S::kWarps, ST = S::kStages, KP = S::KP, MP = S::MP;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  // Pieces that warps leave: the row (-1: none), kv head, chunk, and whether the
  // piece has the stream's first (1) and last (2) page; and of the row its new
  // tokens, keys, first token and units of a stream.
  __shared__ int4 left[kWarps * 2], left_row[kWarps * 2];
  __shared__ float* where[kWarps * 2];
  __shared__ int slots_taken;
  __shared__ int order[kWarps * 2 + 1], chains[kWarps * 2 + 1], chain_count;
  __shared__ long long units_before;  // units before the row of the CTA's first one
  // Launched behind the tile pass this one runs beside it: that pass lets its
  // successor start once all its CTAs have seen the work before them complete,
  // and the two share no output.  It then waits before it ends, so that what
  // follows it follows both.
  if (!beside) griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  const int hkv = a.cache.hkv;

  if (lane == 0 && warp < 2) prefetch_tensormap(warp ? &maps.v : &maps.k);
  if (threadIdx.x == 0) slots_taken = 0;
  // The block tables and the queries are needed only after the lengths: a line
  // of each a thread comes to L2 meanwhile.
  {
    const long long i = static_cast<long long>(blockIdx.x) * S::kThreads + threadIdx.x;
    if (i * 32 < static_cast<long long>(a.rows) * a.max_blocks) prefetch_l2(a.tables + i * 32);
    const long long per = (static_cast<long long>(a.hq) * D + 63) / 64;
    if (i < per * a.tokens) prefetch_l2(a.q + divide(i, per) * a.ld_q + (i - divide(i, per) * per) * 64);
  }
  // All units: their number up to each row of a group of 128 rows, one scan.
  long long upto[4];
  int4 rows[4];  // a lane's rows: new tokens, keys, first token, chunks
  auto scan = [&](int base, bool report) {  // returns the group's units
    long long sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = base + 32 * k + lane;
      upto[k] = 0;
      if (r < a.rows) {
        const Kv8Row x = kv8_row(a, r, group, kCols, tile_from, report);
        upto[k] = row_units<KP>(x, hkv);
        rows[k] = make_int4(x.count, x.len, x.t0, x.chunks);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (base + 32 * k < a.rows) {
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const long long v = __shfl_up_sync(0xffffffffu, upto[k], off);
          if (lane >= off) upto[k] += v;
        }
        upto[k] += sum;
        sum = __shfl_sync(0xffffffffu, upto[k], 31);
      }
    }
    return sum;
  };
  long long total = 0;
  for (int base = 0; base < a.rows; base += 128) total += scan(base, blockIdx.x == 0 && warp == 0);
  // A CTA takes kLeast units at least, where there are so many.
  const Cut cut = make_cut(total, gridDim.x, kLeast);
  Record* records = reinterpret_cast<Record*>(a.workspace);
  if (total == 0 || static_cast<int>(blockIdx.x) >= cut.ctas) {
    if (threadIdx.x == 0) records[blockIdx.x].first = -1;
    if (beside) griddep_wait();
    return;
  }
  const long long c0 = cut_begin(cut, blockIdx.x);
  const int units = static_cast<int>(cut_begin(cut, blockIdx.x + 1) - c0);
  const int from = static_cast<int>(divide(static_cast<long long>(units) * warp, kWarps));
  const int n = static_cast<int>(divide(static_cast<long long>(units) * (warp + 1), kWarps)) - from;
  const long long w0 = c0 + from;

  float o[NT][D / 16][4];
  float m[NT][2], l[NT][2];
  uint8_t* const ring = smem + warp * S::kWarpBytes;
  uint64_t* const full = reinterpret_cast<uint64_t*>(ring + S::kBarsAt);
  if (lane < 2) left[warp * 2 + lane].x = -1;
  if (lane == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&full[i], 33);  // the boxes, and every lane's scales
    fence_mbar_init();
  }
  __syncthreads();  // slots_taken

  if (n > 0) {
    // The row of the warp's first unit.
    int row = -1;
    long long before = 0;  // units before the row
    for (int base = 0; row < 0; base += 128) {
      long long next = before;
      if (a.rows > 128) next += scan(base, false);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (row >= 0 || base + 32 * k >= a.rows) continue;
        const unsigned hit = __ballot_sync(0xffffffffu, before + upto[k] > w0);
        if (hit) {
          row = base + 32 * k + __ffs(hit) - 1;
          if (row > base) {
            // Units up to the row before it, which may be the last of the 32 before.
            const int prev = row - base - 1;
            const long long of = prev < 32 ? upto[0] : prev < 64 ? upto[1] : prev < 96 ? upto[2] : upto[3];
            before += __shfl_sync(0xffffffffu, of, prev & 31);
          }
        }
      }
      if (row < 0) before = next;
    }
    if (w0 == c0 && lane == 0) units_before = before;
    const float sl2 = a.scale * kLog2e;
    // Where the arithmetic is, and the loader, ST - 1 units ahead of it.
    struct Cursor {
      int row, kvh, chunk, unit, units;  // units: of the stream
      Kv8Row x;
    };
    Cursor at;
    at.row = row;
    {
      const int k = row % 128 >> 5;
      const int4 r = k == 0 ? rows[0] : k == 1 ? rows[1] : k == 2 ? rows[2] : rows[3];
      at.x.count = __shfl_sync(0xffffffffu, r.x, row & 31);
      at.x.len = __shfl_sync(0xffffffffu, r.y, row & 31);
      at.x.t0 = __shfl_sync(0xffffffffu, r.z, row & 31);
      at.x.chunks = __shfl_sync(0xffffffffu, r.w, row & 31);
      at.x.pages = kv8_pages(at.x.len);
    }
    at.units = stream_units<KP>(at.x);
    {
      const long long skip = w0 - before;
      const int stream = static_cast<int>(divide(skip, at.units));
      at.unit = static_cast<int>(skip - static_cast<long long>(stream) * at.units);
      at.kvh = at.x.chunks == 1 ? stream : stream / at.x.chunks;
      at.chunk = stream - at.kvh * at.x.chunks;
    }
    Cursor ahead = at;
    auto advance = [&](Cursor& c) {
      if (++c.unit < c.units) return;
      c.unit = 0;
      if (++c.chunk < c.x.chunks) return;
      c.chunk = 0;
      if (++c.kvh < hkv) return;
      c.kvh = 0;
      while (++c.row < a.rows) {
        c.x = kv8_row(a, c.row, group, kCols, tile_from, false);
        c.units = stream_units<KP>(c.x);
        if (c.x.chunks) return;
      }
    };
    // The block table in pieces of 32 entries, one a lane.  With the memory busy
    // a load takes microseconds, so the next piece, the row's first one (for its
    // next stream) and the next row's first one are on their way well ahead, to
    // shared memory, where each lane reads its own entries.
    int* const tables = reinterpret_cast<int*>(ring + S::kTableAt) + lane;  // + 32 k: first, next, next row's
    auto table = [&](int k, int r, int piece) {
      const int i = piece * 32 + lane;
      if (r < a.rows && i < a.max_blocks)
        copy4_async(smem_u32(tables + 32 * k), a.tables + static_cast<size_t>(r) * a.max_blocks + i, true);
    };
    int tab_row = at.row, tab_piece = at.unit * KP >> 5;
    table(0, tab_row, 0);
    table(1, tab_row, tab_piece + 1);
    table(2, tab_row + 1, 0);
    int tab = tab_piece * 32 + lane < a.max_blocks
                  ? __ldg(a.tables + static_cast<size_t>(tab_row) * a.max_blocks + tab_piece * 32 + lane)
                  : -1;
    // The queries of a stream, in shared memory: each lane copies what it reads.
    // They arrive with the stream's first unit, unless an earlier stream's are
    // still there (streams of one unit), and then are loaded when it is their turn.
    int entered = 0, opened = 0, queries_of = 0;  // streams that the loader, the arithmetic, the copy are at
    constexpr int kHalves = S::KW / 2;            // 16-byte pieces of a lane's words
    auto query_of = [&](const Cursor& c, int nt, bool* live) {
      const int col = c.chunk * kCols + nt * 8 + g;
      *live = col < c.x.count * group;
      const int token = *live && c.x.count > 1 ? col / group : 0;
      return a.q + static_cast<size_t>(c.x.t0 + token) * a.ld_q +
             static_cast<size_t>(c.kvh * group + (*live ? col - token * group : 0)) * D + tq * S::KW * 4;
    };
    auto copy_queries = [&](const Cursor& c) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        bool live;
        const __half* src = query_of(c, nt, &live);
#pragma unroll
        for (int s = 0; s < S::KS; ++s)
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            copy16_async(smem_u32(ring + S::kQueriesAt + (((nt * S::KS + s) * kHalves + h) * 32 + lane) * 16),
                         src + s * S::KW * 16 + h * 8, live);
      }
    };
    uint32_t qb[NT][D / 16][2];  // the queries as B fragments, in the keys' order
    auto take_queries = [&](bool copied) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        bool live;
        const __half* src = query_of(at, nt, &live);
#pragma unroll
        for (int s = 0; s < S::KS; ++s)
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (copied)
              v = *reinterpret_cast<const uint4*>(ring + S::kQueriesAt +
                                                  (((nt * S::KS + s) * kHalves + h) * 32 + lane) * 16);
            else if (live)
              v = __ldg(reinterpret_cast<const uint4*>(src + s * S::KW * 16 + h * 8));
            qb[nt][s * S::KW + 2 * h][0] = v.x;
            qb[nt][s * S::KW + 2 * h][1] = v.y;
            qb[nt][s * S::KW + 2 * h + 1][0] = v.z;
            qb[nt][s * S::KW + 2 * h + 1][1] = v.w;
          }
      }
    };
    unsigned have = 0;  // bit stage * KP + j: page j of the stage is there
    auto fetch = [&](int stage, bool first) {
      const int q0 = ahead.unit * KP;
      if (ahead.row != tab_row || q0 >> 5 != tab_piece) {
        copy_wait();
        if (ahead.row != tab_row) {
          if (ahead.row != tab_row + 1) {
            table(2, ahead.row, 0);
            copy_wait();
          }
          tab_row = ahead.row;
          tables[0] = tables[64];
          table(2, tab_row + 1, 0);
        }
        tab_piece = q0 >> 5;
        tab = tables[tab_piece ? 32 : 0];
        if ((tab_piece + 1) * 32 < ahead.x.pages) table(1, tab_row, tab_piece + 1);
      }
      // A page past the last key is none (-2), whatever its entry holds.
      auto page_at = [&](int j) {
        const int b = __shfl_sync(0xffffffffu, tab, (q0 & 31) + j);
        return (q0 + j) * kKv8Page >= ahead.x.len ? -2 : b < 0 || b >= a.cache.blocks ? -1 : b;
      };
      uint64_t* const bar = &full[stage];
      const uint32_t scales = smem_u32(ring + S::kScalesAt + stage * (32 * KP));
      // Scales: eight words a page, four of K and four of V.
      {
        const int b = page_at(lane >> 3 & (KP - 1));
        if (lane < 8 * KP) {
          const size_t page = static_cast<size_t>(max(b, 0)) * hkv + ahead.kvh;
          copy4_async(scales + lane * 4,
                      (lane & 4 ? a.cache.v_scale : a.cache.k_scale) + page * kKv8Page + (lane & 3) * 4,
                      b >= 0);
        }
        if (ahead.unit == 0 && !first) {
          ++entered;
          if (queries_of <= opened) {
            queries_of = entered;
            copy_queries(ahead);
          }
        }
        copy_arrive(bar);
      }
      int b[KP], there = 0;
#pragma unroll
      for (int j = 0; j < KP; ++j) {
        b[j] = page_at(j);
        there |= b[j] >= 0 ? 1 << j : 0;
      }
      have = (have & ~(((1u << KP) - 1u) << (stage * KP))) | static_cast<unsigned>(there) << (stage * KP);
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, __popc(there) * S::kPage);
        uint8_t* to = ring + stage * S::kStage;
#pragma unroll
        for (int j = 0; j < KP; ++j) {
          if (b[j] >= 0) {
            const int page = b[j] * hkv + ahead.kvh;
#pragma unroll
            for (int box = 0; box < D / S::BOX; ++box) {
              tma_load_3d(to + j * S::kPage + box * (16 * S::BOX), &maps.k, bar, box * S::BOX, 0, page);
              tma_load_3d(to + j * S::kPage + 16 * D + box * (16 * S::BOX), &maps.v, bar, box * S::BOX, 0,
                          page);
            }
          } else if (b[j] == -1) {
            atomicOr(a.status, kDevBadIndex);
          }
        }
      }
      advance(ahead);
    };

    int lim[NT][2];              // last key that columns 2t, 2t + 1 see
    int edge;                    // least of them over the stream's columns

    auto open = [&]() {
      const int x0 = at.chunk * kCols, cols = at.x.count * group;
      edge = 0x7fffffff;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int cc = x0 + nt * 8 + 2 * tq + e;
          // Columns beyond the stream's see everything; nothing of them is stored.
          const int tok = at.x.count > 1 ? cc / group : 0;
          lim[nt][e] = cc < cols ? max(-1, at.x.len - at.x.count + tok) : 0x7fffffff;
          edge = min(edge, lim[nt][e]);
          m[nt][e] = kNoReference;
          l[nt][e] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
      }
      edge = __reduce_min_sync(0xffffffffu, edge);
    };

    // Swapped value rows (Layout) are put right by the permutes that pair them.
    const bool swap = S::swapped(g, tq);
    const uint32_t pair_lo = swap ? 0x1504u : 0x5140u, pair_hi = swap ? 0x3726u : 0x7362u;
    const int mine = S::key_of(g);  // key of score row g
    auto multiply = [&](const uint8_t* unit, const uint8_t* scales, unsigned there, int key) {
      float s[MP][NT][2][4];
#pragma unroll
      for (int j = 0; j < MP; ++j) {
        const uint8_t* page = unit + j * S::kPage;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][nt][0][e] = s[j][nt][1][e] = 0.f;
#pragma unroll
        for (int st = 0; st < S::KS; ++st) {
          uint32_t k0[S::KW], k1[S::KW];
          read_words<S::KW>(k0, page + S::k_at(g, tq, st));
          read_words<S::KW>(k1, page + S::k_at(g, tq, st) + 8 * S::BOX);
#pragma unroll
          for (int w = 0; w < S::KW; ++w) {
            const int i = st * S::KW + w;
            const uint32_t a0 = kv8_half2_lo(k0[w]), a2 = kv8_half2_hi(k0[w]);
            const uint32_t a1 = kv8_half2_lo(k1[w]), a3 = kv8_half2_hi(k1[w]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(s[j][nt][i & 1], a0, a1, a2, a3, qb[nt][i][0], qb[nt][i][1]);
          }
        }
      }
      float ks[MP][2];
      uint32_t vb[MP][2];
#pragma unroll
      for (int j = 0; j < MP; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* sc = scales + j * 32 + mine + 8 * h;
          ks[j][h] = __uint_as_float(static_cast<uint32_t>(sc[0]) << 23) * sl2;
          // (A byte 0, which no write leaves, counts as the least normal number.)
          vb[j][h] = max(static_cast<uint32_t>(sc[16]), 1u);
        }
#pragma unroll
      for (int j = 0; j < MP; ++j)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[j][nt][0][e] = (s[j][nt][0][e] + s[j][nt][1][e]) * ks[j][e >> 1];
      const bool at_edge = key + MP * kKv8Page - 1 > edge || there != (1u << MP) - 1u;
      int end[MP];  // first key of the page that is not there
#pragma unroll
      for (int j = 0; j < MP; ++j) end[j] = there >> j & 1u ? at.x.len : 0;
      if (at_edge) {
        // A unit that ends past the last key or some column's, or lacks a page.
#pragma unroll
        for (int j = 0; j < MP; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = key + j * kKv8Page + mine + 8 * h;
            if (k >= end[j]) vb[j][h] = 127u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (k > lim[nt][e] || k >= end[j]) s[j][nt][0][2 * h + e] = -INFINITY;
          }
      }
      float p[MP][NT][4], top;
      auto weigh = [&]() {
        top = 0.f;
#pragma unroll
        for (int j = 0; j < MP; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[j][nt][1][e] = ex2(s[j][nt][0][e] - m[nt][e & 1]);
              p[j][nt][e] = s[j][nt][1][e] * __uint_as_float(vb[j][e >> 1] << 23);
              top = fmaxf(top, p[j][nt][e]);
            }
      };
      weigh();
      if (__any_sync(0xffffffffu, top > kMostWeight)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < MP; ++j)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                mx = fmaxf(mx, s[j][nt][0][2 * h + e] + static_cast<float>(static_cast<int>(vb[j][h]) - 127));
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float to = mx - kTop;
            if (to > m[nt][e]) {
              const float f = ex2(m[nt][e] - to);
              m[nt][e] = to;
              l[nt][e] *= f;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) {
                o[nt][i][e] *= f;
                o[nt][i][e + 2] *= f;
              }
            }
          }
        weigh();
      }
#pragma unroll
      for (int j = 0; j < MP; ++j) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          l[nt][0] += s[j][nt][1][0] + s[j][nt][1][2];
          l[nt][1] += s[j][nt][1][1] + s[j][nt][1][3];
          pb[nt][0] = transpose8x8(half2_bits(p[j][nt][0], p[j][nt][1]));
          pb[nt][1] = transpose8x8(half2_bits(p[j][nt][2], p[j][nt][3]));
        }
        const uint8_t* page = unit + j * S::kPage + 16 * D;
#pragma unroll
        for (int st = 0; st < S::VS; ++st) {
          uint32_t v[4][S::VW];
#pragma unroll
          for (int h = 0; h < 4; ++h)
            read_words<S::VW>(v[h], page + S::v_at(g, tq, h ^ (swap ? 1 : 0), st));
          if (at_edge) {
            // Rows past the last key may hold anything, NaN among it.
#pragma unroll
            for (int h = 0; h < 4; ++h)
              if (key + j * kKv8Page + S::value_key(tq, h ^ (swap ? 1 : 0)) >= end[j]) {
#pragma unroll
                for (int w = 0; w < S::VW; ++w) v[h][w] = 0u;
              }
          }
#pragma unroll
          for (int w = 0; w < S::VW; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t sel = h ? pair_hi : pair_lo;
              const uint32_t lo = __byte_perm(v[0][w], v[1][w], sel);
              const uint32_t hi = __byte_perm(v[2][w], v[3][w], sel);
              const uint32_t a0 = kv8_half2_lo(lo), a1 = kv8_half2_hi(lo);
              const uint32_t a2 = kv8_half2_lo(hi), a3 = kv8_half2_hi(hi);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816(o[nt][(st * S::VW + w) * 2 + h], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
            }
        }
      }
    };

    // Value rows of a unit that some columns see and others do not: a weight of 0
    // would not hide a NaN code.  Such codes make NaN of the sums of the columns
    // that see them, and become zeros, before the unit is multiplied.
    auto hide_nan = [&](uint8_t* unit, unsigned there, int key) {
      const int r0 = max(0, edge + 1 - key), r1 = min(KP * kKv8Page, at.x.len - key);
      auto codes = [&](int r, int byte) {
        return unit + r / kKv8Page * S::kPage + 16 * D + S::byte_at(r % kKv8Page, byte);
      };
      uint32_t nan = 0u;
#pragma unroll 1
      for (int r = r0; r < r1; ++r)
        if (there >> r / kKv8Page & 1u)
          for (int w = lane; w < D / 4; w += 32)
            nan |= kv8_nan_codes(*reinterpret_cast<const uint32_t*>(codes(r, 4 * w)));
      if (!__any_sync(0xffffffffu, nan != 0u)) return;
#pragma unroll 1
      for (int r = r0; r < r1; ++r) {
        if (!(there >> r / kKv8Page & 1u)) continue;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t two = *reinterpret_cast<const uint16_t*>(codes(r, S::dim_of(i, g)));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if ((two >> (e >> 1) * 8 & 0x7fu) == 0x7fu && key + r <= lim[nt][e & 1])
                o[nt][i][e] = __uint_as_float(0x7fffffffu);
        }
        __syncwarp();
        for (int w = lane; w < D / 4; w += 32) {
          uint32_t* const at_w = reinterpret_cast<uint32_t*>(codes(r, 4 * w));
          *at_w &= ~kv8_nan_codes(*at_w);
        }
      }
      fence_proxy_async();  // the slot's next boxes come after these stores
      __syncwarp();
    };

    auto sum_l = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int off = 4; off < 32; off <<= 1)
            l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
    };

    bool starts = at.unit == 0;
    // The stream's sums so far: its output where this warp had it whole, else a piece.
    auto close = [&](bool ends, bool last) {
      sum_l();
      if (starts && ends) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int col = at.chunk * kCols + nt * 8 + 2 * tq;
          const Output c0 = output_of(a, at.x, group, at.kvh, col, l[nt][0]);
          const Output c1 = output_of(a, at.x, group, at.kvh, col + 1, l[nt][1]);
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            store_unit(c0, c1, S::dim_of(i, g),
                       make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]));
        }
        return;
      }
      const int p = warp * 2 + (starts ? 1 : 0);
      float* piece = reinterpret_cast<float*>(ring);
      if (!last) {
        const int slot = __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(&slots_taken, 1) : 0, 0);
        piece = slot < S::kSlots
                    ? reinterpret_cast<float*>(smem + kWarps * S::kWarpBytes + slot * S::kPieceBytes)
                    : reinterpret_cast<float*>(records + gridDim.x) +
                          (static_cast<size_t>(gridDim.x) * 2 + blockIdx.x * kWarps + warp) * S::kPiece;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          *reinterpret_cast<float4*>(piece + ((nt * (D / 16) + i) * 32 + lane) * 4) =
              make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]);
        if (g == 0)
          *reinterpret_cast<float4*>(piece + S::kUnits * 4 + (nt * 8 + 2 * tq) * 2) =
              make_float4(m[nt][0], l[nt][0], m[nt][1], l[nt][1]);
      }
      if (lane == 0) {
        left[p] = make_int4(at.row, at.kvh, at.chunk, (starts ? 1 : 0) | (ends ? 2 : 0));
        left_row[p] = make_int4(at.x.count, at.x.len, at.x.t0, at.units);
        where[p] = piece;
      }
    };

#pragma unroll
    for (int i = 0; i < ST - 1; ++i)
      if (i < n) fetch(i, i == 0);
    take_queries(false);
    open();
    int stage = 0, next = ST - 1;  // of the page at hand, and of the one to fetch
    unsigned phases = 0;           // bit s: parity of stage s's next page
    int i = 0;
    bool fresh = false;  // a stream's first unit, whose queries are not taken yet
    for (; i < n; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phases >> stage & 1u, a.status))) break;
      phases ^= 1u << stage;
      if (fresh) {  // copied queries have arrived with the unit
        take_queries(queries_of == opened);
        fresh = false;
      }
      const unsigned there = have >> (stage * KP) & ((1u << KP) - 1u);
      if (i + ST - 1 < n) fetch(next, false);  // the stage that every lane has left behind
      const bool ends = at.unit == at.units - 1, more = i + 1 < n;
      if (CHUNKS && edge < at.x.len - 1 && (at.unit + 1) * (KP * kKv8Page) - 1 > edge)
        hide_nan(ring + stage * S::kStage, there, at.unit * (KP * kKv8Page));
#pragma unroll 1
      for (int j = 0; j < KP; j += MP)
        if (const unsigned some = there >> j & ((1u << MP) - 1u))
          multiply(ring + stage * S::kStage + j * S::kPage, ring + S::kScalesAt + stage * (32 * KP) + j * 32,
                   some, (at.unit * KP + j) * kKv8Page);
      __syncwarp();
      if (ends || !more) close(ends, !more);
      if (ends && more) {
        advance(at);
        starts = fresh = true;
        ++opened;
        open();
      } else {
        ++at.unit;
      }
      stage = stage + 1 == ST ? 0 : stage + 1;
      next = next + 1 == ST ? 0 : next + 1;
    }
    copy_wait();
    // After a wait that ran out: pages in flight land before the warp goes on (bounded too).
    for (int k = 0; i < n && k < ST - 1 && i + k < n; ++k) {
      const int f = (stage + k) % ST;
      mbar_wait(&full[f], phases >> f & 1u, a.status);
    }
  }
  __syncthreads();

  // Join the warps' pieces: a chain is a run of pieces of one stream.  One warp
  // lists the pieces that there are and where chains begin.
  if (warp == 0) {
    const int4 p = lane < kWarps * 2 ? left[lane] : make_int4(-1, 0, 0, 0);
    const unsigned live = __ballot_sync(0xffffffffu, p.x >= 0);
    const unsigned before = live & ((1u << lane) - 1u);
    const int prev = before ? 31 - __clz(before) : lane;
    const int row = __shfl_sync(0xffffffffu, p.x, prev), kvh = __shfl_sync(0xffffffffu, p.y, prev),
              chunk = __shfl_sync(0xffffffffu, p.z, prev);
    const bool begin = p.x >= 0 && (!before || row != p.x || kvh != p.y || chunk != p.z);
    const unsigned begins = __ballot_sync(0xffffffffu, begin);
    if (p.x >= 0) order[__popc(before)] = lane;
    if (begin) chains[__popc(begins & ((1u << lane) - 1u))] = __popc(before);
    if (lane == 0) {
      chain_count = __popc(begins);
      chains[__popc(begins)] = __popc(live);
    }
  }
  __syncthreads();
  Record rec{-1, 0, 0, 0, 0, 0, {0, 0}};
  for (int ch = 0; ch < chain_count; ++ch) {
    const int k0 = chains[ch], k1 = chains[ch + 1];
    const int4 p = left[order[k0]];
    const bool begins = p.w & 1, ends = left[order[k1 - 1]].w & 2;
    const int4 of = left_row[order[k0]];
    const Kv8Row x{of.x, of.y, of.z, 0, static_cast<int>((static_cast<long long>(of.x) * group + kCols - 1) / kCols)};
    const int kvh = p.y, x0 = p.z * kCols;
    float* dst = reinterpret_cast<float*>(records + gridDim.x) +
                 (static_cast<size_t>(blockIdx.x) * 2 + (begins ? 1 : 0)) * S::kPiece;
    for (int u = threadIdx.x; u < S::kUnits; u += S::kThreads) {
      const int nt = u / (D / 16 * 32), col = nt * 8 + 2 * (u & 3);
      if (x0 + col >= x.count * group) continue;
      auto ml_of = [&](int k) {  // (m, l) of the unit's two columns
        return *reinterpret_cast<const float4*>(where[order[k]] + S::kUnits * 4 + col * 2);
      };
      float2 M = make_float2(kNoReference, kNoReference), L = make_float2(0.f, 0.f);
#pragma unroll 4
      for (int k = k0; k < k1; ++k) {
        const float4 ml = ml_of(k);
        M = make_float2(fmaxf(M.x, ml.x), fmaxf(M.y, ml.z));
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int k = k0; k < k1; ++k) {
        const float4 ml = ml_of(k);
        const float f0 = ex2(ml.x - M.x), f1 = ex2(ml.z - M.y);
        L.x += ml.y * f0;
        L.y += ml.w * f1;
        const float4 v = *reinterpret_cast<const float4*>(where[order[k]] + u * 4);
        acc.x += v.x * f0;
        acc.y += v.y * f1;
        acc.z += v.z * f0;
        acc.w += v.w * f1;
      }
      if (begins && ends) {
        store_unit(output_of(a, x, group, kvh, x0 + col, L.x), output_of(a, x, group, kvh, x0 + col + 1, L.y),
                   S::dim_of((u >> 5) % (D / 16), (u >> 2) & 7), acc);
      } else {
        *reinterpret_cast<float4*>(dst + u * 4) = acc;
        if (u % (D / 16 * 32) < 4)
          *reinterpret_cast<float4*>(dst + S::kUnits * 4 + col * 2) = make_float4(M.x, L.x, M.y, L.y);
      }
    }
    if (!begins && ends) {
      // The stream that earlier CTAs began ends here: the join pass takes it.
      // It is the CTA's first chain, so its row is the CTA's first.
      const long long stream = static_cast<long long>(kvh) * x.chunks + p.z;
      rec = Record{cut_owner(cut, units_before + stream * of.w), kvh, x0, x.count, x.len, x.t0, {0, 0}};
    }
  }
  if (threadIdx.x == 0) records[blockIdx.x] = rec;
  if (beside) griddep_wait();
}

// Joins the pieces of a stream that spans CTAs, in order; one CTA for each CTA
// of the stream pass, with work where that one ended such a stream.  A thread
// sums a unit over a share of the pieces; the shares meet in shared memory.
template <int D, int NT>
struct Join {
  static constexpr int kUnits = Shape<D, NT>::kUnits;
  static constexpr int kShares = kUnits <= 128 ? 4 : kUnits <= 256 ? 2 : 1;
  static constexpr int kThreads = kUnits * kShares;
};
template <int D, int NT>
__global__ void __launch_bounds__(Join<D, NT>::kThreads, 1) kv8_join_kernel(const Kv8AttnArgs a, int group) {
  using S = Shape<D, NT>;
  constexpr int kShares = Join<D, NT>::kShares;
  __shared__ float4 sums[kShares > 1 ? kShares - 1 : 1][S::kUnits];
  __shared__ float4 refs[kShares > 1 ? kShares - 1 : 1][S::kUnits];
  griddep_enter();
  const Record* records = reinterpret_cast<const Record*>(a.workspace);
  const Record rec = records[blockIdx.x];
  const int first = rec.first, end = blockIdx.x;
  if (first < 0 || first >= end) return;
  const float* base = reinterpret_cast<const float*>(records + gridDim.x);
  const int u = threadIdx.x % S::kUnits, share = threadIdx.x / S::kUnits;
  const int col = u / (D / 16 * 32) * 8 + 2 * (u & 3);
  const bool live = rec.x0 + col < rec.count * group;
  // Piece of CTA c: the one it left open for the first, else the one it continued.
  auto piece = [&](int c) {
    return base + (static_cast<size_t>(c) * 2 + (c == first ? 1 : 0)) * S::kPiece;
  };
  float2 M = make_float2(kNoReference, kNoReference), L = make_float2(0.f, 0.f);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& ml, const float4& v) {
    const float m0 = fmaxf(M.x, ml.x), m1 = fmaxf(M.y, ml.z);
    const float f0 = ex2(M.x - m0), f1 = ex2(M.y - m1), g0 = ex2(ml.x - m0), g1 = ex2(ml.z - m1);
    M = make_float2(m0, m1);
    L = make_float2(L.x * f0 + ml.y * g0, L.y * f1 + ml.w * g1);
    acc = make_float4(acc.x * f0 + v.x * g0, acc.y * f1 + v.y * g1, acc.z * f0 + v.z * g0,
                      acc.w * f1 + v.w * g1);
  };
  if (live) {
    // Eight pieces at a time, all their loads in flight together.
    for (int k = first + share; k <= end; k += 8 * kShares) {
      float4 ml[8], v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i * kShares <= end) {
          const float* p = piece(k + i * kShares);
          ml[i] = __ldcg(reinterpret_cast<const float4*>(p + S::kUnits * 4 + col * 2));
          v[i] = __ldcg(reinterpret_cast<const float4*>(p + u * 4));
        }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i * kShares <= end) add(ml[i], v[i]);
    }
  }
  if (kShares > 1) {
    if (share > 0) {
      sums[share - 1][u] = acc;
      refs[share - 1][u] = make_float4(M.x, L.x, M.y, L.y);
    }
    __syncthreads();
  }
  if (share > 0 || !live) return;
#pragma unroll
  for (int p = 0; p < kShares - 1; ++p) add(refs[p][u], sums[p][u]);
  const Kv8Row x{rec.count, rec.len, rec.t0, 0, 0};
  store_unit(output_of(a, x, group, rec.kvh, rec.x0 + col, L.x),
             output_of(a, x, group, rec.kvh, rec.x0 + col + 1, L.y),
             S::dim_of((u >> 5) % (D / 16), (u >> 2) & 7), acc);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
                           cudaSuccess && q == cudaDriverEntryPointSuccess;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(found ? p : nullptr);
  }();
  return fn;
}

bool make_maps(PoolMaps* maps, const Kv8Cache& c, int box) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(c.dim), kKv8Page,
                              static_cast<cuuint64_t>(c.blocks) * c.hkv};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(c.dim), static_cast<cuuint64_t>(c.dim) * kKv8Page};
  const cuuint32_t boxes[3] = {static_cast<cuuint32_t>(box), kKv8Page, 1}, ones[3] = {1, 1, 1};
  const CUtensorMapSwizzle swizzle = box == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : box == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                 : CU_TENSOR_MAP_SWIZZLE_32B;
  for (int v = 0; v < 2; ++v)
    if (fn(v ? &maps->v : &maps->k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, v ? c.v : c.k, dims, strides, boxes,
           ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  return true;
}

int stream_ctas(int sm_count) { return sm_count; }

template <int D, int NT, bool CHUNKS>
cudaError_t launch_stream(const Kv8AttnArgs& a, int tile_from, bool beside, cudaStream_t stream) {
  using S = Shape<D, NT>;
  PoolMaps maps;
  if (!make_maps(&maps, a.cache, S::BOX)) return cudaErrorUnknown;
  static Kv8Configured configured;
  cudaError_t e = configured.once(kv8_stream_kernel<D, NT, CHUNKS>, S::kSmem);
  if (e != cudaSuccess) return e;
  const int group = a.hq / a.cache.hkv;
  const int ctas = stream_ctas(a.sm_count);
  e = launch_dependent(kv8_stream_kernel<D, NT, CHUNKS>, dim3(ctas), dim3(S::kThreads), S::kSmem, stream,
                       maps, a, group, tile_from, beside);
  if (e != cudaSuccess) return e;
  return launch_dependent(kv8_join_kernel<D, NT>, dim3(ctas), dim3(Join<D, NT>::kThreads), 0, stream, a,
                          group);
}

template <int D, int NT>
cudaError_t by_tokens(const Kv8AttnArgs& a, int tile_from, bool beside, cudaStream_t stream) {
  return a.max_row_tokens > 1 ? launch_stream<D, NT, true>(a, tile_from, beside, stream)
                              : launch_stream<D, NT, false>(a, tile_from, beside, stream);
}

// Bytes of a piece: Shape<dim, nt>::kPieceBytes.
size_t piece_bytes(int dim, int nt) {
  return (static_cast<size_t>(dim) / 16 * nt * 32 * 4 + 8 * nt * 2) * sizeof(float);
}

// Rows with this many columns (new tokens x query heads of a group) go to the
// tile pass: half a tile of queries, from where its products beat walking the
// pages once for every 8 columns.  Eight rows on 8 kv heads behind 4000 keys, tile
// and stream pass: 64 columns 43 and 53 us at head size 64, 56 and 71 at 128; 32
// columns 59 and 33, 67 and 41; 64 columns behind 500 keys 18.6 and 18.5, 20.6 and
// 22.3.
constexpr int kTileFrom = 64;

bool with_tiles(int max_row_tokens, int hq, int hkv, int dim) {
  return kv8_tile_supported(dim) &&
         static_cast<long long>(max_row_tokens) * (hq / hkv) >= kTileFrom;
}
// Records, two pieces a CTA, and one a warp (at most 12).
size_t stream_workspace(int dim, int sm_count) {
  return static_cast<size_t>(stream_ctas(sm_count)) *
         (sizeof(Record) + 14 * piece_bytes(dim, dim <= 128 ? 2 : 1));
}

}  // namespace

size_t kv8_attention_workspace(int max_row_tokens, int hq, int hkv, int dim, int sm_count) {
  return stream_workspace(dim, sm_count) +
         (with_tiles(max_row_tokens, hq, hkv, dim) ? kv8_tile_workspace(dim, sm_count) : 0);
}

cudaError_t kv8_attention_launch(const Kv8AttnArgs& a, cudaStream_t stream) {
  if (a.rows == 0 || a.tokens == 0) return cudaSuccess;
  const bool tiles = with_tiles(a.max_row_tokens, a.hq, a.cache.hkv, a.cache.dim);
  const int tile_from = tiles ? kTileFrom : 0x7fffffff;
  float* partial = a.workspace + stream_workspace(a.cache.dim, a.sm_count) / sizeof(float);
  cudaError_t e = cudaSuccess;
  if (tiles) e = kv8_tile_launch(a, tile_from, partial, stream);
  if (e != cudaSuccess) return e;
  // 16 columns a stream where the rows have them; one-token rows of a group of
  // at most 8 heads have not.
  const bool wide = a.hq / a.cache.hkv > 8 || (a.max_row_tokens > 1 && !tiles);
  switch (a.cache.dim) {
#define HB_KV8_DIM(D)                                                                        \
  case D:                                                                                    \
    e = wide && D <= 128 ? by_tokens<D, D <= 128 ? 2 : 1>(a, tile_from, tiles, stream)       \
                         : by_tokens<D, 1>(a, tile_from, tiles, stream);                     \
    break;
    HB_KV8_DIM(32)
    HB_KV8_DIM(64)
    HB_KV8_DIM(96)
    HB_KV8_DIM(128)
    HB_KV8_DIM(160)
    HB_KV8_DIM(192)
    HB_KV8_DIM(224)
    HB_KV8_DIM(256)
#undef HB_KV8_DIM
    default: return cudaErrorInvalidValue;
  }
  if (e == cudaSuccess && tiles) e = kv8_tile_join_launch(a, tile_from, partial, stream);
  return e;
}

}  // namespace hb
