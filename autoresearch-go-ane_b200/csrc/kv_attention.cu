// Attention of new tokens over a paged KV cache (ane_op_kv_attention).
//
// The query heads of a KV head share its keys, so they are rows of one product: row r of a KV head's queries is token r / group,
// head r % group.  Few rows take m16n8k16 on mma.sync: single tokens are bound by the bytes of the cache, and their
// products take a fraction of the time that the operands need to arrive.
//
//   few rows (up to 32 a KV head): a CTA holds 8, 16 or 32 rows; its warps take 16 of every 96 or 128 keys each, with softmax statistics
//     of their own, joined at the end.  No barrier in the loop: every warp waits for its own copies only.
//   many rows: 128 rows a CTA on tcgen05, see kv_attention_tc.cuh.
//
// Keys and values come by cp.async into a ring of stages.  8-bit ones stay 8-bit until they are in registers, where they
// become f16, which holds e4m3 exactly: queries are brought to f16 by a power of two per row, scales of keys go onto the
// scores, scales of values onto the probabilities.
//
// Work is cut on the device, as only the device knows the lengths: all tiles of keys of all (sequence, row tile, KV head) in one
// line, an even share of the line to each CTA of one wave.  What a CTA did of an item that others share goes to the
// workspace, and a second kernel joins the parts in their order, without atomics: the same sums from call to call.
//
// Single tokens, 32 heads of 128 with 8 for keys, 64 sequences of up to 8000 tokens: 208 to 213 us from bf16 pages (6.4 TB/s, about the
// memory's rate), 125 to 132 from 8-bit ones (5.1 to 5.4 TB/s; the floor is 103).  There widening, scaling and exponentials are chains that six
// warps do not cover: 35 % of the issue slots are taken, 17 % of the warps active, no pipe full.  Small calls are launches and dependent reads: one
// sequence of 256 tokens 5.8 us, 32 of 768 8.9, two of 60000 with two KV heads 19.7 (the floor is 7.3).  Tables of more than 768 tokens add the
// launch of the joining kernel, whatever the sequences hold: with 8192, 8.1 and 11.5 us.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "gemm_tc.cuh"
#include "serving.h"

namespace ane {
namespace {

constexpr int kGroup = 16;  // keys of a product
// A row's maximum follows its scores only where they exceed it by more than this (in log2), so that probabilities are below 2^kSlack: most
// keys then need no exchange of maxima and no new factor on what has been summed.
constexpr float kSlack = 8.f;
constexpr float kLowest = 1.17549435e-38f;

// What enters the products with 8-bit values is a probability times its page's scale, in f16.  Scales of the pages that a row sees may be of any
// sizes, so the unit follows the row's own largest such product w, as the exponents' base follows its largest score: outputs are in units of
// 2^(w - 7), f16 numbers 2^15 at most; those down to 2^-21 of the largest stay normal, below 2^-32 they are 0.  What a row does not see has no part
// in it.  With f = 2^((base - w + 7) / 2) a probability takes the factor scale * f * f, in two steps as base - w may be 134; where it leaves fp32,
// above 2^127, the page is one that the row does not see, or whose probabilities are below 2^-112.
constexpr float kNoUnit = -3e38f;  // log2 of the largest product of a row that has seen none
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float unit_factor(float base, float w) { return exp2_fast(fminf(0.5f * (base - w) + 3.5f, 72.f)); }
__device__ __forceinline__ float into_units(float scale, float f) { return fminf(scale * f * f, 0x1p127f); }

struct Attn {
  PagedKv kv;
  Batch batch;
  const bf16* q;
  bf16* out;
  int ld_q, ld_out, group, max_new, window, capacity, stages;
  bool one_tile;   // no sequence has more rows than a tile
  Div by_group, by_page;
  float scale_log2;
  int4* head;      // [CTAs]: the shared item that begins in this CTA: sequence (< 0: none), row tile, KV head, parts
  float2* stats;   // [2 * CTAs][rows]: maximum (log2) and sum of a part
  float* part;     // [2 * CTAs][rows][head_dim]
  int* status;
};

template <int HD, bool F8>
struct Layout {
  static constexpr int ES = F8 ? 1 : 2;
  static constexpr int RB = HD * ES, GB = kGroup * RB, CPR = RB / 16;  // bytes of a row, of 16 rows; 16-byte pieces of a row
  // 8 bits: bytes that a thread loads of K rows at a time, and of V rows
  static constexpr int VK = HD % 64 == 0 ? 16 : HD % 32 == 0 ? 8 : 4, VV = HD % 128 == 0 ? 16 : HD % 64 == 0 ? 8 : HD % 32 == 0 ? 4 : 2;
};

// A form for few rows: the warps share 8 * NB rows and take a part of the keys each, so that no warp is without rows.
// Eight warps, but six where 8-bit pages and 128 * 8 outputs a warp do not fit the 128 registers that two CTAs of eight leave: 64 sequences of
// 8000 tokens with heads of 128 take 125 us with 168 registers, 130 us with 128 and spills (heads of 64 and 12 rows, 8192 tokens: 68 and 73).
// kGroups: times 16 keys that a warp takes at once.  More keys share their softmax's maximum, exchanges and loop, fewer leave the ring room
// for more stages.
template <int HD_, bool F8_, int NB_>
struct Form {
  static constexpr int HD = HD_, NB = NB_, kWarps = F8_ && HD_ * NB_ == 128 && NB_ <= 2 ? 6 : 8;
  static constexpr bool F8 = F8_, kSplit = true;
  using L = Layout<HD, F8>;
  static constexpr int kGroups = L::RB <= 64 && NB == 1 ? 2 : 1;
  // groups of 16 keys of a tile that a warp fetches; the ring has to hold the warps' outputs
  static constexpr int kLoads = kGroups * 3 * L::ES < NB ? 2 : kGroups;
  static constexpr int kThreads = 32 * kWarps, kTile = kGroup * kWarps * kLoads, kRows = 8 * NB;
  static constexpr int kStage = kWarps * kLoads * 2 * L::GB;
  // resident CTAs wanted: registers for outputs and queries decide
  static constexpr int kRegs = NB * (HD / 16 * 6 + 16);
  static constexpr int kCtas = kRegs > 80 || 3 * kStage > 108 * 1024 ? 1 : 2;
  static constexpr int kRoom = 224 * 1024 / kCtas - 3 * 1024, kFit = kRoom / kStage;
  static constexpr int kStages = kFit < 3 ? 3 : kFit > 6 ? 6 : kFit;
  static constexpr int kMost = 216 * 1024 / kStage, kDeep = kMost > 8 ? 8 : kMost < kStages ? kStages : kMost;  // where a CTA has an SM to itself
  static constexpr int kMostSmem = kDeep * kStage;
  static_assert(kWarps * kRows * HD * 4 <= 3 * kStage, "the warps' outputs are joined in the ring");
  // Tiles of an item that are not worth sharing (joining parts takes a second kernel), the least share of one that is shared, and what another
  // item costs a CTA, as 768, 256 and 768 keys.  us at half and at twice as many beside it, tables as long as the sequences (12 heads of 64 bf16;
  // A with 4 for keys; B 32 heads of 128 with 8, 8 bits):
  //   alone    one of 500 9.3 7.7 7.7, of 1500 9.4 9.4 12.0; A 32 of 600 11.4 8.4 8.4, of 1500 14.7 14.7 12.7; B 4 of 700 11.6 12.9 12.9,
  //            of 1500 13.5 13.5 18.2: few sequences would rather have less, many more
  //   least    one of 1000 9.6 9.4 10.4, of 1500 10.2 9.4 10.4, of 3000 11.1 11.1 10.6; B 4 of 1000 12.0 12.0 13.4
  //   restart  (256, 768, 1536) A 32 of 1500 15.5 14.7 14.7; B 16 of 4000 28.6 28.6 34.3, 12 of 8000 36.6 36.6 41.2
  static constexpr int kAlone = 768 / kTile, kLeast = 256 / kTile;
  static constexpr int kRestart = 768 / kTile;
};

// Where 16-byte piece c of a row lies within 16 rows, so that what is read together lies in different banks.  bf16: the same piece of eight
// rows (ldmatrix).  8 bits: a thread (g, j) reads row g of K at pieces j.. and row 2 j (+ 1, 8, 9) of V at pieces g...
template <int CPR, bool F8, bool V>
__device__ __forceinline__ int piece(int row, int c) {
  if (!F8) {
    if (CPR % 8 == 0) return row * CPR + (c ^ (row & 7));
    if (CPR % 4 == 0) return row * CPR + (c ^ (row >> 1 & 3));
    return row * CPR + (c ^ (row >> 2 & 1));
  }
  if (CPR % 8 == 0) return row * CPR + (c ^ (V ? row & 7 : (row & 1) << 2));
  if (CPR == 4) return (row >> 1) * 8 + ((((row & 1) << 2) | c) ^ ((row >> 1 & 3) << 1));
  if (CPR == 2) return (row >> 2) * 8 + ((((row & 3) << 1) | c) ^ ((row >> 2 & 1) << 1));
  return row * CPR + c;
}
template <bool kTrans>
__device__ __forceinline__ void load_matrices(uint32_t at, uint32_t (&a)[4]) {
  if (kTrans) asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(at));
  else asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(at));
}

template <bool F8>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F8)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same onto zeros.
template <bool F8>
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F8)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void e4m3_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {  // the low and the high two bytes
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
template <bool F8>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  if (F8) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void copy_16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int B>
__device__ __forceinline__ void lds(const char* p, uint32_t* w) {  // B bytes
  if (B == 16) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else if (B == 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x; w[1] = u.y;
  } else if (B == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
}

// ---- cutting the work ---------------------------------------------------------------------------------------------------------
// An item is a (sequence, tile of kRows rows, KV head); its key tiles are those that one of its rows sees.
struct Range {
  int lo, hi;  // positions that some row of the tile sees
  template <class F>
  __device__ int t0() const { return lo / F::kTile; }
  template <class F>
  __device__ int tiles() const { return (hi - 1) / F::kTile - lo / F::kTile + 1; }
};
// The positions that a tile of rows sees; with one tile for all rows of a sequence this takes no quotients.
template <class F>
__device__ __forceinline__ Range range_of(const Attn& a, const Span& s, int mt) {
  if (F::kSplit && a.one_tile) return {a.window ? max(0, s.pos + 1 - a.window) : 0, s.pos + s.n};
  const int t_last = min(s.n - 1, a.by_group((mt + 1) * F::kRows - 1));
  return {a.window ? max(0, s.pos + a.by_group(mt * F::kRows) + 1 - a.window) : 0, s.pos + t_last + 1};
}
template <class F>
__device__ __forceinline__ int row_tiles(const Attn& a, const Span& s) {
  return F::kSplit && a.one_tile ? (s.n > 0 ? 1 : 0) : (s.n * a.group + F::kRows - 1) / F::kRows;
}

// An item, and the tiles of it that are this CTA's.
struct Item {
  int b, mt, head, off;  // off: the first of its tiles that is
  Span s;
  Range range;
  int tiles, count;  // all tiles, this CTA's
  int unit;          // of its first tile here, in the line
};

// How the line of all tiles is cut.  Whole items to a CTA where all are short; one piece of at most `share` tiles of one item to each CTA where
// that makes the largest share little larger than an even one, since another item costs a CTA a new start; else even shares.
enum Cut { kWhole, kPieces, kEven };
// The host has made sure that there are less than 2^31 units where no row belongs to two sequences.
struct Plan {
  int first, last;  // this CTA's units of the line: items, pieces or tiles
  int share;        // tiles (kWhole: items) of a CTA
  int cut;
};

template <class F>
__device__ __forceinline__ void measure(const Attn& a, const Plan& p, Item& it) {
  it.range = range_of<F>(a, it.s, it.mt);
  it.tiles = it.range.template tiles<F>();
  it.count = p.cut == kWhole ? it.tiles : p.cut == kPieces ? min(it.tiles - it.off, p.share) : min(it.tiles - it.off, p.last - it.unit);
}
template <class F>
__device__ __forceinline__ bool next_item(const Attn& a, const Plan& p, Item& it) {
  it.unit += p.cut == kEven ? it.count : 1;
  if (it.unit >= p.last) return false;
  it.off = 0;
  if (++it.head == a.kv.kv_heads) {
    it.head = 0;
    ++it.mt;
    while (it.mt >= row_tiles<F>(a, it.s)) {
      it.mt = 0;
      it.s = span_of(a.batch, ++it.b, a.capacity, a.max_new, a.status);
    }
  }
  measure<F>(a, p, it);
  return true;
}

// n / d rounded up for n + d < 2^31, d > 0: a quotient of floats, put right by one step at most (its error is below 2^-22 of it, so
// from 2^21 on an exact one).
__device__ __forceinline__ int quotient_up(int n, int d) {
  if (n >= 1 << 21) return (int)((uint32_t)(n + d - 1) / (uint32_t)d);
  int q = (int)__fdividef((float)n, (float)d);
  if (q * d < n) ++q;
  if (q * d < n) ++q;
  if ((q - 1) * d >= n && q > 0) --q;
  return q;
}

template <class F>
__device__ __forceinline__ Plan make_plan(const Attn& a, Item& it) {
  constexpr int kWarps = F::kWarps, kThreads = F::kThreads;
  __shared__ int3 all[kWarps];
  __shared__ int sums[kWarps];
  __shared__ int4 at, span;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // A thread has some sequences, or, where those are few and have many tiles of rows, a part of one's: 2^split threads a sequence.
  const int per = (a.batch.n_seq + kThreads - 1) / kThreads;
  const int split = per > 1 || (F::kSplit && a.one_tile) ? 0 : 31 - __clz(kThreads / a.batch.n_seq), part = tid & ((1 << split) - 1);
  const int b0 = min((tid >> split) * per, a.batch.n_seq), b1 = min(b0 + per, a.batch.n_seq);
  Span s = {0, 0, 0};  // of the thread's only sequence, mostly
  int longest = 0;     // INT_MIN: starts fall
  // what(tiles of an item) of all items of a KV head of the thread's sequences, until it says stop
  auto each = [&](auto what) {
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      if (per > 1) s = span_of(a.batch, b, a.capacity, a.max_new, a.status);
      if (s.n < 0) {
        longest = INT_MIN;
        return;
      }
      const int mts = row_tiles<F>(a, s), each_mts = (mts + (1 << split) - 1) >> split, mt1 = min(mts, (part + 1) * each_mts);
#pragma unroll 1
      for (int mt = part * each_mts; mt < mt1; ++mt)
        if (what(b, mt, range_of<F>(a, s, mt).template tiles<F>())) return;
    }
  };
  if (per == 1 && b0 < b1) s = span_of(a.batch, b0, a.capacity, a.max_new, a.status);
  int items = 0, tiles = 0;
  each([&](int, int, int t) {
    ++items;
    tiles += t;
    longest = max(longest, t);
    return false;
  });
  items = __reduce_add_sync(0xffffffffu, items);
  tiles = __reduce_add_sync(0xffffffffu, tiles);
  longest = (int)__reduce_max_sync(0xffffffffu, (uint32_t)longest);
  if (lane == 0) all[warp] = make_int3(items, tiles, longest);
  if (tid == 0) at = make_int4(-1, 0, 0, 0);
  __syncthreads();
  items = tiles = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    items += all[w].x;
    tiles += all[w].y;
    longest = (int)max((uint32_t)longest, (uint32_t)all[w].z);
  }
  Plan p = {};
  if (longest < 0) {  // reported; rows may belong to several sequences, and nothing bounds the line's length then
    it.b = -1;
    return p;
  }
  items *= a.kv.kv_heads;
  tiles *= a.kv.kv_heads;
  const int ctas = gridDim.x;
  p.cut = kWhole;
  p.share = quotient_up(items, ctas);
  if (longest > F::kAlone) {
    const int even = max(quotient_up(tiles, ctas), F::kLeast);
    p.cut = kEven;
    p.share = even;
    if constexpr (F::kSplit) {
      // at most tiles / share + items pieces
      const int pieces = items < ctas ? max(quotient_up(tiles, ctas - items), even) : INT32_MAX;
      if (pieces <= even + F::kRestart) {
        p.cut = kPieces;
        p.share = pieces;
      }
    }
  }
  auto weight = [&](int t) { return p.cut == kWhole ? 1 : p.cut == kPieces ? quotient_up(t, p.share) : t; };
  int mine = 0;
  each([&](int, int, int t) {
    mine += weight(t);
    return false;
  });
  mine *= a.kv.kv_heads;
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += t;
  }
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  int units = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    units += sums[w];
  }
  before -= mine;
  const int step = p.cut == kPieces ? 1 : p.share;
  p.first = (int)min((long long)step * blockIdx.x, (long long)units);
  p.last = min(step, units - p.first) + p.first;
  if (p.first < p.last && p.first >= before && p.first - before < mine) {
    int rest = p.first - before;
    each([&](int b, int mt, int t) {
      const int one = weight(t);
      if (rest >= one * a.kv.kv_heads) {
        rest -= one * a.kv.kv_heads;
        return false;
      }
      const int head = (int)((uint32_t)rest / (uint32_t)one), unit = rest - head * one;
      at = make_int4(b, mt, head, p.cut == kPieces ? unit * p.share : p.cut == kEven ? unit : 0);
      span = make_int4(s.row, s.n, s.pos, 0);
      return true;
    });
  }
  __syncthreads();
  const int4 from = at, of = span;
  it.b = from.x;
  it.mt = from.y;
  it.head = from.z;
  it.off = from.w;
  it.s = {of.x, of.y, of.z};
  it.unit = p.first;
  if (it.b >= 0) measure<F>(a, p, it);
  return p;
}

// ---- the products of 16 keys and a warp's rows ----------------------------------------------------------------------------------
// Scores as K q^T and outputs as V^T p^T: keys, and then columns of the output, are the 16 rows of a product, queries its 8 columns, so
// that a group of up to 8 heads takes half of the products, registers and softmax arithmetic of the other way round.
template <int HD, bool F8, int NB>
struct Rows {  // 8 * NB rows of queries
  uint32_t q[NB][HD / 16][2];  // right operands: the thread's row g of each eight
  float o[NB][HD / 16][4];     // columns of the output column(2 y, g) and column(2 y + 1, g), for rows 2 j and 2 j + 1
  // rows 2 j and 2 j + 1: exponents' base, which is the maximum at the time, the score from which on it is renewed (-infinity: none yet), the sum,
  // and what brings products to scores in log2
  float base[NB][2], limit[NB][2], l[NB][2], mult[NB][2];
  int pos[NB][2];                         // their positions; -1: no such row
  float w[NB][2], f[NB][2];               // 8 bits: log2 of the largest probability times scale, and what makes f16 numbers of such products
};

// The power of two that brings a row's largest value to [256, 512): f16 is exact for what is above 2^-22 of it.
__device__ __forceinline__ float to_f16_range(float top) {
  const int e = min(max((int)(__float_as_uint(top) >> 23), 16), 254);
  return top > 0.f && top < INFINITY ? __uint_as_float((uint32_t)min(254 + 8 - e, 254) << 23) : 1.f;
}
// Where four columns of a part's row lie: rows next to one another where a thread has a whole one, columns next to one another else.
template <class F>
__device__ __forceinline__ float4* part_at(const Attn& a, size_t slot, int row, int col4) {
  return reinterpret_cast<float4*>(a.part) + (F::kSplit ? (slot * F::kRows + row) * (F::HD / 4) + col4 : (slot * (F::HD / 4) + col4) * F::kRows + row);
}
template <bool F16>
__device__ __forceinline__ float from_16(uint16_t w) {
  return F16 ? __half2float(__ushort_as_half(w)) : __uint_as_float((uint32_t)w << 16);
}
// Parts of an item that begins in this CTA and does not end there: its own, and one of each of the next ones until the item ends.
__device__ __forceinline__ void mark_shared(const Attn& a, const Plan& plan, const Item& it) {
  const uint32_t last = plan.cut == kPieces ? blockIdx.x + (uint32_t)(it.tiles - 1) / (uint32_t)plan.share
                                            : (uint32_t)(it.unit + it.tiles - 1) / (uint32_t)plan.share;
  a.head[blockIdx.x] = make_int4(it.b, it.mt, it.head, (int)(last - blockIdx.x) + 1);
}

template <int HD, int NB>
struct RawRows {
  uint2 w[NB][HD / 16];  // the thread's row g of each eight
};
template <int HD, bool F8, int NB>
__device__ __forceinline__ void fetch_queries(const Attn& a, const Item& it, int rows0, RawRows<HD, NB>& raw) {
  using L = Layout<HD, F8>;
  const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3, n_rows = it.s.n * a.group;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = rows0 + 8 * n + g;
    const bool there = row < n_rows;
    const int t = there ? a.by_group(row) : 0, hd = there ? row - t * a.group : 0;
    const bf16* q = a.q + (size_t)(it.s.row + t) * a.ld_q + (size_t)(it.head * a.group + hd) * HD;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
      // 8 bits: the four elements that word i of the thread's bytes of a K row meets
      const int at = F8 ? L::VK * j + i / (L::VK / 4) * 4 * L::VK + i % (L::VK / 4) * 4 : 16 * i + 2 * j;
      if (!there) raw.w[n][i] = make_uint2(0, 0);
      else if (F8) raw.w[n][i] = *reinterpret_cast<const uint2*>(q + at);
      else raw.w[n][i] = make_uint2(*reinterpret_cast<const uint32_t*>(q + at), *reinterpret_cast<const uint32_t*>(q + at + 8));
    }
  }
}

template <int HD, bool F8, int NB>
__device__ __forceinline__ void begin_rows(const Attn& a, const Item& it, int rows0, const RawRows<HD, NB>& raw, Rows<HD, F8, NB>& r) {
  const int lane = threadIdx.x & 31, j = lane & 3, n_rows = it.s.n * a.group;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    float mult = a.scale_log2;
    if (F8) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        const uint2 w = raw.w[n][i];
        top = fmaxf(top, fmaxf(fmaxf(fabsf(__uint_as_float(w.x << 16)), fabsf(__uint_as_float(w.x & 0xffff0000u))),
                               fmaxf(fabsf(__uint_as_float(w.y << 16)), fabsf(__uint_as_float(w.y & 0xffff0000u)))));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float by = to_f16_range(top);
      mult /= by;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        const uint2 w = raw.w[n][i];
        r.q[n][i][0] = pack<true>(__uint_as_float(w.x << 16) * by, __uint_as_float(w.x & 0xffff0000u) * by);
        r.q[n][i][1] = pack<true>(__uint_as_float(w.y << 16) * by, __uint_as_float(w.y & 0xffff0000u) * by);
      }
    } else {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        r.q[n][i][0] = raw.w[n][i].x;
        r.q[n][i][1] = raw.w[n][i].y;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int mine = rows0 + 8 * n + 2 * j + h;
      r.pos[n][h] = mine < n_rows ? it.s.pos + a.by_group(mine) : -1;
      r.base[n][h] = 0.f;
      r.limit[n][h] = -INFINITY;
      r.l[n][h] = 0.f;
      if (F8) {
        r.w[n][h] = kNoUnit;
        r.f[n][h] = unit_factor(0.f, kNoUnit);
      }
      r.mult[n][h] = F8 ? __shfl_sync(0xffffffffu, mult, (2 * j + h) * 4) : mult;
    }
#pragma unroll
    for (int y = 0; y < HD / 16; ++y) r.o[n][y][0] = r.o[n][y][1] = r.o[n][y][2] = r.o[n][y][3] = 0.f;
  }
}

// Whether one of a word's values is infinite or NaN.
template <bool F8>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  if (F8) return (w & 0x7fu) == 0x7fu || (w >> 8 & 0x7fu) == 0x7fu || (w >> 16 & 0x7fu) == 0x7fu || (w >> 24 & 0x7fu) == 0x7fu;
  return (w & 0x7f80u) == 0x7f80u || (w >> 16 & 0x7f80u) == 0x7f80u;
}

// Column of the output that element x of a thread's products with V stands for in the threads with this g.
template <int HD, bool F8>
__device__ __forceinline__ int column(int x, int g) {
  using L = Layout<HD, F8>;
  constexpr int EV = L::VV;
  return F8 ? x / EV * 8 * EV + g * EV + x % EV : 8 * x + g;
}
__device__ __forceinline__ uint32_t transposed(uint32_t w) {  // of an 8 x 8 matrix of 16-bit values
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
  return r;
}

// KG * 16 keys at positions key0.. against the warp's rows; group i of them lies at ring + i * 2 * GB.  `checked`: some row does not
// see some key.
template <int HD, bool F8, int NB, int KG>
__device__ __forceinline__ void take_keys(const char* ring, const float4* scales, int key0, bool checked, int window, Rows<HD, F8, NB>& r) {
  using L = Layout<HD, F8>;
  constexpr int kChains = NB == 1 ? 2 : 1;
  constexpr bool kRest = !F8;  // probabilities have one
  const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  float s[KG][NB][4];  // keys g (0, 1) and g + 8 (2, 3), rows 2 j and 2 j + 1
  float4 scale[KG];    // of keys, of values, log2 of the latter
#pragma unroll
  for (int k = 0; k < KG; ++k) {
    const char* ks = ring + k * 2 * L::GB;
    scale[k] = F8 ? scales[k] : make_float4(1.f, 1.f, 0.f, 0.f);
    float even[NB][4];  // a second chain of products, half as long each
    auto products = [&](const uint32_t (&a)[4], int step) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float(&d)[4] = kChains == 2 && step % 2 == 1 ? even[n] : s[k][n];
        if (step < kChains) mma_first<F8>(d, a, r.q[n][step][0], r.q[n][step][1]);
        else mma<F8>(d, a, r.q[n][step][0], r.q[n][step][1]);
      }
    };
    if (F8) {
#pragma unroll
      for (int i = 0; i < L::RB / (4 * L::VK); ++i) {
        const int byte = L::VK * j + 4 * L::VK * i;
        uint32_t u[L::VK / 4], w[L::VK / 4];  // of keys g and g + 8
        lds<L::VK>(ks + piece<L::CPR, F8, false>(g, byte >> 4) * 16 + (byte & 15), u);
        lds<L::VK>(ks + piece<L::CPR, F8, false>(8 + g, byte >> 4) * 16 + (byte & 15), w);
#pragma unroll
        for (int x = 0; x < L::VK / 4; ++x) {
          uint32_t a[4];
          e4m3_to_f16(u[x], a[0], a[2]);
          e4m3_to_f16(w[x], a[1], a[3]);
          products(a, i * (L::VK / 4) + x);
        }
      }
    } else {
      const uint32_t at = smem_u32(ks);
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        uint32_t a[4];
        load_matrices<false>(at + piece<L::CPR, F8, false>(lane & 15, 2 * i + (lane >> 4)) * 16, a);
        products(a, i);
      }
    }
    if (kChains == 2) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[k][n][i] += even[n][i];
    }
  }
  if (checked) {
#pragma unroll
    for (int k = 0; k < KG; ++k)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + kGroup * k + g + 8 * (i >> 1), pos = r.pos[n][i & 1];
          if (key > pos || (window && key <= pos - window)) s[k][n][i] = -INFINITY;
        }
  }
  uint32_t p[KG][NB][2], rest[kRest ? KG : 1][NB][2];
  bool above = false;
  float mult[KG][NB][2];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = -INFINITY, most = -INFINITY;
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        mult[k][n][h] = F8 ? fmaxf(r.mult[n][h] * scale[k].x, kLowest) : r.mult[n][h];  // not 0, so that hidden scores stay -infinity
        const float high = fmaxf(s[k][n][h], s[k][n][2 + h]) * mult[k][n][h];
        top = fmaxf(top, high);
        if (F8) most = fmaxf(most, high + scale[k].z);
      }
      above |= top > r.limit[n][h] || (F8 && most > r.w[n][h] + kSlack);
    }
  if (__any_sync(0xffffffffu, above)) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float fix[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = -INFINITY, most = -INFINITY;
#pragma unroll
        for (int k = 0; k < KG; ++k) {
          const float high = fmaxf(s[k][n][h], s[k][n][2 + h]) * mult[k][n][h];
          top = fmaxf(top, high);
          if (F8) most = fmaxf(most, high + scale[k].z);
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (F8) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        const bool none = r.limit[n][h] == -INFINITY;
        const float base = none ? (top == -INFINITY ? 0.f : top) : fmaxf(top, r.base[n][h]);
        fix[h] = none ? 1.f : exp2_fast(r.base[n][h] - base);  // sums are still 0 then
        r.base[n][h] = base;
        r.limit[n][h] = none && top == -INFINITY ? -INFINITY : base + kSlack;
        r.l[n][h] *= fix[h];
        if (F8) {
          const float w = fmaxf(most, r.w[n][h]);
          fix[h] = exp2_fast(r.w[n][h] - w);
          r.w[n][h] = w;
          r.f[n][h] = unit_factor(base, w);
        }
      }
#pragma unroll
      for (int y = 0; y < HD / 16; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) r.o[n][y][i] *= fix[i & 1];
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        s[k][n][h] = exp2_fast(fmaf(s[k][n][h], mult[k][n][h], -r.base[n][h]));
        s[k][n][2 + h] = exp2_fast(fmaf(s[k][n][2 + h], mult[k][n][h], -r.base[n][h]));
        sum += s[k][n][h] + s[k][n][2 + h];
      }
      r.l[n][h] += sum;  // the thread's own keys; joined at the end
    }
    // Probabilities in 16 bits.  f16 is finer than the output's type.  bf16 is as coarse, and errors of both add up to 1.4 times the output's own:
    // what rounding has left of it is added.
#pragma unroll
    for (int k = 0; k < KG; ++k) {
      if (F8) {
        const float into[2] = {into_units(scale[k].y, r.f[n][0]), into_units(scale[k].y, r.f[n][1])};
#pragma unroll
        for (int i = 0; i < 4; ++i) s[k][n][i] *= into[i & 1];
      }
      p[k][n][0] = transposed(pack<F8>(s[k][n][0], s[k][n][1]));
      p[k][n][1] = transposed(pack<F8>(s[k][n][2], s[k][n][3]));
      if constexpr (kRest) {
        float left[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) left[i] = s[k][n][i] - __bfloat162float(__float2bfloat16_rn(s[k][n][i]));
        rest[k][n][0] = transposed(pack<F8>(left[0], left[1]));
        rest[k][n][1] = transposed(pack<F8>(left[2], left[3]));
      }
    }
  }
  if (checked) {
    // a value that is infinite or NaN must not reach rows that do not see its key, and 0 * NaN is NaN
    bool odd = false;
#pragma unroll 1
    for (int k = 0; k < KG; ++k)
#pragma unroll 1
      for (int i = lane; i < L::GB / 4; i += 32)
        odd |= not_finite<F8>(*reinterpret_cast<const uint32_t*>(ring + k * 2 * L::GB + L::GB + 4 * i));
    if (__any_sync(0xffffffffu, odd)) {
      // one product after the other, unseen ones left out
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const char* vs = ring + k * 2 * L::GB + L::GB;
#pragma unroll 1
        for (int key = 0; key < kGroup; ++key) {
          const int from = (key & 7) * 4 + j, at_key = key0 + kGroup * k + key;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const float w0 = __shfl_sync(0xffffffffu, key < 8 ? s[k][n][0] : s[k][n][2], from);
            const float w1 = __shfl_sync(0xffffffffu, key < 8 ? s[k][n][1] : s[k][n][3], from);
            const bool see0 = at_key <= r.pos[n][0] && !(window && at_key <= r.pos[n][0] - window);
            const bool see1 = at_key <= r.pos[n][1] && !(window && at_key <= r.pos[n][1] - window);
#pragma unroll
            for (int x = 0; x < HD / 8; ++x) {
              const int byte = column<HD, F8>(x, g) * L::ES;
              const char* at = vs + piece<L::CPR, F8, true>(key, byte >> 4) * 16 + (byte & 15);
              const float v = F8 ? __half2float(__half(__nv_cvt_fp8_to_halfraw(*reinterpret_cast<const unsigned char*>(at), __NV_E4M3)))
                                 : __uint_as_float((uint32_t)*reinterpret_cast<const unsigned short*>(at) << 16);
              if (see0) r.o[n][x >> 1][2 * (x & 1)] += w0 * v;
              if (see1) r.o[n][x >> 1][2 * (x & 1) + 1] += w1 * v;
            }
          }
        }
      }
      return;
    }
  }
  constexpr int EV = L::VV, WV = L::VV >= 4 ? L::VV / 4 : 1;
#pragma unroll
  for (int k = 0; k < KG; ++k) {
    const char* vs = ring + k * 2 * L::GB + L::GB;
    if (!F8) {
      const uint32_t at = smem_u32(vs);
#pragma unroll
      for (int y = 0; y < HD / 16; ++y) {
        uint32_t v[4];
        load_matrices<true>(at + piece<L::CPR, F8, true>((lane & 7) + (lane >> 4) * 8, 2 * y + (lane >> 3 & 1)) * 16, v);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          mma<false>(r.o[n][y], v, p[k][n][0], p[k][n][1]);
          if constexpr (kRest) mma<false>(r.o[n][y], v, rest[k][n][0], rest[k][n][1]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < (F8 ? L::RB / (8 * L::VV) : 0); ++i) {
      const int byte = L::VV * g + 8 * L::VV * i;
      uint32_t w[4][WV];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int row = 2 * j + (m & 1) + 8 * (m >> 1);
        lds<L::VV>(vs + piece<L::CPR, F8, true>(row, byte >> 4) * 16 + (byte & 15), w[m]);
      }
#pragma unroll
      for (int x = 0; x < WV; ++x) {
        // two columns of two keys in a word: (key, key + 1) of one column, then of the next
        uint32_t v[4];
        e4m3_to_f16(__byte_perm(w[0][x], w[1][x], 0x5140), v[0], v[1]);
        e4m3_to_f16(__byte_perm(w[2][x], w[3][x], 0x5140), v[2], v[3]);
        const int y = (i * EV + 4 * x) / 2;
#pragma unroll
        for (int n = 0; n < NB; ++n) mma<true>(r.o[n][y], v, p[k][n][0], p[k][n][1]);
        if (EV > 2) {
          e4m3_to_f16(__byte_perm(w[0][x], w[1][x], 0x7362), v[0], v[1]);
          e4m3_to_f16(__byte_perm(w[2][x], w[3][x], 0x7362), v[2], v[3]);
#pragma unroll
          for (int n = 0; n < NB; ++n) mma<true>(r.o[n][y + (EV > 2)], v, p[k][n][0], p[k][n][1]);
        }
      }
    }
  }
}

// ---- the kernel -------------------------------------------------------------------------------------------------------------------
template <class F>
__global__ void __launch_bounds__(F::kThreads, F::kCtas) kv_attention_kernel(const Attn a) {
  constexpr int HD = F::HD, NB = F::NB;
  constexpr bool F8 = F::F8;
  using L = Layout<HD, F8>;
  constexpr int kRows = F::kRows, kWarps = F::kWarps, kLoads = F::kLoads, kTile = F::kTile, kThreads = F::kThreads;
  extern __shared__ __align__(128) char ring[];
  __shared__ float4 scales[F::kDeep][kWarps * kLoads];
  __shared__ float join_m[kWarps][8 * NB], join_l[kWarps][8 * NB];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j = lane & 3;
  Item it;
  const Plan plan = make_plan<F>(a, it);
  if (tid == 0) a.head[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (it.b < 0) {
    pdl_trigger();
    return;
  }
  const uint32_t ring_at = smem_u32(ring);
  RawRows<HD, NB> raw;
  fetch_queries<HD, F8, NB>(a, it, it.mt * kRows, raw);

  Rows<HD, F8, NB> r;
  for (;;) {
    const int rows0 = it.mt * kRows, tile0 = it.range.template t0<F>() + it.off;
    // copies of tile0 + i, i < count: kLoads groups of 16 keys of each by this warp.  Where they lie (in 16-byte pieces; all ones:
    // nowhere) and their scales, of the next 32 groups, are in its lanes.
    constexpr int kAhead = 32 / kLoads;  // tiles
    uint32_t my_at = 0xffffffffu;
    float my_k = 0.f, my_v = 0.f;
    auto look_up = [&](int i) {
      const int key = (tile0 + i + lane / kLoads) * kTile + (warp * kLoads + lane % kLoads) * kGroup;
      my_at = 0xffffffffu;
      my_k = my_v = 0.f;
      if (i + lane / kLoads < it.count && key < it.range.hi && key + kGroup > it.range.lo) {
        const int slot = a.by_page(key), p = a.kv.table[(size_t)it.b * a.kv.table_pitch + slot];
        if (p < 0 || p >= a.kv.n_pages) {
          atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
        } else {
          my_at = (uint32_t)(((unsigned long long)p * a.kv.page_stride +
                              ((size_t)it.head * a.kv.page_size + key - slot * a.kv.page_size) * HD) * L::ES >> 4);
          if (F8) {
            my_k = a.kv.k_scale[(size_t)p * a.kv.kv_heads + it.head];
            my_v = a.kv.v_scale[(size_t)p * a.kv.kv_heads + it.head];
          }
        }
      }
    };
    int to_stage = 0, from_stage = 0;
    auto copy = [&](int i) {
      if (i < it.count) {
        if (i % kAhead == 0) look_up(i);
        const char* none = reinterpret_cast<const char*>(a.kv.k);
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
          const uint32_t at = __shfl_sync(0xffffffffu, my_at, i % kAhead * kLoads + n);
          const int key0 = (tile0 + i) * kTile + (warp * kLoads + n) * kGroup;
          const uint32_t to = ring_at + to_stage * F::kStage + (warp * kLoads + n) * 2 * L::GB;
          const char *k = none + (size_t)at * 16, *v = reinterpret_cast<const char*>(a.kv.v) + (size_t)at * 16;
          if (key0 >= it.range.lo && key0 + kGroup <= it.range.hi && at != 0xffffffffu) {
#pragma unroll
            for (int c0 = 0; c0 < L::GB / 16; c0 += 32) {
              const int c = c0 + lane;
              if ((L::GB / 16) % 32 == 0 || c < L::GB / 16) {
                const int row = c / L::CPR, in_row = c % L::CPR;
                copy_16(to + piece<L::CPR, F8, false>(row, in_row) * 16, k + c * 16, true);
                copy_16(to + L::GB + piece<L::CPR, F8, true>(row, in_row) * 16, v + c * 16, true);
              }
            }
          } else {
            // rows that no query sees are filled with zeros: whatever lies there must not count
            const int lo = it.range.lo - key0, hi = at == 0xffffffffu ? 0 : it.range.hi - key0;
#pragma unroll 1
            for (int c = lane; c < L::GB / 16; c += 32) {
              const int row = c / L::CPR, in_row = c % L::CPR;
              const bool take = row >= lo && row < hi;
              copy_16(to + piece<L::CPR, F8, false>(row, in_row) * 16, take ? k + c * 16 : none, take);
              copy_16(to + L::GB + piece<L::CPR, F8, true>(row, in_row) * 16, take ? v + c * 16 : none, take);
            }
          }
        }
        if (++to_stage == a.stages) to_stage = 0;
      }
      copy_commit();
    };
    // scales follow their copies, as they arrive later than the pages' numbers
    int scaled = 0, scale_stage = 0;
    auto put_scales = [&]() {
      if (F8 && scaled < it.count) {
        if (lane / kLoads == scaled % kAhead) scales[scale_stage][warp * kLoads + lane % kLoads] = make_float4(my_k, my_v, __log2f(my_v), 0.f);
        ++scaled;
        if (++scale_stage == a.stages) scale_stage = 0;
      }
    };
#pragma unroll 1
    for (int i = 0; i < a.stages - 1; ++i) copy(i);
#pragma unroll 1
    for (int i = 0; i < a.stages - 1; ++i) put_scales();
    begin_rows<HD, F8, NB>(a, it, rows0, raw, r);
    // positions of the first and last row
    const int p_first = it.s.pos + (a.one_tile ? 0 : a.by_group(rows0));
    const int p_last = it.s.pos + (a.one_tile ? it.s.n - 1 : min(it.s.n - 1, a.by_group(rows0 + 8 * NB - 1)));
#pragma unroll 1
    for (int i = 0; i < it.count; ++i) {
      if (a.stages == F::kStages) copy_wait<F::kStages - 2>();
      else copy_wait<F::kDeep - 2>();
      __syncwarp();
      copy(i + a.stages - 1);
      put_scales();
      const char* at = ring + from_stage * F::kStage;
      constexpr int KG = F::kGroups;
      const int key_tile = (tile0 + i) * kTile;
#pragma unroll 1
      for (int w = warp * kLoads; w < (warp + 1) * kLoads; w += KG) {
        const int key0 = key_tile + w * kGroup;
        if (key0 > p_last || (a.window && key0 + KG * kGroup - 1 <= p_first - a.window)) continue;
        const bool checked = key0 + KG * kGroup - 1 > p_first || (a.window && key0 <= p_last - a.window);
        take_keys<HD, F8, NB, KG>(at + w * 2 * L::GB, &scales[from_stage][w], key0, checked, a.window, r);
      }
      if (++from_stage == a.stages) from_stage = 0;
    }
    copy_wait<0>();

    // the item's end; the queries of the next one are fetched meanwhile
    const Item done = it;
    const bool another = next_item<F>(a, plan, it);
    if (another) fetch_queries<HD, F8, NB>(a, it, it.mt * kRows, raw);
    // rows' sums over their threads, and over the warps where those took different keys
    const bool begins = done.off == 0, ends = done.off + done.count == done.tiles, complete = begins && ends;
    const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        r.l[n][h] += __shfl_xor_sync(0xffffffffu, r.l[n][h], 4);
        r.l[n][h] += __shfl_xor_sync(0xffffffffu, r.l[n][h], 8);
        r.l[n][h] += __shfl_xor_sync(0xffffffffu, r.l[n][h], 16);
      }
    __syncthreads();  // all warps are done with the ring, which now takes their outputs
    float* o_at = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = 8 * n + 2 * j + h;
        const float unit = F8 ? 1.f / r.f[n][h] : 1.f;
        if (g == 0) {
          join_m[warp][row] = r.limit[n][h] == -INFINITY ? -INFINITY : r.base[n][h];
          join_l[warp][row] = r.l[n][h];
        }
#pragma unroll
        for (int y = 0; y < HD / 16; ++y) {
          float* at = o_at + (warp * kRows + row) * HD;
          at[column<HD, F8>(2 * y, g)] = F8 ? r.o[n][y][h] * unit * unit : r.o[n][y][h];
          at[column<HD, F8>(2 * y + 1, g)] = F8 ? r.o[n][y][2 + h] * unit * unit : r.o[n][y][2 + h];
        }
      }
    __syncthreads();
    const int first = done.mt * kRows, n_rows = min(kRows, done.s.n * a.group - first);
    for (int k = tid; k < n_rows * (HD / 4); k += kThreads) {
      const int row = k / (HD / 4), col = k % (HD / 4) * 4;
      float top = join_m[0][row];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, join_m[w][row]);
      const float base = top == -INFINITY ? 0.f : top;
      float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float by = exp2_fast(join_m[w][row] - base);
        const float4 v = *reinterpret_cast<const float4*>(o_at + (w * kRows + row) * HD + col);
        l += join_l[w][row] * by;
        o[0] += v.x * by; o[1] += v.y * by; o[2] += v.z * by; o[3] += v.w * by;
      }
      if (complete) {
        const float by = l == 0.f ? 0.f : 1.f / l;
        const int t = a.by_group(first + row), hd = first + row - t * a.group;
        *reinterpret_cast<uint2*>(a.out + (size_t)(done.s.row + t) * a.ld_out + (size_t)(done.head * a.group + hd) * HD + col) =
            make_uint2(pack<false>(o[0] * by, o[1] * by), pack<false>(o[2] * by, o[3] * by));
      } else {
        *part_at<F>(a, slot, row, col / 4) = make_float4(o[0], o[1], o[2], o[3]);
        if (col == 0) a.stats[(size_t)slot * kRows + row] = make_float2(top, l);
      }
    }
    if (!complete && begins && tid == 0) mark_shared(a, plan, done);
    if (!another) break;
    __syncthreads();  // the ring and the join buffers are free again
  }
  pdl_trigger();  // not earlier: the next kernel's CTAs would take the room of this one's second half
}

}  // namespace
}  // namespace ane
#include "kv_attention_tc.cuh"
namespace ane {
namespace {

// Joins the parts of shared items: a block for each CTA of the first kernel and row of a tile.  Factors of all parts first, so that the
// parts themselves are read without waiting for one another.
constexpr int kJoinThreads = 256, kMostParts = 1024;

template <class F>
__device__ __forceinline__ void join_row(const Attn& a, int cta, int4 item, int row) {
  constexpr int HD = F::HD, kRows = F::kRows;
  const Span s = span_of(a.batch, item.x, INT32_MAX, INT32_MAX, a.status);
  const int at = item.y * kRows + row, parts = item.w, tid = threadIdx.x, warp = tid >> 5;
  if (at >= s.n * a.group) return;
  // part i: the first CTA's second slot, then the first slot of each
  auto slot = [&](int i) { return (size_t)(i == 0 ? 2 * cta + 1 : 2 * (cta + i)); };
  constexpr int lanes = HD / 4, teams = kJoinThreads / lanes, kMine = kMostParts / kJoinThreads;  // a team takes every teams-th part
  __shared__ float factor[kMostParts];
  __shared__ float most[kJoinThreads / 32], total[kJoinThreads / 32];
  __shared__ float4 sums[teams][lanes];
  const int team = tid / lanes, lane = tid % lanes;
  float2 st[kMine];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int i = tid + k * kJoinThreads;
    st[k] = i < parts ? a.stats[slot(i) * kRows + row] : make_float2(-INFINITY, 0.f);
  }
  constexpr int kEarly = 8;  // parts that are on their way before the factors are known
  float4 early[kEarly];
#pragma unroll
  for (int k = 0; k < kEarly; ++k) {
    const int i = team + k * teams;
    early[k] = team < teams && i < parts ? *part_at<F>(a, slot(i), row, lane) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int k = 0; k < kMine; ++k) m = fmaxf(m, st[k].x);
  m = warp_max(m);
  if ((tid & 31) == 0) most[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) m = fmaxf(m, most[i]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int i = tid + k * kJoinThreads;
    const float f = exp2_fast(st[k].x - base);
    if (i < parts) factor[i] = f;
    l += st[k].y * f;
  }
  l = warp_sum(l);
  if ((tid & 31) == 0) total[warp] = l;
  __syncthreads();
  if (team < teams) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, float f) {
      o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
    };
#pragma unroll
    for (int k = 0; k < kEarly; ++k)
      if (team + k * teams < parts) add(early[k], factor[team + k * teams]);
#pragma unroll 4
    for (int i = team + kEarly * teams; i < parts; i += teams)
      add(*part_at<F>(a, slot(i), row, lane), factor[i]);
    sums[team][lane] = o;
  }
  __syncthreads();
  if (tid >= lanes) return;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) l += total[i];
  float4 o = sums[0][tid];
  for (int i = 1; i < min(teams, parts); ++i) {
    const float4 v = sums[i][tid];
    o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
  }
  const float by = l == 0.f ? 0.f : 1.f / l;
  const int t = a.by_group(at), hd = at - t * a.group;
  *reinterpret_cast<uint2*>(a.out + (size_t)(s.row + t) * a.ld_out + (size_t)(item.z * a.group + hd) * HD + tid * 4) =
      make_uint2(pack<false>(o.x * by, o.y * by), pack<false>(o.z * by, o.w * by));
}

// The same of eight rows from `row` on by a block, for at most kFew parts: a row takes as many lanes as it has groups of four columns, rounded up to
// a power of two.
constexpr int kFew = 6;
template <class F>
__device__ __forceinline__ void join_rows(const Attn& a, int cta, int4 item, int row0) {
  constexpr int HD = F::HD, kRows = F::kRows, lanes = HD <= 32 ? 8 : HD <= 64 ? 16 : 32;
  const Span s = span_of(a.batch, item.x, INT32_MAX, INT32_MAX, a.status);
  const int tid = threadIdx.x, parts = item.w, lane = F::kSplit ? tid % lanes : tid / 8, row = row0 + (F::kSplit ? tid / lanes : tid % 8);
  const int at = item.y * kRows + row;
  if (tid >= 8 * lanes || row >= kRows || at >= s.n * a.group) return;
  const bool mine = lane * 4 < HD;
  float2 st[kFew];
  float4 v[kFew];
#pragma unroll
  for (int i = 0; i < kFew; ++i) {
    // part i: the first CTA's second slot, then the first slot of each
    const size_t slot = (size_t)(i == 0 ? 2 * cta + 1 : 2 * (cta + i));
    st[i] = i < parts ? a.stats[slot * kRows + row] : make_float2(-INFINITY, 0.f);
    v[i] = i < parts && mine ? *part_at<F>(a, slot, row, lane) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kFew; ++i) m = fmaxf(m, st[i].x);
  const float base = m == -INFINITY ? 0.f : m;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kFew; ++i) {
    const float f = exp2_fast(st[i].x - base);
    l = fmaf(st[i].y, f, l);
    o.x = fmaf(v[i].x, f, o.x); o.y = fmaf(v[i].y, f, o.y); o.z = fmaf(v[i].z, f, o.z); o.w = fmaf(v[i].w, f, o.w);
  }
  const float by = l == 0.f ? 0.f : 1.f / l;
  const int t = a.by_group(at), hd = at - t * a.group;
  if (mine)
    *reinterpret_cast<uint2*>(a.out + (size_t)(s.row + t) * a.ld_out + (size_t)(item.z * a.group + hd) * HD + lane * 4) =
        make_uint2(pack<false>(o.x * by, o.y * by), pack<false>(o.z * by, o.w * by));
}

// Rows of shared items, task t: row t % rows of the item that begins in CTA t / rows.  Most CTAs of the first kernel begin none: 32 tasks are
// looked at together.  Items of up to kFew parts take a part of a block a row, eight rows from every eighth task, others a block.
// The grid's size is odd where a block has several tasks, so that those are spread evenly.
template <class F>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const Attn a, int ctas, int rows) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, tasks = ctas * rows;  // this block's: blockIdx.x, + gridDim.x, ...
  for (int t0 = blockIdx.x; t0 < tasks; t0 += 32 * gridDim.x) {
    const int mine = t0 + lane * (int)gridDim.x, my_cta = mine / rows, my_row = mine - my_cta * rows;
    const int4 item = mine < tasks ? a.head[my_cta] : make_int4(-1, 0, 0, 0);
    for (uint32_t left = __ballot_sync(0xffffffffu, item.x >= 0 && (item.w > kFew || my_row % 8 == 0)); left; left &= left - 1) {
      const int from = __ffs(left) - 1, cta = __shfl_sync(0xffffffffu, my_cta, from), row = __shfl_sync(0xffffffffu, my_row, from);
      const int4 one = make_int4(__shfl_sync(0xffffffffu, item.x, from), __shfl_sync(0xffffffffu, item.y, from),
                                 __shfl_sync(0xffffffffu, item.z, from), __shfl_sync(0xffffffffu, item.w, from));
      if (one.w <= kFew) {
        join_rows<F>(a, cta, one, row);
        continue;
      }
      join_row<F>(a, cta, one, row);
      __syncthreads();
    }
  }
}

template <class F>
cudaError_t run(Attn a, int sms, void* workspace, cudaStream_t s) {
  constexpr int kRows = F::kRows, kTile = F::kTile, most = F::kCtas;
  static_assert(most * kRows <= (F::HD <= 64 ? 256 : 128), "the workspace is sized for these");
  static unsigned long long opted = 0;
  auto kernel = [] {
    if constexpr (F::kSplit) return kv_attention_kernel<F>;
    else return kv_prompt_kernel<F>;
  }();
  if (!smem_opt_in(kernel, F::kMostSmem, opted)) return cudaGetLastError();
  a.one_tile = (long long)a.max_new * a.group <= kRows;
  // no more CTAs than there can be units: items, or shares of F::kLeast tiles of them
  const long long longest = a.window ? min((long long)a.capacity, (long long)a.window + (kRows - 1) / a.group + kTile) : a.capacity;
  const long long items = (((long long)a.batch.n_tokens * a.group) / kRows + a.batch.n_seq) * a.kv.kv_heads;
  const long long tiles = (longest + kTile - 1) / kTile + (a.window ? 1 : 0);
  if (items * tiles > INT32_MAX) return cudaErrorInvalidValue;
  const bool may_share = tiles > F::kAlone;
  const int ctas = (int)min(min((long long)sms * most, (long long)kMostParts), may_share ? items * (tiles / F::kLeast + 2) : items);
  // a CTA that has an SM to itself may fetch further ahead
  a.stages = ctas <= sms ? F::kDeep : F::kStages;
  char* at = reinterpret_cast<char*>(workspace);
  a.head = reinterpret_cast<int4*>(at);
  at += sizeof(int4) * (size_t)sms * most;
  a.stats = reinterpret_cast<float2*>(at);
  at += sizeof(float2) * 2 * (size_t)sms * most * kRows;
  a.part = reinterpret_cast<float*>(at);
  cudaError_t e = launch_pdl(kernel, dim3((unsigned)ctas), dim3(F::kThreads), F::kSplit ? a.stages * F::kStage : F::kMostSmem, s, a);
  if (e != cudaSuccess || !may_share) return e;
  const int rows = (int)min((long long)kRows, (long long)a.max_new * a.group);
  return launch_pdl(kv_join_kernel<F>, dim3((unsigned)min((long long)ctas * rows, (kRows > 32 ? 8ll : 4ll) * sms - 1)), dim3(kJoinThreads), 0, s, a, ctas, rows);
}

// Which form, by the rows of one KV head that a sequence has at most.  Up to 32 the warps share them: as one tile, or, of wide heads, whose outputs
// do not fit the registers otherwise, two tiles that read their keys again; more are products of 128 rows.  us, the first and the second:
//   two sequences of 60000 tokens   20 rows of 64 81 and 94, 32 83 and 95, 48 142 and 98, 64 142 and 102 (bf16 136 and 89);
//                                   32 rows of 128 36 and 40 (bf16 35 and 34)
//   64 sequences of 8192            32 rows of 64 290 and 292, 64 474 and 301; 24 rows of 128 83 and 99, 32 88 and 100
//   16 sequences of 500             20 rows of 48 11.6 and 12.7, 48 12.2 and 12.9, 64 21.0 and 13.4
template <int HD, bool F8>
cudaError_t run_rows(const Attn& a, int sms, void* workspace, cudaStream_t s) {
  const long long rows = (long long)a.max_new * a.group;
  if (rows <= 8) return run<Form<HD, F8, 1>>(a, sms, workspace, s);
  if (rows <= (HD <= 64 ? 16 : 32)) return run<Form<HD, F8, 2>>(a, sms, workspace, s);
  if constexpr (HD <= 64)
    if (rows <= 32) return run<Form<HD, F8, 4>>(a, sms, workspace, s);
  return run<Prompt<HD, F8>>(a, sms, workspace, s);
}
template <int HD>
cudaError_t run_hd(const Attn& a, int sms, void* workspace, cudaStream_t s) {
  return a.kv.e4m3 ? run_rows<HD, true>(a, sms, workspace, s) : run_rows<HD, false>(a, sms, workspace, s);
}

}  // namespace

bool kv_head_dim_supported(int hd) { return hd == 32 || hd == 48 || hd == 64 || hd == 96 || hd == 128; }

template <int HD>
static size_t workspace_of(int sms) {
  auto bytes = [&](size_t per_sm, size_t rows) {
    return sms * per_sm * (sizeof(int4) + 2 * rows * (sizeof(float2) + sizeof(float) * HD));
  };
  return bytes(HD <= 64 ? 2 : 1, 128);  // the form of most rows
}
size_t kv_attention_workspace(int sms, int hd) {  // the same for both types of cache
  switch (hd) {
    case 32: return workspace_of<32>(sms);
    case 48: return workspace_of<48>(sms);
    case 64: return workspace_of<64>(sms);
    case 96: return workspace_of<96>(sms);
  }
  return workspace_of<128>(sms);
}

cudaError_t kv_attention(const PagedKv& kv, const Batch& batch, int heads, const bf16* q, int ld_q, bf16* out, int ld_out,
                         int max_new, int window, float scale, void* workspace, int* status, cudaStream_t s) {
  if (batch.n_seq == 0 || batch.n_tokens == 0) return cudaSuccess;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  Attn a = {};
  a.kv = kv;
  a.batch = batch;
  a.q = q; a.out = out; a.ld_q = ld_q; a.ld_out = ld_out;
  a.group = heads / kv.kv_heads;
  a.capacity = (int)min((long long)kv.table_pitch * kv.page_size, (long long)INT32_MAX - kv.page_size);
  a.by_group = Div(a.group);
  a.by_page = Div(kv.page_size);
  a.max_new = max_new;
  a.window = window;
  a.scale_log2 = (scale == 0.f ? (float)(1.0 / sqrt((double)kv.head_dim)) : scale) * 1.4426950408889634f;
  a.status = status;
  switch (kv.head_dim) {
    case 32: return run_hd<32>(a, sms, workspace, s);
    case 48: return run_hd<48>(a, sms, workspace, s);
    case 64: return run_hd<64>(a, sms, workspace, s);
    case 96: return run_hd<96>(a, sms, workspace, s);
    case 128: return run_hd<128>(a, sms, workspace, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace ane
