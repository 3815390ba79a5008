// Attention of new tokens over a paged KV cache (ane_op_kv_attention).
//
// The query heads of a KV head share its keys, so they are rows of one product: row r of a KV head's queries is token r / group,
// head r % group.  Products are m16n8k16 on mma.sync: single tokens are bound by the bytes of the cache, and their
// products take a fraction of the time that the operands need to arrive.
//
//   few rows (up to 16 a KV head): a CTA holds 8 or 16 rows; its four warps take 16 of every 64 keys each, with softmax statistics
//     of their own, joined at the end.  No barrier in the loop: every warp waits for its own copies only.
//   many rows: a CTA holds 64 or 128 rows, a warp a quarter of them, and all warps go over all keys.
//
// Keys and values come by cp.async into a ring of stages of 64 keys.  8-bit ones stay 8-bit until they are in registers, where they
// become f16, which holds e4m3 exactly: queries are brought to f16 by a power of two per row, scales of keys go onto the
// scores, scales of values onto the probabilities.
//
// Work is cut on the device, as only the device knows the lengths: all tiles of 64 keys of all (sequence, row tile, KV head) in
// one line, an even share of the line to each CTA of one wave.  What a CTA did of an item that others share goes to the
// workspace, and a second kernel joins the parts in their order, without atomics: the same sums from call to call.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "serving.h"

namespace ane {
namespace {

constexpr int kTile = 64, kGroup = 16, kWarps = 4, kThreads = kWarps * 32;
constexpr int kLeast = 4;  // tiles of an item that are not worth sharing: joining parts takes the time of about four
constexpr float kPScale = 32768.f;  // of f16 probabilities: those down to 2^-29 of the row's largest stay normal
constexpr float kLowest = 1.17549435e-38f;

struct Attn {
  PagedKv kv;
  Batch batch;
  const bf16* q;
  bf16* out;
  int ld_q, ld_out, group, max_new, window;
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
  static constexpr int VK = RB % 64 == 0 ? 16 : RB % 32 == 0 ? 8 : 4;   // bytes that a thread loads of K rows at a time
  static constexpr int VV = RB % 128 == 0 ? 16 : RB % 64 == 0 ? 8 : RB % 32 == 0 ? 4 : 2;  // of V rows
  static constexpr int STAGE = kWarps * 2 * GB;
};

// Where 16-byte piece c of a row lies within 16 rows, so that the threads of a fragment load find it in different banks: a thread
// (g, j) reads row g of K at pieces j.. and row 2 j (+ 1, 8, 9) of V at pieces g...
template <int CPR, bool V>
__device__ __forceinline__ int piece(int row, int c) {
  if (CPR % 8 == 0) return row * CPR + (c ^ (V ? row & 7 : (row & 1) << 2));
  if (CPR == 4) return (row >> 1) * 8 + ((((row & 1) << 2) | c) ^ ((row >> 1 & 3) << 1));
  if (CPR == 2) return (row >> 2) * 8 + ((((row & 3) << 1) | c) ^ ((row >> 2 & 1) << 1));
  return row * CPR + c;
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
__device__ __forceinline__ uint32_t e4m3_to_f16(uint32_t pair) {  // the low two bytes
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)pair));
  return r;
}
template <bool F8>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  if (F8) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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
  __device__ int t0() const { return lo / kTile; }
  __device__ int tiles() const { return (hi - 1) / kTile - lo / kTile + 1; }
};
__device__ __forceinline__ Range range_of(const Span& s, int rows0, int rows, int group, int window) {
  const int t_first = rows0 / group, t_last = min(s.n - 1, (rows0 + rows - 1) / group);
  return {window ? max(0, s.pos + t_first + 1 - window) : 0, s.pos + t_last + 1};
}

struct Plan {
  long long units, first, last;  // of the line: all, and this CTA's
  long long share;
  bool whole;                    // units are items, not tiles
  int b, mt, head, off;          // where `first` lies
};

template <int kRows>
__device__ __forceinline__ void weigh(const Attn& a, const Span& s, int& items, long long& tiles, int& longest) {
  items = 0;
  tiles = 0;
  for (int r = 0; r < s.n * a.group; r += kRows) {
    const int t = range_of(s, r, kRows, a.group, a.window).tiles();
    ++items;
    tiles += t;
    longest = max(longest, t);
  }
}

template <int kRows>
__device__ Plan make_plan(const Attn& a, int capacity) {
  __shared__ long long sums[2][kWarps];
  __shared__ int longest_of[kWarps];
  __shared__ Plan plan;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.batch.n_seq + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.batch.n_seq), b1 = min(b0 + per, a.batch.n_seq);
  long long items = 0, tiles = 0;
  int longest = 0;
  for (int b = b0; b < b1; ++b) {
    const Span s = span_of(a.batch, b, capacity, a.max_new, a.status);
    int i;
    long long t;
    weigh<kRows>(a, s, i, t, longest);
    items += (long long)i * a.kv.kv_heads;
    tiles += t * a.kv.kv_heads;
  }
  long long before_items = items, before_tiles = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long i = __shfl_up_sync(0xffffffffu, before_items, o), t = __shfl_up_sync(0xffffffffu, before_tiles, o);
    if (lane >= o) {
      before_items += i;
      before_tiles += t;
    }
    longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
  }
  if (lane == 31) {
    sums[0][warp] = before_items;
    sums[1][warp] = before_tiles;
    longest_of[warp] = longest;
  }
  if (tid == 0) plan.b = -1;
  __syncthreads();
  long long all_items = 0, all_tiles = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      before_items += sums[0][w];
      before_tiles += sums[1][w];
    }
    all_items += sums[0][w];
    all_tiles += sums[1][w];
    longest = max(longest, longest_of[w]);
  }
  const bool whole = longest <= kLeast;
  const long long units = whole ? all_items : all_tiles;
  long long share = (units + gridDim.x - 1) / gridDim.x;
  if (!whole) share = max(share, (long long)kLeast);
  const long long first = share * blockIdx.x;
  const long long mine = whole ? items : tiles, before = (whole ? before_items : before_tiles) - mine;
  if (first < units && first >= before && first < before + mine) {
    long long rest = first - before;
    for (int b = b0; b < b1; ++b) {
      const Span s = span_of(a.batch, b, capacity, a.max_new, a.status);
      int mt = 0;
      bool found = false;
      for (int r = 0; r < s.n * a.group; r += kRows, ++mt) {
        const int t = whole ? 1 : range_of(s, r, kRows, a.group, a.window).tiles();
        const long long w = (long long)t * a.kv.kv_heads;
        if (rest < w) {
          plan.b = b;
          plan.mt = mt;
          plan.head = (int)(rest / t);
          plan.off = (int)(rest % t);
          found = true;
          break;
        }
        rest -= w;
      }
      if (found) break;
    }
  }
  __syncthreads();
  Plan p = plan;
  p.units = units;
  p.share = share;
  p.whole = whole;
  p.first = first;
  p.last = min(first + share, units);
  return p;
}

// ---- the products of 16 keys and a warp's rows ----------------------------------------------------------------------------------
// Scores as K q^T and outputs as V^T p^T: keys, and then columns of the output, are the 16 rows of a product, queries its 8 columns, so
// that a group of up to 8 heads takes half of the products, registers and softmax arithmetic of the other way round.
template <int HD, bool F8, int NB>
struct Rows {  // 8 * NB rows of queries
  uint32_t q[NB][HD / 16][2];  // right operands: the thread's row g of each eight
  float o[NB][HD / 16][4];     // columns of the output column(2 y, g) and column(2 y + 1, g), for rows 2 j and 2 j + 1
  float m[NB][2], l[NB][2], mult[NB][2];  // rows 2 j and 2 j + 1; mult: what brings products to scores in log2
  int pos[NB][2];                         // their positions; -1: no such row
  float v_ref, v_inv;                     // 8 bits: o is in units of v_ref / kPScale; v_inv = kPScale / v_ref
};

template <int HD, bool F8, int NB>
__device__ __forceinline__ void load_queries(const Attn& a, const Span& s, int rows0, int head, Rows<HD, F8, NB>& r) {
  using L = Layout<HD, F8>;
  const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3, n_rows = s.n * a.group;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = rows0 + 8 * n + g;
    const bool there = row < n_rows;
    const int t = there ? row / a.group : 0, hd = there ? row - t * a.group : 0;
    const bf16* q = a.q + (size_t)(s.row + t) * a.ld_q + (size_t)(head * a.group + hd) * HD;
    float mult = a.scale_log2;
    if (F8) {
      uint2 w[HD / 16];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        // word i of the thread's bytes of a K row: four elements
        const int at = L::VK * j + i / (L::VK / 4) * 4 * L::VK + i % (L::VK / 4) * 4;
        w[i] = there ? *reinterpret_cast<const uint2*>(q + at) : make_uint2(0, 0);
        top = fmaxf(top, fmaxf(fmaxf(fabsf(__uint_as_float(w[i].x << 16)), fabsf(__uint_as_float(w[i].x & 0xffff0000u))),
                               fmaxf(fabsf(__uint_as_float(w[i].y << 16)), fabsf(__uint_as_float(w[i].y & 0xffff0000u)))));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the power of two that brings the row's largest value to [256, 512): f16 is exact for what is above 2^-22 of it
      const int e = min(max((int)(__float_as_uint(top) >> 23), 16), 254);
      const bool fine = top > 0.f && top < INFINITY;
      const float by = fine ? __uint_as_float((uint32_t)min(254 + 8 - e, 254) << 23) : 1.f;
      mult /= by;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        r.q[n][i][0] = pack<true>(__uint_as_float(w[i].x << 16) * by, __uint_as_float(w[i].x & 0xffff0000u) * by);
        r.q[n][i][1] = pack<true>(__uint_as_float(w[i].y << 16) * by, __uint_as_float(w[i].y & 0xffff0000u) * by);
      }
    } else {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        // words 2 i and 2 i + 1 of the thread's bytes of a K row
        const int word = 2 * i, at = (L::VK * j + word / (L::VK / 4) * 4 * L::VK + word % (L::VK / 4) * 4) / 2;
        const uint2 w = there ? *reinterpret_cast<const uint2*>(q + at) : make_uint2(0, 0);
        r.q[n][i][0] = w.x;
        r.q[n][i][1] = w.y;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int mine = rows0 + 8 * n + 2 * j + h;
      r.pos[n][h] = mine < n_rows ? s.pos + mine / a.group : -1;
      r.m[n][h] = -INFINITY;
      r.l[n][h] = 0.f;
      r.mult[n][h] = F8 ? __shfl_sync(0xffffffffu, mult, (2 * j + h) * 4) : mult;
    }
#pragma unroll
    for (int y = 0; y < HD / 16; ++y) r.o[n][y][0] = r.o[n][y][1] = r.o[n][y][2] = r.o[n][y][3] = 0.f;
  }
  r.v_ref = kLowest;
  r.v_inv = kPScale / kLowest;
}

// Whether one of a word's values is infinite or NaN.
template <bool F8>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  if (F8) return (w & 0x7fu) == 0x7fu || (w >> 8 & 0x7fu) == 0x7fu || (w >> 16 & 0x7fu) == 0x7fu || (w >> 24 & 0x7fu) == 0x7fu;
  return (w & 0x7f80u) == 0x7f80u || (w >> 16 & 0x7f80u) == 0x7f80u;
}

// Column of the output that group x of a thread's bytes of V rows (element x) stands for in the threads with this g.
template <int HD, bool F8>
__device__ __forceinline__ int column(int x, int g) {
  using L = Layout<HD, F8>;
  constexpr int EV = L::VV / L::ES;
  return x / EV * 8 * EV + g * EV + x % EV;
}
__device__ __forceinline__ uint32_t transposed(uint32_t w) {  // of an 8 x 8 matrix of 16-bit values
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
  return r;
}

// 16 keys at positions key0.. against the warp's rows.  `checked`: some row does not see some key.
template <int HD, bool F8, int NB>
__device__ __forceinline__ void keys_16(const char* ks, const char* vs, int key0, bool checked, int window, float k_scale,
                                        float v_scale, Rows<HD, F8, NB>& r) {
  using L = Layout<HD, F8>;
  const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  float s[NB][4];  // keys g (0, 1) and g + 8 (2, 3), rows 2 j and 2 j + 1
#pragma unroll
  for (int n = 0; n < NB; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
  for (int i = 0; i < L::RB / (4 * L::VK); ++i) {
    const int byte = L::VK * j + 4 * L::VK * i;
    uint32_t u[L::VK / 4], w[L::VK / 4];  // of keys g and g + 8
    lds<L::VK>(ks + piece<L::CPR, false>(g, byte >> 4) * 16 + (byte & 15), u);
    lds<L::VK>(ks + piece<L::CPR, false>(8 + g, byte >> 4) * 16 + (byte & 15), w);
#pragma unroll
    for (int x = 0; x < L::VK / 4; x += F8 ? 1 : 2) {
      const uint32_t k[4] = {F8 ? e4m3_to_f16(u[x]) : u[x], F8 ? e4m3_to_f16(w[x]) : w[x], F8 ? e4m3_to_f16(u[x] >> 16) : u[x + !F8],
                             F8 ? e4m3_to_f16(w[x] >> 16) : w[x + !F8]};
      const int step = F8 ? i * (L::VK / 4) + x : (i * (L::VK / 4) + x) / 2;
#pragma unroll
      for (int n = 0; n < NB; ++n) mma<F8>(s[n], k, r.q[n][step][0], r.q[n][step][1]);
    }
  }
  uint32_t seen = 0xffffffffu;  // bit 4 n + i of s[n][i]
  if (checked) {
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + g + 8 * (i >> 1), pos = r.pos[n][i & 1];
        if (key > pos || (window && key <= pos - window)) {
          s[n][i] = -INFINITY;
          seen &= ~(1u << (4 * n + i));
        }
      }
  }
  float into = 1.f;
  if (F8) {
    if (v_scale > r.v_ref) {  // statistics keep their unit, the output changes to the new one
      const float by = r.v_ref / v_scale;
      r.v_ref = v_scale;
      r.v_inv = kPScale / v_scale;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int y = 0; y < HD / 16; ++y)
#pragma unroll
          for (int i = 0; i < 4; ++i) r.o[n][y][i] *= by;
    }
    into = v_scale * r.v_inv;
  }
  uint32_t p[NB][2];
  bool moved = false;
  float fix[NB][2];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float mult = F8 ? fmaxf(r.mult[n][h] * k_scale, kLowest) : r.mult[n][h];  // not 0, so that hidden scores stay -infinity
      float top = fmaxf(s[n][h], s[n][2 + h]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      top = fmaxf(top * mult, r.m[n][h]);
      const float base = top == -INFINITY ? 0.f : top;  // nothing seen yet: exp2 of -infinity, which is 0
      fix[n][h] = exp2_fast(r.m[n][h] - base);
      moved |= r.m[n][h] != top;
      r.m[n][h] = top;
      s[n][h] = exp2_fast(fmaf(s[n][h], mult, -base));
      s[n][2 + h] = exp2_fast(fmaf(s[n][2 + h], mult, -base));
      r.l[n][h] = fmaf(r.l[n][h], fix[n][h], s[n][h] + s[n][2 + h]);  // the thread's own keys; joined at the end
      if (F8) {
        s[n][h] *= into;
        s[n][2 + h] *= into;
      }
    }
    // probabilities in 16 bits: their rounding is half a step of the output's own type or less
    p[n][0] = transposed(pack<F8>(s[n][0], s[n][1]));
    p[n][1] = transposed(pack<F8>(s[n][2], s[n][3]));
  }
  if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int y = 0; y < HD / 16; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) r.o[n][y][i] *= fix[n][i & 1];
  }
  bool odd = false;
  if (checked) {
    // a value that is infinite or NaN must not reach rows that do not see its key, and 0 * NaN is NaN
#pragma unroll 1
    for (int i = lane; i < L::GB / 4; i += 32) odd |= not_finite<F8>(*reinterpret_cast<const uint32_t*>(vs + 4 * i));
    odd = __any_sync(0xffffffffu, odd);
  }
  if (odd) {
    // one product after the other, unseen ones left out
#pragma unroll 1
    for (int k = 0; k < kGroup; ++k) {
      const int from = (k & 7) * 4 + j;
      const uint32_t see = __shfl_sync(0xffffffffu, seen, from) >> (k < 8 ? 0 : 2);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const float w0 = __shfl_sync(0xffffffffu, k < 8 ? s[n][0] : s[n][2], from), w1 = __shfl_sync(0xffffffffu, k < 8 ? s[n][1] : s[n][3], from);
#pragma unroll
        for (int x = 0; x < HD / 8; ++x) {
          const int byte = column<HD, F8>(x, g) * L::ES;
          const char* at = vs + piece<L::CPR, true>(k, byte >> 4) * 16 + (byte & 15);
          const float v = F8 ? __half2float(__half(__nv_cvt_fp8_to_halfraw(*reinterpret_cast<const unsigned char*>(at), __NV_E4M3)))
                             : __uint_as_float((uint32_t)*reinterpret_cast<const unsigned short*>(at) << 16);
          if (see >> (4 * n) & 1u) r.o[n][x >> 1][2 * (x & 1)] += w0 * v;
          if (see >> (4 * n + 1) & 1u) r.o[n][x >> 1][2 * (x & 1) + 1] += w1 * v;
        }
      }
    }
    return;
  }
  constexpr int EV = L::VV / L::ES, WV = L::VV >= 4 ? L::VV / 4 : 1;
#pragma unroll
  for (int i = 0; i < L::RB / (8 * L::VV); ++i) {
    const int byte = L::VV * g + 8 * L::VV * i;
    uint32_t w[4][WV];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = 2 * j + (k & 1) + 8 * (k >> 1);
      lds<L::VV>(vs + piece<L::CPR, true>(row, byte >> 4) * 16 + (byte & 15), w[k]);
    }
#pragma unroll
    for (int x = 0; x < WV; ++x) {
      if (F8) {
        // two columns of two keys in a word: (key, key + 1) of one column, then of the next
        const uint32_t b0 = __byte_perm(w[0][x], w[1][x], 0x5140), b1 = __byte_perm(w[2][x], w[3][x], 0x5140);
        const uint32_t v[4] = {e4m3_to_f16(b0), e4m3_to_f16(b0 >> 16), e4m3_to_f16(b1), e4m3_to_f16(b1 >> 16)};
        const int y = (i * EV + 4 * x) / 2;
#pragma unroll
        for (int n = 0; n < NB; ++n) mma<true>(r.o[n][y], v, p[n][0], p[n][1]);
        if (EV > 2) {
          const uint32_t c0 = __byte_perm(w[0][x], w[1][x], 0x7362), c1 = __byte_perm(w[2][x], w[3][x], 0x7362);
          const uint32_t u[4] = {e4m3_to_f16(c0), e4m3_to_f16(c0 >> 16), e4m3_to_f16(c1), e4m3_to_f16(c1 >> 16)};
#pragma unroll
          for (int n = 0; n < NB; ++n) mma<true>(r.o[n][y + 1], u, p[n][0], p[n][1]);
        }
      } else {
        const uint32_t v[4] = {__byte_perm(w[0][x], w[1][x], 0x5410), __byte_perm(w[0][x], w[1][x], 0x7632),
                               __byte_perm(w[2][x], w[3][x], 0x5410), __byte_perm(w[2][x], w[3][x], 0x7632)};
        const int y = (i * EV + 2 * x) / 2;
#pragma unroll
        for (int n = 0; n < NB; ++n) mma<false>(r.o[n][y], v, p[n][0], p[n][1]);
      }
    }
  }
}

// ---- the kernel -------------------------------------------------------------------------------------------------------------------
// kSplit: the four warps share 8 * NB rows and take 16 of every 64 keys each; otherwise each has 8 * NB rows and takes all keys.
template <int HD, bool F8, int NB, bool kSplit>
struct Form {
  using L = Layout<HD, F8>;
  static constexpr int kRows = kSplit ? 8 * NB : 8 * NB * kWarps;
  // resident CTAs wanted: registers for outputs and queries decide
  static constexpr int kRegs = NB * (HD / 16 * 6 + 16);
  static constexpr int kCtas = kRegs <= 80 ? 4 : kRegs <= 112 ? 3 : 2;
  static constexpr int kRoom = 224 * 1024 / kCtas - 4096, kFit = kRoom / L::STAGE;
  static constexpr int kStages = kFit < 3 ? 3 : kFit > 6 ? 6 : kFit;
  static constexpr int kJoin = kSplit ? kWarps * kRows * HD * 4 : 0;
  static constexpr int kSmem = kStages * L::STAGE > kJoin ? kStages * L::STAGE : kJoin;
};

template <int HD, bool F8, int NB, bool kSplit>
__global__ void __launch_bounds__(kThreads, Form<HD, F8, NB, kSplit>::kCtas) kv_attention_kernel(const Attn a) {
  using L = Layout<HD, F8>;
  using F = Form<HD, F8, NB, kSplit>;
  constexpr int kRows = F::kRows, kStages = F::kStages;
  extern __shared__ __align__(128) char ring[];
  __shared__ float2 scales[kStages][kWarps];
  __shared__ float join_m[kWarps][8 * NB], join_l[kWarps][8 * NB];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j = lane & 3;
  const int page = a.kv.page_size;
  const int capacity = (int)min((long long)a.kv.table_pitch * page, (long long)INT32_MAX);
  const Plan plan = make_plan<kRows>(a, capacity);
  if (tid == 0) a.head[blockIdx.x] = make_int4(-1, 0, 0, 0);
  const uint32_t ring_at = smem_u32(ring);
  int b = plan.b, mt = plan.mt, head = plan.head, off = plan.off;
  if (b < 0) {
    pdl_trigger();
    return;
  }
  Span s = span_of(a.batch, b, capacity, a.max_new, a.status);
  for (long long unit = plan.first; unit < plan.last;) {
    const int rows0 = mt * kRows;
    const Range range = range_of(s, rows0, kRows, a.group, a.window);
    const int tiles = range.tiles();
    const int count = plan.whole ? tiles : (int)min((long long)(tiles - off), plan.last - unit);
    const int tile0 = range.t0() + off;

    // copies of tile0 + i, i < count: this warp's 16 keys of each.  Where they lie (in 16-byte pieces; all ones: nowhere) and their scales,
    // of 32 tiles ahead, are in its lanes.
    uint32_t my_at = 0xffffffffu;
    float my_k = 1.f, my_v = 1.f;
    auto look_up = [&](int i) {
      const int key = (tile0 + i + lane) * kTile + warp * kGroup;
      my_at = 0xffffffffu;
      my_k = my_v = 1.f;
      if (i + lane < count && key < range.hi && key + kGroup > range.lo) {
        const int slot = key / page, p = a.kv.table[(size_t)b * a.kv.table_pitch + slot];
        if (p < 0 || p >= a.kv.n_pages) {
          atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
        } else {
          my_at = (uint32_t)(((unsigned long long)p * a.kv.page_stride + ((size_t)head * page + key - slot * page) * HD) * L::ES >> 4);
          if (F8) {
            my_k = a.kv.k_scale[(size_t)p * a.kv.kv_heads + head];
            my_v = a.kv.v_scale[(size_t)p * a.kv.kv_heads + head];
          }
        }
      }
    };
    int to_stage = 0, from_stage = 0;
    auto copy = [&](int i) {
      if (i < count) {
        if ((i & 31) == 0) look_up(i);
        const uint32_t at = __shfl_sync(0xffffffffu, my_at, i & 31);
        const int key0 = (tile0 + i) * kTile + warp * kGroup;
        if (F8) {
          const float ks = __shfl_sync(0xffffffffu, my_k, i & 31), vs = __shfl_sync(0xffffffffu, my_v, i & 31);
          if (lane == 0) scales[to_stage][warp] = make_float2(ks, vs);
        }
        const uint32_t to = ring_at + to_stage * L::STAGE + warp * 2 * L::GB;
        const char *k = reinterpret_cast<const char*>(a.kv.k) + (size_t)at * 16, *v = reinterpret_cast<const char*>(a.kv.v) + (size_t)at * 16;
        if (key0 >= range.lo && key0 + kGroup <= range.hi && at != 0xffffffffu) {
#pragma unroll
          for (int c0 = 0; c0 < L::GB / 16; c0 += 32) {
            const int c = c0 + lane;
            if ((L::GB / 16) % 32 == 0 || c < L::GB / 16) {
              const int row = c / L::CPR, in_row = c % L::CPR;
              copy_16(to + piece<L::CPR, false>(row, in_row) * 16, k + c * 16, true);
              copy_16(to + L::GB + piece<L::CPR, true>(row, in_row) * 16, v + c * 16, true);
            }
          }
        } else {
          // rows that no query sees are filled with zeros: whatever lies there must not count
          const int lo = range.lo - key0, hi = at == 0xffffffffu ? 0 : range.hi - key0;
#pragma unroll 1
          for (int c = lane; c < L::GB / 16; c += 32) {
            const int row = c / L::CPR, in_row = c % L::CPR;
            const bool take = row >= lo && row < hi;
            copy_16(to + piece<L::CPR, false>(row, in_row) * 16, take ? k + c * 16 : reinterpret_cast<const char*>(a.kv.k), take);
            copy_16(to + L::GB + piece<L::CPR, true>(row, in_row) * 16, take ? v + c * 16 : reinterpret_cast<const char*>(a.kv.v), take);
          }
        }
        if (++to_stage == kStages) to_stage = 0;
      }
      copy_commit();
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) copy(i);

    Rows<HD, F8, NB> r;
    const int my_rows0 = rows0 + (kSplit ? 0 : warp * 8 * NB);
    load_queries<HD, F8, NB>(a, s, my_rows0, head, r);
    // positions of the warp's first and last row
    const bool any_row = my_rows0 < s.n * a.group;
    const int p_first = s.pos + my_rows0 / a.group, p_last = s.pos + min(s.n - 1, (my_rows0 + 8 * NB - 1) / a.group);

#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      copy_wait<kStages - 2>();
      if (kSplit) __syncwarp();
      else __syncthreads();
      copy(i + kStages - 1);
      const char* at = ring + from_stage * L::STAGE;
#pragma unroll 1
      for (int w = kSplit ? warp : 0; w < (kSplit ? warp + 1 : kWarps); ++w) {
        const int key0 = (tile0 + i) * kTile + w * kGroup;
        if (!any_row || key0 > p_last || (a.window && key0 + kGroup - 1 <= p_first - a.window)) continue;
        const bool checked = key0 + kGroup - 1 > p_first || (a.window && key0 <= p_last - a.window);
        const float2 scale = F8 ? scales[from_stage][w] : make_float2(1.f, 1.f);
        keys_16<HD, F8, NB>(at + w * 2 * L::GB, at + w * 2 * L::GB + L::GB, key0, checked, a.window, scale.x, scale.y, r);
      }
      if (++from_stage == kStages) from_stage = 0;
    }
    copy_wait<0>();

    // the item's end: rows' sums over their threads, and over the warps where those took different keys
    const bool begins = off == 0, ends = off + count == tiles, complete = begins && ends;
    const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
    float unit_o = 1.f;
    if (F8) unit_o = r.v_ref * (1.f / kPScale);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        r.l[n][h] += __shfl_xor_sync(0xffffffffu, r.l[n][h], 4);
        r.l[n][h] += __shfl_xor_sync(0xffffffffu, r.l[n][h], 8);
        r.l[n][h] += __shfl_xor_sync(0xffffffffu, r.l[n][h], 16);
      }
    if (kSplit) {
      __syncthreads();  // all warps are done with the ring, which now takes their outputs
      float* o_at = reinterpret_cast<float*>(ring);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = 8 * n + 2 * j + h;
          if (g == 0) {
            join_m[warp][row] = r.m[n][h];
            join_l[warp][row] = r.l[n][h];
          }
#pragma unroll
          for (int y = 0; y < HD / 16; ++y)
            *reinterpret_cast<float2*>(o_at + (warp * kRows + row) * HD + column<HD, F8>(2 * y, g)) =
                make_float2(r.o[n][y][h] * unit_o, r.o[n][y][2 + h] * unit_o);
        }
      __syncthreads();
      const int n_rows = min(kRows, s.n * a.group - rows0);
      for (int i = tid; i < n_rows * (HD / 4); i += kThreads) {
        const int row = i / (HD / 4), col = i % (HD / 4) * 4;
        float top = join_m[0][row];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, join_m[w][row]);
        const float base = top == -INFINITY ? 0.f : top;
        float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float by = exp2_fast(join_m[w][row] - base);
          const float4 v = *reinterpret_cast<const float4*>(o_at + (w * kRows + row) * HD + col);
          if (join_m[w][row] == -INFINITY && join_l[w][row] == 0.f) continue;  // saw nothing
          l += join_l[w][row] * by;
          o[0] += v.x * by; o[1] += v.y * by; o[2] += v.z * by; o[3] += v.w * by;
        }
        if (complete) {
          const float by = l == 0.f ? 0.f : 1.f / l;
          const int t = (rows0 + row) / a.group, hd = (rows0 + row) % a.group;
          *reinterpret_cast<uint2*>(a.out + (size_t)(s.row + t) * a.ld_out + (size_t)(head * a.group + hd) * HD + col) =
              make_uint2(pack<false>(o[0] * by, o[1] * by), pack<false>(o[2] * by, o[3] * by));
        } else {
          *reinterpret_cast<float4*>(a.part + ((size_t)slot * kRows + row) * HD + col) = make_float4(o[0], o[1], o[2], o[3]);
          if (col == 0) a.stats[(size_t)slot * kRows + row] = make_float2(top, l);
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = warp * 8 * NB + 8 * n + 2 * j + h, at = rows0 + row;
          if (at >= s.n * a.group) continue;
          const float by = complete ? (r.l[n][h] == 0.f ? 0.f : unit_o / r.l[n][h]) : unit_o;
          const int t = at / a.group, hd = at % a.group;
          bf16* out = a.out + (size_t)(s.row + t) * a.ld_out + (size_t)(head * a.group + hd) * HD;
          float* part = a.part + ((size_t)slot * kRows + row) * HD;
          if (!complete && g == 0) a.stats[(size_t)slot * kRows + row] = make_float2(r.m[n][h], r.l[n][h]);
#pragma unroll
          for (int y = 0; y < HD / 16; ++y) {
            const int col = column<HD, F8>(2 * y, g);
            const float u = r.o[n][y][h] * by, v = r.o[n][y][2 + h] * by;
            if (complete) *reinterpret_cast<uint32_t*>(out + col) = pack<false>(u, v);
            else *reinterpret_cast<float2*>(part + col) = make_float2(u, v);
          }
        }
    }
    if (!complete && begins && tid == 0) {
      // parts: this CTA's and one of each of the next ones until the item ends
      const long long end = unit + tiles;
      a.head[blockIdx.x] = make_int4(b, mt, head, (int)((end - 1) / plan.share - blockIdx.x) + 1);
    }
    __syncthreads();  // the ring and the join buffers are free again
    unit += plan.whole ? 1 : count;
    off = 0;
    if (unit < plan.last && ++head == a.kv.kv_heads) {
      head = 0;
      ++mt;
      while (mt * kRows >= s.n * a.group) {
        mt = 0;
        s = span_of(a.batch, ++b, capacity, a.max_new, a.status);
      }
    }
  }
  pdl_trigger();
}

// Joins the parts of shared items: a block for each CTA of the first kernel and row of a tile.
template <int HD, int kRows>
__global__ void __launch_bounds__(kThreads) kv_join_kernel(const Attn a) {
  pdl_trigger();
  pdl_wait();
  const int4 item = a.head[blockIdx.x];
  if (item.x < 0) return;
  const Span s = span_of(a.batch, item.x, INT32_MAX, INT32_MAX, a.status);
  const int row = blockIdx.y, at = item.y * kRows + row, parts = item.w, tid = threadIdx.x;
  if (at >= s.n * a.group) return;
  // part i: the first CTA's second slot, then the first slot of each
  auto slot = [&](int i) { return (size_t)(i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i)) * kRows + row; };
  constexpr int lanes = HD / 4, teams = kThreads / lanes;  // a team goes over every teams-th part
  __shared__ float4 sums[teams][lanes];
  __shared__ float2 stats[teams];
  const int team = tid / lanes, lane = tid % lanes;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (team < teams) {
#pragma unroll 4
    for (int i = team; i < parts; i += teams) {
      const float2 st = a.stats[slot(i)];
      const float4 v = *reinterpret_cast<const float4*>(a.part + slot(i) * HD + lane * 4);
      if (st.x == -INFINITY && st.y == 0.f) continue;
      const float top = fmaxf(m, st.x), base = top == -INFINITY ? 0.f : top;
      const float f = exp2_fast(m - base), by = exp2_fast(st.x - base);
      m = top;
      l = l * f + st.y * by;
      o.x = o.x * f + v.x * by; o.y = o.y * f + v.y * by; o.z = o.z * f + v.z * by; o.w = o.w * f + v.w * by;
    }
    sums[team][lane] = o;
    if (lane == 0) stats[team] = make_float2(m, l);
  }
  __syncthreads();
  if (tid >= lanes) return;
  m = -INFINITY;
#pragma unroll
  for (int i = 0; i < teams; ++i) m = fmaxf(m, stats[i].x);
  const float base = m == -INFINITY ? 0.f : m;
  l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < teams; ++i) {
    if (stats[i].x == -INFINITY && stats[i].y == 0.f) continue;
    const float by = exp2_fast(stats[i].x - base);
    const float4 v = sums[i][tid];
    l += stats[i].y * by;
    o.x += v.x * by; o.y += v.y * by; o.z += v.z * by; o.w += v.w * by;
  }
  const float by = l == 0.f ? 0.f : 1.f / l;
  const int t = at / a.group, hd = at % a.group;
  *reinterpret_cast<uint2*>(a.out + (size_t)(s.row + t) * a.ld_out + (size_t)(item.z * a.group + hd) * HD + tid * 4) =
      make_uint2(pack<false>(o.x * by, o.y * by), pack<false>(o.z * by, o.w * by));
}

// CTAs of a wave: bounded so that the workspace's size is known without asking for the occupancy.
constexpr int kMostPerSm = 4;

template <int HD, bool F8, int NB, bool kSplit>
cudaError_t run(Attn a, int sms, void* workspace, cudaStream_t s) {
  using F = Form<HD, F8, NB, kSplit>;
  constexpr int kRows = F::kRows, most = F::kCtas;
  static_assert(most <= kMostPerSm, "the workspace is sized for this many");
  static unsigned long long opted = 0;
  auto kernel = kv_attention_kernel<HD, F8, NB, kSplit>;
  if (!smem_opt_in(kernel, F::kSmem, opted)) return cudaGetLastError();
  // no more CTAs than there can be units: items, or pieces of kLeast tiles of them
  const long long capacity = (long long)a.kv.table_pitch * a.kv.page_size;
  const long long longest = a.window ? min(capacity, (long long)a.window + (kRows - 1) / a.group + kTile) : capacity;
  const long long items = (((long long)a.batch.n_tokens * a.group) / kRows + a.batch.n_seq) * a.kv.kv_heads;
  const long long pieces = ((longest + kTile - 1) / kTile + 1 + kLeast - 1) / kLeast;
  const bool may_share = (longest + kTile - 1) / kTile > kLeast;
  const int ctas = (int)min((long long)sms * most, may_share ? items * pieces : items);
  char* at = reinterpret_cast<char*>(workspace);
  a.head = reinterpret_cast<int4*>(at);
  at += sizeof(int4) * (size_t)sms * most;
  a.stats = reinterpret_cast<float2*>(at);
  at += sizeof(float2) * 2 * (size_t)sms * most * kRows;
  a.part = reinterpret_cast<float*>(at);
  cudaError_t e = launch_pdl(kernel, dim3((unsigned)ctas), dim3(kThreads), F::kSmem, s, a);
  if (e != cudaSuccess || !may_share) return e;
  const int rows = (int)min((long long)kRows, (long long)a.max_new * a.group);
  return launch_pdl(kv_join_kernel<HD, kRows>, dim3((unsigned)ctas, (unsigned)rows), dim3(kThreads), 0, s, a);
}

// Rows of one KV head at most: which form.
template <int HD, bool F8>
cudaError_t run_rows(const Attn& a, int sms, void* workspace, cudaStream_t s) {
  constexpr int kMany = HD <= 64 ? 4 : 2;
  const long long rows = (long long)a.max_new * a.group;
  if (rows <= 8) return run<HD, F8, 1, true>(a, sms, workspace, s);
  if (rows <= 16) return run<HD, F8, 2, true>(a, sms, workspace, s);
  return run<HD, F8, kMany, false>(a, sms, workspace, s);
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
  using A = Form<HD, false, 1, true>;
  using B = Form<HD, false, 2, true>;
  using C = Form<HD, false, HD <= 64 ? 4 : 2, false>;
  size_t most = bytes(A::kCtas, A::kRows);
  if (bytes(B::kCtas, B::kRows) > most) most = bytes(B::kCtas, B::kRows);
  if (bytes(C::kCtas, C::kRows) > most) most = bytes(C::kCtas, C::kRows);
  return most;
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
