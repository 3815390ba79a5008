// Appending keys and values to a paged cache, rotated by their positions on the way (ane_op_kv_append).
//
// q|k|v read, rotated q and the cache's rows written, once each: bound by HBM in the limit.  10368 tokens of 32 prompts, 12 + 4 heads of 64 into
// 8-bit pages take 18.8 us (50 MB, 2.7 TB/s; the floor is 7.7), into bf16 pages 19.1 (8.5): no pipe is full, 40 % of the issue slots are taken and 33 %
// of the warps active, so that it is the reads that a short block waits for one after the other: sequence, page, rows.  64 single tokens take
// 3.3 us, one 2.8: launches.
#include <cuda_fp8.h>

#include "serving.h"

namespace ane {

PagedKv paged_kv(const ane_kv_cache& c) {
  PagedKv kv;
  kv.k = c.d_k; kv.v = c.d_v; kv.k_scale = c.d_k_scale; kv.v_scale = c.d_v_scale;
  kv.page_stride = c.page_stride ? c.page_stride : (long long)c.n_kv_heads * c.page_size * c.head_dim;
  kv.n_pages = c.n_pages; kv.page_size = c.page_size; kv.kv_heads = c.n_kv_heads; kv.head_dim = c.head_dim;
  kv.table = c.d_page_table; kv.table_pitch = c.table_pitch;
  kv.e4m3 = c.dtype == ANE_KV_E4M3;
  return kv;
}

namespace {

constexpr int kThreads = 128, kMany = 4;  // two rows a thread: 20.1 us for 10368 tokens, four 19.0, eight 23.1

struct Append {
  PagedKv kv;
  Batch batch;
  const bf16* qkv;  // may be q: every element is read by the thread that writes it
  bf16* q;
  const float *cosb, *sinb;
  int ld_qkv, ld_q, heads;
  int n_positions;  // that may be written: those of the tables, or any
  int rows_blocks;  // blocks that rotate rows; the others are 8-bit pages
  int units;        // bound of the pages that are touched
  int capacity;     // tokens of a sequence
  int q_vec, kv_vec;  // groups of eight elements of a row's queries, and keys or values, that the former take
  Div by_row, by_head, by_page;  // by those groups of a row, by groups of a head, by tokens of a page
  int* status;
};

// The first sequence whose end, as end(i) gives it for start[i + 1], lies behind `at`, and what the batch says of it: all of a team's T threads
// look at other sequences, so that this takes one round trip to memory.  n_seq if there is none.
struct Found {
  int b, row, end, pos;
};
template <int T, class End>
__device__ __forceinline__ Found find(const Batch& a, int at, int lane, End end) {
  Found f = {a.n_seq, 0, 0, 0};
  bool mine = false;
  for (int i = lane; i < a.n_seq && !mine; i += T) {
    const int from = a.start[i], to = a.start[i + 1], pos = a.pos[i];
    mine = end(to, i + 1) > at && (i == 0 || end(from, i) <= at);
    if (mine) f = {i, from, to, pos};
  }
  if constexpr (T == 32) {
    const uint32_t who = __ballot_sync(0xffffffffu, mine);
    const int from = who ? __ffs(who) - 1 : 0;
    return {__shfl_sync(0xffffffffu, f.b, from), __shfl_sync(0xffffffffu, f.row, from), __shfl_sync(0xffffffffu, f.end, from),
            __shfl_sync(0xffffffffu, f.pos, from)};
  } else {
    __shared__ Found found;
    if (lane == 0) found = {a.n_seq, 0, 0, 0};
    __syncthreads();
    if (mine) found = f;
    __syncthreads();
    return found;
  }
}

// Eight elements of a row, rotated by their position if c is given.  Products and sums are rounded one by one.
struct Eight {
  float x[8];
};
struct Raw {
  uint4 x;
  float4 c, s;
};
__device__ __forceinline__ Raw fetch_eight(const bf16* p, const float* c, const float* s) {
  Raw r;
  r.x = *reinterpret_cast<const uint4*>(p);
  r.c = c ? *reinterpret_cast<const float4*>(c) : make_float4(0.f, 0.f, 0.f, 0.f);
  r.s = c ? *reinterpret_cast<const float4*>(s) : make_float4(0.f, 0.f, 0.f, 0.f);
  return r;
}
__device__ __forceinline__ Eight turned(const Raw& r, bool turn) {
  const uint32_t w[4] = {r.x.x, r.x.y, r.x.z, r.x.w};
  const float c[4] = {r.c.x, r.c.y, r.c.z, r.c.w}, s[4] = {r.s.x, r.s.y, r.s.z, r.s.w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __uint_as_float(w[i] << 16), b = __uint_as_float(w[i] & 0xffff0000u);
    e.x[2 * i] = turn ? __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i])) : a;
    e.x[2 * i + 1] = turn ? __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i])) : b;
  }
  return e;
}
__device__ __forceinline__ void store_eight(bf16* p, const Eight& e) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(e.x[2 * i], e.x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Groups of eight elements of the tokens' rows: the queries of all caches, keys and values too of a bf16 one.  A thread has the same group of
// kEach rows in a row, so that what the group is is found out once, and all its loads are on their way before the first is used.
template <int kEach>
__device__ __forceinline__ void append_rows(const Append& a, int block) {
  const int tid = threadIdx.x, hd = a.kv.head_dim, half = hd >> 1, page = a.kv.page_size;
  const int vec = a.q_vec + 2 * a.kv_vec, u = block * kThreads + tid, rows = a.by_row(u), v = u - rows * vec, row0 = rows * kEach;
  // the sequence of the block's first row; the next ones are found from there
  const Found f = find<kThreads>(a.batch, a.by_row(block * kThreads) * kEach, tid, [](int to, int) { return to; });
  int b = f.b, end = f.end;
  Span s = span_of(f.row, f.end, f.pos, a.batch, a.capacity, INT32_MAX, a.status);
  const int part = v < a.q_vec ? 0 : v < a.q_vec + a.kv_vec ? 1 : 2;
  const int in_part = part == 0 ? v : v - a.q_vec - (part - 1) * a.kv_vec;  // within q, k or v
  const int head = a.by_head(in_part), in_head = in_part * 8 - head * hd;
  const bool turn = part < 2 && a.cosb;
  const bf16* from = a.qkv + (size_t)row0 * a.ld_qkv + (part == 0 ? 0 : (a.heads + (part - 1) * a.kv.kv_heads) * hd) + in_part * 8;
  const float *cosb = turn ? a.cosb + (in_head >> 1) : nullptr, *sinb = turn ? a.sinb + (in_head >> 1) : nullptr;
  bf16* cache = reinterpret_cast<bf16*>(part == 1 ? a.kv.k : a.kv.v) + (size_t)head * page * hd + in_head;
  Raw raw[kEach];
  int number[kEach], off[kEach];  // of the page; place in it, negative: nothing to write
#pragma unroll
  for (int i = 0; i < kEach; ++i, from += a.ld_qkv) {
    const int row = row0 + i;
    off[i] = -1;
    number[i] = 0;
    if (row >= a.batch.n_tokens) continue;
    while (b < a.batch.n_seq && end <= row)
      if (++b < a.batch.n_seq) {
        end = a.batch.start[b + 1];
        s = span_of(a.batch, b, a.capacity, INT32_MAX, a.status);
      }
    if (b == a.batch.n_seq || s.n <= 0 || row < s.row) continue;
    const int pos = s.pos + row - s.row;
    if (pos >= a.n_positions) {
      atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
      continue;
    }
    raw[i] = fetch_eight(from, turn ? cosb + (size_t)pos * half : nullptr, turn ? sinb + (size_t)pos * half : nullptr);
    off[i] = 0;
    if (part != 0) {
      const int slot = a.by_page(pos);
      number[i] = a.kv.table[(size_t)b * a.kv.table_pitch + slot];
      off[i] = pos - slot * page;
    }
  }
  bf16* q = a.q + (size_t)row0 * a.ld_q + in_part * 8;
#pragma unroll
  for (int i = 0; i < kEach; ++i, q += a.ld_q) {
    if (off[i] < 0) continue;
    if ((unsigned)number[i] >= (unsigned)a.kv.n_pages) {
      atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
      continue;
    }
    store_eight(part == 0 ? q : cache + number[i] * a.kv.page_stride + off[i] * hd, turned(raw[i], turn));
  }
}

// Exponent of the smallest power of two, at least 2^-126, that brings a finite |x| within 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float largest) {
  const uint32_t u = __float_as_uint(largest);
  return max((int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
}
__device__ __forceinline__ uint2 to_e4m3(const Eight& e, float scale, bool power, float inverse) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t pair[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float2 f = make_float2(e.x[4 * i + 2 * j], e.x[4 * i + 2 * j + 1]);
      // dividing by a power of two is multiplying by its inverse
      f = power ? make_float2(f.x * inverse, f.y * inverse) : make_float2(__fdiv_rn(f.x, scale), __fdiv_rn(f.y, scale));
      pair[j] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
    }
    w[i] = pair[0] | pair[1] << 16;
  }
  return make_uint2(w[0], w[1]);
}

// One page and head of 8-bit keys or values by a team of T threads: the largest new value gives the scale, then the new rows
// are rounded, and the rows that the page held before if the scale has grown.  A thread keeps its first kKeep groups of eight in registers;
// others are read again, from L1 or L2.
//
// Unit u is a page that some sequence touches, found without a list: with U(b) = start[b] / page_size + 2 b sequence b has the
// units U(b) .. U(b + 1) - 1, at least as many as the pages its tokens can touch.
template <int T>
__device__ __forceinline__ void append_page(const Append& a, int unit, int head, bool values, int lane) {
  constexpr int kKeep = T == 32 ? 2 : 4;
  const int hd = a.kv.head_dim, half = hd >> 1, page = a.kv.page_size;
  const Found f = find<T>(a.batch, unit, lane, [&](int to, int i) { return a.by_page(max(to, 0)) + 2 * i; });
  const int b = f.b;
  if (b >= a.batch.n_seq) return;
  const Span s = span_of(f.row, f.end, f.pos, a.batch, a.capacity, INT32_MAX, a.status);
  if (s.n <= 0) return;
  const int ahead = unit - (a.by_page(s.row) + 2 * b), slot = a.by_page(s.pos) + ahead;
  if (ahead < 0 || slot > a.by_page(s.pos + s.n - 1)) return;
  const int p = a.kv.table[(size_t)b * a.kv.table_pitch + slot];
  const bool turn = !values && a.cosb;
  if (s.pos + s.n > a.n_positions && lane == 0) atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
  const int page0 = slot * page;
  const int lo = max(s.pos, page0) - page0, hi = min(min(s.pos + s.n, a.n_positions), page0 + page) - page0;  // new rows of the page
  if (hi <= lo) return;
  const bf16* in = a.qkv + (size_t)(s.row + page0 + lo - s.pos) * a.ld_qkv + (a.heads + (values ? a.kv.kv_heads : 0) + head) * hd;
  const float* c = turn ? a.cosb + (size_t)(page0 + lo) * half : nullptr;
  const float* n = turn ? a.sinb + (size_t)(page0 + lo) * half : nullptr;
  const int per_row = hd / 8, vecs = (hi - lo) * per_row;
  // group lane, lane + T ... of the rows: row and group within it
  const int step_rows = a.by_head(T), step_groups = T - step_rows * per_row;
  int r = a.by_head(lane), v = lane - r * per_row;
  auto fetch_next = [&]() {
    const size_t at = (size_t)r * half + v * 4;
    const Raw raw = fetch_eight(in + (size_t)r * a.ld_qkv + v * 8, turn ? c + at : nullptr, turn ? n + at : nullptr);
    r += step_rows;
    v += step_groups;
    if (v >= per_row) {
      v -= per_row;
      ++r;
    }
    return raw;
  };
  // the rows are on their way while the page's number arrives
  Raw raw[kKeep];
#pragma unroll
  for (int k = 0; k < kKeep; ++k)
    if (lane + k * T < vecs) raw[k] = fetch_next();
  if (p < 0 || p >= a.kv.n_pages) {
    if (lane == 0) atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
    return;
  }
  float* scale_at = (values ? a.kv.v_scale : a.kv.k_scale) + (size_t)p * a.kv.kv_heads + head;
  const float old = lo > 0 ? *scale_at : 0.f;
  const int r_kept = r, v_kept = v;
  float top = 0.f;
  auto look_at = [&](const Eight& e) {
    float most = fabsf(e.x[0]);  // maxima pass NaN over
#pragma unroll
    for (int j = 1; j < 8; ++j) most = fmaxf(most, fabsf(e.x[j]));
    if (most == INFINITY) {  // nor does what is infinite count
      most = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(e.x[j]) == INFINITY ? 0.f : fabsf(e.x[j]));
    }
    top = fmaxf(top, most);
  };
  Eight kept[kKeep];
#pragma unroll
  for (int k = 0; k < kKeep; ++k)
    if (lane + k * T < vecs) look_at(kept[k] = turned(raw[k], turn));
#pragma unroll 4
  for (int i = lane + kKeep * T; i < vecs; i += T) look_at(turned(fetch_next(), turn));
  top = warp_max(top);
  if constexpr (T > 32) {
    __shared__ float tops[T / 32];
    if ((lane & 31) == 0) tops[lane >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 32; ++i) top = fmaxf(top, tops[i]);
  }
  const float scale = fmaxf(old, __uint_as_float((uint32_t)(scale_exponent(top) + 127) << 23));
  unsigned char* out = reinterpret_cast<unsigned char*>(values ? a.kv.v : a.kv.k) + p * a.kv.page_stride + (size_t)head * page * hd;
  if (T > 32) __syncthreads();
  else __syncwarp();
  if (lane == 0) *scale_at = scale;  // all have read it
  const bool power = (__float_as_uint(scale) & 0x7fffffu) == 0 && scale < 1.7014118e38f;
  const float inverse = power ? __uint_as_float((254u << 23) - __float_as_uint(scale)) : 0.f;
#pragma unroll
  for (int k = 0; k < kKeep; ++k)
    if (lane + k * T < vecs)
      *reinterpret_cast<uint2*>(out + (size_t)lo * hd + (size_t)(lane + k * T) * 8) = to_e4m3(kept[k], scale, power, inverse);
  r = r_kept;
  v = v_kept;
#pragma unroll 4
  for (int i = lane + kKeep * T; i < vecs; i += T)
    *reinterpret_cast<uint2*>(out + (size_t)lo * hd + (size_t)i * 8) = to_e4m3(turned(fetch_next(), turn), scale, power, inverse);
  if (lo > 0 && old != scale) {
    const float ratio = __fdiv_rn(old, scale);
    for (int i = lane; i < lo * per_row; i += T) {
      uint2* at = reinterpret_cast<uint2*>(out + (size_t)i * 8);
      const uint2 u = *at;
      Eight e;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 2 ? u.x : u.y) >> (16 * (j & 1))), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        e.x[2 * j] = f.x * ratio;
        e.x[2 * j + 1] = f.y * ratio;
      }
      *at = to_e4m3(e, 1.f, true, 1.f);
    }
  }
}

// T: threads of a team that has a page and head, kEach: rows of a thread that rotates.
template <int T, int kEach>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const Append a) {
  pdl_trigger();
  pdl_wait();
  if ((int)blockIdx.x < a.rows_blocks) {
    append_rows<kEach>(a, blockIdx.x);
    return;
  }
  constexpr int teams = kThreads / T;
  const long long task = (long long)(blockIdx.x - a.rows_blocks) * teams + threadIdx.x / T;
  // heads within a unit: neighbours read the same rows
  const int per_unit = 2 * a.kv.kv_heads, unit = (int)(task / per_unit), rest = (int)(task - (long long)unit * per_unit);
  if (unit < a.units) append_page<T>(a, unit, rest >> 1, rest & 1, threadIdx.x % T);
}

}  // namespace

cudaError_t kv_append(const PagedKv& kv, const Batch& batch, int heads, const bf16* qkv, int ld_qkv, bf16* q, int ld_q,
                      const float* cosb, const float* sinb, int n_positions, int* status, cudaStream_t s) {
  if (batch.n_seq == 0 || batch.n_tokens == 0) return cudaSuccess;
  Append a = {kv, batch, qkv, q, cosb, sinb, ld_qkv, ld_q, heads, cosb ? n_positions : INT32_MAX};
  a.status = status;
  a.capacity = (int)min((long long)kv.table_pitch * kv.page_size, (long long)INT32_MAX);
  a.q_vec = q ? heads * kv.head_dim / 8 : 0;
  a.kv_vec = kv.e4m3 ? 0 : kv.kv_heads * kv.head_dim / 8;
  const int row_vec = a.q_vec + 2 * a.kv_vec;
  a.by_row = Div(row_vec ? row_vec : 1);
  a.by_head = Div(kv.head_dim / 8);
  a.by_page = Div(kv.page_size);
  // A warp a page and head, and a row a thread, where sequences bring a token or two; a block, and kMany rows, where they bring whole pages.
  const bool small = batch.n_tokens <= 4ll * batch.n_seq;
  const int each = small ? 1 : kMany;
  const long long vec = ((long long)batch.n_tokens + each - 1) / each * row_vec;
  if (vec > INT32_MAX - kThreads) return cudaErrorInvalidValue;
  a.rows_blocks = (int)((vec + kThreads - 1) / kThreads);
  long long tasks = 0;
  if (kv.e4m3) {
    a.units = batch.n_tokens / kv.page_size + 2 * batch.n_seq;
    tasks = (long long)a.units * 2 * kv.kv_heads;
  }
  const long long blocks = a.rows_blocks + (small ? (tasks * 32 + kThreads - 1) / kThreads : tasks);
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  return small ? launch_pdl(kv_append_kernel<32, 1>, dim3((unsigned)blocks), dim3(kThreads), 0, s, a)
               : launch_pdl(kv_append_kernel<kThreads, kMany>, dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
}

}  // namespace ane
