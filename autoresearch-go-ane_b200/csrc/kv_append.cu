// Appending keys and values to a paged cache, rotated by their positions on the way (ane_op_kv_append).
//
// Bound by HBM for prompts (q|k|v read, rotated q and the cache's rows written, once each) and by latency for single tokens.
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

constexpr int kThreads = 128;
constexpr int kEach = 4;  // groups of eight elements that a thread rotates

struct Append {
  PagedKv kv;
  Batch batch;
  const bf16* qkv;  // may be q: every element is read by the thread that writes it
  bf16* q;
  const float *cosb, *sinb;
  int ld_qkv, ld_q, heads, n_positions;
  int rows_blocks;  // blocks that rotate rows; the others are 8-bit pages
  int units;        // bound of the pages that are touched
  int* status;
};

// The last sequence whose first row is not behind `row` (a block's threads compare one sequence each, which is one round trip to
// memory where a binary search takes one for each halving); n_seq if all rows of sequences lie before it.
template <int T, class Less>
__device__ __forceinline__ int count_before(int n, int lane, Less before) {
  int c = 0;
  for (int i = lane; i < n; i += T) c += before(i) ? 1 : 0;
  if constexpr (T == 32) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    return c;
  } else {
    __shared__ int part[T / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if ((lane & 31) == 0) part[lane >> 5] = c;
    __syncthreads();
    c = 0;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) c += part[i];
    return c;
  }
}

// Eight elements of a row, rotated where cos / sin are given.  Products and sums are rounded one by one.
struct Eight {
  float x[8];
};
__device__ __forceinline__ Eight load_eight(const bf16* p, const float* c, const float* s) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e.x[2 * i] = __uint_as_float(w[i] << 16);
    e.x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  if (c) {
    const float4 c4 = *reinterpret_cast<const float4*>(c), s4 = *reinterpret_cast<const float4*>(s);
    const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = e.x[2 * i], b = e.x[2 * i + 1];
      e.x[2 * i] = __fsub_rn(__fmul_rn(a, cc[i]), __fmul_rn(b, ss[i]));
      e.x[2 * i + 1] = __fadd_rn(__fmul_rn(b, cc[i]), __fmul_rn(a, ss[i]));
    }
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

// kEach * kThreads groups of eight elements of the tokens' rows, in the order of memory: the queries of all caches, keys and values too of a
// bf16 one.
__device__ __forceinline__ void append_rows(const Append& a, int block) {
  const int tid = threadIdx.x;
  const int hd = a.kv.head_dim, half = hd >> 1, page = a.kv.page_size;
  const int capacity = (int)min((long long)a.kv.table_pitch * page, (long long)INT32_MAX);
  const int q_vec = a.q ? a.heads * hd / 8 : 0, kv_vec = a.kv.e4m3 ? 0 : a.kv.kv_heads * hd / 8, vec = q_vec + 2 * kv_vec;
  const long long begin = (long long)block * (kEach * kThreads);
  const int first = (int)(begin / vec), v0 = (int)(begin - (long long)first * vec);
  // the sequence of the block's first row; the next ones are found from there
  int b = count_before<kThreads>(a.batch.n_seq, tid, [&](int i) { return a.batch.start[i + 1] <= first; });
  Span s = {0, 0, 0};
  int known = -1;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int u = v0 + tid + i * kThreads, row = first + u / vec, v = u % vec;
    if (row >= a.batch.n_tokens) break;
    while (b < a.batch.n_seq && a.batch.start[b + 1] <= row) ++b;
    if (b == a.batch.n_seq) break;
    if (b != known) s = span_of(a.batch, known = b, capacity, INT32_MAX, a.status);
    if (s.n == 0 || row < s.row) continue;
    const int pos = s.pos + row - s.row;
    const int part = v < q_vec ? 0 : v < q_vec + kv_vec ? 1 : 2;
    const int col = (part == 0 ? v : v - q_vec - (part - 1) * kv_vec) * 8;  // within q, k or v
    const bool turn = part < 2 && a.cosb;
    if (turn && pos >= a.n_positions) {
      atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
      continue;
    }
    const int in_col = col + (part == 0 ? 0 : (a.heads + (part - 1) * a.kv.kv_heads) * hd);
    const int head = col / hd, in_head = col - head * hd;
    const size_t at = (size_t)pos * half + (in_head >> 1);
    const Eight e = load_eight(a.qkv + (size_t)row * a.ld_qkv + in_col, turn ? a.cosb + at : nullptr, turn ? a.sinb + at : nullptr);
    if (part == 0) {
      store_eight(a.q + (size_t)row * a.ld_q + col, e);
      continue;
    }
    const int slot = pos / page, p = a.kv.table[(size_t)b * a.kv.table_pitch + slot];
    if (p < 0 || p >= a.kv.n_pages) {
      atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
      continue;
    }
    bf16* cache = reinterpret_cast<bf16*>(part == 1 ? a.kv.k : a.kv.v);
    store_eight(cache + p * a.kv.page_stride + ((size_t)head * page + pos - slot * page) * hd + in_head, e);
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
// are rounded, and the rows that the page held before if the scale has grown.  The page's rows are read twice: the
// second time they are in L1 or L2.
//
// Unit u is a page that some sequence touches, found without a list: with U(b) = start[b] / page_size + 2 b sequence b has the
// units U(b) .. U(b + 1) - 1, at least as many as the pages its tokens can touch.
template <int T>
__device__ __forceinline__ void append_page(const Append& a, int unit, int head, bool values, int lane) {
  const int hd = a.kv.head_dim, half = hd >> 1, page = a.kv.page_size;
  const int capacity = (int)min((long long)a.kv.table_pitch * page, (long long)INT32_MAX);
  const int b = count_before<T>(a.batch.n_seq, lane, [&](int i) { return a.batch.start[i + 1] / page + 2 * (i + 1) <= unit; });
  if (b >= a.batch.n_seq) return;
  const Span s = span_of(a.batch, b, capacity, INT32_MAX, a.status);
  const int ahead = unit - (a.batch.start[b] / page + 2 * b), slot = s.pos / page + ahead;
  if (s.n == 0 || ahead < 0 || slot > (s.pos + s.n - 1) / page) return;
  const int p = a.kv.table[(size_t)b * a.kv.table_pitch + slot];
  if (p < 0 || p >= a.kv.n_pages || (!values && a.cosb && s.pos + s.n > a.n_positions)) {
    if (lane == 0) atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
    return;
  }
  const int page0 = slot * page;
  const int lo = max(s.pos, page0) - page0, hi = min(s.pos + s.n, page0 + page) - page0;  // new rows of the page
  const bf16* in = a.qkv + (size_t)(s.row + page0 + lo - s.pos) * a.ld_qkv + (a.heads + (values ? a.kv.kv_heads : 0) + head) * hd;
  const bool turn = !values && a.cosb;
  const float* c = turn ? a.cosb + (size_t)(page0 + lo) * half : nullptr;
  const float* n = turn ? a.sinb + (size_t)(page0 + lo) * half : nullptr;
  const int per_row = hd / 8, vecs = (hi - lo) * per_row;
  auto load = [&](int i) {
    const int r = i / per_row, v = i - r * per_row;
    const size_t at = (size_t)r * half + v * 4;
    return load_eight(in + (size_t)r * a.ld_qkv + v * 8, turn ? c + at : nullptr, turn ? n + at : nullptr);
  };
  float top = 0.f;
#pragma unroll 4
  for (int i = lane; i < vecs; i += T) {
    const Eight e = load(i);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = fabsf(e.x[j]);
      if (x <= 3.402823466e38f) top = fmaxf(top, x);  // not what is infinite or NaN
    }
  }
  top = warp_max(top);
  if constexpr (T > 32) {
    __shared__ float tops[T / 32];
    if ((lane & 31) == 0) tops[lane >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 32; ++i) top = fmaxf(top, tops[i]);
  }
  float* scale_at = (values ? a.kv.v_scale : a.kv.k_scale) + (size_t)p * a.kv.kv_heads + head;
  const float old = lo > 0 ? *scale_at : 0.f;
  const float scale = fmaxf(old, __uint_as_float((uint32_t)(scale_exponent(top) + 127) << 23));
  unsigned char* out = reinterpret_cast<unsigned char*>(values ? a.kv.v : a.kv.k) + p * a.kv.page_stride + (size_t)head * page * hd;
  if (T > 32) __syncthreads();
  else __syncwarp();
  if (lane == 0) *scale_at = scale;  // all have read it
  const bool power = (__float_as_uint(scale) & 0x7fffffu) == 0 && scale < 1.7014118e38f;
  const float inverse = power ? __uint_as_float((254u << 23) - __float_as_uint(scale)) : 0.f;
#pragma unroll 4
  for (int i = lane; i < vecs; i += T)
    *reinterpret_cast<uint2*>(out + (size_t)lo * hd + (size_t)i * 8) = to_e4m3(load(i), scale, power, inverse);
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

template <int T>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const Append a) {
  pdl_trigger();
  pdl_wait();
  if ((int)blockIdx.x < a.rows_blocks) {
    append_rows(a, blockIdx.x);
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
  Append a = {kv, batch, qkv, q, cosb, sinb, ld_qkv, ld_q, heads, n_positions, 0, 0, status};
  const long long vec = (long long)batch.n_tokens * ((q ? heads : 0) + (kv.e4m3 ? 0 : 2 * kv.kv_heads)) * kv.head_dim / 8;
  if ((vec + kEach * kThreads - 1) / (kEach * kThreads) > INT32_MAX) return cudaErrorInvalidValue;
  a.rows_blocks = (int)((vec + kEach * kThreads - 1) / (kEach * kThreads));
  long long tasks = 0;
  if (kv.e4m3) {
    a.units = batch.n_tokens / kv.page_size + 2 * batch.n_seq;
    tasks = (long long)a.units * 2 * kv.kv_heads;
  }
  // a warp a page and head where sequences bring a token or two, a block where they bring whole pages
  const bool small = batch.n_tokens <= 4ll * batch.n_seq;
  const long long blocks = a.rows_blocks + (small ? (tasks * 32 + kThreads - 1) / kThreads : tasks);
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  return small ? launch_pdl(kv_append_kernel<32>, dim3((unsigned)blocks), dim3(kThreads), 0, s, a)
               : launch_pdl(kv_append_kernel<kThreads>, dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
}

}  // namespace ane
