// Penalties, biases and grammar masks on rows of logits (ane_op_logit_rules).
//
// Bound by HBM: logits in, logits out, once each.  Many logits take two kernels: one copies them, masked, which needs no token; the other, a
// block a row, reads the row's lists once, gathers what there is to know of each token in a table in shared memory, and forms
// the few logits again that there is something to know of.  Few logits take one kernel, which saves a launch: a block has a short
// stretch of a row's vocabulary, counts the row's tokens that fall into it and goes over the stretch.  Counts and marks are
// integers, so that the order does not matter.
// 255 rows of 128000 bf16 logits with lists of 6000 tokens take 63 us (3.2 TB/s; 38 the copy, the floor is 31), 64 of 32000 fp32 9.4 us, one 3.0.
#include "serving.h"

namespace ane {
namespace {

struct Rules {
  ane_logit_rules_args a;
  int* status;
  bool vec;  // 16-byte accesses are aligned
};

constexpr int kGroup = 8;  // logits that a thread copies at a time
// 64 rows of 32000 logits take 9.4 us in one kernel and 12.8 in two, 16 of 128000 12.4 and 15.1; 128 of 32000 19.3 and 15.8, 32 of 128000 22.2
// and 20.5, 255 of 128000 180 and 63.
constexpr long long kFewLogits = 3 << 20;

template <bool BF>
struct Logits {  // kGroup of them, as they are stored
  uint4 x[BF ? 1 : 2];
  __device__ __forceinline__ float get(int i) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
    if (BF) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    return __uint_as_float(w[i]);
  }
};
template <bool BF>
__device__ __forceinline__ Logits<BF> load_logits(const void* logits, size_t at, int n, bool vec) {
  Logits<BF> f = {};
  const char* p = reinterpret_cast<const char*>(logits) + at * (BF ? 2 : 4);
  if (vec && n >= kGroup) {
#pragma unroll
    for (int i = 0; i < (BF ? 1 : 2); ++i) f.x[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(f.x);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      if (i >= n) break;
      if (BF) w[i >> 1] |= (uint32_t)reinterpret_cast<const unsigned short*>(p)[i] << (16 * (i & 1));
      else w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
  }
  return f;
}

// What there is to know of a token: how often the row's output names it, whether its prompt does, and the place of its last bias in the row's
// list, from 1.  Rules in the order of the header, each operation rounded.
struct Known {
  uint32_t count, bias;
  bool seen;
};
struct Penalties {
  float rep, freq, pres;
};
__device__ __forceinline__ Penalties penalties(const ane_logit_rules_args& a, int row) {
  return {a.d_repetition ? a.d_repetition[row] : 1.f, a.d_frequency ? a.d_frequency[row] : 0.f, a.d_presence ? a.d_presence[row] : 0.f};
}
__device__ __forceinline__ float ruled(const ane_logit_rules_args& a, float y, const Known& k, const Penalties& p, float bias) {
  if (k.seen || k.count) {
    if (a.d_repetition) y = y > 0.f ? __fdiv_rn(y, p.rep) : __fmul_rn(y, p.rep);
    if (k.count) {
      if (a.d_frequency) y = __fsub_rn(y, __fmul_rn(p.freq, (float)k.count));
      if (a.d_presence) y = __fsub_rn(y, p.pres);
    }
  }
  return k.bias ? __fadd_rn(y, bias) : y;
}

// A row's lists, none where their sizes make no sense.
struct Lists {
  const int* tokens;
  int n_tokens, prompt, first_bias, n_bias;
};
__device__ __forceinline__ Lists lists_of(const Rules& r, int row) {
  const ane_logit_rules_args& a = r.a;
  Lists l = {nullptr, 0, 0, 0, 0};
  if (a.d_tokens) {
    l.tokens = a.d_tokens + (size_t)row * a.ld_tokens;
    l.n_tokens = a.d_n_tokens[row];
    if (a.d_n_prompt) l.prompt = a.d_n_prompt[row];
  }
  if (a.d_bias_start) {
    l.first_bias = a.d_bias_start[row];
    l.n_bias = a.d_bias_start[row + 1] - l.first_bias;
  }
  const bool no_tokens = l.n_tokens < 0 || l.n_tokens > a.ld_tokens, no_bias = l.n_bias < 0 || l.n_bias > 65535 || l.first_bias < 0;
  if ((no_tokens || no_bias) && threadIdx.x == 0) atomicCAS(r.status, DEV_OK, DEV_BAD_INDEX);
  if (no_tokens) l.n_tokens = 0;
  if (no_bias) l.n_bias = 0;
  return l;
}
// The row's mask; nullptr: all are allowed.
__device__ __forceinline__ const uint32_t* mask_of(const Rules& r, int row) {
  const ane_logit_rules_args& a = r.a;
  if (!a.d_mask) return nullptr;
  const int m = a.d_mask_row ? a.d_mask_row[row] : row;
  if (m >= a.n_masks && threadIdx.x == 0) atomicCAS(r.status, DEV_OK, DEV_BAD_INDEX);
  return m < 0 || m >= a.n_masks ? nullptr : a.d_mask + (size_t)m * a.ld_mask;
}

template <bool BF>
__device__ __forceinline__ void store_masked(const Rules& r, int row, int v, int n, const Logits<BF>& x, uint32_t bits) {
  float* out = r.a.d_out + (size_t)row * r.a.ld_out + v;
  float y[kGroup];
#pragma unroll
  for (int k = 0; k < kGroup; ++k) y[k] = bits >> k & 1u ? x.get(k) : -INFINITY;
  if (r.vec && n >= kGroup) {
#pragma unroll
    for (int k = 0; k < kGroup; k += 4) *reinterpret_cast<float4*>(out + k) = make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]);
  } else {
#pragma unroll
    for (int k = 0; k < kGroup; ++k)
      if (k < n) out[k] = y[k];
  }
}

// ---- few logits: one kernel ---------------------------------------------------------------------------------------------------------
// W: 16 bits of count and mark and 16 of bias for lists below 2^15, 32 of each for others.
template <bool BF, class W>
__global__ void __launch_bounds__(256) rules_stretch_kernel(const Rules r) {
  constexpr int kThreads = 256, kStretch = 1024, kBias = 4 * sizeof(W);
  constexpr W kSeen = (W)1 << (kBias - 1), kCount = kSeen - 1;
  constexpr int kAtOnce = 4;  // tokens of a thread that are on their way together
  __shared__ __align__(16) W known[kStretch];
  const ane_logit_rules_args& a = r.a;
  pdl_trigger();
  const int row = blockIdx.y, v0 = blockIdx.x * kStretch, tid = threadIdx.x, len = min(kStretch, a.vocab - v0);
  for (int i = tid; i < kStretch; i += kThreads) known[i] = 0;
  pdl_wait();
  float x[kStretch / kThreads];
#pragma unroll
  for (int i = 0; i < kStretch / kThreads; ++i) {
    const int v = i * kThreads + tid;
    const size_t at = (size_t)row * a.ld_logits + v0 + v;
    if (v < len) x[i] = BF ? __bfloat162float(reinterpret_cast<const bf16*>(a.d_logits)[at]) : reinterpret_cast<const float*>(a.d_logits)[at];
  }
  const Lists l = lists_of(r, row);
  const uint32_t* mask = mask_of(r, row);
  const Penalties p = penalties(a, row);
  int t[kAtOnce];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = i0 + k * kThreads + tid;
      t[k] = i < l.n_tokens ? l.tokens[i] - v0 : -1;
    }
  };
  fetch(0);
  __syncthreads();
  if (l.n_bias) {
    for (int i = tid; i < l.n_bias; i += kThreads) {
      const int at = a.d_bias_token[l.first_bias + i] - v0;
      if ((unsigned)at < (unsigned)len) atomicMax(known + at, (W)(i + 1) << kBias);  // nothing else is there yet
    }
    __syncthreads();
  }
  for (int i0 = 0; i0 < l.n_tokens; i0 += kAtOnce * kThreads) {
    if (i0) fetch(i0);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if ((unsigned)t[k] >= (unsigned)len) continue;
      if (i0 + k * kThreads + tid < l.prompt) atomicOr(known + t[k], kSeen);
      else atomicAdd(known + t[k], (W)1);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kStretch / kThreads; ++i) {
    const int v = i * kThreads + tid;
    if (v >= len) break;
    float y = x[i];
    const W c = known[v];
    if (c) {
      const Known k = {(uint32_t)(c & kCount), (uint32_t)(c >> kBias), (c & kSeen) != 0};
      y = ruled(a, y, k, p, k.bias ? a.d_bias[l.first_bias + k.bias - 1] : 0.f);
    }
    if (mask && !(mask[(v0 + v) >> 5] >> ((v0 + v) & 31) & 1u)) y = -INFINITY;
    a.d_out[(size_t)row * a.ld_out + v0 + v] = y;
  }
}

// ---- many logits: copies, then the ones to be formed ----------------------------------------------------------------------------------
template <bool BF>
__global__ void __launch_bounds__(256) rules_copy_kernel(const Rules r) {
  constexpr int kThreads = 256, kEach = 4, kStretch = kThreads * kEach * kGroup;
  const ane_logit_rules_args& a = r.a;
  pdl_trigger();
  const int row = blockIdx.y, v0 = blockIdx.x * kStretch + threadIdx.x * kGroup;
  pdl_wait();
  Logits<BF> x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int v = v0 + i * kThreads * kGroup;
    if (v < a.vocab) x[i] = load_logits<BF>(a.d_logits, (size_t)row * a.ld_logits + v, a.vocab - v, r.vec);
  }
  const uint32_t* mask = mask_of(r, row);
  uint32_t bits[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int v = v0 + i * kThreads * kGroup;
    bits[i] = mask && v < a.vocab ? mask[v >> 5] >> (v & 31) : ~0u;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int v = v0 + i * kThreads * kGroup;
    if (v < a.vocab) store_masked<BF>(r, row, v, a.vocab - v, x[i], bits[i]);
  }
}

// A row's table: an open one by a hash of the token where its lists are short, of which a quarter stays empty; else passes over ranges of the
// vocabulary with an entry for every token.
template <int kBits>
struct Table {
  static constexpr int kSlots = 1 << kBits, kMostUsed = kSlots / 4 * 3, kThreads = kSlots / 16;
  static constexpr size_t kBytes = (size_t)kSlots * 8 + kMostUsed * 2;
};

template <bool BF, int kBits>
__global__ void __launch_bounds__(Table<kBits>::kThreads) rules_form_kernel(const Rules r) {
  constexpr int kSlots = Table<kBits>::kSlots, kMostUsed = Table<kBits>::kMostUsed, kThreads = Table<kBits>::kThreads, kAtOnce = 4;
  constexpr uint32_t kNone = 0xffffffffu;
  extern __shared__ __align__(16) uint32_t table[];
  uint32_t *first = table, *second = table + kSlots;
  unsigned short* used = reinterpret_cast<unsigned short*>(second + kSlots);  // [kMostUsed] slots of the open table
  __shared__ int n_used;
  const ane_logit_rules_args& a = r.a;
  pdl_trigger();
  const int row = blockIdx.x, tid = threadIdx.x;
  pdl_wait();
  const Lists l = lists_of(r, row);
  const uint32_t* mask = mask_of(r, row);
  const Penalties p = penalties(a, row);
  // Forms the logits of n entries: what(i, token) is known of entry i, if anything.
  auto form = [&](int n, auto what) {
#pragma unroll 1
    for (int i0 = tid; i0 < n; i0 += kAtOnce * kThreads) {
      Known k[kAtOnce];
      float x[kAtOnce], bias[kAtOnce];
      bool write[kAtOnce];
      int v[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        write[j] = false;
        if (i0 + j * kThreads >= n) continue;
        k[j] = what(i0 + j * kThreads, v[j]);
        write[j] = k[j].seen || k[j].count || k[j].bias;
        if (!write[j]) continue;
        const size_t at = (size_t)row * a.ld_logits + v[j];  // where the output is the input, an allowed logit is still what it was
        x[j] = BF ? __bfloat162float(reinterpret_cast<const bf16*>(a.d_logits)[at]) : reinterpret_cast<const float*>(a.d_logits)[at];
        if (mask) write[j] = mask[v[j] >> 5] >> (v[j] & 31) & 1u;
        bias[j] = k[j].bias ? a.d_bias[l.first_bias + k[j].bias - 1] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (write[j]) a.d_out[(size_t)row * a.ld_out + v[j]] = ruled(a, x[j], k[j], p, bias[j]);
    }
  };
  // what(i, token) for the list's tokens
  auto each_token = [&](auto what) {
#pragma unroll 1
    for (int i0 = tid; i0 < l.n_tokens; i0 += kAtOnce * kThreads) {
      int t[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) t[j] = i0 + j * kThreads < l.n_tokens ? l.tokens[i0 + j * kThreads] : -1;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if ((unsigned)t[j] < (unsigned)a.vocab) what(i0 + j * kThreads, t[j]);
    }
  };
  auto each_bias = [&](auto what) {
    for (int i = tid; i < l.n_bias; i += kThreads) {
      const int t = a.d_bias_token[l.first_bias + i];
      if ((unsigned)t < (unsigned)a.vocab) what(i, t);
    }
  };
  if (l.n_tokens + l.n_bias <= kMostUsed) {
    // first: the token, second: kBits of count, one of mark, the others of bias
    constexpr uint32_t kSeen = 1u << kBits;
    static_assert(2 * kBits + 1 <= 32, "counts and places fit");
    for (int i = tid; i < kSlots / 4; i += kThreads) {
      reinterpret_cast<uint4*>(first)[i] = make_uint4(kNone, kNone, kNone, kNone);
      reinterpret_cast<uint4*>(second)[i] = make_uint4(0, 0, 0, 0);
    }
    if (tid == 0) n_used = 0;
    __syncthreads();
    auto slot_of = [&](int v) {  // there is an empty one: at most kMostUsed tokens are asked for
      uint32_t at = (uint32_t)v * 2654435761u >> (32 - kBits);
      for (;; at = (at + 1) % kSlots) {
        const uint32_t was = atomicCAS(first + at, kNone, (uint32_t)v);
        if (was == kNone) used[atomicAdd(&n_used, 1)] = (unsigned short)at;
        if (was == kNone || was == (uint32_t)v) return second + at;
      }
    };
    if (l.n_bias) {
      each_bias([&](int i, int v) { atomicMax(slot_of(v), (uint32_t)(i + 1) << (kBits + 1)); });  // nothing else is there yet
      __syncthreads();
    }
    each_token([&](int i, int v) {
      if (i < l.prompt) atomicOr(slot_of(v), kSeen);
      else atomicAdd(slot_of(v), 1u);
    });
    __syncthreads();
    form(n_used, [&](int i, int& v) {
      const uint32_t at = used[i], c = second[at];
      v = (int)first[at];
      return Known{c & (kSeen - 1), c >> (kBits + 1), (c & kSeen) != 0};
    });
    return;
  }
  // first: the bias, second: the count and, as its highest bit, the mark
  for (int v0 = 0; v0 < a.vocab; v0 += kSlots) {
    for (int i = tid; i < kSlots / 2; i += kThreads) reinterpret_cast<uint4*>(first)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    each_bias([&](int i, int v) {
      if ((unsigned)(v - v0) < (unsigned)kSlots) atomicMax(first + (v - v0), (uint32_t)(i + 1));
    });
    each_token([&](int i, int v) {
      if ((unsigned)(v - v0) >= (unsigned)kSlots) return;
      if (i < l.prompt) atomicOr(second + (v - v0), 1u << 31);
      else atomicAdd(second + (v - v0), 1u);
    });
    __syncthreads();
    form(kSlots, [&](int i, int& v) {
      v = v0 + i;
      return Known{second[i] & 0x7fffffffu, first[i], second[i] >> 31 != 0};
    });
    __syncthreads();
  }
}

// Rows in slices of what a grid's second dimension holds.
template <class Launch>
cudaError_t by_rows(const Rules& r, Launch launch) {
  for (int row = 0; row < r.a.rows; row += 65535) {
    Rules part = r;
    ane_logit_rules_args& a = part.a;
    a.rows = r.a.rows - row < 65535 ? r.a.rows - row : 65535;
    a.d_logits = reinterpret_cast<const char*>(r.a.d_logits) + (size_t)row * r.a.ld_logits * (a.dtype == ANE_DTYPE_BF16 ? 2 : 4);
    a.d_out += (size_t)row * r.a.ld_out;
    if (a.d_tokens) {
      a.d_tokens += (size_t)row * a.ld_tokens;
      a.d_n_tokens += row;
      if (a.d_n_prompt) a.d_n_prompt += row;
    }
    if (a.d_mask) {
      if (a.d_mask_row) {
        a.d_mask_row += row;
      } else {
        a.d_mask += (size_t)row * a.ld_mask;
        a.n_masks -= row;
      }
    }
    if (a.d_bias_start) a.d_bias_start += row;
    if (a.d_repetition) a.d_repetition += row;
    if (a.d_presence) a.d_presence += row;
    if (a.d_frequency) a.d_frequency += row;
    const cudaError_t e = launch(part);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <bool BF>
cudaError_t run(const Rules& r, cudaStream_t s) {
  const ane_logit_rules_args& all = r.a;
  const bool lists = all.d_tokens || all.d_bias_start;
  const unsigned stretches = (unsigned)(((long long)all.vocab + 1023) / 1024);
  if ((long long)all.rows * all.vocab <= kFewLogits)
    return by_rows(r, [&](const Rules& p) {
      const dim3 grid(stretches, (unsigned)p.a.rows);
      return all.d_tokens && all.ld_tokens >= 1 << 15 ? launch_pdl(rules_stretch_kernel<BF, unsigned long long>, grid, dim3(256), 0, s, p)
                                                      : launch_pdl(rules_stretch_kernel<BF, uint32_t>, grid, dim3(256), 0, s, p);
    });
  // the table is open for lists of up to three quarters of its slots; room for a thousand biases
  const bool small = !all.d_tokens || all.ld_tokens <= Table<13>::kMostUsed - 1024;
  static unsigned long long opted[2] = {0, 0};
  if (!(small ? smem_opt_in(rules_form_kernel<BF, 13>, Table<13>::kBytes, opted[0]) : smem_opt_in(rules_form_kernel<BF, 14>, Table<14>::kBytes, opted[1])))
    return cudaGetLastError();
  const bool same = all.d_logits == all.d_out;
  return by_rows(r, [&](const Rules& p) {
    cudaError_t e = cudaSuccess;
    if (!same || all.d_mask) e = launch_pdl(rules_copy_kernel<BF>, dim3((stretches + 7) / 8, (unsigned)p.a.rows), dim3(256), 0, s, p);
    if (e != cudaSuccess || !lists) return e;
    const dim3 grid((unsigned)p.a.rows);
    return small ? launch_pdl(rules_form_kernel<BF, 13>, grid, dim3(Table<13>::kThreads), Table<13>::kBytes, s, p)
                 : launch_pdl(rules_form_kernel<BF, 14>, grid, dim3(Table<14>::kThreads), Table<14>::kBytes, s, p);
  });
}

}  // namespace

cudaError_t logit_rules(const ane_logit_rules_args& a, int* status, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  const bool bf = a.dtype == ANE_DTYPE_BF16;
  const Rules r = {a, status, reinterpret_cast<uintptr_t>(a.d_logits) % 16 == 0 && a.ld_logits % (bf ? 8 : 4) == 0 &&
                                  reinterpret_cast<uintptr_t>(a.d_out) % 16 == 0 && a.ld_out % 4 == 0};
  return bf ? run<true>(r, s) : run<false>(r, s);
}

}  // namespace ane
