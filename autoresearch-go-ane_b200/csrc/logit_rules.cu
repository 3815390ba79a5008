// Penalties, biases and grammar masks on rows of logits (ane_op_logit_rules).
//
// Bound by HBM: logits in, logits out, once each.  A block takes a stretch of a row's vocabulary.  It counts the row's tokens that
// fall into the stretch in shared memory (integers: the order of the additions does not matter) while its first logits are on
// their way, and then goes over the stretch once.  Short stretches give few rows enough blocks, long ones read the row's token list
// less often.
#include "serving.h"

namespace ane {
namespace {

constexpr int kThreads = 256;

// What a stretch keeps of a token: how often it is in the output, whether it is in the prompt, and 1 + its last bias' place in the row's
// list.  32 bits where token lists are shorter than 2^15, 64 otherwise.
template <class W>
struct Entry;
template <>
struct Entry<uint32_t> {
  static constexpr int kBias = 16;
  static constexpr uint32_t kSeen = 1u << 15, kCount = kSeen - 1;
};
template <>
struct Entry<unsigned long long> {
  static constexpr int kBias = 32;
  static constexpr unsigned long long kSeen = 1ull << 31, kCount = kSeen - 1;
};

struct Rules {
  ane_logit_rules_args a;
  int* status;
  bool vec;  // 16-byte fp32 and 8-byte bf16 accesses are aligned
};

template <bool BF>
__device__ __forceinline__ float4 load4(const Rules& r, size_t at, int n) {
  if (r.vec && n >= 4) {
    if (!BF) return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(r.a.d_logits) + at);
    const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const bf16*>(r.a.d_logits) + at);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
  }
  float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) x[i] = BF ? __bfloat162float(reinterpret_cast<const bf16*>(r.a.d_logits)[at + i]) : reinterpret_cast<const float*>(r.a.d_logits)[at + i];
  return make_float4(x[0], x[1], x[2], x[3]);
}

template <bool BF, int kStretch, class W>
__global__ void __launch_bounds__(kThreads) logit_rules_kernel(const Rules r) {
  using E = Entry<W>;
  constexpr int kEach = kStretch / (kThreads * 4);  // groups of four logits of a thread
  __shared__ __align__(16) W seen[kStretch];
  const ane_logit_rules_args& a = r.a;
  pdl_trigger();
  const int row = blockIdx.y, v0 = blockIdx.x * kStretch, tid = threadIdx.x;
  const int len = min(kStretch, a.vocab - v0);
  const bool marks = a.d_tokens || a.d_bias_start;
  if (marks)
    for (int i = tid; i < kStretch * (int)sizeof(W) / 16; i += kThreads) reinterpret_cast<uint4*>(seen)[i] = make_uint4(0, 0, 0, 0);
  pdl_wait();
  float4 x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int v = (i * kThreads + tid) * 4;
    if (v < len) x[i] = load4<BF>(r, (size_t)row * a.ld_logits + v0 + v, len - v);
  }
  const uint32_t* mask = nullptr;
  if (a.d_mask) {
    const int m = a.d_mask_row ? a.d_mask_row[row] : row;
    if (m >= a.n_masks) {
      if (tid == 0) atomicCAS(r.status, DEV_OK, DEV_BAD_INDEX);
    } else if (m >= 0) {
      mask = a.d_mask + (size_t)m * a.ld_mask;
    }
  }
  if (marks) __syncthreads();
  int first_bias = 0;
  if (a.d_bias_start) {
    first_bias = a.d_bias_start[row];
    int n = a.d_bias_start[row + 1] - first_bias;
    if (n < 0 || n > 65535 || first_bias < 0) {
      if (tid == 0) atomicCAS(r.status, DEV_OK, DEV_BAD_INDEX);
      n = 0;
    }
    for (int i = tid; i < n; i += kThreads) {
      const int t = a.d_bias_token[first_bias + i];
      if (t >= v0 && t - v0 < len) atomicMax(seen + (t - v0), (W)(i + 1) << E::kBias);  // nothing else is there yet
    }
    __syncthreads();
  }
  if (a.d_tokens) {
    int n = a.d_n_tokens[row];
    if (n < 0 || n > a.ld_tokens) {
      if (tid == 0) atomicCAS(r.status, DEV_OK, DEV_BAD_INDEX);
      n = 0;
    }
    const int prompt = a.d_n_prompt ? a.d_n_prompt[row] : 0;
    const int* tokens = a.d_tokens + (size_t)row * a.ld_tokens;
    // eight at a time, so that as many are on their way
    for (int i0 = 0; i0 < n; i0 += 8 * kThreads) {
      int t[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k * kThreads + tid;
        t[k] = i < n ? tokens[i] - v0 : -1;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if ((unsigned)t[k] >= (unsigned)len) continue;
        if (i0 + k * kThreads + tid < prompt) atomicOr(seen + t[k], E::kSeen);
        else atomicAdd(seen + t[k], (W)1);
      }
    }
  }
  const float rep = a.d_repetition ? a.d_repetition[row] : 1.f, freq = a.d_frequency ? a.d_frequency[row] : 0.f;
  const float pres = a.d_presence ? a.d_presence[row] : 0.f;
  if (marks) __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int v = (i * kThreads + tid) * 4;
    if (v >= len) break;
    float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    if (marks) {
      W c[4];
#pragma unroll
      for (int k = 0; k < (int)sizeof(W) / 4; ++k) reinterpret_cast<uint4*>(c)[k] = reinterpret_cast<const uint4*>(seen + v)[k];
      if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c[k] & (E::kSeen | E::kCount)) {
            if (a.d_repetition) y[k] = y[k] > 0.f ? __fdiv_rn(y[k], rep) : __fmul_rn(y[k], rep);
            const uint32_t n = (uint32_t)(c[k] & E::kCount);
            if (n) {
              if (a.d_frequency) y[k] = __fsub_rn(y[k], __fmul_rn(freq, (float)n));
              if (a.d_presence) y[k] = __fsub_rn(y[k], pres);
            }
          }
          const uint32_t at = (uint32_t)(c[k] >> E::kBias);
          if (at) y[k] = __fadd_rn(y[k], a.d_bias[first_bias + at - 1]);
        }
      }
    }
    if (mask) {
      const uint32_t bits = mask[(v0 + v) >> 5] >> ((v0 + v) & 31);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (!(bits >> k & 1u)) y[k] = -INFINITY;
    }
    float* out = a.d_out + (size_t)row * a.ld_out + v0 + v;
    if (r.vec && len - v >= 4) {
      *reinterpret_cast<float4*>(out) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (v + k < len) out[k] = y[k];
    }
  }
}

template <bool BF, int kStretch, class W>
cudaError_t run(const Rules& r, cudaStream_t s) {
  // rows in slices of what a grid's second dimension holds
  for (int row = 0; row < r.a.rows; row += 65535) {
    Rules part = r;
    ane_logit_rules_args& a = part.a;
    a.rows = r.a.rows - row < 65535 ? r.a.rows - row : 65535;
    a.d_logits = reinterpret_cast<const char*>(r.a.d_logits) + (size_t)row * r.a.ld_logits * (BF ? 2 : 4);
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
    const dim3 grid((unsigned)((a.vocab + kStretch - 1) / kStretch), (unsigned)a.rows);
    const cudaError_t e = launch_pdl(logit_rules_kernel<BF, kStretch, W>, grid, dim3(kThreads), 0, s, part);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t logit_rules(const ane_logit_rules_args& a, int* status, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  const bool bf = a.dtype == ANE_DTYPE_BF16;
  const Rules r = {a, status, reinterpret_cast<uintptr_t>(a.d_logits) % (bf ? 8 : 16) == 0 && a.ld_logits % 4 == 0 &&
                                  reinterpret_cast<uintptr_t>(a.d_out) % 16 == 0 && a.ld_out % 4 == 0};
  const bool few = (long long)a.rows * a.vocab <= 1024ll * 1024;
  if (a.d_tokens && a.ld_tokens >= 1 << 15) return bf ? run<true, 4096, unsigned long long>(r, s) : run<false, 4096, unsigned long long>(r, s);
  if (bf) return few ? run<true, 1024, uint32_t>(r, s) : run<true, 4096, uint32_t>(r, s);
  return few ? run<false, 1024, uint32_t>(r, s) : run<false, 4096, uint32_t>(r, s);
}

}  // namespace ane
