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
constexpr uint32_t kCount = 0xffffffu, kSeen = 1u << 24;  // entry of a token: how often in the output, and whether at all

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

template <bool BF, int kStretch>
__global__ void __launch_bounds__(kThreads) logit_rules_kernel(const Rules r) {
  constexpr int kEach = kStretch / (kThreads * 4);  // groups of four logits of a thread
  extern __shared__ uint32_t shared[];
  uint32_t* seen = shared;                                                   // [kStretch]
  uint32_t* bias_at = shared + (r.a.d_tokens ? kStretch : 0);  // [kStretch]: 1 + entry in the row's list
  const ane_logit_rules_args& a = r.a;
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.y, v0 = blockIdx.x * kStretch, tid = threadIdx.x;
  const int len = min(kStretch, a.vocab - v0);
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
  if (a.d_tokens)
    for (int i = tid; i < len; i += kThreads) seen[i] = 0;
  if (a.d_bias_start)
    for (int i = tid; i < len; i += kThreads) bias_at[i] = 0;
  __syncthreads();
  if (a.d_tokens) {
    int n = a.d_n_tokens[row];
    if (n < 0 || n > a.ld_tokens) {
      if (tid == 0) atomicCAS(r.status, DEV_OK, DEV_BAD_INDEX);
      n = 0;
    }
    const int prompt = a.d_n_prompt ? a.d_n_prompt[row] : 0;
    const int* tokens = a.d_tokens + (size_t)row * a.ld_tokens;
#pragma unroll 4
    for (int i = tid; i < n; i += kThreads) {
      const int t = tokens[i];
      if (t < v0 || t - v0 >= len) continue;
      if (i < prompt) atomicOr(seen + (t - v0), kSeen);
      else atomicAdd(seen + (t - v0), 1u);
    }
  }
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
      if (t >= v0 && t - v0 < len) atomicMax(bias_at + (t - v0), (uint32_t)i + 1u);
    }
  }
  const float rep = a.d_repetition ? a.d_repetition[row] : 1.f, freq = a.d_frequency ? a.d_frequency[row] : 0.f;
  const float pres = a.d_presence ? a.d_presence[row] : 0.f;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int v = (i * kThreads + tid) * 4;
    if (v >= len) break;
    float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    if (a.d_tokens) {
      const uint4 c4 = *reinterpret_cast<const uint4*>(seen + v);
      const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (v + k < len && c[k]) {
          if (a.d_repetition) y[k] = y[k] > 0.f ? __fdiv_rn(y[k], rep) : __fmul_rn(y[k], rep);
          const uint32_t n = c[k] & kCount;
          if (n) {
            if (a.d_frequency) y[k] = __fsub_rn(y[k], __fmul_rn(freq, (float)n));
            if (a.d_presence) y[k] = __fsub_rn(y[k], pres);
          }
        }
    }
    if (a.d_bias_start) {
      const uint4 c4 = *reinterpret_cast<const uint4*>(bias_at + v);
      const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (v + k < len && c[k]) y[k] = __fadd_rn(y[k], a.d_bias[first_bias + c[k] - 1]);
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

template <bool BF, int kStretch>
cudaError_t run(const Rules& r, cudaStream_t s) {
  static unsigned long long opted = 0;
  const size_t smem = sizeof(uint32_t) * kStretch * ((r.a.d_tokens ? 1 : 0) + (r.a.d_bias_start ? 1 : 0));
  if (!smem_opt_in(logit_rules_kernel<BF, kStretch>, 2 * sizeof(uint32_t) * kStretch, opted)) return cudaGetLastError();
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
    const cudaError_t e = launch_pdl(logit_rules_kernel<BF, kStretch>, grid, dim3(kThreads), smem, s, part);
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
  if (bf) return few ? run<true, 1024>(r, s) : run<true, 8192>(r, s);
  return few ? run<false, 1024>(r, s) : run<false, 8192>(r, s);
}

}  // namespace ane
