// Launchers of the serving kernels (kv_append.cu, kv_attention.cu, logit_rules.cu).  Arguments have been checked by their C entry
// points (ops_api.cu) or by the engine; each launcher returns the status of its launches.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/ane_b200.h"
#include "common.cuh"

namespace ane {

// A paged cache as the kernels see it; strides in elements.
struct PagedKv {
  void *k, *v;
  float *k_scale, *v_scale;
  long long page_stride;
  int n_pages, page_size, kv_heads, head_dim;
  const int* table;
  int table_pitch;
  bool e4m3;
};
PagedKv paged_kv(const ane_kv_cache& c);

// The sequences of a batch: new rows [start[b], start[b + 1]) at positions pos[b]...
struct Batch {
  const int *start, *pos;
  int n_seq, n_tokens;
};

bool kv_head_dim_supported(int head_dim);
cudaError_t kv_append(const PagedKv& kv, const Batch& batch, int heads, const bf16* qkv, int ld_qkv, bf16* q, int ld_q,
                      const float* cosb, const float* sinb, int n_positions, int* status, cudaStream_t s);
cudaError_t kv_attention(const PagedKv& kv, const Batch& batch, int heads, const bf16* q, int ld_q, bf16* out, int ld_out,
                         int max_new, int window, float scale, void* workspace, int* status, cudaStream_t s);
size_t kv_attention_workspace(int sms, int head_dim);
cudaError_t logit_rules(const ane_logit_rules_args& a, int* status, cudaStream_t s);

#ifdef __CUDACC__
// Quotients by a number known at launch, in five instructions: floor(2^32 / d) gives them or one less.
struct Div {
  uint32_t d, m;
  Div() = default;
  explicit Div(int by) : d(by), m(by == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / by)) {}
  __device__ __forceinline__ int operator()(int n) const {
    const uint32_t q = __umulhi((uint32_t)n, m);
    return (int)(q + ((uint32_t)n - q * d >= d ? 1u : 0u));
  }
};

// New rows and place of sequence b; none (and the status word) where its entries make no sense, n < 0 where its rows would begin behind their end.
struct Span {
  int row, n, pos;
};
__device__ __forceinline__ Span span_of(int row, int end, int pos, const Batch& a, int capacity, int most, int* status) {
  if (row == end) return {row, 0, pos};
  if (row < 0 || end < row || end > a.n_tokens || end - row > most || pos < 0 || end - row > capacity - pos) {
    atomicCAS(status, DEV_OK, DEV_BAD_INDEX);
    return {row, end < row ? -1 : 0, pos};
  }
  return {row, end - row, pos};
}
__device__ __forceinline__ Span span_of(const Batch& a, int b, int capacity, int most, int* status) {
  return span_of(a.start[b], a.start[b + 1], a.pos[b], a, capacity, most, status);
}
#endif

}  // namespace ane
