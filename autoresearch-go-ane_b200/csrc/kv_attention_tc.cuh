// Attention over a paged cache for many rows: 128 rows of a KV head's queries to a CTA, tiles of 64 keys, products on tcgen05.
//
//   warps 0-3    a thread has a row: it brings its queries to shared memory, turns the row's scores into probabilities, and its outputs, which
//                stay in tensor memory, into what is written
//   next 2 or 4  fetch 32 or 16 of a tile's keys and values each, by cp.async, with no wait for one another; 8-bit ones pass through a ring of
//                their own and become f16 on their way into the tile, once for all 128 rows
//   last         one thread issues the products: the next tile's scores before it waits for this tile's probabilities
//
// Probabilities take the place of their scores in tensor memory, in the operands' 16 bits: f16, which is finer than the output's type, for 8-bit
// pages; bf16 otherwise, and behind it what that leaves of them, a second product, without which the error is 1.4 times that of rounding
// the result.  Outputs are renewed only with a row's maximum, which follows its scores with some slack.
//
// The 8192 exponentials of a tile take 512 cycles of an SM at 16 a cycle; the products 256 with heads of 64, 384 over bf16 pages.  Heads of up to
// 64 have two CTAs an SM, so that one's waits and copies run under the other's softmax: 850 to 1000 cycles a tile and SM.  Eight sequences of
// 400 tokens over 1500, 12 heads of 64 with 4 for keys: 48 us from 8-bit pages and 45 from bf16, 41 without the second product (8.2 GFLOP; by
// mma.sync, every warp converting all keys, 74 and 59).  Its 4452 tiles, 30 an SM, are about 15 of the 48; cutting the work is 4, joining shared
// items 8, launches, starts and ends of items and what is uneven the rest.  Two of 100 over 60000, 16 heads of 128 with 2, 165 and 155 (334 by
// mma.sync).  Two threads a row, with half of the keys each, took 60 and 49 in place of 52 and 45: registers for 22 warps are too few; half of the
// scores loaded under the maximum of the others 50.4 and 42.6 in place of 49.2 and 41.6 (bf16 without the second product, both).
// Every wait is bounded and reports through the status word.
#pragma once

namespace ane {
namespace {

template <int HD_, bool F8_>
struct Prompt {
  static constexpr int HD = HD_;
  static constexpr bool F8 = F8_, kSplit = false, kRest = !F8_;  // probabilities have one
  // copying warps: two are all that the registers of two CTAs allow; 60000 tokens of heads of 128 took 213 us with two, 184 with four
  static constexpr int kLoaders = HD <= 64 ? 2 : 4, kEach = 4 / kLoaders, kWarps = 5 + kLoaders, kThreads = 32 * kWarps;
  static constexpr int kRows = 128, kTile = 64, kCtas = HD <= 64 ? 2 : 1;
  // tiles of 128 bytes a row, swizzled as the products want them: 64 columns each
  static constexpr int kAtoms = (HD + 63) / 64, kAtomQ = kRows * 128, kAtomX = kTile * 128;
  static constexpr int kQ = kAtoms * kAtomQ, kX = kAtoms * kAtomX, kStage = 2 * kX;
  static constexpr int kStages = F8 ? 3 : 4, kDeep = kStages, kLag = F8 && HD > 64 ? 3 : 2;  // tiles whose copies are under way while an earlier one's are waited for
  static constexpr int kRaw = F8 ? kTile * 2 * HD : 0, kRaws = kLag + 1;
  static constexpr int kMostSmem = 1024 + kQ + kStages * kStage + kRaws * kRaw;
  static constexpr int kInfo = 8;  // tiles whose scales and marks are kept
  static_assert(kLag + kStages < kInfo, "a tile's scales are written again when it is done with");
  // as in Form; us at half, as is, and at twice as many.  alone: 8 x 400 over 200 35.0 20.3 20.3, over 500 39.2 39.2 25.2, 100 over 600 (bf16)
  // 21.5 18.6 18.6; least: 8 x 100 over 1000 29.5 25.9 25.1, 50 over 3000 37.0 37.1 30.9
  static constexpr int kAlone = 768 / kTile, kLeast = 256 / kTile;
};

// f16 or bf16 operands, 128 rows, n columns; values lie with their columns together
__host__ __device__ constexpr uint32_t product_of(bool f16, bool values, int n) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | (values ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const float (&v)[16]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld_32x1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  return r;
}
// D[tmem] (+)= A[tmem, two 16-bit elements a column] * B[smem desc]; issued by a single thread.
__device__ __forceinline__ void tc_mma_from_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Two products, sums or both in one instruction.
__device__ __forceinline__ uint64_t both(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void each(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_both(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_both(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_both(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred P;\n\tmbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n\tselp.u32 %0, 1, 0, P;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// Where 16-byte piece c of a row lies in a tile of `atom` bytes per 64 columns.
__device__ __forceinline__ int swizzled(int row, int c, int atom) { return (c >> 3) * atom + row * 128 + (((c & 7) ^ (row & 7)) << 4); }

// Barriers and small things of a CTA.  Its tensor memory has two tiles' scores, 64 columns each, whose place their probabilities take (in
// 16 bits, 32 columns), and the outputs behind them.
template <class F>
struct PromptMemory {
  uint64_t full[F::kStages], empty[F::kStages], scores[2], outputs[2], probs[2], queries;
  float4 scales[F::kInfo][4];      // of a tile's groups of 16 keys: of keys, of values, log2 of the latter
  alignas(4) unsigned char odd[F::kInfo][4];  // not 0: a value is infinite or NaN and hidden from some row
  uint32_t tmem;
};
template <class F>
struct PromptPlaces {
  char *q, *tiles, *raw;
};

// A wait of a whole warp for two barriers, with one answer.
__device__ __forceinline__ bool warp_wait(uint64_t& one, uint32_t parity_one, uint64_t& two, uint32_t parity_two, int* status, int code) {
  const bool now_one = mbar_test(smem_u32(&one), parity_one), now_two = mbar_test(smem_u32(&two), parity_two);
  if (__all_sync(0xffffffffu, now_one && now_two)) return true;
  return __all_sync(0xffffffffu, mbar_wait(smem_u32(&one), parity_one, status, code) && mbar_wait(smem_u32(&two), parity_two, status, code));
}
// The same for one.
__device__ __forceinline__ bool warp_wait(uint64_t& bar, uint32_t parity, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar), parity, status, code));
}

// Keys and values of tile n of the CTA lie in stage n % kStages.
template <class F>
__device__ __forceinline__ void prompt_load(const Attn& a, const Plan& plan, Item it, PromptMemory<F>& m, const PromptPlaces<F>& at) {
  constexpr int HD = F::HD, ES = F::F8 ? 1 : 2;
  constexpr int kAhead = 32 / F::kEach;  // tiles
  const int lane = threadIdx.x & 31, group0 = ((threadIdx.x >> 5) - 4) * F::kEach;
  uint32_t issued = 0, finished = 0, edges = 0;  // edges: bit i, of the i-th last tile issued
  bool ok = true;
  // whether piece c, of a lane's i-th, of 16 keys and their values is one of values
  auto values = [](int i, int c) { return HD % 32 == 0 ? i >= HD / 32 : c >= HD; };
  auto stage_free = [&](uint32_t n) {
    return n < F::kStages || warp_wait(m.empty[n % F::kStages], ((n / F::kStages) & 1) ^ 1, a.status, DEV_MBAR_TIMEOUT_PRODUCER);
  };
  auto finish = [&]() {  // the copies of tile `finished` are there
    const uint32_t n = finished;
    char* k = at.tiles + n % F::kStages * F::kStage;
    const bool edge = edges >> (issued - n - 1) & 1;
    bool odd = false;
    if (F::F8) {
      if (!(ok = ok && stage_free(n))) return;
#pragma unroll
      for (int h = 0; h < F::kEach; ++h) {
        const uint4* raw = reinterpret_cast<const uint4*>(at.raw + n % F::kRaws * F::kRaw + (group0 + h) * (F::kRaw / 4));
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          const int c = i * 32 + lane, in = values(i, c) ? c - HD : c, row = (group0 + h) * kGroup + in / (HD / 16), piece = in % (HD / 16);
          const uint4 w = raw[c];
          uint4 lo, hi;
          e4m3_to_f16(w.x, lo.x, lo.y);
          e4m3_to_f16(w.y, lo.z, lo.w);
          e4m3_to_f16(w.z, hi.x, hi.y);
          e4m3_to_f16(w.w, hi.z, hi.w);
          char* to = values(i, c) ? k + F::kX : k;
          const int first = piece >> 2 & 1;  // of the two; what is written together lies in different banks then
          *reinterpret_cast<uint4*>(to + swizzled(row, 2 * piece + first, F::kAtomX)) = first ? hi : lo;
          *reinterpret_cast<uint4*>(to + swizzled(row, 2 * piece + 1 - first, F::kAtomX)) = first ? lo : hi;
          if (edge && values(i, c)) odd |= not_finite<true>(w.x) || not_finite<true>(w.y) || not_finite<true>(w.z) || not_finite<true>(w.w);
        }
      }
    } else if (edge) {
#pragma unroll
      for (int i = 0; i < F::kEach * HD / 16; ++i) {
        const int c = i * 32 + lane;
        const uint4 w = *reinterpret_cast<const uint4*>(k + F::kX + swizzled(group0 * kGroup + c / (HD / 8), c % (HD / 8), F::kAtomX));
        odd |= not_finite<false>(w.x) || not_finite<false>(w.y) || not_finite<false>(w.z) || not_finite<false>(w.w);
      }
    }
    odd = __any_sync(0xffffffffu, odd);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      m.odd[n % F::kInfo][group0 / F::kEach] = odd;
      mbar_arrive(smem_u32(&m.full[n % F::kStages]));
    }
    ++finished;
  };
  for (;;) {
    const int tile0 = it.range.template t0<F>() + it.off;
    const int p_first = it.s.pos + a.by_group(it.mt * F::kRows);
    const int p_last = it.s.pos + min(it.s.n - 1, a.by_group(it.mt * F::kRows + F::kRows - 1));
    // where the groups of the next tiles lie (in 16-byte pieces; all ones: nowhere) and their scales, a group a lane
    uint32_t my_at = 0xffffffffu;
    float my_k = 0.f, my_v = 0.f;
#pragma unroll 1
    for (int i = 0; i < it.count && ok; ++i) {
      if (i % kAhead == 0) {
        const int key = (tile0 + i + lane / F::kEach) * F::kTile + (group0 + lane % F::kEach) * kGroup;
        my_at = 0xffffffffu;
        my_k = my_v = 0.f;
        if (i + lane / F::kEach < it.count && key < it.range.hi && key + kGroup > it.range.lo) {
          const int slot = a.by_page(key), p = a.kv.table[(size_t)it.b * a.kv.table_pitch + slot];
          if (p < 0 || p >= a.kv.n_pages) {
            atomicCAS(a.status, DEV_OK, DEV_BAD_INDEX);
          } else {
            my_at = (uint32_t)(((unsigned long long)p * a.kv.page_stride +
                                ((size_t)it.head * a.kv.page_size + key - slot * a.kv.page_size) * HD) * ES >> 4);
            if (F::F8) {
              my_k = a.kv.k_scale[(size_t)p * a.kv.kv_heads + it.head];
              my_v = a.kv.v_scale[(size_t)p * a.kv.kv_heads + it.head];
            }
          }
        }
      }
      const uint32_t n = issued;
      if (!F::F8) {
        // earlier tiles first: the place for this one becomes free with products that may want them
        if (issued - finished == F::kLag) {
          copy_wait<F::kLag - 1>();
          finish();
        }
        if (!(ok = ok && stage_free(n))) break;
      }
      const char* none = reinterpret_cast<const char*>(a.kv.k);
#pragma unroll
      for (int h = 0; h < F::kEach; ++h) {
        const uint32_t from = __shfl_sync(0xffffffffu, my_at, i % kAhead * F::kEach + h);
        const int key0 = (tile0 + i) * F::kTile + (group0 + h) * kGroup;
        // rows that no query sees are filled with zeros: whatever lies there must not count
        const int lo = it.range.lo - key0, hi = from == 0xffffffffu ? 0 : it.range.hi - key0;
        const char *k = none + (size_t)from * 16, *v = reinterpret_cast<const char*>(a.kv.v) + (size_t)from * 16;
        if (F::F8) {
          const uint32_t to = smem_u32(at.raw) + n % F::kRaws * F::kRaw + (group0 + h) * (F::kRaw / 4);
#pragma unroll
          for (int x = 0; x < HD / 16; ++x) {
            const int c = x * 32 + lane, in = values(x, c) ? c - HD : c, row = in / (HD / 16);
            const bool take = row >= lo && row < hi;
            copy_16(to + c * 16, take ? (values(x, c) ? v : k) + in * 16 : none, take);
          }
        } else {
          const uint32_t to = smem_u32(at.tiles) + n % F::kStages * F::kStage;
#pragma unroll
          for (int x = 0; x < HD / 16; ++x) {
            const int c = x * 32 + lane, row = c / (HD / 8), place = swizzled((group0 + h) * kGroup + row, c % (HD / 8), F::kAtomX);
            const bool take = row >= lo && row < hi;
            copy_16(to + place, take ? k + c * 16 : none, take);
            copy_16(to + F::kX + place, take ? v + c * 16 : none, take);
          }
        }
      }
      copy_commit();
      if (F::F8 && lane / F::kEach == i % kAhead) m.scales[n % F::kInfo][group0 + lane % F::kEach] = make_float4(my_k, my_v, __log2f(my_v), 0.f);
      ++issued;
      const int first = (tile0 + i) * F::kTile;
      edges = edges << 1 | (first + F::kTile - 1 > p_first || (a.window && first <= p_last - a.window) ? 1u : 0u);
      if (F::F8 && issued - finished > F::kLag) {
        copy_wait<F::kLag>();
        finish();
      }
    }
    if (!ok || !next_item<F>(a, plan, it)) break;
  }
  copy_wait<0>();
  while (ok && finished < issued) finish();
}

// One thread.
template <class F>
__device__ __forceinline__ void prompt_issue(const Attn& a, const Plan& plan, Item it, PromptMemory<F>& m, const PromptPlaces<F>& at) {
  constexpr int HD = F::HD;
  constexpr uint32_t for_scores = product_of(F::F8, false, F::kTile), for_outputs = product_of(F::F8, true, F::kAtoms * 64);
  const uint32_t q = smem_u32(at.q), tiles = smem_u32(at.tiles), tmem = m.tmem;
  uint32_t n = 0;
  auto scores = [&](uint32_t n) {
    if (!mbar_wait(smem_u32(&m.full[n % F::kStages]), (n / F::kStages) & 1, a.status, DEV_MBAR_TIMEOUT_MMA)) return false;
    // the probabilities of the tile before last lie where these scores go
    if (n >= 2 && !mbar_wait(smem_u32(&m.outputs[n & 1]), ((n - 2) >> 1) & 1, a.status, DEV_MBAR_TIMEOUT_MMA)) return false;
    tc_fence_after();
    const uint32_t k = tiles + n % F::kStages * F::kStage;
#pragma unroll
    for (int x = 0; x < HD / 16; ++x)
      tc_mma_bf16(tmem + (n & 1) * F::kTile, make_smem_desc(q + x / 4 * F::kAtomQ + x % 4 * 32, 16, 1024),
                  make_smem_desc(k + x / 4 * F::kAtomX + x % 4 * 32, 16, 1024), for_scores, x > 0 ? 1u : 0u);
    tc_commit(smem_u32(&m.scores[n & 1]));
    return true;
  };
  for (uint32_t items = 0;; ++items) {
    if (!mbar_wait(smem_u32(&m.queries), items & 1, a.status, DEV_MBAR_TIMEOUT_MMA)) return;
    tc_fence_after();
    if (!scores(n)) return;
    for (int i = 0; i < it.count; ++i, ++n) {
      if (i + 1 < it.count && !scores(n + 1)) return;
      if (!mbar_wait(smem_u32(&m.probs[n & 1]), n >> 1 & 1, a.status, DEV_MBAR_TIMEOUT_MMA)) return;
      tc_fence_after();
      if (*reinterpret_cast<const volatile uint32_t*>(m.odd[n % F::kInfo]) == 0) {
        const uint32_t v = tiles + n % F::kStages * F::kStage + F::kX;
#pragma unroll
        for (int x = 0; x < F::kTile / 16; ++x) {
          const uint64_t values = make_smem_desc(v + x * 2048, F::kAtomX, 1024);
          const uint32_t p = tmem + (n & 1) * F::kTile + x * 8;
          tc_mma_from_tmem(tmem + 2 * F::kTile, p, values, for_outputs, i > 0 || x > 0 ? 1u : 0u);
          if (F::kRest) tc_mma_from_tmem(tmem + 2 * F::kTile, p + F::kTile / 2, values, for_outputs, 1u);
        }
      }
      tc_commit(smem_u32(&m.outputs[n & 1]));
      tc_commit(smem_u32(&m.empty[n % F::kStages]));
    }
    if (!next_item<F>(a, plan, it)) return;
  }
}

template <class F>
__device__ __forceinline__ void prompt_rows(const Attn& a, const Plan& plan, Item it, PromptMemory<F>& m, const PromptPlaces<F>& at) {
  constexpr int HD = F::HD, kTile = F::kTile;
  const int row = threadIdx.x, warp = row >> 5, lane = row & 31;
  const uint32_t tmem = m.tmem + ((uint32_t)(warp * 32) << 16), tmem_o = tmem + 2 * kTile;
  uint4 raw[HD / 8];
  auto fetch = [&](const Item& it) {
    const int n = it.mt * F::kRows + row;
    const bool there = n < it.s.n * a.group;
    const int t = there ? a.by_group(n) : 0, hd = there ? n - t * a.group : 0;
    const uint4* q = reinterpret_cast<const uint4*>(a.q + (size_t)(it.s.row + t) * a.ld_q + (size_t)(it.head * a.group + hd) * HD);
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) raw[i] = there ? q[i] : make_uint4(0, 0, 0, 0);
  };
  // The queries become an operand; what brings products to scores in log2 is returned.
  auto put = [&]() {
    float mult = a.scale_log2;
    if (F::F8) {
      float top = 0.f;
      auto most = [&](uint32_t w) { top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u)))); };
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) most(raw[i].x), most(raw[i].y), most(raw[i].z), most(raw[i].w);
      const float by = to_f16_range(top);
      mult /= by;
      auto f16 = [&](uint32_t w) { return pack<true>(__uint_as_float(w << 16) * by, __uint_as_float(w & 0xffff0000u) * by); };
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) raw[i] = make_uint4(f16(raw[i].x), f16(raw[i].y), f16(raw[i].z), f16(raw[i].w));
    }
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) *reinterpret_cast<uint4*>(at.q + swizzled(row, i, F::kAtomQ)) = raw[i];
    tc_fence_before();
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&m.queries));
    return mult;
  };
  fetch(it);
  float mult = put();
  uint32_t n = 0;
  for (;;) {
    const int rows0 = it.mt * F::kRows + warp * 32, n_rows = it.s.n * a.group, tile0 = it.range.template t0<F>() + it.off;
    const int pos = it.mt * F::kRows + row < n_rows ? it.s.pos + a.by_group(it.mt * F::kRows + row) : -1;
    const int p_first = it.s.pos + a.by_group(rows0), p_last = it.s.pos + min(it.s.n - 1, a.by_group(rows0 + 31));
    float base = 0.f, limit = -INFINITY, l = 0.f, w = kNoUnit, f = unit_factor(0.f, kNoUnit);
#pragma unroll 1
    for (int i = 0; i < it.count; ++i, ++n) {
      const int key0 = (tile0 + i) * kTile;
      // what the copying warps have written is read, too
      if (!warp_wait(m.full[n % F::kStages], (n / F::kStages) & 1, m.scores[n & 1], n >> 1 & 1, a.status, DEV_MBAR_TIMEOUT_EPILOGUE)) return;
      tc_fence_after();
      const bool odd = *reinterpret_cast<const volatile uint32_t*>(m.odd[n % F::kInfo]) != 0;
      float s[kTile];
      tmem_ld_32x32(tmem + (n & 1) * kTile, s);
      tmem_ld_32x32(tmem + (n & 1) * kTile + 32, s + 32);
      tmem_ld_wait();
      if (key0 + kTile - 1 > p_first || (a.window && key0 <= p_last - a.window)) {
#pragma unroll
        for (int e = 0; e < kTile; ++e)
          if (key0 + e > pos || (a.window && key0 + e <= pos - a.window)) s[e] = -INFINITY;
      }
      float mults[4], into[4], most = -INFINITY, top = -INFINITY;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float high = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) high = fmaxf(high, s[16 * g + e]);
        mults[g] = mult;
        into[g] = 1.f;
        if (F::F8) {
          const float4 scale = m.scales[n % F::kInfo][g];
          mults[g] = fmaxf(mult * scale.x, kLowest);  // not 0, so that hidden scores stay -infinity
          into[g] = scale.y;
          most = fmaxf(most, fmaf(high, mults[g], scale.z));
        }
        top = fmaxf(top, high * mults[g]);
      }
      if (__any_sync(0xffffffffu, top > limit || (F::F8 && most > w + kSlack))) {
        const bool none = limit == -INFINITY;
        const float up = top > limit ? (none ? (top == -INFINITY ? 0.f : top) : fmaxf(top, base)) : base;
        float fix = none ? 1.f : exp2_fast(base - up);  // the sum is still 0 then
        base = up;
        limit = none && top == -INFINITY ? -INFINITY : base + kSlack;
        l *= fix;
        if (F::F8) {  // outputs have a unit of their own
          const float now = most > w + kSlack ? most : w;
          fix = exp2_fast(w - now);
          w = now;
          f = unit_factor(base, w);
        }
        if (i > 0) {
          if (!warp_wait(m.outputs[(n - 1) & 1], (n - 1) >> 1 & 1, a.status, DEV_MBAR_TIMEOUT_EPILOGUE)) return;
          tc_fence_after();
#pragma unroll 1
          for (int x = 0; x < HD; x += 16) {
            float o[16];
            tmem_ld_32x16(tmem_o + x, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= fix;
            tmem_st_32x16(tmem_o + x, o);
          }
          tmem_st_wait();
        }
      }
      uint64_t sums[2] = {0, 0};
      uint32_t p[kTile / 2], rest[F::kRest ? kTile / 2 : 1];
      const uint64_t less = both(-base, -base), minus = both(-1.f, -1.f);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint64_t by = both(mults[g], mults[g]);
        if (F::F8) into[g] = into_units(into[g], f);
#pragma unroll
        for (int e = 8 * g; e < 8 * g + 8; ++e) {
          float lo, hi;
          each(fma_both(both(s[2 * e], s[2 * e + 1]), by, less), lo, hi);
          uint64_t two = both(exp2_fast(lo), exp2_fast(hi));
          sums[e & 1] = add_both(sums[e & 1], two);
          if (F::F8) two = mul_both(two, both(into[g], into[g]));
          each(two, lo, hi);
          p[e] = pack<F::F8>(lo, hi);
          if constexpr (F::kRest) {
            float lo_left, hi_left;
            each(fma_both(both(__uint_as_float(p[e] << 16), __uint_as_float(p[e] & 0xffff0000u)), minus, two), lo_left, hi_left);
            rest[e] = pack<false>(lo_left, hi_left);
          }
        }
      }
      {
        float lo, hi;
        each(add_both(sums[0], sums[1]), lo, hi);
        l += lo + hi;
      }
      // The place is free: the products with the tile before last were complete before this one's scores.
      tmem_st_32x32(tmem + (n & 1) * kTile, p);
      if constexpr (F::kRest) tmem_st_32x32(tmem + (n & 1) * kTile + kTile / 2, rest);
      tmem_st_wait();
      if (odd) {
        // A value that is infinite or NaN must not reach rows that do not see its key, and 0 * NaN is NaN: one product after the other, unseen
        // ones left out, instead of the tile's.
        const char* v = at.tiles + n % F::kStages * F::kStage + F::kX;
        if (i > 0) {
          if (!warp_wait(m.outputs[(n - 1) & 1], (n - 1) >> 1 & 1, a.status, DEV_MBAR_TIMEOUT_EPILOGUE)) return;
          tc_fence_after();
        }
#pragma unroll 1
        for (int x = 0; x < HD; x += 16) {
          float o[16];
          if (i > 0) {
            tmem_ld_32x16(tmem_o + x, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0.f;
          }
#pragma unroll 1
          for (int key = 0; key < kTile; ++key) {
            const uint32_t two = tmem_ld_32x1(tmem + (n & 1) * kTile + key / 2);
            const uint32_t left = F::kRest ? tmem_ld_32x1(tmem + (n & 1) * kTile + kTile / 2 + key / 2) : 0u;
            tmem_ld_wait();
            float w = from_16<F::F8>((uint16_t)(key & 1 ? two >> 16 : two));
            if (F::kRest) w += from_16<false>((uint16_t)(key & 1 ? left >> 16 : left));
            const bool seen = key0 + key <= pos && !(a.window && key0 + key <= pos - a.window);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (seen) o[e] = fmaf(w, from_16<F::F8>(*reinterpret_cast<const uint16_t*>(v + swizzled(key, (x + e) / 8, F::kAtomX) + e % 8 * 2)), o[e]);
          }
          __syncwarp();
          tmem_st_32x16(tmem_o + x, o);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&m.probs[n & 1]));
    }

    // the item's end: all its scores have been formed, so the next one's queries may take the place of its
    const Item done = it;
    const bool another = next_item<F>(a, plan, it);
    if (another) fetch(it);
    if (!warp_wait(m.outputs[(n - 1) & 1], (n - 1) >> 1 & 1, a.status, DEV_MBAR_TIMEOUT_EPILOGUE)) return;
    tc_fence_after();
    if (another) mult = put();
    const bool begins = done.off == 0, ends = done.off + done.count == done.tiles, complete = begins && ends;
    const int slot = 2 * blockIdx.x + (begins ? 1 : 0), of = done.mt * F::kRows + row;
    const bool there = of < n_rows;
    const int t = a.by_group(of), hd = of - t * a.group;
    const float unit = F::F8 ? 1.f / f : 1.f, by = !complete ? unit : l == 0.f ? 0.f : unit / l;
    bf16* out = a.out + (size_t)(done.s.row + t) * a.ld_out + (size_t)(done.head * a.group + hd) * HD;
    if (!complete && there) a.stats[(size_t)slot * F::kRows + row] = make_float2(limit == -INFINITY ? -INFINITY : base, l);
#pragma unroll 1
    for (int x = 0; x < HD; x += 16) {
      float o[16];
      tmem_ld_32x16(tmem_o + x, o);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] *= by, o[e] *= unit;
      if (!there) {
      } else if (complete) {
#pragma unroll
        for (int e = 0; e < 16; e += 8)
          *reinterpret_cast<uint4*>(out + x + e) =
              make_uint4(pack<false>(o[e], o[e + 1]), pack<false>(o[e + 2], o[e + 3]), pack<false>(o[e + 4], o[e + 5]), pack<false>(o[e + 6], o[e + 7]));
      } else {
#pragma unroll
        for (int e = 0; e < 16; e += 4) *part_at<F>(a, slot, row, (x + e) / 4) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      }
      __syncwarp();
    }
    if (!complete && begins && row == 0) mark_shared(a, plan, done);
    if (!another) return;
  }
}

template <class F>
__global__ void __launch_bounds__(F::kThreads, F::kCtas) kv_prompt_kernel(const Attn a) {
  extern __shared__ __align__(128) char ring[];
  __shared__ __align__(16) PromptMemory<F> m;
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5;
  Item it;
  const Plan plan = make_plan<F>(a, it);
  if (tid == 0) a.head[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (it.b < 0) {
    pdl_trigger();
    return;
  }
  if (tid < F::kInfo) *reinterpret_cast<uint32_t*>(m.odd[tid]) = 0;
  if (tid == 0) {
    for (int i = 0; i < F::kStages; ++i) {
      mbar_init(smem_u32(&m.full[i]), F::kLoaders);
      mbar_init(smem_u32(&m.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&m.scores[i]), 1);
      mbar_init(smem_u32(&m.outputs[i]), 1);
      mbar_init(smem_u32(&m.probs[i]), 4);
    }
    mbar_init(smem_u32(&m.queries), 4);
    fence_mbar_init();
  }
  if (warp == F::kWarps - 1) {
    tmem_alloc(smem_u32(&m.tmem), 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  PromptPlaces<F> at;
  at.q = ring + ((1024 - (smem_u32(ring) & 1023)) & 1023);
  at.tiles = at.q + F::kQ;
  at.raw = at.tiles + F::kStages * F::kStage;
  if (warp < 4) prompt_rows<F>(a, plan, it, m, at);
  else if (warp < F::kWarps - 1) prompt_load<F>(a, plan, it, m, at);
  else if (elect_one()) prompt_issue<F>(a, plan, it, m, at);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == F::kWarps - 1) {
    tc_fence_after();
    tmem_dealloc(m.tmem, 256);
  }
  pdl_trigger();  // not earlier: the next kernel's CTAs would take the room of this one's second half
}

}  // namespace
}  // namespace ane
