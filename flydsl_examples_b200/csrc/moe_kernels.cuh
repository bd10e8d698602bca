// A mixture-of-experts layer for a few tokens (up to 64) in two kernels, for sm_100a.
//
//   p = softmax(logits); the top_k experts of each token, ties to the lowest index (optionally renormalised)
//   y[t] = sum over its experts e of p[t, e] * W2[e] * (silu(G) * U),   [G; U] = W13[e] * x[t]
//
// Bound by reading the weights of the experts that any token chose, once: 6 * H * I bytes each. Everything else is arranged
// around that stream.
//  * Weights sit on the 128-row side of tcgen05.mma, tokens on its N axis (16, 32 or 64 columns). All tokens take part in
//    every expert's product and the epilogue keeps the pairs that the router chose: no gather, and the tensor core has
//    the time (64 columns need a quarter of what the weights' bytes take).
//  * First kernel: every block routes for itself (a warp per token, top_k rounds of a warp-wide maximum; the logits are a
//    few kilobytes), so no launch and no pass of its own. A tile is 64 gate rows over 64 up rows of one expert; its
//    epilogue writes h[slot][t][i] = round16(p * silu(gate) * up), zero for pairs that were not chosen. The weight of the
//    pair is folded in before the one rounding that the second product's 16-bit operand needs.
//  * Second kernel: the sum over experts is the K axis of one product, y[h, t] = sum over (slot, i) of W2 * h, accumulated
//    in TMEM. K is cut into contiguous spans over the CTAs of a cluster, which add up through distributed shared
//    memory in rank order: no atomics, the same bits every time.
// Both keep about 190 KB of TMA loads in flight per SM.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace b200 {

constexpr int kMoeThreads = 192;  // warp 0 TMA producer, warp 1 TMEM and MMA, warps 2-5 epilogue
constexpr int kMoeMaxTokens = 64, kMoeMaxExperts = 512, kMoeMaxTopK = 16;
constexpr int kMoeTK = 128;       // K elements per stage: two 64-element swizzle spans
constexpr int kMoeUBytes = 128 * kMoeTK * 2;

struct alignas(64) MoeParams {
  CUtensorMap tmap_u;  // W13 as {H, 2I, E}, box {64, 64, 1}; or W2 as {I, H, E}, box {64, 128, 1}
  CUtensorMap tmap_v;  // x as {H, T}, box {64, TN}; or h as {I, T, slots}, box {64, TN, 1}
  const void* logits;
  long long logits_row, logits_col;
  int logits_dtype;  // 1 fp32, 2 bf16, 3 fp16
  int T, E, H, I, top_k, renorm;
  int dtype;         // 2 bf16, 3 fp16
  uint16_t* h;       // [slot][T][I]
  int* active;       // [0] = number of experts chosen by any token, then their indices in increasing order
  void* out;
  long long ldo;
  int cluster_split;
  uint32_t idesc, desc_hi;
  int* status;
  unsigned long long wait_limit_ns;
};

template <int TN, int STAGES, bool UP>
struct SmemMoe {
  static constexpr int kVBox = TN * 128;
  static constexpr int kStageBytes = kMoeUBytes + 2 * kVBox;
  static constexpr int kXOff = STAGES * kStageBytes;                 // UP: the up half's sums [TN][64]; otherwise recv[src][col][128]
  static constexpr int kXBytes = UP ? TN * 64 * 4 : TN * 128 * 4;
  static constexpr int kRouteOff = kXOff + kXBytes;                  // ids, weights [64][16]; active list; weights of one expert
  static constexpr int kRouteBytes = UP ? kMoeMaxTokens * kMoeMaxTopK * 8 + (kMoeMaxExperts + 16 + kMoeMaxExperts / 32 + kMoeMaxTokens) * 4 : 0;
  static constexpr int kBarOff = (kRouteOff + kRouteBytes + 7) / 8 * 8;
  static constexpr int kMiscOff = kBarOff + (2 * STAGES + 4) * 8;
  static constexpr int kTotal = kMiscOff + 16;
  static constexpr int kDynBytes = kTotal + 1024;
};

__device__ __forceinline__ void report_abort_moe(int* status, int role, int unit) {
  if (status != nullptr && atomicCAS(status, 0, 1) == 0) {
    status[1] = blockIdx.x;
    status[2] = role;
    status[3] = unit;
  }
}

// Order-preserving integer of a logit; NaN above everything, the two zeros alike.
__device__ __forceinline__ uint32_t logit_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float load_logit(const MoeParams& p, int t, int e) {
  const long long i = (long long)t * p.logits_row + (long long)e * p.logits_col;
  if (p.logits_dtype == 1) return reinterpret_cast<const float*>(p.logits)[i];
  if (p.logits_dtype == 2) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.logits)[i]);
  return __half2float(reinterpret_cast<const __half*>(p.logits)[i]);
}

// One warp routes token t: ids[0..top_k), weights[0..top_k) (a weight of zero: not chosen), and the experts' bits in `mask`.
__device__ __forceinline__ void route_token(const MoeParams& p, int t, int lane, int* ids, float* weights, uint32_t* mask) {
  constexpr int kPer = kMoeMaxExperts / 32;
  uint32_t key[kPer];  // 0: no expert, or taken already (no logit maps to 0)
  float top = -INFINITY, total = 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    key[j] = 0;
    if (j * 32 < p.E) {
      const int e = j * 32 + lane;
      if (e < p.E) key[j] = logit_key(load_logit(p, t, e));
    }
  }
  auto value = [](uint32_t k) {  // the logit of a key
    return k == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  };
  float mine = 0.f;  // lane r holds the r-th chosen logit and index
  int my_id = 0;
  for (int r = 0; r < p.top_k; ++r) {
    uint32_t best = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j * 32 < p.E) best = max(best, key[j]);
    best = __reduce_max_sync(0xffffffffu, best);
    int at = 0x7fffffff;
#pragma unroll
    for (int j = kPer - 1; j >= 0; --j)
      if (j * 32 < p.E && key[j] == best) at = j * 32 + lane;
    at = (int)__reduce_min_sync(0xffffffffu, (unsigned)at);
    if (r == 0) {
      top = value(best);
      if (!p.renorm) {  // the softmax's sum over all experts
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (j * 32 + lane < p.E) total += expf(value(key[j]) - top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      }
    }
    if (lane == r) mine = value(best), my_id = at;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j * 32 + lane == at) key[j] = 0;
  }
  float w = lane < p.top_k ? expf(mine - top) : 0.f;
  if (p.renorm) {
    total = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  w = top == -INFINITY ? 0.f : w / total;  // a token whose logits are all -inf goes nowhere
  if (lane < p.top_k) {
    ids[lane] = w == 0.f ? -1 : my_id;
    weights[lane] = w;
    if (w != 0.f) atomicOr(mask + (my_id >> 5), 1u << (my_id & 31));
  }
}

// UP: the first kernel (gate and up products, SiLU), otherwise the second (down product and sum).
template <int TN, int STAGES, bool UP>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_a16w16_sm100_kernel(const __grid_constant__ MoeParams p) {
  using L = SmemMoe<TN, STAGES, UP>;
  constexpr uint32_t kTmemCols = 2 * TN < 32 ? 32 : 2 * TN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const uint32_t bar0 = base + L::kBarOff;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto accf_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto acce_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + 2 + b); };
  volatile uint32_t* tmem_ptr_s = reinterpret_cast<volatile uint32_t*>(sm + L::kMiscOff);
  volatile int* abort_s = reinterpret_cast<volatile int*>(sm + L::kMiscOff + 4);
  volatile int* epi_abort_s = reinterpret_cast<volatile int*>(sm + L::kMiscOff + 8);
  int* ids = reinterpret_cast<int*>(sm + L::kRouteOff);
  float* weights = reinterpret_cast<float*>(ids + kMoeMaxTokens * kMoeMaxTopK);
  int* list = reinterpret_cast<int*>(weights + kMoeMaxTokens * kMoeMaxTopK);  // [0] = count, [16..] = experts
  uint32_t* mask = reinterpret_cast<uint32_t*>(list + 16 + kMoeMaxExperts);
  float* pair_w = reinterpret_cast<float*>(mask + kMoeMaxExperts / 32);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool cluster_mode = !UP && p.cluster_split > 1;
  const int rank = cluster_mode ? (int)cluster_ctarank() : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf_bar(b), 1);
      mbar_init(acce_bar(b), 4);
    }
    *abort_s = 0;
    *epi_abort_s = 0;
    fence_mbar_init();
    prefetch_tmap(&p.tmap_u);
    prefetch_tmap(&p.tmap_v);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_ptr_s)), kTmemCols);
    tmem_relinquish<1>();
  }
  if (UP && threadIdx.x < kMoeMaxExperts / 32) mask[threadIdx.x] = 0;
  tc_fence_before();
  __syncthreads();
  bool cluster_wait_due = false;
  if (cluster_mode) {
    cluster_arrive();
    cluster_wait_due = true;
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr_s;
  grid_dependency_wait();
  grid_launch_dependents();

  int n_active;
  const int* experts;
  if constexpr (UP) {
    for (int t = warp; t < p.T; t += kMoeThreads / 32) route_token(p, t, lane, ids + t * kMoeMaxTopK, weights + t * kMoeMaxTopK, mask);
    __syncthreads();
    if (warp == 0) {  // the chosen experts in increasing order
      uint32_t m = lane < kMoeMaxExperts / 32 ? mask[lane] : 0;
      int before = __popc(m);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      if (lane == 31) list[0] = before;
      int at = before - __popc(m);
      while (m) {
        list[16 + at++] = lane * 32 + __ffs(m) - 1;
        m &= m - 1;
      }
    }
    __syncthreads();
    n_active = list[0];
    experts = list + 16;
    if (blockIdx.x == 0) {  // for the second kernel
      for (int i = threadIdx.x; i < n_active; i += kMoeThreads) p.active[16 + i] = experts[i];
      if (threadIdx.x == 0) p.active[0] = n_active;
    }
  } else {
    n_active = *reinterpret_cast<volatile int*>(p.active);
    experts = p.active + 16;
  }

  // UP: unit = (slot, 64 gate rows), K = H. Otherwise one unit per CTA: 128 rows of H, a span of the K axis (slot, I).
  const int k_blocks = UP ? (p.H + kMoeTK - 1) / kMoeTK : (p.I + kMoeTK - 1) / kMoeTK;
  const int tiles = UP ? (p.I + 63) / 64 : 1;
  const int S = cluster_mode ? p.cluster_split : 1;
  const long long span = (long long)n_active * k_blocks;
  const int row_tile = UP ? 0 : (int)blockIdx.x / S;
  const int u_first = UP ? (int)blockIdx.x : 0, u_step = UP ? (int)gridDim.x : 1;
  const int u_end = UP ? n_active * tiles : 1;
  const int b_first = UP ? 0 : (int)(span * rank / S), b_end = UP ? k_blocks : (int)(span * (rank + 1) / S);

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
#pragma unroll 1
    for (int u = u_first; ok && u < u_end; u += u_step) {
      const int slot0 = UP ? u / tiles : 0, i0 = UP ? (u - slot0 * tiles) * 64 : 0;
      int expert = UP ? experts[slot0] : 0, slot = UP ? slot0 : -1;
#pragma unroll 1
      for (int b = b_first; b < b_end; ++b) {
        int kb = b;
        if constexpr (!UP) {
          const int s = b / k_blocks;
          kb = b - s * k_blocks;
          if (s != slot) slot = s, expert = experts[s];
        }
        if (issued >= STAGES) {
          int good = 1;
          if (lane == 0) good = mbar_wait(empty_bar(stage), phase ^ 1u, abort_s, p.wait_limit_ns) ? 1 : 0;
          good = __shfl_sync(0xffffffffu, good, 0);
          if (!good) {
            if (lane == 0) report_abort_moe(p.status, 0, u);
            ok = false;
            break;
          }
        }
        if (elect_one()) {
          const uint32_t fb = full_bar(stage);
          const uint32_t su = base + stage * L::kStageBytes, sv = su + kMoeUBytes;
          mbar_arrive_expect_tx(fb, L::kStageBytes);
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            const int k0 = kb * kMoeTK + sub * 64;
            if constexpr (UP) {
              tma_load_3d(su + sub * 16384, &p.tmap_u, k0, i0, expert, fb);
              tma_load_3d(su + sub * 16384 + 8192, &p.tmap_u, k0, p.I + i0, expert, fb);
              tma_load_2d(sv + sub * L::kVBox, &p.tmap_v, k0, 0, fb);
            } else {
              tma_load_3d(su + sub * 16384, &p.tmap_u, k0, row_tile * 128, expert, fb);
              tma_load_3d(sv + sub * L::kVBox, &p.tmap_v, k0, 0, slot, fb);
            }
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == STAGES) stage = 0, phase ^= 1u;
      }
    }
    if (!ok && lane == 0) {  // loads in flight still write shared memory: a bounded time to land
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    int stage = 0, it = 0;
    uint32_t phase = 0;
    bool ok = true;
#pragma unroll 1
    for (int u = u_first; ok && u < u_end && b_first < b_end; u += u_step, ++it) {
      const int buf = it & 1;
      int good = 1;
      if (lane == 0) good = mbar_wait(acce_bar(buf), ((it >> 1) & 1) ^ 1u, abort_s, p.wait_limit_ns) ? 1 : 0;
      good = __shfl_sync(0xffffffffu, good, 0);
      if (!good) {
        if (lane == 0) report_abort_moe(p.status, 1, u);
        break;
      }
      tc_fence_after();
#pragma unroll 1
      for (int b = b_first; b < b_end; ++b) {
        if (lane == 0) good = mbar_wait(full_bar(stage), phase, abort_s, p.wait_limit_ns) ? 1 : 0;
        good = __shfl_sync(0xffffffffu, good, 0);
        if (!good) {
          if (lane == 0) report_abort_moe(p.status, 2, u);
          ok = false;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t su = base + stage * L::kStageBytes, sv = su + kMoeUBytes;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            // K-major rows of 128 swizzled bytes, groups of eight 1024 bytes apart
            const uint64_t du = (uint64_t(p.desc_hi) << 32) | uint64_t((1u << 16) | (((su + sub * 16384) >> 4) & 0x3fffu));
            const uint64_t dv = (uint64_t(p.desc_hi) << 32) | uint64_t((1u << 16) | (((sv + sub * L::kVBox) >> 4) & 0x3fffu));
#pragma unroll
            for (int j = 0; j < 4; ++j)
              umma_f16<1>(tmem_base + buf * TN, du + uint64_t(2 * j), dv + uint64_t(2 * j), p.idesc, (b != b_first || sub || j) ? 1u : 0u);
          }
          umma_commit(empty_bar(stage));
          if (b + 1 == b_end) umma_commit(accf_bar(buf));
        }
        __syncwarp();
        if (++stage == STAGES) stage = 0, phase ^= 1u;
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue (warps 2..5)
    const int quarter = warp & 3, row = quarter * 32 + lane, et = threadIdx.x - 64;
    float* xs = reinterpret_cast<float*>(sm + L::kXOff);
    int it = 0;
#pragma unroll 1
    for (int u = u_first; u < u_end; u += u_step, ++it) {
      const int buf = it & 1;
      const int slot = UP ? u / tiles : 0;
      if constexpr (UP) {  // the weights of this expert's pairs; ordered by the barriers below
        if (et < TN) {
          float w = 0.f;
          if (et < p.T)
            for (int j = 0; j < p.top_k; ++j)
              if (ids[et * kMoeMaxTopK + j] == experts[slot]) w = weights[et * kMoeMaxTopK + j];
          pair_w[et] = w;
        }
      }
      float v[TN];
      if (b_first < b_end) {
        // The 128 threads meet at barriers: one whose limit ran out leaves a note that later finishers read.
        if (!mbar_wait<false, false>(accf_bar(buf), (it >> 1) & 1, abort_s, p.wait_limit_ns)) *epi_abort_s = 1;
        named_bar_sync(1, 128);
        if (*epi_abort_s != 0) {
          if (et == 0) report_abort_moe(p.status, 3, u);
          break;
        }
        tc_fence_after();
        const uint32_t t_acc = tmem_base + buf * TN + (uint32_t(quarter * 32) << 16);
        uint32_t r[32];
#pragma unroll
        for (int c = 0; c < TN; c += 32) {
          if constexpr (TN >= 32)
            tmem_ld_32x32(t_acc + c, r);
          else
            tmem_ld_32x16(t_acc + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < (TN < 32 ? TN : 32); ++i) v[c + i] = __uint_as_float(r[i]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acce_bar(buf));
      } else {
#pragma unroll
        for (int i = 0; i < TN; ++i) v[i] = 0.f;
      }
      if constexpr (UP) {
        // lanes 64..127 hold the up rows of the gate rows in lanes 0..63
        if (row >= 64) {
#pragma unroll
          for (int t = 0; t < TN; ++t) xs[t * 64 + row - 64] = v[t];
        }
        named_bar_sync(2, 128);
        const int i = (u - slot * tiles) * 64 + row;
        if (row < 64 && i < p.I) {
          uint16_t* dst = p.h + ((size_t)slot * p.T) * p.I + i;
#pragma unroll
          for (int t = 0; t < TN; ++t) {
            if (t < p.T) {
              const float w = pair_w[t], g = v[t];
              // a pair that was not chosen is zero whatever its sums are
              const float a = w == 0.f ? 0.f : w * (g / (1.f + __expf(-g))) * xs[t * 64 + row];
              uint16_t bits;
              if (p.dtype == 2) {
                const __nv_bfloat16 h = __float2bfloat16_rn(a);
                bits = *reinterpret_cast<const uint16_t*>(&h);
              } else {
                const __half h = __float2half_rn(a);
                bits = *reinterpret_cast<const uint16_t*>(&h);
              }
              dst[(size_t)t * p.I] = bits;
            }
          }
        }
        named_bar_sync(1, 128);  // xs and pair_w may be rewritten
      } else if (cluster_mode) {
        // Column t belongs to CTA t / (TN / S): a warp's 32 rows are 128 contiguous bytes of recv[source][own column][row].
        if (cluster_wait_due) {
          cluster_wait();
          cluster_wait_due = false;
        }
        const int own_log2 = __ffs(TN / S) - 1;
        const uint32_t recv = base + L::kXOff + (uint32_t)row * 4u;
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          const uint32_t dst = mapa_cluster(recv + (uint32_t)(((rank << own_log2) + (t & ((1 << own_log2) - 1))) * 128) * 4u, (uint32_t)(t >> own_log2));
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(v[t]) : "memory");
        }
      } else {
        const int hrow = row_tile * 128 + row;
        if (hrow < p.H) {
#pragma unroll
          for (int t = 0; t < TN; ++t)
            if (t < p.T) {
              if (p.dtype == 2)
                reinterpret_cast<__nv_bfloat16*>(p.out)[(long long)t * p.ldo + hrow] = __float2bfloat16_rn(v[t]);
              else
                reinterpret_cast<__half*>(p.out)[(long long)t * p.ldo + hrow] = __float2half_rn(v[t]);
            }
        }
      }
    }
  }

  // ---------------------------------------------------------------------- teardown
  if (cluster_wait_due) cluster_wait();
  tc_fence_before();
  __syncthreads();
  if (cluster_mode) {
    cluster_arrive();
    cluster_wait();
    if (warp >= 2) {
      const int own = TN / S, row = threadIdx.x - 64, hrow = row_tile * 128 + row;
      const float* recv = reinterpret_cast<const float*>(sm + L::kXOff) + row;
      if (hrow < p.H) {
        for (int c = 0; c < own; ++c) {
          const int t = rank * own + c;
          if (t >= p.T) break;
          float x = 0.f;
          for (int src = 0; src < S; ++src) x += recv[(src * own + c) * 128];
          if (p.dtype == 2)
            reinterpret_cast<__nv_bfloat16*>(p.out)[(long long)t * p.ldo + hrow] = __float2bfloat16_rn(x);
          else
            reinterpret_cast<__half*>(p.out)[(long long)t * p.ldo + hrow] = __float2half_rn(x);
        }
      }
    }
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, kTmemCols);
  }
}

typedef void (*MoeFn)(const MoeParams);

}  // namespace b200
