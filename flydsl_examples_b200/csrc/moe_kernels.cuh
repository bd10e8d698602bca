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
//  * Every block of the first kernel routes for itself (the logits are a few kilobytes), so routing has no launch and no pass
//    of its own; the list of chosen experts goes to the second kernel. (The second kernel routing again, in order to fill
//    its ring with weights while the first one's last tiles run, took 26.2 instead of 24.4 us for one token of 8 / 128
//    experts, 169 instead of 171 us for 8 tokens of 2 / 16: its blocks mostly start when the first kernel's end. The first
//    kernel asking for the down weights into L2 behind its own last loads: 28.0 instead of 24.4 us for one token.)
//  * First kernel: a tile is 64 gate rows over 64 up rows of one expert; its epilogue computes h[slot][t][i] = p * silu(gate) *
//    up, zero for pairs that were not chosen, with the weight of the pair folded in. h is the second product's 16-bit
//    operand; it is stored as two of them, the rounded value and the rounded remainder, which cost that product columns
//    (2 TN instead of TN) that it has to spare. Rounded once, h would put as much error into y as y's own rounding does. The two
//    have accumulators of their own, so each may have a power of two of its own, undone when they are added. In fp16 the value
//    is that of h / 16 and the remainder is kept 2^11 times as large: together they are exact to 2^-22 of h, or 2^-32 for
//    |h| below 2^-10, up to 2^20 (with no such factors: infinite from 65520 on, and half steps of 2^-25). bf16 has fp32's range: 2^-16 of h.
//  * Second kernel: the sum over experts is the K axis of one product, y[h, t] = sum over (slot, i) of W2 * h, accumulated
//    in TMEM. K is cut into contiguous spans over the CTAs of a cluster, which add up through distributed shared
//    memory in rank order: no atomics, the same bits every time.
// Both keep about 190 KB of TMA loads in flight per SM. 32 tokens, 8 of 32 experts, H 7168, I 2048 (2.8 GB): 431 - 452 us, 95 to
// 100 % of the copy rate; 8 tokens, 2 of 16, 4096, 3584: 143 - 169 us by the experts chosen, 93 to 98 %; 64 tokens, 8 of 32, 4096, 2048 (1.6
// GB): 287 - 290 us, 85 % (each weight tile comes with h for all tokens, as many bytes again); one token, 8 of 128, 2048, 768 (75 MB): 24.6
// us, 47 %, bound by the latencies of two dependent kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace b200 {

constexpr int kMoeThreads = 384;  // warp 0 TMA producer, warp 1 TMEM and MMA, warps 2-5 epilogue; 6-11 only help to route
constexpr int kMoeMaxTokens = 64, kMoeMaxExperts = 512, kMoeMaxTopK = 16;

// Powers of two with which h is kept in fp16, see above.
constexpr float kMoeValueScale = 1.f / 16, kMoeRestScale = 2048.f;

struct alignas(64) MoeParams {
  CUtensorMap tmap_u;  // W13 as {H, 2I, E}, box {64, 64, 1}; or W2 as {I, H, E}, box {64, 128, 1}
  CUtensorMap tmap_v;  // x as {H, T}, box {64, TN}; or h as {I, T, 2 slots}, box {64, TN, 1}
  const void* logits;
  long long logits_row, logits_col;
  int logits_dtype;  // 1 fp32, 2 bf16, 3 fp16
  int T, E, H, I, top_k, renorm;
  int dtype;         // 2 bf16, 3 fp16
  uint16_t* h;       // [slot][value, remainder][T][I]
  float value_scale, value_back, rest_back;  // h's value is that of h * value_scale; the factors that undo that and kMoeRestScale in the sums
  int* list;         // [0] = number of experts that a token chose, [16..] = their indices in increasing order
  void* out;
  long long ldo;
  int cluster_split;
  uint32_t idesc, desc_hi;
  int* status;
  unsigned long long wait_limit_ns;
};

// A stage holds SUBS swizzle spans (64 K elements) of 128 weight rows and of the tokens' rows (the second kernel's twice: value
// and remainder).
template <int TN, int STAGES, int SUBS, bool UP>
struct SmemMoe {
  static constexpr int kVRows = UP ? TN : 2 * TN;
  static constexpr int kVBox = kVRows * 128;
  static constexpr int kUBytes = SUBS * 16384;
  static constexpr int kStageBytes = kUBytes + SUBS * kVBox;
  static constexpr int kXOff = STAGES * kStageBytes;                 // UP: the up half's sums [TN][64]; otherwise recv[t / S][source][128], t / S <= (TN - 1) / S
  static constexpr int kXBytes = UP ? TN * 64 * 4 : (TN + 15) * 128 * 4;
  static constexpr int kRouteOff = kXOff + kXBytes;
  // the list of experts; first kernel: their bits, one expert's weights, and ids and weights [TN][16]
  static constexpr int kPairs = TN * kMoeMaxTopK;
  static constexpr int kRouteBytes = (kMoeMaxExperts + 16) * 4 + (UP ? (kMoeMaxExperts / 32 + kMoeMaxTokens) * 4 + kPairs * 8 : 0);
  static constexpr int kBarOff = (kRouteOff + kRouteBytes + 7) / 8 * 8;
  static constexpr int kMiscOff = kBarOff + (2 * STAGES + 4) * 8;
  static constexpr int kTotal = kMiscOff + 16;
  static_assert(!UP || STAGES * kStageBytes >= TN * (kMoeMaxExperts + 4) * 4, "the ring holds all logits while routing");
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
  if (f != f) return 0xfffffffeu;  // one below the largest integer: ranks add 1 to keys
  const uint32_t b = __float_as_uint(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float logit_of_key(uint32_t k) {
  return k == 0xfffffffeu ? __uint_as_float(0x7fffffffu) : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Logits as keys into shared memory; 0 marks no expert, or one taken already (no logit maps to 0). Four loads of a thread travel
// together: one by one, each costs an L2 round trip of 0.4 us.
template <typename T>
__device__ __forceinline__ void stage_logits(const MoeParams& p, const T* logits, uint32_t* keys, int e4, int stride) {
  const int total = p.T * e4;
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < total; i0 += 4 * kMoeThreads) {
    T raw[4];
    int at[4];
    bool in[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int i = i0 + n * kMoeThreads, t = i / e4, e = i - t * e4;
      at[n] = i < total ? t * stride + e : -1;
      in[n] = i < total && e < p.E;
      raw[n] = logits[in[n] ? t * p.logits_row + e * p.logits_col : 0];
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (at[n] >= 0) keys[at[n]] = in[n] ? logit_key((float)raw[n]) : 0u;
  }
}

// The whole block routes all tokens: ids[t][r], weights[t][r] for r < top_k (-1 and zero: not chosen), the chosen experts' bits
// in `mask`. `keys` is scratch for T * stride integers.
//
// A single token has latencies to pay one after the other, many tokens have instructions to issue; both are kept few: logits
// as ordered integers in shared memory, loads in batches, short rolled loops. One token of 128 experts takes 3 us (1 us of
// it for its logits to come), 32 of 32 5.4 us, 64 of 64 8 us.
__device__ __forceinline__ void route_all(const MoeParams& p, uint32_t* keys, int* ids, float* weights, uint32_t* mask) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int e4 = (p.E + 3) & ~3, stride = e4 + 4;  // rows of 16-byte pieces, on different banks
  if (p.logits_dtype == 1)
    stage_logits(p, reinterpret_cast<const float*>(p.logits), keys, e4, stride);
  else if (p.logits_dtype == 2)
    stage_logits(p, reinterpret_cast<const __nv_bfloat16*>(p.logits), keys, e4, stride);
  else
    stage_logits(p, reinterpret_cast<const __half*>(p.logits), keys, e4, stride);
  __syncthreads();
  const int G = p.E <= 128 ? 4 : 16;  // lanes to a token where tokens share warps
  if (p.T * p.E <= kMoeThreads && p.E <= 128) {
    // A thread per (token, expert): its rank is the number of experts ahead of it (larger, or equal with a lower index).
    const int t = tid / p.E, e = tid - t * p.E;
    uint32_t* row = keys + min(t, p.T - 1) * stride;
    const uint32_t mine = row[e];
    int rank = 0;
#pragma unroll 2
    for (int o = 0; o < e4; o += 4) {
      const uint4 k = *reinterpret_cast<const uint4*>(row + o);
      rank += (k.x + (o < e) > mine) + (k.y + (o + 1 < e) > mine) + (k.z + (o + 2 < e) > mine) + (k.w + (o + 3 < e) > mine);
    }
    const bool chosen = t < p.T && rank < p.top_k;
    if (chosen) {
      ids[t * kMoeMaxTopK + rank] = e;
      weights[t * kMoeMaxTopK + rank] = logit_of_key(mine);
    }
    __syncthreads();
    if (chosen) row[e] = 0;
  } else {
    // More pairs of experts than threads to compare them: top_k rounds per token, each taking out the largest.
    const int sub = lane & (G - 1);
#pragma unroll 1
    for (int t0 = 0; t0 < p.T; t0 += kMoeThreads / G) {
      const int t = t0 + tid / G;
      uint32_t* row = keys + min(t, p.T - 1) * stride;
#pragma unroll 1
      for (int r = 0; r < p.top_k; ++r) {
        uint32_t best = 0;
        int at = 0x7fffffff;
#pragma unroll 2
        for (int e = 4 * sub; e < e4; e += 4 * G) {
          const uint4 k = *reinterpret_cast<const uint4*>(row + e);
          if (k.x > best) best = k.x, at = e;
          if (k.y > best) best = k.y, at = e + 1;
          if (k.z > best) best = k.z, at = e + 2;
          if (k.w > best) best = k.w, at = e + 3;
        }
        for (int o = G >> 1; o > 0; o >>= 1) {
          const uint32_t k2 = __shfl_xor_sync(0xffffffffu, best, o);
          const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
          if (k2 > best || (k2 == best && a2 < at)) best = k2, at = a2;
        }
        __syncwarp();
        if (t < p.T && sub == 0) {
          row[at] = 0;
          ids[t * kMoeMaxTopK + r] = at;
          weights[t * kMoeMaxTopK + r] = logit_of_key(best);
        }
        __syncwarp();
      }
    }
  }
  __syncthreads();
  // softmax over the chosen logits, with the others' share of the sum unless the weights are renormalised
  const int WG = p.T <= kMoeThreads / 32 ? 32 : G, sub = lane & (WG - 1);
#pragma unroll 1
  for (int t0 = 0; t0 < p.T; t0 += kMoeThreads / WG) {
    const int t = t0 + tid / WG, at = min(t, p.T - 1);
    int* id = ids + at * kMoeMaxTopK;
    float* weight = weights + at * kMoeMaxTopK;
    const float top = weight[0];
    float total = 0.f;
    if (!p.renorm)
      for (int e = sub; e < p.E; e += WG)
        if (keys[at * stride + e] != 0) total += expf(logit_of_key(keys[at * stride + e]) - top);
    for (int r = sub; r < p.top_k; r += WG) total += expf(weight[r] - top);
    for (int o = WG >> 1; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    __syncwarp();  // every lane has read weight[0]
    if (t < p.T)
      for (int r = sub; r < p.top_k; r += WG) {
        // a token whose logits are all -inf goes nowhere
        const float w = top == -INFINITY ? 0.f : expf(weight[r] - top) / total;
        weight[r] = w;
        if (w != 0.f)
          atomicOr(mask + (id[r] >> 5), 1u << (id[r] & 31));
        else
          id[r] = -1;
      }
  }
}

// UP: the first kernel (gate and up products, SiLU), otherwise the second (down product and sum).
template <int TN, int STAGES, int SUBS, bool UP>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_a16w16_sm100_kernel(const __grid_constant__ MoeParams p) {
  using L = SmemMoe<TN, STAGES, SUBS, UP>;
  constexpr int kTK = 64 * SUBS;
  constexpr int NC = L::kVRows;  // accumulator columns
  constexpr uint32_t kTmemCols = 2 * NC < 32 ? 32 : 2 * NC;
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
  int* list = reinterpret_cast<int*>(sm + L::kRouteOff);  // [0] = number of experts that a token chose, [16..] = their indices
  uint32_t* mask = reinterpret_cast<uint32_t*>(list + 16 + kMoeMaxExperts);
  float* pair_w = reinterpret_cast<float*>(mask + kMoeMaxExperts / 32);
  int* ids = reinterpret_cast<int*>(pair_w + kMoeMaxTokens);
  float* weights = reinterpret_cast<float*>(ids + L::kPairs);

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
  // The logits are on the critical path and often no longer (or not yet) in L2: ask for them ahead of the wait. L2 is where
  // all writes meet, so a line that is written after this is still read right.
  if (UP && blockIdx.x == 0) {
    const int es = p.logits_dtype == 1 ? 4 : 2;
    for (int i = threadIdx.x; i < p.T * ((p.E * es + 127) / 128 + 1); i += kMoeThreads) {
      const int t = i % p.T, e = min((i / p.T) * (128 / es), p.E - 1);
      prefetch_l2(reinterpret_cast<const char*>(p.logits) + ((long long)t * p.logits_row + (long long)e * p.logits_col) * es);
    }
  }
  grid_dependency_wait();
  if (!UP) grid_launch_dependents();
  if constexpr (UP) {
    route_all(p, reinterpret_cast<uint32_t*>(sm), ids, weights, mask);  // the ring is free until the first load
    fence_proxy_async_smem();
    __syncthreads();
    // the chosen experts in increasing order
    for (int e = threadIdx.x; e < kMoeMaxExperts; e += kMoeThreads) {
      const int w = e >> 5;
      int at = __popc(mask[w] & ((1u << (e & 31)) - 1u));
      for (int j = 0; j < w; ++j) at += __popc(mask[j]);
      if (mask[w] >> (e & 31) & 1u) list[16 + at] = e;
      if (e == kMoeMaxExperts - 1) list[0] = at + (int)(mask[w] >> 31);
    }
    __syncthreads();
    if (blockIdx.x == 0)  // for the second kernel
      for (int i = threadIdx.x; i < 16 + list[0]; i += kMoeThreads) p.list[i] = list[i];
  } else {
    for (int i = threadIdx.x; i < 16 + min(p.E, p.T * p.top_k); i += kMoeThreads) list[i] = p.list[i];
    __syncthreads();
  }
  const int n_active = list[0];
  const int* experts = list + 16;

  // UP: unit = (slot, 64 gate rows), K = H. Otherwise one unit per CTA: 128 rows of H, a span of the K axis (slot, I).
  const int k_blocks = ((UP ? p.H : p.I) + kTK - 1) / kTK;
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
#pragma unroll 1
      for (int b = b_first; b < b_end; ++b) {
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
          const uint32_t fb = full_bar(stage), su = base + stage * L::kStageBytes, sv = su + L::kUBytes;
          const int s = UP ? slot0 : b / k_blocks, kb = UP ? b : b - s * k_blocks;
          const int expert = experts[s];
          mbar_arrive_expect_tx(fb, L::kStageBytes);
#pragma unroll
          for (int sub = 0; sub < SUBS; ++sub) {
            const int k0 = kb * kTK + sub * 64;
            if constexpr (UP) {
              tma_load_3d(su + sub * 16384, &p.tmap_u, k0, i0, expert, fb);
              tma_load_3d(su + sub * 16384 + 8192, &p.tmap_u, k0, p.I + i0, expert, fb);
              tma_load_2d(sv + sub * L::kVBox, &p.tmap_v, k0, 0, fb);
            } else {
              tma_load_3d(su + sub * 16384, &p.tmap_u, k0, row_tile * 128, expert, fb);
              tma_load_3d(sv + sub * L::kVBox, &p.tmap_v, k0, 0, 2 * s, fb);
              tma_load_3d(sv + sub * L::kVBox + TN * 128, &p.tmap_v, k0, 0, 2 * s + 1, fb);
            }
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == STAGES) stage = 0, phase ^= 1u;
      }
    }
    // The second kernel may take the SMs that this one leaves; not before all of this block's loads are on their way (1 %).
    if (UP) grid_launch_dependents();
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
          const uint32_t su = base + stage * L::kStageBytes, sv = su + L::kUBytes;
#pragma unroll
          for (int sub = 0; sub < SUBS; ++sub) {
            // K-major rows of 128 swizzled bytes, groups of eight 1024 bytes apart
            const uint64_t du = (uint64_t(p.desc_hi) << 32) | uint64_t((1u << 16) | (((su + sub * 16384) >> 4) & 0x3fffu));
            const uint64_t dv = (uint64_t(p.desc_hi) << 32) | uint64_t((1u << 16) | (((sv + sub * L::kVBox) >> 4) & 0x3fffu));
#pragma unroll
            for (int j = 0; j < 4; ++j)
              umma_f16<1>(tmem_base + buf * NC, du + uint64_t(2 * j), dv + uint64_t(2 * j), p.idesc, (b != b_first || sub || j) ? 1u : 0u);
          }
          umma_commit(empty_bar(stage));
          if (b + 1 == b_end) umma_commit(accf_bar(buf));
        }
        __syncwarp();
        if (++stage == STAGES) stage = 0, phase ^= 1u;
      }
    }
  } else if (warp < 6) {
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
          pair_w[et] = w * p.value_scale;
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
        const uint32_t t_acc = tmem_base + buf * NC + (uint32_t(quarter * 32) << 16);
        uint32_t r[32];
#pragma unroll
        for (int c = 0; c < NC; c += TN < 32 ? TN : 32) {
          if constexpr (TN >= 32)
            tmem_ld_32x32(t_acc + c, r);
          else
            tmem_ld_32x16(t_acc + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < (TN < 32 ? TN : 32); ++i) {
            if (c < TN)
              v[c + i] = __uint_as_float(r[i]);
            else
              v[c - TN + i] = fmaf(__uint_as_float(r[i]), p.rest_back, v[c - TN + i]) * p.value_back;  // the remainders' part
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acce_bar(buf));
      } else {
#pragma unroll
        for (int i = 0; i < TN; ++i) v[i] = 0.f;
      }
      if constexpr (UP) {
        // Lanes 64..127 hold the up rows of the gate rows in lanes 0..63: the halves swap sums through shared memory, so that
        // the first finishes the first half of the tokens and the second the others.
        const bool is_gate = row < 64;
        const int r64 = row & 63;
#pragma unroll
        for (int t = 0; t < TN; ++t)
          if ((t < TN / 2) != is_gate) xs[t * 64 + r64] = v[t];
        named_bar_sync(2, 128);
        const int i = (u - slot * tiles) * 64 + r64;
        if (i < p.I) {
          const size_t plane = (size_t)p.T * p.I;
          uint16_t* dst = p.h + 2 * slot * plane + i;
#pragma unroll
          for (int j = 0; j < TN / 2; ++j) {
            const int t = is_gate ? j : TN / 2 + j;
            if (t < p.T) {
              const float w = pair_w[t], other = xs[t * 64 + r64], own = is_gate ? v[j] : v[TN / 2 + j];
              const float g = is_gate ? own : other, up = is_gate ? other : own;
              // a pair that was not chosen is zero whatever its sums are
              const float a = w == 0.f ? 0.f : w * __fdividef(g, 1.f + __expf(-g)) * up;
              uint16_t bits, rest;
              if (p.dtype == 2) {
                const __nv_bfloat16 h = __float2bfloat16_rn(a), l = __float2bfloat16_rn(a - __bfloat162float(h));
                bits = __bfloat16_as_ushort(h), rest = __bfloat16_as_ushort(l);
              } else {
                const __half h = __float2half_rn(a), l = __float2half_rn((a - __half2float(h)) * kMoeRestScale);
                bits = __half_as_ushort(h), rest = __half_as_ushort(l);
              }
              if ((p.dtype == 2 ? bits & 0x7f80u : bits & 0x7c00u) == (p.dtype == 2 ? 0x7f80u : 0x7c00u)) rest = 0;  // infinite or NaN
              dst[(size_t)t * p.I] = bits;
              dst[plane + (size_t)t * p.I] = rest;
            }
          }
        }
        named_bar_sync(1, 128);  // xs and pair_w may be rewritten
      } else if (cluster_mode) {
        // Column t belongs to CTA t % S: a warp's 32 rows are 128 contiguous bytes of recv[t / S][source][row].
        if (cluster_wait_due) {
          cluster_wait();
          cluster_wait_due = false;
        }
        const uint32_t recv = base + L::kXOff + (uint32_t)row * 4u;
        int slab = 0, owner = 0;
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          if (t < p.T) {
            const uint32_t dst = mapa_cluster(recv + (uint32_t)((slab + rank) * 128) * 4u, (uint32_t)owner);
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(v[t]) : "memory");
            if (++owner == S) owner = 0, slab += S;
          }
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
    if (warp >= 2 && warp < 6) {
      const int row = threadIdx.x - 64, hrow = row_tile * 128 + row;
      const float* recv = reinterpret_cast<const float*>(sm + L::kXOff) + row;
      if (hrow < p.H) {
        for (int t = rank; t < p.T; t += S, recv += S * 128) {
          float x = 0.f;
          for (int src = 0; src < S; ++src) x += recv[src * 128];  // in rank order
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
