// 8-bit floating-point GEMM with one fp32 scale per block of 128 along K, for sm_100a.
//
//   D[p, q] = sum over K blocks b of  us[p, b] * vs[q, b] * (sum over k in block b of U[p, k] * V[q, k])  (+ bias)
//
// U is the operand on the 128-row MMA axis, V the one on the MMA N axis ((A, B), or (B, A) for swap_ab, which writes D^T).
// A scale belongs to one row of its operand or to 128 of them; either operand may be K-contiguous or row-contiguous.
//
// Mathematics and split of the work. The products of a K block are exact in fp32 and summed by tcgen05.mma (kind::f8f6f4,
// four K = 32 instructions) into an accumulator in TMEM that starts at zero for every block; scales are not powers of
// two in general, so the tensor core cannot apply them. Eight epilogue warps read that accumulator, multiply by
// us[p] * vs[q] and add to the running sums, which stay in their registers for the whole tile (128 fp32 values per
// thread of a 256-column tile). TMEM holds two (256 columns) or four accumulators, so the tensor core works on the next
// blocks meanwhile. Per 128 x 256 half-tile and block the tensor core needs 512 cycles and the eight warps about 400 issue
// slots per scheduler; a block takes 750 to 830 cycles, the rest being the chain accumulator done -> read -> handed back ->
// next instructions, twice deep. 8192^3: 454 us in a burst (2420 TFLOP/s), 534 us under the power cap; 2048 x 4096 x 4096:
// 33 us; with a scale per row on both sides (two multiplications and a shared-memory read per element) 647 us.
//
// PACKED: where all scales are powers of two (what the quantizer makes), the tensor core applies them itself
// (kind::mxf8f6f4, one exponent per row and 32 elements): up to 32 K blocks are summed in one accumulator (k8Chunk says why no more),
// the epilogue warps only drain it, and the operands' way into the SM is what is left (with plain kind::f8f6f4 and no scales at all
// 31.1 us where this took 31.3, 2048 x 4096 x 4096, before its fifth ring stage). Replayed from a graph, operands in L2: 8192^3 374 -
// 382 us in a burst in any layout, 2048 x 4096 x 4096 32.8 us, 4096 x 4096 x 2048 with both operands row-contiguous 34.4 us (a scale per
// row on both sides above: 56 us).
//
// Roles (384 threads): warp 0 = TMA producer, warp 1 = TMEM owner and MMA issuer, warps 2-3 = scale loaders (PACKED: idle, the
// producer loads the exponents), warps 4-11 = epilogue (warp w reads TMEM lanes 32 * (w % 4).. and column half (w - 4) / 4). The
// scale loaders copy the scales of a K block into an eight-deep ring with 4-byte cp.async, whose completion arrives on the
// ring's barrier by itself: any strides are served, nobody waits for a load, and rows outside the operand get zero.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace b200 {

constexpr int k8TileP = 128;   // U rows per CTA
constexpr int k8TK = 128;      // K elements per block and pipeline stage: one scale, one 128-byte swizzle span
constexpr int k8Threads = 384;
constexpr int k8EpiThreads = 256;
constexpr int k8ScaleStages = 8;
constexpr int k8UBytes = k8TileP * k8TK;
// PACKED: K blocks that the tensor core sums by itself. Its additions do not round to nearest, they cut off: sums of positive
// products in one accumulator come out 1e-6 too small at K = 4096, 4.5e-5 at 65536 (values of either sign: off by 2.2e-7 and 7.6e-6). So
// the sums over each 32 blocks are added in fp32 registers. That costs small products of long sums 4 to 5 % (1024 x 1024 x 65536, 256 x
// 2048 x 16384) and, for the addition to nothing that short sums have, 4096 x 4096 x 512 4 %, else 1 % at most. (Kernels without it for up to 32 blocks: a linear layer's step
// that uses both kinds takes 4 to 8 us more, 1000 x 3000 x 4100 118 instead of 110.)
constexpr int k8Chunk = 32;

struct alignas(64) Gemm8Params {
  CUtensorMap tmap_u;
  CUtensorMap tmap_v;
  CUtensorMap tmap_us, tmap_vs;  // PACKED: the exponent tiles as rows of 128 bytes, box 4 rows
  CUtensorMap tmap_out;  // box = 32 rows x 128 bytes (valid when tma_store != 0)
  const float* u_scale;
  const float* v_scale;
  long long us_row, us_kb, vs_row, vs_kb;  // element strides of the scales: per row (or block of 128 rows), per K block
  int us_shift, vs_shift;                  // 0: a scale per row, 7: per 128 rows
  void* out;
  const void* bias;
  int* status;
  long long ldo;
  int P, Q;
  int tiles_p, tiles_q, num_tiles, kb_total;
  int cluster_split;  // > 1: that many CTAs of a cluster share a tile's K blocks and reduce through distributed shared memory
  int group_p;        // grouped rasterisation over tile rows of P (0 = off)
  int swap_out;       // 1: D^T is written (out[q * ldo + p]); bias indexed by p
  int tma_store;
  int out_dtype, bias_dtype;  // 1 fp32, 2 bf16, 3 fp16
  int u_mn_major, v_mn_major;
  uint32_t idesc;
  uint32_t u_desc_hi, u_desc_lo, v_desc_hi, v_desc_lo;
  uint32_t u_kstep, v_kstep;  // start-address increment (16-byte units) per K = 32 MMA
  unsigned long long wait_limit_ns;
};

// VVEC: V has a scale per row; otherwise one per 128 rows, so one value serves each half of a tile's columns.
// PACKED: scales are powers of two, in exponent tiles, and the tensor core applies them.
template <int TILE_Q, int STAGES, int CG, bool VVEC, bool PACKED>
struct Smem8 {
  static constexpr int kVRows = TILE_Q / CG;
  static constexpr int kVBytes = kVRows * k8TK;
  static constexpr int kStageBytes = k8UBytes + kVBytes;
  static constexpr int kOutOff = STAGES * kStageBytes;
  // swizzled 32 x 128-byte images of the epilogue warps on their way out: two each where a warp has two or more segments to
  // send (2 % on 256 columns; the fifth ring stage that they displace gained nothing), else one. PACKED has the fifth stage:
  // 2048 x 4096 x 4096 4 % faster when it was chosen (a short K pays: 4096 x 4096 x 512 15.8 instead of 14.5 us)
  static constexpr int kImages = TILE_Q >= 256 && !PACKED ? 2 : 1;
  static constexpr int kStagingBytes = TILE_Q >= 64 ? 8 * kImages * 4096 : 0;
  static constexpr int kRecvBytes = CG == 1 && !PACKED ? k8TileP * TILE_Q * 4 : 0;   // cluster split: [source][own column][128] fp32
  static constexpr int kOutBytes = kRecvBytes > kStagingBytes ? kRecvBytes : kStagingBytes;
  static constexpr int kScaleOff = kOutOff + kOutBytes;
  static constexpr int kScaleVals = k8TileP + (VVEC ? TILE_Q : 4);
  static constexpr int kTileBytes = 512 * (1 + TILE_Q / 128);  // PACKED: exponents of a stage, U's then V's
  static constexpr int kScaleBytes = PACKED ? STAGES * kTileBytes : k8ScaleStages * kScaleVals * 4;
  // accumulators in TMEM; PACKED needs the other columns for the exponents of its stages
  static constexpr int kBufs = PACKED ? 256 / TILE_Q : TILE_Q > 128 ? 2 : 4;
  static constexpr int kBarOff = kScaleOff + kScaleBytes;
  static constexpr int kNumBars = 2 * STAGES + 2 * k8ScaleStages + kBufs;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kTotal = kMiscOff + 16;
  static constexpr int kDynBytes = kTotal + 1024;  // slack for manual 1024-byte alignment
};

__device__ __forceinline__ void report_abort8(int* status, int role, int unit) {
  if (status != nullptr && atomicCAS(status, 0, 1) == 0) {
    status[1] = blockIdx.x;
    status[2] = role;
    status[3] = unit;
  }
}

__device__ __forceinline__ float load_as_float(const void* ptr, long long i, int dtype) {
  if (dtype == 1) return reinterpret_cast<const float*>(ptr)[i];
  if (dtype == 2) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(ptr)[i]);
  return __half2float(reinterpret_cast<const __half*>(ptr)[i]);
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, int dtype) {
  if (dtype == 2) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void store_one(void* out, long long i, float x, int dtype) {
  if (dtype == 1)
    reinterpret_cast<float*>(out)[i] = x;
  else if (dtype == 2)
    reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(x);
  else
    reinterpret_cast<__half*>(out)[i] = __float2half_rn(x);
}

// bias[q .. q + 8) added to v; entries outside Q are skipped.
__device__ __forceinline__ void add_bias8(const Gemm8Params& p, float (&v)[8], int q) {
  if (p.bias == nullptr) return;
  const char* src = reinterpret_cast<const char*>(p.bias) + (long long)q * (p.bias_dtype == 1 ? 4 : 2);
  if (p.bias_dtype != 1 && q + 8 <= p.Q && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const uint4 w = *reinterpret_cast<const uint4*>(src);
    const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p.bias_dtype == 2) {
        v[2 * i] += __uint_as_float(wd[i] << 16);
        v[2 * i + 1] += __uint_as_float(wd[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&wd[i]));
        v[2 * i] += f.x, v[2 * i + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (q + i < p.Q) v[i] += load_as_float(p.bias, q + i, p.bias_dtype);
  }
}

// Eight consecutive values of row `prow` from column q on: vectors where the address allows, single values at ragged edges.
__device__ __forceinline__ void store_row8(const Gemm8Params& p, const float (&v)[8], int prow, int q) {
  const long long i = (long long)prow * p.ldo + q;
  char* dst = reinterpret_cast<char*>(p.out) + i * (p.out_dtype == 1 ? 4 : 2);
  if (q + 8 <= p.Q && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
    if (p.out_dtype == 1) {
      reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack16(v[0], v[1], p.out_dtype), pack16(v[2], v[3], p.out_dtype),
                                                  pack16(v[4], v[5], p.out_dtype), pack16(v[6], v[7], p.out_dtype));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (q + j < p.Q) store_one(p.out, i + j, v[j], p.out_dtype);
  }
}

__device__ __forceinline__ void raster8(const Gemm8Params& p, int tile, int& tp, int& tq) {
  if (p.group_p > 0) {
    const int per_group = p.group_p * p.tiles_q;
    const int g = tile / per_group;
    const int first = g * p.group_p;
    const int rows = min(p.tiles_p - first, p.group_p);
    const int r = tile - g * per_group;
    tp = first + r % rows;
    tq = r / rows;
  } else {
    tp = tile / p.tiles_q;
    tq = tile - tp * p.tiles_q;
  }
}

// Both barriers' phases, the whole warp with one verdict. The two probes are in flight together; nothing else is on the path
// of a warp that finds them complete.
__device__ __forceinline__ bool wait_two(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1, volatile int* abort_flag,
                                         unsigned long long limit) {
  const bool a = mbar_try_wait(bar0, parity0), b = mbar_try_wait(bar1, parity1);
  if (__all_sync(0xffffffffu, a && b)) return true;
  const bool good = mbar_wait(bar0, parity0, abort_flag, limit) && mbar_wait(bar1, parity1, abort_flag, limit);
  return __all_sync(0xffffffffu, good);
}

template <int TILE_Q, int STAGES, int CG, bool VVEC, bool PACKED>
__global__ void __launch_bounds__(k8Threads, 1) gemm_a8w8_sm100_kernel(const __grid_constant__ Gemm8Params p) {
  using L = Smem8<TILE_Q, STAGES, CG, VVEC, PACKED>;
  constexpr int HC = TILE_Q / 2;               // columns per epilogue warp (the two warps of a lane quarter split the tile)
  constexpr int CW = HC < 32 ? HC : 32;        // columns per tcgen05.ld
  constexpr int NCH = HC / CW;
  constexpr int kBufs = L::kBufs;
  constexpr uint32_t kTmemCols = PACKED ? 512 : TILE_Q * kBufs < 32 ? 32 : TILE_Q * kBufs;
  constexpr uint32_t kExpCols = 4 * (1 + TILE_Q / 128);  // TMEM columns of a stage's exponents, behind the accumulators
  static_assert(!PACKED || (TILE_Q % 128 == 0 && 256 + STAGES * kExpCols <= 512), "exponents in TMEM");
  // 128 running sums, 32 loaded values and addresses do not fit the 168 registers a thread of 384 gets at launch: the
  // wide tile moves registers to the epilogue, 128 * 40 + 256 * 232 = 384 * 168.
  constexpr bool kMoveRegs = HC > 64;
  // Look for the next block's barriers before this block's last additions. It pays where those are long (256 columns with a
  // scale each: 58.8 -> 54.2 us at 4096 x 4096 x 2048) and costs elsewhere (one scale per half: 454 -> 479 us at 8192^3; 128
  // columns: 61 -> 64 us).
  constexpr bool kLookAhead = VVEC && HC > 64;
  constexpr uint32_t kTxBytes = CG * L::kStageBytes;  // both CTAs of a pair count on the leader's barrier

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const uint32_t bar0 = base + L::kBarOff;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  // The MMAs of the K block in stage s are done: the stage may be loaded again, and the block's accumulator may be read. One
  // commit per block serves both: an accumulator is read before its stage can have come round again (kBufs < STAGES).
  auto done_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto sfull_bar = [&](int s) { return bar0 + 8u * (2 * STAGES + s); };
  auto sempty_bar = [&](int s) { return bar0 + 8u * (2 * STAGES + k8ScaleStages + s); };
  auto acce_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + 2 * k8ScaleStages + b); };
  static_assert(kBufs <= STAGES, "an accumulator is read before its stage is loaded again");
  volatile uint32_t* tmem_ptr_s = reinterpret_cast<volatile uint32_t*>(sm + L::kMiscOff);
  volatile int* abort_s = reinterpret_cast<volatile int*>(sm + L::kMiscOff + 4);
  const unsigned long long wait_limit = p.wait_limit_ns;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const bool cluster_mode = CG == 1 && p.cluster_split > 1;
  const int rank = (CG == 2 || cluster_mode) ? (int)cluster_ctarank() : 0;
  const int prank = CG == 2 ? rank : 0;  // rank inside a pair; 0 issues the MMAs
  // cluster split: one tile per cluster, slice `rank` takes K blocks rank, rank + S, ...; otherwise this walker (CTA or
  // pair) takes tiles walker, walker + walkers, ... with all their K blocks
  const int walkers = CG == 2 ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const int tile0 = cluster_mode ? (int)blockIdx.x / p.cluster_split : CG == 2 ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int tile_step = cluster_mode ? p.num_tiles : walkers;
  const int kb0 = cluster_mode ? rank : 0;
  const int kbstep = cluster_mode ? p.cluster_split : 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(done_bar(s), 1);
    }
    for (int s = 0; s < k8ScaleStages; ++s) {
      mbar_init(sfull_bar(s), PACKED ? 1 : 64);  // PACKED: the first of them are the accumulators' "complete"
      mbar_init(sempty_bar(s), 8);
    }
    for (int b = 0; b < kBufs; ++b) mbar_init(acce_bar(b), 8 * CG);
    *abort_s = 0;
    fence_mbar_init();
    prefetch_tmap(&p.tmap_u);
    prefetch_tmap(&p.tmap_v);
    if (p.tma_store) prefetch_tmap(&p.tmap_out);
    if (PACKED) {
      prefetch_tmap(&p.tmap_us);
      prefetch_tmap(&p.tmap_vs);
    }
  }
  if (warp == 1) {
    tmem_alloc<CG>(smem_u32(const_cast<uint32_t*>(tmem_ptr_s)), kTmemCols);
    tmem_relinquish<CG>();
  }
  tc_fence_before();
  __syncthreads();
  // Every CTA of a cluster must be running before anything is sent across it: a pair needs that before its first load,
  // cluster split-K only before the epilogue sends its sums (each thread arrives now and waits later).
  bool cluster_wait_due = false;
  if (CG == 2) {
    cluster_arrive();
    cluster_wait();
  } else if (cluster_mode) {
    cluster_arrive();
    cluster_wait_due = true;
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr_s;
  grid_dependency_wait();
  grid_launch_dependents();

  if (warp < 4) {
    if constexpr (kMoveRegs) reg_dec<40>();
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer (one per CTA)
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      auto load = [&](uint32_t dst, const void* map, int x, int y, uint32_t fb) {
        if constexpr (CG == 2)
          tma_load_2d_pair(dst, map, x, y, fb);
        else
          tma_load_2d(dst, map, x, y, fb);
      };
#pragma unroll 1
      for (int tile = tile0; ok && tile < p.num_tiles; tile += tile_step) {
        int tp, tq;
        raster8(p, tile, tp, tq);
        const int p0 = (tp * CG + prank) * k8TileP, q0 = tq * TILE_Q + prank * L::kVRows;
#pragma unroll 1
        for (int kb = kb0; kb < p.kb_total; kb += kbstep) {
          if (issued >= STAGES) {
            int good = 1;
            if (lane == 0) good = mbar_wait(done_bar(stage), phase ^ 1u, abort_s, wait_limit) ? 1 : 0;
            good = __shfl_sync(0xffffffffu, good, 0);
            if (!good) {
              if (lane == 0) report_abort8(p.status, 0, tile);
              ok = false;
              break;
            }
          }
          uint32_t fb = full_bar(stage);
          if constexpr (CG == 2) fb = mapa_cluster(fb, 0);
          if (elect_one()) {
            const uint32_t su = base + stage * L::kStageBytes, sv = su + k8UBytes;
            const int k0 = kb * k8TK;
            const bool exps = PACKED && (kb & 3) == 0;  // with the first of four blocks
            if (prank == 0) mbar_arrive_expect_tx(full_bar(stage), exps ? kTxBytes + CG * L::kTileBytes : kTxBytes);
            if (!p.u_mn_major)
              load(su, &p.tmap_u, k0, p0, fb);
            else
              load(su, &p.tmap_u, p0, k0, fb);
            if (!p.v_mn_major)
              load(sv, &p.tmap_v, k0, q0, fb);
            else
              load(sv, &p.tmap_v, q0, k0, fb);
            if (exps) {
              const uint32_t se = base + L::kScaleOff + stage * L::kTileBytes;
              const int q = kb >> 2;
              load(se, &p.tmap_us, 0, 4 * (int)(q * p.us_kb + (tp * CG + prank) * p.us_row), fb);
#pragma unroll
              for (int j = 0; j < TILE_Q / 128; ++j)  // both CTAs of a pair need V's
                load(se + 512u * (1 + j), &p.tmap_vs, 0, 4 * (int)(q * p.vs_kb + (tq * (TILE_Q / 128) + j) * p.vs_row), fb);
            }
          }
          __syncwarp();
          ++issued;
          if (++stage == STAGES) stage = 0, phase ^= 1u;
        }
      }
      if (!ok && lane == 0) {
        // Loads already issued still write shared memory: give them a bounded time to land before the block ends.
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) {
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issuer (the pair's leader only)
      if (prank == 0) {
        int stage = 0;
        uint32_t phase = 0;
        int g = 0;  // K blocks so far; each has an accumulator of its own (PACKED: chunks)
        int group = -1;  // PACKED: fours of K blocks so far
        bool ok = true;
#pragma unroll 1
        for (int tile = tile0; ok && tile < p.num_tiles; tile += tile_step, g += PACKED) {
#pragma unroll 1
          for (int kb = kb0; kb < p.kb_total; kb += kbstep, g += !PACKED) {
            if (PACKED && kb != 0 && kb % k8Chunk == 0) ++g;
            const int buf = g % kBufs;
            if (PACKED && (kb & 3) == 0) ++group;
            if (!wait_two(acce_bar(buf), ((g / kBufs) & 1) ^ 1u, full_bar(stage), phase, abort_s, wait_limit)) {
              if (lane == 0) report_abort8(p.status, 1, tile);
              ok = false;
              break;
            }
            tc_fence_after();
            if (elect_one()) {
              const uint32_t su = base + stage * L::kStageBytes, sv = su + k8UBytes;
              const uint64_t du = (uint64_t(p.u_desc_hi) << 32) | uint64_t(p.u_desc_lo | ((su >> 4) & 0x3fffu));
              const uint64_t dv = (uint64_t(p.v_desc_hi) << 32) | uint64_t(p.v_desc_lo | ((sv >> 4) & 0x3fffu));
              const uint32_t d_tmem = tmem_base + buf * TILE_Q;
              if constexpr (PACKED) {
                // Four blocks share a place in TMEM, one byte each. There are STAGES places: before one is written again its four
                // blocks have left the ring.
                const uint32_t se = base + L::kScaleOff + stage * L::kTileBytes, exps = tmem_base + 256 + (group % STAGES) * kExpCols;
                // rows of 16 bytes without swizzle, eight of them 128 bytes apart from the next eight
                const uint64_t de = (uint64_t((128u >> 4) | (1u << 14)) << 32) | uint64_t((1u << 16) | ((se >> 4) & 0x3fffu));
                if ((kb & 3) == 0) {
#pragma unroll
                  for (int j = 0; j <= TILE_Q / 128; ++j) tmem_copy_scales<CG>(exps + 4 * j, de + uint64_t(j * (512 >> 4)));
                }
                const uint32_t idesc = p.idesc | (uint32_t)(kb & 3) << 4 | (uint32_t)(kb & 3) << 29;  // the byte of V's and of U's
#pragma unroll
                for (int j = 0; j < k8TK / 32; ++j)
                  umma_mxf8<CG>(d_tmem, du + uint64_t(j * p.u_kstep), dv + uint64_t(j * p.v_kstep), idesc, exps, exps + 4,
                                kb % k8Chunk != 0 || j != 0 ? 1u : 0u);
              }
#pragma unroll
              for (int j = 0; j < (PACKED ? 0 : k8TK / 32); ++j)
                umma_f8<CG>(d_tmem, du + uint64_t(j * p.u_kstep), dv + uint64_t(j * p.v_kstep), p.idesc, j != 0 ? 1u : 0u);
              if constexpr (CG == 2) {
                umma_commit_pair(mapa_cluster(done_bar(stage), 0));
                umma_commit_pair(mapa_cluster(done_bar(stage), 1));
              } else {
                umma_commit(done_bar(stage));
              }
              if (PACKED && (kb + 1 == p.kb_total || kb % k8Chunk == k8Chunk - 1)) {
                if constexpr (CG == 2) {
                  umma_commit_pair(mapa_cluster(sfull_bar(buf), 0));
                  umma_commit_pair(mapa_cluster(sfull_bar(buf), 1));
                } else {
                  umma_commit(sfull_bar(buf));
                }
              }
            }
            __syncwarp();
            if (++stage == STAGES) stage = 0, phase ^= 1u;
          }
        }
      }
    } else if constexpr (!PACKED) {
      // ------------------------------------------------------------------ scale loaders (warps 2 and 3)
      const int lt = threadIdx.x - 64;
      int g = 0;
      bool ok = true;
#pragma unroll 1
      for (int tile = tile0; ok && tile < p.num_tiles; tile += tile_step) {
        int tp, tq;
        raster8(p, tile, tp, tq);
        const int p0 = (tp * CG + prank) * k8TileP, q0 = tq * TILE_Q;
        // source of each value this thread fetches, without the K block's offset; a row outside the operand has none
        const float* us[2];
        bool uin[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = p0 + lt + 64 * i;
          uin[i] = row < p.P;
          us[i] = p.u_scale + (long long)((uin[i] ? row : 0) >> p.us_shift) * p.us_row;
        }
        constexpr int kVPer = VVEC ? (TILE_Q + 63) / 64 : 1;
        const float* vs[kVPer];
        bool vin[kVPer], vmine[kVPer];
#pragma unroll
        for (int i = 0; i < kVPer; ++i) {
          const int c = VVEC ? lt + 64 * i : lt * HC;  // blocks of 128: one value per column half
          vmine[i] = VVEC ? c < TILE_Q : lt < 2;
          const int col = q0 + c;
          vin[i] = vmine[i] && col < p.Q;
          vs[i] = p.v_scale + (long long)((vin[i] ? col : 0) >> p.vs_shift) * p.vs_row;
        }
#pragma unroll 1
        for (int kb = kb0; kb < p.kb_total; kb += kbstep, ++g) {
          const int ss = g % k8ScaleStages;
          if (g >= k8ScaleStages && !mbar_wait(sempty_bar(ss), ((g / k8ScaleStages) & 1) ^ 1u, abort_s, wait_limit)) {
            report_abort8(p.status, 2, tile);
            ok = false;
            break;
          }
          const uint32_t dst = base + L::kScaleOff + (uint32_t)(ss * L::kScaleVals) * 4u;
#pragma unroll
          for (int i = 0; i < 2; ++i) cp_async_4(dst + (uint32_t)(lt + 64 * i) * 4u, us[i] + (uin[i] ? kb * p.us_kb : 0), uin[i] ? 4 : 0);
#pragma unroll
          for (int i = 0; i < kVPer; ++i)
            if (vmine[i]) cp_async_4(dst + (uint32_t)(k8TileP + lt + 64 * i) * 4u, vs[i] + (vin[i] ? kb * p.vs_kb : 0), vin[i] ? 4 : 0);
          cp_async_arrive(sfull_bar(ss));
        }
      }
      cp_async_commit();
      cp_async_wait<0>();  // nothing writes shared memory after the block has ended
    }
  } else {
    // -------------------------------------------------------------------- epilogue (warps 4..11)
    if constexpr (kMoveRegs) reg_inc<232>();
    const int quarter = warp & 3;
    const int half = (warp - 4) >> 2;
    const int row = quarter * 32 + lane;
    const float* ring = reinterpret_cast<const float*>(sm + L::kScaleOff);
    const uint32_t image0 = base + L::kOutOff + (uint32_t)((warp - 4) * L::kImages) * 4096u;
    uint32_t image = image0;
    int g = 0, stage = 0;
    uint32_t phase = 0;
#pragma unroll 1
    for (int tile = tile0; tile < p.num_tiles; tile += tile_step) {
      int tp, tq;
      raster8(p, tile, tp, tq);
      const int prow = (tp * CG + prank) * k8TileP + row;
      const int qbase = tq * TILE_Q + half * HC;
      uint64_t acc2[HC / 2];  // two neighbouring columns each: fma.rn.f32x2 does both in one issue slot
#pragma unroll
      for (int i = 0; i < HC / 2; ++i) acc2[i] = 0;
      auto acc = [&](int i) { return __uint_as_float((uint32_t)(i & 1 ? acc2[i >> 1] >> 32 : acc2[i >> 1])); };
      bool ok = true, seen = false;
      if constexpr (PACKED) {
        // The sums of one chunk, added to those of the chunks before.
        auto take = [&]() {
          const int buf = g % kBufs;
          const uint32_t done = (g / kBufs) & 1;
          ++g;
          ok = wait_two(sfull_bar(buf), done, sfull_bar(buf), done, abort_s, wait_limit);
          if (ok) {
            tc_fence_after();
            const uint32_t t_acc = tmem_base + buf * TILE_Q + half * HC + (uint32_t(quarter * 32) << 16);
#pragma unroll
            for (int c = 0; c < NCH; c += 2) {
              uint32_t r[2][32];
              tmem_ld_32x32(t_acc + c * 32, r[0]);
              tmem_ld_32x32(t_acc + c * 32 + 32, r[1]);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 64; i += 2)
                acc2[(c * 32 + i) / 2] = add_f32x2(acc2[(c * 32 + i) / 2], pack_u32x2(r[i >> 5][i & 31], r[i >> 5][(i & 31) + 1]));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (CG == 2 && prank != 0)
                mbar_arrive_remote(acce_bar(buf), 0);
              else
                mbar_arrive(acce_bar(buf));
            }
          }
        };
        // The last one stands apart: with all of them in the loop 4096 x 4096 x 512 takes 18.5 us instead of 17.1.
#pragma unroll 1
        for (int kb = k8Chunk; ok && kb < p.kb_total; kb += k8Chunk) take();
        if (ok) take();
      }
#pragma unroll 1
      for (int kb = kb0; !PACKED && kb < p.kb_total; kb += kbstep, ++g) {
        const int buf = g % kBufs, ss = g % k8ScaleStages;
        // The verdict is the warp's: tcgen05.ld needs all its lanes.
        if (!(kLookAhead && __all_sync(0xffffffffu, seen)) &&
            !wait_two(sfull_bar(ss), (g / k8ScaleStages) & 1, done_bar(stage), phase, abort_s, wait_limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t t_acc = tmem_base + buf * TILE_Q + half * HC + (uint32_t(quarter * 32) << 16);
        uint32_t ra[32], rb[32];
        auto load_chunk = [&](uint32_t(&r)[32], int c) {
          if constexpr (CW == 32)
            tmem_ld_32x32(t_acc + c * CW, r);
          else if constexpr (CW == 16)
            tmem_ld_32x16(t_acc + c * CW, r);
          else
            tmem_ld_32x8(t_acc + c * CW, r);
        };
        load_chunk(ra, 0);
        if (NCH > 1) load_chunk(rb, 1);
        const float* sc = ring + ss * L::kScaleVals;
        // The two scales are multiplied first: their product has to be in fp32's normal range, see the header. (A second copy of
        // these additions for products outside it, chosen by a vote, costs all calls: 8192^3 429 -> 577 us.)
        const float su = VVEC ? sc[row] : sc[row] * sc[k8TileP + half];
        const float* sv = sc + k8TileP + half * HC;
        const uint64_t su2 = pack_f32x2(su, su);
        auto add_chunk = [&](const uint32_t(&r)[32], int c) {
#pragma unroll
          for (int i = 0; i < CW; i += 4) {
            uint64_t s0 = su2, s1 = su2;
            if constexpr (VVEC) {
              const float4 v4 = *reinterpret_cast<const float4*>(sv + c * CW + i);
              s0 = mul_f32x2(su2, pack_f32x2(v4.x, v4.y));
              s1 = mul_f32x2(su2, pack_f32x2(v4.z, v4.w));
            }
            uint64_t* a = acc2 + (c * CW + i) / 2;
            a[0] = fma_f32x2(pack_u32x2(r[i], r[i + 1]), s0, a[0]);
            a[1] = fma_f32x2(pack_u32x2(r[i + 2], r[i + 3]), s1, a[1]);
          }
        };
        auto release = [&]() {  // the accumulator has been read: it may be written again
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2 && prank != 0)
              mbar_arrive_remote(acce_bar(buf), 0);
            else
              mbar_arrive(acce_bar(buf));
          }
        };
        // Two loads travel together and each buffer is refilled as soon as its values are added.
#pragma unroll
        for (int c = 0; c < NCH; c += 2) {
          tmem_ld_wait();
          if (c + 2 >= NCH) {
            release();
            if constexpr (kLookAhead) {
              const int nstage = stage + 1 == STAGES ? 0 : stage + 1;
              seen = mbar_test(sfull_bar((g + 1) % k8ScaleStages), ((g + 1) / k8ScaleStages) & 1) &&
                     mbar_test(done_bar(nstage), nstage == 0 ? phase ^ 1u : phase);
            }
          }
          add_chunk(ra, c);
          if (c + 2 < NCH) load_chunk(ra, c + 2);
          if (c + 1 < NCH) add_chunk(rb, c + 1);
          if (c + 3 < NCH) load_chunk(rb, c + 3);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(sempty_bar(ss));  // the scales are read
        if (++stage == STAGES) stage = 0, phase ^= 1u;
      }
      if (!ok) {
        if (lane == 0) report_abort8(p.status, 3, tile);
        break;
      }

      if (cluster_mode) {
        // Column c of the tile belongs to CTA c / (TILE_Q / S): the 32 rows of a warp are 128 contiguous bytes of that CTA's
        // recv[source][own column][row].
        if (cluster_wait_due) {
          cluster_wait();
          cluster_wait_due = false;
        }
        const int own_log2 = __ffs(TILE_Q / p.cluster_split) - 1;
        const uint32_t recv = base + L::kOutOff + (uint32_t)row * 4u;
#pragma unroll
        for (int i = 0; i < HC; ++i) {
          const int c = half * HC + i;
          const uint32_t dst = mapa_cluster(recv + (uint32_t)(((rank << own_log2) + (c & ((1 << own_log2) - 1))) * k8TileP) * 4u,
                                            (uint32_t)(c >> own_log2));
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(acc(i)) : "memory");
        }
      } else if (p.swap_out) {
        // D^T: the lanes of a warp write neighbouring addresses
        if (prow < p.P) {
          const float b = p.bias != nullptr ? load_as_float(p.bias, prow, p.bias_dtype) : 0.f;
#pragma unroll
          for (int i = 0; i < HC; ++i)
            if (qbase + i < p.Q) store_one(p.out, (long long)(qbase + i) * p.ldo + prow, acc(i) + b, p.out_dtype);
        }
      } else if constexpr (HC >= 32) {
        // One 128-byte row segment per lane into the warp's swizzled image (16-byte piece j of row t at j ^ (t % 8)). The image
        // leaves by TMA, clipped at the matrix's edges; where C's rows do not start on 16 bytes the warp writes it row by
        // row, neighbouring lanes neighbouring values (a lane per row would touch 32 sectors for every value).
        const int row0 = (tp * CG + prank) * k8TileP + quarter * 32;
        uint32_t row_base = image + (uint32_t)lane * 128u;
        auto acquire = [&]() {  // the store that last read the next image is done with it
          if (lane == 0) tma_store_wait_read<L::kImages - 1>();
          __syncwarp();
          if (L::kImages > 1) {
            image = image0 + ((image - image0) ^ 4096u);
            row_base = image + (uint32_t)lane * 128u;
          }
        };
        auto flush = [&](int col0, int ncols) {  // ncols: columns of this segment inside the tile
          if (p.tma_store) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (row0 < p.P && col0 < p.Q) tma_store_2d(&p.tmap_out, col0, row0, image);
              tma_store_commit();
            }
            return;
          }
          __syncwarp();
          const int rows = min(32, p.P - row0), cols = min(ncols, p.Q - col0);
          if (p.out_dtype == 1) {
            float* dst = reinterpret_cast<float*>(p.out) + (long long)row0 * p.ldo + col0 + lane;
            for (int t = 0; t < rows; ++t, dst += p.ldo)
              if (lane < cols) *dst = *reinterpret_cast<const float*>(sm + (image - base) + t * 128 + ((((lane >> 2) ^ (t & 7)) << 4) | ((lane & 3) << 2)));
          } else {
            uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (long long)row0 * p.ldo + col0;
            for (int t = 0; t < rows; ++t, dst += p.ldo) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(sm + (image - base) + t * 128 + ((((lane >> 2) ^ (t & 7)) << 4) | ((lane & 3) << 2)));
              if (2 * lane + 1 < cols && (reinterpret_cast<uintptr_t>(dst) & 3) == 0) {
                reinterpret_cast<uint32_t*>(dst)[lane] = w;
              } else {
                if (2 * lane < cols) dst[2 * lane] = (uint16_t)w;
                if (2 * lane + 1 < cols) dst[2 * lane + 1] = (uint16_t)(w >> 16);
              }
            }
          }
          __syncwarp();  // the image may be rewritten
        };
        if (p.out_dtype == 1) {
#pragma unroll
          for (int f = 0; f < HC / 32; ++f) {
            acquire();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = acc(f * 32 + j * 8 + i);
              add_bias8(p, v, qbase + f * 32 + j * 8);
#pragma unroll
              for (int h = 0; h < 2; ++h)
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(row_base + (uint32_t)(((2 * j + h) ^ (lane & 7)) << 4)),
                             "f"(v[4 * h]), "f"(v[4 * h + 1]), "f"(v[4 * h + 2]), "f"(v[4 * h + 3])
                             : "memory");
            }
            flush(qbase + f * 32, 32);
          }
        } else {
          constexpr int FC = HC < 64 ? HC : 64;  // columns of a row segment
#pragma unroll
          for (int f = 0; f < HC / FC; ++f) {
            acquire();
#pragma unroll
            for (int j = 0; j < FC / 8; ++j) {
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = acc(f * FC + j * 8 + i);
              add_bias8(p, v, qbase + f * FC + j * 8);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_base + (uint32_t)((j ^ (lane & 7)) << 4)),
                           "r"(pack16(v[0], v[1], p.out_dtype)), "r"(pack16(v[2], v[3], p.out_dtype)),
                           "r"(pack16(v[4], v[5], p.out_dtype)), "r"(pack16(v[6], v[7], p.out_dtype))
                           : "memory");
            }
            flush(qbase + f * FC, FC);
          }
        }
      } else if (prow < p.P) {
#pragma unroll
        for (int j = 0; j < HC / 8; ++j) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = acc(j * 8 + i);
          add_bias8(p, v, qbase + j * 8);
          store_row8(p, v, prow, qbase + j * 8);
        }
      }
    }
    if (lane == 0) tma_store_wait_all<0>();  // images and C are complete before the CTA leaves
  }

  // ---------------------------------------------------------------------- teardown
  if (cluster_wait_due) cluster_wait();
  tc_fence_before();
  __syncthreads();
  if (CG == 2 || cluster_mode) {
    // a pair: no CTA leaves while its peer may still signal it; cluster split: every CTA's sums have arrived
    cluster_arrive();
    cluster_wait();
  }
  if constexpr (CG == 1) {
    if (cluster_mode && warp >= 4 && tile0 < p.num_tiles) {
      // This CTA finishes `own` columns: the S sources are added in rank order, so the result does not depend on timing.
      const int S = p.cluster_split, own = TILE_Q / S;
      const int et = threadIdx.x - 128, row = et & 127, part = et >> 7;
      int tp, tq;
      raster8(p, tile0, tp, tq);
      const int prow = tp * k8TileP + row;
      const float* recv = reinterpret_cast<const float*>(sm + L::kOutOff) + row;
      auto sum = [&](int c) {
        float x = 0.f;
        for (int src = 0; src < S; ++src) x += recv[(src * own + c) * k8TileP];
        return x;
      };
      const int q0 = tq * TILE_Q + rank * own;
      if (prow < p.P) {
        if (!p.swap_out && own >= 16) {
          for (int c = part * (own / 2); c < (part + 1) * (own / 2); c += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = sum(c + i);
            add_bias8(p, v, q0 + c);
            store_row8(p, v, prow, q0 + c);
          }
        } else {
          for (int c = part; c < own; c += 2) {
            if (q0 + c < p.Q) {
              float x = sum(c);
              if (p.bias != nullptr) x += load_as_float(p.bias, p.swap_out ? prow : q0 + c, p.bias_dtype);
              store_one(p.out, p.swap_out ? (long long)(q0 + c) * p.ldo + prow : (long long)prow * p.ldo + q0 + c, x, p.out_dtype);
            }
          }
        }
      }
    }
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc<CG>(tmem_base, kTmemCols);
  }
}

typedef void (*Kernel8Fn)(const Gemm8Params);

}  // namespace b200
