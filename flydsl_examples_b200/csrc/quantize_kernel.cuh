// Quantization to 8-bit floating point with one power-of-two scale per group of 128, for sm_100a.
//
//   s = 2^ceil(log2(amax / MAX))  (amax: largest finite magnitude of the group; MAX = 448 or 57344, both 1.75 * 2^n; s = 1 for
//   a group of zeros, never below 2^-126),  q = round_to_nearest_even(x / s)
//
// s is read off amax's exponent and mantissa (m * 2^e with 1 <= m < 2: s = 2^(e - n), doubled when m > 1.75), so x / s is an
// exact product with a power of two and the conversion's is the only rounding. NaN becomes NaN; an infinity becomes NaN in
// e4m3 and stays infinite in e5m2; neither touches its group's scale.
//
// Memory-bound: one pass. A block of 256 threads holds a 128 x 128 tile in registers (eight 16-byte loads of 16-bit values
// in flight per thread, four blocks per SM), so the groups along rows (16 lanes: four shuffles), along columns and whole
// blocks (one trip through shared memory) come from the same read, whichever of them are asked for. 16384 x 8192 bf16: rows
// 64 us (6.3 TB/s), rows and columns 89 us (6.1 TB/s), blocks 63 us; fp32 102, 129 and 102 us.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "ptx.cuh"

namespace b200 {

constexpr int kQuantThreads = 256;

struct QuantParams {
  const void* x;
  long long ldx;  // elements between rows of x (columns are contiguous)
  int rows, cols;
  uint8_t* q_row;  // groups along a row (and 128 x 128 blocks, in block mode)
  long long ldq_row;
  float* s_row;
  long long sr_row, sr_group;  // element strides of s_row: per row (per block of rows), per group
  uint8_t* q_col;              // groups along a column
  long long ldq_col;
  float* s_col;
  long long sc_group, sc_col;
  int packed;  // scales as exponent bytes in tiles for the tensor core, see store_packed; s_col of mode 4: with K along the rows
  float* colsum;  // optional: sums of the tile's columns, [tile row][cols_pitch]
  long long colsum_ld;
};

// Exponent bits of the scale of a group with largest magnitude `amax` (finite, >= 0), in place in an fp32 word; 2^n * 1.75 is
// the format's largest value.
__device__ __forceinline__ uint32_t scale_bits(float amax, int n) {
  const uint32_t bits = __float_as_uint(amax);
  if (bits == 0) return 127u << 23;
  int e = (int)(bits >> 23);
  uint32_t man = bits & 0x7fffffu;
  if (e == 0) return 1u << 23;  // an fp32 subnormal: the smallest scale
  e += (man > 0x600000u) - n;   // mantissa above 1.75
  return (uint32_t)(e < 1 ? 1 : e) << 23;
}
// 1 / s for a power of two s = 2^(b - 127), as fp32 bits; b is between 1 and 247, so the result is normal.
__device__ __forceinline__ float inverse_of_scale(uint32_t bits) { return __uint_as_float((254u << 23) - bits); }

// Four values to the format, to nearest even (beyond its range: its largest value; NaN: NaN), the first in the lowest byte.
template <bool E5M2>
__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
  uint32_t r;
  if constexpr (E5M2)
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e5m2x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e5m2x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
  else
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// Eight consecutive elements, and what the groups' maxima need: magnitudes compare like unsigned integers, so 16-bit values
// are compared two to an instruction as they are (`Mag` = two of them), fp32 values one by one.
template <typename T>
struct RawRow {
  static constexpr int kWords = sizeof(T) == 4 ? 8 : 4;
  uint32_t w[kWords];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    } else {
      const __half2 h = *reinterpret_cast<const __half2*>(&w[i >> 1]);
      return i & 1 ? __high2float(h) : __low2float(h);
    }
  }
};
template <typename T>
struct Mag {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr uint32_t kAbs = kWide ? 0x7fffffffu : 0x7fff7fffu;
  static constexpr uint32_t kInf = kWide ? 0x7f800000u : std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;  // and above: NaN
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    if constexpr (kWide) return max(a, b);
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  // an infinity of either sign to a NaN (both halves of a word)
  static __device__ __forceinline__ uint32_t no_inf(uint32_t w) {
    if constexpr (kWide) return (w & kAbs) == kInf ? w | 1u : w;
    return w | ((w & 0x7fffu) == kInf ? 1u : 0u) | ((w >> 16 & 0x7fffu) == kInf ? 0x10000u : 0u);
  }
  static __device__ __forceinline__ bool any_odd(uint32_t m) { return kWide ? m >= kInf : (m & 0xffffu) >= kInf || (m >> 16) >= kInf; }
  static __device__ __forceinline__ uint32_t only_finite(uint32_t m) {
    if constexpr (kWide) return m >= kInf ? 0u : m;
    return ((m & 0xffffu) >= kInf ? 0u : m & 0xffffu) | ((m >> 16) >= kInf ? 0u : m & 0xffff0000u);
  }
  // the magnitude in half h of the word, as fp32
  static __device__ __forceinline__ float value(uint32_t m, int h) {
    if constexpr (kWide) return __uint_as_float(m);
    const uint32_t b = h ? m >> 16 : m & 0xffffu;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(b << 16);
    return __half2float(__ushort_as_half((unsigned short)b));
  }
};

// The rows and columns at a ragged edge, or off 16-byte boundaries: element by element. Not inlined: the kernel's straight path is
// long as it is, and waits for instructions where it outgrows the cache.
template <typename T>
__device__ __noinline__ RawRow<T> load_row8_slow(const T* src, int n) {
  RawRow<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = i < n ? __float_as_uint(src[i]) : 0u;
  } else {
    const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.w[i] = (uint32_t)(2 * i < n ? s[2 * i] : 0) | ((uint32_t)(2 * i + 1 < n ? s[2 * i + 1] : 0) << 16);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ RawRow<T> load_row8(const T* src, int n, bool vec) {
  if (!(n >= 8 && vec)) return load_row8_slow(src, n);
  RawRow<T> r;
  const uint4 a = __ldcs(reinterpret_cast<const uint4*>(src));  // read once
  r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
  if constexpr (sizeof(T) == 4) {
    const uint4 b = __ldcs(reinterpret_cast<const uint4*>(src) + 1);
    r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
  }
  return r;
}
static __device__ __noinline__ void store_row8_slow(uint8_t* dst, uint32_t lo, uint32_t hi, int n) {
  const uint64_t v = (uint64_t(hi) << 32) | lo;
#pragma unroll 1
  for (int j = 0; j < min(n, 8); ++j) dst[j] = (uint8_t)(v >> (8 * j));
}

// Packed scales: 512 bytes for 128 rows of an operand and four K blocks, as the tensor core takes them; row r and block b are byte
// r % 32 * 16 + r / 32 * 4 + b % 4, the scale's exponent. `step`: tiles from four blocks to the next four.
__device__ __forceinline__ void store_packed(float* tiles, long long step, int row_tile, int block, int r, uint32_t bits) {
  reinterpret_cast<uint8_t*>(tiles)[((block >> 2) * step + row_tile) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (block & 3)] = (uint8_t)(bits >> 23);
}

// Which of a thread's eight columns have infinities of one sign and no NaN (bit j +inf, bit 8 + j -inf): those sums stay infinite although v gets
// NaN in their place.
template <typename T>
__device__ __forceinline__ uint32_t infinite_columns(const RawRow<T> (&v)[8]) {
  uint32_t up = 0, down = 0, nan = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = v[i].get(j);
      up |= (f == INFINITY ? 1u : 0u) << j, down |= (f == -INFINITY ? 1u : 0u) << j, nan |= (f != f ? 1u : 0u) << j;
    }
  nan |= up & down;
  return (up & ~nan) | (down & ~nan) << 8;
}

// MODE: 1 = groups along rows, 2 = along columns, 4 = 128 x 128 blocks (written through the row members).
template <typename T, int MODE, bool E5M2>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 4 ? 2 : 4) quantize_a8_kernel(const QuantParams p) {
  constexpr int kPasses = 8;  // rows per thread: ty, ty + 16, ...
  __shared__ float red[8][128];
  __shared__ float red2[8][128];
  __shared__ uint32_t infinite[MODE & 2 ? kQuantThreads : 1];  // of a thread that met an infinity or NaN (a register costs all: 1.7 %)
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, warp = threadIdx.x >> 5;
  const int tiles_c = (p.cols + 127) >> 7;
  const int tr = blockIdx.x / tiles_c, tc = blockIdx.x - tr * tiles_c;
  const int r0 = tr * 128, col = tc * 128 + tx * 8;
  const int ncol = min(8, p.cols - col);  // may be <= 0
  const int nrow = min(128, p.rows - r0);
  const T* x = reinterpret_cast<const T*>(p.x);
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ((p.ldx * (long long)sizeof(T)) & 15) == 0;
  constexpr int n = E5M2 ? 15 : 8;

  grid_dependency_wait();
  grid_launch_dependents();
  RawRow<T> v[kPasses];
  const T* src = x + (long long)(r0 + ty) * p.ldx + col;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const bool in = ty + 16 * i < nrow && ncol > 0;
    v[i] = load_row8<T>(in ? src : x, in ? ncol : 0, vec);
    src += 16 * p.ldx;
  }

  // Largest magnitudes per row (over the thread's eight columns) and per column (over its eight rows).
  using M = Mag<T>;
  constexpr int kW = RawRow<T>::kWords;
  uint32_t rmag[kPasses], cmag[kW];
  auto maxima = [&](auto finite) {
#pragma unroll
    for (int j = 0; j < kW; ++j) cmag[j] = 0;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      rmag[i] = 0;
#pragma unroll
      for (int j = 0; j < kW; ++j) {
        const uint32_t m = finite(v[i].w[j] & M::kAbs);
        if (MODE & 5) rmag[i] = M::max2(rmag[i], m);
        if (MODE & 2) cmag[j] = M::max2(cmag[j], m);
      }
    }
  };
  maxima([](uint32_t m) { return m; });
  uint32_t all = 0;
  if (MODE & 2) {
#pragma unroll
    for (int j = 0; j < kW; ++j) all = M::max2(all, cmag[j]);
  } else {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) all = M::max2(all, rmag[i]);
  }
  const bool odd = M::any_odd(all);  // an infinity or a NaN among them: it counts as zero
  if (odd) {
    maxima([](uint32_t m) { return M::only_finite(m); });
    if constexpr (!E5M2) {  // the conversion clamps infinities, e4m3 has none
      if (MODE & 2) infinite[threadIdx.x] = infinite_columns<T>(v);
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
#pragma unroll
        for (int j = 0; j < kW; ++j) v[i].w[j] = M::no_inf(v[i].w[j]);
    }
  }
  float rmax[kPasses], cmax[8];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) rmax[i] = M::kWide ? M::value(rmag[i], 0) : fmaxf(M::value(rmag[i], 0), M::value(rmag[i], 1));
#pragma unroll
  for (int j = 0; j < 8; ++j) cmax[j] = M::kWide ? M::value(cmag[j % kW], 0) : M::value(cmag[(j >> 1) % kW], j & 1);
  // Eight values of one row times their inverse scales, converted and stored.
  auto put = [&](uint8_t* dst, const RawRow<T>& raw, const float (&inv)[8], bool dvec) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = pack_fp8x4<E5M2>(raw.get(4 * h) * inv[4 * h], raw.get(4 * h + 1) * inv[4 * h + 1], raw.get(4 * h + 2) * inv[4 * h + 2],
                              raw.get(4 * h + 3) * inv[4 * h + 3]);
    if constexpr (E5M2) {
      if (odd) {  // the conversion clamps infinities to the largest value
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = __float_as_uint(raw.get(j));
          if ((b & 0x7fffffffu) == 0x7f800000u) {
            const uint32_t code = 0x7cu | ((b >> 24) & 0x80u);
            w[j >> 2] = (w[j >> 2] & ~(0xffu << (8 * (j & 3)))) | (code << (8 * (j & 3)));
          }
        }
      }
    }
    if (dvec && ncol >= 8)
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else
      store_row8_slow(dst, w[0], w[1], ncol);
  };
  const bool rvec = (reinterpret_cast<uintptr_t>(p.q_row) & 7) == 0 && (p.ldq_row & 7) == 0;
  const bool cvec = (reinterpret_cast<uintptr_t>(p.q_col) & 7) == 0 && (p.ldq_col & 7) == 0;

  if constexpr (MODE & 1) {
    // Eight rows over 16 lanes: each exchange halves the rows a lane answers for, so that eight shuffles (instead of 32) leave
    // lane tx with the maximum of row ty + 16 * (tx / 2, its three bits) and one scale to work out.
#pragma unroll
    for (int h = 4; h > 0; h >>= 1) {
      const bool up = tx & (2 * h);
#pragma unroll
      for (int j = 0; j < h; ++j) {
        const float mine = up ? rmax[j + h] : rmax[j], other = up ? rmax[j] : rmax[j + h];
        rmax[j] = fmaxf(mine, __shfl_xor_sync(0xffffffffu, other, 2 * h));
      }
    }
    const uint32_t sb = scale_bits(fmaxf(rmax[0], __shfl_xor_sync(0xffffffffu, rmax[0], 1)), n);
    const int own = ty + 16 * (tx >> 1);
    if ((tx & 1) == 0 && own < nrow) {
      if (p.packed)
        store_packed(p.s_row, p.sr_group, tr, tc, own, sb);
      else
        p.s_row[(long long)(r0 + own) * p.sr_row + (long long)tc * p.sr_group] = __uint_as_float(sb);
    }
    const float own_inv = inverse_of_scale(sb);
    uint8_t* dst = p.q_row + (long long)(r0 + ty) * p.ldq_row + col;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const float s = __shfl_sync(0xffffffffu, own_inv, 2 * i, 16);
      const float inv[8] = {s, s, s, s, s, s, s, s};
      if (ty + 16 * i < nrow && ncol > 0) put(dst, v[i], inv, rvec);
      dst += 16 * p.ldq_row;
    }
  }
  if constexpr (MODE & 2) {
    float csum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      cmax[j] = fmaxf(cmax[j], __shfl_xor_sync(0xffffffffu, cmax[j], 16));
      csum[j] = 0.f;
    }
    if (p.colsum != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < kPasses; ++i) csum[j] += v[i].get(j);
      if (!E5M2 && odd) {
        const uint32_t bits = infinite[threadIdx.x];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (bits >> j & 0x101u) csum[j] = __uint_as_float(bits >> j & 1u ? 0x7f800000u : 0xff800000u);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) csum[j] += __shfl_xor_sync(0xffffffffu, csum[j], 16);
    }
    if ((threadIdx.x & 16) == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        red[warp][tx * 8 + j] = cmax[j];
        if (p.colsum != nullptr) red2[warp][tx * 8 + j] = csum[j];
      }
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      float m = 0.f, t = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w][threadIdx.x]);
      const uint32_t sb = scale_bits(m, n);
      const int c = tc * 128 + threadIdx.x;
      if (c < p.cols) {
        if (p.packed)
          store_packed(p.s_col, p.sc_group, tc, tr, threadIdx.x, sb);
        else
          p.s_col[(long long)tr * p.sc_group + (long long)c * p.sc_col] = __uint_as_float(sb);
        if (p.colsum != nullptr) {
#pragma unroll
          for (int w = 0; w < 8; ++w) t += red2[w][threadIdx.x];
          p.colsum[(long long)tr * p.colsum_ld + c] = t;
        }
      }
      red[0][threadIdx.x] = inverse_of_scale(sb);
    }
    __syncthreads();
    if (ncol > 0) {
      float inv[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) inv[j] = red[0][tx * 8 + j];
      uint8_t* dst = p.q_col + (long long)(r0 + ty) * p.ldq_col + col;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        if (ty + 16 * i < nrow) put(dst, v[i], inv, cvec);
        dst += 16 * p.ldq_col;
      }
    }
  }
  if constexpr (MODE & 4) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) m = fmaxf(m, rmax[i]);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) red[0][warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = fmaxf(m, red[0][w]);
    const uint32_t sb = scale_bits(m, n);
    if (p.packed) {
      const int i = threadIdx.x & 127;
      if (threadIdx.x < 128 && i < nrow) store_packed(p.s_row, p.sr_group, tr, tc, i, sb);
      if (threadIdx.x >= 128 && p.s_col != nullptr && tc * 128 + i < p.cols) store_packed(p.s_col, p.sc_group, tc, tr, i, sb);
    } else if (threadIdx.x == 0) {
      p.s_row[(long long)tr * p.sr_row + (long long)tc * p.sr_group] = __uint_as_float(sb);
    }
    const float s = inverse_of_scale(sb);
    const float inv[8] = {s, s, s, s, s, s, s, s};
    if (ncol > 0) {
      uint8_t* dst = p.q_row + (long long)(r0 + ty) * p.ldq_row + col;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        if (ty + 16 * i < nrow) put(dst, v[i], inv, rvec);
        dst += 16 * p.ldq_row;
      }
    }
  }
}

}  // namespace b200
