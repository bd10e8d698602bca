// Host side of the 8-bit block-scaled GEMM and its quantizer: validation, plan, tensor maps, launch. Exports the
// b200_gemm_a8w8_* and b200_gemm_quantize_a8 entry points of include/b200_gemm.h. No device allocation, no synchronisation.
#include <cstring>
#include <initializer_list>

#include "../../include/b200_gemm.h"
#include "gemm_a8w8_variants.h"
#include "host.h"
#include "quantize_kernel.cuh"

namespace b200 {

struct Call8 {
  Gemm8Params params;
  Variant8 var;
  int grid, cluster, pdl;
};

static bool is_fp8(int dt) { return dt == B200_GEMM_DTYPE_E4M3 || dt == B200_GEMM_DTYPE_E5M2; }

// Everything that needs no device; also what b200_gemm_a8w8_plan_query answers.
static int resolve8(const b200_gemm_a8w8_args* a, int sms, b200_gemm_plan* out, Variant8* var) {
  if (a == nullptr || a->m <= 0 || a->n <= 0 || a->k <= 0) return B200_GEMM_ERR_BAD_ARG;
  if (a->m > 0x7fffff00LL || a->n > 0x7fffff00LL || a->k > 0x7fffff00LL) return B200_GEMM_ERR_TOO_LARGE;
  if (!is_fp8(a->a_dtype) || !is_fp8(a->b_dtype)) return B200_GEMM_ERR_BAD_ARG;
  if (a->out_dtype < 1 || a->out_dtype > 3) return B200_GEMM_ERR_BAD_ARG;
  if (a->lda < (a->a_trans ? a->m : a->k) || a->ldb < (a->b_trans ? a->k : a->n) || a->ldo < a->n) return B200_GEMM_ERR_BAD_ARG;
  // exponent tiles: for both operands or for neither
  if (a->a_block < 0 || a->a_block > 2 || a->b_block < 0 || a->b_block > 2 || (a->a_block == 2) != (a->b_block == 2)) return B200_GEMM_ERR_BAD_ARG;
  const int packed = a->a_block == 2;
  const b200_gemm_policy& pol = a->policy;
  // this kernel has one ring depth and one K depth per tile, and no stream-K, ticket, atomic or loader-warp mode
  if (pol.stages != 0 || pol.stream_k != 0 || pol.tile_k != 0 || pol.loader != 0) return B200_GEMM_ERR_BAD_POLICY;
  b200_gemm_plan pl;
  memset(&pl, 0, sizeof(pl));
  pl.cta_group = pol.cta_group == 0 ? 1 : pol.cta_group;
  pl.swap_ab = pol.swap_ab ? 1 : 0;
  pl.tile_n = pol.tile_n;
  pl.tile_k = k8TK;
  const int v_vector = (pl.swap_ab ? a->a_block : a->b_block) ? 0 : 1;
  if (packed && (pl.swap_ab || pol.split_k > 1)) return B200_GEMM_ERR_BAD_POLICY;
  if (!variant8(pl.tile_n, pl.cta_group, v_vector, packed, var)) return B200_GEMM_ERR_BAD_POLICY;
  pl.tile_m = k8TileP * pl.cta_group;
  pl.stages = var->stages;
  pl.smem_bytes = var->smem_bytes;
  // a row-contiguous operand arrives in boxes of 128 rows: each CTA's share of the tile has to be one
  const int v_mn = pl.swap_ab ? (a->a_trans ? 1 : 0) : (a->b_trans ? 0 : 1);
  if (v_mn && pl.tile_n / pl.cta_group != 128) return B200_GEMM_ERR_BAD_POLICY;
  const int64_t P = pl.swap_ab ? a->n : a->m, Q = pl.swap_ab ? a->m : a->n;
  pl.tiles_p = (int)((P + pl.tile_m - 1) / pl.tile_m);
  pl.tiles_q = (int)((Q + pl.tile_n - 1) / pl.tile_n);
  // all tile rows are one group at most: the kernel multiplies by tiles_q in 32 bits
  pl.group_m = pol.group_m < 0 ? 0 : pol.group_m < pl.tiles_p ? pol.group_m : pl.tiles_p;
  const int64_t tiles = (int64_t)pl.tiles_p * pl.tiles_q;
  const int kb_total = (int)((a->k + k8TK - 1) / k8TK);
  int s = 1;
  if (pol.split_k > 1) {  // the K blocks of a tile over the CTAs of a cluster: a power of two, no slice empty, a column each
    if (pl.cta_group != 1) return B200_GEMM_ERR_BAD_POLICY;
    s = 16;
    while (s > pol.split_k || s > kb_total || s > pl.tile_n) s >>= 1;
  }
  pl.split_k = s;
  pl.cluster_split = s > 1 ? s : 0;
  if (tiles * s > 0x3fffffffLL) return B200_GEMM_ERR_TOO_LARGE;
  pl.num_units = (int)(tiles * s);
  int cap = (pol.max_ctas > 0 ? pol.max_ctas : sms) / pl.cta_group;
  if (cap < 1) cap = 1;
  pl.grid = s > 1 ? pl.num_units : (int)(tiles < cap ? tiles : cap) * pl.cta_group;
  pl.tmem_cols = packed || pl.tile_n > 128 ? 512 : pl.tile_n * 4;
  *out = pl;
  return 0;
}

static int encode8(CUtensorMap* map, const void* ptr, int mn_major, int64_t rows, int64_t k, int64_t ld, int box_rows) {
  EncodeTiledFn enc = get_encode_fn();
  if (enc == nullptr) return B200_GEMM_ERR_DRIVER;
  // K-contiguous: dims {K, rows}, box {128, rows of a tile}; row-contiguous: dims {rows, K}, box {128, 128}
  cuuint64_t dims[2] = {(cuuint64_t)(mn_major ? rows : k), (cuuint64_t)(mn_major ? k : rows)};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {128, (cuuint32_t)(mn_major ? k8TK : box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult res = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return res == CUDA_SUCCESS ? 0 : B200_GEMM_ERR_TENSOR_MAP;
}

constexpr int64_t kMaxTiles = 0x0fffffff;  // 32-bit coordinates, with room for the tiles that a CTA asks for past the last row

// The exponent tiles of an operand, 512 bytes each, as rows of 128 bytes.
static int encode_tiles(CUtensorMap* map, const void* ptr, int64_t row_tiles, int64_t k_groups, int64_t s_row, int64_t s_kb) {
  EncodeTiledFn enc = get_encode_fn();
  if (enc == nullptr) return B200_GEMM_ERR_DRIVER;
  const int64_t tiles = (row_tiles - 1) * s_row + (k_groups - 1) * s_kb + 1;
  if (tiles > kMaxTiles) return B200_GEMM_ERR_TOO_LARGE;
  cuuint64_t dims[2] = {128, (cuuint64_t)(4 * tiles)};
  cuuint64_t strides[1] = {128};
  cuuint32_t box[2] = {128, 4};
  cuuint32_t estr[2] = {1, 1};
  const CUresult res = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return res == CUDA_SUCCESS ? 0 : B200_GEMM_ERR_TENSOR_MAP;
}

// Shared-memory descriptor without the start address (fields as for the 16-bit kernel): K-contiguous rows are 128 bytes
// apart, groups of eight 1024 bytes, a K = 32 step is 32 bytes; a row-contiguous box is [128 K rows x 128 bytes], groups of
// eight K rows 1024 bytes apart, a K = 32 step is 4096 bytes.
static void make_desc8(int mn_major, uint32_t* hi, uint32_t* lo, uint32_t* kstep) {
  *lo = (mn_major ? (16384u >> 4) : 1u) << 16;
  *hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  *kstep = mn_major ? (4096 >> 4) : (32 >> 4);
}

static int prepare8(const b200_gemm_a8w8_args* a, Call8* h) {
  int dev = 0, sms = 0;
  b200_gemm_plan pl;
  Variant8 var;
  int rc = resolve8(a, 148, &pl, &var);  // refusals first: they need no device
  if (rc) return rc;
  if (a->a == nullptr || a->b == nullptr || a->out == nullptr || a->a_scale == nullptr || a->b_scale == nullptr)
    return B200_GEMM_ERR_BAD_ARG;
  const int es = a->out_dtype == B200_GEMM_DTYPE_FP32 ? 4 : 2;
  auto aligned = [](const void* ptr, int64_t to) { return (reinterpret_cast<uintptr_t>(ptr) % (uintptr_t)to) == 0; };
  if (!aligned(a->a, 16) || !aligned(a->b, 16) || a->lda % 16 != 0 || a->ldb % 16 != 0) return B200_GEMM_ERR_BAD_ARG;
  const int packed = a->a_block == 2;
  if (packed)
    for (const int64_t s : {a->sa_row, a->sa_kb, a->sb_col, a->sb_kb}) {
      if (s < 0) return B200_GEMM_ERR_BAD_ARG;
      if (s > kMaxTiles) return B200_GEMM_ERR_TOO_LARGE;
    }
  if (!aligned(a->a_scale, packed ? 16 : 4) || !aligned(a->b_scale, packed ? 16 : 4) || !aligned(a->out, es)) return B200_GEMM_ERR_BAD_ARG;
  if (a->bias != nullptr && (a->bias_dtype < 1 || a->bias_dtype > 3 || !aligned(a->bias, a->bias_dtype == 1 ? 4 : 2)))
    return B200_GEMM_ERR_BAD_ARG;
  rc = current_sms(&dev, &sms);
  if (rc) return rc;
  ensure_context();
  rc = resolve8(a, sms, &pl, &var);
  if (rc) return rc;

  memset(h, 0, sizeof(*h));
  Gemm8Params& p = h->params;
  const int a_mn = a->a_trans ? 1 : 0, b_mn = a->b_trans ? 0 : 1;
  const bool sw = pl.swap_ab != 0;
  p.P = (int)(sw ? a->n : a->m), p.Q = (int)(sw ? a->m : a->n);
  p.u_mn_major = sw ? b_mn : a_mn, p.v_mn_major = sw ? a_mn : b_mn;
  rc = encode8(&p.tmap_u, sw ? a->b : a->a, p.u_mn_major, p.P, a->k, sw ? a->ldb : a->lda, k8TileP);
  if (rc) return rc;
  rc = encode8(&p.tmap_v, sw ? a->a : a->b, p.v_mn_major, p.Q, a->k, sw ? a->lda : a->ldb, pl.tile_n / pl.cta_group);
  if (rc) return rc;
  if (packed) {
    const int64_t kb = (a->k + 4 * k8TK - 1) / (4 * k8TK);
    rc = encode_tiles(&p.tmap_us, a->a_scale, (a->m + 127) / 128, kb, a->sa_row, a->sa_kb);
    if (!rc) rc = encode_tiles(&p.tmap_vs, a->b_scale, (a->n + 127) / 128, kb, a->sb_col, a->sb_kb);
    if (rc) return rc;
  }
  p.u_scale = sw ? a->b_scale : a->a_scale, p.v_scale = sw ? a->a_scale : a->b_scale;
  p.us_row = sw ? a->sb_col : a->sa_row, p.us_kb = sw ? a->sb_kb : a->sa_kb;
  p.vs_row = sw ? a->sa_row : a->sb_col, p.vs_kb = sw ? a->sa_kb : a->sb_kb;
  p.us_shift = (sw ? a->b_block : a->a_block) ? 7 : 0;
  p.vs_shift = (sw ? a->a_block : a->b_block) ? 7 : 0;
  p.out = a->out, p.bias = a->bias, p.status = a->status;
  p.ldo = a->ldo;
  p.tiles_p = pl.tiles_p, p.tiles_q = pl.tiles_q, p.num_tiles = pl.tiles_p * pl.tiles_q;
  p.kb_total = (int)((a->k + k8TK - 1) / k8TK);
  p.cluster_split = pl.cluster_split;
  p.group_p = pl.group_m;
  p.swap_out = pl.swap_ab;
  p.out_dtype = a->out_dtype, p.bias_dtype = a->bias_dtype;
  if (!sw && pl.tile_n >= 128 && !pl.cluster_split && aligned(a->out, 16) && (a->ldo * es) % 16 == 0) {
    EncodeTiledFn enc = get_encode_fn();
    const CUtensorMapDataType dt = a->out_dtype == B200_GEMM_DTYPE_FP32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : a->out_dtype == B200_GEMM_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    cuuint64_t dims[2] = {(cuuint64_t)a->n, (cuuint64_t)a->m};
    cuuint64_t strides[1] = {(cuuint64_t)(a->ldo * es)};
    cuuint32_t box[2] = {(cuuint32_t)(128 / es), 32};
    cuuint32_t estr[2] = {1, 1};
    if (enc(&p.tmap_out, dt, 2, a->out, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS)
      p.tma_store = 1;
  }
  const uint32_t u_fmt = (sw ? a->b_dtype : a->a_dtype) == B200_GEMM_DTYPE_E5M2 ? 1u : 0u;
  const uint32_t v_fmt = (sw ? a->a_dtype : a->b_dtype) == B200_GEMM_DTYPE_E5M2 ? 1u : 0u;
  // instruction descriptor: fp32 accumulator, the operands' 8-bit formats, their major-ness, N / 8, M / 16
  p.idesc = (1u << 4) | (u_fmt << 7) | (v_fmt << 10) | (uint32_t(p.u_mn_major) << 15) | (uint32_t(p.v_mn_major) << 16) |
            (uint32_t(pl.tile_n >> 3) << 17) | (uint32_t(pl.tile_m >> 4) << 24);
  // with scales the accumulator is always fp32; bits 4-5 and 29-30 name B's and A's exponent byte, bit 23 the scales' type
  if (packed) p.idesc = (p.idesc & ~(3u << 4)) | (1u << 23);
  make_desc8(p.u_mn_major, &p.u_desc_hi, &p.u_desc_lo, &p.u_kstep);
  make_desc8(p.v_mn_major, &p.v_desc_hi, &p.v_desc_lo, &p.v_kstep);
  p.wait_limit_ns = a->policy.wait_limit_us > 0 ? (unsigned long long)a->policy.wait_limit_us * 1000ull : kWaitLimitNs;

  h->var = var;
  h->grid = pl.grid;
  h->cluster = pl.cta_group == 2 ? 2 : pl.cluster_split;
  h->pdl = a->policy.no_pdl ? 0 : 1;
  return allow_launch(reinterpret_cast<const void*>(var.fn), var.smem_bytes, dev);
}

static int run8(const Call8* h, cudaStream_t stream) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(h->grid, 1, 1);
  cfg.blockDim = dim3(k8Threads, 1, 1);
  cfg.dynamicSmemBytes = h->var.smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (h->cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = h->cluster, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (h->pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = n ? attr : nullptr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, h->var.fn, h->params);
  return e == cudaSuccess ? 0 : set_cuda_error(e);
}

template <typename T, bool E5M2>
static void* quant_fn(int mode) {
  switch (mode) {
    case 1: return reinterpret_cast<void*>(quantize_a8_kernel<T, 1, E5M2>);
    case 2: return reinterpret_cast<void*>(quantize_a8_kernel<T, 2, E5M2>);
    case 3: return reinterpret_cast<void*>(quantize_a8_kernel<T, 3, E5M2>);
    default: return reinterpret_cast<void*>(quantize_a8_kernel<T, 4, E5M2>);
  }
}
template <typename T>
static void* quant_fn(int mode, bool e5m2) {
  return e5m2 ? quant_fn<T, true>(mode) : quant_fn<T, false>(mode);
}

}  // namespace b200

extern "C" {

int b200_gemm_a8w8_plan_query(const b200_gemm_a8w8_args* args, b200_gemm_plan* plan) {
  if (plan == nullptr) return B200_GEMM_ERR_BAD_ARG;
  int dev = 0, sms = 0;
  if (b200::current_sms(&dev, &sms) != 0) sms = 148;
  b200::Variant8 var;
  return b200::resolve8(args, sms, plan, &var);
}

int b200_gemm_a8w8(const b200_gemm_a8w8_args* args, void* cuda_stream) {
  b200::Call8 h;
  const int rc = b200::prepare8(args, &h);
  return rc ? rc : b200::run8(&h, reinterpret_cast<cudaStream_t>(cuda_stream));
}

int b200_gemm_quantize_a8(const b200_gemm_quantize_args* a, void* cuda_stream) {
  if (a == nullptr || a->rows < 0 || a->cols < 0) return B200_GEMM_ERR_BAD_ARG;
  if (a->in_dtype < 1 || a->in_dtype > 3 || !b200::is_fp8(a->out_dtype)) return B200_GEMM_ERR_BAD_ARG;
  if (a->mode < 1 || a->mode > 4 || a->packed < 0 || a->packed > 1) return B200_GEMM_ERR_BAD_ARG;
  if (a->rows == 0 || a->cols == 0) return 0;
  if (a->rows > 0x7fffff00LL || a->cols > 0x7fffff00LL) return B200_GEMM_ERR_TOO_LARGE;
  const bool row = a->mode != 2, col = a->mode == 2 || a->mode == 3;
  const int es = a->in_dtype == B200_GEMM_DTYPE_FP32 ? 4 : 2;
  if (a->x == nullptr || a->ldx < a->cols || reinterpret_cast<uintptr_t>(a->x) % es != 0) return B200_GEMM_ERR_BAD_ARG;
  if (row && (a->q_row == nullptr || a->s_row == nullptr || a->ldq_row < a->cols)) return B200_GEMM_ERR_BAD_ARG;
  if (col && (a->q_col == nullptr || a->s_col == nullptr || a->ldq_col < a->cols)) return B200_GEMM_ERR_BAD_ARG;
  if (a->colsum != nullptr && (!col || a->colsum_ld < a->cols)) return B200_GEMM_ERR_BAD_ARG;
  auto off = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 4 != 0; };
  if (!a->packed && ((row && off(a->s_row)) || (col && off(a->s_col)))) return B200_GEMM_ERR_BAD_ARG;
  if (off(a->colsum)) return B200_GEMM_ERR_BAD_ARG;
  const int64_t tiles = ((a->rows + 127) / 128) * ((a->cols + 127) / 128);
  if (tiles > 0x7fffffffLL) return B200_GEMM_ERR_TOO_LARGE;
  b200::QuantParams p;
  memset(&p, 0, sizeof(p));
  p.x = a->x, p.ldx = a->ldx, p.rows = (int)a->rows, p.cols = (int)a->cols;
  p.q_row = static_cast<uint8_t*>(a->q_row), p.ldq_row = a->ldq_row, p.s_row = a->s_row, p.sr_row = a->sr_row, p.sr_group = a->sr_group;
  p.q_col = static_cast<uint8_t*>(a->q_col), p.ldq_col = a->ldq_col, p.s_col = a->s_col, p.sc_group = a->sc_group, p.sc_col = a->sc_col;
  p.colsum = a->colsum, p.colsum_ld = a->colsum_ld;
  p.packed = a->packed;
  const bool e5m2 = a->out_dtype == B200_GEMM_DTYPE_E5M2;
  void* fn = a->in_dtype == B200_GEMM_DTYPE_FP32   ? b200::quant_fn<float>(a->mode, e5m2)
             : a->in_dtype == B200_GEMM_DTYPE_BF16 ? b200::quant_fn<__nv_bfloat16>(a->mode, e5m2)
                                                    : b200::quant_fn<__half>(a->mode, e5m2);
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)tiles, 1, 1);
  cfg.blockDim = dim3(b200::kQuantThreads, 1, 1);
  cfg.stream = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  void* kargs[1] = {&p};
  const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, kargs);
  return e == cudaSuccess ? 0 : b200::set_cuda_error(e);
}

int b200_gemm_sequence(const void* records, void* cuda_stream) {
  const char* r = static_cast<const char*>(records);
  if (r == nullptr || reinterpret_cast<uintptr_t>(r) % 8 != 0) return B200_GEMM_ERR_BAD_ARG;
  for (;;) {
    const int64_t kind = *reinterpret_cast<const int64_t*>(r);
    r += 8;
    int rc = B200_GEMM_ERR_BAD_ARG;
    if (kind == 0) return 0;
    if (kind == 1) {
      rc = b200_gemm_a8w8(reinterpret_cast<const b200_gemm_a8w8_args*>(r), cuda_stream);
      r += sizeof(b200_gemm_a8w8_args);
    } else if (kind == 2) {
      rc = b200_gemm_quantize_a8(reinterpret_cast<const b200_gemm_quantize_args*>(r), cuda_stream);
      r += sizeof(b200_gemm_quantize_args);
    } else if (kind == 3) {
      const b200_gemm_reduce_args* a = reinterpret_cast<const b200_gemm_reduce_args*>(r);
      rc = b200_gemm_reduce_slots(a->slots, a->slot_stride, a->n_slots, a->out, a->bias, a->rows, a->cols, a->out_dtype, a->bias_dtype, cuda_stream);
      r += sizeof(b200_gemm_reduce_args);
    }
    if (rc) return rc;
  }
}

}  // extern "C"
