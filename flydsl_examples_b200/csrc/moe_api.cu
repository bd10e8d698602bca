// Host side of the few-token mixture-of-experts layer (b200_gemm_moe_* in include/b200_gemm.h): validation, tensor maps, the two
// launches. No device allocation, no synchronisation.
#include <cstring>
#include <mutex>

#include "../../include/b200_gemm.h"
#include "host.h"
#include "moe_kernels.cuh"

namespace b200 {

// Ring depths: as many stages (128 deep, the widest second kernel's 64) as fit 227 KB next to the exchange area.
struct MoeVariant {
  MoeFn up, down;
  int up_smem, down_smem, cols, down_k;
};
template <int TN, int UP_STAGES, int DOWN_STAGES, int DOWN_SUBS>
static MoeVariant moe_make() {
  using Up = SmemMoe<TN, UP_STAGES, 2, true>;
  using Down = SmemMoe<TN, DOWN_STAGES, DOWN_SUBS, false>;
  static_assert(Up::kDynBytes <= 227 * 1024 && Down::kDynBytes <= 227 * 1024, "shared memory");
  return {moe_a16w16_sm100_kernel<TN, UP_STAGES, 2, true>, moe_a16w16_sm100_kernel<TN, DOWN_STAGES, DOWN_SUBS, false>, Up::kDynBytes,
          Down::kDynBytes, TN, 64 * DOWN_SUBS};
}
static MoeVariant moe_variant(int64_t t) {
  return t <= 16 ? moe_make<16, 5, 5, 2>() : t <= 32 ? moe_make<32, 5, 4, 2>() : moe_make<64, 4, 5, 1>();
}

constexpr uint64_t kMoeListBytes = 4096;  // the list of chosen experts at the start of the scratch

static int moe_check(const b200_gemm_moe_args* a) {
  if (a == nullptr || a->tokens <= 0 || a->hidden <= 0 || a->inner <= 0 || a->experts <= 0) return B200_GEMM_ERR_BAD_ARG;
  if (a->tokens > kMoeMaxTokens || a->experts > kMoeMaxExperts || a->hidden > (1 << 24) || a->inner > (1 << 24)) return B200_GEMM_ERR_TOO_LARGE;
  if (a->top_k < 1 || a->top_k > kMoeMaxTopK || a->top_k > a->experts) return B200_GEMM_ERR_BAD_ARG;
  if (a->dtype != B200_GEMM_DTYPE_BF16 && a->dtype != B200_GEMM_DTYPE_FP16) return B200_GEMM_ERR_BAD_ARG;
  if (a->logits_dtype < 1 || a->logits_dtype > 3) return B200_GEMM_ERR_BAD_ARG;
  // TMA describes all operands: rows of whole 16-byte pieces
  if (a->hidden % 8 != 0 || a->inner % 8 != 0) return B200_GEMM_ERR_BAD_ARG;
  if (a->ldx < a->hidden || a->w13_row < a->hidden || a->w2_row < a->inner || a->ldo < a->hidden) return B200_GEMM_ERR_BAD_ARG;
  if (a->ldx % 8 != 0 || a->w13_row % 8 != 0 || a->w13_expert % 8 != 0 || a->w2_row % 8 != 0 || a->w2_expert % 8 != 0) return B200_GEMM_ERR_BAD_ARG;
  if (a->experts > 1 && (a->w13_expert < 2 * a->inner * a->w13_row - (a->w13_row - a->hidden) ||
                         a->w2_expert < a->hidden * a->w2_row - (a->w2_row - a->inner)))
    return B200_GEMM_ERR_BAD_ARG;
  return 0;
}

static int64_t moe_slots(const b200_gemm_moe_args* a) {
  const int64_t pairs = a->tokens * a->top_k;
  return pairs < a->experts ? pairs : a->experts;
}

static int encode3(CUtensorMap* map, int dtype, const void* ptr, int64_t d0, int64_t d1, int64_t d2, int64_t s1, int64_t s2, int box1) {
  EncodeTiledFn enc = get_encode_fn();
  if (enc == nullptr) return B200_GEMM_ERR_DRIVER;
  cuuint64_t dims[3] = {(cuuint64_t)d0, (cuuint64_t)d1, (cuuint64_t)d2};
  cuuint64_t strides[2] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box1, 1}, estr[3] = {1, 1, 1};
  const CUresult res = enc(map, dtype == B200_GEMM_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           d2 > 0 ? 3 : 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return res == CUDA_SUCCESS ? 0 : B200_GEMM_ERR_TENSOR_MAP;
}

struct MoeCall {
  MoeParams up, down;
  MoeVariant var;
  int grid_up, grid_down, pdl;
};

// Clusters of `size` CTAs of the second kernel that the device holds at once; asked once for each kernel and size.
static int max_clusters(const MoeVariant& var, int size, int dev) {
  static std::mutex mutex;
  static int known[kMaxDevices][3][17];  // 0: not asked yet
  int& n = known[dev][var.cols == 16 ? 0 : var.cols == 32 ? 1 : 2][size];
  std::lock_guard<std::mutex> lock(mutex);
  if (n == 0) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(size, 1, 1), cfg.blockDim = dim3(kMoeThreads, 1, 1), cfg.dynamicSmemBytes = var.down_smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = size, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, reinterpret_cast<const void*>(var.down), &cfg) != cudaSuccess) {
      cudaGetLastError();  // not a launch error: this size is not used
      got = 0;
    }
    n = got > 0 ? got : -1;
  }
  return n;
}

static int moe_prepare(const b200_gemm_moe_args* a, MoeCall* h) {
  int rc = moe_check(a);
  if (rc) return rc;
  if (a->x == nullptr || a->logits == nullptr || a->w13 == nullptr || a->w2 == nullptr || a->out == nullptr) return B200_GEMM_ERR_BAD_ARG;
  auto off = [](const void* ptr, uintptr_t to) { return (reinterpret_cast<uintptr_t>(ptr) % to) != 0; };
  if (off(a->x, 16) || off(a->w13, 16) || off(a->w2, 16) || off(a->out, 2) || off(a->logits, a->logits_dtype == 1 ? 4 : 2))
    return B200_GEMM_ERR_BAD_ARG;
  if (a->workspace == nullptr || off(a->workspace, 256) || a->workspace_bytes < b200_gemm_moe_workspace_bytes(a)) return B200_GEMM_ERR_WORKSPACE;
  int dev = 0, sms = 0;
  rc = current_sms(&dev, &sms);
  if (rc) return rc;
  ensure_context();

  memset(h, 0, sizeof(*h));
  h->var = moe_variant(a->tokens);
  const int cols = h->var.cols;
  MoeParams& u = h->up;
  u.logits = a->logits, u.logits_row = a->logits_row, u.logits_col = a->logits_col, u.logits_dtype = a->logits_dtype;
  u.T = (int)a->tokens, u.E = (int)a->experts, u.H = (int)a->hidden, u.I = (int)a->inner, u.top_k = a->top_k, u.renorm = a->renormalize ? 1 : 0;
  u.dtype = a->dtype;
  u.list = static_cast<int*>(a->workspace);
  u.h = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(a->workspace) + kMoeListBytes);
  const bool fp16 = a->dtype == B200_GEMM_DTYPE_FP16;
  u.value_scale = fp16 ? kMoeValueScale : 1.f, u.value_back = 1.f / u.value_scale, u.rest_back = fp16 ? 1.f / kMoeRestScale : 1.f;
  u.out = a->out, u.ldo = a->ldo;
  u.status = a->status;
  u.wait_limit_ns = a->wait_limit_us > 0 ? (unsigned long long)a->wait_limit_us * 1000ull : kWaitLimitNs;
  const uint32_t fmt = a->dtype == B200_GEMM_DTYPE_BF16 ? 1u : 0u;
  u.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (uint32_t(cols >> 3) << 17) | (uint32_t(128 >> 4) << 24);  // N = the tokens' rows
  u.desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  h->down = u;
  h->down.idesc = (u.idesc & ~(0x3fu << 17)) | (uint32_t(2 * cols >> 3) << 17);
  const int64_t slots = moe_slots(a);
  const int64_t one13 = a->experts > 1 ? a->w13_expert : 2 * a->inner * a->w13_row, one2 = a->experts > 1 ? a->w2_expert : a->hidden * a->w2_row;
  rc = encode3(&h->up.tmap_u, a->dtype, a->w13, a->hidden, 2 * a->inner, a->experts, a->w13_row, one13, 64);
  if (!rc) rc = encode3(&h->up.tmap_v, a->dtype, a->x, a->hidden, a->tokens, 0, a->ldx, 0, cols);
  if (!rc) rc = encode3(&h->down.tmap_u, a->dtype, a->w2, a->inner, a->hidden, a->experts, a->w2_row, one2, 128);
  if (!rc) rc = encode3(&h->down.tmap_v, a->dtype, u.h, a->inner, a->tokens, 2 * slots, a->inner, a->tokens * a->inner, cols);
  if (rc) return rc;

  const int64_t units = slots * ((a->inner + 63) / 64);
  h->grid_up = (int)(units < sms ? units : sms);
  rc = allow_launch(reinterpret_cast<const void*>(h->var.up), h->var.up_smem, dev);
  if (!rc) rc = allow_launch(reinterpret_cast<const void*>(h->var.down), h->var.down_smem, dev);
  if (rc) return rc;
  // The down product's K axis goes over the CTAs of clusters, as large as still fit the GPU all at once (how many do depends
  // on how its SMs are grouped: 16 clusters of 8 have been seen to take two turns); no CTA without a K block or a token's
  // column to finish.
  const int row_tiles = (int)((a->hidden + 127) / 128);
  const int64_t blocks = slots * ((a->inner + h->var.down_k - 1) / h->var.down_k);
  int s = 16;
  if (s > blocks) s = (int)blocks;
  while (s > 1 && (row_tiles * s > sms || max_clusters(h->var, s, dev) < row_tiles)) --s;
  h->down.cluster_split = s;
  h->grid_down = row_tiles * s;
  h->pdl = a->no_pdl ? 0 : 1;
  return 0;
}

static int moe_run(const MoeCall* h, cudaStream_t stream) {
  for (int second = 0; second < 2; ++second) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(second ? h->grid_down : h->grid_up, 1, 1);
    cfg.blockDim = dim3(kMoeThreads, 1, 1);
    cfg.dynamicSmemBytes = second ? h->var.down_smem : h->var.up_smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (second && h->down.cluster_split > 1) {
      attr[n].id = cudaLaunchAttributeClusterDimension;
      attr[n].val.clusterDim.x = h->down.cluster_split, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
      ++n;
    }
    if (h->pdl) {
      attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[n].val.programmaticStreamSerializationAllowed = 1;
      ++n;
    }
    cfg.attrs = n ? attr : nullptr;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, second ? h->var.down : h->var.up, second ? h->down : h->up);
    if (e != cudaSuccess) return set_cuda_error(e);
  }
  return 0;
}

}  // namespace b200

extern "C" {

uint64_t b200_gemm_moe_workspace_bytes(const b200_gemm_moe_args* args) {
  if (b200::moe_check(args) != 0) return 0;
  return b200::kMoeListBytes + (uint64_t)(b200::moe_slots(args) * args->tokens * args->inner) * 4;
}

int b200_gemm_moe_a16w16(const b200_gemm_moe_args* args, void* cuda_stream) {
  b200::MoeCall h;
  const int rc = b200::moe_prepare(args, &h);
  return rc ? rc : b200::moe_run(&h, reinterpret_cast<cudaStream_t>(cuda_stream));
}

}  // extern "C"
