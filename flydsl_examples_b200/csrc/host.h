// Host-side helpers shared by the translation units that export the C ABI.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

constexpr int kMaxDevices = 16;

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, looked up once; null when the driver does not have it.
EncodeTiledFn get_encode_fn();

// The driver encodes only with a context, which a thread gets with its first runtime call that needs one; where a call of this
// library is the thread's first, its device's is made current. Called once before a call's tensor maps are encoded.
void ensure_context();

// Keeps the error's text for b200_gemm_strerror and returns B200_GEMM_ERR_LAUNCH.
int set_cuda_error(cudaError_t e);

// The current device and its number of SMs.
int current_sms(int* dev, int* sms);

// Lets `fn` launch with `smem_bytes` of dynamic shared memory and clusters of up to 16 CTAs on device `dev`; done once for each.
int allow_launch(const void* fn, int smem_bytes, int dev);

}  // namespace b200
