// Dropout, residual add and LayerNorm forward, 16-bit updates (residual_fwd.cuh).
#include "residual_fwd.cuh"

namespace triattn {

using H = __half;
using B = __nv_bfloat16;

cudaError_t launch_fused16_fwd(const NormFwdArgs& a, int z, int y, int out, int vec, cudaStream_t st) {
  if (z == DT_F32 && y == DT_F16 && out == DT_F16) return fwd_types<float, H, H, kFused>(a, vec, st);
  if (z == DT_F32 && y == DT_BF16 && out == DT_BF16) return fwd_types<float, B, B, kFused>(a, vec, st);
  if (z == DT_F16 && y == DT_F16 && out == DT_F16) return fwd_types<H, H, H, kFused>(a, vec, st);
  if (z == DT_BF16 && y == DT_BF16 && out == DT_BF16) return fwd_types<B, B, B, kFused>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
