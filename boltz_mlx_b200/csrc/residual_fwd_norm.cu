// LayerNorm forward (residual_fwd.cuh).
#include "residual_fwd.cuh"

namespace triattn {

using H = __half;
using B = __nv_bfloat16;

cudaError_t launch_norm_fwd(const NormFwdArgs& a, int z, int out, int vec, cudaStream_t st) {
  if (z == DT_F32 && out == DT_F32) return fwd_types<float, float, float, kNorm>(a, vec, st);
  if (z == DT_F32 && out == DT_F16) return fwd_types<float, float, H, kNorm>(a, vec, st);
  if (z == DT_F32 && out == DT_BF16) return fwd_types<float, float, B, kNorm>(a, vec, st);
  if (z == DT_F16 && out == DT_F16) return fwd_types<H, H, H, kNorm>(a, vec, st);
  if (z == DT_BF16 && out == DT_BF16) return fwd_types<B, B, B, kNorm>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
