// Gradients of dropout, residual add and LayerNorm, fp32 updates on an fp32 stream (residual_bwd.cuh).
#include "residual_bwd.cuh"

namespace triattn {

using H = __half;
using B = __nv_bfloat16;

cudaError_t launch_fused_bwd(const NormBwdArgs& a, int x, int y, int dout, int vec, cudaStream_t st) {
  if (x != DT_F32 || y != DT_F32) return launch_fused16_bwd(a, x, y, dout, vec, st);
  if (dout == DT_F32) return bwd_types<float, float, float, true>(a, vec, st);
  if (dout == DT_F16) return bwd_types<float, float, H, true>(a, vec, st);
  if (dout == DT_BF16) return bwd_types<float, float, B, true>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
