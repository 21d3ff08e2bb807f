// Gradients of dropout, residual add and LayerNorm, 16-bit updates (residual_bwd.cuh).
#include "residual_bwd.cuh"

namespace triattn {

using H = __half;
using B = __nv_bfloat16;

cudaError_t launch_fused16_bwd(const NormBwdArgs& a, int x, int y, int dout, int vec, cudaStream_t st) {
  if (x == DT_F32 && y == DT_F16 && dout == DT_F16) return bwd_types<float, H, H, true>(a, vec, st);
  if (x == DT_F32 && y == DT_BF16 && dout == DT_BF16) return bwd_types<float, B, B, true>(a, vec, st);
  if (x == DT_F16 && y == DT_F16 && dout == DT_F16) return bwd_types<H, H, H, true>(a, vec, st);
  if (x == DT_BF16 && y == DT_BF16 && dout == DT_BF16) return bwd_types<B, B, B, true>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
