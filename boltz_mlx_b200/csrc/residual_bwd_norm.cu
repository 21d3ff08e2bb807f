// LayerNorm backward (residual_bwd.cuh).
#include "residual_bwd.cuh"

namespace triattn {

using H = __half;
using B = __nv_bfloat16;

int norm_bwd_max_ctas() { return device_sm_count() * kCtasPerSm * kPartials; }

cudaError_t launch_norm_bwd(const NormBwdArgs& a, int x, int dout, int vec, cudaStream_t st) {
  if (x == DT_F32 && dout == DT_F32) return bwd_types<float, float, float, false>(a, vec, st);
  if (x == DT_F32 && dout == DT_F16) return bwd_types<float, float, H, false>(a, vec, st);
  if (x == DT_F32 && dout == DT_BF16) return bwd_types<float, float, B, false>(a, vec, st);
  if (x == DT_F16 && dout == DT_F16) return bwd_types<H, H, H, false>(a, vec, st);
  if (x == DT_BF16 && dout == DT_BF16) return bwd_types<B, B, B, false>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
