// Dropout, residual add and LayerNorm forward, fp32 updates on an fp32 stream (residual_fwd.cuh).
#include "residual_fwd.cuh"

namespace triattn {

using H = __half;
using B = __nv_bfloat16;

cudaError_t launch_fused_fwd(const NormFwdArgs& a, int z, int y, int out, int vec, cudaStream_t st) {
  if (z != DT_F32 || y != DT_F32) return launch_fused16_fwd(a, z, y, out, vec, st);
  if (out == DT_F32) return fwd_types<float, float, float, kFused>(a, vec, st);
  if (out == DT_F16) return fwd_types<float, float, H, kFused>(a, vec, st);
  if (out == DT_BF16) return fwd_types<float, float, B, kFused>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
