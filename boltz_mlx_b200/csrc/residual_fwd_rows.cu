// Dropout and residual add by rows of up to 512 channels (residual_fwd.cuh without the norm).
#include "residual_fwd.cuh"

namespace triattn {

using H = __half;
using B = __nv_bfloat16;

template <class TX, class TY, Does DO>
static cudaError_t rows(const NormFwdArgs& a, int vec, cudaStream_t st) {
  constexpr int VEC = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;
  if (vec >= VEC) {
    const int C = a.dim / VEC;
    if (C <= 8) return fwd_one<TX, TY, TX, VEC, 8, 1, 4, 2, DO, false>(a, 8, 256, st);
    if (C <= 32) return fwd_one<TX, TY, TX, VEC, 32, 1, 4, 2, DO, false>(a, 32, 256, st);
    if (C <= 64) return fwd_one<TX, TY, TX, VEC, 32, 2, 2, 2, DO, false>(a, 32, 256, st);
    if constexpr (VEC == 4) {
      if (C <= 96) return fwd_one<TX, TY, TX, VEC, 32, 3, 2, 2, DO, false>(a, 32, 256, st);
      return fwd_one<TX, TY, TX, VEC, 32, 4, 2, 2, DO, false>(a, 32, 256, st);
    }
  }
  if (a.dim <= 128) return fwd_one<TX, TY, TX, 1, 32, 4, 2, 2, DO, false>(a, 32, 256, st);
  if (a.dim <= 256) return fwd_one<TX, TY, TX, 1, 32, 8, 1, 3, DO, false>(a, 32, 256, st);
  if (a.dim <= 384) return fwd_one<TX, TY, TX, 1, 32, 12, 1, 3, DO, false>(a, 32, 256, st);
  return fwd_one<TX, TY, TX, 1, 32, 16, 1, 3, DO, false>(a, 32, 256, st);
}

cudaError_t launch_dropout_rows(const NormFwdArgs& a, int y, int out, int vec, cudaStream_t st) {
  if (a.z) {
    if (out == DT_F32 && y == DT_F32) return rows<float, float, kAdd>(a, vec, st);
    if (out == DT_F32 && y == DT_F16) return rows<float, H, kAdd>(a, vec, st);
    if (out == DT_F32 && y == DT_BF16) return rows<float, B, kAdd>(a, vec, st);
    if (out == DT_F16 && y == DT_F16) return rows<H, H, kAdd>(a, vec, st);
    if (out == DT_BF16 && y == DT_BF16) return rows<B, B, kAdd>(a, vec, st);
    return cudaErrorInvalidValue;
  }
  if (out == DT_F32 && y == DT_F32) return rows<float, float, kDrop>(a, vec, st);
  if (out == DT_F16 && y == DT_F32) return rows<H, float, kDrop>(a, vec, st);
  if (out == DT_BF16 && y == DT_F32) return rows<B, float, kDrop>(a, vec, st);
  if (out == DT_F16 && y == DT_F16) return rows<H, H, kDrop>(a, vec, st);
  if (out == DT_BF16 && y == DT_BF16) return rows<B, B, kDrop>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
