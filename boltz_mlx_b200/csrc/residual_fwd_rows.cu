// Dropout and residual add of rows that are dropped or kept whole (residual_fwd.cuh without the norm): the rows that
// are dropped are known a batch ahead, so that their updates are not read.
#include "residual_fwd.cuh"

namespace triattn {

using H = __half;
using B = __nv_bfloat16;

template <class TX, class TY, Does DO>
static cudaError_t rows(const NormFwdArgs& a, cudaStream_t st) {
  constexpr int VEC = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;
  const int C = a.dim / VEC;
  if (C <= 32) return fwd_one<TX, TY, TX, VEC, 32, 1, 4, 2, DO, true>(a, 32, 256, st);
  if (C <= 64) return fwd_one<TX, TY, TX, VEC, 32, 2, 2, 2, DO, true>(a, 32, 256, st);
  if constexpr (VEC == 4)
    if (C <= 128) return fwd_one<TX, TY, TX, VEC, 32, 4, 2, 2, DO, true>(a, 32, 256, st);
  return cudaErrorInvalidValue;
}

cudaError_t launch_dropout_rows(const NormFwdArgs& a, int y, int out, int vec, cudaStream_t st) {
  if (a.z) {
    if (out == DT_F32 && y == DT_F32) return rows<float, float, kAdd>(a, st);
    if (out == DT_F32 && y == DT_F16) return rows<float, H, kAdd>(a, st);
    if (out == DT_F32 && y == DT_BF16) return rows<float, B, kAdd>(a, st);
    if (out == DT_F16 && y == DT_F16) return rows<H, H, kAdd>(a, st);
    if (out == DT_BF16 && y == DT_BF16) return rows<B, B, kAdd>(a, st);
    return cudaErrorInvalidValue;
  }
  if (out == DT_F32 && y == DT_F32) return rows<float, float, kDrop>(a, st);
  if (out == DT_F16 && y == DT_F32) return rows<H, float, kDrop>(a, st);
  if (out == DT_BF16 && y == DT_F32) return rows<B, float, kDrop>(a, st);
  if (out == DT_F16 && y == DT_F16) return rows<H, H, kDrop>(a, st);
  if (out == DT_BF16 && y == DT_BF16) return rows<B, B, kDrop>(a, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
