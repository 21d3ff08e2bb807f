// Dropout and residual add by rows of up to 8192 channels (residual_fwd.cuh without the norm).
#include "residual_fwd.cuh"

namespace triattn {

using H = __half;
using B = __nv_bfloat16;

#define LAUNCH(VEC, LPR, NCH, R, S, WIDTH, THREADS) return fwd_one<TX, TY, TX, VEC, LPR, NCH, R, S, DO, false>(a, WIDTH, THREADS, st)

template <class TX, class TY, Does DO, int VEC>
static cudaError_t pieces(const NormFwdArgs& a, cudaStream_t st) {
  const int C = a.dim / VEC;
  if (C <= 8) LAUNCH(VEC, 8, 1, 4, 2, 8, 256);
  if (C <= 16) LAUNCH(VEC, 16, 1, 4, 2, 16, 256);
  if (C <= 32) LAUNCH(VEC, 32, 1, 4, 2, 32, 256);
  if (C <= 64) LAUNCH(VEC, 32, 2, 2, 2, 32, 256);
  if constexpr (VEC == 4) {
    if (C <= 96) LAUNCH(VEC, 32, 3, 2, 2, 32, 256);
    if (C <= 128) LAUNCH(VEC, 32, 4, 2, 2, 32, 256);
  }
  const RowWidth w = row_width<VEC>(C, 256);
  if constexpr (VEC == 4) {
    if (w.pieces == 2) LAUNCH(VEC, 0, 2, 1, 3, w.width, w.threads);
    if (w.pieces == 3) LAUNCH(VEC, 0, 3, 1, 3, w.width, w.threads);
  }
  LAUNCH(VEC, 0, 16 / VEC, 1, 3, w.width, w.threads);
}

template <class TX, class TY, Does DO>
static cudaError_t rows(const NormFwdArgs& a, int vec, cudaStream_t st) {
  if constexpr (sizeof(TX) == 2 && sizeof(TY) == 2)
    if (vec == 8) return pieces<TX, TY, DO, 8>(a, st);
  if (vec >= 4) return pieces<TX, TY, DO, 4>(a, st);
  if (a.dim <= 16) LAUNCH(1, 8, 2, 4, 2, 8, 256);
  if (a.dim <= 32) LAUNCH(1, 8, 4, 2, 2, 8, 256);
  if (a.dim <= 64) LAUNCH(1, 16, 4, 2, 2, 16, 256);
  if (a.dim <= 128) LAUNCH(1, 32, 4, 2, 2, 32, 256);
  if (a.dim <= 256) LAUNCH(1, 32, 8, 1, 3, 32, 256);
  if (a.dim <= 384) LAUNCH(1, 32, 12, 1, 3, 32, 256);
  if (a.dim <= 512) LAUNCH(1, 32, 16, 1, 3, 32, 256);
  const RowWidth w = row_width<1>(a.dim, 256);
  if (w.pieces == 12) LAUNCH(1, 0, 12, 1, 3, w.width, w.threads);
  LAUNCH(1, 0, 16, 1, 3, w.width, w.threads);
}

#undef LAUNCH

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
