// LayerNorm forward, alone or behind dropout + residual add (residual.cuh has the formulas).
//
// Bound by HBM: one read of every input and one write of every output; about 40 issued instructions per
// 128-channel row against 1 KB of traffic.  A row stays in the registers of LPR lanes (or of a whole CTA
// when it is longer than 512 channels), NCH accesses of VEC elements each, so that both statistics passes
// (mean, then centred squares) run without a second read; R rows per group are in flight to cover the
// latency of the loads.
#include "residual.cuh"

namespace triattn {
namespace {

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, bool HASY>
__global__ void __launch_bounds__(LPR ? 256 : 512) norm_fwd_kernel(const NormFwdArgs a) {
  constexpr int EPL = VEC * NCH;
  __shared__ float red[LPR ? 1 : 2 * 2 * RES_MAX_WARPS];
  int phase = 0;
  const int width = LPR ? LPR : blockDim.x;  // lanes of a row
  const int lane = LPR ? threadIdx.x & (width - 1) : threadIdx.x;
  const int group = LPR ? threadIdx.x / width : 0, groups = LPR ? blockDim.x / width : 1;
  const int D = a.dim;
  const float inv_d = 1.0f / (float)D;
  const TX* z = static_cast<const TX*>(a.z);
  const TY* y = static_cast<const TY*>(a.y);
  TX* sum = static_cast<TX*>(a.sum);
  TO* out = static_cast<TO*>(a.out);

  bool act[NCH];
  float w[EPL], b[EPL];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (lane + c * width) * VEC;
    act[c] = col < D;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      w[c * VEC + v] = act[c] ? load_param(a.weight, a.param_dtype, col + v, 1.0f) : 0.0f;
      b[c * VEC + v] = act[c] ? load_param(a.bias, a.param_dtype, col + v, 0.0f) : 0.0f;
    }
  }
  const Philox rng(a.drop);

  const uint32_t step = gridDim.x * groups * R;
  // the loop's count is the same for every lane of a CTA (whole-warp shuffles, CTA barriers)
  for (uint32_t base = blockIdx.x * groups * R; base < a.map.rows; base += step) {
    const uint32_t row0 = base + group * R;
    float x[R][EPL];
    RowIndex idx[R];
    Pack<TX, VEC> zr[R][NCH];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = row0 + r;
      idx[r] = a.map.at(row < a.map.rows ? row : a.map.rows - 1);
      const TX* p = z + row_offset(a.zs, row, idx[r], D);
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        if (act[c] && row < a.map.rows) zr[r][c] = load_pack<TX, VEC>(p + (lane + c * width) * VEC);
    }
    if constexpr (HASY) {
      Pack<TY, VEC> yr[R][NCH];
      bool keep_row[R];
      if (a.drop.on && !a.drop.per_channel) {
        // one draw per row: lane k of a group takes the R rows' draws in turn and hands them round
        bool k;
        if constexpr (LPR && R > 1) {
          const int mine = lane & (R - 1);
          uint64_t pos = 0;
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (r == mine) pos = mask_base(a.drop, idx[r]);
          k = rng.word(pos) > a.drop.drop_max;
#pragma unroll
          for (int r = 0; r < R; ++r) keep_row[r] = __shfl_sync(0xffffffffu, (int)k, r, LPR) != 0;
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r) keep_row[r] = rng.word(mask_base(a.drop, idx[r])) > a.drop.drop_max;
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) keep_row[r] = true;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t row = row0 + r;
        const TY* p = y + row_offset(a.ys, row, idx[r], D);
#pragma unroll
        for (int c = 0; c < NCH; ++c)  // a row that is dropped whole is not read
          if (act[c] && row < a.map.rows && keep_row[r]) yr[r][c] = load_pack<TY, VEC>(p + (lane + c * width) * VEC);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t row = row0 + r;
        const bool live = row < a.map.rows;
        const uint64_t mb = mask_base(a.drop, idx[r]);
        TX* p = sum + row_offset(a.ss, row, idx[r], D);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          const int col = (lane + c * width) * VEC;
          uint32_t bits = keep_row[r] ? 0xffu : 0u;
          if (a.drop.on && a.drop.per_channel) bits = keep_bits<VEC>(rng, mb + col, a.drop.drop_max);
          Pack<TX, VEC> s;
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            float f = 0.0f;
            if (act[c] && live) {
              f = to_f32(zr[r][c].v[v]);
              if (bits >> v & 1) f = fmaf(to_f32(yr[r][c].v[v]), a.drop.scale, f);
            }
            s.v[v] = from_f32<TX>(f);
            x[r][c * VEC + v] = to_f32(s.v[v]);  // the norm is taken of the stream as it is held
          }
          if (act[c] && live) store_pack(p + col, s);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int v = 0; v < VEC; ++v)
            x[r][c * VEC + v] = act[c] && row0 + r < a.map.rows ? to_f32(zr[r][c].v[v]) : 0.0f;
    }

    float mean[R], var[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) mean[r] += x[r][i];
    }
    row_sum<LPR, R>(mean, red, phase);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] *= inv_d;
      var[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        x[r][i] = act[i / VEC] ? x[r][i] - mean[r] : 0.0f;
        var[r] = fmaf(x[r][i], x[r][i], var[r]);
      }
    }
    row_sum<LPR, R>(var, red, phase);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = row0 + r;
      if (row >= a.map.rows) continue;
      const float rstd = rsqrtf(fmaf(var[r], inv_d, a.eps));
      if (lane == 0) {
        if (a.mean) a.mean[row] = mean[r];
        if (a.rstd) a.rstd[row] = rstd;
      }
      TO* p = out + row_offset(a.os, row, idx[r], D);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        if (!act[c]) continue;
        Pack<TO, VEC> h;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const int i = c * VEC + v;
          h.v[v] = from_f32<TO>(fmaf(x[r][i] * rstd, w[i], b[i]));
        }
        store_pack(p + (lane + c * width) * VEC, h);
      }
    }
  }
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, bool HASY>
cudaError_t launch_one(const NormFwdArgs& a, int threads, cudaStream_t st) {
  auto kernel = norm_fwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, HASY>;
  const int per_cta = (LPR ? threads / (LPR ? LPR : 1) : 1) * R;
  const long long need = ((long long)a.map.rows + per_cta - 1) / per_cta;
  const long long cap = (long long)device_sm_count() * (2048 / threads);
  kernel<<<(unsigned)(need < cap ? need : cap), threads, 0, st>>>(a);
  return cudaGetLastError();
}

// Lanes per row by the row's number of accesses C = ceil(dim / VEC): the fewest that keep a lane's share
// within 16 elements (registers), and no more than C rounded up to a power of two below one warp.
template <class TX, class TY, class TO, int VEC, bool HASY>
cudaError_t launch_vec(const NormFwdArgs& a, cudaStream_t st) {
  constexpr int M = 16 / VEC;  // accesses per lane at most
  const int C = (a.dim + VEC - 1) / VEC;
  if constexpr (VEC > 1) {
    if (C <= 8) return launch_one<TX, TY, TO, VEC, 8, 1, 4, HASY>(a, 256, st);
    if (C <= 16) return launch_one<TX, TY, TO, VEC, 16, 1, 4, HASY>(a, 256, st);
    if (C <= 32) return launch_one<TX, TY, TO, VEC, 32, 1, VEC == 4 ? 4 : 2, HASY>(a, 256, st);
    if (C <= 64) return launch_one<TX, TY, TO, VEC, 32, 2, VEC == 4 ? 2 : 1, HASY>(a, 256, st);
    if constexpr (VEC == 4)
      if (C <= 128) return launch_one<TX, TY, TO, VEC, 32, 4, 1, HASY>(a, 256, st);
  } else {
    if (C <= 128) return launch_one<TX, TY, TO, VEC, 32, 4, 2, HASY>(a, 256, st);
    if (C <= 512) return launch_one<TX, TY, TO, VEC, 32, 16, 1, HASY>(a, 256, st);
  }
  const int threads = ((C + M - 1) / M + 31) / 32 * 32;
  return launch_one<TX, TY, TO, VEC, 0, M, 1, HASY>(a, threads, st);
}

template <class TX, class TY, class TO, bool HASY>
cudaError_t launch_types(const NormFwdArgs& a, int vec, cudaStream_t st) {
  constexpr int FULL = sizeof(TX) == 2 && sizeof(TY) == 2 && sizeof(TO) == 2 ? 8 : 4;
  if (vec >= FULL) return launch_vec<TX, TY, TO, FULL, HASY>(a, st);
  return launch_vec<TX, TY, TO, 1, HASY>(a, st);
}

}  // namespace

cudaError_t launch_norm_fwd(const NormFwdArgs& a, int z_dtype, int y_dtype, int out_dtype, int vec, cudaStream_t st) {
  using H = __half;
  using B = __nv_bfloat16;
  if (!a.y) {
    if (z_dtype == DT_F32 && out_dtype == DT_F32) return launch_types<float, float, float, false>(a, vec, st);
    if (z_dtype == DT_F32 && out_dtype == DT_F16) return launch_types<float, float, H, false>(a, vec, st);
    if (z_dtype == DT_F32 && out_dtype == DT_BF16) return launch_types<float, float, B, false>(a, vec, st);
    if (z_dtype == DT_F16 && out_dtype == DT_F16) return launch_types<H, H, H, false>(a, vec, st);
    if (z_dtype == DT_BF16 && out_dtype == DT_BF16) return launch_types<B, B, B, false>(a, vec, st);
    return cudaErrorInvalidValue;
  }
  if (z_dtype == DT_F32 && y_dtype == DT_F32) {
    if (out_dtype == DT_F32) return launch_types<float, float, float, true>(a, vec, st);
    if (out_dtype == DT_F16) return launch_types<float, float, H, true>(a, vec, st);
    if (out_dtype == DT_BF16) return launch_types<float, float, B, true>(a, vec, st);
  }
  if (z_dtype == DT_F32 && y_dtype == DT_F16 && out_dtype == DT_F16) return launch_types<float, H, H, true>(a, vec, st);
  if (z_dtype == DT_F32 && y_dtype == DT_BF16 && out_dtype == DT_BF16) return launch_types<float, B, B, true>(a, vec, st);
  if (z_dtype == DT_F16 && y_dtype == DT_F16 && out_dtype == DT_F16) return launch_types<H, H, H, true>(a, vec, st);
  if (z_dtype == DT_BF16 && y_dtype == DT_BF16 && out_dtype == DT_BF16) return launch_types<B, B, B, true>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
