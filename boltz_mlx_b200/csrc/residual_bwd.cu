// LayerNorm backward, alone or with the gradients of the residual add and the dropout in front of it:
//
//   xh = (x - mean) rstd,  g = dout w
//   dx = rstd (g - mean_c(g) - xh mean_c(g xh)) (+ ds),  dy = keep ? dx scale : 0
//   dweight = sum_rows dout xh,  dbias = sum_rows dout
//
// Bound by HBM like the forward pass: x, dout (and ds) are read once, dx (and dy) written once.  A lane
// owns the same channels in every row that its group handles, so the two column sums stay in its
// registers until the CTA has seen its last row; they are then joined in shared memory, written as one
// partial row per CTA and summed by a second small kernel in the order of the CTAs: no atomics, the same
// bits on every run.
#include "residual.cuh"

namespace triattn {
namespace {

constexpr int kCtasPerSm = 4;

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, bool HASY>
__global__ void __launch_bounds__(LPR ? 256 : 512) norm_bwd_kernel(const NormBwdArgs a) {
  constexpr int EPL = VEC * NCH;
  extern __shared__ float colsum[];  // LPR: [warps][2][dim] of the column sums
  __shared__ float red[LPR ? 1 : 2 * 2 * RES_MAX_WARPS];
  int phase = 0;
  const int width = LPR ? LPR : blockDim.x;
  const int lane = LPR ? threadIdx.x & (width - 1) : threadIdx.x;
  const int group = LPR ? threadIdx.x / width : 0, groups = LPR ? blockDim.x / width : 1;
  const int D = a.dim;
  const float inv_d = 1.0f / (float)D;
  const TX* x = static_cast<const TX*>(a.x);
  const TX* ds = static_cast<const TX*>(a.ds);
  const TO* dout = static_cast<const TO*>(a.dout);
  TX* dx = static_cast<TX*>(a.dx);
  TY* dy = static_cast<TY*>(a.dy);

  bool act[NCH];
  float w[EPL], dw[EPL], db[EPL];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (lane + c * width) * VEC;
    act[c] = col < D;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      w[c * VEC + v] = act[c] ? load_param(a.weight, a.param_dtype, col + v, 1.0f) : 0.0f;
      dw[c * VEC + v] = db[c * VEC + v] = 0.0f;
    }
  }
  const Philox rng(a.drop);

  const uint32_t step = gridDim.x * groups * R;
  for (uint32_t base = blockIdx.x * groups * R; base < a.map.rows; base += step) {
    const uint32_t row0 = base + group * R;
    RowIndex idx[R];
    Pack<TX, VEC> xr[R][NCH], sr[R][NCH];
    Pack<TO, VEC> gr[R][NCH];
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = row0 + r;
      const bool live = row < a.map.rows;
      idx[r] = a.map.at(live ? row : a.map.rows - 1);
      const TX* px = x + row_offset(a.xs, row, idx[r], D);
      const TO* pg = dout + row_offset(a.dos, row, idx[r], D);
      const TX* ps = ds + (HASY && ds ? row_offset(a.dss, row, idx[r], D) : 0);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int col = (lane + c * width) * VEC;
        if (act[c] && live) {
          xr[r][c] = load_pack<TX, VEC>(px + col);
          gr[r][c] = load_pack<TO, VEC>(pg + col);
          if (HASY && ds) sr[r][c] = load_pack<TX, VEC>(ps + col);
        }
      }
      mean[r] = live ? a.mean[row] : 0.0f;
      rstd[r] = live ? a.rstd[row] : 0.0f;
    }
    // v[2 r] = sum g, v[2 r + 1] = sum g xh
    float xh[R][EPL], g[R][EPL], v[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = row0 + r < a.map.rows;
      v[2 * r] = v[2 * r + 1] = 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const bool in = act[i / VEC] && live;
        const float d = in ? to_f32(gr[r][i / VEC].v[i % VEC]) : 0.0f;
        xh[r][i] = in ? (to_f32(xr[r][i / VEC].v[i % VEC]) - mean[r]) * rstd[r] : 0.0f;
        dw[i] = fmaf(d, xh[r][i], dw[i]);
        db[i] += d;
        g[r][i] = d * w[i];
        v[2 * r] += g[r][i];
        v[2 * r + 1] = fmaf(g[r][i], xh[r][i], v[2 * r + 1]);
      }
    }
    row_sum<LPR, 2 * R>(v, red, phase);
    bool keep_row[R];
    if constexpr (HASY) {
      if (dy && a.drop.on && !a.drop.per_channel) {
        if constexpr (LPR && R > 1) {
          const int mine = lane & (R - 1);
          uint64_t pos = 0;
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (r == mine) pos = mask_base(a.drop, idx[r]);
          const bool k = rng.word(pos) > a.drop.drop_max;
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
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = row0 + r;
      if (row >= a.map.rows) continue;
      const float c1 = v[2 * r] * inv_d, c2 = v[2 * r + 1] * inv_d;
      const uint64_t mb = mask_base(a.drop, idx[r]);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        if (!act[c]) continue;
        const int col = (lane + c * width) * VEC;
        Pack<TX, VEC> o;
        float f[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const int i = c * VEC + k;
          f[k] = rstd[r] * (g[r][i] - c1 - xh[r][i] * c2);
          if (HASY && ds) f[k] += to_f32(sr[r][c].v[k]);
          o.v[k] = from_f32<TX>(f[k]);
        }
        if (dx) store_pack(dx + (int64_t)row * D + col, o);
        if constexpr (HASY) {
          if (dy) {
            uint32_t bits = keep_row[r] ? 0xffu : 0u;
            if (a.drop.on && a.drop.per_channel) bits = keep_bits<VEC>(rng, mb + col, a.drop.drop_max);
            Pack<TY, VEC> q;
#pragma unroll
            for (int k = 0; k < VEC; ++k) q.v[k] = from_f32<TY>(bits >> k & 1 ? f[k] * a.drop.scale : 0.0f);
            store_pack(dy + (int64_t)row * D + col, q);
          }
        }
      }
    }
  }

  if (!a.partial) return;
  float* part = a.partial + (size_t)blockIdx.x * 2 * D;
  if constexpr (LPR == 0) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      if (act[c]) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const int col = (lane + c * width) * VEC + v;
          part[col] = dw[c * VEC + v];
          part[D + col] = db[c * VEC + v];
        }
      }
  } else {
    // groups of one warp first (they own the same channels), then the warps through shared memory
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
        db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
      }
    }
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    float* mine = colsum + (size_t)warp * 2 * D;
    if ((threadIdx.x & 31) < LPR) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        if (act[c]) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            const int col = (lane + c * width) * VEC + v;
            mine[col] = dw[c * VEC + v];
            mine[D + col] = db[c * VEC + v];
          }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) {
      float s = 0.0f;
      for (int k = 0; k < warps; ++k) s += colsum[(size_t)k * 2 * D + i];
      part[i] = s;
    }
  }
}

// Column sums of the CTAs' partial rows: 32 columns per CTA, 16 warps over the partial rows.
template <class TP>
__global__ void __launch_bounds__(512) norm_bwd_join_kernel(const float* __restrict__ partial, int ctas, int dim,
                                                            TP* __restrict__ dweight, TP* __restrict__ dbias) {
  __shared__ float part[16][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;  // of 2 * dim
  float s = 0.0f;
  if (col < 2 * dim)
    for (int i = warp; i < ctas; i += 16) s += partial[(size_t)i * 2 * dim + col];
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < 2 * dim) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += part[i][lane];
    if (col < dim) {
      if (dweight) dweight[col] = from_f32<TP>(s);
    } else if (dbias) {
      dbias[col - dim] = from_f32<TP>(s);
    }
  }
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, bool HASY>
cudaError_t launch_one(const NormBwdArgs& a, int threads, cudaStream_t st) {
  auto kernel = norm_bwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, HASY>;
  const int per_cta = (LPR ? threads / (LPR ? LPR : 1) : 1) * R;
  const long long need = ((long long)a.map.rows + per_cta - 1) / per_cta;
  const long long cap = (long long)device_sm_count() * (threads > 256 ? 2 : kCtasPerSm);
  const unsigned grid = (unsigned)(need < cap ? need : cap);
  const size_t smem = LPR && a.partial ? (size_t)(threads / 32) * 2 * a.dim * 4 : 0;  // at most 32 KB: dim <= 512
  kernel<<<grid, threads, smem, st>>>(a);
  if (!a.partial) return cudaGetLastError();
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  const int blocks = (2 * a.dim + 31) / 32;
  if (a.param_dtype == DT_F32)
    norm_bwd_join_kernel<<<blocks, 512, 0, st>>>(a.partial, (int)grid, a.dim, static_cast<float*>(a.dweight),
                                                static_cast<float*>(a.dbias));
  else if (a.param_dtype == DT_F16)
    norm_bwd_join_kernel<<<blocks, 512, 0, st>>>(a.partial, (int)grid, a.dim, static_cast<__half*>(a.dweight),
                                                static_cast<__half*>(a.dbias));
  else
    norm_bwd_join_kernel<<<blocks, 512, 0, st>>>(a.partial, (int)grid, a.dim, static_cast<__nv_bfloat16*>(a.dweight),
                                                static_cast<__nv_bfloat16*>(a.dbias));
  return cudaGetLastError();
}

template <class TX, class TY, class TO, int VEC, bool HASY>
cudaError_t launch_vec(const NormBwdArgs& a, cudaStream_t st) {
  constexpr int M = 16 / VEC;
  const int C = (a.dim + VEC - 1) / VEC;
  if constexpr (VEC > 1) {
    if (C <= 8) return launch_one<TX, TY, TO, VEC, 8, 1, 2, HASY>(a, 256, st);
    if (C <= 16) return launch_one<TX, TY, TO, VEC, 16, 1, 2, HASY>(a, 256, st);
    if (C <= 32) return launch_one<TX, TY, TO, VEC, 32, 1, 2, HASY>(a, 256, st);
    if (C <= 64) return launch_one<TX, TY, TO, VEC, 32, 2, 1, HASY>(a, 256, st);
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
cudaError_t launch_types(const NormBwdArgs& a, int vec, cudaStream_t st) {
  constexpr int FULL = sizeof(TX) == 2 && sizeof(TY) == 2 && sizeof(TO) == 2 ? 8 : 4;
  if (vec >= FULL) return launch_vec<TX, TY, TO, FULL, HASY>(a, st);
  return launch_vec<TX, TY, TO, 1, HASY>(a, st);
}

}  // namespace

int norm_bwd_max_ctas() { return device_sm_count() * kCtasPerSm; }

cudaError_t launch_norm_bwd(const NormBwdArgs& a, int x_dtype, int y_dtype, int dout_dtype, int vec, cudaStream_t st) {
  using H = __half;
  using B = __nv_bfloat16;
  if (!a.dy && !a.ds) {
    if (x_dtype == DT_F32 && dout_dtype == DT_F32) return launch_types<float, float, float, false>(a, vec, st);
    if (x_dtype == DT_F32 && dout_dtype == DT_F16) return launch_types<float, float, H, false>(a, vec, st);
    if (x_dtype == DT_F32 && dout_dtype == DT_BF16) return launch_types<float, float, B, false>(a, vec, st);
    if (x_dtype == DT_F16 && dout_dtype == DT_F16) return launch_types<H, H, H, false>(a, vec, st);
    if (x_dtype == DT_BF16 && dout_dtype == DT_BF16) return launch_types<B, B, B, false>(a, vec, st);
    return cudaErrorInvalidValue;
  }
  if (x_dtype == DT_F32 && y_dtype == DT_F32) {
    if (dout_dtype == DT_F32) return launch_types<float, float, float, true>(a, vec, st);
    if (dout_dtype == DT_F16) return launch_types<float, float, H, true>(a, vec, st);
    if (dout_dtype == DT_BF16) return launch_types<float, float, B, true>(a, vec, st);
  }
  if (x_dtype == DT_F32 && y_dtype == DT_F16 && dout_dtype == DT_F16) return launch_types<float, H, H, true>(a, vec, st);
  if (x_dtype == DT_F32 && y_dtype == DT_BF16 && dout_dtype == DT_BF16) return launch_types<float, B, B, true>(a, vec, st);
  if (x_dtype == DT_F16 && y_dtype == DT_F16 && dout_dtype == DT_F16) return launch_types<H, H, H, true>(a, vec, st);
  if (x_dtype == DT_BF16 && y_dtype == DT_BF16 && dout_dtype == DT_BF16) return launch_types<B, B, B, true>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
