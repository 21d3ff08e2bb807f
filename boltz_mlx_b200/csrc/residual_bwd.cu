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

template <class TX, class TO, int VEC, int NCH, int R, bool HASY>
constexpr int stage_bytes(int width, int dim) {
  return R * ((HASY ? 2 : 1) * row_slot<TX, VEC, NCH>(width, dim) + row_slot<TO, VEC, NCH>(width, dim));
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, bool HASY>
__global__ void __launch_bounds__(LPR ? 256 : 512) norm_bwd_kernel(const NormBwdArgs a, int width) {
  constexpr int EPL = VEC * NCH;
  extern __shared__ __align__(16) char smem[];  // the groups' stages; at the end [groups][2][dim] column sums
  using L = Lanes<VEC, LPR, NCH>;
  __shared__ float red[L::red_floats];
  int phase = 0;
  const L l(a.dim, width);
  using CX = RowCopy<TX, VEC, LPR, NCH>;
  using CO = RowCopy<TO, VEC, LPR, NCH>;
  const int D = a.dim;
  const float inv_d = 1.0f / (float)D;
  const TX* x = static_cast<const TX*>(a.x);
  const TX* ds = static_cast<const TX*>(a.ds);
  const TO* dout = static_cast<const TO*>(a.dout);
  TX* dx = static_cast<TX*>(a.dx);
  TY* dy = static_cast<TY*>(a.dy);

  float w[EPL], dw[EPL], db[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    w[i] = l.act[i / VEC] ? load_param(a.weight, a.param_dtype, l.col(i / VEC) + i % VEC, 1.0f) : 0.0f;
    dw[i] = db[i] = 0.0f;
  }
  const Philox rng(a.drop);
  const bool has_ds = HASY && ds, has_dy = HASY && dy;
  const bool row_draw = has_dy && a.drop.on && !a.drop.per_channel, draw = has_dy && a.drop.on && a.drop.per_channel;

  const int slot_x = row_slot<TX, VEC, NCH>(l.width, D), slot_o = row_slot<TO, VEC, NCH>(l.width, D);
  const int stage = stage_bytes<TX, TO, VEC, NCH, R, HASY>(l.width, D);
  char* ring = smem + l.group * S * stage;
  const uint32_t ring32 = smem_u32(ring);

  const uint32_t rows = a.map.rows, step = gridDim.x * l.groups * R;
  const auto issue = [&](uint32_t base, int s) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = base + l.group * R + r;
      if (row >= rows) continue;
      const uint32_t at = ring32 + s * stage;
      CX::issue(l, at + r * slot_x, x + row_offset(a.xs, row, a.map, D));
      CO::issue(l, at + R * slot_x + r * slot_o, dout + row_offset(a.dos, row, a.map, D));
      if constexpr (HASY)
        if (has_ds) CX::issue(l, at + R * (slot_x + slot_o) + r * slot_x, ds + row_offset(a.dss, row, a.map, D));
    }
  };
  float mean[R], rstd[R], mean_next[R], rstd_next[R];  // of the batch in hand and of the next one
  const auto statistics = [&](uint32_t base) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = base + l.group * R + r;
      mean_next[r] = row < rows ? a.mean[row] : 0.0f;
      rstd_next[r] = row < rows ? a.rstd[row] : 0.0f;
    }
  };

  uint32_t ahead = blockIdx.x * l.groups * R;
  statistics(ahead);
#pragma unroll
  for (int s = 0; s < S - 1; ++s, ahead += step) {
    if (ahead < rows) issue(ahead, s);
    copy_commit();
  }
  int s = 0;
  for (uint32_t base = blockIdx.x * l.groups * R; base < rows; base += step, ahead += step) {
    if (ahead < rows) issue(ahead, s == 0 ? S - 1 : s - 1);
    copy_commit();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = mean_next[r];
      rstd[r] = rstd_next[r];
    }
    statistics(base + step);
    copy_wait<S - 1>();
    l.sync();
    const uint32_t row0 = base + l.group * R;
    const char* here = ring + s * stage;
    // v[2 r] = sum g, v[2 r + 1] = sum g xh
    float xh[R][EPL], g[R][EPL], v[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = row0 + r;
      const bool live = row < rows;
      const TX* xrow = x + (VEC == 1 ? row_offset(a.xs, row, a.map, D) : 0);
      const TO* orow = dout + (VEC == 1 ? row_offset(a.dos, row, a.map, D) : 0);
      v[2 * r] = v[2 * r + 1] = 0.0f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        float xv[VEC], dv[VEC];
        const bool in = live && l.act[c];
#pragma unroll
        for (int k = 0; k < VEC; ++k) xv[k] = mean[r], dv[k] = 0.0f;
        if (in) {
          CX::read(l, here + r * slot_x, xrow, c, xv);
          CO::read(l, here + R * slot_x + r * slot_o, orow, c, dv);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const int i = c * VEC + k;
          xh[r][i] = (xv[k] - mean[r]) * rstd[r];
          dw[i] = fmaf(dv[k], xh[r][i], dw[i]);
          db[i] += dv[k];
          g[r][i] = dv[k] * w[i];
          v[2 * r] += g[r][i];
          v[2 * r + 1] = fmaf(g[r][i], xh[r][i], v[2 * r + 1]);
        }
      }
    }
    l.sum(v, red, phase);
    uint32_t whole = ~0u;  // bit r: row r is not dropped whole
    if constexpr (HASY) {
      if (row_draw) {
        if constexpr (LPR && R > 1) {
          const uint32_t row = row0 + (l.lane & (R - 1));
          const bool k = row < rows && rng.word(mask_base(a.drop, a.map.at(row))) > a.drop.drop_max;
          whole = 0;
#pragma unroll
          for (int r = 0; r < R; ++r) whole |= __shfl_sync(0xffffffffu, (uint32_t)k, r, LPR) << r;
        } else {
          whole = 0;
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (row0 + r < rows && rng.word(mask_base(a.drop, a.map.at(row0 + r))) > a.drop.drop_max) whole |= 1u << r;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = row0 + r;
      const bool live = row < rows;
      const float c1 = v[2 * r] * inv_d, c2 = v[2 * r + 1] * inv_d;
      uint32_t keep[NCH];
#pragma unroll
      for (int c = 0; c < NCH; ++c) keep[c] = whole >> r & 1 ? 0xffu : 0u;
      if constexpr (HASY)
        if (draw) keep_pieces(l, rng, mask_base(a.drop, a.map.at(live ? row : rows - 1)), a.drop.drop_max, keep);
      const TX* srow = ds + (HASY && VEC == 1 && has_ds ? row_offset(a.dss, row, a.map, D) : 0);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        if (!live || !l.act[c]) continue;
        const int col = l.col(c);
        float f[VEC], sv[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const int i = c * VEC + k;
          f[k] = rstd[r] * (g[r][i] - c1 - xh[r][i] * c2);
        }
        if constexpr (HASY) {
          if (has_ds) {
            CX::read(l, here + R * (slot_x + slot_o) + r * slot_x, srow, c, sv);
#pragma unroll
            for (int k = 0; k < VEC; ++k) f[k] += sv[k];
          }
        }
        if (dx) {
          Pack<TX, VEC> o;
#pragma unroll
          for (int k = 0; k < VEC; ++k) o.v[k] = from_f32<TX>(f[k]);
          store_pack(dx + (int64_t)row * D + col, o);
        }
        if constexpr (HASY) {
          if (dy) {
            Pack<TY, VEC> q;
#pragma unroll
            for (int k = 0; k < VEC; ++k) q.v[k] = from_f32<TY>(keep[c] >> k & 1 ? f[k] * a.drop.scale : 0.0f);
            store_pack(dy + (int64_t)row * D + col, q);
          }
        }
      }
    }
    l.sync();
    s = s == S - 1 ? 0 : s + 1;
  }
  copy_wait<0>();

  if (!a.partial) return;
  // groups of one warp first (they own the same channels), then all groups through shared memory
  float* part = a.partial + (size_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int o = LPR ? LPR : 32; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
      db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
    }
  }
  const int sets = LPR ? blockDim.x >> 5 : l.groups;
  const bool writes = LPR ? (threadIdx.x & 31) < LPR : true;
  float* mine = sets == 1 ? part : reinterpret_cast<float*>(smem) + (size_t)(LPR ? threadIdx.x >> 5 : l.group) * 2 * D;
  __syncthreads();  // every warp has read its last rows
  if (writes) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      if (l.act[c]) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          mine[l.col(c) + k] = dw[c * VEC + k];
          mine[D + l.col(c) + k] = db[c * VEC + k];
        }
      }
  }
  if (sets == 1) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) {
    float t = 0.0f;
    for (int k = 0; k < sets; ++k) t += reinterpret_cast<const float*>(smem)[(size_t)k * 2 * D + i];
    part[i] = t;
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

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, bool HASY>
cudaError_t launch_one(const NormBwdArgs& a, int width, int threads, cudaStream_t st) {
  static KernelInfo info;
  const int groups = threads / width, sets = LPR ? threads / 32 : groups;
  size_t smem = (size_t)groups * S * stage_bytes<TX, TO, VEC, NCH, R, HASY>(width, a.dim);
  if (const size_t sums = (size_t)sets * 2 * a.dim * 4; sets > 1 && smem < sums) smem = sums;
  unsigned grid = 0;
  if (cudaError_t e = launch_rows(info, norm_bwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, S, HASY>, a, width, groups * R, threads,
                                  smem, kCtasPerSm, st, &grid);
      e != cudaSuccess || !a.partial)
    return e;
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
  const int C = (a.dim + VEC - 1) / VEC;
  if constexpr (VEC > 1) {
    if (C <= 8) return launch_one<TX, TY, TO, VEC, 8, 1, 2, 3, HASY>(a, 8, 256, st);
    if (C <= 16) return launch_one<TX, TY, TO, VEC, 16, 1, 2, 3, HASY>(a, 16, 256, st);
    if (C <= 32) return launch_one<TX, TY, TO, VEC, 32, 1, 2, 3, HASY>(a, 32, 256, st);
    if (C <= 64) return launch_one<TX, TY, TO, VEC, 32, 2, 1, 3, HASY>(a, 32, 256, st);
    if constexpr (VEC == 4) {
      if (C <= 96) return launch_one<TX, TY, TO, VEC, 32, 3, 1, 3, HASY>(a, 32, 256, st);
      if (C <= 128) return launch_one<TX, TY, TO, VEC, 32, 4, 1, 3, HASY>(a, 32, 256, st);
    }
  } else {
    if (C <= 8) return launch_one<TX, TY, TO, VEC, 8, 1, 2, 3, HASY>(a, 8, 256, st);
    if (C <= 32) return launch_one<TX, TY, TO, VEC, 32, 1, 2, 3, HASY>(a, 32, 256, st);
    if (C <= 128) return launch_one<TX, TY, TO, VEC, 32, 4, 1, 3, HASY>(a, 32, 256, st);
    if (C <= 512) return launch_one<TX, TY, TO, VEC, 32, 16, 1, 3, HASY>(a, 32, 256, st);
  }
  const RowWidth w = row_width<VEC>(C);
  if constexpr (VEC == 4)
    if (w.pieces == 3) return launch_one<TX, TY, TO, VEC, 0, 3, 1, 2, HASY>(a, w.width, w.threads, st);
  return launch_one<TX, TY, TO, VEC, 0, 16 / VEC, 1, 2, HASY>(a, w.width, w.threads, st);
}

template <class TX, class TY, class TO, bool HASY>
cudaError_t launch_types(const NormBwdArgs& a, int vec, cudaStream_t st) {
  if constexpr (sizeof(TX) == 2 && sizeof(TY) == 2 && sizeof(TO) == 2) {
    if (vec == 8) return launch_vec<TX, TY, TO, 8, HASY>(a, st);
  }
  if (vec >= 4) return launch_vec<TX, TY, TO, 4, HASY>(a, st);
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
