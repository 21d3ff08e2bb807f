// LayerNorm forward, alone or behind dropout + residual add (residual.cuh has the formulas).
//
// Bound by HBM: one read of every input and one write of every output.  A persistent grid of row groups; a
// group's next batches of R rows are on their way into shared memory (residual.cuh) while it works on one.
// A row's values stay in registers through both statistics passes (mean, then centred squares).
#include "residual.cuh"

namespace triattn {
namespace {

template <class TX, class TY, int VEC, int NCH, int R, bool HASY>
constexpr int stage_bytes(int width, int dim) {
  return R * (row_slot<TX, VEC, NCH>(width, dim) + (HASY ? row_slot<TY, VEC, NCH>(width, dim) : 0));
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, bool HASY>
__global__ void __launch_bounds__(LPR ? 256 : 512) norm_fwd_kernel(const NormFwdArgs a, int width) {
  constexpr int EPL = VEC * NCH;
  extern __shared__ __align__(16) char smem[];  // LPR: weight and bias in fp32, then the groups' stages
  using L = Lanes<VEC, LPR, NCH>;
  __shared__ float red[L::red_floats];
  int phase = 0;
  const L l(a.dim, width);
  using CX = RowCopy<TX, VEC, LPR, NCH>;
  using CY = RowCopy<TY, VEC, LPR, NCH>;
  const int D = a.dim;
  const float inv_d = 1.0f / (float)D;
  const TX* z = static_cast<const TX*>(a.z);
  const TY* y = static_cast<const TY*>(a.y);
  TX* sum = static_cast<TX*>(a.sum);
  TO* out = static_cast<TO*>(a.out);

  // Whole-CTA rows keep weight and bias in registers, rows of one warp (several at once) in shared memory.
  float* wb = reinterpret_cast<float*>(smem);
  const int wb_pad = LPR ? (D + VEC - 1) / VEC * VEC : 0;
  float w[LPR ? 1 : EPL], b[LPR ? 1 : EPL];
  if constexpr (LPR) {
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
      wb[i] = load_param(a.weight, a.param_dtype, i, 1.0f);
      wb[wb_pad + i] = load_param(a.bias, a.param_dtype, i, 0.0f);
    }
    __syncthreads();
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      w[i] = l.act[i / VEC] ? load_param(a.weight, a.param_dtype, l.col(i / VEC) + i % VEC, 1.0f) : 0.0f;
      b[i] = l.act[i / VEC] ? load_param(a.bias, a.param_dtype, l.col(i / VEC) + i % VEC, 0.0f) : 0.0f;
    }
  }
  const Philox rng(a.drop);
  const bool row_draw = HASY && a.drop.on && !a.drop.per_channel, draw = HASY && a.drop.on && a.drop.per_channel;

  const int slot_x = row_slot<TX, VEC, NCH>(l.width, D), slot_y = row_slot<TY, VEC, NCH>(l.width, D);
  const int stage = stage_bytes<TX, TY, VEC, NCH, R, HASY>(l.width, D);
  char* ring = smem + (wb_pad * 8 + 15) / 16 * 16 + l.group * S * stage;
  const uint32_t ring32 = smem_u32(ring);
  uint32_t kept = ~0u;  // bit s * R + r: row r of stage s is not dropped whole

  const uint32_t rows = a.map.rows, step = gridDim.x * l.groups * R;
  const auto issue = [&](uint32_t base, int s) {
    const uint32_t row0 = base + l.group * R;
    if constexpr (HASY) {
      if (row_draw) {
        // one draw per row: lane k of a group takes that of row k, and hands it round
        if constexpr (LPR && R > 1) {
          const uint32_t row = row0 + (l.lane & (R - 1));
          const bool k = row < rows && rng.word(mask_base(a.drop, a.map.at(row))) > a.drop.drop_max;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const uint32_t bit = 1u << (s * R + r);
            kept = __shfl_sync(0xffffffffu, (int)k, r, LPR) ? kept | bit : kept & ~bit;
          }
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const bool k = row0 + r < rows && rng.word(mask_base(a.drop, a.map.at(row0 + r))) > a.drop.drop_max;
            const uint32_t bit = 1u << (s * R + r);
            kept = k ? kept | bit : kept & ~bit;
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = row0 + r;
      if (row >= rows) continue;
      const uint32_t at = ring32 + s * stage + r * slot_x;
      CX::issue(l, at, z + row_offset(a.zs, row, a.map, D));
      if constexpr (HASY) {
        if (kept >> (s * R + r) & 1)  // a row that is dropped whole is not read
          CY::issue(l, ring32 + s * stage + R * slot_x + r * slot_y, y + row_offset(a.ys, row, a.map, D));
      }
    }
  };

  uint32_t ahead = blockIdx.x * l.groups * R;
#pragma unroll
  for (int s = 0; s < S - 1; ++s, ahead += step) {
    if (ahead < rows) issue(ahead, s);
    copy_commit();
  }
  int s = 0;
  // the loop's count is the same for every lane of a CTA (whole-warp shuffles, CTA barriers)
  for (uint32_t base = blockIdx.x * l.groups * R; base < rows; base += step, ahead += step) {
    if (ahead < rows) issue(ahead, s == 0 ? S - 1 : s - 1);
    copy_commit();
    copy_wait<S - 1>();
    l.sync();
    const uint32_t row0 = base + l.group * R;
    const char* here = ring + s * stage;
    float x[R][EPL];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = row0 + r;
      const bool live = row < rows;
      const TX* zrow = z + (VEC == 1 ? row_offset(a.zs, row, a.map, D) : 0);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        float v[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = 0.0f;
        if (live && l.act[c]) CX::read(l, here + r * slot_x, zrow, c, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[r][c * VEC + k] = v[k];
      }
      if constexpr (HASY) {
        const TY* yrow = y + (VEC == 1 ? row_offset(a.ys, row, a.map, D) : 0);
        uint32_t keep[NCH];
        const uint32_t whole = kept >> (s * R + r) & 1 ? 0xffu : 0u;
#pragma unroll
        for (int c = 0; c < NCH; ++c) keep[c] = whole;
        if (draw) keep_pieces(l, rng, mask_base(a.drop, a.map.at(live ? row : rows - 1)), a.drop.drop_max, keep);
        TX* p = sum + row_offset(a.ss, row, a.map, D);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          if (!live || !l.act[c]) continue;
          float v[VEC];
          if (keep[c]) {
            CY::read(l, here + R * slot_x + r * slot_y, yrow, c, v);
#pragma unroll
            for (int k = 0; k < VEC; ++k)
              if (keep[c] >> k & 1) x[r][c * VEC + k] = fmaf(v[k], a.drop.scale, x[r][c * VEC + k]);
          }
          Pack<TX, VEC> o;
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            o.v[k] = from_f32<TX>(x[r][c * VEC + k]);
            x[r][c * VEC + k] = to_f32(o.v[k]);  // the norm is taken of the stream as it is held
          }
          store_pack(p + l.col(c), o);
        }
      }
    }
    l.sync();

    float mean[R], var[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) mean[r] += x[r][i];
    }
    l.sum(mean, red, phase);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] *= inv_d;
      var[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        x[r][i] = l.act[i / VEC] ? x[r][i] - mean[r] : 0.0f;
        var[r] = fmaf(x[r][i], x[r][i], var[r]);
      }
    }
    l.sum(var, red, phase);
#pragma unroll
    for (int r = 0; r < R; ++r) var[r] = rsqrtf(fmaf(var[r], inv_d, a.eps));  // now rstd
    if (a.mean && l.lane == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row0 + r < rows) {
          a.mean[row0 + r] = mean[r];
          a.rstd[row0 + r] = var[r];
        }
    }
    TO* po[R];
#pragma unroll
    for (int r = 0; r < R; ++r) po[r] = out + row_offset(a.os, row0 + r, a.map, D);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (!l.act[c]) continue;
      const int col = l.col(c);
      Pack<float, VEC> wc, bc;
      if constexpr (LPR) {
        if constexpr (VEC == 8) {
          const Pack<float, 4> w0 = load_pack<float, 4>(wb + col), w1 = load_pack<float, 4>(wb + col + 4);
          const Pack<float, 4> b0 = load_pack<float, 4>(wb + wb_pad + col), b1 = load_pack<float, 4>(wb + wb_pad + col + 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) wc.v[k] = w0.v[k], wc.v[k + 4] = w1.v[k], bc.v[k] = b0.v[k], bc.v[k + 4] = b1.v[k];
        } else {
          wc = load_pack<float, VEC>(wb + col);
          bc = load_pack<float, VEC>(wb + wb_pad + col);
        }
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) wc.v[k] = w[c * VEC + k], bc.v[k] = b[c * VEC + k];
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (row0 + r >= rows) continue;
        Pack<TO, VEC> h;
#pragma unroll
        for (int k = 0; k < VEC; ++k) h.v[k] = from_f32<TO>(fmaf(x[r][c * VEC + k] * var[r], wc.v[k], bc.v[k]));
        store_pack(po[r] + col, h);
      }
    }
    s = s == S - 1 ? 0 : s + 1;
  }
  copy_wait<0>();
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, bool HASY>
cudaError_t launch_one(const NormFwdArgs& a, int width, int threads, cudaStream_t st) {
  static KernelInfo info;
  const int groups = threads / width, wb = LPR ? ((a.dim + VEC - 1) / VEC * VEC * 8 + 15) / 16 * 16 : 0;
  const size_t smem = wb + (size_t)groups * S * stage_bytes<TX, TY, VEC, NCH, R, HASY>(width, a.dim);
  return launch_rows(info, norm_fwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, S, HASY>, a, width, groups * R, threads, smem, 8, st,
                     nullptr);
}

template <class TX, class TY, class TO, int VEC, bool HASY>
cudaError_t launch_vec(const NormFwdArgs& a, cudaStream_t st) {
  const int C = (a.dim + VEC - 1) / VEC;
  constexpr int W = sizeof(TX) == 4 || HASY ? 2 : 4;  // rows of a batch: 16 to 64 bytes a lane and stage
  if constexpr (VEC > 1) {
    if (C <= 8) return launch_one<TX, TY, TO, VEC, 8, 1, W, 3, HASY>(a, 8, 256, st);
    if (C <= 16) return launch_one<TX, TY, TO, VEC, 16, 1, W, 3, HASY>(a, 16, 256, st);
    if (C <= 32) return launch_one<TX, TY, TO, VEC, 32, 1, W, 3, HASY>(a, 32, 256, st);
    if (C <= 64) return launch_one<TX, TY, TO, VEC, 32, 2, W / 2, 3, HASY>(a, 32, 256, st);
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
    if (w.pieces == 3) return launch_one<TX, TY, TO, VEC, 0, 3, 1, 3, HASY>(a, w.width, w.threads, st);
  return launch_one<TX, TY, TO, VEC, 0, 16 / VEC, 1, 3, HASY>(a, w.width, w.threads, st);
}

template <class TX, class TY, class TO, bool HASY>
cudaError_t launch_types(const NormFwdArgs& a, int vec, cudaStream_t st) {
  if constexpr (sizeof(TX) == 2 && sizeof(TY) == 2 && sizeof(TO) == 2) {
    if (vec == 8) return launch_vec<TX, TY, TO, 8, HASY>(a, st);
  }
  if (vec >= 4) return launch_vec<TX, TY, TO, 4, HASY>(a, st);
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
