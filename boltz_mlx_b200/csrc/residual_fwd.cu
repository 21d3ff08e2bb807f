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

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, bool HASY, bool DENSE>
__global__ void __launch_bounds__(LPR ? 256 : 512) norm_fwd_kernel(const NormFwdArgs a, int width, Split split) {
  using L = Lanes<VEC, LPR, NCH>;
  constexpr int P = L::PAIRS;
  extern __shared__ __align__(16) char smem[];  // LPR: weight and bias in fp32, then the groups' stages
  __shared__ __align__(16) float red[L::red_floats];
  int phase = 0;
  const L l(a.dim, width);
  const int D = a.dim;
  const float inv_d = 1.0f / (float)D;

  // Rows of several warps keep weight and bias in registers, rows of one warp (several at once) in shared memory.
  float* wb = reinterpret_cast<float*>(smem);
  const int wb_pad = LPR ? (D + VEC - 1) / VEC * VEC : 0;
  Pair w[LPR ? 1 : P], b[LPR ? 1 : P];
  if constexpr (LPR) {
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
      wb[i] = load_param(a.weight, a.param_dtype, i, 1.0f);
      wb[wb_pad + i] = load_param(a.bias, a.param_dtype, i, 0.0f);
    }
    __syncthreads();
  } else {
    load_pairs(l, a.weight, a.param_dtype, 1.0f, w);
    load_pairs(l, a.bias, a.param_dtype, 0.0f, b);
    l.clear(red);
  }
  const Philox rng(a.drop);
  const bool row_draw = HASY && a.drop.on && !a.drop.per_channel, draw = HASY && a.drop.on && a.drop.per_channel;
  const Pair scale = both(a.drop.scale);

  const int slot_x = row_slot<TX, VEC, NCH>(l.width, D), slot_y = row_slot<TY, VEC, NCH>(l.width, D);
  const int stage = stage_bytes<TX, TY, VEC, NCH, R, HASY>(l.width, D);
  char* ring = smem + (wb_pad * 8 + 15) / 16 * 16 + l.group * S * stage;
  const RowIn<TX, VEC, LPR, NCH, DENSE> z(l, a.map, a.z, a.zs, ring);
  const RowIn<TY, VEC, LPR, NCH, DENSE> y(l, a.map, a.y, a.ys, ring + R * slot_x);
  const RowOut<TX, VEC, LPR, NCH, DENSE> sum(l, a.map, a.sum, a.ss);
  const RowOut<TO, VEC, LPR, NCH, DENSE> out(l, a.map, a.out, a.os);
  for (int k = 0; k < S; ++k) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      z.clear(k * stage + r * slot_x);
      if (HASY) y.clear(k * stage + r * slot_y);
    }
  }
  uint32_t kept = ~0u;  // bit s * R + r: row r of stage s is not dropped whole

  const uint32_t rows = a.map.rows, step = l.groups * R;
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
      z.issue(s * stage + r * slot_x, row);
      if constexpr (HASY) {
        if (kept >> (s * R + r) & 1) y.issue(s * stage + r * slot_y, row);  // a row that is dropped whole is not read
      }
    }
  };

  uint32_t first, end;  // rows of this CTA
  split.range(blockIdx.x, first, end);
  first *= step;
  end *= step;
  uint32_t ahead = first;
#pragma unroll
  for (int s = 0; s < S - 1; ++s, ahead += step) {
    if (ahead < end) issue(ahead, s);
    copy_commit();
  }
  int s = 0;
  // the loop's count is the same for every lane of a CTA (whole-warp shuffles, barriers)
  for (uint32_t base = first; base < end; base += step, ahead += step) {
    if (ahead < end) issue(ahead, s == 0 ? S - 1 : s - 1);
    copy_commit();
    copy_wait<S - 1>();
    l.sync();
    const uint32_t row0 = base + l.group * R;
    // Rows behind the last one are computed from what their place holds, and not stored.
    Pair x[R][P];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = row0 + r;
      const bool live = row < rows;
      z.read(s * stage + r * slot_x, row, live, x[r]);
      if constexpr (HASY) {
        const bool whole = kept >> (s * R + r) & 1;
        if (whole) {
          Pair v[P];
          y.read(s * stage + r * slot_y, row, live, v);
          if (draw) {
            each_kept(l, rng, mask_base(a.drop, a.map.at(live ? row : rows - 1)), a.drop.drop_max, [&](bool k, int i) {
              const float2 xi = halves(x[r][i / 2]), vi = halves(v[i / 2]);
              const float f = i & 1 ? xi.y : xi.x, g = k ? fmaf(i & 1 ? vi.y : vi.x, a.drop.scale, f) : f;
              x[r][i / 2] = i & 1 ? pair(xi.x, g) : pair(g, xi.y);
            });
          } else {
#pragma unroll
            for (int j = 0; j < P; ++j) x[r][j] = fma2(v[j], scale, x[r][j]);
          }
        }
        if constexpr (sizeof(TX) == 2) {  // the norm is taken of the stream as it is held
#pragma unroll
          for (int j = 0; j < P; ++j) {
            TX held[2];
            from_pair(x[r][j], held);
            x[r][j] = to_pair(held);
          }
        }
        if (live) sum.row(row, x[r]);
      }
    }
    l.sync();

    float mean[R], var[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      Pair t = x[r][0];
#pragma unroll
      for (int j = 1; j < P; ++j) t = t + x[r][j];
      mean[r] = total(t);
    }
    l.sum(mean, red, phase);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] *= inv_d;
      const Pair m = both(-mean[r]);
      Pair t = both(0.0f);
      centre(l, m, x[r], t);
      var[r] = total(t);
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
    for (int r = 0; r < R; ++r) po[r] = out.at(row0 + r);
    constexpr int STEP = VEC == 1 && NCH > 1 ? 2 : 1;  // pieces of a pair
#pragma unroll
    for (int c = 0; c < NCH; c += STEP) {
      constexpr int N = VEC > 1 ? VEC / 2 : 1;
      Pair wc[N], bc[N];
      if constexpr (LPR) {
        if constexpr (VEC > 1) {
#pragma unroll
          for (int j = 0; j < N; ++j) wc[j] = bc[j] = both(0.0f);
          if (l.act(c)) {
#pragma unroll
            for (int j = 0; j < N; j += 2) {
              const Pack<float, 4> wq = load_pack<float, 4>(wb + l.col(c) + 2 * j);
              const Pack<float, 4> bq = load_pack<float, 4>(wb + wb_pad + l.col(c) + 2 * j);
              wc[j] = pair(wq.v[0], wq.v[1]), wc[j + 1] = pair(wq.v[2], wq.v[3]);
              bc[j] = pair(bq.v[0], bq.v[1]), bc[j + 1] = pair(bq.v[2], bq.v[3]);
            }
          }
        } else {
          const bool a0 = l.act(c), a1 = STEP == 2 && c + 1 < NCH && l.act(c + 1);
          wc[0] = pair(a0 ? wb[l.col(c)] : 0.0f, a1 ? wb[l.col(c + 1)] : 0.0f);
          bc[0] = pair(a0 ? wb[wb_pad + l.col(c)] : 0.0f, a1 ? wb[wb_pad + l.col(c + 1)] : 0.0f);
        }
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) wc[j] = w[(VEC > 1 ? c * N : c / 2) + j], bc[j] = b[(VEC > 1 ? c * N : c / 2) + j];
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Pair rstd = both(var[r]);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          Pair& h = x[r][(VEC > 1 ? c * N : c / 2) + j];
          h = fma2(h * rstd, wc[j], bc[j]);
        }
        if (row0 + r < rows) {
#pragma unroll
          for (int k = 0; k < STEP; ++k)
            if (c + k < NCH) out.piece(po[r], c + k, x[r]);
        }
      }
    }
    s = s == S - 1 ? 0 : s + 1;
  }
  copy_wait<0>();
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, bool HASY, bool DENSE>
cudaError_t launch_one(const NormFwdArgs& a, int width, int threads, cudaStream_t st) {
  static KernelInfo info;
  const int groups = threads / width, wb = LPR ? ((a.dim + VEC - 1) / VEC * VEC * 8 + 15) / 16 * 16 : 0;
  const size_t smem = wb + (size_t)groups * S * stage_bytes<TX, TY, VEC, NCH, R, HASY>(width, a.dim);
  int fit = 0;
  if (cudaError_t e = info.fit(norm_fwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, S, HASY, DENSE>, threads, smem, &fit);
      e != cudaSuccess)
    return e;
  // Many CTAs of few batches: they are handed to the SMs as these come free.  An equal share for every resident
  // CTA leaves the SMs that the memory system serves last working alone at the end (0.82 of the copy rate
  // instead of 0.98 at 2^20 rows of 128 fp32).  A CTA has to load weight and bias, though, so that long rows
  // want more batches, in 16 bits (half the traffic a row) most (0.70 instead of 0.62 at 8192 rows of 4096).
  const uint32_t per = groups * R, batches = ((uint32_t)a.map.rows + per - 1) / per;
  const uint32_t resident = (uint32_t)(device_sm_count() * fit);
  uint32_t few = (batches + resident - 1) / resident;
  constexpr uint32_t most = LPR ? 5 : VEC == 8 ? 16 : 4;
  if (few > most) few = most;
  norm_fwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, S, HASY, DENSE><<<(batches + few - 1) / few, threads, smem, st>>>(
      a, width, Split{0, 0, few, batches});
  return cudaGetLastError();
}

template <class TX, class TY, class TO, int VEC, bool HASY, bool DENSE>
cudaError_t launch_vec(const NormFwdArgs& a, cudaStream_t st) {
  const int C = (a.dim + VEC - 1) / VEC;
#define LAUNCH(LPR, NCH, R, S, WIDTH, THREADS) \
  return launch_one<TX, TY, TO, VEC, LPR, NCH, R, S, HASY, DENSE>(a, WIDTH, THREADS, st)
  if constexpr (VEC > 1) {
    if (C <= 8) LAUNCH(8, 1, 4, 2, 8, 256);
    if (C <= 16) LAUNCH(16, 1, 4, 2, 16, 256);
    if (C <= 32) LAUNCH(32, 1, 4, 2, 32, 256);
    if (C <= 64) LAUNCH(32, 2, 2, 2, 32, 256);
    if constexpr (VEC == 4) {
      if (C <= 96) LAUNCH(32, 3, 2, 2, 32, 256);
      if (C <= 128) LAUNCH(32, 4, 2, 2, 32, 256);
    }
  } else {
    if (C <= 8) LAUNCH(8, 1, 2, 3, 8, 256);
    if (C <= 32) LAUNCH(32, 1, 2, 3, 32, 256);
    if (C <= 128) LAUNCH(32, 4, 1, 3, 32, 256);
    if (C <= 512) LAUNCH(32, 16, 1, 3, 32, 256);
  }
  const RowWidth w = row_width<VEC>(C, 256);
  if constexpr (VEC == 4) {
    if (w.pieces == 2) LAUNCH(0, 2, 1, 3, w.width, w.threads);
    if (w.pieces == 3) LAUNCH(0, 3, 1, 3, w.width, w.threads);
  }
  LAUNCH(0, 16 / VEC, 1, 3, w.width, w.threads);
#undef LAUNCH
}

template <class TX, class TY, class TO, bool HASY>
cudaError_t launch_types(const NormFwdArgs& a, int vec, cudaStream_t st) {
  const bool dense = a.zs.dense && a.os.dense && (!HASY || (a.ys.dense && a.ss.dense));
  if constexpr (sizeof(TX) == 2 && sizeof(TY) == 2 && sizeof(TO) == 2) {
    if (vec == 8) return dense ? launch_vec<TX, TY, TO, 8, HASY, true>(a, st) : launch_vec<TX, TY, TO, 8, HASY, false>(a, st);
  }
  if (vec >= 4) return dense ? launch_vec<TX, TY, TO, 4, HASY, true>(a, st) : launch_vec<TX, TY, TO, 4, HASY, false>(a, st);
  return launch_vec<TX, TY, TO, 1, HASY, false>(a, st);
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
