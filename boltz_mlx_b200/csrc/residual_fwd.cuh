// LayerNorm forward, alone or behind dropout + residual add, and the add without the norm (residual.cuh has the formulas).
//
// Bound by HBM: one read of every input and one write of every output.  A group's next batches of R rows are on their way
// into shared memory (residual.cuh) while it works on one: with one load in flight for each lane instead, 121 us for 2^20
// rows of 128 bf16, so 84 us.  A row's values stay in registers through both statistics passes (mean, then centred
// squares), as pairs, of which one instruction handles two.
// 2^20 rows of 128: fp32 -> bf16 119 us (1.02 of the copy rate), read transposed 129 us, bf16 84 us, fp32 163 us; with the add
// and one draw per row 262 us, less than a pass that reads every update needs (286; 266 with the kept ones alone); with a
// draw per element 327 us: a draw is 20 multiplications of 32 x 32 bits for four elements, at a quarter of the rate of others.
// On 16-bit streams they show: 16384 rows of 1024 bf16, dropout and add 27 us (floor 15), the multipliers busy 64 % of the
// launch, issue slots 56 %, DRAM 31 %; fused, 8198 rows of 1024 fp16, 18 us (floor 10), 53 / 54 / 20 % at 15 warps an SM.
// 2^25 bf16 in rows of 1024, 2048, 4096, 8192: 24, 25, 27, 30 us (0.84, 0.82, 0.75, 0.68), of which about 5 are the launch,
// the parameters and the first rows' way.
#pragma once
#include "residual.cuh"

namespace triattn {
namespace {

// what a kernel does: LayerNorm; dropout, add and LayerNorm; dropout and add; dropout
enum Does { kNorm, kFused, kAdd, kDrop };

template <class TX, class TY, int VEC, int NCH, int R, Does DO>
constexpr int fwd_stage_bytes(int width, int dim) {
  return R * ((DO != kDrop ? row_slot<TX, VEC, NCH>(width, dim) : 0) + (DO != kNorm ? row_slot<TY, VEC, NCH>(width, dim) : 0));
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, Does DO, bool DENSE>
__global__ void __launch_bounds__(LPR ? 256 : 512) norm_fwd_kernel(const NormFwdArgs a, int width, Split split) {
  using L = Lanes<VEC, LPR, NCH>;
  constexpr int P = L::PAIRS;
  constexpr bool HASX = DO != kDrop, HASY = DO != kNorm, NORM = DO == kNorm || DO == kFused;
  extern __shared__ __align__(16) char smem[];  // LPR: weight and bias in fp32, then the groups' stages
  __shared__ __align__(16) float red[L::red_floats];
  int phase = 0;
  const L l(a.dim, width);
  const int D = a.dim;
  const float inv_d = 1.0f / (float)D;

  // Rows of several warps keep weight and bias in registers, rows of one warp (several at once) in shared memory.
  float* wb = reinterpret_cast<float*>(smem);
  const int wb_pad = NORM && LPR ? L::EPL * LPR : 0;  // zeros behind dim
  Pair w[LPR ? 1 : P], b[LPR ? 1 : P];
  if constexpr (!NORM) {
  } else if constexpr (LPR) {
    for (int i = threadIdx.x; i < wb_pad; i += blockDim.x) {
      wb[i] = i < D ? load_param(a.weight, a.param_dtype, i, 1.0f) : 0.0f;
      wb[wb_pad + i] = i < D ? load_param(a.bias, a.param_dtype, i, 0.0f) : 0.0f;
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
  const int stage = fwd_stage_bytes<TX, TY, VEC, NCH, R, DO>(l.width, D);
  char* ring = smem + wb_pad * 8 + l.group * S * stage;
  const RowIn<TX, VEC, LPR, NCH, DENSE> z(l, a.z, a.zs, ring);
  const RowIn<TY, VEC, LPR, NCH, DENSE> y(l, a.y, a.ys, ring + (HASX ? R * slot_x : 0));
  const RowOut<TX, VEC, LPR, NCH, DENSE> sum(l, a.sum, a.ss);
  const RowOut<TO, VEC, LPR, NCH, DENSE> out(l, a.out, a.os);
  for (int k = 0; k < S; ++k) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (HASX) z.clear(k * stage + r * slot_x);
      if (HASY) y.clear(k * stage + r * slot_y);
    }
  }
  uint32_t kept = ~0u;  // bit s * R + r: row r of stage s is not dropped whole

  const RowMap& map = a.map;
  const uint32_t step = l.groups * R;
  using Rows = Batch<DENSE, R>;
  const auto issue = [&](uint32_t base, int s) {
    const Rows batch(l, map, base + l.group * R);
    TX* pz[R];
    TY* py[R];
    if constexpr (HASX) z.rows.at(batch, pz);
    if constexpr (HASY) y.rows.at(batch, py);
    if constexpr (HASY) {
      if (row_draw) {
        // one draw per row: lane r of a group takes that of row r, and hands it round
        const uint32_t mine = batch.first + (LPR ? l.lane & (R - 1) : 0);
        const bool k = rng.word(mask_base(a.drop, map.at(mine))) > a.drop.drop_max;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint32_t bit = 1u << (s * R + r);
          kept = (R > 1 ? __shfl_sync(0xffffffffu, (int)k, r, LPR ? LPR : 32) : (int)k) ? kept | bit : kept & ~bit;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!batch.live(r)) continue;
      // of a row that is dropped whole, y is not read, nor, in place, z
      const bool keep = !HASY || (kept >> (s * R + r) & 1);
      if constexpr (HASX)
        if (keep || !(DO == kAdd && a.in_place)) z.issue(s * stage + r * slot_x, pz[r]);
      if constexpr (HASY)
        if (keep) y.issue(s * stage + r * slot_y, py[r]);
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
    const Rows batch(l, map, base + l.group * R);
    TX *pz[R], *ps[R];
    TY* py[R];
    if constexpr (HASX && VEC == 1) z.rows.at(batch, pz);
    if constexpr (HASY && VEC == 1) y.rows.at(batch, py);
    if constexpr (HASY) sum.rows.at(batch, ps);
    // Rows behind the last one are computed from what their slot holds, and not stored.
    Pair x[R][P];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if constexpr (HASX) {
        z.read(s * stage + r * slot_x, VEC == 1 ? pz[r] : nullptr, x[r]);
      } else {
#pragma unroll
        for (int j = 0; j < P; ++j) x[r][j] = both(0.0f);
      }
      if constexpr (HASY) {
        const bool whole = kept >> (s * R + r) & 1;
        if (whole) {
          Pair v[P];
          y.read(s * stage + r * slot_y, VEC == 1 ? py[r] : nullptr, v);
          if (draw) {
            each_kept(l, rng, mask_base(a.drop, map.at(batch.row(r))), a.drop.drop_max, [&](bool k, int i) {
              const float2 xi = halves(x[r][i / 2]), vi = halves(v[i / 2]);
              const float f = i & 1 ? xi.y : xi.x, g = k ? fmaf(i & 1 ? vi.y : vi.x, a.drop.scale, f) : f;
              x[r][i / 2] = i & 1 ? pair(xi.x, g) : pair(g, xi.y);
            });
          } else {
#pragma unroll
            for (int j = 0; j < P; ++j) x[r][j] = fma2(v[j], scale, x[r][j]);
          }
        }
        if constexpr (NORM && sizeof(TX) == 2) {  // the norm is taken of the stream as it is held
#pragma unroll
          for (int j = 0; j < P; ++j) {
            TX held[2];
            from_pair(x[r][j], held);
            x[r][j] = to_pair(held);
          }
        }
        if (batch.live(r) && (whole || !(DO == kAdd && a.in_place))) sum.row(ps[r], x[r]);
      }
    }
    l.sync();

    if constexpr (NORM) {
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
          if (batch.live(r)) {
            a.mean[batch.row(r)] = mean[r];
            a.rstd[batch.row(r)] = var[r];
          }
      }
      TO* po[R];
      out.rows.at(batch, po);
      constexpr int STEP = VEC == 1 && NCH > 1 ? 2 : 1;  // pieces of a pair
#pragma unroll
      for (int c = 0; c < NCH; c += STEP) {
        constexpr int N = VEC > 1 ? VEC / 2 : 1;
        Pair wc[N], bc[N];
        if constexpr (LPR) {
          if constexpr (VEC > 1) {
#pragma unroll
            for (int j = 0; j < N; j += 2) {
              const Pack<float, 4> wq = load_pack<float, 4>(wb + l.col(c) + 2 * j);
              const Pack<float, 4> bq = load_pack<float, 4>(wb + wb_pad + l.col(c) + 2 * j);
              wc[j] = pair(wq.v[0], wq.v[1]), wc[j + 1] = pair(wq.v[2], wq.v[3]);
              bc[j] = pair(bq.v[0], bq.v[1]), bc[j + 1] = pair(bq.v[2], bq.v[3]);
            }
          } else {
            const int c1 = l.col(c + STEP - 1);
            wc[0] = pair(wb[l.col(c)], wb[c1]);
            bc[0] = pair(wb[wb_pad + l.col(c)], wb[wb_pad + c1]);
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
          if (batch.live(r)) {
#pragma unroll
            for (int k = 0; k < STEP; ++k)
              if (c + k < NCH) out.piece(po[r], c + k, x[r]);
          }
        }
      }
    }
    s = s == S - 1 ? 0 : s + 1;
  }
  copy_wait<0>();
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, Does DO, bool DENSE>
cudaError_t fwd_one(const NormFwdArgs& a, int width, int threads, cudaStream_t st) {
  static KernelInfo info;
  if (!pieces_fit<VEC, NCH>(a.dim, width)) return cudaErrorInvalidConfiguration;
  const int groups = threads / width, wb = DO == kNorm || DO == kFused ? LPR * VEC * NCH * 8 : 0;
  const size_t smem = wb + (size_t)groups * S * fwd_stage_bytes<TX, TY, VEC, NCH, R, DO>(width, a.dim);
  int fit = 0;
  if (cudaError_t e = info.fit(norm_fwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, S, DO, DENSE>, threads, smem, &fit);
      e != cudaSuccess)
    return e;
  // Many CTAs of few batches: they are handed to the SMs as these come free.  An equal share for every resident
  // CTA leaves the SMs that the memory system serves last working alone at the end (0.82 of the copy rate
  // instead of 0.98 at 2^20 rows of 128 fp32).  A CTA has to load weight and bias, though, so that long rows
  // want more batches, in 16 bits (half the traffic a row) most.  2^25 elements in rows of 1024, 2048, 4096 and 8192, 16
  // batches a CTA against 4: bf16 24.3, 24.8, 26.8 and 29.7 us against 27.2, 27.7, 30.2 and 34.5; fp32 49.0, 50.2, 51.4 and
  // 52.8 against 43.9, 44.3, 45.1 and 46.8.
  const uint32_t per = groups * R, batches = (a.map.rows + per - 1) / per;
  const uint32_t resident = (uint32_t)(device_sm_count() * fit);
  uint32_t few = (batches + resident - 1) / resident;
  constexpr uint32_t most = LPR ? 5 : VEC == 8 ? 16 : 4;
  if (few > most) few = most;
  norm_fwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, S, DO, DENSE><<<(batches + few - 1) / few, threads, smem, st>>>(
      a, width, Split{0, 0, few, batches});
  return cudaGetLastError();
}

template <class TX, class TY, class TO, int VEC, Does DO, bool DENSE>
cudaError_t fwd_vec(const NormFwdArgs& a, cudaStream_t st) {
  const int C = (a.dim + VEC - 1) / VEC;
#define LAUNCH(LPR, NCH, R, S, WIDTH, THREADS) \
  return fwd_one<TX, TY, TO, VEC, LPR, NCH, R, S, DO, DENSE>(a, WIDTH, THREADS, st)
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
    // Odd widths: as many rows to a warp as leave its lanes few empty pieces (2^25 fp16 elements: rows of 6, 13, 31 and 63
    // channels 185, 99, 56 and 54 us, against 804, 373, 159 and 103 with one row to a warp).
    if (C <= 8) LAUNCH(8, 1, 4, 2, 8, 256);
    if (C <= 16) LAUNCH(8, 2, 4, 2, 8, 256);
    if (C <= 32) LAUNCH(8, 4, 2, 2, 8, 256);
    if (C <= 64) LAUNCH(16, 4, 2, 2, 16, 256);
    if (C <= 128) LAUNCH(32, 4, 2, 2, 32, 256);
    if (C <= 256) LAUNCH(32, 8, 1, 3, 32, 256);
    if (C <= 384) LAUNCH(32, 12, 1, 3, 32, 256);
    if (C <= 512) LAUNCH(32, 16, 1, 3, 32, 256);
  }
  const RowWidth w = row_width<VEC>(C, 256);
  if constexpr (VEC == 4) {
    if (w.pieces == 2) LAUNCH(0, 2, 1, 3, w.width, w.threads);
    if (w.pieces == 3) LAUNCH(0, 3, 1, 3, w.width, w.threads);
  }
  if constexpr (VEC == 1)
    if (w.pieces == 12) LAUNCH(0, 12, 1, 3, w.width, w.threads);
  LAUNCH(0, 16 / VEC, 1, 3, w.width, w.threads);
#undef LAUNCH
}

template <class TX, class TY, class TO, Does DO>
cudaError_t fwd_types(const NormFwdArgs& a, int vec, cudaStream_t st) {
  const bool dense = a.zs.dense && a.os.dense && (DO == kNorm || (a.ys.dense && a.ss.dense));
  constexpr int FULL = sizeof(TX) == 2 && sizeof(TY) == 2 && sizeof(TO) == 2 ? 8 : 4;
  if (vec >= FULL) return dense ? fwd_vec<TX, TY, TO, FULL, DO, true>(a, st) : fwd_vec<TX, TY, TO, FULL, DO, false>(a, st);
  // 16-bit rows of whole pieces of four (2^25 bf16 elements: rows of 60, 100 and 1004 channels 29, 36 and 29 us, read one by
  // one 55, 67 and 48; backward 51, 54 and 42 against 86, 104 and 54)
  if constexpr (FULL == 8)
    if (vec == 4) return dense ? fwd_vec<TX, TY, TO, 4, DO, true>(a, st) : fwd_vec<TX, TY, TO, 4, DO, false>(a, st);
  return dense ? fwd_vec<TX, TY, TO, 1, DO, true>(a, st) : fwd_vec<TX, TY, TO, 1, DO, false>(a, st);
}

}  // namespace
}  // namespace triattn
