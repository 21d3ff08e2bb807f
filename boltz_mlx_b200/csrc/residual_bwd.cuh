// LayerNorm backward, alone or with the gradients of the residual add and the dropout in front of it:
//
//   xh = (x - mean) rstd,  g = dout w
//   dx = rstd (g - mean_c(g) - xh mean_c(g xh)) (+ ds),  dy = keep ? dx scale : 0
//   dweight = sum_rows dout xh,  dbias = sum_rows dout
//
// Bound by HBM like the forward pass: x, dout (and ds) are read once, dx (and dy) written once; x and dout are brought
// in as the forward pass brings in its rows (residual.cuh).  A lane owns the same channels in every row that its group
// handles, so the two column sums stay in its registers until the CTA has seen its last row; they are then joined in
// shared memory, written as one partial row per CTA and summed by a second small kernel in the order of the CTAs: no
// atomics, the same bits on every run.
// 2^20 rows of 128, fp32 <- bf16: 211 us, 6.4 TB/s (0.97 of the copy rate); bf16: 128 us (0.95); with ds and dy, 768^2 rows:
// 212 us (0.97).  2^25 bf16 in rows of 1024, 2048, 4096 and 8192: 39, 42, 44 and 47 us (0.78, 0.73, 0.70 and 0.66): latency
// at 16 warps an SM, whose registers hold the column sums; nothing is full (8192 rows of 4096: DRAM 50 %, issue slots 56 %,
// multipliers 43 %), and up to 10 MB of partial sums are written and read.
#pragma once
#include <cooperative_groups.h>

#include "residual.cuh"

namespace triattn {
namespace {

constexpr int kCtasPerSm = 4;  // resident at most
constexpr int kPartials = 4;   // CTAs of a launch at most, times those

template <class TX, class TO, int VEC, int NCH, int R, bool HASY>
constexpr int bwd_stage_bytes(int width, int dim) {
  return R * ((HASY ? 2 : 1) * row_slot<TX, VEC, NCH>(width, dim) + row_slot<TO, VEC, NCH>(width, dim));
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, bool HASY, bool DENSE>
__global__ void __launch_bounds__(LPR ? 256 : 512) norm_bwd_kernel(const NormBwdArgs a, int width, Split split) {
  using L = Lanes<VEC, LPR, NCH>;
  constexpr int P = L::PAIRS;
  extern __shared__ __align__(16) char smem[];  // the groups' stages; at the end [groups][2][dim] column sums
  __shared__ __align__(16) float red[L::red_floats];
  int phase = 0;
  const L l(a.dim, width);
  const int D = a.dim;
  const float inv_d = 1.0f / (float)D;

  Pair w[P], dw[P], db[P];
  load_pairs(l, a.weight, a.param_dtype, 1.0f, w);
#pragma unroll
  for (int j = 0; j < P; ++j) dw[j] = db[j] = both(0.0f);
  l.clear(red);
  const Philox rng(a.drop);
  const bool has_ds = HASY && a.ds, has_dy = HASY && a.dy;
  const bool row_draw = has_dy && a.drop.on && !a.drop.per_channel, draw = has_dy && a.drop.on && a.drop.per_channel;

  const int slot_x = row_slot<TX, VEC, NCH>(l.width, D), slot_o = row_slot<TO, VEC, NCH>(l.width, D);
  const int stage = bwd_stage_bytes<TX, TO, VEC, NCH, R, HASY>(l.width, D);
  char* ring = smem + l.group * S * stage;
  const RowIn<TX, VEC, LPR, NCH, DENSE> x(l, a.x, a.xs, ring), ds(l, a.ds, a.dss, ring + R * (slot_x + slot_o));
  const RowIn<TO, VEC, LPR, NCH, DENSE> dout(l, a.dout, a.dos, ring + R * slot_x);
  const RowOut<TX, VEC, LPR, NCH, true> dx(l, a.dx, a.xs);
  const RowOut<TY, VEC, LPR, NCH, true> dy(l, a.dy, a.xs);
  for (int k = 0; k < S; ++k) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      x.clear(k * stage + r * slot_x);
      dout.clear(k * stage + r * slot_o);
      if (HASY) ds.clear(k * stage + r * slot_x);
    }
  }

  const RowMap& map = a.map;
  const uint32_t step = l.groups * R;
  using Rows = Batch<DENSE, R>;
  const auto issue = [&](uint32_t base, int s) {
    const Rows batch(l, map, base + l.group * R);
    TX *px[R], *ps[R];
    TO* po[R];
    x.rows.at(batch, px);
    dout.rows.at(batch, po);
    if constexpr (HASY) ds.rows.at(batch, ps);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!batch.live(r)) {  // adds nothing to the column sums
        x.issue_none(s * stage + r * slot_x);
        dout.issue_none(s * stage + r * slot_o);
        continue;
      }
      x.issue(s * stage + r * slot_x, px[r]);
      dout.issue(s * stage + r * slot_o, po[r]);
      if constexpr (HASY)
        if (has_ds) ds.issue(s * stage + r * slot_x, ps[r]);
    }
  };
  float mean_next[R], rstd_next[R];  // of the next batch
  const auto statistics = [&](uint32_t base) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t row = base + l.group * R + r;
      mean_next[r] = row < map.rows ? a.mean[row] : 0.0f;
      rstd_next[r] = row < map.rows ? a.rstd[row] : 0.0f;
    }
  };

  uint32_t first, end;  // rows of this CTA
  split.range(blockIdx.x, first, end);
  first *= step;
  end *= step;
  uint32_t ahead = first;
  statistics(ahead);
#pragma unroll
  for (int s = 0; s < S - 1; ++s, ahead += step) {
    if (ahead < end) issue(ahead, s);
    copy_commit();
  }
  int s = 0;
  for (uint32_t base = first; base < end; base += step, ahead += step) {
    if (ahead < end) issue(ahead, s == 0 ? S - 1 : s - 1);
    copy_commit();
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = mean_next[r];
      rstd[r] = rstd_next[r];
    }
    statistics(base + step);
    copy_wait<S - 1>();
    l.sync();
    const Rows batch(l, map, base + l.group * R);
    TX *px[R], *ps[R];
    TO* po[R];
    if constexpr (VEC == 1) {
      x.rows.at(batch, px);
      dout.rows.at(batch, po);
      if constexpr (HASY) ds.rows.at(batch, ps);
    }
    // v[2 r] = sum g, v[2 r + 1] = sum g xh
    Pair xh[R][P], g[R][P];
    float v[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      x.read(s * stage + r * slot_x, VEC == 1 ? px[r] : nullptr, xh[r]);
      dout.read(s * stage + r * slot_o, VEC == 1 ? po[r] : nullptr, g[r]);
      const Pair q = both(rstd[r]), m = both(-mean[r]);
      Pair s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        // centred before it is scaled, as in the forward pass: mean * rstd would be rounded at the size of a row far from
        // zero.  Where there is no channel, dout and the weight are zero.
        xh[r][j] = (xh[r][j] + m) * q;
        dw[j] = fma2(g[r][j], xh[r][j], dw[j]);
        db[j] = db[j] + g[r][j];
        g[r][j] = g[r][j] * w[j];
        s1 = s1 + g[r][j];
        s2 = fma2(g[r][j], xh[r][j], s2);
      }
      v[2 * r] = total(s1);
      v[2 * r + 1] = total(s2);
    }
    l.sum(v, red, phase);
    TX* pdx[R];
    TY* pdy[R];
    const Batch<true, R> written(l, map, batch.first);
    dx.rows.at(written, pdx);
    dy.rows.at(written, pdy);
    uint32_t whole = ~0u;  // bit r: row r is not dropped whole
    if constexpr (HASY) {
      if (row_draw) {
        const uint32_t mine = batch.first + (LPR ? l.lane & (R - 1) : 0);
        const bool k = rng.word(mask_base(a.drop, map.at(mine))) > a.drop.drop_max;
        whole = 0;
#pragma unroll
        for (int r = 0; r < R; ++r)
          whole |= (R > 1 ? __shfl_sync(0xffffffffu, (uint32_t)k, r, LPR ? LPR : 32) : (uint32_t)k) << r;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = batch.live(r);
      const float t = -inv_d * rstd[r];
      const Pair c1 = both(v[2 * r] * t), c2 = both(v[2 * r + 1] * t), q = both(rstd[r]);
#pragma unroll
      for (int j = 0; j < P; ++j) g[r][j] = fma2(g[r][j], q, fma2(xh[r][j], c2, c1));
      if constexpr (HASY) {
        if (has_ds) {
          Pair sv[P];
          ds.read(s * stage + r * slot_x, VEC == 1 ? ps[r] : nullptr, sv);
#pragma unroll
          for (int j = 0; j < P; ++j) g[r][j] = g[r][j] + sv[j];
        }
      }
      if (a.dx && live) dx.row(pdx[r], g[r]);
      if constexpr (HASY) {
        if (has_dy) {
          if (draw) {
            each_kept(l, rng, mask_base(a.drop, map.at(batch.row(r))), a.drop.drop_max, [&](bool k, int i) {
              const float2 gi = halves(g[r][i / 2]);
              const float f = k ? (i & 1 ? gi.y : gi.x) * a.drop.scale : 0.0f;
              g[r][i / 2] = i & 1 ? pair(gi.x, f) : pair(f, gi.y);
            });
          } else {
            const Pair scale = both(a.drop.scale);
#pragma unroll
            for (int j = 0; j < P; ++j) g[r][j] = whole >> r & 1 ? g[r][j] * scale : both(0.0f);
          }
          if (live) dy.row(pdy[r], g[r]);
        }
      }
    }
    l.sync();
    s = s == S - 1 ? 0 : s + 1;
  }
  copy_wait<0>();

  if (!a.partial) return;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining kernel may take its places and wait
  // groups of one warp first (they own the same channels), then all groups through shared memory
#pragma unroll
  for (int o = LPR ? LPR : 32; o < 32; o <<= 1) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      dw[j] = dw[j] + Pair{__shfl_xor_sync(0xffffffffu, dw[j].v, o)};
      db[j] = db[j] + Pair{__shfl_xor_sync(0xffffffffu, db[j].v, o)};
    }
  }
  const int sets = LPR ? blockDim.x >> 5 : l.groups;
  float* sums = reinterpret_cast<float*>(smem);
  float* mine = sums + (size_t)(LPR ? threadIdx.x >> 5 : l.group) * 2 * D;
  __syncthreads();  // every warp has read its last rows
  if (!LPR || (threadIdx.x & 31) < LPR) {
#pragma unroll
    for (int i = 0; i < L::EPL; ++i) {
      if (!l.act(i / VEC)) continue;
      const float2 u = halves(dw[i / 2]), t = halves(db[i / 2]);
      mine[l.col(i / VEC) + i % VEC] = i & 1 ? u.y : u.x;
      mine[D + l.col(i / VEC) + i % VEC] = i & 1 ? t.y : t.x;
    }
  }
  __syncthreads();
  float* part = a.partial + (size_t)blockIdx.x * 2 * D;
  for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) {
    float t = 0.0f;
    for (int k = 0; k < sets; ++k) t += sums[(size_t)k * 2 * D + i];
    if (gridDim.x > 1) {
      part[i] = t;
    } else {  // the only CTA's sums are the gradients
      void* grad = i < D ? a.dweight : a.dbias;
      const int c = i < D ? i : i - D;
      if (!grad) continue;
      if (a.param_dtype == DT_F32)
        static_cast<float*>(grad)[c] = t;
      else if (a.param_dtype == DT_F16)
        static_cast<__half*>(grad)[c] = from_f32<__half>(t);
      else
        static_cast<__nv_bfloat16*>(grad)[c] = from_f32<__nv_bfloat16>(t);
    }
  }
}

// A value that another kernel wrote while this one was already there: from L2, and not before what stands in front of it.
__device__ __forceinline__ float ld_written(const float* p) {
  float v;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}

// Column sums of the CTAs' partial rows: a cluster of kJoin CTAs for 32 columns, each of its warps with every
// 16 * kJoin-th row; the cluster's first CTA adds up what the others hold in their shared memory.  One CTA
// alone needs 15 us for the 2000 partial rows of a long launch, a cluster of eight 3; for the few partial rows
// of a short launch, or the many columns of long rows, one is enough.
// The kernel is launched while the rows are still written, so that `partial` is not read-only while it lives: no const
// __restrict__, and loads that go to L2, behind the wait.
template <class TP, int kJoin>
__global__ void __cluster_dims__(kJoin, 1, 1) __launch_bounds__(512)
    norm_bwd_join_kernel(float* partial, int ctas, int dim, TP* dweight, TP* dbias) {
  namespace cg = cooperative_groups;
  __shared__ float part[16][33];
  __shared__ float sum[32];
  const auto cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x / kJoin * 32 + lane;  // of 2 * dim
  float s = 0.0f;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // all partial rows are written
  if (col < 2 * dim) {
#pragma unroll 8
    for (int i = rank * 16 + warp; i < ctas; i += 16 * kJoin) s += ld_written(partial + (size_t)i * 2 * dim + col);
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += part[i][lane];
    sum[lane] = s;
  }
  cluster.sync();
  if (rank == 0 && warp == 0 && col < 2 * dim) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) s += *cluster.map_shared_rank(&sum[lane], i);
    if (col < dim) {
      if (dweight) dweight[col] = from_f32<TP>(s);
    } else if (dbias) {
      dbias[col - dim] = from_f32<TP>(s);
    }
  }
  cluster.sync();  // no CTA leaves while its sums are read
}

template <class TP>
cudaError_t launch_join(const NormBwdArgs& a, int ctas, cudaStream_t st) {
  const int blocks = (2 * a.dim + 31) / 32;
  TP *dw = static_cast<TP*>(a.dweight), *db = static_cast<TP*>(a.dbias);
  const int size = ctas > 320 && blocks <= 64 ? 8 : 1;
  // launched while the last CTAs that write partial rows still run (a pass of 48 us becomes one of 47)
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(blocks * size);
  c.blockDim = dim3(512);
  c.stream = st;
  c.attrs = &early;
  c.numAttrs = 1;
  float* partial = a.partial;
  if (size == 8) return cudaLaunchKernelEx(&c, norm_bwd_join_kernel<TP, 8>, partial, ctas, (int)a.dim, dw, db);
  return cudaLaunchKernelEx(&c, norm_bwd_join_kernel<TP, 1>, partial, ctas, (int)a.dim, dw, db);
}

// Three quarters of the batches go to the CTAs that are resident from the start, in equal shares; the rest in
// shares an eighth as large, to whichever SM comes free: equal shares alone leave the SMs that the memory
// system serves last working alone at the end (0.82 of the copy rate instead of 0.97 at 2^20 rows of 128).  Every CTA
// costs a partial row of 16 bytes a channel (written and read), so a share has kRows rows at least, or there is one
// kind of CTA only.  What a CTA adds up goes by its index, not by when it runs.
constexpr uint32_t kRows = 64;
constexpr uint32_t kAlone = 4;  // so few batches one CTA works off alone, and needs no second kernel to add up
Split share(uint32_t batches, uint32_t resident, uint32_t per) {
  if (batches <= kAlone) return Split{1, batches, 0, batches};
  Split s{resident, batches / 4 * 3 / resident, 0, batches};
  const uint32_t rest = batches - resident * s.many, most = (kPartials - 1) * resident;  // short shares, at most
  const auto up = [](uint32_t a, uint32_t b) { return (a + b - 1) / b; };
  s.few = s.many / 8;
  if (s.few * per < kRows) s.few = up(kRows, per);
  if (s.few < up(rest, most)) s.few = up(rest, most);
  if (s.few * 2 > s.many) {
    s.many = up(batches, resident);
    s.big = up(batches, s.many);
    s.few = 0;
  }
  return s;
}

template <class TX, class TY, class TO, int VEC, int LPR, int NCH, int R, int S, bool HASY, bool DENSE>
cudaError_t bwd_one(const NormBwdArgs& a, int width, int threads, cudaStream_t st) {
  static KernelInfo info;
  if (!pieces_fit<VEC, NCH>(a.dim, width)) return cudaErrorInvalidConfiguration;
  const int groups = threads / width, sets = LPR ? threads / 32 : groups;
  size_t smem = (size_t)groups * S * bwd_stage_bytes<TX, TO, VEC, NCH, R, HASY>(width, a.dim);
  if (const size_t sums = (size_t)sets * 2 * a.dim * 4; smem < sums) smem = sums;
  int fit = 0;
  if (cudaError_t e = info.fit(norm_bwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, S, HASY, DENSE>, threads, smem, &fit);
      e != cudaSuccess)
    return e;
  if (fit > kCtasPerSm) fit = kCtasPerSm;
  const uint32_t per = groups * R, batches = (a.map.rows + per - 1) / per;
  const Split split = share(batches, (uint32_t)(device_sm_count() * fit), per);
  const uint32_t grid = split.big + (split.few ? (batches - split.big * split.many + split.few - 1) / split.few : 0);
  if (grid > (uint32_t)norm_bwd_max_ctas()) return cudaErrorInvalidConfiguration;  // the partial sums have no room for more
  norm_bwd_kernel<TX, TY, TO, VEC, LPR, NCH, R, S, HASY, DENSE><<<grid, threads, smem, st>>>(a, width, split);
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess || !a.partial || grid == 1) return e;
  if (a.param_dtype == DT_F32) return launch_join<float>(a, (int)grid, st);
  if (a.param_dtype == DT_F16) return launch_join<__half>(a, (int)grid, st);
  return launch_join<__nv_bfloat16>(a, (int)grid, st);
}

template <class TX, class TY, class TO, int VEC, bool HASY, bool DENSE>
cudaError_t bwd_vec(const NormBwdArgs& a, cudaStream_t st) {
  const int C = (a.dim + VEC - 1) / VEC;
#define LAUNCH(LPR, NCH, R, S, WIDTH, THREADS) \
  return bwd_one<TX, TY, TO, VEC, LPR, NCH, R, S, HASY, DENSE>(a, WIDTH, THREADS, st)
  if constexpr (VEC > 1) {
    if (C <= 8) LAUNCH(8, 1, 4, 2, 8, 256);
    if (C <= 16) LAUNCH(16, 1, 4, 2, 16, 256);
    if (C <= 32) LAUNCH(32, 1, 16 / VEC, 2, 32, 256);
    if (C <= 64) LAUNCH(32, 2, 2, 2, 32, 256);
    if constexpr (VEC == 4) {
      if (C <= 96) LAUNCH(32, 3, 1, 3, 32, 256);
      if (C <= 128) LAUNCH(32, 4, 1, 3, 32, 256);
    }
  } else {
    // Several narrow rows to a warp, as in the forward pass (2^25 fp16 elements: rows of 6, 13, 31 and 63 channels 361, 183, 96
    // and 84 us, against 1328, 616, 266 and 156 with one row to a warp).
    if (C <= 8) LAUNCH(8, 1, 4, 2, 8, 256);
    if (C <= 16) LAUNCH(8, 2, 4, 2, 8, 256);
    if (C <= 32) LAUNCH(8, 4, 2, 2, 8, 256);
    if (C <= 64) LAUNCH(16, 4, 2, 2, 16, 256);
    if (C <= 128) LAUNCH(32, 4, 2, 2, 32, 256);
    if (C <= 256) LAUNCH(32, 8, 1, 3, 32, 256);
    if (C <= 384) LAUNCH(32, 12, 1, 3, 32, 256);
    if (C <= 512) LAUNCH(32, 16, 1, 3, 32, 256);
  }
  // Long rows: one CTA of 512 threads on an SM leaves half the partial sums that two of 256 do.  2^25 elements in rows of
  // 2560, 4096 and 8192, 512 against 256: bf16 42.3, 44.0 and 46.5 us against 46.7, 45.1 and 46.5, fp32 70.3, 72.5 and 73.7
  // against 74.5, 74.6 and 73.8; of 1024, 1536 and 2048: bf16 44.9, 40.1 and 40.6 against 39.5, 42.1 and 42.1, fp32 68.3, 67.4
  // and 71.1 against 71.1, 67.3 and 73.0.
  const RowWidth w = row_width<VEC>(C, C * VEC > 2048 ? 512 : 256);
  if constexpr (VEC == 4) {
    if (w.pieces == 2) LAUNCH(0, 2, 1, 2, w.width, w.threads);
    if (w.pieces == 3) LAUNCH(0, 3, 1, 2, w.width, w.threads);
  }
  if constexpr (VEC == 1)
    if (w.pieces == 12) LAUNCH(0, 12, 1, 2, w.width, w.threads);
  LAUNCH(0, 16 / VEC, 1, VEC == 8 ? 3 : 2, w.width, w.threads);
#undef LAUNCH
}

template <class TX, class TY, class TO, bool HASY>
cudaError_t bwd_types(const NormBwdArgs& a, int vec, cudaStream_t st) {
  const bool dense = a.xs.dense && a.dos.dense && (!HASY || !a.ds || a.dss.dense);
  constexpr int FULL = sizeof(TX) == 2 && sizeof(TY) == 2 && sizeof(TO) == 2 ? 8 : 4;
  if (vec >= FULL) return dense ? bwd_vec<TX, TY, TO, FULL, HASY, true>(a, st) : bwd_vec<TX, TY, TO, FULL, HASY, false>(a, st);
  if constexpr (FULL == 8)
    if (vec == 4) return dense ? bwd_vec<TX, TY, TO, 4, HASY, true>(a, st) : bwd_vec<TX, TY, TO, 4, HASY, false>(a, st);
  return dense ? bwd_vec<TX, TY, TO, 1, HASY, true>(a, st) : bwd_vec<TX, TY, TO, 1, HASY, false>(a, st);
}

}  // namespace
}  // namespace triattn
