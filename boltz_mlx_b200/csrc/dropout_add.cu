// Dropout and dropout + residual add: out = (z ? z : 0) + (keep ? y * scale : 0), residual.cuh's mask.
//
// Bound by HBM: z and y read once, out written once; a draw costs about 50 instructions for four
// positions, which the loads cover.  A thread handles chunks of VEC consecutive elements, kUnroll of them
// in flight.  FLAT: every tensor is dense, so a chunk is VEC consecutive elements of the whole tensor,
// whatever dim is, and its elements may lie in two rows (or more, for dim < VEC); else a chunk lies in
// one row.
#include "residual.cuh"

namespace triattn {
namespace {

constexpr int kThreads = 256, kUnroll = 4;

// position of the mask of element (row, col)
__device__ __forceinline__ uint64_t mask_pos(const DropoutAddArgs& a, uint32_t row, uint32_t col) {
  return mask_base(a.drop, a.map.at(row)) + (a.drop.per_channel ? col : 0);
}

template <class T, int VEC>
__device__ __forceinline__ void load_some(Pack<T, VEC>& r, const T* p, int n) {
  if (VEC == 1 || n == VEC) {
    r = load_pack<T, VEC>(p);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (k < n) r.v[k] = p[k];
  }
}

template <class TZ, class TY, class TO, int VEC, bool FLAT, bool HASZ>
__global__ void __launch_bounds__(kThreads) dropout_add_kernel(const DropoutAddArgs a, FastDiv per_row,
                                                               uint64_t elements) {
  const TZ* z = static_cast<const TZ*>(a.z);
  const TY* y = static_cast<const TY*>(a.y);
  TO* out = static_cast<TO*>(a.out);
  const uint32_t D = (uint32_t)a.dim;
  const Philox rng(a.drop);
  const uint64_t chunks = FLAT ? (elements + VEC - 1) / VEC : elements / VEC;
  const uint64_t tiles = (chunks + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  const bool whole_rows = a.drop.on && !a.drop.per_channel;
  const bool linear = a.drop.m[2] == (int64_t)D && a.drop.m[1] == (int64_t)D * a.map.n2.d &&
                      a.drop.m[0] == (int64_t)D * a.map.n2.d * a.map.n1.d;  // every element has its own position
  for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const uint64_t first = tile * (kThreads * kUnroll);  // chunk
    // first row of the tile and the place in it (elements if FLAT, chunks if not)
    const uint64_t at0 = FLAT ? first * VEC : first;
    const uint32_t row_base = (uint32_t)(at0 / per_row.d), rest = (uint32_t)(at0 - (uint64_t)row_base * per_row.d);
    Pack<TZ, VEC> zr[kUnroll];
    Pack<TY, VEC> yr[kUnroll];
    uint32_t bits[kUnroll];
    int64_t oo[kUnroll];
    int n[kUnroll];  // elements of the chunk
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t q = u * kThreads + threadIdx.x;
      const bool live = first + q < chunks;
      n[u] = 0;
      bits[u] = VEC == 8 ? 0xffu : (1u << VEC) - 1u;
      if (!live) continue;
      n[u] = VEC;
      int64_t zo, yo;
      uint32_t row, col;
      if constexpr (FLAT) {
        const uint64_t e = (first + q) * VEC;
        if (elements - e < VEC) n[u] = (int)(elements - e);
        const uint32_t t = rest + q * VEC, dr = per_row.div(t);
        row = row_base + dr;
        col = t - dr * D;
        zo = yo = oo[u] = (int64_t)e;
      } else {
        const uint32_t t = rest + q, dr = per_row.div(t);
        row = row_base + dr;
        col = (t - dr * per_row.d) * VEC;
        zo = row_offset(a.zs, row, a.map, D) + col;
        yo = row_offset(a.ys, row, a.map, D) + col;
        oo[u] = row_offset(a.os, row, a.map, D) + col;
      }
      if (HASZ && !a.in_place) load_some(zr[u], z + zo, n[u]);
      if (a.drop.on) {
        if constexpr (!FLAT) {
          if (whole_rows)
            bits[u] = rng.word(mask_pos(a, row, 0)) > a.drop.drop_max ? bits[u] : 0u;
          else
            bits[u] = keep_bits<VEC>(rng, mask_pos(a, row, col), a.drop.drop_max);
        } else if (linear) {
          bits[u] = keep_bits<VEC>(rng, (first + q) * VEC, a.drop.drop_max);
        } else if (whole_rows && col + VEC <= D) {
          bits[u] = rng.word(mask_pos(a, row, 0)) > a.drop.drop_max ? bits[u] : 0u;
        } else {
          // element by element, a block of four words at a time while the positions stay in it
          uint64_t have = ~0ull;
          uint4 w = make_uint4(0, 0, 0, 0);
          uint32_t r = row, c = col;
          bits[u] = 0;
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            if (k < n[u]) {
              const uint64_t pos = mask_pos(a, r, c);
              if (pos >> 2 != have) {
                have = pos >> 2;
                w = rng.block(have);
              }
              const uint32_t lo = (pos & 1) ? w.y : w.x, hi = (pos & 1) ? w.w : w.z;
              if (((pos & 2) ? hi : lo) > a.drop.drop_max) bits[u] |= 1u << k;
              if (++c == D) {
                c = 0;
                ++r;
              }
            }
          }
        }
      }
      if (bits[u]) {  // what is dropped whole is not read
        load_some(yr[u], y + yo, n[u]);
        if (HASZ && a.in_place) load_some(zr[u], z + zo, n[u]);
      } else if (HASZ && a.in_place) {
        n[u] = 0;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!n[u]) continue;
      Pack<TO, VEC> o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float f = 0.0f;
        if (k < n[u]) {
          if (HASZ) f = to_f32(zr[u].v[k]);
          if (bits[u] >> k & 1) f = HASZ ? fmaf(to_f32(yr[u].v[k]), a.drop.scale, f) : to_f32(yr[u].v[k]) * a.drop.scale;
        }
        o.v[k] = from_f32<TO>(f);
      }
      if (VEC == 1 || n[u] == VEC) {
        store_pack(out + oo[u], o);
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          if (k < n[u]) out[oo[u] + k] = o.v[k];
      }
    }
  }
}

template <class TZ, class TY, class TO, int VEC, bool FLAT, bool HASZ>
cudaError_t launch_one(const DropoutAddArgs& a, cudaStream_t st) {
  const uint64_t elements = (uint64_t)a.map.rows * a.dim;
  const FastDiv per_row = FastDiv::make(FLAT ? a.dim : a.dim / VEC);
  const uint64_t chunks = (elements + VEC - 1) / VEC, tiles = (chunks + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  const uint64_t cap = (uint64_t)device_sm_count() * 32;
  dropout_add_kernel<TZ, TY, TO, VEC, FLAT, HASZ><<<(unsigned)(tiles < cap ? tiles : cap), kThreads, 0, st>>>(a, per_row,
                                                                                                           elements);
  return cudaGetLastError();
}

template <class TZ, class TY, class TO, bool HASZ>
cudaError_t launch_types(const DropoutAddArgs& a, int vec, cudaStream_t st) {
  constexpr int FULL = sizeof(TZ) == 2 && sizeof(TY) == 2 && sizeof(TO) == 2 ? 8 : 4;
  const auto aligned = [](const void* p, size_t b) { return reinterpret_cast<uintptr_t>(p) % b == 0; };
  if (vec >= FULL) return launch_one<TZ, TY, TO, FULL, false, HASZ>(a, st);
  if ((!a.z || a.zs.dense) && a.ys.dense && a.os.dense && aligned(a.z, FULL * sizeof(TZ)) &&
      aligned(a.y, FULL * sizeof(TY)) && aligned(a.out, FULL * sizeof(TO)))
    return launch_one<TZ, TY, TO, FULL, true, HASZ>(a, st);
  return launch_one<TZ, TY, TO, 1, false, HASZ>(a, st);
}

}  // namespace

cudaError_t launch_dropout_add(const DropoutAddArgs& a, int z_dtype, int y_dtype, int out_dtype, int vec,
                               cudaStream_t st) {
  using H = __half;
  using B = __nv_bfloat16;
  if (!a.z) {
    if (y_dtype == DT_F32 && out_dtype == DT_F32) return launch_types<float, float, float, false>(a, vec, st);
    if (y_dtype == DT_F32 && out_dtype == DT_F16) return launch_types<float, float, H, false>(a, vec, st);
    if (y_dtype == DT_F32 && out_dtype == DT_BF16) return launch_types<float, float, B, false>(a, vec, st);
    if (y_dtype == DT_F16 && out_dtype == DT_F16) return launch_types<H, H, H, false>(a, vec, st);
    if (y_dtype == DT_BF16 && out_dtype == DT_BF16) return launch_types<B, B, B, false>(a, vec, st);
    return cudaErrorInvalidValue;
  }
  if (z_dtype != out_dtype) return cudaErrorInvalidValue;
  if (z_dtype == DT_F32 && y_dtype == DT_F32) return launch_types<float, float, float, true>(a, vec, st);
  if (z_dtype == DT_F32 && y_dtype == DT_F16) return launch_types<float, H, float, true>(a, vec, st);
  if (z_dtype == DT_F32 && y_dtype == DT_BF16) return launch_types<float, B, float, true>(a, vec, st);
  if (z_dtype == DT_F16 && y_dtype == DT_F16) return launch_types<H, H, H, true>(a, vec, st);
  if (z_dtype == DT_BF16 && y_dtype == DT_BF16) return launch_types<B, B, B, true>(a, vec, st);
  return cudaErrorInvalidValue;
}

}  // namespace triattn
