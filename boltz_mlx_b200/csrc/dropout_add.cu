// Dropout and dropout + residual add: out = (z ? z : 0) + (keep ? y * scale : 0), residual.cuh's mask.
//
// Bound by HBM: z and y read once, out written once; a draw of four positions is 20 wide multiplications and as many
// exclusive ors, which other warps' loads cover as long as enough of them are resident (fp32).  A thread handles chunks of VEC consecutive
// elements, U of them in flight.
#include "residual.cuh"

namespace triattn {
namespace {

constexpr int kThreads = 256;

// Where a chunk lies.  kVector: every tensor is dense and every element has a position of its own (or nothing
// is dropped), so that the tensor is one long vector.  kRows: in one row, found by strides.  kMixed: tensors are
// dense, but draws are shared and dim is not a multiple of VEC: a chunk is VEC elements of the whole tensor,
// in two rows or more.
enum Where { kVector, kRows, kMixed };

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

template <class TZ, class TY, class TO, int VEC, int U, Where W, bool HASZ>
__global__ void __launch_bounds__(kThreads, W == kMixed ? 2 : 4) dropout_add_kernel(const DropoutAddArgs a, FastDiv per_row,
                                                               uint64_t elements) {
  const TZ* z = static_cast<const TZ*>(a.z);
  const TY* y = static_cast<const TY*>(a.y);
  TO* out = static_cast<TO*>(a.out);
  const uint32_t D = (uint32_t)a.dim, drop_max = a.drop.drop_max;
  const float scale = a.drop.scale;
  const Philox rng(a.drop);
  constexpr bool FLAT = W != kRows;
  const uint64_t chunks = FLAT ? (elements + VEC - 1) / VEC : elements / VEC;
  const uint64_t tiles = (chunks + kThreads * U - 1) / (kThreads * U);
  const bool row_draw = W != kVector && a.drop.on && !a.drop.per_channel;
  for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const uint64_t first = tile * (kThreads * U);  // chunk
    // first row of the tile and the place in it (elements if FLAT, chunks if not)
    const uint64_t at0 = FLAT ? first * VEC : first;
    uint32_t row_base = 0, rest = 0;
    if (W != kVector) {
      row_base = (uint32_t)(at0 / per_row.d);
      rest = (uint32_t)(at0 - (uint64_t)row_base * per_row.d);
    }
    Pack<TZ, VEC> zr[U];
    Pack<TY, VEC> yr[U];
    bool kept[U];
    uint32_t row[U], col[U];
    int64_t oo[U];
    int n[U];  // elements of the chunk
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t q = u * kThreads + threadIdx.x;
      n[u] = first + q < chunks ? VEC : 0;
      kept[u] = true;
      row[u] = col[u] = 0;
      oo[u] = 0;
      if (!n[u]) continue;
      int64_t zo, yo;
      if constexpr (FLAT) {
        const uint64_t e = (first + q) * VEC;
        if (elements - e < VEC) n[u] = (int)(elements - e);
        if (W == kMixed) {
          const uint32_t t = rest + q * VEC, dr = per_row.div(t);
          row[u] = row_base + dr;
          col[u] = t - dr * D;
        }
        zo = yo = oo[u] = (int64_t)e;
      } else {
        const uint32_t t = rest + q, dr = per_row.div(t);
        row[u] = row_base + dr;
        col[u] = (t - dr * per_row.d) * VEC;
        zo = row_offset(a.zs, row[u], a.map, D) + col[u];
        yo = row_offset(a.ys, row[u], a.map, D) + col[u];
        oo[u] = row_offset(a.os, row[u], a.map, D) + col[u];
      }
      if (HASZ && !a.in_place) load_some(zr[u], z + zo, n[u]);
      if (row_draw && (W == kRows || col[u] + VEC <= D)) kept[u] = rng.word(mask_pos(a, row[u], 0)) > drop_max;
      if (kept[u]) {  // what is dropped whole is not read, and in place not touched
        load_some(yr[u], y + yo, n[u]);
        if (HASZ && a.in_place) load_some(zr[u], z + zo, n[u]);
      } else if (HASZ && a.in_place) {
        n[u] = 0;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!n[u]) continue;
      float f[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = HASZ ? to_f32(zr[u].v[k]) : 0.0f;
      const auto add = [&](bool k, int i) {
        const float v = to_f32(yr[u].v[i]);
        if (k) f[i] = HASZ ? fmaf(v, scale, f[i]) : v * scale;
      };
      if (!a.drop.on || (row_draw && (W == kRows || col[u] + VEC <= D))) {
        if (kept[u]) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) add(true, k);
        }
      } else if (VEC == 1) {
        add(rng.word(mask_pos(a, row[u], col[u])) > drop_max, 0);
      } else if (W != kMixed) {
        const uint64_t pos = W == kVector ? (uint64_t)oo[u] : mask_pos(a, row[u], col[u]);
#pragma unroll
        for (int k = 0; k + 3 < VEC; k += 4) {
          const uint4 w = rng.block((pos + k) >> 2);
          add(w.x > drop_max, k);
          add(w.y > drop_max, k + 1);
          add(w.z > drop_max, k + 2);
          add(w.w > drop_max, k + 3);
        }
      } else {
        // a chunk that lies in several rows: element by element, a block of four words at a time while the
        // positions stay in it
        uint64_t have = ~0ull;
        uint4 w = make_uint4(0, 0, 0, 0);
        uint32_t r = row[u], c = col[u];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          if (k < n[u]) {
            const uint64_t pos = mask_pos(a, r, c);
            if (pos >> 2 != have) {
              have = pos >> 2;
              w = rng.block(have);
            }
            const uint32_t lo = (pos & 1) ? w.y : w.x, hi = (pos & 1) ? w.w : w.z;
            add(((pos & 2) ? hi : lo) > drop_max, k);
            if (++c == D) {
              c = 0;
              ++r;
            }
          }
        }
      }
      Pack<TO, VEC> o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.v[k] = from_f32<TO>(f[k]);
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

template <class TZ, class TY, class TO, int VEC, Where W, bool HASZ>
cudaError_t launch_one(const DropoutAddArgs& a, cudaStream_t st) {
  constexpr int U = VEC == 8 ? 2 : 4;
  const uint64_t elements = (uint64_t)a.map.rows * a.dim;
  const FastDiv per_row = FastDiv::make(W == kRows ? a.dim / VEC : a.dim);
  const uint64_t chunks = (elements + VEC - 1) / VEC, tiles = (chunks + kThreads * U - 1) / (kThreads * U);
  // a few tiles a CTA, handed out as SMs come free
  const uint64_t per = tiles / ((uint64_t)device_sm_count() * 64) + 1, grid = (tiles + per - 1) / per;
  dropout_add_kernel<TZ, TY, TO, VEC, U, W, HASZ><<<(unsigned)grid, kThreads, 0, st>>>(a, per_row, elements);
  return cudaGetLastError();
}

template <class TZ, class TY, class TO, bool HASZ>
cudaError_t launch_types(const DropoutAddArgs& a, int vec, cudaStream_t st) {
  constexpr int FULL = sizeof(TZ) == 2 && sizeof(TY) == 2 && sizeof(TO) == 2 ? 8 : 4;
  const auto aligned = [](const void* p, size_t b) { return reinterpret_cast<uintptr_t>(p) % b == 0; };
  const bool flat = (!a.z || a.zs.dense) && a.ys.dense && a.os.dense && aligned(a.z, FULL * sizeof(TZ)) &&
                    aligned(a.y, FULL * sizeof(TY)) && aligned(a.out, FULL * sizeof(TO));
  if (flat && a.vector) return launch_one<TZ, TY, TO, FULL, kVector, HASZ>(a, st);
  if (vec >= FULL) return launch_one<TZ, TY, TO, FULL, kRows, HASZ>(a, st);
  if (flat) return launch_one<TZ, TY, TO, FULL, kMixed, HASZ>(a, st);
  return launch_one<TZ, TY, TO, 1, kRows, HASZ>(a, st);
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
