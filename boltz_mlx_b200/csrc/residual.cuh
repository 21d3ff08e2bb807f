// Residual path of the pair stack: what the LayerNorm, dropout and residual-add kernels share.
//
//   h = (x - mean) * rstd * w + b                      per row of dim channels, statistics in fp32
//   s = z + keep ? y * scale : 0, scale = fp32(1 / (1 - p))
//
// Tensors are [n0][n1][n2][dim] with unit stride along dim and any strides of the three leading axes; a
// row is one (i0, i1, i2).  The keep mask is a function of (seed, offset, position) alone and is never
// stored: position m of the mask tensor (size 1 along every shared axis) takes word m % 4 of
// Philox4x32-10 with key = seed and counter = (m / 4, offset), and is kept if that word is above
// drop_max.  So forward and backward, any launch shape, layout or type see the same mask.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "triattn_internal.cuh"

namespace triattn {

constexpr int RES_MAX_DIM = 8192;  // a row lives in the registers of at most 512 threads, 16 channels each

// Division of n < 2^31 by a run-time d >= 1 (Granlund and Montgomery, Division by invariant integers
// using multiplication, 1994): l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1, q = (hi(m n) + n) >> l.
struct FastDiv {
  uint32_t d, m, l;
  static FastDiv make(uint32_t d) {
    uint32_t l = 0;
    while (l < 31 && (1u << l) < d) ++l;
    const uint64_t m = (((1ull << l) - d) << 32) / d + 1;
    return FastDiv{d, (uint32_t)m, l};
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> l; }
};

struct Strides3 {
  int64_t s[3];
  bool dense;  // rows follow one another without gaps
};

struct RowIndex {
  uint32_t i0, i1, i2;
};
struct RowMap {
  uint32_t rows;
  FastDiv n1, n2;
  __device__ __forceinline__ RowIndex at(uint32_t row) const {
    const uint32_t q = n2.div(row), i0 = n1.div(q);
    return RowIndex{i0, q - i0 * n1.d, row - q * n2.d};
  }
};
__device__ __forceinline__ int64_t row_offset(const Strides3& s, uint32_t row, const RowIndex& i, int dim) {
  return s.dense ? (int64_t)row * dim : s.s[0] * i.i0 + s.s[1] * i.i1 + s.s[2] * i.i2;
}

// ---- the keep mask ------------------------------------------------------------------------------
struct Dropout {
  int on;                // 0: everything is kept and scale is 1
  uint32_t drop_max;     // a word u is dropped if u <= drop_max
  float scale;
  uint64_t seed, offset;
  const uint64_t* state;  // device {seed, offset} instead of the two above, or nullptr
  int64_t m[3];           // strides of the mask tensor's leading axes, 0 where shared
  int per_channel;        // 1: every channel has its own position, 0: one for the whole row
};

struct Philox {
  uint32_t k0, k1, o0, o1;
  __device__ __forceinline__ explicit Philox(const Dropout& d) {
    const uint64_t seed = d.state ? d.state[0] : d.seed, offset = d.state ? d.state[1] : d.offset;
    k0 = (uint32_t)seed;
    k1 = (uint32_t)(seed >> 32);
    o0 = (uint32_t)offset;
    o1 = (uint32_t)(offset >> 32);
  }
  // the four words of block (positions 4 * block .. 4 * block + 3); Salmon, Moraes, Dror, Shaw,
  // Parallel random numbers: as easy as 1, 2, 3 (2011), 10 rounds
  __device__ __forceinline__ uint4 block(uint64_t block) const {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = o0, c3 = o1, a = k0, b = k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      const uint64_t p = (uint64_t)0xD2511F53u * c0, q = (uint64_t)0xCD9E8D57u * c2;
      c0 = (uint32_t)(q >> 32) ^ c1 ^ a;
      c1 = (uint32_t)q;
      c2 = (uint32_t)(p >> 32) ^ c3 ^ b;
      c3 = (uint32_t)p;
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
  }
  __device__ __forceinline__ uint32_t word(uint64_t pos) const {
    const uint4 w = block(pos >> 2);
    const uint32_t lo = (pos & 1) ? w.y : w.x, hi = (pos & 1) ? w.w : w.z;
    return (pos & 2) ? hi : lo;
  }
};
__device__ __forceinline__ uint64_t mask_base(const Dropout& d, const RowIndex& i) {
  return (uint64_t)(d.m[0] * i.i0 + d.m[1] * i.i1 + d.m[2] * i.i2);
}
// keep bits of positions pos .. pos + VEC - 1 (VEC 4 or 8: pos is a multiple of 4)
template <int VEC>
__device__ __forceinline__ uint32_t keep_bits(const Philox& rng, uint64_t pos, uint32_t drop_max) {
  if constexpr (VEC == 1) {
    return rng.word(pos) > drop_max ? 1u : 0u;
  } else {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j) {
      const uint4 w = rng.block((pos >> 2) + j);
      bits |= ((w.x > drop_max ? 1u : 0u) | (w.y > drop_max ? 2u : 0u) | (w.z > drop_max ? 4u : 0u) |
               (w.w > drop_max ? 8u : 0u))
              << (4 * j);
    }
    return bits;
  }
}

// ---- element types --------------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC consecutive elements, moved with one access of VEC * sizeof(T) bytes (4 x fp32 and 8 x 16-bit: 16)
template <typename T, int VEC>
struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) Pack {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  using P = Pack<T, VEC>;
  P r;
  if constexpr (sizeof(P) == 16) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    __builtin_memcpy(&r, &u, 16);
  } else if constexpr (sizeof(P) == 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    __builtin_memcpy(&r, &u, 8);
  } else {
    r.v[0] = *p;
  }
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& r) {
  using P = Pack<T, VEC>;
  if constexpr (sizeof(P) == 16) {
    uint4 u;
    __builtin_memcpy(&u, &r, 16);
    *reinterpret_cast<uint4*>(p) = u;
  } else if constexpr (sizeof(P) == 8) {
    uint2 u;
    __builtin_memcpy(&u, &r, 8);
    *reinterpret_cast<uint2*>(p) = u;
  } else {
    *p = r.v[0];
  }
}
// a LayerNorm parameter, held in any of the three types; `absent` where the pointer is null
__device__ __forceinline__ float load_param(const void* p, int dtype, int i, float absent) {
  if (!p) return absent;
  if (dtype == DT_F32) return static_cast<const float*>(p)[i];
  if (dtype == DT_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// ---- sums over the lanes that hold one row -------------------------------------------------------------
// LPR lanes of one warp (8, 16 or 32), or LPR = 0: the whole CTA.
constexpr int RES_MAX_WARPS = 16;
template <int LPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* smem, int& phase) {
  constexpr int W = LPR ? LPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
  if constexpr (LPR == 0) {
    // one barrier per sum: consecutive sums use the two halves of smem ([2][K <= 2][RES_MAX_WARPS]) in
    // turn, and a warp can only reach the same half again after the barrier in between
    float* s = smem + phase * 2 * RES_MAX_WARPS;
    phase ^= 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) s[k * RES_MAX_WARPS + warp] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = lane < warps ? s[k * RES_MAX_WARPS + lane] : 0.0f;
#pragma unroll
      for (int o = RES_MAX_WARPS / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
      v[k] = __shfl_sync(0xffffffffu, v[k], 0);
    }
  }
}

// ---- arguments ------------------------------------------------------------------------------------
// forward: out = LN(x), x = z, or (with y) x = s = z + dropout(y) rounded to z's type and stored in sum
struct NormFwdArgs {
  const void *z, *y;
  void *sum, *out;
  Strides3 zs, ys, ss, os;
  RowMap map;
  int dim;
  const void *weight, *bias;
  int param_dtype;
  float eps;
  float *mean, *rstd;  // [rows] or nullptr
  Dropout drop;
};
// backward: dx = ds + LN'(dout), dy = dropout(dx), partial column sums of dout * xhat and dout
struct NormBwdArgs {
  const void *dout, *x, *ds;
  Strides3 dos, xs, dss;
  RowMap map;
  int dim;
  const void* weight;
  int param_dtype;
  const float *mean, *rstd;
  void *dx, *dy;          // dense, or nullptr
  void *dweight, *dbias;  // param_dtype, or nullptr
  float* partial;         // [launched CTAs][2][dim]
  Dropout drop;
};
// out = (z ? z : 0) + dropout(y)
struct DropoutAddArgs {
  const void *z, *y;
  void* out;
  Strides3 zs, ys, os;
  RowMap map;
  int dim;
  int in_place;  // out is z: what is dropped whole is neither read nor written
  Dropout drop;
};

// what every tensor of a call allows: elements moved at a time (8, 4 or 1)
cudaError_t launch_norm_fwd(const NormFwdArgs& a, int z_dtype, int y_dtype, int out_dtype, int vec, cudaStream_t st);
cudaError_t launch_norm_bwd(const NormBwdArgs& a, int x_dtype, int y_dtype, int dout_dtype, int vec, cudaStream_t st);
cudaError_t launch_dropout_add(const DropoutAddArgs& a, int z_dtype, int y_dtype, int out_dtype, int vec,
                               cudaStream_t st);
int device_sm_count();
// CTAs of launch_norm_bwd at most (rows of its partial sums)
int norm_bwd_max_ctas();

}  // namespace triattn
