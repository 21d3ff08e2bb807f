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
#include <mutex>

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
__device__ __forceinline__ int64_t row_offset(const Strides3& s, uint32_t row, const RowMap& map, int dim) {
  if (s.dense) return (int64_t)row * dim;
  const RowIndex i = map.at(row);
  return s.s[0] * i.i0 + s.s[1] * i.i1 + s.s[2] * i.i2;
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

// ---- rows on their way to a lane ------------------------------------------------------------------------
// Every lane brings its own share of its next rows into shared memory with asynchronous copies, kStages
// batches deep, and reads it back when its turn comes.  What is in flight then costs no registers (an SM
// needs about 50 KB of it to keep HBM busy), and as a lane reads only what it copied itself, no barrier
// stands between the two.
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  static_assert(BYTES == 4 || BYTES == 8 || BYTES == 16, "");
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// the first `bytes` (1..16) of 16; what follows them is not read
__device__ __forceinline__ void copy_async_part(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// How a row of dim channels lies on its lanes: LPR lanes of one warp (8, 16 or 32), or with LPR = 0 `width`
// lanes of several warps, each with NCH pieces of VEC consecutive channels, piece c at channel
// (lane + c * width) * VEC.  A CTA holds several such groups.
// VEC > 1: a piece is copied by its own lane.  VEC = 1, for rows that start anywhere (an odd dim, an odd
// stride or address): the row's lanes copy the 16-byte blocks that hold it, so what a lane reads was
// copied by its neighbours, and a barrier of the row's lanes (sync) stands before and after the reading.
constexpr int RES_MAX_WARPS = 16;  // of a CTA
template <int VEC, int LPR, int NCH>
struct Lanes {
  int width, lane, group, groups, dim;
  bool act[NCH];
  __device__ __forceinline__ Lanes(int d, int w) : dim(d) {
    width = LPR ? LPR : w;
    group = threadIdx.x / width;
    lane = threadIdx.x - group * width;
    groups = blockDim.x / width;
#pragma unroll
    for (int c = 0; c < NCH; ++c) act[c] = col(c) < dim;
  }
  __device__ __forceinline__ int col(int c) const { return (lane + c * width) * VEC; }
  __device__ __forceinline__ void barrier() const {  // of the row's lanes
    if constexpr (LPR)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(width) : "memory");
  }
  __device__ __forceinline__ void sync() const {
    if constexpr (VEC == 1) barrier();
  }
  // Sums over the row's lanes.  Several warps: one barrier per call; consecutive calls use the two halves
  // of red in turn, and a warp reaches the same half again only after the barrier in between.
  static constexpr int red_floats = LPR ? 1 : RES_MAX_WARPS * 2 * 2;
  template <int K>
  __device__ __forceinline__ void sum(float (&v)[K], float* red, int& phase) const {
    constexpr int W = LPR ? LPR : 32;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
    if constexpr (LPR == 0) {
      static_assert(K <= 2, "");
      float* s = red + phase * RES_MAX_WARPS * 2;
      phase ^= 1;
      const int wl = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = width >> 5, first = group * warps;
      if (wl == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) s[k * RES_MAX_WARPS + warp] = v[k];
      }
      barrier();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        v[k] = wl < warps ? s[k * RES_MAX_WARPS + first + wl] : 0.0f;
#pragma unroll
        for (int o = RES_MAX_WARPS / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
        v[k] = __shfl_sync(0xffffffffu, v[k], 0);
      }
    }
  }
};

// Rows of several warps: C pieces (of VEC channels) on `width` lanes, 16 channels a lane at most (registers).
// fp32 rows take three pieces a lane instead of four where that leaves fewer lanes idle (dim 768, 1536).
struct RowWidth {
  int pieces, width, threads;
};
template <int VEC>
RowWidth row_width(int C) {
  const auto lanes = [C](int n) { return ((C + n - 1) / n + 31) / 32 * 32; };
  int n = 16 / VEC;
  if (VEC == 4 && lanes(3) * 3 < lanes(4) * 4 && lanes(3) <= 512) n = 3;
  const int width = lanes(n), groups = width < 256 ? 256 / width : 1;
  return RowWidth{n, width, width * groups};
}

// Bytes of shared memory that one row of a tensor takes in one stage, per row's group of lanes.
template <class T, int VEC, int NCH>
__host__ __device__ constexpr int row_slot(int width, int dim) {
  return VEC > 1 ? width * NCH * VEC * (int)sizeof(T) : (dim * (int)sizeof(T) + 15) / 16 * 16 + 16;
}

// One row of a tensor, copied to `slot` and read back from it.
template <class T, int VEC, int LPR, int NCH>
struct RowCopy {
  using L = Lanes<VEC, LPR, NCH>;
  __device__ __forceinline__ static void issue(const L& l, uint32_t slot, const T* row) {
    if constexpr (VEC > 1) {
      constexpr int B = VEC * sizeof(T);
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        if (l.act[c]) {
          const uint32_t dst = slot + (l.lane + c * l.width) * B;
          const T* src = row + l.col(c);
          if constexpr (B <= 16) {
            copy_async<B>(dst, src);
          } else {
#pragma unroll
            for (int k = 0; k < B; k += 16) copy_async<16>(dst + k, reinterpret_cast<const char*>(src) + k);
          }
        }
    } else {
      // the block that holds the row's first byte begins at most 15 bytes before it, inside the same
      // 16-byte block of memory; behind the row's last byte nothing is read
      const uintptr_t first = reinterpret_cast<uintptr_t>(row), last = first + (uintptr_t)l.dim * sizeof(T);
      uintptr_t at = (first & ~(uintptr_t)15) + (uintptr_t)l.lane * 16;
      for (uint32_t dst = slot + l.lane * 16; at < last; at += (uintptr_t)l.width * 16, dst += l.width * 16) {
        const int n = last - at < 16 ? (int)(last - at) : 16;
        copy_async_part(dst, reinterpret_cast<const void*>(at), n);
      }
    }
  }
  // piece c, as floats
  __device__ __forceinline__ static void read(const L& l, const char* slot, const T* row, int c, float (&v)[VEC]) {
    if constexpr (VEC > 1) {
      const Pack<T, VEC> p = load_pack<T, VEC>(reinterpret_cast<const T*>(slot) + (l.lane + c * l.width) * VEC);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = to_f32(p.v[k]);
    } else {
      v[0] = to_f32(reinterpret_cast<const T*>(slot + (reinterpret_cast<uintptr_t>(row) & 15))[l.col(c)]);
    }
  }
};

// Keep bits of the NCH pieces of a lane: bit k of keep[c].  pos0: position of the row's first channel.
template <int VEC, int LPR, int NCH>
__device__ __forceinline__ void keep_pieces(const Lanes<VEC, LPR, NCH>& l, const Philox& rng, uint64_t pos0,
                                            uint32_t drop_max, uint32_t (&keep)[NCH]) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) keep[c] = keep_bits<VEC>(rng, pos0 + l.col(c), drop_max);
  } else if constexpr (NCH < 3) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) keep[c] = keep_bits<1>(rng, pos0 + l.col(c), drop_max);
  } else {
    // The 32 channels of a warp's piece lie in at most 9 blocks of four positions: lanes 0..8, 9..17 and
    // 18..26 draw those of three pieces at a time, and every lane fetches its bit.
    const int wl = threadIdx.x & 31, third = wl >= 27 ? 2 : wl / 9, block = wl - third * 9;
    const int warp0 = l.lane - wl;  // first channel of the warp in piece 0
#pragma unroll
    for (int c = 0; c < NCH; c += 3) {
      const uint64_t mine = pos0 + warp0 + (c + third) * l.width;
      const uint32_t bits = keep_bits<4>(rng, ((mine >> 2) + block) << 2, drop_max);
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        if (c + j < NCH) {
          const uint32_t at = (uint32_t)(pos0 + warp0 + (c + j) * l.width) & 3;  // in the first block
          const uint32_t b = __shfl_sync(0xffffffffu, bits, j * 9 + ((at + wl) >> 2));
          keep[c + j] = b >> ((at + wl) & 3) & 1;
        }
      }
    }
  }
}

int device_sm_count();

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

// A persistent launch over rows: as many CTAs as fit on the GPU at once, `most` per SM at most, or as the rows
// need (per_cta rows each per sweep).  What a kernel needs to be known for that is asked for once per device.
struct KernelInfo {
  std::mutex mu;
  int regs[64] = {0};
};
template <class Kernel, class Args>
cudaError_t launch_rows(KernelInfo& info, Kernel kernel, const Args& a, int width, int per_cta, int threads, size_t smem,
                        int most, cudaStream_t st, unsigned* ctas) {
  constexpr int kSmem = 227 * 1024, kStatic = 1024;  // of an SM; a CTA's static and reserved share, rounded up
  int dev = 0, regs = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  {
    std::lock_guard<std::mutex> lk(info.mu);
    if (!info.regs[dev]) {
      cudaFuncAttributes f;
      if (cudaError_t e = cudaFuncGetAttributes(&f, kernel); e != cudaSuccess) return e;
      if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kSmem - (int)f.sharedSizeBytes);
          e != cudaSuccess)
        return e;
      info.regs[dev] = f.numRegs;
    }
    regs = info.regs[dev];
  }
  const int warps = threads / 32;
  int fit = 65536 / ((regs + 7) / 8 * 8 * 32 * warps);
  if (fit > 64 / warps) fit = 64 / warps;
  if (fit > (int)(kSmem / (smem + 2 * kStatic))) fit = (int)(kSmem / (smem + 2 * kStatic));
  if (fit < 1) fit = 1;
  if (fit > most) fit = most;
  const long long need = ((long long)a.map.rows + per_cta - 1) / per_cta, cap = (long long)device_sm_count() * fit;
  const unsigned grid = (unsigned)(need < cap ? need : cap);
  if (ctas) *ctas = grid;
  kernel<<<grid, threads, smem, st>>>(a, width);
  return cudaGetLastError();
}

// what every tensor of a call allows: elements moved at a time (8, 4 or 1)
cudaError_t launch_norm_fwd(const NormFwdArgs& a, int z_dtype, int y_dtype, int out_dtype, int vec, cudaStream_t st);
cudaError_t launch_norm_bwd(const NormBwdArgs& a, int x_dtype, int y_dtype, int dout_dtype, int vec, cudaStream_t st);
cudaError_t launch_dropout_add(const DropoutAddArgs& a, int z_dtype, int y_dtype, int out_dtype, int vec,
                               cudaStream_t st);
// CTAs of launch_norm_bwd at most (rows of its partial sums)
int norm_bwd_max_ctas();

}  // namespace triattn
