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
  static RowMap make(const int64_t* n, int64_t rows) {
    const auto size = [](int64_t v) { return (uint32_t)(v > 0 ? v : 1); };
    return RowMap{(uint32_t)rows, FastDiv::make(size(n[1])), FastDiv::make(size(n[2]))};
  }
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

constexpr uint32_t PHILOX_M0 = 0xD2511F53u, PHILOX_M1 = 0xCD9E8D57u;  // multipliers of Philox4x32
constexpr uint32_t PHILOX_W0 = 0x9E3779B9u, PHILOX_W1 = 0xBB67AE85u;  // steps of its key

// ---- the keep mask ------------------------------------------------------------------------------
struct Dropout {
  int on;                // 0: everything is kept and scale is 1
  uint32_t drop_max;     // a word u is dropped if u <= drop_max
  float scale;
  uint64_t offset;
  uint32_t key[10][2];    // the ten rounds' keys, from the seed
  const uint64_t* state;  // device {seed, offset} instead of the two above, or nullptr
  int64_t m[3];           // strides of the mask tensor's leading axes, 0 where shared
  int per_channel;        // 1: every channel has its own position, 0: one for the whole row
};

// The generator of one launch.  The rounds' keys are operands from the kernel's parameters where the host knows the
// seed; where the device holds it, they are worked out as they are used (20 additions more, beside a block's 20 wide multiplications and 20 exclusive ors).
struct Philox {
  const Dropout& d;
  uint32_t k0, k1, o0, o1;
  __device__ __forceinline__ explicit Philox(const Dropout& drop) : d(drop) {
    k0 = k1 = 0;
    uint64_t offset = d.offset;
    if (d.state) {
      k0 = (uint32_t)d.state[0];
      k1 = (uint32_t)(d.state[0] >> 32);
      offset = d.state[1];
    }
    o0 = (uint32_t)offset;
    o1 = (uint32_t)(offset >> 32);
  }
  static __device__ __forceinline__ void round(uint32_t& c0, uint32_t& c1, uint32_t& c2, uint32_t& c3, uint32_t a, uint32_t b) {
    const uint64_t p = (uint64_t)PHILOX_M0 * c0, q = (uint64_t)PHILOX_M1 * c2;
    c0 = (uint32_t)(q >> 32) ^ c1 ^ a;
    c1 = (uint32_t)q;
    c2 = (uint32_t)(p >> 32) ^ c3 ^ b;
    c3 = (uint32_t)p;
  }
  // the four words of block (positions 4 * block .. 4 * block + 3); Salmon, Moraes, Dror, Shaw,
  // Parallel random numbers: as easy as 1, 2, 3 (2011), 10 rounds
  __device__ __forceinline__ uint4 block(uint64_t block) const {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = o0, c3 = o1;
    if (!d.state) {
#pragma unroll
      for (int r = 0; r < 10; ++r) round(c0, c1, c2, c3, d.key[r][0], d.key[r][1]);
    } else {
      uint32_t a = k0, b = k1;
#pragma unroll
      for (int r = 0; r < 10; ++r) {
        round(c0, c1, c2, c3, a, b);
        a += PHILOX_W0;
        b += PHILOX_W1;
      }
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
// keep bits of a block's four positions
__device__ __forceinline__ uint32_t keep_bits(const Philox& rng, uint64_t block, uint32_t drop_max) {
  const uint4 w = rng.block(block);
  return (w.x > drop_max ? 1u : 0u) | (w.y > drop_max ? 2u : 0u) | (w.z > drop_max ? 4u : 0u) | (w.w > drop_max ? 8u : 0u);
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

// ---- two fp32 values a register pair: one instruction does both --------------------------------------
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ Pair both(float v) { return pair(v, v); }
__device__ __forceinline__ float2 halves(Pair a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float total(Pair a) {
  const float2 h = halves(a);
  return h.x + h.y;
}
// two neighbouring elements of type T
template <class T>
__device__ __forceinline__ Pair to_pair(const T* p) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    uint32_t u;
    __builtin_memcpy(&u, p, 4);
    return pair(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  } else if constexpr (std::is_same<T, __half>::value) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(p));
    return pair(f.x, f.y);
  } else {
    return pair(p[0], p[1]);
  }
}
template <class T>
__device__ __forceinline__ void from_pair(Pair a, T* p) {
  const float2 h = halves(a);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(h.x, h.y);
    __builtin_memcpy(p, &r, 4);
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 r = __floats2half2_rn(h.x, h.y);
    __builtin_memcpy(p, &r, 4);
  } else {
    p[0] = h.x;
    p[1] = h.y;
  }
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
template <int BYTES>
__device__ __forceinline__ void copy_zero(uint32_t dst, const void* any) {  // `any` is not read
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, 0;" ::"r"(dst), "l"(any) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, 0;" ::"r"(dst), "l"(any), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// How a row of dim channels lies on its lanes: LPR lanes of one warp (8, 16 or 32), or with LPR = 0 `width`
// lanes of several warps, each with NCH pieces of VEC consecutive channels, piece c at channel
// (lane + c * width) * VEC.  A CTA holds several such groups.
// VEC > 1: a piece is copied by its own lane.  All pieces but the last are there on every lane; where the last is
// not, its place in shared memory holds zeros.
// VEC = 1, for rows that start anywhere (an odd dim, an odd stride or address): the row's lanes copy the
// 16-byte blocks that hold it, so what a lane reads was copied by its neighbours, and a barrier of the
// row's lanes (sync) stands before and after the reading.  All pieces but the last four are there.
constexpr int RES_MAX_WARPS = 16;  // of a CTA
constexpr int RES_MAX_GROUPS = 8;  // of several warps, in a CTA
constexpr int RES_MAX_SUMS = 4;    // of one call
template <int VEC, int LPR, int NCH>
struct Lanes {
  static constexpr int EPL = VEC * NCH, PAIRS = (EPL + 1) / 2;  // channels of a lane, and the pairs that hold them
  int width, lane, group, groups, dim;
  bool last;  // the last piece is there
  __device__ __forceinline__ Lanes(int d, int w) : dim(d) {
    width = LPR ? LPR : w;
    group = threadIdx.x / width;
    lane = threadIdx.x - group * width;
    groups = blockDim.x / width;
    last = col(NCH - 1) < dim;
  }
  __device__ __forceinline__ bool act(int c) const {
    return VEC > 1 ? (c < NCH - 1 || last) : (c < NCH - 4 || col(c) < dim);
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
  static constexpr int red_floats = LPR ? 4 : 2 * RES_MAX_SUMS * RES_MAX_GROUPS * RES_MAX_WARPS;
  // what sum() reads beyond a group's warps: zeros
  __device__ __forceinline__ void clear(float* red) const {
    if constexpr (LPR == 0) {
      for (int i = threadIdx.x; i < red_floats; i += blockDim.x) red[i] = 0.0f;
      __syncthreads();
    }
  }
  template <int K>
  __device__ __forceinline__ void sum(float (&v)[K], float* red, int& phase) const {
    constexpr int W = LPR ? LPR : 32;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
    if constexpr (LPR == 0) {
      static_assert(K <= RES_MAX_SUMS, "");
      float* s = red + (phase * RES_MAX_GROUPS + group) * RES_MAX_SUMS * RES_MAX_WARPS;
      phase ^= 1;
      const int warps = width >> 5;
      if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) s[k * RES_MAX_WARPS + (lane >> 5)] = v[k];
      }
      barrier();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        v[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < RES_MAX_WARPS; i += 4) {
          if (i < warps) {
            const float4 f = *reinterpret_cast<const float4*>(s + k * RES_MAX_WARPS + i);
            v[k] += (f.x + f.y) + (f.z + f.w);
          }
        }
      }
    }
  }
};

// R rows of a group that are worked on together, from `first` on.  DENSE: all tensors are dense, and a row's number
// is all that is needed; else lane r of the group holds the index of row r.
template <bool DENSE, int R>
struct Batch {
  uint32_t first, rows;
  RowIndex mine;
  template <class L>
  __device__ __forceinline__ Batch(const L& l, const RowMap& map, uint32_t f) : first(f), rows(map.rows) {
    if constexpr (!DENSE) {
      static_assert((R & (R - 1)) == 0, "");
      const uint32_t row = first + (R > 1 ? l.lane & (R - 1) : 0);
      mine = map.at(row < rows ? row : rows - 1);
    }
  }
  __device__ __forceinline__ uint32_t row(int r) const { return first + r; }
  __device__ __forceinline__ bool live(int r) const { return first + r < rows; }
};

// Rows of several warps: C pieces (of VEC channels) on `width` lanes, 16 channels a lane at most (registers); the
// number of pieces a lane that leaves the fewest lanes idle, all but the last full.
struct RowWidth {
  int pieces, width, threads;
};
template <int VEC>
RowWidth row_width(int C, int threads) {  // a CTA of about so many threads
  RowWidth best{16 / VEC, 512, 512};
  int cost = 1 << 30;
  for (int n = 16 / VEC; n >= 2; n -= VEC == 1 ? 4 : 1) {
    const int width = ((C + n - 1) / n + 31) / 32 * 32;
    if (width > 512 || (VEC > 1 ? (n - 1) * width > C : (n < 12 || (n - 4) * width >= C))) continue;
    if (width * n < cost) {
      cost = width * n;
      best = RowWidth{n, width, width < threads ? threads / width * width : width};
    }
  }
  return best;
}

// What Lanes::act takes for granted: the pieces that are always there are, and the others reach the row's end.  Every
// launch asks.
template <int VEC, int NCH>
bool pieces_fit(int dim, int width) {
  const int always = VEC > 1 ? NCH - 1 : NCH - 4;
  return always * width * VEC <= dim && NCH * width * VEC >= dim && dim % VEC == 0;
}

// Bytes of shared memory that one row of a tensor takes in one stage, per row's group of lanes.
template <class T, int VEC, int NCH>
__host__ __device__ constexpr int row_slot(int width, int dim) {
  return VEC > 1 ? width * NCH * VEC * (int)sizeof(T) : (dim * (int)sizeof(T) + 15) / 16 * 16 + 16;
}

// A tensor's rows.  A dense one's row is found by one multiply-add; of a strided one lane r of a group works out where
// row r lies, and hands it round (every lane of a warp takes part).
template <class T, int LPR, bool DENSE>
struct RowsOf {
  char* base;
  uint32_t pitch;  // bytes of a dense row
  bool dense;
  int64_t s0, s1, s2;
  __device__ __forceinline__ RowsOf(const void* p, const Strides3& s, int dim, int lane_elements) {
    base = static_cast<char*>(const_cast<void*>(p)) + lane_elements * (int)sizeof(T);
    pitch = dim * (uint32_t)sizeof(T);
    if constexpr (!DENSE) {
      dense = s.dense;
      s0 = s.s[0] * (int)sizeof(T);
      s1 = s.s[1] * (int)sizeof(T);
      s2 = s.s[2] * (int)sizeof(T);
    }
  }
  template <int R>
  __device__ __forceinline__ void at(const Batch<DENSE, R>& batch, T* (&p)[R]) const {
    if (DENSE || dense) {
#pragma unroll
      for (int r = 0; r < R; ++r) p[r] = reinterpret_cast<T*>(base + (uint64_t)batch.row(r) * pitch);
    } else {
      const int64_t off = s0 * batch.mine.i0 + s1 * batch.mine.i1 + s2 * batch.mine.i2;
#pragma unroll
      for (int r = 0; r < R; ++r)
        p[r] = reinterpret_cast<T*>(base + (R > 1 ? __shfl_sync(0xffffffffu, off, r, LPR ? LPR : 32) : off));
    }
  }
};

// An input's rows on their way through shared memory: copied to a slot and read back from it.  `off` is the
// slot's place in the group's ring.
template <class T, int VEC, int LPR, int NCH, bool DENSE>
struct RowIn {
  using L = Lanes<VEC, LPR, NCH>;
  static constexpr int B = VEC * sizeof(T);
  static_assert(VEC == 1 || B == 8 || B == 16, "");
  const L& l;
  RowsOf<T, LPR, DENSE> rows;
  char* ring;  // VEC > 1: at the lane's first piece
  uint32_t ring32;
  __device__ __forceinline__ RowIn(const L& l_, const void* p, const Strides3& s, char* r)
      : l(l_), rows(p, s, l_.dim, VEC > 1 ? l_.lane * VEC : 0) {
    ring = r + (VEC > 1 ? l.lane * B : 0);
    ring32 = smem_u32(ring);
  }
  __device__ __forceinline__ int step() const { return l.width * B; }  // between pieces
  // zeros where a lane has no last piece, once for every slot
  __device__ __forceinline__ void clear(int off) const {
    if constexpr (VEC > 1) {
      if (!l.last) {
        uint64_t* p = reinterpret_cast<uint64_t*>(ring + off + (NCH - 1) * step());
#pragma unroll
        for (int k = 0; k < B / 8; ++k) p[k] = 0;
      }
    }
  }
  // row p = rows.at(...)
  __device__ __forceinline__ void issue(int off, const T* p) const {
    if constexpr (VEC > 1) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        if (l.act(c)) copy_async<B>(ring32 + off + c * step(), reinterpret_cast<const char*>(p) + c * step());
    } else {
      // the block that holds the row's first byte begins at most 15 bytes before it, inside the same
      // 16-byte block of memory; behind the row's last byte nothing is read
      const uintptr_t first = reinterpret_cast<uintptr_t>(p), end = first + (uintptr_t)l.dim * sizeof(T);
      uintptr_t at = (first & ~(uintptr_t)15) + (uintptr_t)l.lane * 16;
      for (uint32_t dst = ring32 + off + l.lane * 16; at < end; at += (uintptr_t)l.width * 16, dst += l.width * 16)
        copy_async_part(dst, reinterpret_cast<const void*>(at), end - at < 16 ? (int)(end - at) : 16);
    }
  }
  // A row that is not there: zeros.  The address, of which nothing is read, is one that a copy may have: of a tensor that
  // starts anywhere the 16-byte block that holds its start.
  __device__ __forceinline__ void issue_none(int off) const {
    if constexpr (VEC > 1) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) copy_zero<B>(ring32 + off + c * step(), rows.base);
    } else {
      const void* any = reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(rows.base) & ~(uintptr_t)15);
      for (int i = l.lane * 16; i < row_slot<T, VEC, NCH>(l.width, l.dim); i += l.width * 16)
        copy_zero<16>(ring32 + off + i, any);
    }
  }
  __device__ __forceinline__ void read(int off, const T* row, Pair (&x)[L::PAIRS]) const {
    if constexpr (VEC > 1) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const Pack<T, VEC> p = load_pack<T, VEC>(reinterpret_cast<const T*>(ring + off + c * step()));
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) x[c * VEC / 2 + j] = to_pair(p.v + 2 * j);
      }
    } else {
      const T* p = reinterpret_cast<const T*>(ring + off + (reinterpret_cast<uintptr_t>(row) & 15));
      float v[2 * L::PAIRS];
#pragma unroll
      for (int c = 0; c < 2 * L::PAIRS; ++c) v[c] = c < NCH && l.act(c) ? to_f32(p[l.col(c)]) : 0.0f;
#pragma unroll
      for (int j = 0; j < L::PAIRS; ++j) x[j] = pair(v[2 * j], v[2 * j + 1]);
    }
  }
};
// An output's rows.
template <class T, int VEC, int LPR, int NCH, bool DENSE>
struct RowOut {
  using L = Lanes<VEC, LPR, NCH>;
  const L& l;
  RowsOf<T, LPR, DENSE> rows;
  __device__ __forceinline__ RowOut(const L& l_, const void* p, const Strides3& s) : l(l_), rows(p, s, l_.dim, l_.lane * VEC) {}
  // piece c of a row's values, if the lane has it; p = rows.at(...)
  __device__ __forceinline__ void piece(T* p, int c, const Pair (&x)[L::PAIRS]) const {
    if (!l.act(c)) return;
    if constexpr (VEC > 1) {
      Pack<T, VEC> o;
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) from_pair(x[c * VEC / 2 + j], o.v + 2 * j);
      store_pack(p + c * l.width * VEC, o);
    } else {
      const float2 h = halves(x[c / 2]);
      p[c * l.width] = from_f32<T>(c & 1 ? h.y : h.x);
    }
  }
  __device__ __forceinline__ void row(T* p, const Pair (&x)[L::PAIRS]) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) piece(p, c, x);
  }
};

// a lane's channels of a LayerNorm parameter; zero where it has none
template <class T, int VEC, int LPR, int NCH, int P>
__device__ __forceinline__ void load_pairs_of(const Lanes<VEC, LPR, NCH>& l, const T* p, Pair (&x)[P]) {
  if (VEC > 1 && (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0) {
    Pack<T, 4> v[(VEC * NCH + 3) / 4];  // all on their way before the first is used
#pragma unroll
    for (int q = 0; q < VEC * NCH / 4; ++q)
      if (l.act(q * 4 / VEC)) v[q] = load_pack<T, 4>(p + l.col(q * 4 / VEC) + q * 4 % VEC);
#pragma unroll
    for (int q = 0; q < VEC * NCH / 4; ++q) {
      const bool a = l.act(q * 4 / VEC);
      x[2 * q] = a ? to_pair(v[q].v) : both(0.0f);
      x[2 * q + 1] = a ? to_pair(v[q].v + 2) : both(0.0f);
    }
  } else {
    float v[2 * P];
#pragma unroll
    for (int i = 0; i < 2 * P; ++i)
      v[i] = i < VEC * NCH && l.act(i / VEC) ? to_f32(p[l.col(i / VEC) + i % VEC]) : 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j) x[j] = pair(v[2 * j], v[2 * j + 1]);
  }
}
template <int VEC, int LPR, int NCH, int P>
__device__ __forceinline__ void load_pairs(const Lanes<VEC, LPR, NCH>& l, const void* p, int dtype, float absent, Pair (&x)[P]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < P; ++j)
      x[j] = pair(2 * j < VEC * NCH && l.act(2 * j / VEC) ? absent : 0.0f,
                  2 * j + 1 < VEC * NCH && l.act((2 * j + 1) / VEC) ? absent : 0.0f);
  } else if (dtype == DT_F32) {
    load_pairs_of(l, static_cast<const float*>(p), x);
  } else if (dtype == DT_F16) {
    load_pairs_of(l, static_cast<const __half*>(p), x);
  } else {
    load_pairs_of(l, static_cast<const __nv_bfloat16*>(p), x);
  }
}
// x += m on the channels that are there, and t += x * x
template <int VEC, int LPR, int NCH, int P>
__device__ __forceinline__ void centre(const Lanes<VEC, LPR, NCH>& l, Pair m, Pair (&x)[P], Pair& t) {
  if constexpr (VEC > 1) {
    constexpr int N = VEC / 2;
#pragma unroll
    for (int j = 0; j < P - N; ++j) {
      x[j] = x[j] + m;
      t = fma2(x[j], x[j], t);
    }
    if (l.last) {
#pragma unroll
      for (int j = P - N; j < P; ++j) {
        x[j] = x[j] + m;
        t = fma2(x[j], x[j], t);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const Pair d = x[j] + m;
      if (2 * j + 1 < NCH - 4) {
        x[j] = d;
      } else {
        const float2 h = halves(d);
        x[j] = pair(l.act(2 * j) ? h.x : 0.0f, 2 * j + 1 < NCH && l.act(2 * j + 1) ? h.y : 0.0f);
      }
      t = fma2(x[j], x[j], t);
    }
  }
}

// f(kept, i) for a lane's channels i = 0 .. EPL - 1, drawn at the positions from pos0 (the row's first) on.
template <int VEC, int LPR, int NCH, class F>
__device__ __forceinline__ void each_kept(const Lanes<VEC, LPR, NCH>& l, const Philox& rng, uint64_t pos0,
                                          uint32_t drop_max, F&& f) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
#pragma unroll
      for (int q = 0; q < VEC; q += 4) {
        const uint4 w = rng.block((pos0 + l.col(c) + q) >> 2);
        f(w.x > drop_max, c * VEC + q);
        f(w.y > drop_max, c * VEC + q + 1);
        f(w.z > drop_max, c * VEC + q + 2);
        f(w.w > drop_max, c * VEC + q + 3);
      }
    }
  } else if constexpr (LPR && NCH > 1) {
    // A row's channels are next to one another: lane i draws block i of four positions, LPR blocks at a time, and every
    // lane fetches its bits.  The row may begin inside a block, so that the last piece of four reaches one block further:
    // the first lane's of the next round.  (Every lane of a warp takes part.)
    const uint64_t block = (pos0 >> 2) + l.lane;
    const uint32_t at = ((uint32_t)pos0 & 3) + l.lane;
    uint32_t bits = keep_bits(rng, block, drop_max);
#pragma unroll
    for (int n = 0; n < NCH; n += 4) {
      uint32_t next = 0;
      if (NCH >= 4 && (n + 4) * LPR < l.dim + 3) next = keep_bits(rng, block + (n / 4 + 1) * LPR, drop_max);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (n + j < NCH) {
          const uint32_t drawn = j == 3 && l.lane == 0 ? next : bits;
          const uint32_t from = (at >> 2) + j * (LPR / 4);
          f(__shfl_sync(0xffffffffu, drawn, from & (LPR - 1), LPR) >> (at & 3) & 1, n + j);
        }
      }
      bits = next;
    }
  } else if constexpr (NCH == 1) {
    f(rng.word(pos0 + l.col(0)) > drop_max, 0);
  } else {
    // The 32 channels of a warp's piece lie in at most 9 blocks of four positions: lanes 0..8, 9..17 and
    // 18..26 draw those of three pieces at a time, and every lane fetches its bit.
    const int wl = threadIdx.x & 31, third = wl >= 27 ? 2 : wl / 9, block = wl - third * 9;
    const int warp0 = l.lane - wl;  // first channel of the warp in piece 0
#pragma unroll
    for (int c = 0; c < NCH; c += 3) {
      if (c >= NCH - 4 && warp0 + c * l.width >= l.dim) break;  // the row ends before
      const uint64_t mine = (pos0 + warp0 + (c + third) * l.width) >> 2;
      const uint32_t bits = keep_bits(rng, mine + block, drop_max);
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        if (c + j < NCH) {
          const uint32_t at = ((uint32_t)(pos0 + warp0 + (c + j) * l.width) & 3) + wl;  // from the first block on
          f(__shfl_sync(0xffffffffu, bits, j * 9 + (at >> 2)) >> (at & 3) & 1, c + j);
        }
      }
    }
  }
}

int device_sm_count();

// ---- arguments ------------------------------------------------------------------------------------
// forward: out = LN(x), x = z, or (with y) x = s = z + dropout(y) rounded to sum's type (z's) and stored in sum;
// the sum alone, with or without z, for triattn_dropout_add
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
  int in_place;        // sum is z
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
  int vector;    // the tensors are one long vector each, and so is the mask
  Dropout drop;
};

// How the batches of a launch (groups * R rows each) are shared out: the first `big` CTAs take `many` batches
// each, the others `few`.
struct Split {
  uint32_t big, many, few, batches;
  __device__ __forceinline__ void range(uint32_t cta, uint32_t& first, uint32_t& end) const {
    first = cta < big ? cta * many : big * many + (cta - big) * few;
    end = first + (cta < big ? many : few);
    if (end > batches) end = batches;
  }
};

// What a kernel needs to be known for its launches, asked for once per device.
struct KernelInfo {
  std::mutex mu;
  int regs[64] = {0}, own[64] = {0};  // registers of a thread, static shared memory of a CTA
  // CTAs of a launch that fit on an SM at once
  template <class Kernel>
  cudaError_t fit(Kernel kernel, int threads, size_t smem, int* ctas) {
    constexpr int kSmem = 227 * 1024, kReserved = 1024;  // of an SM; of a CTA, beside what it asks for
    int dev = 0, r = 0, fixed = 0;
    if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    {
      std::lock_guard<std::mutex> lk(mu);
      if (!regs[dev]) {
        cudaFuncAttributes f;
        if (cudaError_t e = cudaFuncGetAttributes(&f, kernel); e != cudaSuccess) return e;
        if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kSmem - (int)f.sharedSizeBytes);
            e != cudaSuccess)
          return e;
        regs[dev] = f.numRegs;
        own[dev] = (int)f.sharedSizeBytes;
      }
      r = regs[dev];
      fixed = own[dev];
    }
    const int warps = threads / 32;
    int n = 65536 / ((r + 7) / 8 * 8 * 32 * warps);
    if (n > 64 / warps) n = 64 / warps;
    if (n > (int)(kSmem / (smem + kReserved + fixed))) n = (int)(kSmem / (smem + kReserved + fixed));
    *ctas = n < 1 ? 1 : n;
    return cudaSuccess;
  }
};

// vec: what every tensor of a call allows, elements moved at a time (8, 4 or 1)
cudaError_t launch_norm_fwd(const NormFwdArgs& a, int z_dtype, int out_dtype, int vec, cudaStream_t st);
cudaError_t launch_fused_fwd(const NormFwdArgs& a, int z_dtype, int y_dtype, int out_dtype, int vec, cudaStream_t st);
cudaError_t launch_fused16_fwd(const NormFwdArgs& a, int z_dtype, int y_dtype, int out_dtype, int vec, cudaStream_t st);
cudaError_t launch_norm_bwd(const NormBwdArgs& a, int x_dtype, int dout_dtype, int vec, cudaStream_t st);
cudaError_t launch_fused_bwd(const NormBwdArgs& a, int x_dtype, int y_dtype, int dout_dtype, int vec, cudaStream_t st);
cudaError_t launch_fused16_bwd(const NormBwdArgs& a, int x_dtype, int y_dtype, int dout_dtype, int vec, cudaStream_t st);
cudaError_t launch_dropout_add(const DropoutAddArgs& a, int z_dtype, int y_dtype, int out_dtype, int vec,
                               cudaStream_t st);
// triattn_dropout_add by rows, dim up to RES_MAX_DIM
cudaError_t launch_dropout_rows(const NormFwdArgs& a, int y_dtype, int out_dtype, int vec, cudaStream_t st);
int norm_bwd_max_ctas();  // of a launch: rows of its partial sums

}  // namespace triattn
