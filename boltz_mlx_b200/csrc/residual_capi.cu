// extern "C" entry points of the residual path (declared in include/triattn.h): argument checks, strides
// and mask positions, launches on the caller's stream.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <numeric>
#include <utility>

#include "residual.cuh"
#include "triattn.h"

using namespace triattn;

namespace {

int fail(int code, const char* what, const char* fmt, ...) {
  char msg[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return record_error(code, what, msg);
}

int finish(cudaError_t e, const char* what) {
  return e == cudaSuccess ? TRIATTN_OK : record_error(TRIATTN_ECUDA, what, cudaGetErrorString(e));
}

bool known(int dtype) { return dtype == DT_F32 || dtype == DT_F16 || dtype == DT_BF16; }
size_t bytes_of(int dtype) { return dtype == DT_F32 ? 4 : 2; }

// Shape of a call, and the widest access that all its tensors allow.
struct Shape {
  const char* what;
  int64_t n[3];
  int dim;
  int64_t rows;
  int vec;

  int init(const char* name, const int64_t* shape, int64_t d, int64_t max_dim) {
    what = name;
    vec = 8;
    if (!shape) return fail(TRIATTN_EINVAL, what, "shape is NULL");
    if (d < 1) return fail(TRIATTN_EINVAL, what, "dim=%lld must be >= 1", (long long)d);
    if (d > max_dim)
      return fail(TRIATTN_EUNSUPPORTED, what, "dim=%lld above the supported %lld", (long long)d, (long long)max_dim);
    rows = 1;
    for (int k = 0; k < 3; ++k) {
      n[k] = shape[k];
      if (n[k] < 0) return fail(TRIATTN_EINVAL, what, "a negative size");
      if (n[k] > 0x7fffffffLL) return fail(TRIATTN_EUNSUPPORTED, what, "2^31 rows or more");
    }
    for (int k = 0; k < 3; ++k) {
      if (n[k] == 0) {
        rows = 0;
        break;
      }
      rows *= n[k];  // each factor and the product so far are below 2^31
      if (rows > 0x7fffffffLL - (1 << 20)) {
        // an empty axis further on still makes the call empty
        for (int l = k + 1; l < 3; ++l)
          if (n[l] == 0) rows = 0;
        if (rows) return fail(TRIATTN_EUNSUPPORTED, what, "about 2^31 rows or more");
        break;
      }
    }
    dim = (int)d;
    while (dim % vec) vec = vec == 8 ? 4 : 1;
    return TRIATTN_OK;
  }
  RowMap map() const { return RowMap::make(n, rows); }
  // A tensor of this shape: its strides (NULL = dense), and what they and its address allow.  `written`:
  // no two rows may share memory.
  int tensor(const char* name, const void* p, int dtype, const int64_t* strides, Strides3* out, bool written) {
    const size_t es = bytes_of(dtype);
    if (!p) return fail(TRIATTN_EINVAL, what, "%s is NULL", name);
    if (reinterpret_cast<uintptr_t>(p) % es) return fail(TRIATTN_EINVAL, what, "%s is not aligned to its elements", name);
    const int64_t dense[3] = {n[1] * n[2] * dim, n[2] * dim, dim};
    Strides3 s;
    s.dense = true;
    for (int k = 0; k < 3; ++k) {
      s.s[k] = strides ? strides[k] : dense[k];
      if (s.s[k] < 0) return fail(TRIATTN_EINVAL, what, "%s: negative stride", name);
      if (n[k] > 1 && s.s[k] != dense[k]) s.dense = false;
    }
    if (written && !s.dense) {  // from the smallest stride up, each must clear what lies below it
      int order[3] = {0, 1, 2};
      for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2 - i; ++j)
          if (s.s[order[j]] > s.s[order[j + 1]]) std::swap(order[j], order[j + 1]);
      int64_t extent = dim;
      for (int k : order) {
        if (n[k] <= 1) continue;
        if (s.s[k] < extent) return fail(TRIATTN_EINVAL, what, "%s: rows overlap", name);
        extent += s.s[k] * (n[k] - 1);
      }
    }
    // Dense rows need no check of the leading strides; others must allow the access at every row start.
    while (vec > 1) {
      bool ok = reinterpret_cast<uintptr_t>(p) % (vec * es < 16 ? vec * es : 16) == 0;
      for (int k = 0; k < 3; ++k) ok = ok && (n[k] <= 1 || s.s[k] % vec == 0);
      if (ok) break;
      vec = vec == 8 ? 4 : 1;
    }
    *out = s;
    return TRIATTN_OK;
  }
  // A tensor that is written and another one of the call: they share no memory, or, where `same` allows it, they are one
  // tensor under two names (a row is read before it is written, and by the lanes that write it).
  int apart(const char* written, const void* p, const Strides3& s, int dtype, const char* other, const void* q,
            const Strides3& t, int other_dtype, bool same) const {
    const int64_t es = (int64_t)bytes_of(dtype), et = (int64_t)bytes_of(other_dtype);
    const intptr_t delta = reinterpret_cast<intptr_t>(q) - reinterpret_cast<intptr_t>(p);
    bool strides = es == et;  // are the same
    for (int k = 0; k < 3; ++k) strides = strides && (n[k] <= 1 || s.s[k] == t.s[k]);
    if (same && delta == 0 && strides && dtype == other_dtype) return TRIATTN_OK;
    if (!meet(s, es, t, et, strides, delta)) return TRIATTN_OK;
    return fail(TRIATTN_EINVAL, what, "%s overlaps %s%s", written, other, same ? " with other strides, or in part" : "");
  }
  // Whether rows of dim elements at strides s and, delta bytes further on, at strides t can have a byte in common.  Exact for
  // equal strides, and where both lie at multiples of a common pitch; else as their ranges say.
  bool meet(const Strides3& s, int64_t es, const Strides3& t, int64_t et, bool equal, int64_t delta) const {
    const int64_t ws = dim * es, wt = dim * et;  // bytes of a row
    int64_t last_s = 0, last_t = 0, pitch = 0;
    for (int k = 0; k < 3; ++k) {
      if (n[k] <= 1) continue;
      last_s += s.s[k] * es * (n[k] - 1);
      last_t += t.s[k] * et * (n[k] - 1);
      pitch = std::gcd(pitch, std::gcd(s.s[k] * es, t.s[k] * et));
    }
    if (delta >= last_s + ws || -delta >= last_t + wt) return false;
    if (pitch > 0) {  // side by side in every pitch
      const int64_t d = (delta % pitch + pitch) % pitch;
      if (d >= ws && pitch - d >= wt) return false;
    }
    if (!equal) return true;
    // rows i of one and j of the other lie delta + sum of (j - i) strides apart
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) { return s.s[a] > s.s[b]; });
    const auto near = [&](const auto& self, int at, int64_t d) -> bool {
      if (at == 3) return d < ws && -d < wt;
      const int k = order[at];
      if (n[k] <= 1 || s.s[k] == 0) return self(self, at + 1, d);
      int64_t rest = 0;  // what the smaller strides add at most
      for (int l = at + 1; l < 3; ++l) rest += n[order[l]] > 1 ? s.s[order[l]] * es * (n[order[l]] - 1) : 0;
      const int64_t step = s.s[k] * es, around = -d / step, more = (rest + (ws > wt ? ws : wt)) / step + 2;
      for (int64_t j = around - more; j <= around + more; ++j)
        if (j > -n[k] && j < n[k] && self(self, at + 1, d + j * step)) return true;
      return false;
    };
    return near(near, 0, delta);
  }
  // `share`: bit k = axis k (3: the channels) shares one draw
  int dropout(int share, double p, uint64_t seed, uint64_t offset, const uint64_t* state, Dropout* out) const {
    if (!(p >= 0.0 && p <= 1.0)) return fail(TRIATTN_EINVAL, what, "p=%g must lie in [0, 1]", p);
    if (share < 0 || share > 15) return fail(TRIATTN_EINVAL, what, "share=%d is not a set of the axes 0..3", share);
    if (reinterpret_cast<uintptr_t>(state) % 8) return fail(TRIATTN_EINVAL, what, "rng_state must be 8-byte aligned");
    Dropout d{};
    const uint64_t threshold = (uint64_t)(p * 4294967296.0 + 0.5);  // a word below it is dropped
    d.on = threshold > 0;
    d.drop_max = d.on ? (uint32_t)(threshold - 1) : 0;
    d.scale = !d.on ? 1.0f : p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
    for (auto& k : d.key) {
      k[0] = k0;
      k[1] = k1;
      k0 += PHILOX_W0;
      k1 += PHILOX_W1;
    }
    d.offset = offset;
    d.state = state;
    d.per_channel = share >> 3 & 1 ? 0 : 1;
    int64_t m = d.per_channel ? dim : 1;
    for (int k = 2; k >= 0; --k) {
      d.m[k] = share >> k & 1 ? 0 : m;
      if (!(share >> k & 1)) m *= n[k];
    }
    *out = d;
    return TRIATTN_OK;
  }
};

// The type pairs that the kernels are built for: an fp32 stream with an fp32 or 16-bit result, or one
// 16-bit type throughout; y in the stream's type or in the result's.
int check_types(const char* what, int z, int y, int out) {
  if (!known(z) || !known(y) || !known(out)) return fail(TRIATTN_EUNSUPPORTED, what, "dtype %d, %d, %d", z, y, out);
  const bool ok = z == DT_F32 ? (y == DT_F32 || y == out) : (y == z && out == z);
  return ok ? TRIATTN_OK : fail(TRIATTN_EUNSUPPORTED, what, "type combination %d, %d -> %d", z, y, out);
}

int check_params(const char* what, const void* w, const void* b, int dtype, float eps) {
  if (!known(dtype)) return fail(TRIATTN_EUNSUPPORTED, what, "parameter dtype %d", dtype);
  const size_t es = bytes_of(dtype);
  if (reinterpret_cast<uintptr_t>(w) % es || reinterpret_cast<uintptr_t>(b) % es)
    return fail(TRIATTN_EINVAL, what, "a parameter is not aligned to its elements");
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail(TRIATTN_EINVAL, what, "eps=%g must be finite and >= 0", (double)eps);
  return TRIATTN_OK;
}

int check_stats(const char* what, const float* mean, const float* rstd) {
  if (!mean != !rstd) return fail(TRIATTN_EINVAL, what, "mean without rstd, or rstd without mean");
  if (reinterpret_cast<uintptr_t>(mean) % 4 || reinterpret_cast<uintptr_t>(rstd) % 4)
    return fail(TRIATTN_EINVAL, what, "mean / rstd are not aligned to their elements");
  return TRIATTN_OK;
}

// Narrow rows that leave over a quarter of the row form's lanes idle, which draw all the same (draws per channel cost the
// most).  2^24 elements with draws shared along an axis, by rows / by chunks in us.  Whole pieces on lanes for 8, 16 or 32:
// fp32 8 channels 111 / 37, 40: 47 / 37, 72: 50 / 38, bf16 72: 40 / 37 (and not: fp32 64: 34 / 38, 96: 41 / 38, bf16 96:
// 34 / 37).  Odd widths on lanes for 32, 64 or 128 channels: fp32 13: 135 / 104, 38: 102 / 83, 66: 115 / 83 (and not: 27:
// 76 / 104, 55: 72 / 101, 107: 75 / 95).  16-bit rows of four-element pieces, which chunks read one by one: bf16 4: 207 / 82
// (and not: 12: 71 / 86, 100: 39 / 86).
bool leaves_lanes_idle(int dim, int vec, int full) {
  if (dim <= 8) return true;
  if (vec > 1 && vec < full) return false;
  int held = vec == 1 ? 32 : 8 * full;
  const int most = vec == 1 ? 128 : 32 * full;
  if (dim > most) return false;
  while (held < dim) held *= 2;
  return 4 * dim < 3 * held;
}

// Every tensor is dense, and every element has a position of its own, the elements' order (or nothing is dropped).
bool is_vector(const DropoutAddArgs& a) {
  const int64_t m2 = a.dim, m1 = m2 * a.map.n2.d, m0 = m1 * a.map.n1.d;
  const bool own = !a.drop.on || (a.drop.per_channel && (a.map.n2.d == 1 || a.drop.m[2] == m2) &&
                                  (a.map.n1.d == 1 || a.drop.m[1] == m1) &&
                                  (a.map.rows == a.map.n1.d * a.map.n2.d || a.drop.m[0] == m0));
  return own && (!a.z || a.zs.dense) && a.ys.dense && a.os.dense;
}

}  // namespace

extern "C" {

int triattn_layer_norm(const void* x, int x_dtype, const int64_t* x_strides, const int64_t* shape, int64_t dim,
                       const void* weight, const void* bias, int param_dtype, float eps, void* out, int out_dtype,
                       const int64_t* out_strides, float* mean, float* rstd, void* stream) {
  const char* what = "layer_norm";
  Shape s;
  if (int r = s.init(what, shape, dim, RES_MAX_DIM)) return r;
  if (int r = check_types(what, x_dtype, x_dtype, out_dtype)) return r;
  if (int r = check_params(what, weight, bias, param_dtype, eps)) return r;
  if (int r = check_stats(what, mean, rstd)) return r;
  if (s.rows == 0) return TRIATTN_OK;
  NormFwdArgs a{};
  if (int r = s.tensor("x", x, x_dtype, x_strides, &a.zs, false)) return r;
  if (int r = s.tensor("out", out, out_dtype, out_strides, &a.os, true)) return r;
  if (int r = s.apart("out", out, a.os, out_dtype, "x", x, a.zs, x_dtype, false)) return r;
  a.z = x; a.out = out; a.map = s.map(); a.dim = s.dim;
  a.weight = weight; a.bias = bias; a.param_dtype = param_dtype; a.eps = eps;
  a.mean = mean; a.rstd = rstd;
  return finish(launch_norm_fwd(a, x_dtype, out_dtype, s.vec, static_cast<cudaStream_t>(stream)), what);
}

int triattn_dropout_add(const void* z, int z_dtype, const int64_t* z_strides, const void* y, int y_dtype,
                        const int64_t* y_strides, const int64_t* shape, int64_t dim, int share, double p, uint64_t seed,
                        uint64_t offset, const uint64_t* rng_state, void* out, int out_dtype,
                        const int64_t* out_strides, void* stream) {
  const char* what = "dropout_add";
  Shape s;
  DropoutAddArgs a{};
  if (int r = s.init(what, shape, dim, 1 << 30)) return r;
  if (!known(y_dtype) || !known(out_dtype) || (z && z_dtype != out_dtype))
    return fail(TRIATTN_EUNSUPPORTED, what, "type combination %d, %d -> %d", z ? z_dtype : -1, y_dtype, out_dtype);
  if (z ? (out_dtype != DT_F32 && y_dtype != out_dtype) : (y_dtype != DT_F32 && y_dtype != out_dtype))
    return fail(TRIATTN_EUNSUPPORTED, what, "type combination %d, %d -> %d", z ? z_dtype : -1, y_dtype, out_dtype);
  if (int r = s.dropout(share, p, seed, offset, rng_state, &a.drop)) return r;
  if (s.rows == 0) return TRIATTN_OK;
  if (z)
    if (int r = s.tensor("z", z, z_dtype, z_strides, &a.zs, false)) return r;
  if (int r = s.tensor("y", y, y_dtype, y_strides, &a.ys, false)) return r;
  if (int r = s.tensor("out", out, out_dtype, out_strides, &a.os, true)) return r;
  a.z = z; a.y = y; a.out = out; a.map = s.map(); a.dim = s.dim;
  a.in_place = z == out;
  if (z)
    if (int r = s.apart("out", out, a.os, out_dtype, "z", z, a.zs, z_dtype, true)) return r;
  if (int r = s.apart("out", out, a.os, out_dtype, "y", y, a.ys, y_dtype, true)) return r;
  // By chunks: one long vector, rows of more than 8192 channels, and what leaves_lanes_idle names.  Else by rows: which of
  // them are dropped whole is then known a batch ahead, and what is dropped is not read (N=1024, one draw per row: 218 us
  // against 280 by chunks; 8192 x 4096 bf16: 28 against 55), and the loads run ahead of the draws (8192 x 4096 bf16, draws
  // shared along an axis: 43 against 70).
  const int full = y_dtype != DT_F32 && out_dtype != DT_F32 ? 8 : 4;
  const bool dense = (!z || a.zs.dense) && a.ys.dense && a.os.dense;
  if (s.dim <= RES_MAX_DIM && !is_vector(a) && !(a.drop.on && a.drop.per_channel && dense && leaves_lanes_idle(s.dim, s.vec, full))) {
    NormFwdArgs f{};
    f.z = z; f.y = y; f.sum = out;
    f.zs = z ? a.zs : a.os; f.ys = a.ys; f.ss = f.os = a.os;
    f.map = a.map; f.dim = a.dim; f.in_place = a.in_place; f.drop = a.drop;
    return finish(launch_dropout_rows(f, y_dtype, out_dtype, s.vec, static_cast<cudaStream_t>(stream)), what);
  }
  a.vector = is_vector(a);
  // A 16-bit vector goes by rows, too, cut into rows of a warp's 256 elements, whose loads run ahead of the draws (16384 x
  // 1024 bf16: 27 us against 34 by chunks; fp32, with twice the traffic for each draw, gains nothing).
  const int64_t n = s.rows * s.dim;
  if (a.vector && full == 8 && s.vec == 8 && n % 256 == 0 && n / 256 < 0x7fffffffLL - (1 << 20)) {
    NormFwdArgs f{};
    f.z = z; f.y = y; f.sum = out;
    f.zs = f.ys = f.ss = f.os = a.os;
    f.dim = 256; f.in_place = a.in_place; f.drop = a.drop;
    const int64_t shape1[3] = {1, 1, n / 256};
    f.map = RowMap::make(shape1, n / 256);
    f.drop.m[0] = f.drop.m[1] = 0;
    f.drop.m[2] = 256;
    return finish(launch_dropout_rows(f, y_dtype, out_dtype, 8, static_cast<cudaStream_t>(stream)), what);
  }
  return finish(launch_dropout_add(a, z_dtype, y_dtype, out_dtype, s.vec, static_cast<cudaStream_t>(stream)), what);
}

int triattn_dropout_add_layer_norm(const void* z, int z_dtype, const int64_t* z_strides, const void* y, int y_dtype,
                                   const int64_t* y_strides, const int64_t* shape, int64_t dim, int share, double p,
                                   uint64_t seed, uint64_t offset, const uint64_t* rng_state, const void* weight,
                                   const void* bias, int param_dtype, float eps, void* sum, const int64_t* sum_strides,
                                   void* out, int out_dtype, const int64_t* out_strides, float* mean, float* rstd,
                                   void* stream) {
  const char* what = "dropout_add_layer_norm";
  Shape s;
  NormFwdArgs a{};
  if (int r = s.init(what, shape, dim, RES_MAX_DIM)) return r;
  if (int r = check_types(what, z_dtype, y_dtype, out_dtype)) return r;
  if (int r = check_params(what, weight, bias, param_dtype, eps)) return r;
  if (int r = check_stats(what, mean, rstd)) return r;
  if (int r = s.dropout(share, p, seed, offset, rng_state, &a.drop)) return r;
  if (s.rows == 0) return TRIATTN_OK;
  if (int r = s.tensor("z", z, z_dtype, z_strides, &a.zs, false)) return r;
  if (int r = s.tensor("y", y, y_dtype, y_strides, &a.ys, false)) return r;
  if (int r = s.tensor("sum", sum, z_dtype, sum_strides, &a.ss, true)) return r;
  if (int r = s.tensor("out", out, out_dtype, out_strides, &a.os, true)) return r;
  if (int r = s.apart("sum", sum, a.ss, z_dtype, "z", z, a.zs, z_dtype, true)) return r;
  if (int r = s.apart("sum", sum, a.ss, z_dtype, "y", y, a.ys, y_dtype, true)) return r;
  if (int r = s.apart("out", out, a.os, out_dtype, "z", z, a.zs, z_dtype, false)) return r;
  if (int r = s.apart("out", out, a.os, out_dtype, "y", y, a.ys, y_dtype, true)) return r;
  if (int r = s.apart("out", out, a.os, out_dtype, "sum", sum, a.ss, z_dtype, false)) return r;
  a.z = z; a.y = y; a.sum = sum; a.out = out; a.map = s.map(); a.dim = s.dim;
  a.weight = weight; a.bias = bias; a.param_dtype = param_dtype; a.eps = eps;
  a.mean = mean; a.rstd = rstd;
  return finish(launch_fused_fwd(a, z_dtype, y_dtype, out_dtype, s.vec, static_cast<cudaStream_t>(stream)), what);
}

size_t triattn_layer_norm_backward_workspace_bytes(int64_t rows, int64_t dim) {
  if (rows < 1 || dim < 1 || dim > RES_MAX_DIM) return 0;
  const int64_t ctas = norm_bwd_max_ctas();  // a CTA has one row at least
  return (size_t)(rows < ctas ? rows : ctas) * 2 * (size_t)dim * sizeof(float);
}

int triattn_layer_norm_backward(const void* dout, int dout_dtype, const int64_t* dout_strides, const void* x, int x_dtype,
                                const int64_t* x_strides, const int64_t* shape, int64_t dim, const void* weight,
                                int param_dtype, const float* mean, const float* rstd, const void* dsum,
                                const int64_t* dsum_strides, int share, double p, uint64_t seed, uint64_t offset,
                                const uint64_t* rng_state, void* dx, void* dy, int y_dtype, void* dweight, void* dbias,
                                void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "layer_norm_backward";
  Shape s;
  NormBwdArgs a{};
  Strides3 dense;
  struct Written {
    const char* name;
    const void* p;
    int dtype;
  };
  if (int r = s.init(what, shape, dim, RES_MAX_DIM)) return r;
  if (!dy) y_dtype = x_dtype;
  if (int r = check_types(what, x_dtype, y_dtype, dout_dtype)) return r;
  if (int r = check_params(what, weight, dweight, param_dtype, 0.0f)) return r;
  if (int r = check_params(what, weight, dbias, param_dtype, 0.0f)) return r;
  if (int r = s.dropout(share, p, seed, offset, rng_state, &a.drop)) return r;
  if (s.rows && (dweight || dbias)) {
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)
      return fail(TRIATTN_EINVAL, what, "dweight / dbias need a 16-byte aligned workspace");
    const size_t need = triattn_layer_norm_backward_workspace_bytes(s.rows, dim);
    if (workspace_bytes < need) return fail(TRIATTN_ENOSPACE, what, "workspace %zu bytes < %zu needed", workspace_bytes, need);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (s.rows == 0) {  // empty sums
    const size_t n = (size_t)dim * bytes_of(param_dtype);
    if (dweight)
      if (int r = finish(cudaMemsetAsync(dweight, 0, n, st), what)) return r;
    if (dbias)
      if (int r = finish(cudaMemsetAsync(dbias, 0, n, st), what)) return r;
    return TRIATTN_OK;
  }
  if (!mean || !rstd) return fail(TRIATTN_EINVAL, what, "mean / rstd are NULL");
  if (int r = check_stats(what, mean, rstd)) return r;
  if (int r = s.tensor("dout", dout, dout_dtype, dout_strides, &a.dos, false)) return r;
  if (int r = s.tensor("x", x, x_dtype, x_strides, &a.xs, false)) return r;
  if (dsum)
    if (int r = s.tensor("dsum", dsum, x_dtype, dsum_strides, &a.dss, false)) return r;
  if (dx)
    if (int r = s.tensor("dx", dx, x_dtype, nullptr, &dense, true)) return r;
  if (dy)
    if (int r = s.tensor("dy", dy, y_dtype, nullptr, &dense, true)) return r;
  for (const auto& [name, p, dtype] : {Written{"dx", dx, x_dtype}, Written{"dy", dy, y_dtype}}) {
    if (!p) continue;
    if (int r = s.apart(name, p, dense, dtype, "dout", dout, a.dos, dout_dtype, true)) return r;
    if (int r = s.apart(name, p, dense, dtype, "x", x, a.xs, x_dtype, true)) return r;
    if (dsum)
      if (int r = s.apart(name, p, dense, dtype, "dsum", dsum, a.dss, x_dtype, true)) return r;
  }
  if (dx && dy)
    if (int r = s.apart("dx", dx, dense, x_dtype, "dy", dy, dense, y_dtype, false)) return r;
  if (!dx && !dy && !dweight && !dbias) return TRIATTN_OK;
  a.dout = dout; a.x = x; a.ds = dsum; a.map = s.map(); a.dim = s.dim;
  a.weight = weight; a.param_dtype = param_dtype; a.mean = mean; a.rstd = rstd;
  a.dx = dx; a.dy = dy; a.dweight = dweight; a.dbias = dbias;
  a.partial = dweight || dbias ? static_cast<float*>(workspace) : nullptr;
  const bool fused = dy || dsum;
  return finish(fused ? launch_fused_bwd(a, x_dtype, y_dtype, dout_dtype, s.vec, st)
                      : launch_norm_bwd(a, x_dtype, dout_dtype, s.vec, st),
                what);
}

}  // extern "C"
