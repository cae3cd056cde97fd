// glu.hip -- the gated feed-forward block and its gradients (include/ggemm_glu.h).
#include <algorithm>
#include <type_traits>

#include "simple.hpp"

namespace ggemm {
namespace {

template <class T>
__device__ __forceinline__ float as_f(const void* p, int64_t i) { return (float)static_cast<const T*>(p)[i]; }

// The row of x that row r stands for, -1: none.
__device__ __forceinline__ int64_t source_row(const ggemm_glu_t& p, int r) {
  if (!p.index) return r;
  const int i = p.index[r];
  return i >= 0 && i < p.x_rows ? i : -1;
}

// h, gate, up
template <class T, int ACT>
struct Up {
  using Acc = float;
  static constexpr int kPairs = 2;
  ggemm_glu_t p;
  T* h;
  int64_t ldh;
  int g, lo, hi, n0;
  __device__ bool place(int t) {
    if (!simple_rows(p.offsets, p.groups, p.rows, ceil_div(p.d_ff, 64), t, g, lo, hi, n0)) return false;
    n0 *= 64;
    return true;
  }
  __device__ int depth() const { return p.d_model; }
  __device__ float a(int i, int k) const {
    if (lo + i >= hi || k >= p.d_model) return 0.0f;
    const int64_t s = source_row(p, lo + i);
    return s < 0 ? 0.0f : as_f<T>(p.x, s * p.ldx + k);
  }
  __device__ float b(int z, int j, int k) const {
    if (n0 + j >= p.d_ff || k >= p.d_model) return 0.0f;
    return as_f<T>(z ? p.w_up : p.w_gate, g * p.w_stride + (n0 + j) * p.ldw + k);
  }
  __device__ void emit(int i, int j, const float* s) const {
    if (lo + i >= hi || n0 + j >= p.d_ff) return;
    const int64_t r = lo + i, c = n0 + j;
    h[r * ldh + c] = (T)(act_value<ACT>(s[0]) * s[1]);
    if (p.gate) {
      static_cast<T*>(p.gate)[r * p.ldg + c] = (T)s[0];
      static_cast<T*>(p.up)[r * p.ldg + c] = (T)s[1];
    }
  }
};

// y = h Wd^T
template <class T>
struct Down {
  using Acc = float;
  static constexpr int kPairs = 1;
  ggemm_glu_t p;
  const T* h;
  int64_t ldh;
  int g, lo, hi, n0;
  __device__ bool place(int t) {
    if (!simple_rows(p.offsets, p.groups, p.rows, ceil_div(p.d_model, 64), t, g, lo, hi, n0)) return false;
    n0 *= 64;
    return true;
  }
  __device__ int depth() const { return p.d_ff; }
  __device__ float a(int i, int k) const { return lo + i < hi && k < p.d_ff ? (float)h[(lo + i) * ldh + k] : 0.0f; }
  __device__ float b(int, int j, int k) const {
    return n0 + j < p.d_model && k < p.d_ff ? as_f<T>(p.w_down, g * p.d_stride + (n0 + j) * p.ldd + k) : 0.0f;
  }
  __device__ void emit(int i, int j, const float* s) const {
    if (lo + i < hi && n0 + j < p.d_model) static_cast<T*>(p.y)[(lo + i) * p.ldy + n0 + j] = (T)s[0];
  }
};

// dh = dy Wd, and from it dgate, dup and h
template <class T, int ACT>
struct Inner {
  using Acc = float;
  static constexpr int kPairs = 1;
  ggemm_glu_t p;
  ggemm_glu_grad_t d;
  T *dg, *du, *h;
  int64_t ldh;
  int g, lo, hi, n0;
  __device__ bool place(int t) {
    if (!simple_rows(p.offsets, p.groups, p.rows, ceil_div(p.d_ff, 64), t, g, lo, hi, n0)) return false;
    n0 *= 64;
    return true;
  }
  __device__ int depth() const { return p.d_model; }
  __device__ float a(int i, int k) const { return lo + i < hi && k < p.d_model ? as_f<T>(d.dy, (lo + i) * d.lddy + k) : 0.0f; }
  __device__ float b(int, int j, int k) const {
    return n0 + j < p.d_ff && k < p.d_model ? as_f<T>(p.w_down, g * p.d_stride + k * p.ldd + n0 + j) : 0.0f;
  }
  __device__ void emit(int i, int j, const float* s) const {
    if (lo + i >= hi || n0 + j >= p.d_ff) return;
    const int64_t r = lo + i, c = n0 + j;
    const bool live = source_row(p, (int)r) >= 0;
    const float v = as_f<T>(p.gate, r * p.ldg + c), u = as_f<T>(p.up, r * p.ldg + c);
    float q, dq;
    act_parts<ACT>(v, q, dq);
    dg[r * ldh + c] = live ? (T)(s[0] * u * (q + v * dq)) : (T)0.0f;
    du[r * ldh + c] = live ? (T)(s[0] * (v * q)) : (T)0.0f;
    h[r * ldh + c] = live ? (T)(v * q * u) : (T)0.0f;
  }
};

// dx = dgate Wg + dup Wu
template <class T>
struct Dx {
  using Acc = float;
  static constexpr int kPairs = 1;
  ggemm_glu_t p;
  ggemm_glu_grad_t d;
  const T *dg, *du;
  int64_t ldh;
  int g, lo, hi, n0;
  __device__ bool place(int t) {
    if (!simple_rows(p.offsets, p.groups, p.rows, ceil_div(p.d_model, 64), t, g, lo, hi, n0)) return false;
    n0 *= 64;
    return true;
  }
  __device__ int depth() const { return 2 * p.d_ff; }
  __device__ float a(int i, int k) const {
    if (lo + i >= hi || k >= 2 * p.d_ff) return 0.0f;
    return k < p.d_ff ? (float)dg[(lo + i) * ldh + k] : (float)du[(lo + i) * ldh + k - p.d_ff];
  }
  __device__ float b(int, int j, int k) const {
    if (n0 + j >= p.d_model || k >= 2 * p.d_ff) return 0.0f;
    return k < p.d_ff ? as_f<T>(p.w_gate, g * p.w_stride + k * p.ldw + n0 + j)
                      : as_f<T>(p.w_up, g * p.w_stride + (k - p.d_ff) * p.ldw + n0 + j);
  }
  __device__ void emit(int i, int j, const float* s) const {
    if (lo + i < hi && n0 + j < p.d_model) static_cast<T*>(d.dx)[(lo + i) * d.lddx + n0 + j] = (T)s[0];
  }
};

// Gradients of the weights: dWg = dgate^T x and dWu = dup^T x (kDown false, z = 0, 1), dWd = dy^T h
template <class T, class W, bool kDown>
struct Dw {
  using Acc = float;
  static constexpr int kPairs = 1;
  ggemm_glu_t p;
  ggemm_glu_grad_t d;
  const T *left, *right;
  int64_t ldl, ldr;
  W* out;
  int g, lo, hi, m0, n0;
  __device__ int m() const { return kDown ? p.d_model : p.d_ff; }
  __device__ int n() const { return kDown ? p.d_ff : p.d_model; }
  __device__ bool place(int t) {
    const int mt = ceil_div(m(), 64), nt = ceil_div(n(), 64);
    g = t / (mt * nt);
    m0 = t / nt % mt * 64;
    n0 = t % nt * 64;
    lo = p.offsets ? min(max(p.offsets[g], 0), p.rows) : 0;
    hi = p.offsets ? min(max(p.offsets[g + 1], 0), p.rows) : p.rows;
    return true;
  }
  __device__ int depth() const { return max(hi - lo, 0); }
  __device__ float a(int i, int k) const {
    if (lo + k >= hi || m0 + i >= m()) return 0.0f;
    return source_row(p, lo + k) < 0 ? 0.0f : (float)left[(lo + k) * ldl + m0 + i];
  }
  __device__ float b(int, int j, int k) const {
    if (lo + k >= hi || n0 + j >= n()) return 0.0f;
    const int64_t s = source_row(p, lo + k);
    return s < 0 ? 0.0f : (float)right[(kDown ? lo + k : s) * ldr + n0 + j];
  }
  __device__ void emit(int i, int j, const float* s) const {
    if (m0 + i >= m() || n0 + j >= n()) return;
    W* const c = out + (kDown ? g * d.dd_stride + (m0 + i) * d.lddd : g * d.dw_stride + (m0 + i) * d.lddw) + n0 + j;
    *c = (W)(d.dw_beta != 0.0f ? s[0] + d.dw_beta * (float)*c : s[0]);
  }
};

bool rows_ok(const void* x, int64_t ld, int cols) { return x && aligned(x, 16) && ld % 8 == 0 && ld >= cols && ld <= GGEMM_GLU_MAX_LD; }

// Sizes and leading dimensions.
bool shape_ok(const ggemm_glu_t* p) {
  if (!p || p->groups < 1 || p->groups > GGEMM_GLU_MAX_GROUPS || p->rows < 0 || p->d_model < 1 || p->d_ff < 1 ||
      p->d_model > GGEMM_GLU_MAX_LD || p->d_ff > GGEMM_GLU_MAX_LD || (p->dtype != GGEMM_BF16 && p->dtype != GGEMM_F16) ||
      !act_known(p->act))
    return false;
  auto pitch = [](int64_t ld, int cols) { return ld % 8 == 0 && ld >= cols && ld <= GGEMM_GLU_MAX_LD; };
  return pitch(p->ldx, p->d_model) && pitch(p->ldw, p->d_model) && pitch(p->ldd, p->d_ff) && p->w_stride % 8 == 0 && p->d_stride % 8 == 0;
}
bool args_ok(const ggemm_glu_t* p) {
  if (!shape_ok(p) || (!p->offsets && p->groups != 1) || !aligned(p->offsets, 4) || !aligned(p->index, 4)) return false;
  if (p->index && (p->x_rows < 0 || p->x_rows * p->ldx >= (1 << 30))) return false;
  if (p->rows == 0) return true;
  if ((!p->x && !(p->index && p->x_rows == 0)) || !aligned(p->x, 16)) return false;
  return p->w_gate && p->w_up && p->w_down && aligned(p->w_gate, 16) && aligned(p->w_up, 16) && aligned(p->w_down, 16);
}
int64_t ld_hidden(const ggemm_glu_t& p) { return (int64_t)align_up((size_t)p.d_ff, 8); }
size_t hidden_bytes(const ggemm_glu_t& p) { return align_up((size_t)p.rows * ld_hidden(p) * 2, 256); }
int64_t row_tiles(const ggemm_glu_t& p, int tm) { return p.groups > 1 ? (int64_t)p.rows / tm + std::min(p.groups, p.rows) : ceil_div(p.rows, tm); }

}  // namespace

size_t glu_workspace(const ggemm_glu_t* p) { return shape_ok(p) ? hidden_bytes(*p) : 0; }

int glu(const ggemm_glu_t* p, void* ws, size_t ws_bytes, hipStream_t s) {
  if (!args_ok(p) || !p->gate != !p->up) return GGEMM_ERR_INVALID;
  if (p->rows == 0) return GGEMM_OK;
  if (!p->y || !aligned(p->y, 2) || p->ldy < p->d_model) return GGEMM_ERR_INVALID;
  if (p->gate && (!aligned(p->gate, 2) || !aligned(p->up, 2) || p->ldg < p->d_ff)) return GGEMM_ERR_INVALID;
  if (ws_bytes < glu_workspace(p)) return GGEMM_ERR_WORKSPACE;
  if (!ws || !aligned(ws, 16)) return GGEMM_ERR_INVALID;
  const int64_t up = row_tiles(*p, 64) * ceil_div(p->d_ff, 64), down = row_tiles(*p, 64) * ceil_div(p->d_model, 64);
  if (std::max(up, down) >= (1 << 23)) return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(p->dtype, [&](auto dt) { with_act(p->act, [&](auto act) {
    if constexpr (decltype(dt)::value != GGEMM_F32) {
      using T = typename Elem<decltype(dt)::value>::T;
      T* const h = static_cast<T*>(ws);
      simple_kernel<<<(unsigned)up, 256, 0, s>>>(Up<T, decltype(act)::value>{*p, h, ld_hidden(*p)});
      simple_kernel<<<(unsigned)down, 256, 0, s>>>(Down<T>{*p, h, ld_hidden(*p)});
    }
  }); }); });
}

size_t glu_backward_workspace(const ggemm_glu_t* p, const ggemm_glu_grad_t* d) {
  return shape_ok(p) && d ? 3 * hidden_bytes(*p) : 0;
}

int glu_backward(const ggemm_glu_t* p, const ggemm_glu_grad_t* d, void* ws, size_t ws_bytes, hipStream_t s) {
  if (!args_ok(p) || !d || !elem_known(d->dw_dtype) || !d->dw_gate != !d->dw_up) return GGEMM_ERR_INVALID;
  const size_t es = elem_bytes(d->dw_dtype);
  auto grads = [&](const void* w, int64_t ld, int64_t stride, int m, int n) {
    return !w || (aligned(w, es) && ld >= n && (p->groups == 1 || stride >= (m - 1) * ld + n));
  };
  if (!grads(d->dw_gate, d->lddw, d->dw_stride, p->d_ff, p->d_model) || !grads(d->dw_up, d->lddw, d->dw_stride, p->d_ff, p->d_model) ||
      !grads(d->dw_down, d->lddd, d->dd_stride, p->d_model, p->d_ff))
    return GGEMM_ERR_INVALID;
  if (p->rows > 0 && (!rows_ok(d->dy, d->lddy, p->d_model) || !p->gate || !p->up || !aligned(p->gate, 2) || !aligned(p->up, 2) ||
                      p->ldg < p->d_ff || (d->dx && (!aligned(d->dx, 2) || d->lddx < p->d_model))))
    return GGEMM_ERR_INVALID;
  if (ws_bytes < glu_backward_workspace(p, d)) return GGEMM_ERR_WORKSPACE;
  if (p->rows > 0 && (!ws || !aligned(ws, 16))) return GGEMM_ERR_INVALID;
  const int64_t in = row_tiles(*p, 64) * ceil_div(p->d_ff, 64), dx = row_tiles(*p, 64) * ceil_div(p->d_model, 64);
  const int64_t dw = (int64_t)p->groups * ceil_div(p->d_ff, 64) * ceil_div(p->d_model, 64);
  if (std::max(std::max(in, dx), dw) >= (1 << 23)) return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(p->dtype, [&](auto dt) { with_act(p->act, [&](auto act) { with_elem(d->dw_dtype, [&](auto wt) {
    if constexpr (decltype(dt)::value != GGEMM_F32) {
      using T = typename Elem<decltype(dt)::value>::T;
      using W = typename Elem<decltype(wt)::value>::T;
      uint8_t* const b = static_cast<uint8_t*>(ws);
      const size_t n = hidden_bytes(*p);
      T *const dg = reinterpret_cast<T*>(b), *const du = reinterpret_cast<T*>(b + n), *const h = reinterpret_cast<T*>(b + 2 * n);
      const int64_t ldh = ld_hidden(*p);
      if (in) simple_kernel<<<(unsigned)in, 256, 0, s>>>(Inner<T, decltype(act)::value>{*p, *d, dg, du, h, ldh});
      if (dx && d->dx) simple_kernel<<<(unsigned)dx, 256, 0, s>>>(Dx<T>{*p, *d, dg, du, ldh});
      if (d->dw_gate) {
        simple_kernel<<<(unsigned)dw, 256, 0, s>>>(Dw<T, W, false>{*p, *d, dg, static_cast<const T*>(p->x), ldh, p->ldx, static_cast<W*>(d->dw_gate)});
        simple_kernel<<<(unsigned)dw, 256, 0, s>>>(Dw<T, W, false>{*p, *d, du, static_cast<const T*>(p->x), ldh, p->ldx, static_cast<W*>(d->dw_up)});
      }
      if (d->dw_down)
        simple_kernel<<<(unsigned)dw, 256, 0, s>>>(Dw<T, W, true>{*p, *d, static_cast<const T*>(d->dy), h, d->lddy, ldh, static_cast<W*>(d->dw_down)});
    }
  }); }); }); });
}

}  // namespace ggemm

extern "C" size_t ggemm_glu_workspace(const ggemm_glu_t* p) { return ggemm::glu_workspace(p); }
extern "C" int ggemm_glu(const ggemm_glu_t* p, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  return ggemm::glu(p, workspace, workspace_bytes, stream);
}
extern "C" size_t ggemm_glu_backward_workspace(const ggemm_glu_t* p, const ggemm_glu_grad_t* d) { return ggemm::glu_backward_workspace(p, d); }
extern "C" int ggemm_glu_backward(const ggemm_glu_t* p, const ggemm_glu_grad_t* d, void* workspace, size_t workspace_bytes,
                                  hipStream_t stream) {
  return ggemm::glu_backward(p, d, workspace, workspace_bytes, stream);
}
