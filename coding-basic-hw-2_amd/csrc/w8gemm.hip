// w8gemm.hip -- grouped products of 8-bit integers with scales for rows and columns (include/ggemm_w8.h).
#include <algorithm>
#include <type_traits>

#include "ggemm_w8.h"
#include "simple.hpp"

namespace ggemm {
namespace {

template <class T, int ACT>
struct Product {
  using Acc = int;
  static constexpr int kPairs = ACT ? 2 : 1;
  ggemm_w8_gemm_t p;
  int g, lo, hi, n0;
  __device__ bool place(int t) {
    if (!simple_rows(p.offsets, p.groups, p.m, ceil_div(p.n, 64), t, g, lo, hi, n0)) return false;
    n0 *= 64;
    return true;
  }
  __device__ int depth() const { return p.k; }
  __device__ int a(int i, int k) const { return lo + i < hi && k < p.k ? p.a[(lo + i) * p.lda + k] : 0; }
  __device__ int b(int z, int j, int k) const {
    return n0 + j < p.n && k < p.k ? (z ? p.b_up : p.b)[g * p.b_stride + (n0 + j) * p.ldb + k] : 0;
  }
  __device__ void emit(int i, int j, const int* s) const {
    if (lo + i >= hi || n0 + j >= p.n) return;
    const int64_t c = g * p.b_scales_stride + n0 + j;
    float v = (float)s[0] * p.a_scales[lo + i] * p.b_scales[c];
    if constexpr (ACT != 0) v = act_value<ACT>(v) * ((float)s[1] * p.a_scales[lo + i] * p.b_up_scales[c]);
    static_cast<T*>(p.c)[(lo + i) * p.ldc + n0 + j] = (T)v;
  }
};

// Sizes, leading dimensions and strides.
bool shape_ok(const ggemm_w8_gemm_t* p) {
  if (!p || p->groups < 1 || p->groups > GGEMM_W8_MAX_GROUPS || p->m < 0 || p->n < 0 || p->k < 0 || p->k >= GGEMM_W8_MAX_COLS ||
      !elem_known(p->dtype) || (p->act != 0 && !act_known(p->act)))
    return false;
  if (p->m == 0 || p->n == 0) return true;
  if (p->ldc < p->n) return false;
  auto pitch = [&](int64_t ld) { return ld % 16 == 0 && ld >= p->k && ld <= GGEMM_W8_MAX_LD; };
  return p->k == 0 || (pitch(p->lda) && pitch(p->ldb) && (p->groups == 1 || p->b_stride % 16 == 0));
}
bool args_ok(const ggemm_w8_gemm_t* p) {
  if (!shape_ok(p) || (!p->offsets && p->groups != 1) || !aligned(p->offsets, 4)) return false;
  if (p->m == 0 || p->n == 0) return true;
  if (!p->c || !aligned(p->c, elem_bytes(p->dtype))) return false;
  auto scales = [](const float* s) { return s && aligned(s, 4); };
  if (!scales(p->a_scales) || !scales(p->b_scales) || (p->act && !scales(p->b_up_scales))) return false;
  auto operand = [](const int8_t* x) { return x && aligned(x, 16); };
  return p->k == 0 || (operand(p->a) && operand(p->b) && (!p->act || operand(p->b_up)));
}
int64_t row_tiles(const ggemm_w8_gemm_t& p, int tm) { return p.groups > 1 ? (int64_t)p.m / tm + std::min(p.groups, p.m) : ceil_div(p.m, tm); }

}  // namespace

size_t w8_gemm_workspace(const ggemm_w8_gemm_t*) { return 0; }

int w8_gemm(const ggemm_w8_gemm_t* p, void* ws, size_t ws_bytes, hipStream_t s) {
  if (!args_ok(p)) return GGEMM_ERR_INVALID;
  if (p->m == 0 || p->n == 0) return GGEMM_OK;
  const size_t need = w8_gemm_workspace(p);
  if (ws_bytes < need) return GGEMM_ERR_WORKSPACE;
  if (need && (!ws || !aligned(ws, 16))) return GGEMM_ERR_INVALID;
  const int64_t tiles = row_tiles(*p, 64) * ceil_div(p->n, 64);
  if (tiles >= (1 << 23)) return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(p->dtype, [&](auto d) {
    using T = typename Elem<decltype(d)::value>::T;
    if (!p->act) simple_kernel<<<(unsigned)tiles, 256, 0, s>>>(Product<T, 0>{*p});
    else with_act(p->act, [&](auto act) { simple_kernel<<<(unsigned)tiles, 256, 0, s>>>(Product<T, decltype(act)::value>{*p}); });
  }); });
}

}  // namespace ggemm

extern "C" size_t ggemm_w8_gemm_workspace(const ggemm_w8_gemm_t* p) { return ggemm::w8_gemm_workspace(p); }
extern "C" int ggemm_w8_gemm(const ggemm_w8_gemm_t* p, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  return ggemm::w8_gemm(p, workspace, workspace_bytes, stream);
}
