// w8quant.hip -- rows to 8-bit integers with a scale each, and back (include/ggemm_w8.h).
#include <algorithm>

#include "ggemm_w8.h"
#include "mx4.hpp"

namespace ggemm {
namespace {

// x / s to the nearest whole number, ties to even, for |x| <= 127 s (1 + 2^-24) and a normal s; r = 1 / s to a few
// bits.  A first guess from x r is off by at most one, and only next to a half.  The rest x - q s is exact
// in 32 bits (a multiple of the smaller unit of x and s, at most s or so), so comparing it with s / 2 (exact) decides.
__device__ __forceinline__ float whole_quotient(float x, float s, float r) {
  float q = rintf(x * r);
  const float rest = fmaf(-q, s, x), half = 0.5f * s;
  const bool odd = fmaf(-2.0f, rintf(0.5f * q), q) != 0.0f;
  if (rest > half || (rest == half && odd)) q += 1.0f;
  else if (rest < -half || (rest == -half && odd)) q -= 1.0f;
  return q;
}

template <int D>
__global__ void __launch_bounds__(256) quant_kernel(ggemm_w8_quant_t p) {
  using T = typename Elem<D>::T;
  __shared__ uint32_t top[4];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    int64_t src = row;
    if (p.index) {
      src = p.index[row];
      if (src < 0 || src >= p.x_rows) src = -1;
    }
    const T* const x = static_cast<const T*>(p.x) + src * p.ld;
    uint32_t m = 0;
    for (int j = threadIdx.x; src >= 0 && j < p.cols; j += 256) m = max(m, __float_as_uint((float)x[j]) & 0x7fffffffu);
    for (int d = 1; d < 64; d *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    __syncthreads();
    if (threadIdx.x % 64 == 0) top[threadIdx.x / 64] = m;
    __syncthreads();
    m = max(max(top[0], top[1]), max(top[2], top[3]));
    const bool bad = m >= 0x7f800000u;
    const float s = fmaxf(__uint_as_float(m) / 127.0f, 0x1p-126f), r = 1.0f / s;
    for (int j = threadIdx.x; j < p.cols; j += 256)
      p.q[row * p.ldq + j] = (int8_t)(bad || src < 0 ? 0.0f : whole_quotient((float)x[j], s, r));
    if (threadIdx.x == 0) p.scales[row] = bad ? __uint_as_float(0x7fc00000u) : s;
  }
}

template <int D>
__global__ void __launch_bounds__(256) dequant_kernel(ggemm_w8_dequant_t p) {
  using T = typename Elem<D>::T;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x)
    for (int j = threadIdx.x; j < p.cols; j += 256) static_cast<T*>(p.y)[row * p.ld + j] = (T)((float)p.q[row * p.ldq + j] * p.scales[row]);
}

}  // namespace

int w8_quantize(const ggemm_w8_quant_t* p, hipStream_t s) {
  if (!p || p->rows < 0 || p->cols < 0 || p->cols >= GGEMM_W8_MAX_COLS || !elem_known(p->dtype) || (p->index && p->x_rows < 0) ||
      !aligned(p->index, 4))
    return GGEMM_ERR_INVALID;
  if (p->rows == 0) return GGEMM_OK;
  if (!p->scales || !aligned(p->scales, 4)) return GGEMM_ERR_INVALID;
  if (p->cols > 0 && ((!p->x && !(p->index && p->x_rows == 0)) || !aligned(p->x, elem_bytes(p->dtype)) || p->ld < p->cols || !p->q || p->ldq < p->cols))
    return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(p->dtype, [&](auto d) {
    quant_kernel<decltype(d)::value><<<(unsigned)std::min(p->rows, 1 << 20), 256, 0, s>>>(*p);
  }); });
}

int w8_dequantize(const ggemm_w8_dequant_t* p, hipStream_t s) {
  if (!p || p->rows < 0 || p->cols < 0 || p->cols >= GGEMM_W8_MAX_COLS || !elem_known(p->dtype)) return GGEMM_ERR_INVALID;
  if (p->rows == 0 || p->cols == 0) return GGEMM_OK;
  if (!p->q || p->ldq < p->cols || !p->scales || !aligned(p->scales, 4) || !p->y || !aligned(p->y, elem_bytes(p->dtype)) || p->ld < p->cols)
    return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(p->dtype, [&](auto d) {
    dequant_kernel<decltype(d)::value><<<(unsigned)std::min(p->rows, 1 << 20), 256, 0, s>>>(*p);
  }); });
}

}  // namespace ggemm

extern "C" int ggemm_w8_quantize(const ggemm_w8_quant_t* q, hipStream_t stream) { return ggemm::w8_quantize(q, stream); }
extern "C" int ggemm_w8_dequantize(const ggemm_w8_dequant_t* d, hipStream_t stream) { return ggemm::w8_dequantize(d, stream); }
