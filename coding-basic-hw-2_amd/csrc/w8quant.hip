// w8quant.hip -- rows to 8-bit integers with a scale each, and back (include/ggemm_w8.h).
//
// One pass: a row is held in registers while its largest magnitude is found, the next row's values on their way and the
// index entry of the row after (without: 32768 gathered rows of 4096 bf16 86 us, with 62; 70 on two other cards).
// Bound: HBM; 5.8 to 6.4 TB/s with every gathered row counted, 16384 rows read twice each.
#include <algorithm>

#include "ggemm_w8.h"
#include "mx4.hpp"

namespace ggemm {
namespace {

// Eight consecutive values of a row from column c0 on, zeros past its end.
template <int D>
__device__ __forceinline__ Run<typename Elem<D>::T, 8> load8(const void* x, int64_t row_at, int c0, int cols) {
  using T = typename Elem<D>::T;
  const T* const p = static_cast<const T*>(x) + row_at + c0;
  if (c0 + 8 <= cols) return Run<T, 8>::load(p);
  Run<T, 8> w;
#pragma unroll
  for (int e = 0; e < 8; ++e) w.x[e] = c0 + e < cols ? p[e] : (T)0.0f;
  return w;
}
// The largest magnitude as bits without the sign, NaN above Inf above all else: 16-bit values two in a word.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <int D>
__device__ __forceinline__ uint32_t largest(const Run<typename Elem<D>::T, 8>& v, uint32_t m) {
  if constexpr (D == GGEMM_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v.x[e]) & 0x7fffffffu);
  } else {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu)));
  }
  return m;
}
// The bits of the 32-bit float that `largest` of a lane stands for.
template <int D>
__device__ __forceinline__ uint32_t largest_bits(uint32_t m) {
  if constexpr (D == GGEMM_F32) return m;
  m = max(m & 0xffffu, m >> 16);
  if constexpr (D == GGEMM_BF16) return m << 16;
  return __float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)m));
}

// x / s to the nearest whole number, ties to even, in the low byte: s = max(fl(a / 127), 2^-126), |x| <= a, r from
// row_factor.  Adding 1.5 2^23 to x r in one multiply-add rounds once, to a whole number.
// r = fl(1 / s), so x r is off x / s by 2 parts in 2^24 at most and the number by one at most, next to a half.
// The rest x - q s is exact (a multiple of the smaller unit of x and s, about s at most), and comparing twice it with s
// decides, exact too (s / 2 would lose a bit where s is below 2^-125; twice the rest is below 2^123).
// bf16 needs no such step.  With x and a of 8 bits, |254 x - (2 n + 1) a| is either a unit of x or more, i.e.
// 127 x / a lies a part of 7 10^-6 or more beside the half, where the roundings of s and r come to 2.4 10^-7; or 0:
// then a is 127 or 254 times a power of two, s and r are powers of two and all is exact, or x = a / 2, n = 63, and for
// that value row_factor has moved r to the side where it belongs.
constexpr float kWhole = 12582912.0f;
template <int D>
__device__ __forceinline__ float row_factor(float a, float s) {
  float r = 1.0f / s;
  if constexpr (D == GGEMM_BF16) {
    const float h = 0.5f * a;
    // h / s of 63.5 or more: 64.  a - 127 s is a whole number of 2^-149, so its sign is right (half of it can come out as zero).
    const bool up = fmaf(-127.0f, s, a) >= 0.0f;
    // s is a power of two at its least, and r exact
    if (s > 0x1p-126f && fmaf(h, r, kWhole) - kWhole != (up ? 64.0f : 63.0f)) r = __uint_as_float(__float_as_uint(r) + (up ? 1u : ~0u));
  }
  return r;
}
template <int D>
__device__ __forceinline__ uint32_t whole_quotient(float x, float s, float r) {
  const float big = fmaf(x, r, kWhole);
  if constexpr (D == GGEMM_BF16) return __float_as_uint(big);
  const float q = big - kWhole, rest = fmaf(-q, s, x), twice = rest + rest;
  const uint32_t w = __float_as_uint(big), odd = w & 1u;
  if (twice > s || (twice == s && odd)) return w + 1u;
  if (twice < -s || (twice == -s && odd)) return w - 1u;
  return w;
}
template <int D>
__device__ __forceinline__ u32x2 quotients(const Run<typename Elem<D>::T, 8>& v, float s, float r) {
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = whole_quotient<D>((float)v.x[e], s, r);
  u32x2 o;
#pragma unroll
  for (int h = 0; h < 2; ++h)   // the low bytes of four words
    o[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[4 * h + 3], w[4 * h + 2], 0x0c0c0400u),
                                 __builtin_amdgcn_perm(w[4 * h + 1], w[4 * h], 0x0c0c0400u), 0x05040100u);
  return o;
}
template <bool kStream>
__device__ __forceinline__ void store8(int8_t* p, u32x2 w, int ok) {
  typedef u32x2 at_any __attribute__((aligned(1)));
  if (ok >= 8) {
    if constexpr (kStream) __builtin_nontemporal_store(w, reinterpret_cast<at_any*>(p));
    else *reinterpret_cast<at_any*>(p) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < ok) p[e] = (int8_t)(w[e / 4] >> (8 * (e % 4)));
  }
}

// L lanes share a row (up to 64: part of a wave, else a whole workgroup), N chunks of 8 values a lane in registers; the chunks of
// a longer row past those are read a second time, out of the caches.
template <int D, int L, int N, bool kStream>
__global__ void __launch_bounds__(256) quant_kernel(ggemm_w8_quant_t p) {
  using V = Run<typename Elem<D>::T, 8>;
  constexpr int R = 256 / L;   // rows at a time
  __shared__ uint32_t top[4];
  const int lane = threadIdx.x % L, chunks = ceil_div(p.cols, 8);
  const int64_t step = (int64_t)gridDim.x * R;
  int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / L;
  auto source = [&](int64_t r) -> int64_t {   // the row of x, -1: none
    if (r >= p.rows) return -1;
    if (!p.index) return r;
    const int i = p.index[r];
    return (uint32_t)i < (uint32_t)p.x_rows ? i : -1;
  };
  auto load = [&](int64_t src, V (&v)[N]) {
#pragma unroll
    for (int c = 0; c < N; ++c) v[c] = src >= 0 && lane + c * L < chunks ? load8<D>(p.x, src * p.ld, 8 * (lane + c * L), p.cols) : V{};
  };
  // a row ahead of the one in hand, and the index entry of the row after
  int64_t src = source(row), coming = source(row + step);
  V next[N];
  load(src, next);
  for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < p.rows; row0 += step, row += step) {
    const int have = src >= 0 ? chunks : 0;
    const int64_t at = src * p.ld;
    V v[N];
#pragma unroll
    for (int c = 0; c < N; ++c) v[c] = next[c];
    src = coming;
    if (row0 + step < p.rows) {
      load(src, next);
      coming = source(row + 2 * step);
    }
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < N; ++c) m = largest<D>(v[c], m);
    for (int c = lane + N * L; c < have; c += L) m = largest<D>(load8<D>(p.x, at, 8 * c, p.cols), m);
    m = largest_bits<D>(m);
#pragma unroll
    for (int d = 1; d < (L < 64 ? L : 64); d *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    if constexpr (L > 64) {
      __syncthreads();
      if (threadIdx.x % 64 == 0) top[threadIdx.x / 64] = m;
      __syncthreads();
      m = max(max(top[0], top[1]), max(top[2], top[3]));
    }
    const bool bad = m >= 0x7f800000u;
    const float a = __uint_as_float(m), s = fmaxf(a / 127.0f, 0x1p-126f), r = bad ? 0.0f : row_factor<D>(a, s);
    if (row >= p.rows) continue;
    int8_t* const out = p.q + row * p.ldq;
    auto put = [&](int c, const V& x) {
      u32x2 w = quotients<D>(x, s, r);
      if (bad) w = u32x2{0, 0};
      store8<kStream>(out + 8 * c, w, p.cols - 8 * c);
    };
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (lane + c * L < chunks) put(lane + c * L, v[c]);
    for (int c = lane + N * L; c < chunks; c += L) put(c, c < have ? load8<D>(p.x, at, 8 * c, p.cols) : V{});
    if (lane == 0) p.scales[row] = bad ? __uint_as_float(0x7fc00000u) : s;
  }
}

// Back to values: 256 lanes cover cx chunks of 8 columns (a power of two) of 256 / cx rows, a workgroup for every row of a large
// matrix: 32768 x 4096 to bf16 66 us, 6.1 TB/s; 1024 to 16384 workgroups that walk over rows 74 to 88, with non-temporal
// stores 68.
template <int D>
__device__ __forceinline__ typename Elem<D>::T dequant_one(int b, float s) {
  float v = (float)b * s;
  asm("" : "+v"(v));   // a 32-bit product, then the type's rounding: not one instruction that rounds once
  return (typename Elem<D>::T)v;
}
template <int D>
__device__ __forceinline__ void dequant_store(const ggemm_w8_dequant_t& p, int64_t row, int c0, u32x2 w, float s) {
  using T = typename Elem<D>::T;
  Run<T, 8> o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o.x[e] = dequant_one<D>((int8_t)(w[e / 4] >> (8 * (e % 4))), s);
  o.template store<false>(static_cast<T*>(p.y) + row * p.ld + c0);
}
template <int D>
__global__ void __launch_bounds__(256) dequant_kernel(ggemm_w8_dequant_t p, int log_cx) {
  const int c0 = 8 * ((blockIdx.y << log_cx) + (threadIdx.x & ((1 << log_cx) - 1)));
  if (c0 >= p.cols) return;
  const int64_t step = (int64_t)gridDim.x << (8 - log_cx);
  int64_t row = ((int64_t)blockIdx.x << (8 - log_cx)) + (threadIdx.x >> log_cx);
  if (c0 + 8 > p.cols) {
    for (; row < p.rows; row += step)
      for (int c = c0; c < p.cols; ++c)
        static_cast<typename Elem<D>::T*>(p.y)[row * p.ld + c] = dequant_one<D>(p.q[row * p.ldq + c], p.scales[row]);
    return;
  }
  typedef u32x2 at_any __attribute__((aligned(1)));
  auto load = [&](int64_t r) { return (u32x2)*reinterpret_cast<const at_any*>(p.q + r * p.ldq + c0); };
  for (; row < p.rows; row += step) dequant_store<D>(p, row, c0, load(row), p.scales[row]);
}

// kStream: non-temporal stores, for more integers than the next reader finds in the caches anyway (32768 x 4096: 72 and 62 us).
template <int D, int L, int N>
void run_quant(const ggemm_w8_quant_t& p, hipStream_t s) {
  const int64_t all = ((int64_t)p.rows + 256 / L - 1) / (256 / L);
  const unsigned grid = (unsigned)std::min((int64_t)(L > 64 ? 4096 : 2048), all);
  if ((int64_t)p.rows * p.cols >= (64 << 20)) quant_kernel<D, L, N, true><<<grid, 256, 0, s>>>(p);
  else quant_kernel<D, L, N, false><<<grid, 256, 0, s>>>(p);
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
    constexpr int D = decltype(d)::value;
    // 16-bit rows of up to 4096: a wave for each (32768 rows 62 us, a workgroup for each 64); one row: 5.3 and 2.9
    if (p->cols <= 256) run_quant<D, 8, 4>(*p, s);
    else if (p->cols <= 1024) run_quant<D, 64, 2>(*p, s);
    else if (p->cols <= 2048) run_quant<D, 64, 4>(*p, s);
    else if (p->cols <= 4096 && D != GGEMM_F32 && p->rows >= 2048) run_quant<D, 64, 8>(*p, s);
    else if (p->cols <= 4096) run_quant<D, 256, 2>(*p, s);
    else run_quant<D, 256, 4>(*p, s);
  }); });
}

int w8_dequantize(const ggemm_w8_dequant_t* p, hipStream_t s) {
  if (!p || p->rows < 0 || p->cols < 0 || p->cols >= GGEMM_W8_MAX_COLS || !elem_known(p->dtype)) return GGEMM_ERR_INVALID;
  if (p->rows == 0 || p->cols == 0) return GGEMM_OK;
  if (!p->q || p->ldq < p->cols || !p->scales || !aligned(p->scales, 4) || !p->y || !aligned(p->y, elem_bytes(p->dtype)) || p->ld < p->cols)
    return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(p->dtype, [&](auto d) {
    const int chunks = ceil_div(p->cols, 8);
    int log_cx = 0;
    while (log_cx < 8 && (1 << log_cx) < chunks) ++log_cx;
    const int64_t rows = ((int64_t)p->rows + (256 >> log_cx) - 1) >> (8 - log_cx);
    dequant_kernel<decltype(d)::value><<<dim3((unsigned)std::min((int64_t)1 << 16, rows), ceil_div(chunks, 1 << log_cx)), 256, 0, s>>>(*p, log_cx);
  }); });
}

}  // namespace ggemm

extern "C" int ggemm_w8_quantize(const ggemm_w8_quant_t* q, hipStream_t stream) { return ggemm::w8_quantize(q, stream); }
extern "C" int ggemm_w8_dequantize(const ggemm_w8_dequant_t* d, hipStream_t stream) { return ggemm::w8_dequantize(d, stream); }
