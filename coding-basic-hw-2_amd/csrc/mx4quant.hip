// mx4quant.hip -- quantisation to microscaled 4-bit floating point and back (include/ggemm_mx4.h).
//
// Per block of 32 values: s = max(exponent(max |v|) - 2, 0) as a biased byte, codes = v / 2^(s - 127) on the
// grid 0, 0.5, 1, 1.5, 2, 3, 4, 6.  The quotient by a power of two is exact, so the conversion
// instruction (v_cvt_scalef32_pk_fp4_*: two values a time, nearest, ties to even, saturating) rounds
// once; the largest magnitude lands in [4, 8).
// Along the rows a lane holds 8 consecutive values and the four lanes of a block exchange their
// maxima; down the columns a lane holds a block of its own column.
// Bound: HBM.
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"

namespace ggemm {
namespace {

constexpr int kThreads = 256;

// Eight consecutive values of a row.
template <int D>
struct Oct {
  typename Elem<D>::T v[8];
};

template <int D>
__device__ __forceinline__ uint32_t mag_bits(typename Elem<D>::T v) {   // |v| as the bits of a 32-bit float
  return __float_as_uint((float)v) & 0x7fffffffu;
}

// codes of 8 values, the first in the low four bits
template <int D>
__device__ __forceinline__ uint32_t codes8(const typename Elem<D>::T (&v)[8], float scale) {
  uint32_t r = 0;
  if constexpr (D == GGEMM_F32) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
  } else if constexpr (D == GGEMM_BF16) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2{v[0], v[1]}, scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2{v[2], v[3]}, scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2{v[4], v[5]}, scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2{v[6], v[7]}, scale, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2{v[0], v[1]}, scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2{v[2], v[3]}, scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2{v[4], v[5]}, scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2{v[6], v[7]}, scale, 3);
  }
  return r;
}

__device__ __forceinline__ int64_t source_row(const ggemm_mx4_quant_t& q, int row) {
  if (!q.index) return row;
  const int r = q.index[row];
  return r >= 0 && r < q.x_rows ? r : -1;
}

// Chunk `chunk` of a row; the four lanes of a block call it together.
template <int D, bool kVec>
__device__ __forceinline__ void quant_chunk(const ggemm_mx4_quant_t& q, int64_t row, int chunk) {
  using T = typename Elem<D>::T;
  const int64_t src = source_row(q, (int)row);
  const int c0 = 8 * chunk;
  Oct<D> o;
  const T* p = static_cast<const T*>(q.x) + src * q.ld + c0;
  if (kVec && src >= 0 && c0 + 8 <= q.cols) {
    o = *reinterpret_cast<const Oct<D>*>(__builtin_assume_aligned(p, 16));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = src >= 0 && c0 + i < q.cols ? p[i] : (T)0.0f;
  }
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, mag_bits<D>(o.v[i]));
  amax = max(amax, dpp<kDppXor1>(amax));
  amax = max(amax, dpp<kDppXor2>(amax));
  const uint32_t s = mx4_scale_byte(amax);
  const uint32_t w = s == 255u ? 0u : codes8<D>(o.v, mx4_scale(s));
  *reinterpret_cast<uint32_t*>(q.codes + row * q.ld_codes + 4 * chunk) = w;
  if ((chunk & 3) == 0) q.scales[row * q.ld_scales + (chunk >> 2)] = (uint8_t)s;
}

// Blocks along the rows.  A workgroup of 256 lanes covers cx chunks of 8 columns (cx a power of two)
// of 256 / cx rows.
template <int D, bool kVec>
__global__ void __launch_bounds__(kThreads) quant_rows_kernel(ggemm_mx4_quant_t q, int log_cx) {
  const int chunks = 4 * ceil_div(q.cols, 32);
  const int chunk = (blockIdx.y << log_cx) + (threadIdx.x & ((1 << log_cx) - 1));
  if (chunk >= chunks) return;   // whole blocks: four lanes together
  for (int64_t row = ((int64_t)blockIdx.x << (8 - log_cx)) + (threadIdx.x >> log_cx); row < q.rows;
       row += (int64_t)gridDim.x << (8 - log_cx))
    quant_chunk<D, kVec>(q, row, chunk);
}

// Block b (32 rows) of column col.
template <int D>
__device__ __forceinline__ void quant_column_block(const ggemm_mx4_quant_t& q, int64_t col, int64_t b) {
  using T = typename Elem<D>::T;
  const int64_t r0 = 32 * b;
  T v[32];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[i] = (T)0.0f;
    if (r0 + i < q.rows) {
      const int64_t src = source_row(q, (int)(r0 + i));
      if (src >= 0) v[i] = static_cast<const T*>(q.x)[src * q.ld + col];
    }
    amax = max(amax, mag_bits<D>(v[i]));
  }
  const uint32_t s = mx4_scale_byte(amax);
  u32x4 w = {0u, 0u, 0u, 0u};
  if (s != 255u) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = v[8 * i + j];
      w[i] = codes8<D>(u, mx4_scale(s));
    }
  }
  *reinterpret_cast<u32x4*>(q.codes_t + col * q.ld_codes_t + 16 * b) = w;
  q.scales_t[col * q.ld_scales_t + b] = (uint8_t)s;
}

// Blocks down the columns: a lane quantises 32 rows of one column.
template <int D>
__global__ void __launch_bounds__(kThreads) quant_cols_kernel(ggemm_mx4_quant_t q) {
  const int64_t col = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  if (col >= q.cols) return;
  for (int64_t b = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6); 32 * b < q.rows; b += 4 * (int64_t)gridDim.y)
    quant_column_block<D>(q, col, b);
}

// A lane turns 8 codes into values.
template <int D, bool kVec>
__device__ __forceinline__ void dequant_chunk(const ggemm_mx4_dequant_t& d, int64_t row, int chunk) {
  using T = typename Elem<D>::T;
  const uint32_t w = *reinterpret_cast<const uint32_t*>(d.codes + row * d.ld_codes + 4 * chunk);
  const uint32_t s = d.scales[row * d.ld_scales + (chunk >> 2)];
  Oct<D> o;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = w >> (4 * i), e = (c >> 1) & 3u, m = c & 1u;
    // magnitude: e = 0: m / 2, else (1 + m / 2) 2^(e - 1); exact in 32 bits times any scale
    const float mag = e ? __uint_as_float(((126u + e) << 23) | (m << 22)) : 0.5f * (float)m;
    float v = mag * mx4_scale(s);
    v = c & 8u ? -v : v;
    o.v[i] = (T)(s == 255u ? __uint_as_float(0x7fc00000u) : v);
  }
  const int c0 = 8 * chunk;
  T* p = static_cast<T*>(d.y) + row * d.ld + c0;
  if (kVec && c0 + 8 <= d.cols) {
    *reinterpret_cast<Oct<D>*>(__builtin_assume_aligned(p, 16)) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < d.cols) p[i] = o.v[i];
  }
}

template <int D, bool kVec>
__global__ void __launch_bounds__(kThreads) dequant_kernel(ggemm_mx4_dequant_t d, int log_cx) {
  const int chunks = ceil_div(d.cols, 8);
  const int chunk = (blockIdx.y << log_cx) + (threadIdx.x & ((1 << log_cx) - 1));
  if (chunk >= chunks) return;
  for (int64_t row = ((int64_t)blockIdx.x << (8 - log_cx)) + (threadIdx.x >> log_cx); row < d.rows;
       row += (int64_t)gridDim.x << (8 - log_cx))
    dequant_chunk<D, kVec>(d, row, chunk);
}

// Lanes of a workgroup along a row of `chunks` chunks: the power of two at or above, at most 256.
int log_lanes(int chunks) {
  int l = 2;
  while (l < 8 && (1 << l) < chunks) ++l;
  return l;
}

// Grid of a row kernel: x strides over the rows (at most 2^20 workgroups), y stays within its 65535 for
// every valid size.
dim3 row_grid(int rows, int chunks, int log_cx) {
  const int per = 256 >> log_cx;
  return dim3((unsigned)std::min(ceil_div(rows, per), 1 << 20), (unsigned)ceil_div(chunks, 1 << log_cx));
}

constexpr int kMaxCols = 1 << 26;   // 8 columns a lane, 256 lanes a workgroup: at most 32768 workgroups along a row

bool codes_ok(const uint8_t* codes, int64_t ld_codes, const uint8_t* scales, int64_t ld_scales, int cols) {
  const int64_t nb = ceil_div(cols, 32);
  return codes && scales && aligned(codes, 16) && aligned(scales, 4) && ld_codes % 16 == 0 && ld_codes >= 16 * nb &&
         ld_scales % 4 == 0 && ld_scales >= nb;
}

}  // namespace

int mx4_quantize(const ggemm_mx4_quant_t* q, hipStream_t s) {
  if (!q || q->rows < 0 || q->cols < 0 || !elem_known(q->dtype)) return GGEMM_ERR_INVALID;
  const bool along = q->codes || q->scales, down = q->codes_t || q->scales_t;
  if (!along && !down) return GGEMM_ERR_INVALID;
  if (q->cols > kMaxCols || (down && q->rows > kMaxCols)) return GGEMM_ERR_INVALID;
  if (q->rows == 0 || q->cols == 0) return GGEMM_OK;
  if (!q->x || q->ld < q->cols || !aligned(q->x, elem_bytes(q->dtype)) || (q->index && (q->x_rows < 0 || !aligned(q->index, 4))))
    return GGEMM_ERR_INVALID;
  if (along && !codes_ok(q->codes, q->ld_codes, q->scales, q->ld_scales, q->cols)) return GGEMM_ERR_INVALID;
  if (down && !codes_ok(q->codes_t, q->ld_codes_t, q->scales_t, q->ld_scales_t, q->rows)) return GGEMM_ERR_INVALID;
  with_elem(q->dtype, [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (along) {
      const int chunks = 4 * ceil_div(q->cols, 32), l = log_lanes(chunks);
      const dim3 grid = row_grid(q->rows, chunks, l);
      if (aligned(q->x, 16) && q->ld * elem_bytes(D) % 16 == 0)
        quant_rows_kernel<D, true><<<grid, kThreads, 0, s>>>(*q, l);
      else
        quant_rows_kernel<D, false><<<grid, kThreads, 0, s>>>(*q, l);
    }
    if (down) {
      const dim3 grid((unsigned)ceil_div(q->cols, 64), (unsigned)std::min(ceil_div(q->rows, 128), 32768));
      quant_cols_kernel<D><<<grid, kThreads, 0, s>>>(*q);
    }
  });
  return hipGetLastError() == hipSuccess ? GGEMM_OK : GGEMM_ERR_CUDA;
}

int mx4_dequantize(const ggemm_mx4_dequant_t* d, hipStream_t s) {
  if (!d || d->rows < 0 || d->cols < 0 || d->cols > kMaxCols || !elem_known(d->dtype)) return GGEMM_ERR_INVALID;
  if (d->rows == 0 || d->cols == 0) return GGEMM_OK;
  if (!codes_ok(d->codes, d->ld_codes, d->scales, d->ld_scales, d->cols) || !d->y || d->ld < d->cols ||
      !aligned(d->y, elem_bytes(d->dtype)))
    return GGEMM_ERR_INVALID;
  with_elem(d->dtype, [&](auto t) {
    constexpr int D = decltype(t)::value;
    const int chunks = ceil_div(d->cols, 8), l = log_lanes(chunks);
    const dim3 grid = row_grid(d->rows, chunks, l);
    if (aligned(d->y, 16) && d->ld * elem_bytes(D) % 16 == 0)
      dequant_kernel<D, true><<<grid, kThreads, 0, s>>>(*d, l);
    else
      dequant_kernel<D, false><<<grid, kThreads, 0, s>>>(*d, l);
  });
  return hipGetLastError() == hipSuccess ? GGEMM_OK : GGEMM_ERR_CUDA;
}

}  // namespace ggemm

extern "C" int ggemm_mx4_quantize(const ggemm_mx4_quant_t* q, hipStream_t stream) {
  return ggemm::mx4_quantize(q, stream);
}
extern "C" int ggemm_mx4_dequantize(const ggemm_mx4_dequant_t* d, hipStream_t stream) {
  return ggemm::mx4_dequantize(d, stream);
}
