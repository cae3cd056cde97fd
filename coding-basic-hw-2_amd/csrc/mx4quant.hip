// mx4quant.hip -- quantisation to microscaled 4-bit floating point and back (include/ggemm_mx4.h).
//
// Per block of 32 values: s = max(exponent(max |v|) - 2, 0) as a biased byte, codes = v / 2^(s - 127) on the
// grid 0, 0.5, 1, 1.5, 2, 3, 4, 6.  The quotient by a power of two is exact, so the conversion
// instruction (v_cvt_scalef32_pk_fp4_*: two values a time, nearest, ties to even, saturating) rounds
// once; the largest magnitude lands in [4, 8).  Magnitudes are compared as integers with the sign bit
// cleared (two 16-bit ones in a word), which orders them with NaN above Inf above all else.
// Along the rows a lane holds 8 consecutive values and the four lanes of a block exchange their
// maxima.  Down the columns a workgroup turns a tile through LDS: it is read once, quantised along
// the rows on the way if that is asked too, and a lane then walks down a block of its columns.
// Bound: HBM.
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"

namespace ggemm {
namespace {

constexpr int kThreads = 256;

// kStream: non-temporal stores, which leave what is still to be read in the caches.  32768 x 4096 bf16: along the rows 64
// -> 51 us, down the columns 72 -> 62, both 88 -> 76, back to values 72 -> 51 (f32 138 -> 99).  Where rows end inside a
// line the parts of a line come one by one and each has to be read first (30001 x 1000 f32, both: 28 us by way of the
// caches, 34; 32768 x 1001 back to bf16: 15, 18), so the rows have to be whole lines of 128 bytes (codes turned through
// LDS) or 64 (values); along the rows a wave's 256 bytes are mostly whole whatever the rows' length.
template <bool kStream, class V>
__device__ __forceinline__ void put(V v, void* p) {
  if constexpr (kStream) __builtin_nontemporal_store(v, static_cast<V*>(p));
  else *static_cast<V*>(p) = v;
}

// Eight consecutive values: two vectors of four, or one.
template <int D>
struct Oct {
  typename Elem<D>::T v[8];
};
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// The larger magnitudes of two words of two 16-bit values, sign bits cleared.
__device__ __forceinline__ uint32_t max_mag2(uint32_t m, uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
// A 16-bit magnitude (low half) as the bits of a 32-bit float.
template <int D>
__device__ __forceinline__ uint32_t wide_mag(uint32_t m) {
  if constexpr (D == GGEMM_BF16) return m << 16;
  else return __float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)m));
}
// The largest of 8 magnitudes (16-bit: both halves of a word; 32-bit: bits).
template <int D>
__device__ __forceinline__ uint32_t oct_mag(const Oct<D>& o) {
  uint32_t m = 0;
  if constexpr (D == GGEMM_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(o.v[i]) & 0x7fffffffu);
  } else {
    const u32x4 w = __builtin_bit_cast(u32x4, o);
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max_mag2(m, w[i]);
    m = max(m & 0xffffu, m >> 16);
  }
  return m;
}
// Scale byte of a block from the largest magnitude that oct_mag gave.
template <int D>
__device__ __forceinline__ uint32_t block_scale(uint32_t m) {
  if constexpr (D == GGEMM_F32) return mx4_scale_byte(m);
  else return mx4_scale_byte(wide_mag<D>(m));
}

// A byte of codes of two values (word: two 16-bit values) into byte I of r.
template <int D, int I>
__device__ __forceinline__ uint32_t code2(uint32_t r, uint32_t w, float scale) {
  if constexpr (D == GGEMM_BF16) return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w), scale, I);
  else return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, w), scale, I);
}
// codes of 8 values, the first in the low four bits
template <int D>
__device__ __forceinline__ uint32_t codes8(const Oct<D>& o, float scale) {
  uint32_t r = 0;
  if constexpr (D == GGEMM_F32) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, o.v[0], o.v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, o.v[2], o.v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, o.v[4], o.v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, o.v[6], o.v[7], scale, 3);
  } else {
    const u32x4 w = __builtin_bit_cast(u32x4, o);
    r = code2<D, 0>(r, w[0], scale);
    r = code2<D, 1>(r, w[1], scale);
    r = code2<D, 2>(r, w[2], scale);
    r = code2<D, 3>(r, w[3], scale);
  }
  return r;
}

__device__ __forceinline__ int64_t source_row(const ggemm_mx4_quant_t& q, int row) {
  if (!q.index) return row;
  const int r = q.index[row];
  return r >= 0 && r < q.x_rows ? r : -1;
}

// Columns 8 chunk .. of a row (zeros past its end and for a row that does not exist).
template <int D>
__device__ __forceinline__ Oct<D> load_chunk(const ggemm_mx4_quant_t& q, int64_t src, int chunk) {
  using T = typename Elem<D>::T;
  constexpr int N = 16 / (int)sizeof(T);
  const int c0 = 8 * chunk;
  const T* p = static_cast<const T*>(q.x) + src * q.ld + c0;
  Oct<D> o;
  if (src >= 0 && c0 + 8 <= q.cols) {
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      const Run<T, N> w = Run<T, N>::load(p + i);
#pragma unroll
      for (int j = 0; j < N; ++j) o.v[i + j] = w.x[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = src >= 0 && c0 + i < q.cols ? p[i] : (T)0.0f;
  }
  return o;
}
// Its codes, and the block's scale byte; the four lanes of a block call it together.
template <int D>
__device__ __forceinline__ uint32_t code_chunk(const Oct<D>& o, uint32_t& s) {
  uint32_t m = oct_mag<D>(o);
  m = max(m, dpp<kDppXor1>(m));
  m = max(m, dpp<kDppXor2>(m));
  s = block_scale<D>(m);
  return s == 255u ? 0u : codes8<D>(o, mx4_scale(s));
}
template <int D>
__device__ __forceinline__ void store_chunk(const ggemm_mx4_quant_t& q, int64_t row, int chunk, const Oct<D>& o) {
  uint32_t s;
  const uint32_t w = code_chunk<D>(o, s);
  put<true>(w, q.codes + row * q.ld_codes + 4 * chunk);
  if ((chunk & 3) == 0) put<true>((uint8_t)s, q.scales + row * q.ld_scales + (chunk >> 2));
}

// Blocks along the rows.  A workgroup of 256 lanes covers cx chunks of 8 columns (cx a power of two)
// of 256 / cx rows.
template <int D>
__global__ void __launch_bounds__(kThreads) quant_rows_kernel(ggemm_mx4_quant_t q, int log_cx) {
  const int chunks = 4 * ceil_div(q.cols, 32);
  const int chunk = (blockIdx.y << log_cx) + (threadIdx.x & ((1 << log_cx) - 1));
  if (chunk >= chunks) return;   // whole blocks: four lanes together
  const int64_t step = (int64_t)gridDim.x << (8 - log_cx);
  int64_t row = ((int64_t)blockIdx.x << (8 - log_cx)) + (threadIdx.x >> log_cx);
  for (; row + step < q.rows; row += 2 * step) {   // two rows' loads before their stores
    const int64_t s0 = source_row(q, (int)row), s1 = source_row(q, (int)(row + step));
    const Oct<D> a = load_chunk<D>(q, s0, chunk), b = load_chunk<D>(q, s1, chunk);
    store_chunk<D>(q, row, chunk, a);
    store_chunk<D>(q, row + step, chunk, b);
  }
  if (row < q.rows) store_chunk<D>(q, row, chunk, load_chunk<D>(q, source_row(q, (int)row), chunk));
}

// Blocks down the columns, and along the rows too with kAlong: a workgroup takes a tile of kRows rows (a
// memory line of codes of every column; half of one for 32-bit values) and 128 columns through 64 KB of LDS.
// Codes and scales of both kinds go back through LDS and leave as 16 and 4 bytes a lane, runs of 128 (64)
// bytes.  A tile has 4 scale bytes of a row; runs of tiles side by side go to one XCD and these bytes are stored
// the ordinary way, so that its L2 makes lines of them (32768 x 4096 bf16, both kinds: 127 us as they come, 104
// this way; 76 with the present loads, the two kinds one after the other 114).  Half the tile and twice the workgroups per compute unit is slower
// by 5 to 20 %.
template <int D>
struct Turn {
  static constexpr int kRows = D == GGEMM_F32 ? 128 : 256, kCols = 128, kThreads = 512;
  static constexpr int kLanes = kCols / 8;   // lanes of a row
  static constexpr int kBlocks = kRows / 32, kRowBytes = kCols * (int)sizeof(typename Elem<D>::T);
};
template <int D, bool kAlong, bool kStream>
__global__ void __launch_bounds__(Turn<D>::kThreads, 4) quant_turn_kernel(ggemm_mx4_quant_t q) {
  using T = typename Elem<D>::T;
  using U = Turn<D>;
  constexpr int B = U::kBlocks;
  constexpr int kAlongCodes = U::kCols * B * 16;            // the rows' codes in the tile's LDS, after the columns'
  constexpr int kPer = D == GGEMM_F32 ? 1 : 2;              // columns of a lane
  constexpr int kStep = U::kThreads / U::kLanes, kN = U::kRows / kStep;   // rows at a time, rows of a lane
  __shared__ __attribute__((aligned(16))) uint8_t tile[U::kRows * U::kRowBytes];
  __shared__ __attribute__((aligned(4))) uint8_t down_scale[U::kCols][B], along_scale[U::kRows][4];
  const int tid = threadIdx.x, lane_row = tid / U::kLanes, lane_chunk = tid % U::kLanes;
  const int tiles_c = ceil_div(q.cols, U::kCols);
  const int64_t tiles = (int64_t)ceil_div(q.rows, U::kRows) * tiles_c;
  for (int64_t it = blockIdx.x; it < tiles; it += gridDim.x) {
    const int64_t t = kAlong ? tile_number((int)it, (int)tiles) : it;
    const int64_t r0 = t / tiles_c * U::kRows;
    const int c0 = (int)(t % tiles_c) * U::kCols;
    const int rows_left = (int)min((int64_t)U::kRows, q.rows - r0), cols_left = min(U::kCols, q.cols - c0);
    uint32_t wa[kAlong ? kN : 1], sa[kAlong ? kN : 1];
    {
      Oct<D> o[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r = i * kStep + lane_row;
        o[i] = load_chunk<D>(q, r < rows_left ? source_row(q, (int)(r0 + r)) : -1, c0 / 8 + lane_chunk);
      }
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        *reinterpret_cast<Oct<D>*>(tile + (i * kStep + lane_row) * U::kRowBytes + lane_chunk * (int)sizeof o[i]) = o[i];
        if constexpr (kAlong) wa[i] = code_chunk<D>(o[i], sa[i]);
      }
    }
    __syncthreads();
    u32x4 w[kPer];
    uint32_t sc[kPer];
    const int col = kPer * (tid % (U::kCols / kPer)), blk = tid / (U::kCols / kPer);
    if constexpr (D == GGEMM_F32) {
      const T* p = reinterpret_cast<const T*>(tile) + 32 * blk * U::kCols + col;
      Oct<D> y[4];
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[i].v[j] = p[(8 * i + j) * U::kCols];
        m = max(m, oct_mag<D>(y[i]));
      }
      sc[0] = block_scale<D>(m);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[0][i] = sc[0] == 255u ? 0u : codes8<D>(y[i], mx4_scale(sc[0]));
    } else {                          // two columns side by side in a word
      const uint32_t* p = reinterpret_cast<const uint32_t*>(tile) + 32 * blk * (U::kCols / 2) + col / 2;
      uint32_t x[32], m = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        x[i] = p[i * (U::kCols / 2)];
        m = max_mag2(m, x[i]);
      }
      sc[0] = block_scale<D>(m & 0xffffu);
      sc[1] = block_scale<D>(m >> 16);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float scale = mx4_scale(sc[c]);
        const uint32_t pick = c ? 0x07060302u : 0x05040100u;   // the column's halves of two rows
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t r = 0;
          r = code2<D, 0>(r, __builtin_amdgcn_perm(x[8 * i + 1], x[8 * i], pick), scale);
          r = code2<D, 1>(r, __builtin_amdgcn_perm(x[8 * i + 3], x[8 * i + 2], pick), scale);
          r = code2<D, 2>(r, __builtin_amdgcn_perm(x[8 * i + 5], x[8 * i + 4], pick), scale);
          r = code2<D, 3>(r, __builtin_amdgcn_perm(x[8 * i + 7], x[8 * i + 6], pick), scale);
          w[c][i] = sc[c] == 255u ? 0u : r;
        }
      }
    }
    __syncthreads();
    // the columns' codes: [column][block] of 16 bytes, the block's place exchanged by the column against bank conflicts
    auto place = [&](int c, int b) { return tile + (c * B + (b ^ (c / kPer & (B - 1)))) * 16; };
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      *reinterpret_cast<u32x4*>(place(col + c, blk)) = w[c];
      down_scale[col + c][blk] = (uint8_t)sc[c];
    }
    if constexpr (kAlong) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r = i * kStep + lane_row;
        *reinterpret_cast<uint32_t*>(tile + kAlongCodes + r * 64 + 4 * lane_chunk) = wa[i];
        if ((lane_chunk & 3) == 0) along_scale[r][lane_chunk / 4] = (uint8_t)sa[i];
      }
    }
    __syncthreads();
    // up to four scale bytes of a row or column; a word's bytes past the last block are not written
    auto put_scales = [&](const uint8_t* from, uint8_t* to, int left, auto stream) {
      if (left < 4) {
        for (int i = 0; i < left; ++i) to[i] = from[i];
      } else {
        put<decltype(stream)::value>(*reinterpret_cast<const uint32_t*>(from), to);
      }
    };
    const int blocks_down = ceil_div(rows_left, 32), blocks_along = ceil_div(cols_left, 32);
    for (int i = tid; i < U::kCols * B; i += U::kThreads) {
      const int c = i / B, b = i % B;
      if (c < cols_left && b < blocks_down) put<kStream>(*reinterpret_cast<const u32x4*>(place(c, b)), q.codes_t + (int64_t)(c0 + c) * q.ld_codes_t + r0 / 2 + 16 * b);
    }
    for (int i = tid; i < U::kCols * B / 4; i += U::kThreads) {
      const int c = i / (B / 4), b = i % (B / 4) * 4;
      if (c < cols_left) put_scales(&down_scale[c][b], q.scales_t + (int64_t)(c0 + c) * q.ld_scales_t + r0 / 32 + b, blocks_down - b, std::bool_constant<kStream>{});
    }
    if constexpr (kAlong) {
      for (int i = tid; i < U::kRows * 4; i += U::kThreads) {
        const int r = i / 4, b = i % 4;
        if (r < rows_left && b < blocks_along)
          put<kStream>(*reinterpret_cast<const u32x4*>(tile + kAlongCodes + 16 * i), q.codes + (r0 + r) * q.ld_codes + c0 / 2 + 16 * b);
      }
      for (int r = tid; r < rows_left; r += U::kThreads) put_scales(along_scale[r], q.scales + (r0 + r) * q.ld_scales + c0 / 32, blocks_along, std::false_type{});
    }
    __syncthreads();
  }
}

// 16 bytes of values: 8 (f32: 4) codes w with scale byte s, two a time by the conversion instructions (exact but
// for f16, which rounds).
template <int D>
struct Sixteen {
  static constexpr int N = 16 / (int)sizeof(typename Elem<D>::T);
  using Codes = std::conditional_t<D == GGEMM_F32, uint16_t, uint32_t>;
  typename Elem<D>::T v[N];
};
template <int D>
__device__ __forceinline__ Sixteen<D> values_of(uint32_t w, uint32_t s) {
  const float scale = mx4_scale(s);
  Sixteen<D> o;
  if constexpr (D == GGEMM_F32) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
    o = __builtin_bit_cast(Sixteen<D>, f32x4{a[0], a[1], b[0], b[1]});
  } else {
    auto word = [&](auto x) { return __builtin_bit_cast(uint32_t, x); };
    u32x4 x;
    if constexpr (D == GGEMM_BF16)
      x = u32x4{word(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)), word(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                word(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)), word(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
    else
      x = u32x4{word(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)), word(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
                word(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)), word(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3))};
    o = __builtin_bit_cast(Sixteen<D>, x);
  }
  if (s == 255u) {
#pragma unroll
    for (int i = 0; i < Sixteen<D>::N; ++i) o.v[i] = (typename Elem<D>::T)__uint_as_float(0x7fc00000u);
  }
  return o;
}

// A lane turns the codes of chunk `chunk` (16 bytes of values) of a row into values.
template <int D>
__device__ __forceinline__ void load_codes(const ggemm_mx4_dequant_t& d, int64_t row, int chunk, uint32_t& w, uint32_t& s) {
  constexpr int N = Sixteen<D>::N;
  w = *reinterpret_cast<const typename Sixteen<D>::Codes*>(d.codes + row * d.ld_codes + chunk * (N / 2));
  s = d.scales[row * d.ld_scales + chunk / (32 / N)];
}
template <int D, bool kStream>
__device__ __forceinline__ void store_values(const ggemm_mx4_dequant_t& d, int64_t row, int chunk, uint32_t w, uint32_t s) {
  constexpr int N = Sixteen<D>::N;
  const Sixteen<D> o = values_of<D>(w, s);
  const int c0 = N * chunk;
  auto* p = static_cast<typename Elem<D>::T*>(d.y) + row * d.ld + c0;
  if (c0 + N <= d.cols) {
    __builtin_bit_cast(Run<typename Elem<D>::T, N>, o).template store<kStream>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c0 + i < d.cols) p[i] = o.v[i];
  }
}
template <int D, bool kStream>
__global__ void __launch_bounds__(kThreads) dequant_kernel(ggemm_mx4_dequant_t d, int log_cx) {
  const int chunks = ceil_div(d.cols, Sixteen<D>::N);
  const int chunk = (blockIdx.y << log_cx) + (threadIdx.x & ((1 << log_cx) - 1));
  if (chunk >= chunks) return;
  const int64_t step = (int64_t)gridDim.x << (8 - log_cx);
  int64_t row = ((int64_t)blockIdx.x << (8 - log_cx)) + (threadIdx.x >> log_cx);
  for (; row + 3 * step < d.rows; row += 4 * step) {   // four rows' loads before their stores
    uint32_t w[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) load_codes<D>(d, row + i * step, chunk, w[i], s[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) store_values<D, kStream>(d, row + i * step, chunk, w[i], s[i]);
  }
  for (; row < d.rows; row += step) {
    uint32_t w, s;
    load_codes<D>(d, row, chunk, w, s);
    store_values<D, kStream>(d, row, chunk, w, s);
  }
}

// Lanes of a workgroup along a row of `chunks` chunks: the power of two at or above, at most 256.
int log_lanes(int chunks) {
  int l = 2;
  while (l < 8 && (1 << l) < chunks) ++l;
  return l;
}

// Grid of a row kernel: x strides over the rows, y stays within its 65535 for every valid size.  About 2048
// workgroups, eight a compute unit, so that a lane has several rows in flight (32768 x 4096 bf16 along the
// rows: 77 us with a workgroup for every 256 chunks, 64 with 2048).
dim3 row_grid(int rows, int chunks, int log_cx) {
  const int per = 256 >> log_cx, y = ceil_div(chunks, 1 << log_cx);
  return dim3((unsigned)std::min(ceil_div(rows, per), std::max(1, 2048 / y)), (unsigned)y);
}

// 4 columns a lane or more, 256 lanes a workgroup: at most 32768 workgroups along a row.
constexpr int kMaxCols = GGEMM_MX4_MAX_COLS;

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
  const bool no_rows = q->index && q->x_rows == 0;   // an index that picks from nothing: x is not read
  if ((!q->x && !no_rows) || q->ld < q->cols || !aligned(q->x, elem_bytes(q->dtype)) || (q->index && (q->x_rows < 0 || !aligned(q->index, 4))))
    return GGEMM_ERR_INVALID;
  if (along && !codes_ok(q->codes, q->ld_codes, q->scales, q->ld_scales, q->cols)) return GGEMM_ERR_INVALID;
  if (down && !codes_ok(q->codes_t, q->ld_codes_t, q->scales_t, q->ld_scales_t, q->rows)) return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(q->dtype, [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (down) {
      const int64_t tiles = (int64_t)ceil_div(q->rows, Turn<D>::kRows) * ceil_div(q->cols, Turn<D>::kCols);
      const unsigned grid = (unsigned)std::min<int64_t>(tiles, 1 << 20);
      auto lines = [](const uint8_t* p, int64_t ld) { return aligned(p, 128) && ld % 128 == 0; };
      const bool stream = lines(q->codes_t, q->ld_codes_t) && (!along || lines(q->codes, q->ld_codes));
      auto go = [&](auto a, auto st) {
        quant_turn_kernel<D, decltype(a)::value, decltype(st)::value><<<grid, Turn<D>::kThreads, 0, s>>>(*q);
      };
      using std::true_type;
      using std::false_type;
      if (along) stream ? go(true_type{}, true_type{}) : go(true_type{}, false_type{});
      else stream ? go(false_type{}, true_type{}) : go(false_type{}, false_type{});
    } else {
      const int chunks = 4 * ceil_div(q->cols, 32), l = log_lanes(chunks);
      quant_rows_kernel<D><<<row_grid(q->rows, chunks, l), kThreads, 0, s>>>(*q, l);
    }
  }); });
}

int mx4_dequantize(const ggemm_mx4_dequant_t* d, hipStream_t s) {
  if (!d || d->rows < 0 || d->cols < 0 || d->cols > kMaxCols || !elem_known(d->dtype)) return GGEMM_ERR_INVALID;
  if (d->rows == 0 || d->cols == 0) return GGEMM_OK;
  if (!codes_ok(d->codes, d->ld_codes, d->scales, d->ld_scales, d->cols) || !d->y || d->ld < d->cols ||
      !aligned(d->y, elem_bytes(d->dtype)))
    return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(d->dtype, [&](auto t) {
    constexpr int D = decltype(t)::value;
    const int chunks = ceil_div(d->cols, Sixteen<D>::N), l = log_lanes(chunks);
    const dim3 grid = row_grid(d->rows, chunks, l);
    if (aligned(d->y, 64) && d->ld * elem_bytes(D) % 64 == 0) dequant_kernel<D, true><<<grid, kThreads, 0, s>>>(*d, l);
    else dequant_kernel<D, false><<<grid, kThreads, 0, s>>>(*d, l);
  }); });
}

}  // namespace ggemm

extern "C" int ggemm_mx4_quantize(const ggemm_mx4_quant_t* q, hipStream_t stream) {
  return ggemm::mx4_quantize(q, stream);
}
extern "C" int ggemm_mx4_dequantize(const ggemm_mx4_dequant_t* d, hipStream_t stream) {
  return ggemm::mx4_dequantize(d, stream);
}
