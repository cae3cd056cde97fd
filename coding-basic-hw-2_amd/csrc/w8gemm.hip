// w8gemm.hip -- grouped products of 8-bit integers with scales for rows and columns (include/ggemm_w8.h).
//
// Tiles and the kernel for few rows of tiles.hpp on v_mfma_i32_32x32x32_i8 (16x16x64): sums are exact, k < 2^17 keeps them
// below 2^31.  A row's and a column's scale, the activation and the pair's product come in the epilogue, in 32-bit floating
// point; the sum is rounded to it first (at most 2^-24 of it).
// Bound: large products, the loop's idle cycles, a third (matrix cores busy 65 % of 0.80 million), and the clock, which ranges from 1.43
// to 1.77 GHz over launches one after another (8192^3: 434 to 557 us, 2.0 to 2.5 POP/s); decoding, the bytes of the weights (64
// experts of 4096 x 2048 twice, 8 rows each: 180 us, 5.8 TB/s).
#include <algorithm>
#include <type_traits>

#include "ggemm_w8.h"
#include "act.hpp"
#include "tiles.hpp"

namespace ggemm {
namespace {

struct Place {
  int g, m0, m_end, n0, nk;
  bool whole;   // every row and column of the tile exists
};

// c = (s sa) sb, or act of it times the same of the second weights
template <int D, int ACT>
struct Product {
  using T = typename Elem<D>::T;
  using M = MmaI8;
  using Place = ggemm::Place;
  static constexpr bool kADown = false, kBDown = false, kPair = ACT != 0;
  static constexpr bool kDead = false;
  static constexpr int E = 8;
  ggemm_w8_gemm_t p;
  bool stream;
  __device__ __forceinline__ RowGroups rows() const { return RowGroups{p.offsets, p.groups, p.m}; }
  template <int BM, int BN>
  __device__ __forceinline__ GroupTiles<BM> groups() const { return GroupTiles<BM>(rows(), 0, ceil_div(p.n, kPair ? BN / 2 : BN)); }
  template <class C>
  __device__ __forceinline__ Place place(const GroupTiles<C::BM>& first, int t) const {
    constexpr int width = kPair ? C::BN / 2 : C::BN;
    const int nt = ceil_div(p.n, width);
    const RowSpan s = find_group(rows(), first, t, nt);
    if (s.g < 0) return Place{-1};
    int tm, tn;
    tile_raster(t, ceil_div(s.hi - s.lo, C::BM), nt, tm, tn);
    const int m0 = s.lo + tm * C::BM, n0 = tn * width;
    return Place{s.g, m0, s.hi, n0, ceil_div(p.k, 128), m0 + C::BM <= s.hi && n0 + width <= p.n};
  }
  template <class C>
  struct Src {
    Along<C, C::BM> a;
    Along<C, C::BN, kPair> b;
    __device__ __forceinline__ void prepare(int kt, int wave) {
      a.prepare(kt, wave);
      b.prepare(kt, wave);
    }
    // integers: zeros on one side are enough
    __device__ __forceinline__ bool ragged(int kt) const { return a.ragged(kt); }
    __device__ __forceinline__ void clear(int kt, uint8_t* slot) const { a.clear(kt, slot); }
  };
  template <class C>
  __device__ __forceinline__ Src<C> source(const Place& c, int wave, int lane) const {
    auto bytes = [](const int8_t* x) { return reinterpret_cast<const uint8_t*>(x); };
    const int64_t b0 = c.g * p.b_stride + c.n0 * p.ldb;
    return Src<C>{Along<C, C::BM>(bytes(p.a) + c.m0 * p.lda, nullptr, p.lda, c.m_end - c.m0, p.k, wave, lane, InOrder{(uint32_t)p.lda}),
                  Along<C, C::BN, kPair>(bytes(p.b) + b0, bytes(p.b_up) + b0, p.ldb, p.n - c.n0, p.k, wave, lane, InOrder{(uint32_t)p.ldb})};
  }
  __device__ __forceinline__ FewRows few(const Place& c, int i) const {
    auto bytes = [](const int8_t* x) { return reinterpret_cast<const uint8_t*>(x); };
    const int64_t b0 = c.g * p.b_stride + c.n0 * p.ldb;
    const int end = (p.k + 15) & ~15;
    const int64_t left = (p.n - c.n0 - 1) * p.ldb + end;   // 16 columns on: that much less, nothing if there are none
    const uint32_t vb = (uint32_t)i * (uint32_t)p.ldb;
    return FewRows{bytes(p.a) + c.m0 * p.lda, {bytes(p.b) + b0, kPair ? bytes(p.b_up) + b0 : bytes(p.b) + b0 + 16 * p.ldb},
                   (c.m_end - c.m0 - 1) * p.lda + end, {left, kPair ? left : left - 16 * p.ldb}, (uint32_t)i * (uint32_t)p.lda, {vb, vb}, p.k};
  }
  template <bool kWhole>
  __device__ __forceinline__ Nothing fetch(const Place&, int, int) const {
    return {};
  }
  template <bool kWhole, int E>
  __device__ __forceinline__ void emit(const Place& c, int row, int col, const float (&v)[E], const float (&u)[E], Nothing) const {
    const int64_t r = c.m0 + row, j = c.n0 + col;
    if (!kWhole && (r >= c.m_end || j >= p.n)) return;
    const int ok = kWhole ? E : p.n - (int)j;
    const int64_t sj = c.g * p.b_scales_stride + j;
    const float sa = p.a_scales[r];
    float o[E], s[E];
    load_some(p.b_scales + sj, ok, s);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = v[e] * sa * s[e];
    if constexpr (kPair) {
      load_some(p.b_up_scales + sj, ok, s);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = act_value<ACT>(o[e]) * (u[e] * sa * s[e]);
    }
    store_some(static_cast<T*>(p.c) + r * p.ldc + j, ok, o, stream);
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
// Tiles of BM rows that a call's groups can need at most; cols: of a tile, half of them columns of C where it computes a pair.
int64_t tiles_of(const ggemm_w8_gemm_t& p, int bm, int cols) { return row_tiles(p.groups, p.m, bm) * ceil_div(p.n, p.act ? cols / 2 : cols); }

template <class P>
void run(const P& p, hipStream_t s) {
  const int bm = rows_tile(p.p.groups, p.p.m, p.p.n, P::kPair ? 64 : 128, true);
  if (bm == 256) run_tiles<Tile256>(p, tiles_of(p.p, 256, 256), s);
  else if (bm == 128) run_tiles<Tile128>(p, tiles_of(p.p, 128, 128), s);
  else if (bm == 64) run_tiles<Tile64>(p, tiles_of(p.p, 64, 128), s);
  else few_kernel<P><<<(unsigned)tiles_of(p.p, 16, 32), 256, 0, s>>>(p);
}

}  // namespace

int w8_gemm(const ggemm_w8_gemm_t* p, hipStream_t s) {
  if (!args_ok(p)) return GGEMM_ERR_INVALID;
  if (p->m == 0 || p->n == 0) return GGEMM_OK;
  if (tiles_of(*p, 64, 128) >= (1 << 23)) return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(p->dtype, [&](auto d) {
    constexpr int D = decltype(d)::value;
    const bool stream = whole_runs(p->c, p->ldc * elem_bytes(D));
    if (!p->act) run(Product<D, 0>{*p, stream}, s);
    else with_act(p->act, [&](auto act) { run(Product<D, decltype(act)::value>{*p, stream}, s); });
  }); });
}

}  // namespace ggemm

extern "C" size_t ggemm_w8_gemm_workspace(const ggemm_w8_gemm_t*) { return 0; }
extern "C" int ggemm_w8_gemm(const ggemm_w8_gemm_t* p, void*, size_t, hipStream_t stream) { return ggemm::w8_gemm(p, stream); }
