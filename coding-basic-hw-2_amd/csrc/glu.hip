// glu.hip -- the gated feed-forward block and its gradients (include/ggemm_glu.h).
//
// Five products by the tiles of tiles.hpp, each with the work that belongs to its result in the epilogue: two launches
// forward (gate, up, activation and product; down), three backward (hidden gradients; dx; the weights' gradients), one more
// for the copies of gathered rows.  What is kept between launches is 16-bit: h, dgate and dup are matrix operands.
// Bound: long inner dimensions, the loop's idle cycles: matrix cores busy 66 % of them forward and 55 to 60 % where an operand lies down the
// inner dimension, at 1.55 to 1.95 GHz in the same launches, 1.1 to 1.26 and 1.0 to 1.1 PFLOP/s; short ones, a tile's first loads and
// its stores.
// Registers: the 256 x 256 tiles take all 256; hidden keeps one to three values of the epilogue's in scratch memory over the stages, the
// kernels over rows 23 to 66 scalars in lanes, both outside the loop of the stages.
#include <algorithm>
#include <type_traits>

#include "act.hpp"
#include "tiles.hpp"

namespace ggemm {
namespace {

// Where a tile of rows of a group lies: rows [m0, m_end), first column, stages of the inner dimension.
struct Place {
  int g, m0, m_end, n0, nk;
  bool whole;   // every row and column of the tile exists
};
template <class C>
__device__ __forceinline__ Place row_place(const RowGroups& rows, const GroupTiles<C::BM>& first, int t, int n, int width, int nk) {
  const int nt = ceil_div(n, width);
  const RowSpan s = find_group(rows, first, t, nt);
  if (s.g < 0) return Place{-1};
  int tm, tn;
  tile_raster(t, ceil_div(s.hi - s.lo, C::BM), nt, tm, tn);
  const int m0 = s.lo + tm * C::BM, n0 = tn * width;
  return Place{s.g, m0, s.hi, n0, nk, m0 + C::BM <= s.hi && n0 + width <= n};
}
__device__ __forceinline__ const uint8_t* bytes_of(const void* p) { return static_cast<const uint8_t*>(p); }

// The rows of x that an index picks, or none.
struct Picked {
  const int32_t* index;
  int x_rows;
  // index entry of row r, or -1
  __device__ __forceinline__ int at(int r) const {
    const int i = index[r];
    return (uint32_t)i < (uint32_t)x_rows ? i : -1;
  }
  __device__ __forceinline__ bool live(int r) const { return !index || at(r) >= 0; }
};
// Products over rows that an index may pick: results of rows of which it names none are stored as zeros, not as what zeros times
// the weights give, which is NaN for an Inf.
__device__ __forceinline__ int row_entry(const ggemm_glu_t& p, const Place& c, int row) {
  return p.index && c.m0 + row < c.m_end ? p.index[c.m0 + row] : 0;
}
__device__ __forceinline__ bool names_row(const ggemm_glu_t& p, int entry) { return !p.index || (uint32_t)entry < (uint32_t)p.x_rows; }

// h = act(x Wg^T) (x Wu^T), and gate and up where they are kept.  Both products in one tile: half the columns, twice the
// weights, x read once (8192 x 4096 x 8192: 880 to 1000 us, 1.1 to 1.25 PFLOP/s; 4096 tokens, 2 of 16 experts (1024, 2048), all kept: 107 us, of
// which 18 are the stores).
template <int D, int ACT>
struct Up {
  using T = typename Elem<D>::T;
  using M = typename MmaOf<D>::M;
  using Place = ggemm::Place;
  static constexpr bool kADown = false, kBDown = false, kPair = true;
  static constexpr bool kDead = true;
  static constexpr int E = 8;
  ggemm_glu_t p;
  T* h;
  int64_t ldh;
  bool stream;   // gate and up
  __device__ __forceinline__ int entry(const Place& c, int row) const { return row_entry(p, c, row); }
  __device__ __forceinline__ bool names(int e) const { return names_row(p, e); }
  __device__ __forceinline__ RowGroups rows() const { return RowGroups{p.offsets, p.groups, p.rows}; }
  template <int BM, int BN>
  __device__ __forceinline__ GroupTiles<BM> groups() const { return GroupTiles<BM>(rows(), 0, ceil_div(p.d_ff, BN / 2)); }
  template <class C>
  __device__ __forceinline__ Place place(const GroupTiles<C::BM>& first, int t) const {
    return row_place<C>(rows(), first, t, p.d_ff, C::BN / 2, ceil_div(p.d_model, 64));
  }
  template <class C>
  struct Src {
    Along<C, C::BM> a;
    Along<C, C::BN, true> b;
    __device__ __forceinline__ void prepare(int kt, int wave) {
      a.prepare(kt, wave);
      b.prepare(kt, wave);
    }
    __device__ __forceinline__ bool ragged(int kt) const { return a.ragged(kt); }
    __device__ __forceinline__ void clear(int kt, uint8_t* slot) const {
      a.clear(kt, slot);
      b.clear(kt, slot + C::SA);
    }
  };
  template <class C>
  __device__ __forceinline__ Src<C> source(const Place& c, int wave, int lane) const {
    const int64_t px = 2 * p.ldx, pw = 2 * p.ldw, w0 = 2 * (c.g * p.w_stride + c.n0 * p.ldw);
    const int bytes = 2 * p.d_model, n = p.d_ff - c.n0;
    const Picked pick{p.index, p.x_rows};
    auto at = [&](int row) -> uint32_t {
      if (!p.index) return (uint32_t)row * (uint32_t)px;
      const int i = c.m0 + row < c.m_end ? pick.at(c.m0 + row) : -1;
      return i < 0 ? kOut : (uint32_t)i * (uint32_t)px;
    };
    const uint8_t* const x = bytes_of(p.x) + (p.index ? 0 : c.m0 * px);
    return Src<C>{Along<C, C::BM>(x, nullptr, px, p.index ? p.x_rows : c.m_end - c.m0, bytes, wave, lane, at),
                  Along<C, C::BN, true>(bytes_of(p.w_gate) + w0, bytes_of(p.w_up) + w0, pw, n, bytes, wave, lane, InOrder{(uint32_t)pw})};
  }
  __device__ __forceinline__ FewRows few(const Place& c, int i) const {
    const int64_t px = 2 * p.ldx, pw = 2 * p.ldw, w0 = 2 * (c.g * p.w_stride + c.n0 * p.ldw);
    const int bytes = 2 * p.d_model, end = (bytes + 15) & ~15;
    uint32_t va = (uint32_t)i * (uint32_t)px;
    if (p.index) {
      const int r = c.m0 + i < c.m_end ? Picked{p.index, p.x_rows}.at(c.m0 + i) : -1;
      va = r < 0 ? kOut : (uint32_t)r * (uint32_t)px;
    }
    const int64_t left = (p.d_ff - c.n0 - 1) * pw + end;
    return FewRows{bytes_of(p.x) + (p.index ? 0 : c.m0 * px), {bytes_of(p.w_gate) + w0, bytes_of(p.w_up) + w0},
                   ((p.index ? p.x_rows : c.m_end - c.m0) - 1) * px + end, {left, left}, va, {(uint32_t)i * (uint32_t)pw, (uint32_t)i * (uint32_t)pw},
                   bytes};
  }
  template <bool kWhole>
  __device__ __forceinline__ Nothing fetch(const Place&, int, int) const {
    return {};
  }
  template <bool kWhole, int E>
  __device__ __forceinline__ void emit(const Place& c, int row, int col, const float (&v)[E], const float (&u)[E], Nothing) const {
    const int64_t r = c.m0 + row, j = c.n0 + col;
    if (!kWhole && (r >= c.m_end || j >= p.d_ff)) return;
    const int ok = kWhole ? E : p.d_ff - (int)j;
    float g[E], w[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = v[e], w[e] = u[e], o[e] = act_value<ACT>(v[e]) * u[e];
    store_some(h + r * ldh + j, ok, o, true);
    if (p.gate) {
      store_some(static_cast<T*>(p.gate) + r * p.ldg + j, ok, g, stream);
      store_some(static_cast<T*>(p.up) + r * p.ldg + j, ok, w, stream);
    }
  }
};

// y = h Wd^T (8192 x 8192 x 4096: 430 to 500 us, 1.1 to 1.27 PFLOP/s)
template <int D>
struct DownProduct {
  using T = typename Elem<D>::T;
  using M = typename MmaOf<D>::M;
  using Place = ggemm::Place;
  static constexpr bool kADown = false, kBDown = false, kPair = false;
  static constexpr bool kDead = true;
  static constexpr int E = 8;
  ggemm_glu_t p;
  const T* h;
  int64_t ldh;
  bool stream;
  __device__ __forceinline__ int entry(const Place& c, int row) const { return row_entry(p, c, row); }
  __device__ __forceinline__ bool names(int e) const { return names_row(p, e); }
  __device__ __forceinline__ RowGroups rows() const { return RowGroups{p.offsets, p.groups, p.rows}; }
  template <int BM, int BN>
  __device__ __forceinline__ GroupTiles<BM> groups() const { return GroupTiles<BM>(rows(), 0, ceil_div(p.d_model, BN)); }
  template <class C>
  __device__ __forceinline__ Place place(const GroupTiles<C::BM>& first, int t) const {
    return row_place<C>(rows(), first, t, p.d_model, C::BN, ceil_div(p.d_ff, 64));
  }
  template <class C>
  struct Src {
    Along<C, C::BM> a;
    Along<C, C::BN> b;
    __device__ __forceinline__ void prepare(int kt, int wave) {
      a.prepare(kt, wave);
      b.prepare(kt, wave);
    }
    __device__ __forceinline__ bool ragged(int kt) const { return a.ragged(kt); }
    __device__ __forceinline__ void clear(int kt, uint8_t* slot) const {
      a.clear(kt, slot);
      b.clear(kt, slot + C::SA);
    }
  };
  template <class C>
  __device__ __forceinline__ Src<C> source(const Place& c, int wave, int lane) const {
    const int64_t ph = 2 * ldh, pw = 2 * p.ldd;
    const int bytes = 2 * p.d_ff;
    return Src<C>{Along<C, C::BM>(bytes_of(h) + c.m0 * ph, nullptr, ph, c.m_end - c.m0, bytes, wave, lane, InOrder{(uint32_t)ph}),
                  Along<C, C::BN>(bytes_of(p.w_down) + 2 * (c.g * p.d_stride + c.n0 * p.ldd), nullptr, pw, p.d_model - c.n0, bytes, wave,
                                  lane, InOrder{(uint32_t)pw})};
  }
  __device__ __forceinline__ FewRows few(const Place& c, int i) const {
    const int64_t ph = 2 * ldh, pw = 2 * p.ldd;
    const int bytes = 2 * p.d_ff, end = (bytes + 15) & ~15;
    const uint8_t* const w = bytes_of(p.w_down) + 2 * (c.g * p.d_stride + c.n0 * p.ldd);
    const int64_t left = (p.d_model - c.n0 - 1) * pw + end;   // 16 columns on: that much less, nothing if there are none
    return FewRows{bytes_of(h) + c.m0 * ph, {w, w + 16 * pw}, (c.m_end - c.m0 - 1) * ph + end, {left, left - 16 * pw},
                   (uint32_t)i * (uint32_t)ph, {(uint32_t)i * (uint32_t)pw, (uint32_t)i * (uint32_t)pw}, bytes};
  }
  template <bool kWhole>
  __device__ __forceinline__ Nothing fetch(const Place&, int, int) const {
    return {};
  }
  template <bool kWhole, int E>
  __device__ __forceinline__ void emit(const Place& c, int row, int col, const float (&v)[E], const float (&)[E], Nothing) const {
    const int64_t r = c.m0 + row, j = c.n0 + col;
    if (!kWhole && (r >= c.m_end || j >= p.d_model)) return;
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = v[e];
    store_some(static_cast<T*>(p.y) + r * p.ldy + j, kWhole ? E : p.d_model - (int)j, o, stream);
  }
};

// dh = dy Wd, and from it, gate and up: dgate = dh up act'(gate), dup = dh act(gate), h = act(gate) up.  dh stays in registers.  Bound:
// five matrices pass through the epilogue, under which nothing else is multiplied (32768 rows, (2048, 4096): 760 to 830 us,
// 0.66 to 0.72 PFLOP/s; 632 without reading gate and up, 540 would be the product's).
template <int D, int ACT>
struct Hidden {
  using T = typename Elem<D>::T;
  using M = typename MmaOf<D>::M;
  using Place = ggemm::Place;
  static constexpr bool kADown = false, kBDown = true, kPair = false;
  static constexpr bool kDead = false;
  static constexpr int E = 8;
  ggemm_glu_t p;
  const void* dy;
  int64_t lddy;
  T *dg, *du, *h;   // dg and du or h: NULL where nobody reads them
  int64_t ldh;
  __device__ __forceinline__ RowGroups rows() const { return RowGroups{p.offsets, p.groups, p.rows}; }
  template <int BM, int BN>
  __device__ __forceinline__ GroupTiles<BM> groups() const { return GroupTiles<BM>(rows(), 0, ceil_div(p.d_ff, BN)); }
  template <class C>
  __device__ __forceinline__ Place place(const GroupTiles<C::BM>& first, int t) const {
    return row_place<C>(rows(), first, t, p.d_ff, C::BN, ceil_div(p.d_model, 64));
  }
  template <class C>
  struct Src {
    Along<C, C::BM> a;
    Down<C, C::BN> b;
    __device__ __forceinline__ void prepare(int kt, int wave) {
      a.prepare(kt, wave);
      b.prepare(b.base, kt);
    }
    __device__ __forceinline__ bool ragged(int kt) const { return a.ragged(kt); }
    __device__ __forceinline__ void clear(int kt, uint8_t* slot) const { a.clear(kt, slot); }
  };
  template <class C>
  __device__ __forceinline__ Src<C> source(const Place& c, int wave, int lane) const {
    const int64_t py = 2 * lddy;
    return Src<C>{Along<C, C::BM>(bytes_of(dy) + c.m0 * py, nullptr, py, c.m_end - c.m0, 2 * p.d_model, wave, lane, InOrder{(uint32_t)py}),
                  Down<C, C::BN>(bytes_of(p.w_down) + 2 * (c.g * p.d_stride + c.n0), 2 * p.ldd, p.d_model, p.d_ff - c.n0, wave, lane)};
  }
  struct Kept {
    Run<T, E> g, u;
    bool live;
  };
  template <bool kWhole>
  __device__ __forceinline__ Kept fetch(const Place& c, int row, int col) const {
    Kept k{};
    const int64_t r = c.m0 + row, j = c.n0 + col;
    if (!kWhole && (r >= c.m_end || j >= p.d_ff)) return k;
    const int ok = kWhole ? E : p.d_ff - (int)j;
    k.live = Picked{p.index, p.x_rows}.live((int)r);
    k.g = run_some<T, E>(static_cast<const T*>(p.gate) + r * p.ldg + j, ok);
    k.u = run_some<T, E>(static_cast<const T*>(p.up) + r * p.ldg + j, ok);
    return k;
  }
  template <bool kWhole, int E>
  __device__ __forceinline__ void emit(const Place& c, int row, int col, const float (&v)[E], const float (&)[E], const Kept& k) const {
    const int64_t r = c.m0 + row, j = c.n0 + col;
    if (!kWhole && (r >= c.m_end || j >= p.d_ff)) return;
    const int ok = kWhole ? E : p.d_ff - (int)j;
    const bool live = k.live;
    float g[E], u[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      g[e] = (float)k.g.x[e], u[e] = (float)k.u.x[e];
      float q, dq;
      act_parts<ACT>(g[e], q, dq);
      const float a = g[e] * q, w = u[e];
      u[e] = live ? v[e] * a : 0.0f;
      o[e] = live ? a * w : 0.0f;
      g[e] = live ? v[e] * w * fmaf(g[e], dq, q) : 0.0f;
    }
    if (dg) {
      store_some(dg + r * ldh + j, ok, g, true);
      store_some(du + r * ldh + j, ok, u, true);
    }
    if (h) store_some(h + r * ldh + j, ok, o, true);
  }
};

// dx = dgate Wg + dup Wu: two inner dimensions, one after the other, one sum (32768 rows, (2048, 4096): 1080 us, 1.0
// PFLOP/s).  Weights as they lie, down the inner dimension: a transposed copy of them would be read and written first.
template <int D>
struct InputGrad {
  using T = typename Elem<D>::T;
  using M = typename MmaOf<D>::M;
  using Place = ggemm::Place;
  static constexpr bool kADown = false, kBDown = true, kPair = false;
  static constexpr bool kDead = true;
  static constexpr int E = 8;
  ggemm_glu_t p;
  void* dx;
  int64_t lddx;
  const T *dg, *du;
  int64_t ldh;
  bool stream;
  __device__ __forceinline__ int entry(const Place& c, int row) const { return row_entry(p, c, row); }
  __device__ __forceinline__ bool names(int e) const { return names_row(p, e); }
  __device__ __forceinline__ RowGroups rows() const { return RowGroups{p.offsets, p.groups, p.rows}; }
  template <int BM, int BN>
  __device__ __forceinline__ GroupTiles<BM> groups() const { return GroupTiles<BM>(rows(), 0, ceil_div(p.d_model, BN)); }
  template <class C>
  __device__ __forceinline__ Place place(const GroupTiles<C::BM>& first, int t) const {
    return row_place<C>(rows(), first, t, p.d_model, C::BN, 2 * ceil_div(p.d_ff, 64));
  }
  template <class C>
  struct Src {
    Along<C, C::BM> a;   // base2: dup
    Down<C, C::BN> b;
    const uint8_t* b2;
    int half;            // stages of each
    __device__ __forceinline__ void prepare(int kt, int wave) {
      const bool second = kt >= half;
      a.prepare(second ? a.base2 : a.base, nullptr, second ? kt - half : kt, wave);
      b.prepare(second ? b2 : b.base, second ? kt - half : kt);
    }
    __device__ __forceinline__ bool ragged(int kt) const { return a.ragged(kt >= half ? kt - half : kt); }
    __device__ __forceinline__ void clear(int kt, uint8_t* slot) const { a.clear(kt >= half ? kt - half : kt, slot); }
  };
  template <class C>
  __device__ __forceinline__ Src<C> source(const Place& c, int wave, int lane) const {
    const int64_t ph = 2 * ldh, w0 = 2 * (c.g * p.w_stride + c.n0);
    return Src<C>{Along<C, C::BM>(bytes_of(dg) + c.m0 * ph, bytes_of(du) + c.m0 * ph, ph, c.m_end - c.m0, 2 * p.d_ff, wave, lane,
                                  InOrder{(uint32_t)ph}),
                  Down<C, C::BN>(bytes_of(p.w_gate) + w0, 2 * p.ldw, p.d_ff, p.d_model - c.n0, wave, lane), bytes_of(p.w_up) + w0,
                  ceil_div(p.d_ff, 64)};
  }
  template <bool kWhole>
  __device__ __forceinline__ Nothing fetch(const Place&, int, int) const {
    return {};
  }
  template <bool kWhole, int E>
  __device__ __forceinline__ void emit(const Place& c, int row, int col, const float (&v)[E], const float (&)[E], Nothing) const {
    const int64_t r = c.m0 + row, j = c.n0 + col;
    if (!kWhole && (r >= c.m_end || j >= p.d_model)) return;
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = v[e];
    store_some(static_cast<T*>(dx) + r * lddx + j, kWhole ? E : p.d_model - (int)j, o, stream);
  }
};

// Gradients of the weights: dWg = dgate^T x, dWu = dup^T x (d_ff x d_model), dWd = dy^T h (d_model x d_ff), in one launch, so
// that one last round is partly filled, not three.  Both operands down the inner dimension, a group's rows (16 groups of 2048
// rows, (2048, 4096): 1570 us, 1.05 PFLOP/s; 2 groups 1370: a tile costs about 10 us beside its stages).
struct WeightPlace {
  int g, which, lo, m0, n0, depth, nk;
  bool whole;
};
template <int D, int W>
struct WeightGrad {
  using T = typename Elem<D>::T;
  using O = typename Elem<W>::T;
  using M = typename MmaOf<D>::M;
  using Place = WeightPlace;
  static constexpr bool kADown = true, kBDown = true, kPair = false;
  static constexpr bool kDead = false;
  static constexpr int E = 8;
  ggemm_glu_t p;        // x and dy: one row for each of the call's rows
  ggemm_glu_grad_t d;
  const T *dg, *du, *h;
  int64_t ldh;
  int first_of;   // 0: all three, 2: dWd only
  bool stream;
  __device__ __forceinline__ RowGroups rows() const { return RowGroups{p.offsets, p.groups, p.rows}; }
  template <int BM, int BN>
  __device__ __forceinline__ int groups() const { return 0; }
  template <class C>
  __device__ __forceinline__ Place place(int, int t) const {
    static_assert(C::BM == C::BN, "as many tiles of each matrix");
    const int tf = ceil_div(p.d_ff, C::BM), td = ceil_div(p.d_model, C::BM), per = tf * td;
    Place a;
    a.which = first_of + t / (per * p.groups);
    t %= per * p.groups;
    a.g = t / per;
    int hi, tm, tn;
    rows().span(a.g, a.lo, hi);
    a.depth = max(hi - a.lo, 0);
    a.nk = ceil_div(a.depth, 64);
    const bool down = a.which == 2;
    tile_raster(t % per, down ? td : tf, down ? tf : td, tm, tn);
    a.m0 = tm * C::BM;
    a.n0 = tn * C::BM;
    a.whole = a.m0 + C::BM <= (down ? p.d_model : p.d_ff) && a.n0 + C::BM <= (down ? p.d_ff : p.d_model);
    return a;
  }
  template <class C>
  struct Src {
    Down<C, C::BM> a;
    Down<C, C::BN> b;
    __device__ __forceinline__ void prepare(int kt, int) {
      a.prepare(a.base, kt);
      b.prepare(b.base, kt);
    }
    __device__ __forceinline__ bool ragged(int) const { return false; }
    __device__ __forceinline__ void clear(int, uint8_t*) const {}
  };
  template <class C>
  __device__ __forceinline__ Src<C> source(const Place& c, int wave, int lane) const {
    const bool down = c.which == 2;
    const int64_t pa = 2 * (down ? d.lddy : ldh), pb = 2 * (down ? ldh : p.ldx);
    const uint8_t* const a = bytes_of(down ? d.dy : c.which ? (const void*)du : dg) + c.lo * pa + 2 * c.m0;
    const uint8_t* const b = bytes_of(down ? (const void*)h : p.x) + c.lo * pb + 2 * c.n0;
    const int m = down ? p.d_model : p.d_ff, n = down ? p.d_ff : p.d_model;
    return Src<C>{Down<C, C::BM>(a, pa, c.depth, m - c.m0, wave, lane), Down<C, C::BN>(b, pb, c.depth, n - c.n0, wave, lane)};
  }
  template <bool kWhole>
  __device__ __forceinline__ Nothing fetch(const Place&, int, int) const {
    return {};
  }
  template <bool kWhole, int E>
  __device__ __forceinline__ void emit(const Place& c, int row, int col, const float (&v)[E], const float (&)[E], Nothing) const {
    const bool down = c.which == 2;
    const int m = down ? p.d_model : p.d_ff, n = down ? p.d_ff : p.d_model, i = c.m0 + row, j = c.n0 + col;
    if (!kWhole && (i >= m || j >= n)) return;
    O* const base = static_cast<O*>(down ? d.dw_down : c.which ? d.dw_up : d.dw_gate);
    O* const out = base + (down ? c.g * d.dd_stride + i * d.lddd : c.g * d.dw_stride + i * d.lddw) + j;
    float o[E];
    if (d.dw_beta != 0.0f) {
      load_some(static_cast<const O*>(out), kWhole ? E : n - j, o);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(d.dw_beta, o[e], v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = v[e];
    }
    store_some(out, kWhole ? E : n - j, o, stream);
  }
};

// Rows of x in the call's order and rows of dy, zeros where the index names none, for the weights' gradients: 256 lanes cover cx
// chunks of 8 columns (a power of two) of 256 / cx rows.  (Rows looked up in the products' loop instead: 16 groups of
// 2048 rows, (2048, 4096), 1820 us for the products, 1570 without an index; these copies take 80, 5 TB/s.)  xg or yg may be NULL.
__global__ void __launch_bounds__(256) gather_kernel(ggemm_glu_t p, const void* dy, int64_t lddy, u32x4* xg, u32x4* yg, int chunks, int log_cx) {
  const int c = (blockIdx.y << log_cx) + (threadIdx.x & ((1 << log_cx) - 1));
  if (c >= chunks) return;
  const int64_t step = (int64_t)gridDim.x << (8 - log_cx);
  for (int64_t r = ((int64_t)blockIdx.x << (8 - log_cx)) + (threadIdx.x >> log_cx); r < p.rows; r += step) {
    const int64_t at = Picked{p.index, p.x_rows}.at((int)r);
    u32x4 x{}, y{};
    if (at >= 0 && xg) x = *reinterpret_cast<const u32x4*>(bytes_of(p.x) + 2 * (at * p.ldx + 8 * c));
    if (at >= 0 && yg) y = *reinterpret_cast<const u32x4*>(bytes_of(dy) + 2 * (r * lddy + 8 * c));
    if (xg) xg[r * chunks + c] = x;
    if (yg) yg[r * chunks + c] = y;
  }
}

// Tiles of BM rows and `width` columns that a call's groups can need at most.
int64_t tiles_of(const ggemm_glu_t& p, int bm, int n, int width) { return row_tiles(p.groups, p.rows, bm) * ceil_div(n, width); }

// A product over rows of groups with n columns.
template <class P>
void run_rows(const P& p, int n, hipStream_t s) {
  constexpr int H = P::kPair ? 2 : 1;
  const int bm = rows_tile(p.p.groups, p.p.rows, n, 128 / H, !P::kBDown);
  if (bm == 256) run_tiles<Tile256>(p, tiles_of(p.p, 256, n, 256 / H), s);
  else if (bm == 128) run_tiles<Tile128>(p, tiles_of(p.p, 128, n, 128 / H), s);
  else if (bm == 64) run_tiles<Tile64>(p, tiles_of(p.p, 64, n, 128 / H), s);
  else if constexpr (!P::kBDown) few_kernel<P><<<(unsigned)tiles_of(p.p, 16, n, 32 / H), 256, 0, s>>>(p);
}

// f(integral_constant<int, D>) for a 16-bit type
template <class F>
void with_type(int dtype, F&& f) {
  if (dtype == GGEMM_BF16) f(std::integral_constant<int, GGEMM_BF16>{});
  else f(std::integral_constant<int, GGEMM_F16>{});
}

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
int64_t ld_hidden(const ggemm_glu_t& p) { return (int64_t)align_up((size_t)p.d_ff, 32); }   // rows of whole runs of 64 bytes
size_t hidden_bytes(const ggemm_glu_t& p) { return align_up((size_t)p.rows * ld_hidden(p) * 2, 256); }
// The most tiles that a launch over rows or weights can have, in the smallest shape that it may take.
bool tiles_fit(const ggemm_glu_t& p, bool weights) {
  const int64_t n = std::max(p.d_ff, p.d_model);
  const int64_t w = 3ll * p.groups * ceil_div(p.d_ff, 128) * ceil_div(p.d_model, 128);
  return tiles_of(p, 64, (int)n, 64) < (1 << 23) && (!weights || w < (1 << 23));
}

}  // namespace

size_t glu_workspace(const ggemm_glu_t* p) { return shape_ok(p) && tiles_fit(*p, false) ? hidden_bytes(*p) : 0; }

int glu(const ggemm_glu_t* p, void* ws, size_t ws_bytes, hipStream_t s) {
  if (!args_ok(p) || !p->gate != !p->up || !tiles_fit(*p, false)) return GGEMM_ERR_INVALID;
  if (p->rows == 0) return GGEMM_OK;
  if (!p->y || !aligned(p->y, 2) || p->ldy < p->d_model) return GGEMM_ERR_INVALID;
  if (p->gate && (!aligned(p->gate, 2) || !aligned(p->up, 2) || p->ldg < p->d_ff)) return GGEMM_ERR_INVALID;
  if (ws_bytes < glu_workspace(p)) return GGEMM_ERR_WORKSPACE;
  if (!ws || !aligned(ws, 16)) return GGEMM_ERR_INVALID;
  return launch([&] { with_type(p->dtype, [&](auto dt) { with_act(p->act, [&](auto act) {
    constexpr int D = decltype(dt)::value;
    using T = typename Elem<D>::T;
    T* const h = static_cast<T*>(ws);
    const bool kept = whole_runs(p->gate, 2 * p->ldg) && whole_runs(p->up, 2 * p->ldg);
    run_rows(Up<D, decltype(act)::value>{*p, h, ld_hidden(*p), kept}, p->d_ff, s);
    run_rows(DownProduct<D>{*p, h, ld_hidden(*p), whole_runs(p->y, 2 * p->ldy)}, p->d_model, s);
  }); }); });
}

int64_t ld_model(const ggemm_glu_t& p) { return (int64_t)align_up((size_t)p.d_model, 8); }
size_t model_bytes(const ggemm_glu_t& p) { return align_up((size_t)p.rows * ld_model(p) * 2, 256); }

size_t glu_backward_workspace(const ggemm_glu_t* p, const ggemm_glu_grad_t* d) {
  return shape_ok(p) && d && tiles_fit(*p, d->dw_gate || d->dw_down) ? 3 * hidden_bytes(*p) + (p->index ? 2 * model_bytes(*p) : 0) : 0;
}

int glu_backward(const ggemm_glu_t* p, const ggemm_glu_grad_t* d, void* ws, size_t ws_bytes, hipStream_t s) {
  if (!args_ok(p) || !d || !elem_known(d->dw_dtype) || !d->dw_gate != !d->dw_up || !tiles_fit(*p, d->dw_gate || d->dw_down))
    return GGEMM_ERR_INVALID;
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
  if (!d->dw_gate && !d->dw_down && (!d->dx || p->rows == 0)) return GGEMM_OK;
  return launch([&] { with_type(p->dtype, [&](auto dt) {
    constexpr int D = decltype(dt)::value;
    using T = typename Elem<D>::T;
    uint8_t* const b = static_cast<uint8_t*>(ws);
    const size_t n = hidden_bytes(*p);
    T *const dg = reinterpret_cast<T*>(b), *const du = reinterpret_cast<T*>(b + n), *const h = reinterpret_cast<T*>(b + 2 * n);
    const int64_t ldh = ld_hidden(*p);
    if (p->rows > 0) {
      const bool gu = d->dx || d->dw_gate;
      with_act(p->act, [&](auto act) {
        run_rows(Hidden<D, decltype(act)::value>{*p, d->dy, d->lddy, gu ? dg : nullptr, gu ? du : nullptr, d->dw_down ? h : nullptr, ldh},
                 p->d_ff, s);
      });
      if (d->dx) run_rows(InputGrad<D>{*p, d->dx, d->lddx, dg, du, ldh, whole_runs(d->dx, 2 * d->lddx)}, p->d_model, s);
    }
    if (!d->dw_gate && !d->dw_down) return;
    const int matrices = (d->dw_gate ? 2 : 0) + (d->dw_down ? 1 : 0), from = d->dw_gate ? 0 : 2;
    ggemm_glu_t rows = *p;
    ggemm_glu_grad_t grad = *d;
    if (p->index && p->rows > 0) {
      uint8_t *const xg = b + 3 * n, *const yg = xg + model_bytes(*p);
      const int chunks = (int)(ld_model(*p) / 8);
      int log_cx = 0;
      while (log_cx < 8 && (1 << log_cx) < chunks) ++log_cx;
      const int64_t groups = ((int64_t)p->rows + (256 >> log_cx) - 1) >> (8 - log_cx);
      gather_kernel<<<dim3((unsigned)std::min(groups, (int64_t)1 << 16), ceil_div(chunks, 1 << log_cx)), 256, 0, s>>>(
          *p, d->dy, d->lddy, d->dw_gate ? reinterpret_cast<u32x4*>(xg) : nullptr, d->dw_down ? reinterpret_cast<u32x4*>(yg) : nullptr, chunks,
          log_cx);
      rows.x = xg;
      grad.dy = yg;
      rows.ldx = grad.lddy = ld_model(*p);
    }
    auto runs = [&](const void* w, int64_t ld, int64_t stride) {
      const int64_t es = elem_bytes(d->dw_dtype);
      return !w || (whole_runs(w, ld * es) && (p->groups == 1 || stride * es % 64 == 0));
    };
    const bool stream = runs(d->dw_gate, d->lddw, d->dw_stride) && runs(d->dw_up, d->lddw, d->dw_stride) && runs(d->dw_down, d->lddd, d->dd_stride);
    with_elem(d->dw_dtype, [&](auto wt) {
      const WeightGrad<D, decltype(wt)::value> w{rows, grad, dg, du, h, ldh, from, stream};
      auto tiles = [&](int b) { return (int64_t)matrices * p->groups * ceil_div(p->d_ff, b) * ceil_div(p->d_model, b); };
      // 256 x 256 where they fill the compute units and cover at most a seventh more than 128 x 128 tiles do, whose loop is slower but
      // which fit the edges better and store beside another workgroup.  us, 256 and 128: unfilled, 96 tiles over 8192 rows 194 and
      // 136; filled, 16 groups (2048, 4096) of 2048 rows 1451 and 1912, of 512 rows (1024, 2048) 156 and 167, 384 tiles in a round
      // and a half 154 and 143; a ninth more, 8 groups (1100, 2304) of 4096 rows 545 and 575, 64 groups (1152, 1024) of 1024 rows 655 and
      // 604; a sixth more (1152, 2944) 737 and 674, a third more (384, 1024) 397 and 293, 2.7 times (100, 300) 178 and 71.
      if (tiles(256) >= kCus && 7 * tiles(256) <= 2 * tiles(128)) run_tiles<Tile256>(w, tiles(256), s);
      else run_tiles<Tile128>(w, tiles(128), s);
    });
  }); });
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
