// mx4gemm.hip -- grouped products of microscaled 4-bit matrices (include/ggemm_mx4.h).
//
// C = A B^T on the scaled matrix instructions.  v_mfma_scale_f32_32x32x64_f8f6f4: lane l holds 32 codes (one block, 16
// bytes) of row l % 32 at block l / 32 of two, and that block's scale byte, one of the four bytes of a register
// that the instruction names; products of codes are exact, sums are 32-bit.  The operands are given in the
// order B, A, so that a lane gets four neighbouring columns of one row of C.
// Rates, from registers only with random codes: 32x32x64 6.6 PFLOP/s, 16x16x128 5.8 (zeros: 9.4 and 7.1; the
// card lowers its clock under the products' power), so the tiles use the former.
// Bound: 256 x 256 tiles over a long inner dimension, the loop's cycles at the clock that the products' power leaves
// (8192 x 8192 x 16384: 917 thousand cycles, the matrix cores busy 57 % of them; 501 us, 4.4 PFLOP/s; all zeros
// the same cycles in 380 us); over a short one, also the stores of C (8192 x 8192 x 1024: 53 us), which a tile's first wait
// for its operands waits for too (one counter); few rows, the bytes of B.
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"

namespace ggemm {
namespace {

constexpr int kCus = 256;   // compute units of an MI355X

// The rows [lo, hi) of a group; g = -1: none.
struct Span {
  int g, lo, hi;
};

__device__ __forceinline__ int clamp_to(int x, int n) { return min(max(x, 0), n); }

// The block that an offset along an inner dimension of k starts at.
__device__ __forceinline__ int block_at(int x, int k) { return x >= k ? ceil_div(k, 32) : max(x, 0) / 32; }

// Tiles of the groups in order (TM rows, nt of them along n).  Every wave looks a tile's group up on its own: a lane
// has one of 64 consecutive groups, with an inclusive sum over the lanes of their tile counts.
template <int TM>
struct Groups {
  int lo, hi, own, sum, all;   // this lane's group: rows, tiles, tiles up to it; tiles of the 64
  __device__ __forceinline__ Groups(const ggemm_mx4_gemm_t& p, int g0, int nt) {
    const int lane = threadIdx.x & 63, g = min(g0 + lane, p.groups - 1);
    lo = p.offsets ? clamp_to(p.offsets[g], p.m) : 0;
    hi = p.offsets ? clamp_to(p.offsets[g + 1], p.m) : p.m;
    own = sum = g0 + lane < p.groups ? ceil_div(max(hi - lo, 0), TM) * nt : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int up = __shfl_up(sum, d);
      sum += lane >= d ? up : 0;
    }
    all = __builtin_amdgcn_readlane(sum, 63);
  }
  // The group of tile t; t becomes the number within the group.
  __device__ __forceinline__ bool find(int g0, int& t, Span& s) const {
    if (t >= all) {
      t -= all;
      return false;
    }
    const int l = __builtin_ctzll(__ballot(sum > t));
    t -= __builtin_amdgcn_readlane(sum - own, l);
    s = Span{g0 + l, __builtin_amdgcn_readlane(lo, l), __builtin_amdgcn_readlane(hi, l)};
    return true;
  }
};
// `first`: the first 64 groups, which a kernel looks up in more than once.
template <int TM>
__device__ __forceinline__ Span find_tile(const ggemm_mx4_gemm_t& p, const Groups<TM>& first, int& t, int nt) {
  Span s{-1, 0, 0};
  if (first.find(0, t, s)) return s;
  for (int g0 = 64; g0 < p.groups; g0 += 64)
    if (Groups<TM>(p, g0, nt).find(g0, t, s)) return s;
  return s;
}

// Where results go: c = alpha v + beta c, rounded once.
struct Out {
  float alpha, beta;
  int64_t ldc;
};
template <class T>
__device__ __forceinline__ void store_one(T* c, float v, const Out& o) {
  v *= o.alpha;
  if (o.beta != 0.0f) v += o.beta * (float)*c;
  *c = (T)v;
}
// N values side by side.  kStream: non-temporal stores, for a C of more than the 256 MB of the last-level cache whose rows begin at a multiple
// of 64 bytes: they leave the operands in the caches (32 groups of 2048 x 4096, 32-bit results, 1 GB, inner 32768 in
// all: 358 -> 257 us), but a smaller C is stored faster into the cache (8192 x 8192 bf16, k = 1024: 52 / 55), and a
// line stored in parts has to be read first (20993 x 4062 bf16: 72 / 109).
template <bool kStream, class T, int N>
__device__ __forceinline__ void store_run(T* c, const float (&v)[N], const Out& o) {
  Run<T, N> w;
  float u[N];
#pragma unroll
  for (int e = 0; e < N; ++e) u[e] = o.alpha * v[e];
  if (o.beta != 0.0f) {
    w = Run<T, N>::load(c);
#pragma unroll
    for (int e = 0; e < N; ++e) u[e] += o.beta * (float)w.x[e];
  }
#pragma unroll
  for (int e = 0; e < N; ++e) w.x[e] = (T)u[e];
  w.template store<kStream>(c);
}

// ---------------------------------------------------------------- tiles through LDS
// A workgroup computes a BM x BN tile with WGM x WGN waves of FM x FN blocks of 32 x 32.  The inner dimension goes
// in stages of 256 codes: 128 bytes, one memory line, of every row of A and B, from memory to LDS
// directly, into a ring of two stages.  One barrier a stage: a wave waits for its part of stage s + 1 (a
// whole stage's products old) and for its last fragments of stage s, passes the barrier, sends for stage
// s + 2 into the slot of stage s, and has half of stage s's products still to issue, which cover the
// barrier and the first reads of stage s + 1.
// Scale bytes come in windows of 32 per row (four stages), two windows in LDS: the compute unit's line
// requests bound this kernel, and 8 bytes of every row per stage took as many as the codes (256 x 256 tiles,
// 8192 x 8192 x 16384: 541 us, with windows 525).
// LDS: chunk c (16 bytes, one block's codes) of row r lies at position c ^ (r / 2) % 8 of the row, so that the 16
// rows of a group of lanes reading one chunk hit all banks.  Step t of a stage takes block t of the
// stage's first four from lanes 0-31 and block 4 + t from lanes 32-63 (any pairing will do as long as
// A and B agree), so that one scale word per lane and row block serves the four steps.
// A stage may begin before the group's first block or end past its last one (or the row's).  Those blocks get
// scale byte 0 on both sides: codes are finite, so their products are below 2^11 2^-254, and adding them
// leaves every 32-bit sum as it is.
template <int BM_, int BN_, int WGM_, int WGN_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, NW = WGM * WGN, NT = 64 * NW;
  static constexpr int FM = BM / WGM / 32, FN = BN / WGN / 32;
  static constexpr int SA = BM * 128, SB = BN * 128, STAGE = SA + SB;
  static constexpr int WIN = (BM + BN) * 32;                 // scales of a window
  static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;   // 1 KB pieces of A and B per wave
  static constexpr int NS = (BM + BN) / 32, PS = (NS + NW - 1) / NW;   // 1 KB pieces of a window, and per wave
  static constexpr int EPI = 32 * FN * 32 * 4;               // epilogue bytes per wave, in the second slot
  static constexpr int SMEM = 2 * STAGE + 2 * WIN;
  static constexpr int WAVES = 163840 / SMEM * NW / 4;       // per SIMD, as many workgroups as LDS holds
  static_assert(BM / 8 % NW == 0 && BN / 8 % NW == 0 && NW % 2 == 0, "pieces");
  static_assert(NW * EPI <= STAGE, "epilogue");
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
// 64 lanes' 16 (or 4) bytes at base + off to LDS byte address lds + 16 (4) lane.  Written as assembly so that the
// compiler does not wait for all of them before the next LDS read; the waits are stage_wait's.  s_nop 3: with the move, the five
// wait states that a base written by a vector instruction (the compiler may have kept it in a lane) needs before a memory
// instruction reads it; the compiler's own check does not see in here.
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void dma4(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
// This wave's transfers to LDS landed.
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// This wave's LDS operations done; then every wave's.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// Both.
__device__ __forceinline__ void stage_wait() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ i32x8 frag(u32x4 x) {
  return __builtin_bit_cast(i32x8, __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1));
}

// Sources of a tile's stages and scale windows: uniform bases and this lane's offsets.
template <class C>
struct Source {
  const uint8_t *a, *b, *as, *bs;
  uint32_t va[C::PA], vb[C::PB], vs[C::PS];
  int chunk, nb;   // this lane's chunk of a row, blocks of a row
  int lda_scales, ldb_scales, rows, cols;

  __device__ __forceinline__ Source(const ggemm_mx4_gemm_t& p, const uint8_t* b0, const uint8_t* bs0, int row0, int rows_,
                                    int col0, int cols_, int wave, int lane)
      : a(p.a + (int64_t)row0 * p.lda), b(b0 + (int64_t)col0 * p.ldb), as(p.a_scales + (int64_t)row0 * p.lda_scales),
        bs(bs0 + (int64_t)col0 * p.ldb_scales), nb(ceil_div(p.k, 32)), lda_scales((int)p.lda_scales),
        ldb_scales((int)p.ldb_scales), rows(rows_), cols(cols_) {
    // pieces wave, wave + NW, ... of 8 rows; NW is even, so the swizzle's upper bit is the wave's
    chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
#pragma unroll
    for (int q = 0; q < C::PA; ++q) va[q] = (uint32_t)min(8 * (wave + C::NW * q) + (lane >> 3), rows - 1) * (uint32_t)p.lda + 16 * chunk;
#pragma unroll
    for (int q = 0; q < C::PB; ++q) vb[q] = (uint32_t)min(8 * (wave + C::NW * q) + (lane >> 3), cols - 1) * (uint32_t)p.ldb + 16 * chunk;
    // windows: a piece is 32 rows (of A, then of B) of two 16-byte halves, exchanged in rows with bit 3 set
#pragma unroll
    for (int q = 0; q < C::PS; ++q) vs[q] = scale_row(32 * (wave + C::NW * q) + (lane >> 1)) + 16 * ((lane ^ (lane >> 4)) & 1);
  }
  __device__ __forceinline__ uint32_t scale_row(int r) const {
    return r < C::BM ? (uint32_t)min(r, rows - 1) * (uint32_t)lda_scales : (uint32_t)min(r - C::BM, cols - 1) * (uint32_t)ldb_scales;
  }
  // Blocks blk .. blk + 7 (blk a multiple of 4, blk < nb) into the slot at `slot`.  Chunks past the row's last block
  // are read from the stage's first.
  __device__ __forceinline__ void load(int blk, uint32_t slot, int wave) const {
    const uint32_t back = blk + chunk >= nb ? 16 * chunk : 0;
    const uint8_t *ak = a + (int64_t)16 * blk, *bk = b + (int64_t)16 * blk;
#pragma unroll
    for (int q = 0; q < C::PA; ++q) dma16(ak, va[q] - back, slot + 1024 * (wave + C::NW * q));
#pragma unroll
    for (int q = 0; q < C::PB; ++q) dma16(bk, vb[q] - back, slot + C::SA + 1024 * (wave + C::NW * q));
  }
  // The scale bytes of blocks blk .. blk + 31 (blk a multiple of 32, blk < nb).  A window that the row ends in
  // goes by words: those past the last block are read from the window's first.
  __device__ __forceinline__ void load_scales(int blk, uint32_t slot, int wave, int lane) const {
    if (blk + 32 <= nb) {
#pragma unroll
      for (int q = 0; q < C::PS; ++q) {
        const int piece = wave + C::NW * q;
        if (C::NS % C::NW == 0 || piece < C::NS) dma16((piece < C::BM / 32 ? as : bs) + blk, vs[q], slot + 1024 * piece);
      }
    } else {
#pragma unroll 1
      for (int piece = wave; piece < (C::BM + C::BN) / 8; piece += C::NW) {   // 8 rows of 8 words
        const int r = 8 * piece + (lane >> 3), w = 4 * ((lane & 7) ^ (r >> 1 & 4));
        dma4((piece < C::BM / 8 ? as : bs) + blk, scale_row(r) + (blk + w < nb ? w : 0), slot + 256 * piece);
      }
    }
  }
};

// The codes of blocks blk .. blk + 7 into the slot at offset so of the ring, and the scale window that begins in them.
template <class C>
__device__ __forceinline__ void load_stage(const Source<C>& src, uint32_t ring, int blk, int so, int wave, int lane) {
  const int win = (blk + 7) & ~31;
  if (win >= blk && win < src.nb) src.load_scales(win, ring + 2 * C::STAGE + (win >> 5 & 1) * C::WIN, wave, lane);
  src.load(blk, ring + so, wave);
}
// The first stage of blocks [b0, b1) into the first slot.
template <class C>
__device__ __forceinline__ void load_first(const Source<C>& src, uint32_t ring, int b0, int wave, int lane) {
  const int start = b0 & ~3;
  if (start & 31) src.load_scales(start & ~31, ring + 2 * C::STAGE + (start >> 5 & 1) * C::WIN, wave, lane);
  load_stage(src, ring, start, 0, wave, lane);
}

// The wave's FM x FN blocks, as C's transpose: lane l holds of block (i, j) row 32 i + l % 32 and columns
// 32 j + 8 (r / 4) + 4 (l / 32) + r % 4.  The first stage has landed (every wave's part).
template <class C>
__device__ __forceinline__ void tile_products(uint8_t* lds, const Source<C>& src, int b0, int b1, f32x16 (&acc)[C::FM][C::FN]) {
  constexpr int FM = C::FM, FN = C::FN;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % C::WGM, wn = wave / C::WGM;
  const int start = b0 & ~3, nk = ceil_div(b1 - start, 8);
  const uint32_t base = lds_addr(lds);
  const int fr = lane & 31, half = lane >> 5, x = (fr >> 1) & 7;
  const uint8_t* const pa = lds + (wm * FM * 32 + fr) * 128;
  const uint8_t* const pb = lds + C::SA + (wn * FN * 32 + fr) * 128;
  const uint8_t* const psa = lds + 2 * C::STAGE + (wm * FM * 32 + fr) * 32;
  const uint8_t* const psb = lds + 2 * C::STAGE + (C::BM + wn * FN * 32 + fr) * 32;

  u32x4 a[2][FM], b[2][FN];
  uint32_t sa[FM], sb[FN];
  auto read = [&](int s, int t, int so) {   // fragments of step t of the stage at so, into set s
    const int ch = ((4 * half + t) ^ x) * 16;
#pragma unroll
    for (int i = 0; i < FM; ++i) a[s][i] = *reinterpret_cast<const u32x4*>(pa + so + i * 4096 + ch);
#pragma unroll
    for (int j = 0; j < FN; ++j) b[s][j] = *reinterpret_cast<const u32x4*>(pb + so + j * 4096 + ch);
  };
  auto scales = [&](int kt) {   // of stage kt's four steps; blocks outside [b0, b1) get byte 0
    const int at = start + 8 * kt + 4 * half;
    const int so = (at >> 5 & 1) * C::WIN + ((at & 28) ^ (fr << 1 & 16));
    const int lo = min(max(b0 - at, 0), 4), hi = min(max(b1 - at, 0), 4);
    const uint64_t ones = 0xffffffffull;
    const uint32_t keep = lo < hi ? (uint32_t)(ones << (8 * lo)) & (uint32_t)(ones >> (32 - 8 * hi)) : 0u;
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[i] = *reinterpret_cast<const uint32_t*>(psa + so + i * 1024) & keep;
#pragma unroll
    for (int j = 0; j < FN; ++j) sb[j] = *reinterpret_cast<const uint32_t*>(psb + so + j * 1024) & keep;
  };
  auto products = [&](int s, auto t) {
    constexpr int T = decltype(t)::value;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag(b[s][j]), frag(a[s][i]), acc[i][j], 4, 4, T, (int)sb[j], T, (int)sa[i]);
  };
  // the products issued so far stay before what follows (else they would sink below the next reads and barrier)
  auto pin = [&]() {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) asm volatile("" : "+v"(acc[i][j]));
  };
  using std::integral_constant;
  if (nk > 1) load_stage(src, base, start + 8, C::STAGE, wave, lane);
  scales(0);
  read(0, 0, 0);
  int so = 0;
  for (int kt = 0; kt < nk; ++kt) {
    read(1, 1, so);
    products(0, integral_constant<int, 0>{});
    read(0, 2, so);
    products(1, integral_constant<int, 1>{});
    read(1, 3, so);
    const int sn = C::STAGE - so;
    pin();
    stage_wait();
    if (kt + 2 < nk) load_stage(src, base, start + 8 * (kt + 2), so, wave, lane);
    products(0, integral_constant<int, 2>{});
    read(0, 0, sn);   // after the last stage: what an earlier one left, not used
    products(1, integral_constant<int, 3>{});
    pin();
    scales(kt + 1);
    so = sn;
  }
}

// Blocks to C: a wave turns one row of blocks at a time through its own part of the ring's second slot (32-bit; the
// 16-byte piece q of row r lies at q ^ r % (pieces of a row), which spreads both the writes and the reads over
// the banks), then stores whole 16-byte pieces along C's rows.
// Before the first store it waits for the transfers in flight, the next tile's first stage.
template <class C, int D, bool kStream>
__device__ __forceinline__ void tile_store(uint8_t* lds, const Out& o, typename Elem<D>::T* c, int m_rem, int n_rem,
                                           const f32x16 (&acc)[C::FM][C::FN]) {
  using T = typename Elem<D>::T;
  constexpr int FM = C::FM, FN = C::FN, W = 32 * FN, Q = W / 4;    // columns, 16-byte pieces of an LDS row
  constexpr int E = 16 / (int)sizeof(T), LR = W / E, RI = 64 / LR; // elements a lane, lanes a row, rows at a time
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WGM, wn = wave / C::WGM;
  f32x4* const st = reinterpret_cast<f32x4*>(lds + C::STAGE + wave * C::EPI);
  const int r0 = wm * FM * 32, c0 = wn * W + (lane % LR) * E;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        st[(lane & 31) * Q + ((8 * j + 2 * q + (lane >> 5)) ^ (lane & (Q - 1)))] =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    if (i == 0) landed();
#pragma unroll 2
    for (int r = lane / LR; r < 32; r += RI) {
      const int row = r0 + 32 * i + r;
      float v[E];
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const f32x4 u = st[r * Q + (((lane % LR) * (E / 4) + e / 4) ^ (r & (Q - 1)))];
#pragma unroll
        for (int z = 0; z < 4; ++z) v[e + z] = u[z];
      }
      if (row >= m_rem) continue;
      T* const out = c + (int64_t)row * o.ldc + c0;
      if (c0 + E <= n_rem) {
        store_run<kStream>(out, v, o);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c0 + e < n_rem) store_one(out + e, v[e], o);
      }
    }
  }
}

// Tile t of a rows x cols arrangement of tiles, in bands of 4 rows, down each band's columns.
__device__ __forceinline__ void raster(int t, int rows, int cols, int& r, int& c) {
  const int band = t / (4 * cols), r0 = 4 * band, h = min(4, rows - r0), l = t - r0 * cols;
  r = r0 + l % h;
  c = l / h;
}

// Where a tile lies: its group, first row, the group's last row + 1, first column, blocks of the inner dimension.
struct Place {
  int g, m0, m_end, n0, b0, b1;
};
template <class C, bool kInner>
__device__ __forceinline__ Place place_of(const ggemm_mx4_gemm_t& p, const Groups<C::BM>& first, int t) {
  const int nt = ceil_div(p.n, C::BN);
  Place a{-1, 0, 0, 0, 0, ceil_div(p.k, 32)};
  int tm, tn;
  if constexpr (kInner) {
    const int mt = ceil_div(p.m, C::BM);
    a.g = t / (mt * nt);
    raster(t - a.g * mt * nt, mt, nt, tm, tn);
    a.m0 = tm * C::BM;
    a.m_end = p.m;
    if (p.offsets) {
      a.b0 = block_at(p.offsets[a.g], p.k);
      a.b1 = block_at(p.offsets[a.g + 1], p.k);
    }
  } else {
    const Span s = find_tile(p, first, t, nt);
    a.g = s.g;
    if (s.g < 0) return a;
    raster(t, ceil_div(s.hi - s.lo, C::BM), nt, tm, tn);
    a.m0 = s.lo + tm * C::BM;
    a.m_end = s.hi;
  }
  a.n0 = tn * C::BN;
  return a;
}

// The INNER form's groups by length, longest first, in runs of 64 (a lane has the rank of its group in the
// run), so that the tiles of a round are about equally long: a workgroup gets every 256th tile, with the groups as they
// come the longest ones may all fall to some.
// (32 groups of 2048 x 4096, inner 32768 in all: cut at random 326 -> 295 us, all equal 263 -> 268; of 1024 x 2048, popularities
// of 1 / sqrt(rank) in random order 84 -> 77.)
struct ByLength {
  int run = -1, rank;
  __device__ __forceinline__ int group(const ggemm_mx4_gemm_t& p, int g) {
    if (run != (g & ~63)) {
      run = g & ~63;
      const int lane = threadIdx.x & 63, own = min(run + lane, p.groups - 1);
      const int b0 = block_at(p.offsets[own], p.k), b1 = block_at(p.offsets[own + 1], p.k);
      const int key = run + lane < p.groups ? 64 * ceil_div(max(b1 - (b0 & ~3), 0), 8) + 63 - lane : -1 - lane;
      rank = 0;
#pragma unroll 8
      for (int l = 0; l < 64; ++l) rank += __builtin_amdgcn_readlane(key, l) > key;
    }
    return run + __builtin_ctzll(__ballot(rank == (g & 63)));
  }
};

// Part s of S of the blocks [b0, b1), cut at multiples of four (so that no scale word is shared).
__device__ __forceinline__ void take_part(int& b0, int& b1, int s, int S) {
  const int start = b0 & ~3, words = max(ceil_div(b1 - start, 4), 0);
  const int lo = start + 4 * (int)((int64_t)words * s / S), hi = start + 4 * (int)((int64_t)words * (s + 1) / S);
  b0 = max(b0, lo);
  b1 = min(b1, hi);
}

// Workgroup b takes tiles b, b + grid, ... of `total` (some past the last of a ragged rows form).  The next
// tile's first stage is on its way while this one's results are stored.  kSplit: blockIdx.y is one of gridDim.y parts
// of the inner dimension; its sums go to `parts`, tile after tile, for join_kernel.
template <class C, int D, bool kInner, bool kSplit, bool kStream>
__global__ void __launch_bounds__(C::NT, C::WAVES) gemm_tile_kernel(ggemm_mx4_gemm_t p, int total, float* parts) {
  __shared__ __attribute__((aligned(128))) uint8_t tile_lds[C::SMEM];
  using T = typename Elem<D>::T;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ring = lds_addr(tile_lds);
  const Groups<C::BM> first(p, 0, ceil_div(p.n, C::BN));
  const Out o{p.alpha, p.beta, p.ldc};
  int64_t it = blockIdx.x;
  int number = 0;
  ByLength by_length;
  auto next = [&]() {
    Place a{-1, 0, 0, 0, 0, 0};
    for (; a.g < 0 && it < total; it += gridDim.x) {
      number = tile_number((int)it, total);
      if constexpr (kInner && !kSplit) {
        if (p.offsets && p.groups > 1) {
          const int per = total / p.groups, g = number / per;
          number += (by_length.group(p, g) - g) * per;
        }
      }
      a = place_of<C, kInner>(p, first, number);
      if constexpr (kSplit) take_part(a.b0, a.b1, blockIdx.y, gridDim.y);
    }
    return a;
  };
  auto source = [&](const Place& a) {
    return Source<C>(p, p.b + (kInner ? 0 : a.g * p.b_stride), p.b_scales + (kInner ? 0 : a.g * p.b_scales_stride), a.m0,
                     a.m_end - a.m0, a.n0, p.n - a.n0, wave, lane);
  };
  Place cur = next();
  if (cur.g < 0) return;
  Source<C> src = source(cur);
  if (cur.b0 < cur.b1) load_first(src, ring, cur.b0, wave, lane);
  landed();
  while (true) {
    lds_barrier();
    f32x16 acc[C::FM][C::FN] = {};
    if (cur.b0 < cur.b1) tile_products<C>(tile_lds, src, cur.b0, cur.b1, acc);
    const int done = number;
    const Place nxt = next();
    if (nxt.g >= 0) {
      src = source(nxt);
      if (nxt.b0 < nxt.b1) load_first(src, ring, nxt.b0, wave, lane);
    }
    if constexpr (kSplit) {
      float* const c = parts + ((int64_t)blockIdx.y * total + done) * C::BM * C::BN;
      tile_store<C, GGEMM_F32, false>(tile_lds, Out{1.0f, 0.0f, C::BN}, c, C::BM, C::BN, acc);
    } else {
      T* const c = static_cast<T*>(p.c) + (kInner ? cur.g * p.c_stride : 0) + (int64_t)cur.m0 * p.ldc + cur.n0;
      tile_store<C, D, kStream>(tile_lds, o, c, cur.m_end - cur.m0, p.n - cur.n0, acc);
    }
    if (nxt.g < 0) return;
    cur = nxt;
  }
}

// Sums of the `splits` parts of a tile, in order: a workgroup takes 8 rows of tile blockIdx.x.
template <class C, int D, bool kInner>
__global__ void __launch_bounds__(256) join_kernel(ggemm_mx4_gemm_t p, int total, int splits, const float* __restrict__ parts) {
  using T = typename Elem<D>::T;
  const Groups<C::BM> first(p, 0, ceil_div(p.n, C::BN));
  const int t = blockIdx.x;
  const Place a = place_of<C, kInner>(p, first, t);
  if (a.g < 0) return;
  const Out o{p.alpha, p.beta, p.ldc};
  T* const c = static_cast<T*>(p.c) + (kInner ? a.g * p.c_stride : 0) + (int64_t)a.m0 * p.ldc + a.n0;
  for (int i = threadIdx.x; i < 8 * C::BN; i += 256) {
    const int row = 8 * blockIdx.y + i / C::BN, col = i % C::BN;
    if (a.m0 + row >= a.m_end || a.n0 + col >= p.n) continue;
    float v = 0.0f;
    for (int s = 0; s < splits; ++s) v += parts[((int64_t)s * total + t) * C::BM * C::BN + row * C::BN + col];
    store_one(c + (int64_t)row * p.ldc + col, v, o);
  }
}

// ---------------------------------------------------------------- few rows
// A workgroup computes 16 rows x 32 columns; its NW waves take every NW-th run of 512 codes straight from
// memory into registers and join their sums in LDS in order; the waves of a compute unit (24) cover each
// other's latency.  Products are v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds the block l / 16 of four of
// row l % 16, so that a load takes 64 bytes side by side of each of 16 rows (the 32 x 32 x 64 form takes
// 16 bytes twice of 32 rows, four times the line accesses).  A run's 16 scale bytes of a row are one load of
// every lane of the row, which picks its byte of each word.
// Bound: the bytes of B, which nobody else reads.
struct FewTile {
  static constexpr int BM = 16, BN = 32;
};
template <int D, bool kInner, int NW>
__global__ void __launch_bounds__(64 * NW, 4) gemm_few_kernel(ggemm_mx4_gemm_t p) {
  using T = typename Elem<D>::T;
  __shared__ f32x4 sums[NW][2][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4;
  const Place t = place_of<FewTile, kInner>(p, Groups<FewTile::BM>(p, 0, ceil_div(p.n, FewTile::BN)), blockIdx.x);
  if (t.g < 0) return;
  const int nb = ceil_div(p.k, 32);
  const int row = min(t.m0 + (lane & 15), t.m_end - 1);
  const int col0 = min(t.n0 + (lane & 15), p.n - 1), col1 = min(t.n0 + 16 + (lane & 15), p.n - 1);
  const uint8_t* const b = p.b + (kInner ? 0 : t.g * p.b_stride);
  const uint8_t* const bs = p.b_scales + (kInner ? 0 : t.g * p.b_scales_stride);
  const uint8_t* const codes[3] = {b + (int64_t)col0 * p.ldb, b + (int64_t)col1 * p.ldb, p.a + (int64_t)row * p.lda};
  const uint8_t* const scales[3] = {bs + (int64_t)col0 * p.ldb_scales, bs + (int64_t)col1 * p.ldb_scales,
                                    p.a_scales + (int64_t)row * p.lda_scales};
  const int start = t.b0 & ~3, runs = t.b0 < t.b1 ? ceil_div(t.b1 - start, 16) : 0;
  f32x4 acc[2] = {};
  for (int r = wave; r < runs; r += NW) {
    const int first = start + 16 * r;   // blocks past the row's last are read from the run's first
    u32x4 c[3][4], sc[3];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int at = first + 4 * s + quarter;
      const int64_t off = 16 * (int64_t)(at < nb ? at : first);
#pragma unroll
      for (int i = 0; i < 3; ++i) c[i][s] = *reinterpret_cast<const u32x4*>(codes[i] + off);
    }
    if (first + 16 <= nb) {
      struct __attribute__((packed, aligned(4))) Words { u32x4 w; };
#pragma unroll
      for (int i = 0; i < 3; ++i) sc[i] = reinterpret_cast<const Words*>(scales[i] + first)->w;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int s = 0; s < 4; ++s) sc[i][s] = *reinterpret_cast<const uint32_t*>(scales[i] + (first + 4 * s < nb ? first + 4 * s : first));
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int at = first + 4 * s + quarter;
      const uint32_t keep = at >= t.b0 && at < t.b1 ? 0xffu : 0u;   // blocks outside [b0, b1) get scale byte 0
      uint32_t sb[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) sb[i] = sc[i][s] >> (8 * quarter) & keep;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(frag(c[j][s]), frag(c[2][s]), acc[j], 4, 4, 0, (int)sb[j], 0, (int)sb[2]);
    }
  }
  sums[wave][0][lane] = acc[0];
  sums[wave][1][lane] = acc[1];
  __syncthreads();
  if (wave >= 2) return;
  f32x4 v = sums[0][wave][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) v += sums[w][wave][lane];
  // C's transpose: row lane % 16, columns 16 wave + 4 (lane / 16) + 0 .. 3
  const int i = t.m0 + (lane & 15), j = t.n0 + 16 * wave + 4 * quarter;
  if (i >= t.m_end) return;
  const Out o{p.alpha, p.beta, p.ldc};
  T* const c = static_cast<T*>(p.c) + (kInner ? t.g * p.c_stride : 0) + (int64_t)i * p.ldc + j;
  const float u[4] = {v[0], v[1], v[2], v[3]};
  if (j + 4 <= p.n) {
    store_run<false>(c, u, o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < p.n) store_one(c + e, u[e], o);
  }
}

// Sizes, leading dimensions and strides.
bool shape_ok(const ggemm_mx4_gemm_t* p) {
  if (!p || (p->form != GGEMM_MX4_ROWS && p->form != GGEMM_MX4_INNER) || p->groups < 1 ||
      p->groups > GGEMM_MX4_MAX_GROUPS || p->m < 0 || p->n < 0 || p->k < 0 || !elem_known(p->dtype))
    return false;
  if (p->m == 0 || p->n == 0) return true;
  const bool inner = p->form == GGEMM_MX4_INNER;
  if (p->ldc < p->n) return false;
  if (inner && p->groups > 1 && (p->c_stride < 0 || p->c_stride < (int64_t)(p->m - 1) * p->ldc + p->n)) return false;
  if (p->k == 0) return true;
  const int64_t nb = ceil_div(p->k, 32);
  auto operand = [&](int64_t ld, int64_t lds) { return ld % 16 == 0 && ld >= 16 * nb && lds % 4 == 0 && lds >= nb; };
  return operand(p->lda, p->lda_scales) && operand(p->ldb, p->ldb_scales) &&
         (inner || p->groups == 1 || (p->b_stride % 16 == 0 && p->b_scales_stride % 4 == 0));
}

bool gemm_ok(const ggemm_mx4_gemm_t* p) {
  if (!shape_ok(p) || (!p->offsets && p->groups != 1)) return false;
  if (p->m == 0 || p->n == 0) return true;
  if (!p->c || !aligned(p->c, elem_bytes(p->dtype)) || !aligned(p->offsets, 4)) return false;
  auto operand = [](const uint8_t* x, const uint8_t* s) { return x && s && aligned(x, 16) && aligned(s, 4); };
  return p->k == 0 || (operand(p->a, p->a_scales) && operand(p->b, p->b_scales));
}

// Row tiles of TM rows that the groups can have at most: sum ceil(m_g / TM) <= m / TM + groups with rows.  (Not by
// whether there are offsets: a workspace may be asked for before they exist.)
int64_t row_tiles(const ggemm_mx4_gemm_t& p, int tm) {
  return p.groups > 1 ? (int64_t)p.m / tm + std::min(p.groups, p.m) : ceil_div(p.m, tm);
}

using Tile256 = Tile<256, 256, 2, 4>;
using Tile128 = Tile<128, 128, 2, 2>;
using Tile32 = Tile<32, 128, 1, 4>;

constexpr int64_t kMaxLd = 1 << 23;   // leading dimensions whose 256 rows stay within a 32-bit offset

int64_t tiles_of(const ggemm_mx4_gemm_t& p, int bm, int bn) {
  return (p.form == GGEMM_MX4_INNER ? (int64_t)ceil_div(p.m, bm) * p.groups : row_tiles(p, bm)) * ceil_div(p.n, bn);
}

// How a call is computed.
struct Way {
  int tile;     // rows of a tile: 16, 32, 128 or 256
  int splits;   // parts of the inner dimension
  int64_t tiles;
};
// Rules on the sizes that the host knows (the groups' own are on the device).  Measured, us:
//   few rows or 32 x 128 tiles: by what the card holds at once.  4096 x 2048 weights, one row in each group: 1
//   group 4.2 / 6.5, 8 groups (256 tiles) 8.3 / 8.5, 16 groups 15.3 / 13.6
//   32 x 128 or 128 x 128 tiles: up to 64 rows a group on average.  64 groups of 4096 x 2048: 64 rows each 66 /
//   80, 128 rows 117 / 88
//   128 x 128 or 256 x 256 tiles (one workgroup a compute unit): where the latter make two rounds, half a tile
//   added for every group.  16 groups of n x 1024 weights: n = 2048, 8192 rows in all 18.3 / 17.7, 12288 rows 26 / 31,
//   16384 rows 35 / 30; n = 4096, 8192 rows 33 / 31, 32768 rows 119 / 99
//   parts of the inner dimension: fewer tiles than compute units, so that two tiles' worth per compute unit
//   run, each part four stages or more.  64 rows, 1024 x 16384: 27 us whole, 15.5 in parts
Way way_of(const ggemm_mx4_gemm_t& p) {
  const int64_t widest = std::max(std::max(p.lda, p.ldb), std::max(p.lda_scales, p.ldb_scales));
  const bool inner = p.form == GGEMM_MX4_INNER;
  const int64_t groups = inner ? 1 : p.groups, thin = tiles_of(p, 32, 128);
  if (widest > kMaxLd || (p.m <= 16 * groups && thin <= kCus)) return Way{16, 1, tiles_of(p, 16, 32)};
  Way w{32, 1, thin};
  if (p.m > 64 * groups) {
    const int64_t big = tiles_of(p, 256, 256), nt = ceil_div(p.n, 256);
    const int64_t likely = inner || p.groups == 1 ? big : (2 * (int64_t)p.m / 256 + p.groups) * nt / 2;
    w = likely >= 2 * kCus ? Way{256, 1, big} : Way{128, 1, tiles_of(p, 128, 128)};
  }
  const int64_t runs = ceil_div(p.k, 256) / (inner ? p.groups : 1);
  if (w.tiles < kCus) w.splits = (int)std::max<int64_t>(1, std::min(2 * kCus / w.tiles, runs / 4));
  return w;
}

template <class C, int D, bool kInner>
void launch_tiles(const ggemm_mx4_gemm_t& p, const Way& w, float* parts, hipStream_t s) {
  if (C::BM < 256 && w.splits > 1) {
    if constexpr (C::BM < 256) {
      gemm_tile_kernel<C, D, kInner, true, false><<<dim3((unsigned)w.tiles, w.splits), C::NT, 0, s>>>(p, (int)w.tiles, parts);
      join_kernel<C, D, kInner><<<dim3((unsigned)w.tiles, C::BM / 8), 256, 0, s>>>(p, (int)w.tiles, w.splits, parts);
    }
  } else {
    const int es = elem_bytes(p.dtype);
    const int64_t bytes = (int64_t)p.m * p.n * es * (kInner ? p.groups : 1);
    const bool stream = bytes > ((int64_t)256 << 20) && aligned(p.c, 64) && p.ldc * es % 64 == 0 && p.c_stride * es % 64 == 0;
    const unsigned grid = (unsigned)std::min(w.tiles, (int64_t)kCus * 4 * C::WAVES / C::NW);
    if constexpr (C::BM == 256) {   // a C of that size has so many tiles unless it is very narrow
      if (stream) {
        gemm_tile_kernel<C, D, kInner, false, true><<<grid, C::NT, 0, s>>>(p, (int)w.tiles, nullptr);
        return;
      }
    }
    gemm_tile_kernel<C, D, kInner, false, false><<<grid, C::NT, 0, s>>>(p, (int)w.tiles, nullptr);
  }
}

}  // namespace

size_t mx4_gemm_workspace(const ggemm_mx4_gemm_t* p) {
  if (!shape_ok(p) || p->m == 0 || p->n == 0) return 0;
  const Way w = way_of(*p);
  return w.splits > 1 ? (size_t)w.tiles * w.splits * w.tile * 128 * sizeof(float) : 0;
}

int mx4_gemm(const ggemm_mx4_gemm_t* p, void* ws, size_t ws_bytes, hipStream_t s) {
  if (!gemm_ok(p)) return GGEMM_ERR_INVALID;
  if (p->m == 0 || p->n == 0) return GGEMM_OK;
  const size_t need = mx4_gemm_workspace(p);
  if (ws_bytes < need) return GGEMM_ERR_WORKSPACE;
  if (need && (!ws || !aligned(ws, 16))) return GGEMM_ERR_INVALID;
  const Way w = way_of(*p);
  if (w.tiles >= (1 << 23)) return GGEMM_ERR_INVALID;   // 512 threads each: a grid of 2^32
  return launch([&] { with_elem(p->dtype, [&](auto d) {
    auto go = [&](auto inner) {
      constexpr int D = decltype(d)::value;
      constexpr bool I = decltype(inner)::value;
      float* const parts = static_cast<float*>(ws);
      if (w.tile == 256) launch_tiles<Tile256, D, I>(*p, w, parts, s);
      else if (w.tile == 128) launch_tiles<Tile128, D, I>(*p, w, parts, s);
      else if (w.tile == 32) launch_tiles<Tile32, D, I>(*p, w, parts, s);
      else if (w.tiles < kCus && p->k >= 4096) gemm_few_kernel<D, I, 16><<<(unsigned)w.tiles, 1024, 0, s>>>(*p);
      else gemm_few_kernel<D, I, 4><<<(unsigned)w.tiles, 256, 0, s>>>(*p);
    };
    if (p->form == GGEMM_MX4_INNER) go(std::true_type{});
    else go(std::false_type{});
  }); });
}

}  // namespace ggemm

extern "C" size_t ggemm_mx4_gemm_workspace(const ggemm_mx4_gemm_t* p) { return ggemm::mx4_gemm_workspace(p); }
extern "C" int ggemm_mx4_gemm(const ggemm_mx4_gemm_t* p, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  return ggemm::mx4_gemm(p, workspace, workspace_bytes, stream);
}
