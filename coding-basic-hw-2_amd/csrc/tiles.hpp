// tiles.hpp -- products of 16-bit floating point and 8-bit integers by tiles through LDS, for kernels that bring their own
// operands and epilogue.
//
// A workgroup computes a BM x BN tile with WGM x WGN waves of FM x FN blocks of 32 x 32.  The inner dimension goes in
// stages of 128 bytes of a row (64 16-bit values, 128 integers): from memory to LDS directly, into a ring of two
// stages.  One barrier a stage: a wave waits for its part of stage s + 1 (a whole stage's products old) and for its last
// fragments of stage s, passes the barrier, sends for stage s + 2 into the slot of stage s, and has half of stage
// s's products still to issue, which cover the barrier and the first reads of stage s + 1.
// v_mfma_f32_32x32x16_{bf16,f16} and v_mfma_i32_32x32x32_i8 take the same bytes: lane l holds 16 of row l % 32, from
// byte 16 (l / 32) of the step's 32.  The operands are given in the order B, A, so that a lane gets four neighbouring columns of
// one row of C.
// An operand lies in memory
//   along the inner dimension (Along): rows of the tile are rows in memory.  LDS: chunk c (16 bytes) of row r lies at
//     position c ^ (r / 2) % 8 of the row's 128 bytes, so that the 16 rows of a group of lanes reading one chunk hit
//     all banks;
//   or down it (Down, 16-bit only): rows in memory are steps of the inner dimension, 64 a stage.  LDS: the stage's
//     rows one after another, with the 64-byte units of a row turned by unit ^ f(row), f = row % 4 + 4 (row / 8 % 2);
//     ds_read_b64_tr_b16 turns four rows of 16 columns into fragments, 16 lanes at a time (lane i gives the address of
//     4 columns of row i / 4 and receives column i of the four rows): the eight rows of a wave's read differ in f, so they
//     hit all banks.
// Loads are buffer loads: what lies past an operand's last byte, or has the offset kOut, arrives as zeros.  So rows and
// steps that do not exist need no branches, and nothing that is stored next to them (NaN even) enters a sum.  The few
// bytes between an odd inner dimension and the next 16 are cleared in LDS.
#pragma once
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"

namespace ggemm {

constexpr int kCus = 256;   // compute units of an MI355X
constexpr uint32_t kOut = 0x80000000u;   // a byte offset past every operand's window
constexpr int64_t kWindow = 0x80000000ll;   // the most bytes a buffer load may reach

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct MmaBf16 {
  using Acc = f32x16;
  using Acc4 = f32x4;
  static __device__ __forceinline__ Acc4 mma16(u32x4 b, u32x4 a, Acc4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
  }
  static __device__ __forceinline__ Acc mma(u32x4 b, u32x4 a, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
  }
};
struct MmaF16 {
  using Acc = f32x16;
  using Acc4 = f32x4;
  static __device__ __forceinline__ Acc4 mma16(u32x4 b, u32x4 a, Acc4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
  }
  static __device__ __forceinline__ Acc mma(u32x4 b, u32x4 a, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
  }
};
struct MmaI8 {
  using Acc = i32x16;
  using Acc4 = i32x4;
  static __device__ __forceinline__ Acc4 mma16(u32x4 b, u32x4 a, Acc4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, b), __builtin_bit_cast(i32x4, a), c, 0, 0, 0);
  }
  static __device__ __forceinline__ Acc mma(u32x4 b, u32x4 a, Acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, b), __builtin_bit_cast(i32x4, a), c, 0, 0, 0);
  }
};
template <int D> struct MmaOf { using M = MmaBf16; };
template <> struct MmaOf<GGEMM_F16> { using M = MmaF16; };

// Rows of groups: offsets ascending from the first group's, or NULL for one group of m rows.
struct RowGroups {
  const int32_t* offsets;
  int groups, m;
  __device__ __forceinline__ int at(int g) const { return min(max(offsets[g], 0), m); }
  // the rows of a group
  __device__ __forceinline__ void span(int g, int& lo, int& hi) const {
    lo = offsets ? at(g) : 0;
    hi = offsets ? at(g + 1) : m;
  }
};
struct RowSpan {
  int g, lo, hi;   // g = -1: none
};
// Tiles of the groups in order (TM rows, nt of them along n).  Every wave looks a tile's group up on its own: a lane
// has one of 64 consecutive groups, with an inclusive sum over the lanes of their tile counts.
template <int TM>
struct GroupTiles {
  int lo, hi, own, sum, all;   // this lane's group: rows, tiles, tiles up to it; tiles of the 64
  __device__ __forceinline__ GroupTiles(const RowGroups& p, int g0, int nt) {
    const int lane = threadIdx.x & 63;
    p.span(min(g0 + lane, p.groups - 1), lo, hi);
    // A launch has fewer than 2^23 tiles, so a group may count as 2^24: offsets that are not ascending can name any rows many
    // times over, and their sums must not run over either.
    own = sum = g0 + lane < p.groups ? min(ceil_div(max(hi - lo, 0), TM), (1 << 24) / nt + 1) * nt : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int up = __shfl_up(sum, d);
      sum += lane >= d ? up : 0;
    }
    all = __builtin_amdgcn_readlane(sum, 63);
  }
  // The group of tile t; t becomes the number within the group.
  __device__ __forceinline__ bool find(int g0, int& t, RowSpan& s) const {
    if (t >= all) {
      t -= all;
      return false;
    }
    const int l = __builtin_ctzll(__ballot(sum > t));
    t -= __builtin_amdgcn_readlane(sum - own, l);
    s = RowSpan{g0 + l, __builtin_amdgcn_readlane(lo, l), __builtin_amdgcn_readlane(hi, l)};
    return true;
  }
};
// `first`: the first 64 groups, which a kernel looks up in more than once.
template <int TM>
__device__ __forceinline__ RowSpan find_group(const RowGroups& p, const GroupTiles<TM>& first, int& t, int nt) {
  RowSpan s{-1, 0, 0};
  if (first.find(0, t, s)) return s;
  for (int g0 = 64; g0 < p.groups; g0 += 64)
    if (GroupTiles<TM>(p, g0, nt).find(g0, t, s)) return s;
  return s;
}
// Row tiles of TM rows that groups can have at most: sum ceil(m_g / TM) <= m / TM + groups with rows.  (Not by whether
// there are offsets: a workspace may be asked for before they exist.)
inline int64_t row_tiles(int groups, int m, int tm) {
  return groups > 1 ? (int64_t)m / tm + std::min(groups, m) : ceil_div(m, tm);
}

// Tile t of a rows x cols arrangement of tiles, in bands of 4 rows, down each band's columns.
__device__ __forceinline__ void tile_raster(int t, int rows, int cols, int& r, int& c) {
  const int band = t / (4 * cols), r0 = 4 * band, h = min(4, rows - r0), l = t - r0 * cols;
  r = r0 + l % h;
  c = l / h;
}

template <int BM_, int BN_, int WGM_, int WGN_>
struct TileShape {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, NW = WGM * WGN, NT = 64 * NW;
  static constexpr int FM = BM / WGM / 32, FN = BN / WGN / 32;
  static constexpr int SA = BM * 128, SB = BN * 128, STAGE = SA + SB;
  static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;   // 1 KB pieces of A and B a wave brings
  static constexpr int EPI = 32 * 32 * FN * 4;               // epilogue bytes per wave, from the second slot on
  static constexpr int SMEM = STAGE + (NW * EPI > STAGE ? NW * EPI : STAGE);   // 64 x 128: 56 KB, of which 32 the epilogue's
  static constexpr int PER_CU = 163840 / SMEM;               // workgroups, as many as LDS holds
  static constexpr int WAVES = PER_CU * NW / 4;              // per SIMD
  static_assert(BM / 8 % NW == 0 && BN / 8 % NW == 0 && NW % 2 == 0, "pieces");
};

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
// 64 lanes' 16 bytes at offset off of [base, base + left) to LDS byte address lds + 16 lane, zeros past the end.  Written as
// assembly so that the compiler does not wait for all of them before the next LDS read; the waits are stage_done's.
struct Window {
  i32x4 r;
  Window() = default;
  __device__ __forceinline__ Window(const uint8_t* base, int64_t left) {
    const uint64_t b = (uint64_t)base;
    const int high = (int)(left >> 32);   // compared by halves: scalar instructions
    const uint32_t low = (uint32_t)left, n = high < 0 ? 0u : high > 0 || low > (uint32_t)kWindow ? (uint32_t)kWindow : low;
    r = i32x4{__builtin_amdgcn_readfirstlane((int)b), __builtin_amdgcn_readfirstlane((int)(b >> 32) & 0xffff),
              __builtin_amdgcn_readfirstlane((int)n), 0x00020000};
  }
  // 16 bytes to a register
  __device__ __forceinline__ u32x4 fetch(uint32_t off) const {
    const auto b = __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<void*>(((uint64_t)(uint32_t)r[1] << 32) | (uint32_t)r[0]), 0, r[2], r[3]);
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0));
  }
  __device__ __forceinline__ void send(uint32_t off, uint32_t lds) const {
    // s_nop 3: with the move, the five wait states that a scalar register written by a vector instruction (the compiler may
    // have kept one in a lane) needs before a memory instruction reads it; the compiler's own check does not see in here
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(
                     __builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(r) : "memory");
  }
};
// This wave's transfers to LDS landed.
__device__ __forceinline__ void all_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// This wave's LDS operations done; then every wave's.
__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// Both.
__device__ __forceinline__ void stage_done() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// An operand along the inner dimension: ROWS rows of the tile.  kPair: of two matrices (gate and up), whose rows alternate
// by blocks of 32, so that a wave with two blocks side by side gets both products of the same 32 columns.
template <class C, int ROWS, bool kPair = false>
struct Along {
  static constexpr int P = ROWS / 8 / C::NW;   // 1 KB pieces (8 rows) of a wave
  const uint8_t *base, *base2;
  int64_t left;
  uint32_t v[P], o[P];   // offsets of the pieces in a stage; those of the prepared one
  Window w, w2;
  int chunk, bytes;      // this lane's chunk of a row; bytes of a row
  // rows of the matrix from base (and base2) on, `pitch` and `bytes` bytes each; at(row): a row's offset, or kOut
  template <class At>
  __device__ __forceinline__ Along(const uint8_t* base_, const uint8_t* base2_, int64_t pitch, int64_t rows, int bytes_, int wave,
                                   int lane, At at)
      : base(base_), base2(base2_), left((rows - 1) * pitch + ((bytes_ + 15) & ~15)), bytes(bytes_) {
    chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);   // NW is even, so the swizzle's upper bit is the wave's
#pragma unroll
    for (int q = 0; q < P; ++q) {
      const int p = wave + C::NW * q;
      v[q] = at((kPair ? 32 * (p >> 3) + 8 * (p & 3) : 8 * p) + (lane >> 3)) + 16 * chunk;
    }
  }
  // What stage kt's loads need; from, from2: the bases.
  __device__ __forceinline__ void prepare(const uint8_t* from, const uint8_t* from2, int kt, int wave) {
    const uint32_t out = 128 * kt + 16 * chunk >= bytes ? kOut : 0u;   // v < kOut, or it is out already
#pragma unroll
    for (int q = 0; q < P; ++q) o[q] = v[q] | out;
    const int64_t at = 128 * (int64_t)kt;
    if constexpr (kPair && C::NW < 8) {   // piece p = wave + NW q: its matrix is p's bit 2, a bit of q
      w = Window(from + at, left - at);
      w2 = Window(from2 + at, left - at);
    } else {                               // p = wave + 8 q: the wave's bit 2
      w = Window((kPair && (wave >> 2 & 1) ? from2 : from) + at, left - at);
    }
  }
  __device__ __forceinline__ void prepare(int kt, int wave) { prepare(base, base2, kt, wave); }
  // Sends piece q of the prepared stage.
  __device__ __forceinline__ void send(int q, uint32_t slot, int wave) const {
    static_assert(!kPair || C::NW == 4 || C::NW == 8, "pieces of a pair");
    (kPair && C::NW < 8 && (C::NW * q >> 2 & 1) ? w2 : w).send(o[q], slot + 1024 * (wave + C::NW * q));
  }
  // Whether stage kt ends inside a chunk, and that chunk's rest to zeros.
  __device__ __forceinline__ bool ragged(int kt) const { return bytes % 16 != 0 && bytes - 128 * kt <= 128; }
  __device__ __forceinline__ void clear(int kt, uint8_t* slot) const {
    const int end = bytes - 128 * kt;
    for (int r = threadIdx.x; r < ROWS; r += C::NT) {
      uint8_t* const p = slot + 128 * r + 16 * ((end / 16) ^ (r >> 1 & 7));
      for (int b = end % 16; b < 16; ++b) p[b] = 0;
    }
  }
};
// Rows that lie one after another, the first at offset 0.
struct InOrder {
  uint32_t pitch;
  __device__ __forceinline__ uint32_t operator()(int row) const { return (uint32_t)row * pitch; }
};

// An operand down the inner dimension: COLS columns of the tile, 16-bit.
template <class C, int COLS>
struct Down {
  static constexpr int P = COLS / 8 / C::NW, LANES = COLS / 8, STEPS = 64 / LANES;   // lanes of a row, rows of a piece
  static constexpr int UNITS = COLS / 32;   // of 64 bytes in a row
  const uint8_t* base;
  int64_t stage, left;     // bytes of a stage's rows; bytes from base on
  uint32_t v[P], o[P], col;
  Window w;
  static __device__ __forceinline__ int turn(int k) { return ((k & 3) | (k >> 1 & 4)) & (UNITS - 1); }
  // step of the stage that piece q brings this lane
  static __device__ __forceinline__ int step(int q, int wave, int lane) { return (wave + C::NW * q) * STEPS + lane / LANES; }
  __device__ __forceinline__ Down(const uint8_t* base_, int64_t pitch_, int64_t depth, int cols, int wave, int lane)
      : base(base_), stage(64 * pitch_), left((depth - 1) * pitch_ + ((2 * cols + 15) & ~15)) {
    const int pos = lane % LANES;
    // a wave's pieces lie 16 steps (or a multiple) apart, which f does not see
    static_assert(C::NW * STEPS % 16 == 0, "pieces");
    col = 16 * ((((pos >> 2) ^ turn(step(0, wave, lane))) << 2) | (pos & 3));
#pragma unroll
    for (int q = 0; q < P; ++q) v[q] = (uint32_t)step(q, wave, lane) * (uint32_t)pitch_ + col;
  }
  // What stage kt's loads need; from: the base.
  __device__ __forceinline__ void prepare(const uint8_t* from, int kt) {
    w = Window(from + kt * stage, left - kt * stage);
#pragma unroll
    for (int q = 0; q < P; ++q) o[q] = v[q];
  }
  // Sends piece q of the prepared stage.
  __device__ __forceinline__ void send(int q, uint32_t slot, int wave) const { w.send(o[q], slot + 1024 * (wave + C::NW * q)); }
};

// Fragments of one operand: `blk0` the wave's first 32-row block of the tile.
template <int ROWS, int F, bool kDown>
struct Frags {
  const uint8_t* p[kDown ? F : 1];
  int x, half;
  __device__ __forceinline__ Frags(const uint8_t* lds, int blk0, int lane) {
    half = lane >> 5;
    if constexpr (kDown) {
      const int i = lane & 15, k = 8 * half + (i >> 2);
      constexpr int U = ROWS / 32;
      const int f = ((k & 3) | (k >> 1 & 4)) & (U - 1);
#pragma unroll
      for (int b = 0; b < F; ++b) p[b] = lds + k * ROWS * 2 + 64 * ((blk0 + b) ^ f) + 32 * (lane >> 4 & 1) + 8 * (i & 3);
    } else {
      const int fr = lane & 31;
      x = (fr >> 1) & 7;
      p[0] = lds + (blk0 * 32 + fr) * 128;
    }
  }
  // of step t of the stage at offset so
  __device__ __forceinline__ void read(u32x4 (&out)[F], int t, int so) const {
    if constexpr (kDown) {
      typedef __attribute__((address_space(3))) s16x4 lds4;
#pragma unroll
      for (int b = 0; b < F; ++b) {
        const uint8_t* const q = p[b] + so + 16 * t * ROWS * 2;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)q);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(q + 4 * ROWS * 2));
        const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
        out[b] = u32x4{l[0], l[1], h[0], h[1]};
      }
    } else {
      const int ch = ((2 * t + half) ^ x) * 16;
#pragma unroll
      for (int b = 0; b < F; ++b) out[b] = *reinterpret_cast<const u32x4*>(p[0] + so + b * 4096 + ch);
    }
  }
};

// Stage kt of both operands.  src.prepare(kt, wave) works out what its loads need, src.a and src.b send it.
template <class C, class S>
__device__ __forceinline__ void send_stage(S& src, int kt, uint32_t slot, int wave) {
  src.prepare(kt, wave);
#pragma unroll
  for (int q = 0; q < C::PA; ++q) src.a.send(q, slot, wave);
#pragma unroll
  for (int q = 0; q < C::PB; ++q) src.b.send(q, slot + C::SA, wave);
}

// The wave's FM x FN blocks, as C's transpose: lane l holds of block (i, j) row 32 i + l % 32 and columns
// 32 j + 8 (r / 4) + 4 (l / 32) + r % 4.  src.ragged(kt) and clear(kt, slot) as Along's.  The first stage has landed (every
// wave's part).
// Between the barrier and the next products nothing but sends is left to do, one after each product: the scalar
// work of a stage's loads comes before the barrier, under the products of the first half.  (All of it after the barrier, ahead
// of the products: 8-bit 8192^3 480 us, as it is 456.)
template <class C, class M, bool kADown, bool kBDown, class S>
__device__ __forceinline__ void tile_products(uint8_t* lds, S& src, int nk, typename M::Acc (&acc)[C::FM][C::FN]) {
  constexpr int FM = C::FM, FN = C::FN;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WGM, wn = wave / C::WGM;
  const uint32_t ring = lds_offset(lds);
  const Frags<C::BM, FM, kADown> fa(lds, wm * FM, lane);
  const Frags<C::BN, FN, kBDown> fb(lds + C::SA, wn * FN, lane);
  u32x4 a[2][FM], b[2][FN];
  auto read = [&](int s, int t, int so) {
    fa.read(a[s], t, so);
    fb.read(b[s], t, so);
  };
  auto products = [&](int s) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = M::mma(b[s][j], a[s][i], acc[i][j]);
  };
  // the products issued so far stay before what follows (else they would sink below the next reads and barrier)
  auto pin = [&]() {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) asm volatile("" : "+v"(acc[i][j]));
  };
  if (src.ragged(0)) {
    src.clear(0, lds);
    lds_done();
  }
  if (nk > 1) send_stage<C>(src, 1, ring + C::STAGE, wave);
  read(0, 0, 0);
  int so = 0;
  for (int kt = 0; kt < nk; ++kt) {
    const bool more = kt + 2 < nk;
    read(1, 1, so);
    products(0);
    read(0, 2, so);
    src.prepare(kt + 2, wave);   // past the last stage too (a branch would keep it from mixing with the products)
    products(1);
    read(1, 3, so);
    const int sn = C::STAGE - so;
    pin();
    stage_done();
    if (kt + 1 < nk && src.ragged(kt + 1)) {
      src.clear(kt + 1, lds + sn);
      lds_done();
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        acc[i][j] = M::mma(b[0][j], a[0][i], acc[i][j]);
        asm volatile("" : "+v"(acc[i][j]));
        constexpr int all = C::PA + C::PB;
        const int n = i * FN + j;
        if (more) {
#pragma unroll
          for (int q = n * all / (FM * FN); q < (n + 1) * all / (FM * FN); ++q) {
            if (q < C::PA) src.a.send(q, ring + so, wave);
            else src.b.send(q - C::PA, ring + so + C::SA, wave);
          }
        }
      }
    read(0, 0, sn);   // after the last stage: what an earlier one left, not used
    products(1);
    pin();
    so = sn;
  }
}

// Blocks to an epilogue: a wave turns one row of blocks at a time through its own part of the ring's second slot (32-bit;
// the 16-byte piece q of row r lies at q ^ r % (pieces of a row), which spreads both the writes and the reads over the
// banks), then emit(row, col, v, u, pre) gets E neighbouring columns of a row of the tile.  kPair: blocks alternate between two
// products of the same columns, v and u, and col counts one of them; else u is v.  pre is what fetch(row, col) gave: the
// loads of a row of blocks go together.
// Before the first emit the wave waits for the transfers in flight, the next tile's first stage.
// kWhole: every row and column exists; the rows of a block are unrolled, so that their loads go together.  Else one after another:
// the checks of every row unrolled make the code of a tile longer than the instruction cache (hidden gradients of 32768 rows,
// (2048, 4096): 940 us, so 849).
template <class C, int E, bool kPair, bool kWhole, class Acc, class Fetch, class Emit>
__device__ __forceinline__ void tile_emit(uint8_t* lds, const Acc (&acc)[C::FM][C::FN], Fetch fetch, Emit emit) {
  constexpr int FM = C::FM, FN = C::FN, W = 32 * FN, Q = W / 4;      // columns, 16-byte pieces of an LDS row
  constexpr int LR = (kPair ? W / 2 : W) / E, RI = 64 / LR, N = 32 / RI;   // lanes a row, rows at a time, times
  static_assert(!kPair || FN == 2, "one block of each product");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WGM, wn = wave / C::WGM;
  f32x4* const st = reinterpret_cast<f32x4*>(lds + C::STAGE + wave * C::EPI);
  const int c0 = (lane % LR) * E, row0 = wm * FM * 32 + lane / LR, col0 = wn * (kPair ? W / 2 : W) + c0;
  auto turn = [&](int i) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        st[(lane & 31) * Q + ((8 * j + 2 * q + (lane >> 5)) ^ (lane & (Q - 1)))] =
            f32x4{(float)acc[i][j][4 * q], (float)acc[i][j][4 * q + 1], (float)acc[i][j][4 * q + 2], (float)acc[i][j][4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
    if (i == 0) all_landed();
  };
  auto rows = [&](int i, int n, const auto& pre) {
    const int r = lane / LR + n * RI;
    float v[E], u[E];
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const f32x4 x = st[r * Q + (((c0 + e) / 4) ^ (r & (Q - 1)))];
      f32x4 y = x;
      if constexpr (kPair) y = st[r * Q + ((8 + (c0 + e) / 4) ^ (r & (Q - 1)))];
#pragma unroll
      for (int z = 0; z < 4; ++z) v[e + z] = x[z], u[e + z] = y[z];
    }
    emit(row0 + 32 * i + n * RI, col0, v, u, pre);
  };
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    if constexpr (kWhole) {
      decltype(fetch(0, 0)) pre[N];
#pragma unroll
      for (int n = 0; n < N; ++n) pre[n] = fetch(row0 + 32 * i + n * RI, col0);
      turn(i);
#pragma unroll
      for (int n = 0; n < N; ++n) rows(i, n, pre[n]);
    } else {
      turn(i);
#pragma unroll 1
      for (int n = 0; n < N; ++n) rows(i, n, fetch(row0 + 32 * i + n * RI, col0));
    }
    __builtin_amdgcn_wave_barrier();
  }
}
struct Nothing {};

// Workgroup b takes tiles b, b + grid, ... of `total` (some past the last of ragged groups).  The next tile's first stage
// is on its way while this one's results are stored.
// P: M (products), kADown, kBDown, kPair, E; groups(), what is looked up once for place(that, t), a tile's Place with g (-1:
// none), nk (stages) and whole; source(place) with the operands a and b, prepare(kt, wave), ragged(kt) and clear(kt, slot);
// fetch(place, row, col) and emit(place, row, col, v, u, what fetch gave); kDead: sums of rows for which names(entry(place, row)) is false
// come to emit as zeros.
template <class C, class P>
__global__ void __launch_bounds__(C::NT, C::WAVES) tile_kernel(P p, int total) {
  __shared__ __attribute__((aligned(128))) uint8_t tile_lds[C::SMEM];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ring = lds_offset(tile_lds);
  const auto first = p.template groups<C::BM, C::BN>();
  int64_t it = blockIdx.x;
  auto next = [&]() {
    typename P::Place a{-1};
    for (; a.g < 0 && it < total; it += gridDim.x) a = p.template place<C>(first, tile_number((int)it, total));
    return a;
  };
  auto cur = next();
  if (cur.g < 0) return;
  auto src = p.template source<C>(cur, wave, lane);
  if (cur.nk > 0) send_stage<C>(src, 0, ring, wave);
  all_landed();
  while (true) {
    lds_done();
    typename P::M::Acc acc[C::FM][C::FN] = {};
    if (cur.nk > 0) tile_products<C, typename P::M, P::kADown, P::kBDown>(tile_lds, src, cur.nk, acc);
    // Of row lane % 32 of each of the wave's rows of blocks, the one whose sums the lane has.  Looked at ahead of the epilogue, where a load
    // would wait for the stores before it (forward of 4096 tokens, 2 of 16 experts (1024, 2048): 176 us with a look at each row as it
    // is stored, 157 so and without any).
    int entry[C::FM];
    if constexpr (P::kDead) {
#pragma unroll
      for (int i = 0; i < C::FM; ++i) entry[i] = p.entry(cur, (wave % C::WGM * C::FM + i) * 32 + (lane & 31));
    }
    const auto nxt = next();
    if (nxt.g >= 0) {
      src = p.template source<C>(nxt, wave, lane);
      if (nxt.nk > 0) send_stage<C>(src, 0, ring, wave);
    }
    if constexpr (P::kDead) {
#pragma unroll
      for (int i = 0; i < C::FM; ++i) {
        const bool live = p.names(entry[i]);
        if (!__all(live)) {
#pragma unroll
          for (int j = 0; j < C::FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = live ? acc[i][j][e] : 0;
        }
      }
    }
    auto store = [&](auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      tile_emit<C, P::E, P::kPair, kWhole>(
          tile_lds, acc, [&](int row, int col) { return p.template fetch<kWhole>(cur, row, col); },
          [&](int row, int col, const float (&v)[P::E], const float (&u)[P::E], const auto& pre) {
            p.template emit<kWhole>(cur, row, col, v, u, pre);
          });
    };
    if (cur.whole) store(std::true_type{});
    else store(std::false_type{});
    if (nxt.g < 0) return;
    cur = nxt;
  }
}

// N values side by side, of which the first `ok` exist.
template <class T, int N>
__device__ __forceinline__ Run<T, N> run_some(const T* p, int ok) {
  if (ok >= N) return Run<T, N>::load(p);
  Run<T, N> w;
#pragma unroll
  for (int e = 0; e < N; ++e) w.x[e] = e < ok ? p[e] : (T)0.0f;
  return w;
}
template <class T, int N>
__device__ __forceinline__ void load_some(const T* p, int ok, float (&v)[N]) {
  const Run<T, N> w = run_some<T, N>(p, ok);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (float)w.x[e];
}
// stream: non-temporally, where rows are whole runs of 64 bytes (whole_runs): forward and gradients of 4096 tokens, 2 of 16 experts
// (1024, 2048), 162 -> 156 and 386 -> 367 us, the launches that read the results next included; other rows are stored faster
// by way of the caches (1237 tokens, 3 of 23 experts (1001, 1371), 73 and 76).
template <class T, int N>
__device__ __forceinline__ void store_some(T* p, int ok, const float (&v)[N], bool stream) {
  if (ok >= N) {
    Run<T, N> w;
#pragma unroll
    for (int e = 0; e < N; ++e) w.x[e] = (T)v[e];
    if (stream) {
      asm volatile("");   // else the compiler makes one ordinary store of both
      w.template store<true>(p);
      asm volatile("");
    } else {
      w.template store<false>(p);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < ok) p[e] = (T)v[e];
  }
}
inline bool whole_runs(const void* p, int64_t pitch_bytes) { return aligned(p, 64) && pitch_bytes % 64 == 0; }

// Few rows: a workgroup computes 16 rows x 32 columns (kPair: 16 columns of both products); its 4 waves take every fourth
// run of 256 bytes of the inner dimension straight from memory into registers and join their sums in LDS in order.
// Products are 16 x 16: lane l holds 16 bytes of row l % 16 from byte 16 (l / 16) of 64, so that a load takes 64 bytes side
// by side of each of 16 rows, and the four loads of a run whole lines.
// Bound: the bytes of B, which nobody else reads: 134 MB of 8 experts' weights (2048 x 4096, 16-bit) 29 us, 4.6 TB/s.  8 or 16
// waves: equal where there are fewer workgroups than compute units, up to twice as long (64 experts); two runs
// on the way: 5 to 30 % slower; room for 6 or 8 waves a SIMD: 40 to 90 % slower (fewer loads of a wave at once);
// non-temporal loads: equal to 30 % slower.
struct FewShape {
  static constexpr int BM = 16, BN = 32;
};
// Where a lane's operands are: rows of A and of the two blocks of B, as offsets in windows.
struct FewRows {
  const uint8_t *a, *b[2];
  int64_t a_left, b_left[2];
  uint32_t va, vb[2];
  int bytes;   // of a row
};
template <class P>
__global__ void __launch_bounds__(256, 4) few_kernel(P p) {
  using Acc4 = typename P::M::Acc4;
  constexpr int NW = 4;
  __shared__ Acc4 sums[NW][2][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4;
  const auto c = p.template place<FewShape>(p.template groups<FewShape::BM, FewShape::BN>(), blockIdx.x);
  if (c.g < 0) return;
  const FewRows f = p.few(c, lane & 15);
  int mine;
  if constexpr (P::kDead) mine = p.entry(c, lane & 15);
  Acc4 acc[2] = {};
  const int runs = ceil_div(f.bytes, 256);
  for (int r = wave; r < runs; r += NW) {
    const int64_t at = 256 * (int64_t)r;
    u32x4 x[3][4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t off = 64 * s + 16 * quarter;
      const uint32_t out = at + off >= f.bytes ? kOut : 0u;
      x[0][s] = Window(f.a + at, f.a_left - at).fetch((f.va + off) | out);
#pragma unroll
      for (int j = 0; j < 2; ++j) x[1 + j][s] = Window(f.b[j] + at, f.b_left[j] - at).fetch((f.vb[j] + off) | out);
    }
    if (f.bytes % 16 != 0 && r + 1 == runs) {   // what lies between the row's end and the next 16 bytes
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int have = f.bytes - (int)at - 64 * s - 16 * quarter;   // bytes of this lane's that exist
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int n = have - 4 * w;
            x[i][s][w] &= n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
          }
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[j] = P::M::mma16(x[1 + j][s], x[0][s], acc[j]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) sums[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave >= (P::kPair ? 1 : 2)) return;
  // C's transpose: row lane % 16, columns 4 (lane / 16) + 0 .. 3 of a block
  Acc4 s = sums[0][P::kPair ? 0 : wave][lane], t = sums[0][1][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    s += sums[w][P::kPair ? 0 : wave][lane];
    if constexpr (P::kPair) t += sums[w][1][lane];
  }
  float v[4] = {(float)s[0], (float)s[1], (float)s[2], (float)s[3]};
  float u[4] = {(float)t[0], (float)t[1], (float)t[2], (float)t[3]};
  if constexpr (P::kDead) {
    const bool live = p.names(mine);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = live ? v[e] : 0.0f, u[e] = live ? u[e] : 0.0f;
  }
  p.template emit<false>(c, lane & 15, (P::kPair ? 0 : 16 * wave) + 4 * quarter, v, u, Nothing{});
}

using Tile256 = TileShape<256, 256, 2, 4>;
using Tile128 = TileShape<128, 128, 2, 2>;
using Tile64 = TileShape<64, 128, 2, 2>;
template <class C, class P>
void run_tiles(const P& p, int64_t tiles, hipStream_t s) {
  tile_kernel<C, P><<<(unsigned)std::min(tiles, (int64_t)kCus * C::PER_CU), C::NT, 0, s>>>(p, (int)tiles);
}

// Which kernel computes rows of groups (m in all) times n columns: rows of its tile, 16 for the few rows'.  width: columns of a
// tile of 128 (64 where they are two products').  The host does not know the groups' own rows: half a tile more for each.
// Times of one round of workgroups, all compute units filled, to those of a half-filled one, 8-bit products, n = 4096, k =
// 4096, us: 64 x 128 tiles (two a compute unit) 26, 24; 128 x 128 (two) 40, 29; 256 x 256 (one) 64, 52; the same
// ratios at k = 2048 and 1024.  So the tile with the least rounds times cost is taken; at 2048 rows 52, 42, 54 us, at 3001 78,
// 65, 59, at 4096 101, 79, 67.
// 16-bit products by the same costs: of 48 (twelve blocks from 300 to 65536 rows, forward with gate and up kept, and backward) in all
// three shapes, the one taken is the fastest or within 2 % of it in 42.  The others, 5 to 20 % slower, store three matrices after a short
// inner dimension, which two workgroups on a compute unit do in turns: gate and up of 4096 tokens, 2 of 16 experts
// (1024, 2048), 106 us by 256 x 256, 91 by 128 x 128; hidden gradients of 32768 rows, 8 groups (1024, 1024), 172 and 147.
// Few rows: up to two workgroups a compute unit (n = k = 4096: 64 rows 15.1, by tiles 15.9; 128 rows 25 and 22), up to four
// if groups have 16 rows at most on average, so that nobody else reads their weights (32 groups, 1024 x 1024: 7.6 and 8.7; 8
// experts' 16-bit weights of 4096 x 2048 twice, 8 workgroups a compute unit: 57 and 52).
inline int rows_tile(int groups, int64_t m, int64_t n, int width, bool may_be_few) {
  const int64_t g = std::min<int64_t>(groups, m);
  auto tiles = [&](int bm, int cols) { return (m / bm + (groups > 1 ? (g + 1) / 2 : m % bm != 0)) * ((n + cols - 1) / cols); };
  const bool one = m <= 16 * (int64_t)groups;
  const int64_t few = (one ? g : groups > 1 ? m / 16 + g : (m + 15) / 16) * ((n + width / 4 - 1) / (width / 4));
  if (may_be_few && few <= (one ? 4 : 2) * kCus) return 16;
  auto cost = [](int64_t t, int64_t slots, int full, int half) {
    const int64_t rest = t % slots, over = rest - slots / 2;
    return t / slots * full + (rest == 0 ? 0 : half) + (over > 0 ? (full - half) * over / (slots / 2) : 0);
  };
  const int64_t c64 = cost(tiles(64, width), 2 * kCus, 26, 24), c128 = cost(tiles(128, width), 2 * kCus, 40, 29);
  const int64_t c256 = cost(tiles(256, 2 * width), kCus, 64, 52);
  return c256 <= std::min(c64, c128) ? 256 : c128 <= c64 ? 128 : 64;
}

}  // namespace ggemm
