// route.hip -- the router of a mixture-of-experts layer (include/ggemm_route.h).
//
// A token's logits lie in L lanes of one wave, V experts to a lane (L V >= experts, L a power of two, 64 / L tokens
// a wave), in registers from the load to the last use: in pieces of up to 16 bytes, piece c of lane l at piece
// c L + l of the row, so that the lanes of a load or store lie side by side.  Selection works on
// integer keys that order like the logits (NaN highest, barred experts 0): per place a maximum over the
// lane's keys and then over the L lanes.  16-bit logits have the expert's number, inverted, in the key's low
// half, so that a key is unique and tells the expert to all lanes, and the next place is the largest of
// key - best mod 2^32 (a key below `best` differs by 2^32 - best or more, one above by less): nothing is struck
// out.  32-bit logits take a second reduction, the least expert that holds the maximum, which is struck out.
// Softmax is the usual exp2((x - max) log2 e) over its sum, the maximum being the first choice; its sums are 32-bit.
// Counting: a workgroup takes `span` consecutive tokens.  One bit per (expert, token) in LDS gives each pair
// its rank among the workgroup's tokens by counting bits (no atomic whose order matters), and the
// expert's count.  A second launch turns the workgroups' counts into starting ranks and sums their partial
// softmax sums in a fixed order; a third one writes rows, order and loss, and does the second one's work too
// while the tables are small.  A call of one workgroup does all of it in the first launch.
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"
#include "ggemm_route.h"

namespace ggemm {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896341f;

// Workspace: per workgroup of the first launch and expert the count (then the starting rank) and the
// softmax sum, and per workgroup the tokens used.
struct RouteWs {
  int* hist;     // groups x experts
  float* psum;   // groups x experts
  int* used;     // groups
};

constexpr int kFewCounts = 8192;   // entries of the count table up to which there is no second launch
struct Shape {
  int span, groups;
};
// GGEMM_ROUTE_MAX_TOKENS keeps a token's number plus a workgroup's tokens within 31 bits, and the grids (two threads
// a token at most, where there are many) within 2^32.
// Tokens a workgroup takes (a multiple of 32: whole words of the bit table).  Few tokens are spread over
// the compute units, many take longer spans, which makes the tables of the second launch shorter (16384 x 128:
// 16.5 us with 32, 18 with 64; 32768 x 64: 20.4 and 19.4; 131072 x 256: 78, 68, and 63 with 128).
Shape shape_of(int tokens) {
  const int span = tokens <= 64 ? 64 : tokens <= 16384 ? 32 : tokens <= 65536 ? 64 : 128;
  return Shape{span, tokens > 0 ? ceil_div(tokens, span) : 1};
}

RouteWs carve(void* ws, const Shape& sh, int experts) {
  char* p = static_cast<char*>(ws);
  const size_t table = align_up((size_t)sh.groups * experts * 4, 16);
  return RouteWs{reinterpret_cast<int*>(p), reinterpret_cast<float*>(p + table), reinterpret_cast<int*>(p + 2 * table)};
}

// Keys that order like the logits: 0 for -inf, all ones for NaN, -0 as +0.
__device__ __forceinline__ uint32_t key32(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  if (x != x) return 0xffffffffu;
  if (b == 0xff800000u) return 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key32(uint32_t k) {
  return k == 0xffffffffu ? __uint_as_float(0x7fc00000u) : __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// Two 16-bit logits a word: sign and magnitude to an unsigned order with -0 = +0, then down by what -inf got.  A
// NaN of either sign has to be put right after.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short i16x2 __attribute__((ext_vector_type(2)));
template <int D>
struct Half {
  static constexpr uint32_t kInf = D == GGEMM_BF16 ? 0x7f80u : 0x7c00u, kLow = 0x7fffu - kInf + 1;
};
template <int D>
__device__ __forceinline__ uint32_t order16(uint32_t w) {
  const i16x2 s = __builtin_bit_cast(i16x2, w) >> (short)15;
  const uint32_t o = w ^ (__builtin_bit_cast(uint32_t, s) | 0x80008000u);
  const u16x2 up = __builtin_bit_cast(u16x2, o) - __builtin_bit_cast(u16x2, s);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(up, u16x2{Half<D>::kLow, Half<D>::kLow}));
}
template <int D>
__device__ __forceinline__ float of_order16(uint32_t k) {
  const uint32_t o = k + Half<D>::kLow;
  const unsigned short b = (unsigned short)(o >= 0x8000u ? o ^ 0x8000u : ~(o - 1u));
  return k == 0xffffu ? __uint_as_float(0x7fc00000u) : (float)__builtin_bit_cast(typename Elem<D>::T, b);
}

// Reductions over the L lanes of a token; every lane gets the result.  Up to 16 lanes the exchanges are part of the
// vector instructions: neighbours, pairs, then (quads being alike) mirrored within 8 and 16.
template <int CTRL, class T>
__device__ __forceinline__ T other(T x) {
  return __builtin_bit_cast(T, dpp<CTRL>(__builtin_bit_cast(uint32_t, x)));
}
template <int L, class T, class F>
__device__ __forceinline__ T over_lanes(T x, F&& f) {
  x = f(x, other<kDppXor1>(x));
  x = f(x, other<kDppXor2>(x));
  x = f(x, other<kDppHalfMirror>(x));
  if constexpr (L >= 16) x = f(x, other<kDppMirror>(x));
#pragma unroll
  for (int d = 16; d < L; d *= 2) x = f(x, __shfl_xor(x, d));
  return x;
}
template <int L>
__device__ __forceinline__ float sum_lanes(float x) {
  return over_lanes<L>(x, [](float a, float b) { return a + b; });
}
template <int L>
__device__ __forceinline__ uint32_t max_lanes(uint32_t x) {
  return over_lanes<L>(x, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int L>
__device__ __forceinline__ uint32_t min_lanes(uint32_t x) {
  return over_lanes<L>(x, [](uint32_t a, uint32_t b) { return min(a, b); });
}

// A lane's V values in pieces of N side by side, at most 16 bytes.
template <int D, int V>
struct Piece {
  using T = typename Elem<D>::T;
  static constexpr int N = V * (int)sizeof(T) >= 16 ? 16 / (int)sizeof(T) : V;
  using Type = Run<T, N>;
  // the expert of a lane's value v, less that of its value 0; and that one
  template <int L>
  static __device__ __forceinline__ constexpr int step(int v) { return v / N * L * N + v % N; }
  static __device__ __forceinline__ int first(int lane) { return lane * N; }
};
// The lane's V logits of token t (from expert e0 on; -inf past the last expert), as they lie in memory: a wave has the
// next tokens' on the way while it works on these (131072 x 256 bf16: gradient 48 -> 44 us).  Those of a token
// that is left out are read and not used.
template <int D, int L, int V>
struct Logits {
  using P = Piece<D, V>;
  typename P::Type w[V / P::N];
  unsigned char mask;
  __device__ __forceinline__ void load(const ggemm_router_t& r, int t, int t1, int e0) {
    using T = typename P::T;
    if (t >= t1) return;
    mask = r.mask ? r.mask[t] : 1;
    const T* p = static_cast<const T*>(r.logits) + (int64_t)t * r.ld + e0;
#pragma unroll
    for (int i = 0; i < V / P::N; ++i) {
      constexpr int N = P::N;
      const int at = i * L * N;
      if (e0 + at + N <= r.experts) {
        w[i] = P::Type::load(p + at);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) w[i].x[j] = e0 + at + j < r.experts ? p[at + j] : (T)-__builtin_inff();
      }
    }
  }
  __device__ __forceinline__ bool on(int t, int t1) const { return t < t1 && mask; }   // the token takes part
  __device__ __forceinline__ typename P::T at(int v) const { return w[v / P::N].x[v % P::N]; }
};
template <int D, int L, int V>
__device__ __forceinline__ void store_gradient(typename Elem<D>::T* p, int e0, int experts, const float (&g)[V]) {
  using P = Piece<D, V>;
  constexpr int N = P::N;
#pragma unroll
  for (int i = 0; i < V / N; ++i) {
    const int at = e0 + i * L * N;
    typename P::Type w;
#pragma unroll
    for (int j = 0; j < N; ++j) w.x[j] = (typename P::T)g[i * N + j];
    if (at + N <= experts) {
      w.template store<true>(p + at);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (at + j < experts) p[at + j] = w.x[j];
    }
  }
}

// exp(x - m).  The difference first: it is exact for logits near the maximum, however large they are.
__device__ __forceinline__ float exp_below(float x, float m) { return __builtin_amdgcn_exp2f((x - m) * kLog2e); }
// p[v] = exp(x[v] - max) for a token's lanes, and the reciprocal of the sum.  m: the largest logit;
// a logit of -inf gives 0 unless m is -inf too, where nothing uses p.
// (One fma of x log2 e and -m log2 e was no faster, and its error grows with m.)
template <int L, int V>
__device__ __forceinline__ float exps(const float (&x)[V], float m, float (&p)[V]) {
  float sum = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] = exp_below(x[v], m);
#pragma unroll
  for (int v = 0; v < V; ++v) sum += p[v];
  return 1.0f / sum_lanes<L>(sum);
}

// Rows of order that belong to no pair: expert e's padding, and what follows the last expert.  64-bit: the rows and the
// lanes of a large grid (twice the tokens) together pass 2^31.
__device__ __forceinline__ void pad_order(const ggemm_router_t& r, int from, int to, int64_t lane, int64_t lanes) {
  for (int64_t i = from + lane; i < to; i += lanes) r.order[i] = -1;
}

// The balance loss from counts, probs and the tokens used: one wave, fixed order.
__device__ __forceinline__ void write_loss(const ggemm_router_t& r, const int* counts, const float* probs, int used) {
  const int lane = threadIdx.x & 63;
  float s = 0.0f;
  for (int e = lane; e < r.experts; e += 64) s += (float)counts[e] * probs[e];
  s = sum_lanes<64>(s);
  if (lane == 0) r.loss[0] = used ? s * (r.balance_coef * (float)r.experts / ((float)r.topk * (float)used)) : 0.0f;
}

// Exclusive sums over experts of the counts rounded up to row_align, into off[0 .. experts]; called by
// the whole workgroup (its first kThreads threads, 4 experts each, do it), ends with a barrier.
__device__ __forceinline__ void scan_offsets(const int* counts, int experts, int align, int* off, int* tmp) {
  static_assert(GGEMM_ROUTE_MAX_EXPERTS == 4 * kThreads, "experts a thread");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int c[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = 4 * tid + i;
    c[i] = e < experts ? (counts[e] + align - 1) & -align : 0;
    sum += c[i];
  }
  int inc = sum;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int up = __shfl_up(inc, d);
    inc += lane >= d ? up : 0;
  }
  if (lane == 63 && tid < kThreads) tmp[wave] = inc;
  __syncthreads();
  if (tid < kThreads) {
    int at = inc - sum;
    for (int w = 0; w < wave; ++w) at += tmp[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (4 * tid + i <= experts) off[4 * tid + i] = at;
      at += c[i];
    }
    if (tid == kThreads - 1 && experts == 4 * kThreads) off[experts] = at;
  }
  __syncthreads();
}

// First launch: choices, gates, ranks within the workgroup's tokens (into pos), counts and softmax sums
// per workgroup.  kOne: the only workgroup, which finishes the call.
// (kOne: 16 waves, as long as their sums fit, for the latency of one call)
__host__ __device__ constexpr int first_threads(int experts, bool one) { return one && experts <= 256 ? 1024 : kThreads; }
template <int D, int L, int V, bool kOne>
__global__ void __launch_bounds__(first_threads(L * V, kOne)) route_kernel(ggemm_router_t r, RouteWs ws, int span) {
  using P = Piece<D, V>;
  constexpr int NT = first_threads(L * V, kOne), NW = NT / 64;
  constexpr int kRows = 64 / L, kPar = NW * kRows;   // tokens a wave and a workgroup hold at a time
  extern __shared__ uint32_t lds[];
  const int words = span / 32, E = r.experts, K = r.topk;
  uint32_t* bits = lds;                                        // E x words
  float* part = reinterpret_cast<float*>(lds + E * words);     // NW x (L V): the waves' softmax sums
  __shared__ int s_used[NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = lane & (L - 1), slot = wave * kRows + lane / L, e0 = P::first(sub);
  const int t0 = blockIdx.x * span, t1 = min(t0 + span, r.tokens);
  for (int i = tid; i < E * words; i += NT) bits[i] = 0;
  __syncthreads();
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  int used = 0;
  Logits<D, L, V> ahead;
  ahead.load(r, t0 + slot, t1, e0);
  for (int tb = t0; tb < t1; tb += kPar) {
    const int t = tb + slot;
    const bool in = t < t1;
    const bool on = ahead.on(t, t1);
    float x[V], p[V];
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = (float)ahead.at(v);
    // 16-bit keys: order, then a number that falls with the expert's: within the lane here, the lane's later
    constexpr uint32_t kIn = P::template step<L>(V - 1);
    const uint32_t lane_part = 0xffffu - e0 - kIn;
    if constexpr (D == GGEMM_F32) {
#pragma unroll
      for (int v = 0; v < V; ++v) key[v] = key32(x[v]);
    } else {
      typedef typename Elem<D>::T pair __attribute__((ext_vector_type(2)));
      uint32_t worst = 0;   // the largest magnitudes: a NaN among them?
#pragma unroll
      for (int v = 0; v < V; v += 2) {
        const uint32_t w = __builtin_bit_cast(uint32_t, pair{ahead.at(v), ahead.at(v + 1 < V ? v + 1 : v)});
        worst = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, worst), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
        const uint32_t o = order16<D>(w);
        key[v] = o << 16 | (kIn - P::template step<L>(v));
        if (v + 1 < V) key[v + 1] = (o & 0xffff0000u) | (kIn - P::template step<L>(v + 1));
      }
      if (__ballot(max(worst & 0xffffu, worst >> 16) > Half<D>::kInf)) {
        asm volatile("");   // a branch, not a select per value
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = x[v] != x[v] ? key[v] | 0xffff0000u : key[v];
      }
    }
    ahead.load(r, t + kPar, t1, e0);
    // the largest key of the token below the last one taken (32-bit: of those not struck out), and its expert
    uint32_t best = 0;
    int expert = 0;
    auto take = [&]() {
      if constexpr (D == GGEMM_F32) {
        uint32_t top = key[0];
#pragma unroll
        for (int v = 1; v < V; ++v) top = max(top, key[v]);
        best = max_lanes<L>(top);
        uint32_t e = 0xffffffffu;
#pragma unroll
        for (int v = V - 1; v >= 0; --v) e = key[v] == best ? e0 + P::template step<L>(v) : e;
        expert = (int)min_lanes<L>(e);
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = expert == e0 + P::template step<L>(v) ? 0u : key[v];
      } else {
        const uint32_t from = best - lane_part;
        uint32_t top = key[0] - from;
#pragma unroll
        for (int v = 1; v < V; ++v) top = max(top, key[v] - from);
        best += max_lanes<L>(top);
      }
    };
    auto logit_of = [&](uint32_t k) {
      if constexpr (D == GGEMM_F32) return of_key32(k);
      else return of_order16<D>(k >> 16);
    };
    auto expert_of = [&](uint32_t k, int e) { return D == GGEMM_F32 ? e : 0xffff - (int)(k & 0xffffu); };
    auto any = [&](uint32_t k) { return D == GGEMM_F32 ? k != 0 : k >> 16 != 0; };   // not a barred expert's
    take();
    const float m = logit_of(best);
    const bool live = on && any(best);
    const float inv = exps<L, V>(x, m, p);
    float chosen = 0.0f;
    for (int j0 = 0; j0 < K; j0 += L) {   // lane `sub` keeps place j0 + sub
      uint32_t mine = best;
      int mine_e = expert;
      const int n = min(L, K - j0);
      for (int j = j0 ? 0 : 1; j < n; ++j) {
        take();
        mine = j == sub ? best : mine;
        if constexpr (D == GGEMM_F32) mine_e = j == sub ? expert : mine_e;
      }
      const bool have = live && sub < n && any(mine);
      const int id = have ? expert_of(mine, mine_e) : -1;
      float g = have ? exp_below(logit_of(mine), m) * inv : 0.0f;
      chosen += sum_lanes<L>(g);
      if (r.renormalize && K <= L && have) g = g / chosen;
      if (in && sub < n) {
        r.ids[(int64_t)t * K + j0 + sub] = id;
        r.gates[(int64_t)t * K + j0 + sub] = g;
        if (have) atomicOr(&bits[id * words + ((t - t0) >> 5)], 1u << ((t - t0) & 31));
      }
    }
    if (live) {
      used += sub == 0;
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += p[v] * inv;
      if (r.renormalize && K > L) {   // the sum came after the first places were stored, by the same lanes
        for (int64_t i = (int64_t)t * K + sub; i < (int64_t)(t + 1) * K; i += L)
          if (r.ids[i] >= 0) r.gates[i] = r.gates[i] / chosen;
      }
    }
  }
  // softmax sums: over the tokens of a wave, then over the waves
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int d = L; d < 64; d *= 2) acc[v] += __shfl_xor(acc[v], d);
    if (lane < L) part[wave * L * V + e0 + P::template step<L>(v)] = acc[v];
  }
  used = over_lanes<64>(used, [](int a, int b) { return a + b; });
  if (lane == 0) s_used[wave] = used;
  __syncthreads();
  used = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) used += s_used[w];
  // ranks, counts
  for (int i = tid; i < (t1 - t0) * K; i += NT) {
    const int64_t at = (int64_t)t0 * K + i;
    const int e = r.ids[at], t = i / K;
    int rank = -1;
    if (e >= 0) {
      rank = __popc(bits[e * words + (t >> 5)] & ((1u << (t & 31)) - 1u));
      for (int w = 0; w < t >> 5; ++w) rank += __popc(bits[e * words + w]);
    }
    r.pos[at] = rank;
  }
  __shared__ int s_off[kOne ? GGEMM_ROUTE_MAX_EXPERTS + 1 : 1], s_tmp[4];
  for (int e = tid; e < E; e += NT) {
    int c = 0;
    for (int w = 0; w < words; ++w) c += __popc(bits[e * words + w]);
    float ps = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) ps += part[w * L * V + e];
    if constexpr (kOne) {
      r.counts[e] = c;
      r.probs[e] = used ? ps / (float)used : 0.0f;
    } else {
      ws.hist[(int64_t)blockIdx.x * E + e] = c;
      ws.psum[(int64_t)blockIdx.x * E + e] = ps;
    }
  }
  if constexpr (!kOne) {
    if (tid == 0) ws.used[blockIdx.x] = used;
  } else {
    __syncthreads();
    scan_offsets(r.counts, E, r.row_align, s_off, s_tmp);
    for (int e = tid; e <= E; e += NT) r.offsets[e] = s_off[e];
    for (int i = tid; i < r.tokens * K; i += NT) {
      const int e = r.ids[i];
      if (e >= 0) {
        const int row = s_off[e] + r.pos[i];
        r.pos[i] = row;
        if (row < r.max_rows) r.order[row] = i / K;
      }
    }
    for (int e = tid; e < E; e += NT)
      if (r.row_align > 1) pad_order(r, s_off[e] + r.counts[e], s_off[e + 1], 0, 1);
    pad_order(r, s_off[E], r.max_rows, tid, NT);
    if (tid == 0) r.used[0] = used;
    if (wave == 0) write_loss(r, r.counts, r.probs, used);
  }
}

// Second launch: a workgroup per 16 experts, 64 threads along the workgroups of the first launch each
// taking a run of them: sums per run, then starting ranks.
constexpr int kRuns = 64;
__global__ void __launch_bounds__(16 * kRuns) route_scan_kernel(ggemm_router_t r, RouteWs ws, int groups) {
  __shared__ int s_cnt[kRuns][17], s_use[16];
  __shared__ float s_p[kRuns][17];
  const int i = threadIdx.x & 15, c = threadIdx.x >> 4, e = blockIdx.x * 16 + i, E = r.experts;
  const int run = ceil_div(groups, kRuns), g0 = min(c * run, groups), g1 = min(g0 + run, groups);
  int cnt = 0;
  float ps = 0.0f;
  if (e < E) {
#pragma unroll 8
    for (int g = g0; g < g1; ++g) {
      cnt += ws.hist[(int64_t)g * E + e];
      ps += ws.psum[(int64_t)g * E + e];
    }
  }
  s_cnt[c][i] = cnt;
  s_p[c][i] = ps;
  int use = 0;
  for (int g = threadIdx.x; g < groups; g += 16 * kRuns) use += ws.used[g];
  use = over_lanes<64>(use, [](int a, int b) { return a + b; });
  if ((threadIdx.x & 63) == 0) s_use[threadIdx.x >> 6] = use;
  __syncthreads();
  use = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) use += s_use[w];
  int at = 0;
#pragma unroll 8
  for (int q = 0; q < c; ++q) at += s_cnt[q][i];
  if (e < E) {
    if (c == kRuns - 1) r.counts[e] = at + cnt;
    if (c == 0) {
      float sum = 0.0f;
#pragma unroll 8
      for (int q = 0; q < kRuns; ++q) sum += s_p[q][i];
      r.probs[e] = use ? sum / (float)use : 0.0f;
    }
#pragma unroll 8
    for (int g = g0; g < g1; ++g) {
      int* h = ws.hist + (int64_t)g * E + e;
      const int n = *h;
      *h = at;
      at += n;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) r.used[0] = use;
}

// Third launch: rows of the pairs, order, padding, loss.  Workgroup b takes the pairs of workgroup b of
// the first launch.  kScan: there was no second launch; every workgroup sums the tables for itself (experts <=
// kThreads), which is faster than a launch while the tables are small (4096 x 16: 9.4 us for the call and 11;
// 4096 x 256: 24 and 17.5).
template <bool kScan>
__global__ void __launch_bounds__(kThreads) route_place_kernel(ggemm_router_t r, RouteWs ws, int span) {
  __shared__ int s_off[GGEMM_ROUTE_MAX_EXPERTS + 1], s_tmp[4];
  __shared__ int s_cnt[kThreads], s_rank[kThreads];
  __shared__ float s_p[kThreads];
  const int tid = threadIdx.x, E = r.experts, K = r.topk;
  const int* counts = r.counts;
  const int* rank = ws.hist + (int64_t)blockIdx.x * E;
  const float* probs = r.probs;
  int used = 0;
  if constexpr (kScan) {
    int lanes = 1;   // threads along the experts, the others along the workgroups of the first launch
    while (lanes < E) lanes *= 2;
    const int e = tid & (lanes - 1), c = tid / lanes, runs = kThreads / lanes, groups = gridDim.x;
    int cnt = 0, before = 0;
    float ps = 0.0f;
    if (e < E) {
#pragma unroll 4
      for (int g = c; g < groups; g += runs) {
        const int n = ws.hist[(int64_t)g * E + e];
        cnt += n;
        before += g < (int)blockIdx.x ? n : 0;
        ps += ws.psum[(int64_t)g * E + e];
      }
    }
    for (int g = tid; g < groups; g += kThreads) used += ws.used[g];
    used = over_lanes<64>(used, [](int a, int b) { return a + b; });
    if ((tid & 63) == 0) s_tmp[tid >> 6] = used;
    s_cnt[tid] = cnt;
    s_rank[tid] = before;
    s_p[tid] = ps;
    __syncthreads();
    used = s_tmp[0] + s_tmp[1] + s_tmp[2] + s_tmp[3];
    if (tid < lanes) {
      for (int q = 1; q < runs; ++q) {
        cnt += s_cnt[q * lanes + tid];
        before += s_rank[q * lanes + tid];
        ps += s_p[q * lanes + tid];
      }
      s_cnt[tid] = cnt;
      s_rank[tid] = before;
      s_p[tid] = used ? ps / (float)used : 0.0f;
    }
    __syncthreads();
    counts = s_cnt;
    rank = s_rank;
    probs = s_p;
  }
  scan_offsets(counts, E, r.row_align, s_off, s_tmp);
  const int t0 = blockIdx.x * span, t1 = min(t0 + span, r.tokens);
  for (int i = tid; i < (t1 - t0) * K; i += kThreads) {
    const int64_t at = (int64_t)t0 * K + i;
    const int e = r.ids[at];
    if (e >= 0) {
      const int row = s_off[e] + rank[e] + r.pos[at];
      r.pos[at] = row;
      if (row < r.max_rows) r.order[row] = t0 + i / K;
    }
  }
  const int64_t all = (int64_t)gridDim.x * kThreads, me = (int64_t)blockIdx.x * kThreads + tid;
  if (r.row_align > 1)
    for (int64_t e = me; e < E; e += all) pad_order(r, s_off[e] + counts[e], s_off[e + 1], 0, 1);
  pad_order(r, s_off[E], r.max_rows, me, all);
  if (blockIdx.x == 0) {
    for (int e = tid; e <= E; e += kThreads) r.offsets[e] = s_off[e];
    if constexpr (kScan) {
      if (tid < E) {
        r.counts[tid] = counts[tid];
        r.probs[tid] = probs[tid];
      }
      if (tid == 0) r.used[0] = used;
    }
    if (tid < 64) write_loss(r, counts, probs, kScan ? used : r.used[0]);
  }
}

// Gradient: dx = p (s - <p, s>) + c, with s_e = d_loss coef E counts_e / (topk used^2) and, for the chosen
// places, c_j = g_j (dg_j - <g, dg>) when the gates are renormalised; else s_e takes dg_j too and c = 0.
// The token's dg (or c) by expert goes through a row of LDS that is zero outside the chosen places.
template <int D, int L, int V>
__global__ void __launch_bounds__(kThreads) route_backward_kernel(ggemm_router_t r, const float* __restrict__ d_gates,
                                                                  const float* __restrict__ d_loss, void* d_logits,
                                                                  int64_t ld_d, int per) {
  using T = typename Elem<D>::T;
  using P = Piece<D, V>;
  constexpr int kRows = 64 / L, kPar = 4 * kRows;
  __shared__ float s_row[kPar * L * V];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = lane & (L - 1), slot = wave * kRows + lane / L, e0 = P::first(sub), E = r.experts, K = r.topk;
  float* row = s_row + slot * L * V;
  const int used = r.used[0];
  const float n = (float)used;
  const float f = d_loss && used ? d_loss[0] * (r.balance_coef * (float)E / ((float)K * n * n)) : 0.0f;
  float s[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = e0 + P::template step<L>(v);
    s[v] = e < E ? f * (float)r.counts[e] : 0.0f;
    row[e] = 0.0f;
  }
  const int t0 = blockIdx.x * per, t1 = min(t0 + per, r.tokens);
  // a place of a token: its expert (-1: none), gate and the gate's gradient
  struct Choice {
    int e;
    float g, dg;
  };
  auto choice = [&](int t, int j) {
    Choice c{-1, 0.0f, 0.0f};
    if (t < t1 && j < K) {
      const int64_t at = (int64_t)t * K + j;
      c.e = r.ids[at];
      if (d_gates) {
        c.g = r.gates[at];
        c.dg = d_gates[at];
      }
    }
    return c;
  };
  Logits<D, L, V> ahead;
  ahead.load(r, t0 + slot, t1, e0);
  Choice next = choice(t0 + slot, sub);
  for (int tb = t0; tb < t1; tb += kPar) {
    const int t = tb + slot;
    const bool in = t < t1;
    float x[V], p[V];
    const bool on = ahead.on(t, t1);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = (float)ahead.at(v);
    const Choice mine = next;
    ahead.load(r, t + kPar, t1, e0);
    next = choice(t + kPar, sub);
    float m = x[0];
#pragma unroll
    for (int v = 1; v < V; ++v) m = fmaxf(m, x[v]);
    m = over_lanes<L>(m, [](float a, float b) { return fmaxf(a, b); });
    const float inv = exps<L, V>(x, m, p);
    // the first place is taken unless every expert is barred
    const bool live = on && __shfl(mine.e, lane & ~(L - 1)) >= 0;
    if (d_gates) {
      float dot = 0.0f;
      if (r.renormalize) {
        for (int j = sub; j < K; j += L) {
          const Choice c = j < L ? mine : choice(t, j);
          dot += c.e >= 0 ? c.g * c.dg : 0.0f;
        }
        dot = sum_lanes<L>(dot);
      }
      for (int j = sub; j < K; j += L) {
        const Choice c = j < L ? mine : choice(t, j);
        if (live && c.e >= 0 && c.e < E) row[c.e] = r.renormalize ? c.g * (c.dg - dot) : c.dg;
      }
    }
    __threadfence_block();
    float c[V], ps = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = row[e0 + P::template step<L>(v)];
    if (!live) {
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = 0.0f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] *= inv;
    if (r.renormalize) {
#pragma unroll
      for (int v = 0; v < V; ++v) ps += p[v] * s[v];
      ps = sum_lanes<L>(ps);
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] += p[v] * (s[v] - ps);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        c[v] += s[v];
        ps += p[v] * c[v];
      }
      ps = sum_lanes<L>(ps);
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] = p[v] * (c[v] - ps);
    }
    __threadfence_block();
#pragma unroll
    for (int v = 0; v < V; ++v) row[e0 + P::template step<L>(v)] = 0.0f;
    __threadfence_block();
    // 0 times a NaN or infinite sum is not the 0 of a barred expert or of a token left out
    if (__ballot(!live || !(fabsf(ps) < 1e30f))) {
      asm volatile("");   // a branch, not a select per value
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] = live && x[v] != -__builtin_inff() ? c[v] : 0.0f;
    }
    if (in) store_gradient<D, L, V>(static_cast<T*>(d_logits) + (int64_t)t * ld_d, e0, E, c);
  }
}

// f(L, V) for the lanes and values per lane that hold `experts` logits
template <class F>
void with_lanes(int experts, F&& f) {
#define GGEMM_LV(l, v) f(std::integral_constant<int, l>{}, std::integral_constant<int, v>{})
  if (experts <= 8) GGEMM_LV(8, 1);
  else if (experts <= 16) GGEMM_LV(8, 2);
  else if (experts <= 32) GGEMM_LV(8, 4);
  else if (experts <= 64) GGEMM_LV(16, 4);
  else if (experts <= 128) GGEMM_LV(16, 8);
  else if (experts <= 256) GGEMM_LV(16, 16);
  else if (experts <= 512) GGEMM_LV(32, 16);
  else GGEMM_LV(64, 16);
#undef GGEMM_LV
}

bool sizes_ok(int tokens, int experts, int topk) {
  return tokens >= 0 && tokens <= GGEMM_ROUTE_MAX_TOKENS && experts >= 1 && experts <= GGEMM_ROUTE_MAX_EXPERTS && topk >= 1 &&
         topk <= GGEMM_ROUTE_MAX_TOPK && topk <= experts && (int64_t)tokens * topk <= 0x7fffffff;
}

bool route_ok(const ggemm_router_t* r) {
  if (!r || !sizes_ok(r->tokens, r->experts, r->topk) || !elem_known(r->dtype)) return false;
  if (r->tokens > 0 && (!r->logits || !aligned(r->logits, elem_bytes(r->dtype)) || r->ld < r->experts)) return false;
  if (r->tokens > 0 && (!r->ids || !r->gates)) return false;
  return r->counts && r->used;
}

}  // namespace

size_t route_workspace(int tokens, int experts, int topk) {
  if (!sizes_ok(tokens, experts, topk)) return 0;
  const Shape sh = shape_of(tokens);
  return 2 * align_up((size_t)sh.groups * experts * 4, 16) + align_up((size_t)sh.groups * 4, 16);
}

int route(const ggemm_router_t* r, void* ws, size_t ws_bytes, hipStream_t s) {
  if (!route_ok(r) || !r->offsets || !r->probs || !r->loss || (r->tokens > 0 && !r->pos)) return GGEMM_ERR_INVALID;
  if (r->row_align < 1 || r->row_align > GGEMM_ROUTE_MAX_ALIGN || (r->row_align & (r->row_align - 1)) != 0)
    return GGEMM_ERR_INVALID;
  const int64_t cap = (int64_t)r->tokens * r->topk + (int64_t)r->experts * (r->row_align - 1);
  if (cap > 0x7fffffff || r->max_rows < cap || (r->max_rows > 0 && !r->order)) return GGEMM_ERR_INVALID;
  if (ws_bytes < route_workspace(r->tokens, r->experts, r->topk)) return GGEMM_ERR_WORKSPACE;
  if (!ws || !aligned(ws, 16)) return GGEMM_ERR_INVALID;
  const Shape sh = shape_of(r->tokens);
  const RouteWs w = carve(ws, sh, r->experts);
  return launch([&] {
    with_elem(r->dtype, [&](auto d) {
      with_lanes(r->experts, [&](auto l, auto v) {
        constexpr int D = decltype(d)::value, L = decltype(l)::value, V = decltype(v)::value;
        auto go = [&](auto one) {
          constexpr int NT = first_threads(L * V, decltype(one)::value);
          const size_t lds = (size_t)r->experts * (sh.span / 32) * 4 + NT / 64 * L * V * 4;
          route_kernel<D, L, V, decltype(one)::value><<<sh.groups, NT, lds, s>>>(*r, w, sh.span);
        };
        if (sh.groups == 1) go(std::true_type{});
        else go(std::false_type{});
      });
    });
    if (sh.groups > 1) {
      if (r->experts <= kThreads && (int64_t)sh.groups * r->experts <= kFewCounts) {
        route_place_kernel<true><<<sh.groups, kThreads, 0, s>>>(*r, w, sh.span);
      } else {
        route_scan_kernel<<<ceil_div(r->experts, 16), 16 * kRuns, 0, s>>>(*r, w, sh.groups);
        route_place_kernel<false><<<sh.groups, kThreads, 0, s>>>(*r, w, sh.span);
      }
    }
  });
}

int route_backward(const ggemm_router_t* r, const float* d_gates, const float* d_loss, void* d_logits, int64_t ld_d,
                   hipStream_t s) {
  if (!route_ok(r)) return GGEMM_ERR_INVALID;
  if (r->tokens == 0) return GGEMM_OK;
  if (!d_logits || !aligned(d_logits, elem_bytes(r->dtype)) || ld_d < r->experts) return GGEMM_ERR_INVALID;
  return launch([&] { with_elem(r->dtype, [&](auto d) {
    with_lanes(r->experts, [&](auto l, auto v) {
      constexpr int D = decltype(d)::value, L = decltype(l)::value, V = decltype(v)::value;
      constexpr int kPar = 256 / L;
      const int per = std::max(kPar, (int)align_up((size_t)ceil_div(r->tokens, 2048), kPar));
      route_backward_kernel<D, L, V><<<ceil_div(r->tokens, per), kThreads, 0, s>>>(*r, d_gates, d_loss, d_logits, ld_d, per);
    });
  }); });
}

}  // namespace ggemm

extern "C" size_t ggemm_route_workspace(int tokens, int experts, int topk) {
  return ggemm::route_workspace(tokens, experts, topk);
}
extern "C" int ggemm_route(const ggemm_router_t* r, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  return ggemm::route(r, workspace, workspace_bytes, stream);
}
extern "C" int ggemm_route_backward(const ggemm_router_t* r, const float* d_gates, const float* d_loss, void* d_logits,
                                    int64_t ld_d, hipStream_t stream) {
  return ggemm::route_backward(r, d_gates, d_loss, d_logits, ld_d, stream);
}
