// mx4gemm.hip -- grouped products of microscaled 4-bit matrices (include/ggemm_mx4.h).
//
// C = A B^T by v_mfma_scale_f32_32x32x64_f8f6f4: lane l holds 32 codes (one block, 16 bytes) of row
// l % 32 at k block l / 32 and that block's scale byte; products of codes are exact, sums are 32-bit.
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"

namespace ggemm {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;

// Where a workgroup's tile lies: its group, its first row and the group's end (rows form), or the blocks of
// the inner dimension it sums over (inner form).
struct Span {
  int g, lo, hi;
};

__device__ __forceinline__ int clamp_to(int x, int n) { return min(max(x, 0), n); }

// The block that an offset along an inner dimension of k starts at.
__device__ __forceinline__ int block_at(int x, int k) { return x >= k ? ceil_div(k, 32) : max(x, 0) / 32; }

// Row tile t of the groups' tiles in order, each group cut into tiles of TM rows; g = -1 past the last.
// Every wave finds it on its own: 64 groups a step, an inclusive sum of their tile counts over the lanes.
template <int TM>
__device__ __forceinline__ Span find_rows(const ggemm_mx4_gemm_t& p, int t) {
  const int lane = threadIdx.x & 63;
  if (!p.offsets) return t * TM < p.m ? Span{0, t * TM, p.m} : Span{-1, 0, 0};
  for (int g0 = 0; g0 < p.groups; g0 += 64) {
    const int g = min(g0 + lane, p.groups - 1);
    const int lo = clamp_to(p.offsets[g], p.m), hi = clamp_to(p.offsets[g + 1], p.m);
    int sum = g0 + lane < p.groups ? (max(hi - lo, 0) + TM - 1) / TM : 0;
    const int own = sum;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int up = __shfl_up(sum, d);
      sum += lane >= d ? up : 0;
    }
    const uint64_t hit = __ballot(sum > t);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int before = __shfl(sum - own, l);
      return Span{g0 + l, __shfl(lo, l) + (t - before) * TM, __shfl(hi, l)};
    }
    t -= __shfl(sum, 63);
  }
  return Span{-1, 0, 0};
}

template <int D>
__device__ __forceinline__ void store_c(const ggemm_mx4_gemm_t& p, typename Elem<D>::T* c, float v) {
  v *= p.alpha;
  if (p.beta != 0.0f) v += p.beta * (float)*c;
  *c = (typename Elem<D>::T)v;
}

// Four waves, 32 x 32 each, operands straight from memory.
template <int D, bool kInner>
__global__ void __launch_bounds__(kThreads) gemm_simple_kernel(ggemm_mx4_gemm_t p) {
  using T = typename Elem<D>::T;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * kTile + (wave & 1) * 32;
  int m0, m_end, b0 = 0, b1, g;
  if constexpr (kInner) {
    g = blockIdx.z;
    m0 = blockIdx.y * kTile;
    m_end = p.m;
    b1 = ceil_div(p.k, 32);
    if (p.offsets) {
      b0 = block_at(p.offsets[g], p.k);
      b1 = block_at(p.offsets[g + 1], p.k);
    }
  } else {
    const Span s = find_rows<kTile>(p, blockIdx.y + blockIdx.z * gridDim.y);
    if (s.g < 0) return;
    g = s.g;
    m0 = s.lo;
    m_end = s.hi;
    b1 = ceil_div(p.k, 32);
  }
  m0 += (wave >> 1) * 32;
  const int row = min(m0 + (lane & 31), m_end - 1), col = min(n0 + (lane & 31), p.n - 1);
  const uint8_t* a = p.a + (int64_t)row * p.lda;
  const uint8_t* as = p.a_scales + (int64_t)row * p.lda_scales;
  const uint8_t* b = p.b + (int64_t)col * p.ldb;
  const uint8_t* bs = p.b_scales + (int64_t)col * p.ldb_scales;
  if constexpr (!kInner) {
    b += g * p.b_stride;
    bs += g * p.b_scales_stride;
  }
  f32x16 acc = {};
  for (int k = b0; k < b1; k += 2) {
    const int blk = k + (lane >> 5);
    i32x8 av = {}, bv = {};
    int sa = 127, sb = 127;
    if (blk < b1) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(a + 16 * (int64_t)blk);
      const u32x4 y = *reinterpret_cast<const u32x4*>(b + 16 * (int64_t)blk);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        av[i] = (int)x[i];
        bv[i] = (int)y[i];
      }
      sa = as[blk];
      sb = bs[blk];
    }
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc, 4, 4, 0, sa, 0, sb);
  }
  T* c = static_cast<T*>(p.c) + (kInner ? g * p.c_stride : 0);
  const int j = n0 + (lane & 31);
  if (j >= p.n) return;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int i = m0 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
    if (i < m_end) store_c<D>(p, c + (int64_t)i * p.ldc + j, acc[r]);
  }
}

bool gemm_ok(const ggemm_mx4_gemm_t* p) {
  if (!p || (p->form != GGEMM_MX4_ROWS && p->form != GGEMM_MX4_INNER) || p->groups < 1 ||
      p->groups > GGEMM_MX4_MAX_GROUPS || p->m < 0 || p->n < 0 || p->k < 0 || !elem_known(p->dtype) ||
      (!p->offsets && p->groups != 1))
    return false;
  if (p->m == 0 || p->n == 0) return true;
  const bool inner = p->form == GGEMM_MX4_INNER;
  if (!p->c || !aligned(p->c, elem_bytes(p->dtype)) || p->ldc < p->n || !aligned(p->offsets, 4)) return false;
  if (inner && p->groups > 1 && (p->c_stride < 0 || p->c_stride < (int64_t)(p->m - 1) * p->ldc + p->n)) return false;
  if (p->k == 0) return true;
  const int64_t nb = ceil_div(p->k, 32);
  auto operand = [&](const uint8_t* x, int64_t ld, const uint8_t* s, int64_t lds) {
    return x && s && aligned(x, 16) && aligned(s, 4) && ld % 16 == 0 && ld >= 16 * nb && lds % 4 == 0 && lds >= nb;
  };
  return operand(p->a, p->lda, p->a_scales, p->lda_scales) && operand(p->b, p->ldb, p->b_scales, p->ldb_scales) &&
         (inner || p->groups == 1 || (p->b_stride % 16 == 0 && p->b_scales_stride % 4 == 0));
}

// Row tiles of TM rows that the groups can have at most: sum ceil(m_g / TM) <= m / TM + groups with rows.
int64_t row_tiles(const ggemm_mx4_gemm_t& p, int tm) {
  return p.offsets ? (int64_t)p.m / tm + std::min(p.groups, p.m) : ceil_div(p.m, tm);
}

}  // namespace

size_t mx4_gemm_workspace(const ggemm_mx4_gemm_t* p) {
  if (!gemm_ok(p)) return 0;
  return 16;
}

int mx4_gemm(const ggemm_mx4_gemm_t* p, void* ws, size_t ws_bytes, hipStream_t s) {
  if (!gemm_ok(p)) return GGEMM_ERR_INVALID;
  if (p->m == 0 || p->n == 0) return GGEMM_OK;
  if (ws_bytes < mx4_gemm_workspace(p)) return GGEMM_ERR_WORKSPACE;
  if (!ws || !aligned(ws, 16)) return GGEMM_ERR_INVALID;
  const int nt = ceil_div(p->n, kTile);
  bool fits = true;
  with_elem(p->dtype, [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (p->form == GGEMM_MX4_INNER) {
      const int mt = ceil_div(p->m, kTile);
      if (mt > 65535) { fits = false; return; }
      gemm_simple_kernel<D, true><<<dim3(nt, mt, p->groups), kThreads, 0, s>>>(*p);
    } else {
      const int64_t mt = row_tiles(*p, kTile);
      const int64_t z = (mt + 32767) / 32768;
      gemm_simple_kernel<D, false><<<dim3(nt, (unsigned)std::min<int64_t>(mt, 32768), (unsigned)z), kThreads, 0, s>>>(*p);
    }
  });
  if (!fits) return GGEMM_ERR_INVALID;
  return hipGetLastError() == hipSuccess ? GGEMM_OK : GGEMM_ERR_CUDA;
}

}  // namespace ggemm

extern "C" size_t ggemm_mx4_gemm_workspace(const ggemm_mx4_gemm_t* p) { return ggemm::mx4_gemm_workspace(p); }
extern "C" int ggemm_mx4_gemm(const ggemm_mx4_gemm_t* p, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  return ggemm::mx4_gemm(p, workspace, workspace_bytes, stream);
}
