// mx4.hpp -- what the kernels on microscaled 4-bit operands and the router share: element types, block
// scales, lane exchanges inside a row of 16 lanes.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.hpp"
#include "ggemm_mx4.h"

namespace ggemm {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Element types by their number in the ABI.
template <int D> struct Elem;
template <> struct Elem<GGEMM_F32> { using T = float; };
template <> struct Elem<GGEMM_BF16> { using T = __bf16; };
template <> struct Elem<GGEMM_F16> { using T = _Float16; };

inline int elem_bytes(int dtype) { return dtype == GGEMM_F32 ? 4 : 2; }
inline bool elem_known(int dtype) { return dtype == GGEMM_F32 || dtype == GGEMM_BF16 || dtype == GGEMM_F16; }
inline bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// f(integral_constant<int, D>) for the element type of a call
template <class F>
inline void with_elem(int dtype, F&& f) {
  if (dtype == GGEMM_F32) f(std::integral_constant<int, GGEMM_F32>{});
  else if (dtype == GGEMM_BF16) f(std::integral_constant<int, GGEMM_BF16>{});
  else f(std::integral_constant<int, GGEMM_F16>{});
}

// The status of the launches that f makes.  An error that an earlier call of the program left behind is not theirs.
template <class F>
inline int launch(F&& f) {
  (void)hipGetLastError();
  f();
  return hipGetLastError() == hipSuccess ? GGEMM_OK : GGEMM_ERR_CUDA;
}

// N values of type T side by side, loaded or stored as one vector at any address that suits one of them: the memory
// instructions take that, so that rows of odd length need no path of their own (results of a product, 20993 x 4062 bf16: 123 us value by
// value, 72 this way).
template <class T, int N>
struct Run {
  typedef uint32_t words __attribute__((ext_vector_type(N * sizeof(T) / 4)));
  typedef words at_any __attribute__((aligned(sizeof(T))));
  T x[N];
  static __device__ __forceinline__ Run load(const T* p) {
    return __builtin_bit_cast(Run, (words)*reinterpret_cast<const at_any*>(p));
  }
  // kStream: non-temporally
  template <bool kStream>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kStream) __builtin_nontemporal_store(__builtin_bit_cast(words, *this), reinterpret_cast<at_any*>(p));
    else *reinterpret_cast<at_any*>(p) = __builtin_bit_cast(words, *this);
  }
};
// one 16-bit value
template <>
struct Run<__bf16, 1> {
  __bf16 x[1];
  static __device__ __forceinline__ Run load(const __bf16* p) { return Run{{*p}}; }
  template <bool>
  __device__ __forceinline__ void store(__bf16* p) const { *p = x[0]; }
};
template <>
struct Run<_Float16, 1> {
  _Float16 x[1];
  static __device__ __forceinline__ Run load(const _Float16* p) { return Run{{*p}}; }
  template <bool>
  __device__ __forceinline__ void store(_Float16* p) const { *p = x[0]; }
};

// The scale byte s as a number: 2^(s - 127), exact (s = 0 is the subnormal 2^-127); s < 255.
__device__ __forceinline__ float mx4_scale(uint32_t s) { return __uint_as_float(s ? s << 23 : 1u << 22); }

// Scale byte of a block whose largest magnitude has the bits `amax` (as a 32-bit float, sign cleared):
// 255 for NaN and Inf, else clamp(floor(log2 amax) - 2, -127, 127) + 127 = max(exponent field - 2, 0)
// (zeros and subnormals have field 0, and 252 is the largest result).
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t amax) {
  const uint32_t e = amax >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}

// x of another lane of the same row of 16, by a data-parallel-primitive control word
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);
}
constexpr int kDppXor1 = 0xb1, kDppXor2 = 0x4e;      // quad_perm [1,0,3,2] and [2,3,0,1]
constexpr int kDppHalfMirror = 0x141, kDppMirror = 0x140;   // lane i <-> 7 - i and 15 - i

constexpr int kChunk = 32;   // consecutive tiles that one XCD gets
// The tile of workgroup b: workgroups go to the XCDs in turn, so runs of kChunk tiles that share rows of A and B
// share an L2.  Ragged ends of 8 kChunk tiles keep their number.
__device__ __forceinline__ int tile_number(int b, int total) {
  constexpr int span = kXcds * kChunk;
  if (b >= total / span * span) return b;
  const int q = b / kXcds;
  return q / kChunk * span + b % kXcds * kChunk + q % kChunk;
}

}  // namespace ggemm
