/* ggemm_w8.h -- 8-bit integer matrix products with a scale for each row of both operands on MI355X (activations: for each
 * token; weights: for each output channel), quantisation of rows and back, and the gated pair of products of a
 * feed-forward block.  No counterpart in the reference (its INT8 planes are residues of FP64 operands).
 *
 * Functions work on the caller's stream and memory, allocate nothing, do not synchronise, may be captured into a
 * graph, and return a GGEMM_* code.  Arguments are checked before anything is launched (GGEMM_ERR_INVALID); a launch
 * that fails gives GGEMM_ERR_CUDA.  Pointers are device pointers; leading dimensions and strides count elements.
 * Results are the same bits every time.
 */
#ifndef GGEMM_W8_H
#define GGEMM_W8_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#include "ggemm.h"
#include "ggemm_glu.h"   /* activations */
#include "ggemm_mx4.h"   /* GGEMM_F32, GGEMM_BF16, GGEMM_F16 */

#ifdef __cplusplus
extern "C" {
#endif

#define GGEMM_W8_MAX_COLS (1 << 17)    /* a quantised row, and k of a product (exclusive): sums stay below 2^31 */
#define GGEMM_W8_MAX_GROUPS 4096
#define GGEMM_W8_MAX_LD (1 << 23)      /* leading dimensions of quantised operands */

/* Quantisation of rows: row i is x[i], or with an index x[index[i]], and zeros where index[i] lies outside [0, x_rows)
 * (x may be NULL if x_rows is 0).
 *   scales[i] = max(a / 127, 2^-126), a = max |x| of the row, the quotient rounded to 32 bits
 *   q[i, j]   = x / scales[i] to the nearest whole number, ties to the even one (the quotient itself, not a rounding of it)
 * A row with a NaN or an Inf gets a NaN scale and q = 0.  Columns of q past cols are not written.  Any alignment of x and q
 * that suits their types; as operands of products, q has to be 16-byte aligned with ldq a multiple of 16.  q and scales must
 * not overlap x. */
typedef struct {
  int rows, cols;
  int dtype;                     /* of x: GGEMM_F32, GGEMM_BF16, GGEMM_F16 */
  int x_rows;                    /* rows of x that exist (with an index) */
  const void* x; int64_t ld;
  const int32_t* index;          /* rows entries, or NULL */
  int8_t* q; int64_t ldq;
  float* scales;                 /* rows */
} ggemm_w8_quant_t;
int ggemm_w8_quantize(const ggemm_w8_quant_t* q, hipStream_t stream);

/* y[i, j] = q[i, j] scales[i], in 32 bits, then rounded to y's type.  y must not overlap q and scales. */
typedef struct {
  int rows, cols;
  int dtype;                     /* of y */
  const int8_t* q; int64_t ldq;
  const float* scales;
  void* y; int64_t ld;
} ggemm_w8_dequant_t;
int ggemm_w8_dequantize(const ggemm_w8_dequant_t* d, hipStream_t stream);

/* Grouped products: for the rows r of group e, offsets[e] <= r < offsets[e + 1],
 *   s[r, j] = sum_i a[r, i] b_e[j, i]           a whole number, exact
 *   v[r, j] = (s a_scales[r]) b_scales_e[j]     in 32-bit floating point (s is rounded to it first)
 *   act 0:    c[r, j] = v
 *   GGEMM_SILU, GGEMM_GELU, GGEMM_GELU_TANH (ggemm_glu.h): c[r, j] = act(v) w, with w the same of b_up and its scales
 * rounded once to c's type.  A m x k, B_e n x k (b_stride elements apart, its scales b_scales_stride; b_up alike), C m x n.
 * Rows in no group are not written.  Offsets are read on the device and clamped to [0, m]: wrong ones give wrong results
 * but no access out of bounds.  Every int8 value may occur.  C must not overlap the inputs.
 * Alignment: a, b, b_up 16 bytes, their leading dimensions and strides multiples of 16; scales 4 bytes; C its type's.
 * Of a row of a, b, b_up, what lies up to the next 16 bytes may be read, to no effect.  Products of 2^23 or more tiles (64 x 128 of
 * C, 64 x 64 of a pair) are refused. */
typedef struct {
  int groups;
  int m, n, k;
  int dtype;                     /* of C */
  int act;                       /* 0: one product; else the gated pair */
  const int8_t* a; int64_t lda;
  const float* a_scales;         /* m */
  const int8_t* b; const int8_t* b_up; int64_t ldb; int64_t b_stride;
  const float* b_scales; const float* b_up_scales; int64_t b_scales_stride;
  const int32_t* offsets;        /* groups + 1 ascending values, or NULL for one group of all rows */
  void* c; int64_t ldc;
} ggemm_w8_gemm_t;
/* Bytes of workspace that a call needs: 0, whatever its sizes, in this version of the library. */
size_t ggemm_w8_gemm_workspace(const ggemm_w8_gemm_t* p);
/* workspace and workspace_bytes are not looked at (NULL and 0 will do); they stand for kernels that may come to need some. */
int ggemm_w8_gemm(const ggemm_w8_gemm_t* p, void* workspace, size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
static_assert(sizeof(ggemm_w8_quant_t) == 64, "ggemm_w8_quant_t layout");
static_assert(sizeof(ggemm_w8_dequant_t) == 56, "ggemm_w8_dequant_t layout");
static_assert(sizeof(ggemm_w8_gemm_t) == 128, "ggemm_w8_gemm_t layout");
#endif
#endif
