/* ggemm_mx4.h -- microscaled 4-bit floating point on MI355X: quantisation and grouped products.
 * No counterpart in the reference (its low-precision planes are INT8 residues of FP64 operands).
 *
 * Format.  A matrix is stored row by row.  A row of `cols` values is cut into blocks of 32 (the last
 * one filled up with zeros); a block has one scale byte s, worth 2^(s - 127) (s = 255: NaN), and 32
 * codes of 4 bits, two to a byte, the value of lower column in the low four bits.  A code is a sign
 * (bit 3) and a magnitude 0, 0.5, 1, 1.5, 2, 3, 4, 6 (bits 0-2).
 *
 * Every function works on the caller's stream and memory: it allocates nothing, does not synchronise,
 * may be captured into a graph, and returns a GGEMM_* code.  Arguments are checked before anything is
 * launched (GGEMM_ERR_INVALID); a launch that fails gives GGEMM_ERR_CUDA.  Pointers are device
 * pointers; leading dimensions of typed matrices count elements, those of codes and scales bytes.
 */
#ifndef GGEMM_MX4_H
#define GGEMM_MX4_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#include "ggemm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GGEMM_F32  0
#define GGEMM_BF16 1
#define GGEMM_F16  2

#define GGEMM_MX4_BLOCK 32
#define GGEMM_MX4_MAX_COLS (1 << 25)   /* a quantised row; quantisation and back */
#define GGEMM_MX4_MAX_GROUPS 4096

/* Quantisation of a rows x cols matrix: row i is x[i], or with an index x[index[i]], and zeros where
 * index[i] lies outside [0, x_rows) (rows that pad a group; x may be NULL if x_rows is 0).  Per block of 32 values v, with
 * a = max |v|: s = clamp(floor(log2 a) - 2, -127, 127) + 127 (all zeros: 0), codes = v / 2^(s - 127)
 * rounded to the nearest magnitude, ties to the even code, beyond 6 to 6.  A block that holds a NaN
 * or an Inf gets s = 255 and zero codes: every value of it is NaN.
 *   codes / scales     blocks along the rows:      rows x round_up(cols, 32) / 2 and / 32 bytes
 *   codes_t / scales_t blocks down the columns, stored transposed: cols x round_up(rows, 32) / 2, / 32
 * Either pair may be NULL, not both.  codes 16-byte aligned with ld_codes a multiple of 16; ld of
 * scales a multiple of 4, scales 4-byte aligned; bytes of a scale row past its blocks are not written.
 * cols (with codes_t: and rows) up to GGEMM_MX4_MAX_COLS. */
typedef struct {
  int rows, cols;
  int dtype;                     /* of x: GGEMM_F32, GGEMM_BF16, GGEMM_F16 */
  int x_rows;                    /* rows of x that exist (with an index) */
  const void* x; int64_t ld;
  const int32_t* index;          /* rows entries, or NULL */
  uint8_t* codes;    int64_t ld_codes;
  uint8_t* scales;   int64_t ld_scales;
  uint8_t* codes_t;  int64_t ld_codes_t;
  uint8_t* scales_t; int64_t ld_scales_t;
} ggemm_mx4_quant_t;
int ggemm_mx4_quantize(const ggemm_mx4_quant_t* q, hipStream_t stream);

/* y[i, j] = the value that code and scale stand for, rounded once to y's type (only f16 rounds).  cols up to
 * GGEMM_MX4_MAX_COLS; codes and scales aligned as the quantisation's. */
typedef struct {
  int rows, cols;
  int dtype;                     /* of y */
  const uint8_t* codes;  int64_t ld_codes;
  const uint8_t* scales; int64_t ld_scales;
  void* y; int64_t ld;
} ggemm_mx4_dequant_t;
int ggemm_mx4_dequantize(const ggemm_mx4_dequant_t* d, hipStream_t stream);

/* Grouped products of quantised matrices, sums in 32 bits (subnormals kept), one rounding to C's type.  offsets: device
 * array of groups + 1 ascending values, or NULL for one group that spans everything.
 *   GGEMM_MX4_ROWS   C[r, :] = alpha A[r, :] B_g^T + beta C[r, :] for offsets[g] <= r < offsets[g + 1]
 *                    A m x k, B_g n x k (b_stride / b_scales_stride bytes apart), C m x n.  Rows of C
 *                    in no group are not written.  (Forward and input gradient of an expert layer.)
 *   GGEMM_MX4_INNER  C_g = alpha A[:, K_g] B[:, K_g]^T + beta C_g,  K_g = [offsets[g], offsets[g + 1])
 *                    A m x k, B n x k, C_g m x n (c_stride elements apart); offsets multiples of 32
 *                    (others are rounded down).  (Weight gradient; A and B transposed quantisations.)
 * Offsets are read on the device; they are clamped to [0, m] or [0, k], so wrong ones give wrong
 * results but no access out of bounds.  alpha == 0 still multiplies; with beta == 0 C is not read.  k = 0 (or
 * an empty K_g) gives beta C.  C must not overlap the inputs.
 * Alignment: a, b and their ld and stride multiples of 16 bytes; scales, their ld and stride of 4 bytes: expert e's part
 * of a transposed quantisation, columns k e on, can be B_e if k is a multiple of 128.  C needs its type's alignment only.  Results are the same bits every time.
 * Products of 2^23 or more tiles (16 x 32 to 256 x 256 of C) are refused. */
#define GGEMM_MX4_ROWS  0
#define GGEMM_MX4_INNER 1
typedef struct {
  int form, groups;
  int m, n, k;
  int dtype;                     /* of C */
  float alpha, beta;
  const uint8_t* a;        int64_t lda;
  const uint8_t* a_scales; int64_t lda_scales;
  const uint8_t* b;        int64_t ldb; int64_t b_stride;
  const uint8_t* b_scales; int64_t ldb_scales; int64_t b_scales_stride;
  const int32_t* offsets;
  void* c; int64_t ldc; int64_t c_stride;
} ggemm_mx4_gemm_t;
/* Bytes of workspace (16-byte aligned) that a call with these sizes, leading dimensions and strides needs: often 0, and
 * 0 for invalid ones.  Pointers are not looked at: they may still be NULL. */
size_t ggemm_mx4_gemm_workspace(const ggemm_mx4_gemm_t* p);
/* Too small a workspace: GGEMM_ERR_WORKSPACE.  Its contents need not be kept or cleared between calls;
 * calls that may overlap need one each. */
int ggemm_mx4_gemm(const ggemm_mx4_gemm_t* p, void* workspace, size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
static_assert(sizeof(ggemm_mx4_quant_t) == 104, "ggemm_mx4_quant_t layout");
static_assert(sizeof(ggemm_mx4_dequant_t) == 64, "ggemm_mx4_dequant_t layout");
static_assert(sizeof(ggemm_mx4_gemm_t) == 144, "ggemm_mx4_gemm_t layout");
#endif
#endif
