/* ggemm_glu.h -- the gated feed-forward block of a language model's layer on MI355X, dense or for the experts of a
 * mixture, in 16-bit floating point, and its gradients.  No counterpart in the reference (its application has a
 * tanh between two FP64 products: bench/app/moe_ffn_fp64.cu).
 *
 * For the rows r of group e, offsets[e] <= r < offsets[e + 1] (as ggemm_route writes them):
 *   x_r = x[r], or with an index x[index[r]], and zeros where index[r] lies outside [0, x_rows)
 *   gate = x_r Wg_e^T,  up = x_r Wu_e^T,  h = act(gate) up,  y = h Wd_e^T
 * with d_model columns of x and y, d_ff of gate, up and h; Wg, Wu d_ff x d_model, Wd d_model x d_ff, a group's
 * matrices w_stride (d_stride) elements apart.
 *   GGEMM_SILU       v / (1 + exp(-v))
 *   GGEMM_GELU       v (1 + erf(v / sqrt 2)) / 2, within 5e-7 beside a rounding of 32 bits (of itself 5e-5 at -3, 2e-3 at -5)
 *   GGEMM_GELU_TANH  v (1 + tanh(sqrt(2 / pi) (v + 0.044715 v^3))) / 2
 * Sums, activation and its slope are 32-bit; h, what is kept of gate and up, and every result are each rounded
 * once to their type, and h comes from the unrounded sums.
 *
 * Functions work on the caller's stream and memory, allocate nothing, do not synchronise, may be captured into a
 * graph, and return a GGEMM_* code.  Arguments are checked before anything is launched (GGEMM_ERR_INVALID); a launch
 * that fails gives GGEMM_ERR_CUDA.  Pointers are device pointers; leading dimensions and strides count elements.
 * Results are the same bits every time.
 */
#ifndef GGEMM_GLU_H
#define GGEMM_GLU_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#include "ggemm.h"
#include "ggemm_mx4.h"   /* GGEMM_F32, GGEMM_BF16, GGEMM_F16 */

#ifdef __cplusplus
extern "C" {
#endif

#define GGEMM_SILU 1
#define GGEMM_GELU 2
#define GGEMM_GELU_TANH 3

#define GGEMM_GLU_MAX_GROUPS 4096
#define GGEMM_GLU_MAX_LD (1 << 22)     /* leading dimensions of x, dy and the weights, and d_model, d_ff */

/* Alignment: x, the weights and dy 16 bytes, their leading dimensions and strides multiples of 8 (of a row of them, what lies up
 * to the next 16 bytes may be read, to no effect); gate, up, y, dx and the weights' gradients their type's.  Any d_model and
 * d_ff from 1 on.  With an index, x_rows ldx < 2^30.  Calls of 2^23 or more tiles (64 x 64 of y and gate, 128 x 128 of the
 * weights' gradients) are refused. */
typedef struct {
  int groups, rows;              /* rows: of y, gate, up and index */
  int d_model, d_ff;
  int dtype;                     /* GGEMM_BF16 or GGEMM_F16: x, weights, gate, up, y */
  int act;
  int x_rows;                    /* rows of x that exist (with an index) */
  const void* x; int64_t ldx;
  const int32_t* index;          /* rows entries, or NULL */
  const int32_t* offsets;        /* groups + 1 ascending values, or NULL for one group of all rows */
  const void* w_gate; const void* w_up; int64_t ldw; int64_t w_stride;
  const void* w_down; int64_t ldd; int64_t d_stride;
  void* gate; void* up; int64_t ldg;   /* kept for the backward pass; forward: both NULL if they are not wanted */
  void* y; int64_t ldy;
} ggemm_glu_t;

/* Forward.  Rows in no group are not written; of rows whose index lies outside [0, x_rows), gate, up and y are zeros, whatever the weights
 * hold (an Inf, a NaN).  Offsets are read on the device and clamped to [0, rows]: wrong ones give
 * wrong results but no access out of bounds.  y, gate and up must not overlap the inputs.
 * Workspace: 16-byte aligned, contents need not be kept or cleared between calls; calls that may overlap need one each; too
 * small: GGEMM_ERR_WORKSPACE.  Its size goes by sizes and the inputs' leading dimensions only (pointers may still be NULL), 0 for
 * invalid ones and for more tiles than a call takes. */
size_t ggemm_glu_workspace(const ggemm_glu_t* p);
int ggemm_glu(const ggemm_glu_t* p, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Backward: gradients of sum dy y, from the forward call's struct (y is not looked at) with the gate and up that it kept:
 *   dh = dy Wd_e,  dgate = dh up act'(gate),  dup = dh act(gate),  h = act(gate) up   (each rounded to dtype)
 *   dx[r]  = dgate Wg_e + dup Wu_e         rows x d_model of dtype; with an index the caller adds up a row's copies
 *   dWg_e  = dgate^T x_r + dw_beta dWg_e   of dw_dtype (any of the three), as dWu_e = dup^T x_r
 *   dWd_e  = dy^T h + dw_beta dWd_e        and these too are written for groups without rows
 * Rows whose index lies outside [0, x_rows) count as zeros throughout, dy among them, and get dx = 0, whatever the weights hold.
 * dx may be NULL, dw_gate and dw_up together, and dw_down: what is not wanted is not computed.  Results must not overlap the
 * inputs or each other.  With dw_beta == 0 the
 * gradients of the weights are not read.  The workspace also goes by whether index is NULL, and is 0 for too many tiles of
 * weights' gradients that are not NULL. */
typedef struct {
  const void* dy; int64_t lddy;
  void* dx; int64_t lddx;
  int dw_dtype;
  float dw_beta;
  void* dw_gate; void* dw_up; int64_t lddw; int64_t dw_stride;
  void* dw_down; int64_t lddd; int64_t dd_stride;
} ggemm_glu_grad_t;
size_t ggemm_glu_backward_workspace(const ggemm_glu_t* p, const ggemm_glu_grad_t* d);
int ggemm_glu_backward(const ggemm_glu_t* p, const ggemm_glu_grad_t* d, void* workspace, size_t workspace_bytes,
                       hipStream_t stream);

#ifdef __cplusplus
}
static_assert(sizeof(ggemm_glu_t) == 160, "ggemm_glu_t layout");
static_assert(sizeof(ggemm_glu_grad_t) == 96, "ggemm_glu_grad_t layout");
#endif
#endif
