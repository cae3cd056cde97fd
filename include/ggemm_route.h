/* ggemm_route.h -- the router of a mixture-of-experts layer on MI355X: chosen experts and gates,
 * per-expert counts, the order of the rows by expert that grouped products run on, the balance loss,
 * and the gradient of the logits.  No counterpart in the reference (its application draws the routing
 * on the host: bench/app/moe_ffn_fp64.cu).
 *
 * For token t with logits x over E experts (softmax p over the experts with x > -inf):
 *   ids    the topk largest logits in descending order, equal ones (-0 = +0) by lowest index, NaN
 *          above every number; an expert with x = -inf is barred
 *   gates  p at the chosen experts, or with renormalize divided by their sum
 * A token whose mask byte is 0, or all of whose experts are barred, is left out: its logits count
 * nowhere, ids and pos are -1, gates 0.  A token with fewer than topk experts left has -1, -1 and 0 in the
 * remaining places.  A NaN or +Inf logit of a token that is not left out makes its p NaN, and with it
 * the gates, probs and loss.
 *   counts[e]   pairs (t, j) with ids[t, j] = e;  offsets: exclusive sums of the counts rounded up to
 *               row_align, offsets[E] the rows in all
 *   pos[t, j]   row of the pair: offsets[e] + how many tokens before t chose e
 *   order[row]  the row's token, -1 in padding rows and from offsets[E] on (max_rows entries)
 *   used        tokens not left out;  probs[e] = sum_t p[t, e] / used (0 if used = 0)
 *   loss        balance_coef E sum_e f_e probs[e],  f_e = counts[e] / (topk used)
 * Sums are 32-bit in a fixed order: results are the same bits every time.
 *
 * Functions work on the caller's stream and memory, allocate nothing, do not synchronise, may be
 * captured into a graph, and return a GGEMM_* code; arguments are checked before anything is launched.
 */
#ifndef GGEMM_ROUTE_H
#define GGEMM_ROUTE_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#include "ggemm.h"
#include "ggemm_mx4.h"   /* GGEMM_F32, GGEMM_BF16, GGEMM_F16 */

#ifdef __cplusplus
extern "C" {
#endif

#define GGEMM_ROUTE_MAX_TOKENS (1 << 30)   /* and tokens topk + experts (row_align - 1) < 2^31 */
#define GGEMM_ROUTE_MAX_EXPERTS 1024
#define GGEMM_ROUTE_MAX_TOPK 64
#define GGEMM_ROUTE_MAX_ALIGN 1024

typedef struct {
  int tokens, experts, topk;
  int row_align;                 /* power of two */
  int dtype;                     /* of the logits (and their gradient) */
  int renormalize;
  float balance_coef;
  int max_rows;                  /* entries of order: >= tokens topk + experts (row_align - 1) */
  const void* logits; int64_t ld;
  const uint8_t* mask;           /* tokens bytes, or NULL */
  int32_t* ids;                  /* tokens x topk, contiguous, as gates and pos */
  float* gates;
  int32_t* pos;
  int32_t* counts;               /* experts */
  int32_t* offsets;              /* experts + 1 */
  int32_t* order;                /* max_rows */
  int32_t* used;                 /* 1 */
  float* probs;                  /* experts */
  float* loss;                   /* 1 */
} ggemm_router_t;

/* Bytes of workspace (16-byte aligned) that ggemm_route needs; 0 for sizes out of range. */
size_t ggemm_route_workspace(int tokens, int experts, int topk);
int ggemm_route(const ggemm_router_t* r, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Gradient of d_loss loss + sum d_gates gates with respect to the logits (counts and the choice held
 * fixed): d_logits, tokens x experts of the logits' type, leading dimension ld_d; zeros for tokens
 * left out and barred experts.  r: the struct of the forward call, whose ids, gates, counts and used are read
 * (pos, offsets, order, probs and loss may be NULL).  d_gates (tokens x topk) or d_loss (one device value) may be NULL:
 * taken as zero. */
int ggemm_route_backward(const ggemm_router_t* r, const float* d_gates, const float* d_loss, void* d_logits,
                         int64_t ld_d, hipStream_t stream);

#ifdef __cplusplus
}
static_assert(sizeof(ggemm_router_t) == 128, "ggemm_router_t layout");
#endif
#endif
