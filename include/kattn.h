/*
 * kattn.h — C ABI of libkdecay.so's causal attention over whole prompts: what the
 * recall heads of a hybrid layer run beside its decay heads
 * (/root/reference/src/kilat/arc/attention.py:400-518, torch's
 * scaled_dot_product_attention there).
 *
 *     o_i = sum_{j <= i} softmax_j(scale q_i.k_j) v_j
 *
 * per sequence and head h, with key head h / (H / Hk).  The conventions are kdecay.h's.
 */
#ifndef KATTN_H
#define KATTN_H

#include <stddef.h>
#include <stdint.h>

#include "kdecay.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest head dims: of q and k, and of v. */
#define KATTN_MAX_DK 128
#define KATTN_MAX_DV 128

/*
 * q [B,H,N,Dk], k [B,Hk,N,Dk], v [B,Hk,N,Dv], with strides for their four dimensions, as
 * kdelta.h asks of rows: the last is 1, the others and the bases are multiples of 16
 * bytes, and the head dims of 8.  cu_seqlens and sequences: as in
 * kdelta.h (kdelta_problem).
 */
typedef struct kattn_problem {
  const void *q, *k, *v;
  const int32_t* cu_seqlens;
  int64_t q_strides[4], k_strides[4], v_strides[4];
  int64_t B, Hk, H, N, Dk, Dv, sequences;
  float scale;
  int dtype; /* KDECAY_F32, KDECAY_BF16 or KDECAY_F16: q, k, v and o */
} kattn_problem;

/* o [B,H,N,Dv] of p->dtype; rows of no sequence are set to zero. */
int kattn_fwd(const kattn_problem* p, void* o, const int64_t* o_strides, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KATTN_H */
