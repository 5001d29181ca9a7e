/*
 * kdelta.h — C ABI of libkdecay.so's gated delta rule, the decay scan's
 * content-dependent form.
 *
 * The operation (per sequence, value head h with key head h / (H / Hk)), with
 * a state S of [Dk, Dv] per head:
 *
 *     S_t = a_t (S_{t-1} - b_t k_t (k_t' S_{t-1})) + b_t k_t v_t'     a_t = exp(g_t), b_t = beta_t
 *     o_t = scale S_t' q_t
 *
 * that is, the state decays, what it holds at key k_t is erased by the share
 * b_t, and v_t is written there by the same share.
 *
 * The conventions are kdecay.h's: return codes, strides in elements, device
 * pointers, nothing allocated, nothing synchronised, work enqueued on `stream`
 * of the current device; kdecay_last_error_string() describes a failure.
 */
#ifndef KDELTA_H
#define KDELTA_H

#include <stddef.h>
#include <stdint.h>

#include "kdecay.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest head dims: of q and k, and of v. */
#define KDELTA_MAX_DK 128
#define KDELTA_MAX_DV 256

/*
 * One problem.  Tensors are [B, heads, N, D] with strides for their four
 * dimensions: the last is 1, the others and the base are multiples of 16 bytes
 * (strides of dimensions of size 1 too: give 0), and Dk and Dv are multiples of 8
 * (KDECAY_ELAYOUT, KDECAY_ESHAPE otherwise; zero channels of q and k change nothing).  g and beta are float32
 * [B, H, N] with three strides.  H is a multiple of Hk.
 *
 * cu_seqlens: null for B sequences of N rows.  Otherwise int32 [sequences + 1] on
 * the device, non-decreasing: B is 1, and sequence s is the rows cu_seqlens[s] to
 * cu_seqlens[s + 1].  The library reads the values on the device only and
 * clamps them to 0..N, so that no value makes it read or write out of range;
 * what it computes from values that decrease is unspecified.  Rows of o and of
 * the gradients that belong to no sequence are set to zero.
 *
 * init and final are float32 [sequences, H, Dk, Dv], contiguous (sequences is B
 * without cu_seqlens); null: zeros, and not wanted.
 */
typedef struct kdelta_problem {
  const void *q, *k, *v;
  const float *g, *beta;
  const int32_t* cu_seqlens;
  const float* init;
  int64_t q_strides[4], k_strides[4], v_strides[4], g_strides[3], beta_strides[3];
  int64_t B, Hk, H, N, Dk, Dv, sequences;
  float scale;
  int dtype; /* KDECAY_F32, KDECAY_BF16 or KDECAY_F16: q, k, v, o and their gradients */
} kdelta_problem;

/* Bytes of scratch that the scan or its backward needs (16-byte aligned; its
 * content need not be kept between calls), and floats of the buffer that a
 * scan with a backward fills. */
size_t kdelta_scan_workspace_bytes(const kdelta_problem* p);
size_t kdelta_scan_bwd_workspace_bytes(const kdelta_problem* p);
size_t kdelta_scan_saved_floats(const kdelta_problem* p);

/*
 * The scan over whole sequences.  saved: null, or kdelta_scan_saved_floats()
 * floats (16-byte aligned) that kdelta_scan_bwd takes.
 */
int kdelta_scan_fwd(const kdelta_problem* p, void* o, const int64_t* o_strides, float* final, float* saved,
                    void* workspace, size_t workspace_bytes, void* stream);

/*
 * Its backward, for the same problem: gradients of the inputs from d_o
 * ([B,H,N,Dv] of p->dtype) and d_final (float32, null: zero).  dg and dbeta are
 * float32 [B,H,N] contiguous; d_init is null or like init.  Deterministic: the
 * heads that share a key head are added up in order.
 */
int kdelta_scan_bwd(const kdelta_problem* p, const void* d_o, const int64_t* do_strides, const float* d_final,
                    const float* saved, void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides,
                    void* dv, const int64_t* dv_strides, float* dg, float* dbeta, float* d_init, void* workspace,
                    size_t workspace_bytes, void* stream);

/*
 * One token for a batch, one launch: q, k [B,Hk,Dk], v and out [B,H,Dv], all
 * contiguous and of `dtype` (out: out_dtype, which is dtype or F32); g, beta float32
 * [B,H]; the state float32 [B,H,Dk,Dv].  state_out may be state_in.
 */
int kdelta_step(const void* q, const void* k, const void* v, int dtype, const float* g, const float* beta,
                const float* state_in, float* state_out, void* out, int out_dtype, int64_t B, int64_t Hk, int64_t H,
                int64_t Dk, int64_t Dv, float scale, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KDELTA_H */
