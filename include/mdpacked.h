/*
 * mdpacked.h -- C ABI of attention over packed sequences: prompts and images of different lengths one behind the other without
 * padding, causal or not, heads of q in groups that share a head of k and v, with the backward pass.
 *
 * Part of libmdattn.so, with the conventions and the MDATTN_E_* codes of mdattn.h: a HIP stream first, work only enqueued,
 * nothing allocated or synchronised, arguments checked on the host before any launch, caller-owned device pointers,
 * re-entrant.
 */
#ifndef MDPACKED_H_
#define MDPACKED_H_

#include "mdattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The tensors' sizes and the sequences.  Sequence i is the rows q_offsets[i] .. q_offsets[i + 1] of q and the rows k_offsets[i] ..
 * k_offsets[i + 1] of k and v, of which the first k_lengths[i] are keys where k_lengths is given (a cache with room).  The offsets are
 * int32 in device memory and are read by the kernels: a captured graph follows what they hold when it is replayed.  They
 * must not decrease; whatever they hold, no row outside the tensors is touched.  Rows of q in front of the first sequence and behind the last
 * belong to none.
 *   q_strides, k_strides, v_strides, o_strides   elements between tokens (.seq, below 2^23) and heads (.head, below 2^40; in the backward
 *                  pass, of q and out, below 2^29 * kv_heads / heads), multiples of 8; .batch unused; head dim contiguous
 *   max_q, max_k   hints, the longest sequence's rows: they choose how the work is cut, and nothing else depends on them.  Without them (0) a call
 *                  is planned for one sequence of all rows: single tokens against several caches are then not cut over their keys.
 */
typedef struct {
  const int* q_offsets;
  const int* k_offsets;
  const int* k_lengths; /* or NULL */
  int sequences;        /* both offsets have one element more */
  int q_rows, k_rows;   /* rows of the tensors */
  int heads, kv_heads;  /* heads of q, a multiple of the heads of k and v: head h of q meets head h / (heads / kv_heads) */
  int head_dim;         /* a multiple of 8 up to 128 */
  int causal;           /* of a sequence with m queries and n keys, query i sees the keys up to i + n - m */
  int max_q, max_k;
} mdattn_packed;

/*
 * out = softmax(scale * q k^T) v over each sequence; bf16; scale positive and finite.  rest, strided like out, or NULL: what the rounding of out
 * left, rounded to bf16, for the backward pass (of rows of no sequence it is not written).  lse f32 [heads, q_rows], or NULL: the logarithm of each row's sum.  Rows
 * that see no key, and rows of no sequence: out 0, lse -inf.  Logits, softmax and sums in f32, P rounded to bf16 before its product.
 *   workspace     mdattn_fwd_bf16_packed_workspace_floats floats (0 where one is not needed), with which few rows against many keys are
 *                 split over the keys; with less they are not.  16-byte aligned.
 * A key or value that is infinite or NaN may spoil the rows of its sequence that do not see it.
 */
int64_t mdattn_fwd_bf16_packed_workspace_floats(const mdattn_packed* p);
int mdattn_fwd_bf16_packed(void* stream, const mdattn_packed* p, const void* q, const void* k, const void* v, void* out, void* rest,
                           float* lse, const mdattn_strides* q_strides, const mdattn_strides* k_strides, const mdattn_strides* v_strides,
                           const mdattn_strides* o_strides, float scale, float* workspace, int64_t workspace_floats);

/*
 * Backward of mdattn_fwd_bf16_packed: dq, dk, dv (bf16, strided like q, k and v) from its inputs, out, rest, lse and the
 * gradient of out (strided like it, as rest is).  rest may be NULL, for gradients that are further off where a key has most of a row's weight.
 * k_lengths has to be NULL, and scale 1e-30 at least (lse is divided by it).  Rows of no sequence get zeros.  Deterministic: sums over the rows and
 * over the heads of a group are made in a fixed order.
 *   workspace     mdattn_bwd_bf16_packed_workspace_floats floats; 16-byte aligned
 */
int64_t mdattn_bwd_bf16_packed_workspace_floats(const mdattn_packed* p);
int mdattn_bwd_bf16_packed(void* stream, const mdattn_packed* p, const void* q, const void* k, const void* v, const void* out, const void* rest,
                           const void* dout, const float* lse, void* dq, void* dk, void* dv, const mdattn_strides* q_strides, const mdattn_strides* k_strides,
                           const mdattn_strides* v_strides, const mdattn_strides* o_strides, const mdattn_strides* dq_strides,
                           const mdattn_strides* dk_strides, const mdattn_strides* dv_strides, float scale, float* workspace,
                           int64_t workspace_floats);

#ifdef __cplusplus
}
#endif
#endif /* MDPACKED_H_ */
