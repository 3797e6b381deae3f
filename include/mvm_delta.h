/*
 * mvm_delta.h -- C ABI of the gated delta rule on packed and served sequences
 * (libmvm_scan.so): a recurrence with a matrix state beside the selective
 * scan's diagonal one (the reference has only the latter,
 * mlx_vision_mamba/mamba_block.py:20-74).
 *
 * For each sequence and value head, with the key head hk = h / (value_heads /
 * key_heads) and a state S of dk x dv values:
 *
 *   a_t = exp(g_t)
 *   d_t = beta_t (v_t - a_t S_{t-1}^T k_t)
 *   S_t = a_t S_{t-1} + k_t d_t^T
 *   o_t = scale S_t^T q_t
 *
 * with qk_l2norm q_t and k_t are first divided by sqrt(sum of squares + 1e-6).
 *
 * Conventions are those of mvm_seq.h (sequences, slots, fresh, states) and
 * mvm_scan.h (status codes, mvm_last_error, caller-owned buffers and workspace,
 * host-side validation, deterministic results).
 *
 *   q, k (tokens, key_heads, dk), v (tokens, value_heads, dv): rows and heads
 *   with strides, the last dimension contiguous.  g (tokens, value_heads)
 *   float32, beta the same in beta_dtype: rows with a stride.  o and all
 *   gradients are contiguous.  States: (rows, value_heads, dk, dv) float32.
 *   Strides are at most 2^29 - 1 values, v_stride and value_heads * dv 2^25.
 *
 * g is taken as at least -10000 (exp of which is 0), below which its gradient
 * is zero.  Products run over chunks
 * of 64 tokens: a value that is not finite makes its sequence's outputs
 * meaningless from the start of its chunk on, no other sequence's.
 */
#ifndef MVM_DELTA_H
#define MVM_DELTA_H

#include <stddef.h>
#include <stdint.h>

#include "mvm_seq.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MVM_DELTA_MAX_DK 128
#define MVM_DELTA_MAX_DV 512

typedef struct mvm_delta_desc {
  mvm_seq_desc seq;             /* dim must be 0 */
  int64_t key_heads;            /* >= 1 */
  int64_t value_heads;          /* a multiple of key_heads */
  int64_t dk;                   /* 1..MVM_DELTA_MAX_DK */
  int64_t dv;                   /* 1..MVM_DELTA_MAX_DV */
  int64_t q_stride, q_stride_head, k_stride, k_stride_head, v_stride, v_stride_head;
  int64_t g_stride, beta_stride;
  int64_t max_len;              /* an upper bound of the lengths, 0: unknown.
                                   Only the split over the time axis goes by it */
  float scale;
  int32_t dtype;                /* q, k, v, o and their gradients */
  int32_t beta_dtype;           /* MVM_F32 or dtype */
  int32_t qk_l2norm;
  int32_t split_len;            /* 0: the library picks the time split; else a
                                   multiple of 64, the tokens of a part */
  int32_t reserved;             /* 0 */
} mvm_delta_desc;

/* Validates a descriptor without touching the GPU. */
int mvm_delta_validate(const mvm_delta_desc* desc);

/* float32 elements of the checkpoints that a forward leaves for a backward:
 * each chunk's initial state, the rows d_t, the chunk's triangles and decays.
 * (A head of 128 x 128: 2.1 KiB a token, about twice its q, k, v and o in
 * bfloat16.) */
int64_t mvm_delta_ckpt_elems(const mvm_delta_desc* desc);

/* Workspace bytes: which = 0 forward, with or without checkpoints, 1 backward.
 * The workspace must be 256-byte aligned, the checkpoints 16-byte.  (A head of
 * 128 x 128: 0.6 KiB a token forward, 1.5 backward, and what the parts of the
 * time axis leave each other.) */
int64_t mvm_delta_workspace_bytes(const mvm_delta_desc* desc, int which);

/* h0 (zero), h1 (not stored) and ckpt (no backward) may be NULL; h0 and h1 may
 * be one buffer. */
int mvm_delta_fwd(const mvm_delta_desc* desc, const void* q, const void* k, const void* v,
                  const float* g, const void* beta, const float* h0, float* h1, void* o,
                  float* ckpt, void* workspace, size_t workspace_bytes, void* stream);

/* Gradients for d_o (contiguous) and dh1 (may be NULL: zero).  slots and fresh
 * must be NULL.  dq, dk, dv, dbeta in the types of their primals, dg and dh0
 * (may be NULL; not dh1's buffer) float32; all written in full. */
int mvm_delta_bwd(const mvm_delta_desc* desc, const void* q, const void* k, const void* v,
                  const float* g, const void* beta, const float* ckpt, const void* d_o,
                  const float* dh1, void* dq, void* dk, void* dv, float* dg, void* dbeta,
                  float* dh0, void* workspace, size_t workspace_bytes, void* stream);

/* One token for each sequence (tokens == nseq, offsets NULL, seqlen 1): the
 * states advance in place; a row whose slot is outside [0, state_rows) gets
 * o = 0.  `fresh` is honoured. */
int mvm_delta_step(const mvm_delta_desc* desc, const void* q, const void* k, const void* v,
                   const float* g, const void* beta, float* states, void* o, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MVM_DELTA_H */
