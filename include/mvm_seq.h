/*
 * mvm_seq.h -- C ABI of the packed and served forms of the selective scan and
 * of its causal conv (libmvm_scan.so): sequences of different lengths packed
 * without padding, that start from a state and leave one, and the step of one
 * token.  The reference has neither: its scan and conv start every sequence
 * from zero and drop the final state (mlx_vision_mamba/mamba_block.py:20-74,
 * :170-171).
 *
 * Conventions are those of mvm_scan.h (status codes, mvm_last_error,
 * caller-owned buffers and workspace, host-side validation, deterministic
 * results).
 *
 * Sequences.  `tokens` rows are cut into `nseq` sequences: sequence i holds
 * the rows offsets[i] .. offsets[i + 1] - 1, or i * seqlen .. (i + 1) * seqlen
 * - 1 when offsets is NULL.  offsets lives in device memory and is not
 * inspected on the host: offsets[0] is taken as 0, the others are clamped into
 * [0, tokens], and rows past offsets[nseq] belong to no sequence (outputs and
 * gradients are zero there).  Offsets that decrease give meaningless values,
 * but no access out of bounds.  A sequence may be empty: its state passes
 * through.
 *
 * States.  Row slots[i] (or i when slots is NULL) of a state tensor of
 * `state_rows` rows is sequence i's; a slot outside [0, state_rows) means none:
 * the sequence starts from zero and its final state is dropped.  Two sequences
 * of one call must not share a slot.  fresh[i] != 0 starts sequence i from zero
 * whatever its row holds.  The initial and the final states may be one buffer.
 *
 *   scan: (rows, dim, dstate) float32.   conv: (rows, kwidth - 1, dim) of the
 *   activations' type, the last kwidth - 1 inputs, oldest first.
 *
 * Activations are rows with a stride and contiguous columns.
 */
#ifndef MVM_SEQ_H
#define MVM_SEQ_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct mvm_seq_desc {
  int64_t tokens;
  int64_t nseq;
  int64_t seqlen;          /* with offsets NULL: tokens == nseq * seqlen */
  int64_t dim;             /* channels */
  int64_t state_rows;
  const int32_t* offsets;  /* device (nseq + 1) or NULL */
  const int32_t* slots;    /* device (nseq) or NULL */
  const uint8_t* fresh;    /* device (nseq) or NULL */
} mvm_seq_desc;

typedef struct mvm_seq_scan_desc {
  mvm_seq_desc seq;
  int64_t dstate;          /* 1..MVM_MAX_DSTATE */
  int64_t u_stride, delta_stride, bc_stride, y_stride, z_stride; /* of rows */
  int64_t max_len;         /* an upper bound of the lengths, 0: unknown.  Only
                              the cut into time chunks goes by it */
  int32_t dtype;           /* u, B, C, z, y and their gradients */
  int32_t delta_dtype;     /* delta: MVM_F32 or dtype */
  int32_t delta_softplus;  /* 1: delta = softplus(delta + delta_bias) */
  int32_t a_is_log;        /* 1: A holds A_log, A = -exp(A_log) */
  int32_t chunk_len;       /* 0: the library picks; else a power of two >= 16 */
  int32_t reserved;        /* 0 */
} mvm_seq_scan_desc;

typedef struct mvm_seq_conv_desc {
  mvm_seq_desc seq;
  int64_t kwidth;          /* 1..MVM_CONV_MAX_KWIDTH */
  int64_t x_stride, y_stride;
  int32_t dtype;
  int32_t reserved;        /* 0 */
} mvm_seq_conv_desc;

/* Validates a descriptor without touching the GPU. */
int mvm_seq_scan_validate(const mvm_seq_scan_desc* desc);

/* float32 elements of the checkpoints that a forward leaves for a backward. */
int64_t mvm_seq_scan_ckpt_elems(const mvm_seq_scan_desc* desc);

/* Workspace bytes: which = 0 forward, 1 backward.  The workspace must be
 * 256-byte aligned, the checkpoints 16-byte. */
int64_t mvm_seq_scan_workspace_bytes(const mvm_seq_scan_desc* desc, int which);

/*
 * y_t = (sum_n C_t[n] h_t[n] + D u_t) * silu(z_t),
 * h_t[n] = exp(delta_t A[n]) h_{t-1}[n] + delta_t B_t[n] u_t.
 * A (dim, dstate), Dv and delta_bias (dim) float32.  delta_bias, z (no gate),
 * h0 (zero), h1 (not stored) and ckpt (no backward) may be NULL.
 */
int mvm_seq_scan_fwd(const mvm_seq_scan_desc* desc, const void* u, const void* delta,
                     const float* delta_bias, const float* A, const void* Bm, const void* Cm,
                     const float* Dv, const void* z, const float* h0, float* h1, void* y,
                     float* ckpt, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Gradients for dy (y_stride rows) and dh1 (may be NULL: zero).  slots and
 * fresh must be NULL.  du, ddelta, dz (tokens, dim) and dB, dC (tokens,
 * dstate) are contiguous, in the types of their primals; dA (of A_log with
 * a_is_log), dD, ddelta_bias and dh0 (not dh1's buffer) float32.  All are written in full;
 * ddelta_bias may be NULL, dz is NULL without z, dh0 may be NULL.
 */
int mvm_seq_scan_bwd(const mvm_seq_scan_desc* desc, const void* u, const void* delta,
                     const float* delta_bias, const float* A, const void* Bm, const void* Cm,
                     const float* Dv, const void* z, const float* ckpt, const void* dy,
                     const float* dh1, void* du, void* ddelta, float* ddelta_bias, float* dA,
                     void* dB, void* dC, float* dD, void* dz, float* dh0, void* workspace,
                     size_t workspace_bytes, void* stream);

/* One token for each sequence (tokens == nseq, offsets NULL, seqlen 1): the
 * states advance in place; a row whose slot is outside [0, state_rows) gets
 * y = 0.  `fresh` is honoured. */
int mvm_seq_scan_step(const mvm_seq_scan_desc* desc, const void* u, const void* delta,
                      const float* delta_bias, const float* A, const void* Bm, const void* Cm,
                      const float* Dv, const void* z, float* states, void* y, void* stream);

int mvm_seq_conv_validate(const mvm_seq_conv_desc* desc);

/* Workspace bytes of mvm_seq_conv_bwd (256-byte aligned). */
int64_t mvm_seq_conv_workspace_bytes(const mvm_seq_conv_desc* desc);

/* y = silu(bias + causal depthwise conv(x)); w (dim, kwidth) and bias (dim)
 * float32.  c0 (zero), c1 (not stored) and bias (zero) may be NULL. */
int mvm_seq_conv_fwd(const mvm_seq_conv_desc* desc, const void* x, const float* w,
                     const float* bias, const void* c0, void* c1, void* y, void* stream);

/* Gradients for dy (y_stride rows) and dc1 (may be NULL: zero).  slots and
 * fresh must be NULL.  dx (tokens, dim) and dc0 (nseq, kwidth - 1, dim; may be
 * NULL) in the activations' type, dw and dbias (may be NULL) float32. */
int mvm_seq_conv_bwd(const mvm_seq_conv_desc* desc, const void* x, const float* w,
                     const float* bias, const void* c0, const void* dy, const void* dc1, void* dx,
                     float* dw, float* dbias, void* dc0, void* workspace, size_t workspace_bytes,
                     void* stream);

/* One token for each sequence, the states advanced in place (see
 * mvm_seq_scan_step). */
int mvm_seq_conv_step(const mvm_seq_conv_desc* desc, const void* x, const float* w,
                      const float* bias, void* states, void* y, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MVM_SEQ_H */
