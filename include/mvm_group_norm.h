/*
 * mvm_group_norm.h -- C ABI of the group norm with an activation, channels last
 * (libmvm_scan.so): beside the LayerNorm of mvm_norm.h (the reference's only
 * norm, mlx_vision_mamba/mamba_block.py:201-205), the norm over the heads of a
 * recurrent mixer (positions = 1, groups = heads) and of channels-last maps.
 *
 * x is (batch, positions, channels); channel c belongs to group c / (channels /
 * groups).  Over the positions x channels / groups values of a sample's group
 *
 *   mean, var (biased);   n = (x - mean) / sqrt(var + eps) * weight[c] + bias[c]
 *   y = act(n) * silu(z)           act: n, or silu(n); without z: no factor
 *
 * Conventions are those of mvm_scan.h (status codes, mvm_last_error,
 * caller-owned buffers and workspace, host-side validation, deterministic
 * results).  x, z, y and their gradients are float32 or bfloat16; weight, bias
 * and their gradients, and the statistics, float32.  Rows of channels are
 * contiguous, batch * positions of them a stride apart.  weight (ones), bias
 * (zeros) and z may be NULL.
 */
#ifndef MVM_GROUP_NORM_H
#define MVM_GROUP_NORM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MVM_GROUP_NORM_MAX_CHANNELS 65536

typedef struct mvm_group_norm_desc {
  int64_t batch;       /* >= 0 */
  int64_t positions;   /* >= 0 */
  int64_t channels;    /* 1..MVM_GROUP_NORM_MAX_CHANNELS */
  int64_t groups;      /* divides channels */
  int64_t x_stride;    /* of rows, >= 0 */
  int64_t z_stride;    /* the same; 0 without z */
  float eps;           /* >= 0 */
  int32_t dtype;       /* x, z, y and their gradients */
  int32_t silu;        /* 1: act = silu */
  int32_t reserved;    /* 0 */
} mvm_group_norm_desc;

/* Validates a descriptor without touching the GPU. */
int mvm_group_norm_validate(const mvm_group_norm_desc* desc);

/* Workspace bytes: which = 0 forward, 1 backward (256-byte aligned). */
int64_t mvm_group_norm_workspace_bytes(const mvm_group_norm_desc* desc, int which);

/* y is contiguous.  stats: batch * groups pairs (mean, 1 / sqrt(var + eps)) for
 * the backward, may be NULL. */
int mvm_group_norm_fwd(const mvm_group_norm_desc* desc, const void* x, const float* weight,
                       const float* bias, const void* z, void* y, float* stats, void* workspace,
                       size_t workspace_bytes, void* stream);

/* Gradients for dy (contiguous); dx and dz (NULL without z) are contiguous;
 * dweight and dbias may be NULL.  All are written in full. */
int mvm_group_norm_bwd(const mvm_group_norm_desc* desc, const void* x, const float* weight,
                       const float* bias, const void* z, const float* stats, const void* dy,
                       void* dx, float* dweight, float* dbias, void* dz, void* workspace,
                       size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MVM_GROUP_NORM_H */
