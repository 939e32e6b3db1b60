// Host-side declarations of the learning operators' launchers. Every launcher enqueues its kernels on `stream` and
// returns without waiting; the arguments are checked by the entry points (kgx_learn.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <cstddef>

#include "kgx.h"

namespace kgx {

size_t policy_loss_workspace(int rows, int columns);
void launch_policy_loss(const kg_policy_loss_args& a, hipStream_t s);

// The preference loss's per-row and per-pair results between its kernels, in one workspace: row t's log-probability of its
// label, the softmax's maximum and reciprocal sum, and the factor of its gradient.
struct PrefRow {
  double logp;
  float top, inv_sum;
};
size_t preference_loss_workspace(int rows);
void launch_preference_loss(const kg_preference_loss_args& a, hipStream_t s);

// The AdamW step over `count` tensors, and the moments as numbers.
void launch_adamw(int count, const kg_adamw_tensor* tensors, const kg_adamw_state& state, const kg_adamw_values_t& values,
                  const kg_adamw_values_t* device_values, hipStream_t s);
void launch_adamw_moments(long long blocks, const kg_adamw_state& state, int type, void* m, void* root, hipStream_t s);

// Group norm: how many workgroups share a batch row's points, and the workspace that this asks for.
int group_norm_splits(int batch, int points, int channels);
size_t group_norm_workspace(int batch, int points, int channels, int groups, bool backward);
bool group_norm_fits(const kg_group_norm_args& a);  // its launches' threads fit 32 bits
void launch_group_norm(const kg_group_norm_args& a, hipStream_t s);
void launch_group_norm_backward(const kg_group_norm_args& a, hipStream_t s);

size_t distill_loss_workspace(int rows, int columns, int k);
void launch_distill_loss(const kg_distill_loss_args& a, hipStream_t s);

// Layer norm: the backward pass's sums over parts of the rows.
size_t layer_norm_workspace(int rows, int channels);
void launch_layer_norm(const kg_layer_norm_args& a, hipStream_t s);
void launch_layer_norm_backward(const kg_layer_norm_args& a, hipStream_t s);

// The embedding's backward pass: the tokens sorted, and the sums of runs over several ranges of them.
size_t embedding_backward_workspace(int count, int vocab, int channels);
void launch_embedding(const kg_embedding_args& a, hipStream_t s);
void launch_embedding_backward(const kg_embedding_args& a, hipStream_t s);

}  // namespace kgx
