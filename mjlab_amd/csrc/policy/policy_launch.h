// policy_launch.h -- the per-type launch functions that layer_inst.hip, decay_inst.hip and short_inst.hip define and policy.hip dispatches to.
#pragma once
#include <hip/hip_runtime.h>

#include "../../../include/mjlab_policy.h"

#define MJLAB_POLICY_DECLARE(T)                                                              \
  hipError_t mjlab_launch_layer_forward_##T(const mjlab_layer_t* f, hipStream_t st);         \
  int mjlab_layer_again_##T(const mjlab_layer_t* f);                                         \
  int mjlab_layer_tile_of_##T(const mjlab_layer_t* f, int product);                          \
  long long mjlab_layer_forward_bytes_##T(const mjlab_layer_t* f);                           \
  long long mjlab_layer_backward_bytes_##T(const mjlab_layer_grad_t* g);                     \
  hipError_t mjlab_launch_layer_backward_##T(const mjlab_layer_grad_t* g, hipStream_t st);   \
  long long mjlab_decay_bytes_##T(const mjlab_decay_t* d);                                   \
  hipError_t mjlab_launch_decay_forward_##T(const mjlab_decay_t* d, hipStream_t st);         \
  hipError_t mjlab_launch_decay_backward_##T(const mjlab_decay_grad_t* g, hipStream_t st);   \
  hipError_t mjlab_launch_short_forward_##T(const mjlab_decay_t* d, hipStream_t st);         \
  hipError_t mjlab_launch_short_backward_##T(const mjlab_decay_grad_t* g, hipStream_t st);   \
  hipError_t mjlab_launch_decay_step_##T(const mjlab_decay_t* d, hipStream_t st);
MJLAB_POLICY_DECLARE(f32)
MJLAB_POLICY_DECLARE(f16)
MJLAB_POLICY_DECLARE(bf16)
#undef MJLAB_POLICY_DECLARE
