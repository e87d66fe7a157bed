// policy_type.h -- the element type of this translation unit: -DMJLAB_POLICY_DTYPE=<0 f32 | 1 f16 | 2 bf16> (mjlab_amd/native.py).
#pragma once
#include "policy_common.h"
#include "policy_launch.h"

#if MJLAB_POLICY_DTYPE == 0
using T = float;
#define POLICY_NAME(x) x##_f32
#elif MJLAB_POLICY_DTYPE == 1
using T = _Float16;
#define POLICY_NAME(x) x##_f16
#else
using T = __bf16;
#define POLICY_NAME(x) x##_bf16
#endif

constexpr int CUS = 256;
constexpr long long MAX_BLOCKS = (1LL << 24) - 1;  // of 256 threads: a launch counts its threads in 32 bits

// Dynamic LDS beyond 64 KB has to be asked for, per device and kernel.
template <typename K> inline hipError_t allow_lds(K* kern, int bytes) {
  return bytes > 64 * 1024 ? hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) : hipSuccess;
}
