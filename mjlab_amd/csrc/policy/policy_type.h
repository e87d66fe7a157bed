// policy_type.h -- the element type of this translation unit: -DMJLAB_POLICY_DTYPE=<0 f32 | 1 f16 | 2 bf16> (mjlab_amd/native.py).
#pragma once
#include <atomic>

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

// Dynamic LDS beyond 64 KB has to be asked for, once per device and kernel.
template <typename K> inline hipError_t allow_lds(K* kern, int bytes, std::atomic<unsigned long long>& asked) {
  if (bytes <= 64 * 1024) return hipSuccess;
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
  const unsigned long long bit = 1ULL << (dev & 63);
  if (asked.load(std::memory_order_relaxed) & bit) return hipSuccess;
  const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return e;
}
