// short_inst.hip -- the launches of linear attention with a decay over at most 32 tokens for ONE element type (policy_type.h).
#include "policy_type.h"
#include "decay_short.h"

namespace {

template <int DK, int DV, int FIT, bool BACK> hipError_t launch_sized(const ShortArgs& p, hipStream_t st) {
  constexpr int LDS = (int)sizeof(ShortLds<DK, DV, BACK>);
  auto kern = k_decay_short<T, DK, DV, FIT, BACK>;
  static std::atomic<unsigned long long> asked{0};
  if (hipError_t e = allow_lds(kern, LDS, asked); e != hipSuccess) return e;
  const long long rows = p.d.batch * p.d.heads;  // (below 2^24, and up to 512 threads each: below 2^32 in all is for the caller to check)
  if (rows * short_threads(DK, DV) > 0xffffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)rows), dim3(short_threads(DK, DV)), LDS, st, p);
  return hipGetLastError();
}

template <int DK, int DV, bool BACK> hipError_t launch_pass(const ShortArgs& p, hipStream_t st) {
  constexpr int V = Elem<T>::VEC;
  if (p.d.dk == DK && p.d.dv == DV) return launch_sized<DK, DV, FIT_FULL, BACK>(p, st);
  return p.d.dk % V || p.d.dv % V ? launch_sized<DK, DV, FIT_ANY, BACK>(p, st) : launch_sized<DK, DV, FIT_CHUNKS, BACK>(p, st);
}

template <int DK, bool BACK> hipError_t launch_dv(const ShortArgs& p, hipStream_t st) {
  return p.d.dv <= 32 ? launch_pass<DK, 32, BACK>(p, st) : p.d.dv <= 64 ? launch_pass<DK, 64, BACK>(p, st) : launch_pass<DK, 128, BACK>(p, st);
}

template <bool BACK> hipError_t launch(const ShortArgs& p, hipStream_t st) {
  return p.d.dk <= 32 ? launch_dv<32, BACK>(p, st) : p.d.dk <= 64 ? launch_dv<64, BACK>(p, st) : launch_dv<128, BACK>(p, st);
}

}  // namespace

hipError_t POLICY_NAME(mjlab_launch_short_forward)(const mjlab_decay_t* d, hipStream_t st) {
  ShortArgs p = {};
  p.d = *d;
  return launch<false>(p, st);
}

hipError_t POLICY_NAME(mjlab_launch_short_backward)(const mjlab_decay_grad_t* g, hipStream_t st) {
  ShortArgs p = {};
  p.d = g->f; p.go = g->d_out; p.dq = g->dq; p.dk = g->dk; p.dv = g->dv; p.d_state_out = g->d_state_out; p.d_state = g->d_state;
  return launch<true>(p, st);
}
