// decay_inst.hip -- the launches of linear attention with a decay for ONE element type (policy_type.h).
#include "policy_type.h"
#include "decay.h"

namespace {

struct Split {
  int segments, seg_chunks;
};

// Segments per sequence: one where the sequences fill the device (a workgroup each), else as many as give it a workgroup per CU (two for small
// heads), of four chunks at least: the first pass reads two of the operands again and moves R through memory once per segment.
Split split(const mjlab_decay_t* d) {
  const int C = decay_chunk<T>(d->dk > 64 && d->dv > 64);
  const long long chunks = (d->length + C - 1) / C, rows = d->batch * d->heads, least = d->dk < d->dv ? d->dk : d->dv, most_d = d->dk < d->dv ? d->dv : d->dk;
  const bool alone = DecayCfg<T, false>::N > 1 ? least > 32 || most_d > 64 : most_d > 64 && (least > 32 || DecayCfg<T, false>::P > 1);  // whether LDS holds one workgroup per CU, or two
  const long long slots = alone ? CUS : 2 * CUS;
  if (2 * rows >= slots || chunks < 8) return {1, (int)chunks};
  const long long want = slots / rows, most = chunks / 4, s = want < most ? want : most;
  const long long per = (chunks + s - 1) / s;
  return {(int)((chunks + per - 1) / per), (int)per};
}

long long up256(long long x) { return (x + 255) & ~255LL; }
long long state_bytes(const mjlab_decay_t* d, const Split& s) { return up256(d->batch * d->heads * (s.segments - 1) * (long long)d->dk * d->dv * 4); }

template <int DA, int DC, int FIT, bool EXACT> hipError_t launch_sized(const DecayPass& p, long long rows, hipStream_t st) {
  constexpr int LDS = (int)sizeof(DecayLds<T, DA, DC, false, EXACT>), LDS_FIRST = (int)sizeof(DecayLds<T, DA, DC, true, EXACT>);
  static std::atomic<unsigned long long> asked{0}, asked_first{0};
  hipError_t e;
  if (rows * p.segments * decay_threads<T>(DA, DC) > 0xffffffffLL) return hipErrorInvalidValue;
  if (p.segments > 1 && !p.seg_given) {
    auto first = k_decay_chunks<T, DA, DC, FIT, true, EXACT>;
    if ((e = allow_lds(first, LDS_FIRST, asked_first)) != hipSuccess) return e;
    hipLaunchKernelGGL(first, dim3((unsigned)(rows * (p.segments - 1))), dim3(decay_threads<T>(DA, DC)), LDS_FIRST, st, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL(k_decay_scan<T>, dim3((unsigned)(rows * ((p.da * p.dc + 255) / 256))), dim3(256), 0, st, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  auto kern = k_decay_chunks<T, DA, DC, FIT, false, EXACT>;
  if ((e = allow_lds(kern, LDS, asked)) != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)(rows * p.segments)), dim3(decay_threads<T>(DA, DC)), LDS, st, p);
  return hipGetLastError();
}

template <int DA, int DC, bool EXACT> hipError_t launch_fit(const DecayPass& p, long long rows, hipStream_t st) {
  constexpr int V = Elem<T>::VEC;
  if (p.da == DA && p.dc == DC) return launch_sized<DA, DC, FIT_FULL, EXACT>(p, rows, st);
  return p.da % V || p.dc % V ? launch_sized<DA, DC, FIT_ANY, EXACT>(p, rows, st) : launch_sized<DA, DC, FIT_CHUNKS, EXACT>(p, rows, st);
}

template <int DA, int DC> hipError_t launch_pass(const DecayPass& p, long long rows, hipStream_t st) {
  if (p.state_out && DecayCfg<T, true>::W != DecayCfg<T, false>::W) return launch_fit<DA, DC, DecayCfg<T, true>::W != DecayCfg<T, false>::W>(p, rows, st);
  return launch_fit<DA, DC, false>(p, rows, st);
}

template <int DA> hipError_t launch_dc(const DecayPass& p, long long rows, hipStream_t st) {
  return p.dc <= 32 ? launch_pass<DA, 32>(p, rows, st) : p.dc <= 64 ? launch_pass<DA, 64>(p, rows, st) : launch_pass<DA, 128>(p, rows, st);
}

// out = the pass over a, b (heads of da) and c (of dc); see decay.h
hipError_t launch(const mjlab_decay_t* d, const mjlab_decay_rows_t& a, const mjlab_decay_rows_t& b, const mjlab_decay_rows_t& c, const mjlab_decay_rows_t& out, int da,
                  int dc, bool reverse, const float* state_in, bool turned, float* state_out, hipStream_t st, const void* segments = nullptr) {
  const Split s = split(d);
  DecayPass p = {};
  p.a = a.p; p.a_b = a.batch; p.a_t = a.time; p.a_h = a.head;
  p.b = b.p; p.b_b = b.batch; p.b_t = b.time; p.b_h = b.head;
  p.c = c.p; p.c_b = c.batch; p.c_t = c.time; p.c_h = c.head;
  p.out = (void*)out.p; p.o_b = out.batch; p.o_t = out.time; p.o_h = out.head;
  p.log_decay = d->log_decay;
  p.state_in = state_in; p.in_r = turned ? 1 : dc; p.in_c = turned ? da : 1; p.state_out = state_out;
  p.reset = d->reset; p.reset_bytes = d->reset_bytes; p.reset_b = d->reset_batch; p.reset_t = d->reset_time;
  p.heads = d->heads; p.da = da; p.dc = dc; p.e0 = reverse ? 0 : 1; p.reverse = reverse; p.segments = s.segments; p.seg_chunks = s.seg_chunks;
  p.length = d->length; p.lengths = d->lengths;
  p.ps = d->scale; p.is = reverse ? 1.f : d->scale; p.us = reverse ? d->scale : 1.f;
  p.seg_given = segments != nullptr;
  p.seg_state = segments ? (float*)segments : (float*)d->workspace; p.seg_factor = (float*)((char*)d->workspace + state_bytes(d, s));
  const long long rows = d->batch * d->heads;
  return da <= 32 ? launch_dc<32>(p, rows, st) : da <= 64 ? launch_dc<64>(p, rows, st) : launch_dc<128>(p, rows, st);
}

template <int LPR> hipError_t launch_step(const mjlab_decay_t* d, hipStream_t st) {
  hipLaunchKernelGGL((k_decay_step<T, LPR>), dim3((unsigned)(d->batch * d->heads)), dim3(256), 0, st, *d);
  return hipGetLastError();
}

}  // namespace

long long POLICY_NAME(mjlab_decay_bytes)(const mjlab_decay_t* d) {
  const Split s = split(d);
  return s.segments > 1 ? state_bytes(d, s) + up256(d->batch * d->heads * (s.segments - 1) * 4) : 0;
}

hipError_t POLICY_NAME(mjlab_launch_decay_forward)(const mjlab_decay_t* d, hipStream_t st) {
  if (d->length <= 32) return POLICY_NAME(mjlab_launch_short_forward)(d, st);
  return launch(d, d->q, d->k, d->v, d->o, d->dk, d->dv, false, d->state, false, d->state_out, st);
}

hipError_t POLICY_NAME(mjlab_launch_decay_backward)(const mjlab_decay_grad_t* g, hipStream_t st) {
  const mjlab_decay_t* d = &g->f;
  if (d->length <= 32) return POLICY_NAME(mjlab_launch_short_backward)(g, st);
  hipError_t e;
  // dq's R is the forward pass's transposed, dk's is dv's: the states of their segments serve both
  if (g->dq.p && (e = launch(d, g->d_out, d->v, d->k, g->dq, d->dv, d->dk, false, d->state, true, nullptr, st, g->segments)) != hipSuccess) return e;
  if (g->dv.p && (e = launch(d, d->k, d->q, g->d_out, g->dv, d->dk, d->dv, true, g->d_state_out, false, g->d_state, st)) != hipSuccess) return e;
  if (g->dk.p && (e = launch(d, d->v, g->d_out, d->q, g->dk, d->dv, d->dk, true, g->d_state_out, true, nullptr, st, g->dv.p ? d->workspace : nullptr)) != hipSuccess) return e;
  return hipSuccess;
}

hipError_t POLICY_NAME(mjlab_launch_decay_step)(const mjlab_decay_t* d, hipStream_t st) {
  return d->dv <= 32 ? launch_step<8>(d, st) : d->dv <= 64 ? launch_step<16>(d, st) : launch_step<32>(d, st);
}
