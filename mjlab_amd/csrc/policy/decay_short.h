// decay_short.h -- linear attention with a decay over at most 32 tokens: what an update over stored rollouts is made of (24 steps of thousands of
// environments).  Everything of a sequence and head fits one workgroup at once, so each array is read once and the backward pass is one kernel:
//   A_ij = w_ij q_i . k_j,  B_ij = w_ij do_i . v_j   with w_ij = scale decay^(i-j) for j <= i of one episode
//   o_i  = sum_j A_ij v_j + enter_i S0^T q_i         S_T = through S0 + sum_j leave_j k_j v_j^T
//   dq_i = sum_j B_ij k_j + enter_i S0 do_i          dk_j = sum_i B_ij q_i + leave_j dS_T v_j
//   dv_j = sum_i A_ij do_i + leave_j dS_T^T k_j      dS0 = through dS_T + sum_i enter_i q_i do_i^T
// enter_i = scale decay^(i+1) in the first episode, leave_j = decay^(n-1-j) in the last, through = decay^n if they are one.
// Bound by memory, chiefly the states' bytes, so all types are multiplied as floats; the states go from memory to the matrix cores' registers.
// (1024 sequences of 24 steps, 4 heads of 64, float, forward and backward with states: the chunk kernel 285 us, this one 159 us.)
#pragma once
#include "decay.h"

constexpr int SHORT = 32;

template <int DK, int DV, bool BACK> struct ShortLds {
  static constexpr int LK = DK + 4, LV = DV + 4, LP = SHORT + 4;
  float q[SHORT * LK], k[SHORT * LK], v[SHORT * LV], go[BACK ? SHORT * LV : 4], a[SHORT * LP], b[BACK ? SHORT * LP : 4];
  float enter[SHORT], leave[SHORT];
  int odd[8];
};

constexpr int short_threads(int dk, int dv) { return 4 * (dk > dv ? dk : dv); }  // a wave per 16 columns

struct ShortArgs {
  mjlab_decay_t d;
  mjlab_decay_rows_t go, dq, dk, dv;
  const float* d_state_out;
  float* d_state;
};

template <typename T, int DK, int DV, int FIT, bool BACK> __global__ __launch_bounds__(short_threads(DK, DV)) void k_decay_short(const ShortArgs p) {
  using S = ShortLds<DK, DV, BACK>;
  constexpr bool FULL = FIT == FIT_FULL;
  constexpr int NT = short_threads(DK, DV), NW = NT / 64, V = Elem<T>::VEC, LK = S::LK, LV = S::LV, LP = S::LP, KT = DK / 16, VT = DV / 16;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  S& s = *(S*)lds;
  const mjlab_decay_t& d = p.d;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row4 = (lane >> 4) * 4, colx = lane & 15;
  const long long sh = blockIdx.x, seq = sh / d.heads;
  const int head = (int)(sh % d.heads);
  float g2 = d.log_decay[head] * 1.44269504f;
  g2 = g2 < -1e30f ? -1e30f : g2;  // (finite: its power 0 is 1)
  auto power = [&](int n) { return __builtin_amdgcn_exp2f(n * g2); };
  int n = (int)d.length;
  if (d.lengths) { const int l = d.lengths[seq]; n = l < 0 ? 0 : (l < n ? l : n); }

  // The rows of the tokens, all on their way at once; to LDS as floats below
  constexpr int PK = DK / V, PV = DV / V, NK = (SHORT * PK + NT - 1) / NT, NV = (SHORT * PV + NT - 1) / NT;  // chunks per row, per thread
  auto fetch = [&](auto& c, int per, int real, const mjlab_decay_rows_t& r) {
    const T* base = (const T*)r.p + seq * r.batch + head * r.head;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(c) / sizeof(c[0])); ++i) {
      const int u = tid + i * NT, row = u / per, col = u % per * V;
      c[i] = Chunk<T>{};
      if (row < n) c[i] = load_row<T, FIT>(base + row * r.time + col, col, real);
    }
  };
  Chunk<T> cq[NK], ck[NK], cv[NV], cg[BACK ? NV : 1];
  fetch(cq, PK, d.dk, d.q);
  fetch(ck, PK, d.dk, d.k);
  fetch(cv, PV, d.dv, d.v);
  if constexpr (BACK) fetch(cg, PV, d.dv, p.go);

  // The states' elements that this wave will multiply, likewise where registers allow it.  A state's rows (or, TURNED, columns) from 16 wave on.
  const int r0 = wave * 16;
  const bool has_k = wave < KT, has_v = wave < VT;
  auto at = [&](const float* m, int r, int c) { return FULL || (r < d.dk && c < d.dv) ? m[r * d.dv + c] : 0.f; };
  auto state_frag = [&](const float* m, bool turned, int g) {
    f32x4 f;
    if (!turned && FIT != FIT_ANY) f = __builtin_bit_cast(f32x4, load_row<float, FIT>(m + (r0 + colx) * d.dv + g * 16 + row4, g * 16 + row4, r0 + colx < d.dk ? d.dv : 0));
    else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = turned ? at(m, g * 16 + row4 + e, r0 + colx) : at(m, r0 + colx, g * 16 + row4 + e);
    }
    return f;
  };
  const float* st = d.state ? d.state + sh * d.dk * d.dv : nullptr;
  const float* ds = BACK && p.d_state_out ? p.d_state_out + sh * d.dk * d.dv : nullptr;
  constexpr bool EARLY = BACK ? DK <= 64 && DV <= 64 : true;
  f32x4 fx[EARLY ? (BACK ? VT : KT) : 1], fy[EARLY && BACK ? VT : 1], fz[EARLY && BACK ? KT : 1], acc_state[VT];
  auto early = [&](auto& f, const float* m, bool turned) {
#pragma unroll
    for (int g = 0; g < (int)(sizeof(f) / sizeof(f[0])); ++g) f[g] = state_frag(m, turned, g);
  };
  const bool want_x = BACK ? has_k && p.dq.p && st : has_v && st, want_y = BACK && has_k && p.dk.p && ds, want_z = BACK && has_v && p.dv.p && ds;
  if constexpr (EARLY) {
    if (want_x) early(fx, st, !BACK);
    if (BACK && want_y) early(fy, ds, false);
    if (BACK && want_z) early(fz, ds, true);
  }
  const float* from = BACK ? ds : st;  // what the state that this pass writes comes from
  float* to_state = BACK ? p.d_state : d.state_out;
  const bool want_state = has_k && to_state;
#pragma unroll
  for (int c = 0; c < VT; ++c) acc_state[c] = f32x4{};
  auto early_state = [&]() {
#pragma unroll
    for (int c = 0; c < VT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc_state[c][e] = at(from, r0 + row4 + e, c * 16 + colx);
  };
  if (EARLY && want_state && from) early_state();

  bool odd = false;
  auto bring = [&](float* to, int ld, int per, const auto& c) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(c) / sizeof(c[0])); ++i) {
      const int u = tid + i * NT, row = u / per, col = u % per * V;
      if (row >= SHORT) continue;
      float x[V];
#pragma unroll
      for (int e = 0; e < V; ++e) { x[e] = (float)c[i].e[e]; odd |= not_finite(x[e]); }
#pragma unroll
      for (int e = 0; e < V; e += 4) *(f32x4*)(to + row * ld + col + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
    }
  };

  // bit i: token i is the first of an episode
  unsigned cuts = 0;
  if (d.reset) {
    bool f = false;
    if (lane < n) {
      const long long i = seq * d.reset_batch + lane * d.reset_time;
      f = d.reset_bytes == 1 ? ((const unsigned char*)d.reset)[i] != 0 : ((const int*)d.reset)[i] != 0;
    }
    cuts = (unsigned)__ballot(f);
  }
  auto episode = [&](int i) { return __popc(cuts & ((2u << i) - 1)); };
  const int e_last = n ? episode(n - 1) : 0;
  const bool carries = e_last == 0;
  const float through = power(n);
  if (tid < SHORT) {
    s.enter[tid] = tid < n && episode(tid) == 0 ? d.scale * power(tid + 1) : 0.f;
    s.leave[tid] = tid < n && episode(tid) == e_last ? power(n - 1 - tid) : 0.f;
  }
  bring(s.q, LK, PK, cq);
  bring(s.k, LK, PK, ck);
  bring(s.v, LV, PV, cv);
  if constexpr (BACK) bring(s.go, LV, PV, cg);
  const bool mine = __ballot(odd) != 0;
  if (lane == 0) s.odd[wave] = mine;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) any |= s.odd[i];
  const bool by_term = __builtin_amdgcn_readfirstlane(any) != 0;  // a zero weight times infinity would be NaN: term by term then
  auto linked = [&](int i, int j) { return j <= i && i < n && episode(j) == episode(i); };

  // the pairs, [i][j]: tiles (0, 0), (1, 0), (1, 1); (0, 1) is never read
  auto pairs = [&](float* to, const float* x, const float* y, int ld, int groups, int skip) {  // x rows i, y rows j
    for (int u = (wave + NW - skip % NW) % NW; u < 3; u += NW) {
      const int ti = (u + 1) / 2, tj = u / 2, i = ti * 16 + colx;
      f32x4 acc = {};
#pragma unroll 4
      for (int g = 0; g < groups; ++g) {
        const f32x4 fy = *(const f32x4*)(y + (tj * 16 + colx) * ld + g * 16 + row4), fx = *(const f32x4*)(x + i * ld + g * 16 + row4);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = mma16(fy[e], fx[e], acc);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = tj * 16 + row4 + e;
        acc[e] = linked(i, j) ? d.scale * power(i - j) * acc[e] : 0.f;
      }
      *(f32x4*)(to + i * LP + tj * 16 + row4) = acc;
    }
  };
  pairs(s.a, s.q, s.k, LK, KT, 0);
  if constexpr (BACK) pairs(s.b, s.go, s.v, LV, VT, 3);

  // x[t] (columns: tokens of tile t, rows: 16 wave ..) = factor_t * M y_t, y the tokens' rows in LDS; f: the fragments of M that are here already
  auto state_part = [&](f32x4 (&x)[2], const auto& f, const float* m, bool turned, const float* y, int ld, int groups, const float* factor) {
    f32x4 acc[2] = {};
#pragma unroll
    for (int g = 0; g < groups; ++g) {
      const f32x4 fm = EARLY ? f[EARLY ? g : 0] : state_frag(m, turned, g);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4 fy = *(const f32x4*)(y + (t * 16 + colx) * ld + g * 16 + row4);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t] = mma16(fm[e], fy[e], acc[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float w = factor[t * 16 + colx];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[t][e] = w == 0.f ? 0.f : w * acc[t][e];
    }
  };
  // x[t] += sum over tokens u of W(token of t, u) y_u;  W is w[t][u] (earlier u), or TURNED w[u][t] (later u)
  auto pair_part = [&](f32x4 (&x)[2], const float* w, bool turned, int row0, const float* y, int ld) {
    if (!by_term) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        f32x4 fy;
#pragma unroll
        for (int e = 0; e < 4; ++e) fy[e] = y[(g * 16 + row4 + e) * ld + row0 + colx];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (turned ? g < t : g > t) continue;
          f32x4 fw;
          if (turned) {
#pragma unroll
            for (int e = 0; e < 4; ++e) fw[e] = w[(g * 16 + row4 + e) * LP + t * 16 + colx];
          } else fw = *(const f32x4*)(w + (t * 16 + colx) * LP + g * 16 + row4);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[t] = mma16(fy[e], fw[e], x[t]);
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int i = t * 16 + colx;
        for (int u = 0; u < n; ++u)
          if (turned ? linked(u, i) : linked(i, u)) {
            const float f = turned ? w[u * LP + i] : w[i * LP + u];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[t][e] += f * y[u * ld + row0 + row4 + e];
          }
      }
    }
  };
  auto put_rows = [&](const f32x4 (&x)[2], const mjlab_decay_rows_t& r, int row0, int real) {
    T* base = (T*)r.p + seq * r.batch + head * r.head + row0 + row4;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int i = t * 16 + colx;
      if (i >= d.length) continue;  // (behind the sequence's end x is 0)
      T o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (T)x[t][e];
      T* to = base + i * r.time;
      if (FULL || row0 + row4 + 4 <= real) __builtin_memcpy(to, o, sizeof(o));
      else if (FIT == FIT_ANY) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (row0 + row4 + e < real) to[e] = o[e];
      }
    }
  };
  // the state that this pass writes (dk x dv) = through `from` + sum over tokens of weight_u x_u y_u^T, this wave's 16 rows of it
  auto put_state = [&](const float* x, const float* y, const float* weight) {
    f32x4 (&acc)[VT] = acc_state;
    if (!EARLY && from) early_state();
#pragma unroll
    for (int c = 0; c < VT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[c][e] = from && carries ? through * acc[c][e] : 0.f;
    if (!by_term) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int u = g * 16 + row4 + e;
          const float w = weight[u], fx = w == 0.f ? 0.f : w * x[u * LK + r0 + colx];
#pragma unroll
          for (int c = 0; c < VT; ++c) acc[c] = mma16(fx, y[u * LV + c * 16 + colx], acc[c]);
        }
    } else {
      for (int u = 0; u < n; ++u) {
        const float w = weight[u];
        if (w == 0.f) continue;
#pragma unroll
        for (int c = 0; c < VT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[c][e] += w * x[u * LK + r0 + row4 + e] * y[u * LV + c * 16 + colx];
      }
    }
    float* to = to_state + sh * d.dk * d.dv;
#pragma unroll
    for (int c = 0; c < VT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = r0 + row4 + e, k = c * 16 + colx;
        if (FULL || (r < d.dk && k < d.dv)) to[r * d.dv + k] = acc[c][e];
      }
  };

  f32x4 x[2] = {};
  if constexpr (!BACK) {
    if (want_x) state_part(x, fx, st, true, s.q, LK, KT, s.enter);
    if (want_state) put_state(s.k, s.v, s.leave);
    __syncthreads();
    if (has_v) {
      pair_part(x, s.a, false, r0, s.v, LV);
      put_rows(x, d.o, r0, d.dv);
    }
  } else {
    f32x4 y[2] = {}, z[2] = {};
    if (want_x) state_part(x, fx, st, false, s.go, LV, VT, s.enter);
    if (want_y) state_part(y, fy, ds, false, s.v, LV, VT, s.leave);
    if (want_z) state_part(z, fz, ds, true, s.k, LK, KT, s.leave);
    if (want_state) put_state(s.q, s.go, s.enter);
    __syncthreads();
    if (has_k && p.dq.p) {
      pair_part(x, s.b, false, r0, s.k, LK);
      put_rows(x, p.dq, r0, d.dk);
    }
    if (has_k && p.dk.p) {
      pair_part(y, s.b, true, r0, s.q, LK);
      put_rows(y, p.dk, r0, d.dk);
    }
    if (has_v && p.dv.p) {
      pair_part(z, s.a, true, r0, s.go, LV);
      put_rows(z, p.dv, r0, d.dv);
    }
  }
}
