// decay.h -- linear attention with a decay per head: chunks of tokens on the matrix cores, and the recurrence for one token.
//
// One pass, out_p = ps * sum over pairs j <= p of decay^(p-j) (a_p . b_j) c_j + is * decay^(p+e0) a_p R, carries R (da x dc, 32 bits, in the
// accumulators) from chunk to chunk: R <- decay^n R + us * sum over j of decay^(n-e0-j) b_j c_j^T.  The forward pass and the three gradients are
// this pass with other operands (o: a b c = q k v; dq: do v k; and from the last token to the first dk: v do q, dv: k q do, where the
// carry holds one more decay, e0 = 0).  A link between neighbouring tokens that a reset cuts takes its pairs and the carry out.
// Within a chunk the pairs are two small products, P = a b^T (weighted) and P c; powers of the decay are those of differences >= 0 only, so
// nothing overflows.  A sequence is split into segments when there are few sequences: a first pass forms each segment's own contribution to R, a
// scan along the segments turns these into the R each segment starts from, the second pass does the rest.
#pragma once
#include "policy_common.h"

struct DecayPass {
  const void *a, *b, *c;
  void* out;
  long long a_b, a_t, a_h, b_b, b_t, b_h, c_b, c_t, c_h, o_b, o_t, o_h;  // strides: sequence, token, head
  const float* log_decay;
  const float* state_in;  // or NULL
  float* state_out;       // or NULL
  int in_r, in_c;         // strides of the rows (da) and columns (dc) of state_in; state_out is (da, dc) dense
  const void* reset;
  int reset_bytes, heads, da, dc, e0, reverse, segments, seg_chunks;
  long long reset_b, reset_t, length;
  const int* lengths;
  float ps, is, us;
  float *seg_state, *seg_factor;  // (sequences * heads, segments - 1, da, dc), (sequences * heads, segments - 1)
};

// What the matrix cores read: bf16 as it is; float, and fp16 turned into float (whose products and sums of keys and values may leave fp16's range).
template <typename T> struct DecayCfg {
  using L = float;
  static constexpr int C = 32, KS = 4, PAD = 4;  // tokens per chunk, k per matrix instruction, padding of LDS rows
};
template <> struct DecayCfg<__bf16> {
  using L = __bf16;
  static constexpr int C = 64, KS = 32, PAD = 8;
};

__device__ __forceinline__ f32x4 mma16(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// fragments of 16 rows (or columns) x KS of k: k contiguous / k the row index of the tile
__device__ __forceinline__ s16x8 frag_kc(const __bf16* s, int ld, int r0, int k0, int lane) { return *(const s16x8*)(s + (r0 + (lane & 15)) * ld + k0 + (lane >> 4) * 8); }
__device__ __forceinline__ float frag_kc(const float* s, int ld, int r0, int k0, int lane) { return s[(r0 + (lane & 15)) * ld + k0 + (lane >> 4)]; }
__device__ __forceinline__ s16x8 frag_kr(const __bf16* s, int ld, int r0, int k0, int lane) {
  typedef __attribute__((address_space(3))) s16x4 lds_s4;
  const int t = lane & 15;
  const __bf16* q = s + (k0 + (lane >> 4) * 8 + (t >> 2)) * ld + r0 + (t & 3) * 4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)q);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(q + 4 * ld));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ float frag_kr(const float* s, int ld, int r0, int k0, int lane) { return s[(k0 + (lane >> 4)) * ld + r0 + (lane & 15)]; }

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

__device__ __forceinline__ bool reset_at(const DecayPass& p, long long seq, long long t) {
  const long long i = seq * p.reset_b + t * p.reset_t;
  return p.reset_bytes == 1 ? ((const unsigned char*)p.reset)[i] != 0 : ((const int*)p.reset)[i] != 0;
}

template <typename T, int DA, int DC> struct DecayLds {
  using L = typename DecayCfg<T>::L;
  static constexpr int C = DecayCfg<T>::C, PAD = DecayCfg<T>::PAD, LA = DA + PAD, LC = DC + PAD, LP = C + PAD;
  L a[C * LA], b[C * LA], bw[C * LA], c[C * LC], p[C * LP], r[DC * LA];
  float power[C + 1];
};

// 256 threads per (sequence, head, segment).  STATE: the first pass of a split sequence, the segment's contribution to R alone.
template <typename T, int DA, int DC, bool STATE> __global__ __launch_bounds__(256) void k_decay_chunks(const DecayPass p) {
  using Cfg = DecayCfg<T>;
  using L = typename Cfg::L;
  using S = DecayLds<T, DA, DC>;
  constexpr int C = Cfg::C, KS = Cfg::KS, LA = S::LA, LC = S::LC, LP = S::LP, V = Elem<T>::VEC;
  constexpr int CT = C / 16, NO = CT * (DC / 16) / 4, NR = (DA / 16) * (DC / 16) / 4;  // 16 x 16 tiles per wave: of out, of R
  constexpr int NA = (C * DA / V + 255) / 256, NC = (C * DC / V + 255) / 256;          // 16-byte chunks per thread
  extern __shared__ __attribute__((aligned(16))) char lds[];
  S& s = *(S*)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row4 = (lane >> 4) * 4, colx = lane & 15;
  const int segs = STATE ? p.segments - 1 : p.segments;
  const long long sh = blockIdx.x / segs, seq = sh / p.heads;
  const int seg = (int)(blockIdx.x % segs), head = (int)(sh % p.heads);
  const float g = p.log_decay[head];
  for (int i = tid; i <= C; i += 256) s.power[i] = i ? expf(i * g) : 1.f;
  long long len = p.length;
  if (p.lengths) { const long long l = p.lengths[seq]; len = l < 0 ? 0 : (l < len ? l : len); }
  const T *ga = (const T*)p.a + seq * p.a_b + head * p.a_h, *gb = (const T*)p.b + seq * p.b_b + head * p.b_h, *gc = (const T*)p.c + seq * p.c_b + head * p.c_h;
  T* go = (T*)p.out + seq * p.o_b + head * p.o_h;
  auto token = [&](long long q) { return p.reverse && q < len ? len - 1 - q : q; };

  Chunk<T> xa[NA], xb[NA], xc[NC];
  auto load = [&](long long q0) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int idx = tid + i * 256, row = idx / (DA / V), col = idx % (DA / V) * V;
      const long long q = q0 + row, t = token(q), left = row < C && q < len ? p.da - col : 0;
      if constexpr (!STATE) xa[i] = load_part(ga + t * p.a_t + col, left);
      xb[i] = load_part(gb + t * p.b_t + col, left);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int idx = tid + i * 256, row = idx / (DC / V), col = idx % (DC / V) * V;
      const long long q = q0 + row, t = token(q);
      xc[i] = load_part(gc + t * p.c_t + col, row < C && q < len ? p.dc - col : 0);
    }
  };

  // R, tile i of this wave: rows (of da) tr(i) * 16 + row4 .. + 3, column (of dc) tc(i) * 16 + colx
  f32x4 acc[NR];
  auto tr = [&](int i) { return (wave * NR + i) / (DC / 16); };
  auto tc = [&](int i) { return (wave * NR + i) % (DC / 16); };
  const float* start = STATE ? nullptr : seg ? p.seg_state + (sh * (p.segments - 1) + seg - 1) * p.da * p.dc : p.state_in ? p.state_in + sh * p.da * p.dc : nullptr;
  const int sr = seg ? p.dc : p.in_r, sc = seg ? 1 : p.in_c;
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = tr(i) * 16 + row4 + e, c = tc(i) * 16 + colx;
      acc[i][e] = start && r < p.da && c < p.dc ? start[(long long)r * sr + c * sc] : 0.f;
    }

  const long long first = (long long)seg * p.seg_chunks * C;
  const long long last = first + (long long)p.seg_chunks * C < p.length ? first + (long long)p.seg_chunks * C : p.length;
  float factor = 1.f;
  if (first < last) load(first);
  for (long long q0 = first; q0 < last; q0 += C) {
    const int n = (int)(len - q0 < 0 ? 0 : (len - q0 < C ? len - q0 : C));  // live tokens of the chunk
    // cuts: bit i = the link between tokens i - 1 and i of the chunk (i = 0: the carry that comes in) is cut; out: the link to the carry that goes on
    unsigned long long cuts = 0;
    bool cut_out = false;
    if (p.reset && n) {
      const bool f = lane < n && (p.reverse ? lane > 0 && reset_at(p, seq, token(q0 + lane) + 1) : reset_at(p, seq, q0 + lane));
      cuts = __ballot(f);
      cut_out = p.reverse && reset_at(p, seq, token(q0 + n - 1));
    }
    auto episode = [&](int i) { return __popcll(cuts & ((2ULL << i) - 1)); };
    const int e_last = n ? episode(n - 1) : 0;
    const bool carries = n == 0 || (e_last == 0 && !cut_out);  // R goes through the whole chunk
    auto weight = [&](int j) { return j < n && !cut_out && episode(j) == e_last ? p.us * s.power[n - p.e0 - j] : 0.f; };

    __syncthreads();  // the chunk before is done with LDS (and power[] is there)
    bool odd = false;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int idx = tid + i * 256, row = idx / (DA / V), col = idx % (DA / V) * V;
      if (row >= C) continue;
      const float w = weight(row);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (!STATE) {
          s.a[row * LA + col + e] = (L)(float)xa[i].e[e];
          s.b[row * LA + col + e] = (L)(float)xb[i].e[e];
        }
        s.bw[row * LA + col + e] = w == 0.f ? (L)0.f : (L)(w * (float)xb[i].e[e]);
      }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int idx = tid + i * 256, row = idx / (DC / V), col = idx % (DC / V) * V;
      if (row >= C) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        odd |= not_finite((float)xc[i].e[e]);
        s.c[row * LC + col + e] = (L)(float)xc[i].e[e];
      }
    }
    if constexpr (!STATE) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s.r[(tc(i) * 16 + colx) * LA + tr(i) * 16 + row4 + e] = (L)acc[i][e];
    }
    // A zero weight times infinity would be NaN: a chunk whose c holds one goes term by term.
    const bool by_term = __syncthreads_or(odd);
    if (q0 + C < last) load(q0 + C);

    if constexpr (!STATE) {
      // P, weighted: wave w has the row tile w of 4 (C = 64), or one tile of 2 x 2 (C = 32)
      constexpr int NP = CT * CT / 4;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int ti = (wave * NP + i) / CT, tj = (wave * NP + i) % CT;
        f32x4 x = {};
        if (tj <= ti)
          for (int k = 0; k < DA; k += KS) x = mma16(frag_kc(s.a, LA, ti * 16, k, lane), frag_kc(s.b, LA, tj * 16, k, lane), x);
        const int j = tj * 16 + colx, ej = episode(j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = ti * 16 + row4 + e;
          s.p[r * LP + j] = (L)(j <= r && r < n && ej == episode(r) ? p.ps * s.power[r - j] * x[e] : 0.f);
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        const int ti = (wave * NO + i) / (DC / 16), tj = (wave * NO + i) % (DC / 16);
        f32x4 x = {};
        for (int k = 0; k < DA; k += KS) x = mma16(frag_kc(s.a, LA, ti * 16, k, lane), frag_kc(s.r, LA, tj * 16, k, lane), x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = ti * 16 + row4 + e;
          x[e] = r < n && episode(r) == 0 ? p.is * s.power[r + p.e0] * x[e] : 0.f;
        }
        if (!by_term) {
          for (int k = 0; k < (ti + 1) * 16; k += KS) x = mma16(frag_kc(s.p, LP, ti * 16, k, lane), frag_kr(s.c, LC, tj * 16, k, lane), x);
        } else {
          for (int j = 0; j < n; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = ti * 16 + row4 + e;
              if (j <= r && r < n && episode(j) == episode(r)) x[e] += (float)s.p[r * LP + j] * (float)s.c[j * LC + tj * 16 + colx];
            }
        }
        if (tj * 16 + colx < p.dc) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const long long q = q0 + ti * 16 + row4 + e;
            if (q < p.length) go[token(q) * p.o_t + tj * 16 + colx] = (T)x[e];  // (behind the end x is 0)
          }
        }
      }
    }

    const float through = s.power[n];
    factor = carries ? factor * through : 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = carries ? through * acc[i][e] : 0.f;
      if (!by_term) {
        for (int k = 0; k < C; k += KS) acc[i] = mma16(frag_kr(s.bw, LA, tr(i) * 16, k, lane), frag_kr(s.c, LC, tc(i) * 16, k, lane), acc[i]);
      } else {
        for (int j = 0; j < n; ++j)
          if (weight(j) != 0.f) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (tr(i) * 16 + row4 + e < p.da) acc[i][e] += (float)s.bw[j * LA + tr(i) * 16 + row4 + e] * (float)s.c[j * LC + tc(i) * 16 + colx];
          }
      }
    }
  }

  float* end = STATE ? p.seg_state + (sh * (p.segments - 1) + seg) * p.da * p.dc : seg == p.segments - 1 && p.state_out ? p.state_out + sh * p.da * p.dc : nullptr;
  if (end) {
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = tr(i) * 16 + row4 + e, c = tc(i) * 16 + colx;
        if (r < p.da && c < p.dc) end[(long long)r * p.dc + c] = acc[i][e];
      }
  }
  if (STATE && tid == 0) p.seg_factor[sh * (p.segments - 1) + seg] = factor;
}

// Along the segments: seg_state[s] <- the R that segment s + 1 starts from.  One thread per element of R.
template <typename T> __global__ __launch_bounds__(256) void k_decay_scan(const DecayPass p) {
  const int n = p.da * p.dc, per = (n + 255) / 256;
  const long long sh = blockIdx.x / per;
  const int i = (int)(blockIdx.x % per) * 256 + threadIdx.x;
  if (i >= n) return;
  const int segs = p.segments - 1;
  float* x = p.seg_state + sh * segs * n + i;
  float r = p.state_in ? p.state_in[sh * n + (long long)(i / p.dc) * p.in_r + (i % p.dc) * p.in_c] : 0.f;
  for (int s = 0; s < segs; ++s) {
    const float f = p.seg_factor[sh * segs + s];
    r = (f == 0.f ? 0.f : f * r) + x[(long long)s * n];
    x[(long long)s * n] = r;
  }
}

// One token.  256 threads per (sequence, head): LPR lanes (four columns each) x 256 / LPR rows of S at a time.  Bound by the state's bytes.
template <typename T, int LPR> __global__ __launch_bounds__(256) void k_decay_step(const mjlab_decay_t d) {
  constexpr int RG = 256 / LPR;
  __shared__ float sq[MJLAB_DECAY_MAX_DIM], sk[MJLAB_DECAY_MAX_DIM], red[RG][LPR * 4];
  const int tid = threadIdx.x, lx = tid % LPR, ly = tid / LPR;
  const long long sh = blockIdx.x, seq = sh / d.heads;
  const int head = (int)(sh % d.heads), col = lx * 4, left = d.dv - col;
  const T *q = (const T*)d.q.p + seq * d.q.batch + head * d.q.head, *k = (const T*)d.k.p + seq * d.k.batch + head * d.k.head;
  const T* v = (const T*)d.v.p + seq * d.v.batch + head * d.v.head;
  bool reset = false;
  if (d.reset) {
    const long long i = seq * d.reset_batch;
    reset = d.reset_bytes == 1 ? ((const unsigned char*)d.reset)[i] != 0 : ((const int*)d.reset)[i] != 0;
  }
  const float decay = expf(d.log_decay[head]);
  if (tid < d.dk) { sq[tid] = (float)q[tid]; sk[tid] = (float)k[tid]; }
  float x[4] = {}, o[4] = {};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) x[e] = (float)v[col + e];
  __syncthreads();
  const float* src = d.state + sh * d.dk * d.dv;
  float* dst = d.state_out + sh * d.dk * d.dv;
  if (left > 0) {
#pragma unroll 4
    for (int r = ly; r < d.dk; r += RG) {
      Chunk<float> c = load_part(src + r * d.dv + col, left);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c.e[e] = (reset ? 0.f : decay * c.e[e]) + sk[r] * x[e];
        o[e] += sq[r] * c.e[e];
      }
      store_part(dst + r * d.dv + col, c, left);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) red[ly][lx * 4 + e] = o[e];
  __syncthreads();
  if (tid < d.dv) {
    float t = 0.f;
    for (int y = 0; y < RG; ++y) t += red[y][tid];
    ((T*)d.o.p)[seq * d.o.batch + head * d.o.head + tid] = (T)(d.scale * t);
  }
}
