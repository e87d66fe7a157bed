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
#include <type_traits>

#include "policy_common.h"

struct DecayPass {
  const void *a, *b, *c;
  void* out;
  long long a_b, a_t, a_h, b_b, b_t, b_h, c_b, c_t, c_h, o_b, o_t, o_h;  // strides: sequence, token, head
  const float* log_decay;
  const float* state_in;  // or NULL
  float* state_out;       // or NULL
  int in_r, in_c;         // strides of the rows (da) and columns (dc) of state_in; state_out is (da, dc) dense
  int seg_given;          // the segments' states are there: those of the pass with da and dc exchanged
  const void* reset;
  int reset_bytes, heads, da, dc, e0, reverse, segments, seg_chunks;
  long long reset_b, reset_t, length;
  const int* lengths;
  float ps, is, us;
  float *seg_state, *seg_factor;  // (seg_given: seg_state is read only) (sequences * heads, segments - 1, da, dc), (sequences * heads, segments - 1)
};

// What the matrix cores read.  float as it is.  16 bits: a b^T as it is; what is formed on the way (weighted rows, pairs, R as the outputs read it) as sums of bf16,
// each the nearest to what is left: two leave out 2^-16 of it, which does not show in outputs of 8 or 11 bits (one bf16: off by 1.41 times their own rounding),
// three hold a float -- the weighted rows of a pass whose R is wanted in the end (EXACT), a float output.  fp16: two bf16 hold an fp16 number as well, exactly, and
// sums of keys and values may leave fp16's range, so all but a b^T is multiplied as bf16.
template <typename T, bool EXACT> struct DecayCfg {
  using L = float;
  static constexpr int KS = 4, PAD = 4, A = 1, W = 1, N = 1, P = 1;  // k per matrix instruction, padding of LDS rows, planes of a, of weighted b, of c, of pairs and R
};
template <bool EXACT> struct DecayCfg<__bf16, EXACT> {
  using L = __bf16;
  static constexpr int KS = 32, PAD = 8, A = 1, W = EXACT ? 3 : 2, N = 1, P = 2;
};
template <bool EXACT> struct DecayCfg<_Float16, EXACT> {
  using L = __bf16;
  static constexpr int KS = 32, PAD = 8, A = 2, W = 3, N = 2, P = 2;
};
// tokens per chunk
template <typename T> constexpr int decay_chunk(bool both_large) { return sizeof(T) == 4 || (DecayCfg<T, false>::N > 1 && both_large) ? 32 : 64; }

__device__ __forceinline__ f32x4 mma16(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16h(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// fragments of 16 rows (or columns) x KS of k: k contiguous / k the row index of the tile
template <typename L> __device__ __forceinline__ s16x8 frag_kc(const L* s, int ld, int r0, int k0, int lane) { return *(const s16x8*)(s + (r0 + (lane & 15)) * ld + k0 + (lane >> 4) * 8); }
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

template <typename T, int DA, int DC, bool STATE, bool EXACT> struct DecayLds {
  using Cfg = DecayCfg<T, EXACT>;
  using L = typename Cfg::L;
  static constexpr int C = decay_chunk<T>(DA > 64 && DC > 64), PAD = Cfg::PAD, LA = DA + PAD, LC = DC + PAD, LP = C + PAD;
  static constexpr int SW = C * LA, SC = C * LC, SP = STATE ? 8 : C * LP, SR = STATE ? 8 : DC * LA;  // a plane of each
  // b times its tokens' weights into R.  bf16: the third plane takes the place of b when the pairs are formed (LDS then holds 128 x 128 heads, and two workgroups of 64 x 64)
  static constexpr bool LATE = !STATE && Cfg::W == 3 && Cfg::N == 1;
  L bw[(LATE ? 2 : Cfg::W) * SW];
  T b[STATE ? 8 : C * LA];
  L c[Cfg::N * SC], p[Cfg::P * SP], r[Cfg::P * SR];
  float enter[C];                 // of R into token i
  int episode[C], odd[8];         // the episode a token belongs to, counted in the chunk
};

// N planes of four numbers, `plane` elements apart; and the number that they hold
template <int N> __device__ __forceinline__ void put4(__bf16* at, int plane, f32x4 x) {
  typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const b16x4 h = __builtin_convertvector(x, b16x4);
    *(b16x4*)(at + i * plane) = h;
    if (i + 1 < N) x -= __builtin_convertvector(h, f32x4);
  }
}
template <int N> __device__ __forceinline__ void put4(float* at, int, const f32x4& x) { *(f32x4*)at = x; }
template <int N, typename L> __device__ __forceinline__ float get(const L* at, int plane) {
  float x = (float)*at;
  if (N > 1 && !not_finite(x)) {  // (nothing can be left of an infinity)
#pragma unroll
    for (int i = 1; i < N; ++i) x += (float)at[i * plane];
  }
  return x;
}
// a b over planes: the terms that count
template <int NA, int NB, typename F> __device__ __forceinline__ f32x4 mma_planes(const F* a, const F* b, f32x4 x) {
#pragma unroll
  for (int i = NA - 1; i >= 0; --i)
#pragma unroll
    for (int j = NB - 1; j >= 0; --j)
      if (i + j < (NA > NB ? NA : NB)) x = mma16(a[i], b[j], x);
  return x;
}

// VEC elements of T times w (w 0: zeros, whatever x holds), as N planes of L; `last`: where the third goes instead
template <int N, typename T, typename L> __device__ __forceinline__ void put_weighted(L* at, int plane, const Chunk<T>& x, float w, L* last = nullptr) {
#pragma unroll
  for (int h = 0; h < Elem<T>::VEC; h += 4) {
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = w * (float)x.e[h + e];
    if (w == 0.f) y = f32x4{};
    if constexpr (N == 3) {
      if (last) {
        put4<2>(at + h, plane, y);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] -= (float)(L)y[e];
        put4<1>(last + h, plane, y);
        continue;
      }
    }
    put4<N>(at + h, plane, y);
  }
}

// Whether a chunk held an infinity or a NaN: the largest magnitude's bits, two 16-bit elements at a time
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <typename T> __device__ __forceinline__ void see(unsigned& most, const Chunk<T>& x) {
  unsigned w[4];
  __builtin_memcpy(w, &x, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) most = most > (w[i] & 0x7fffffffu) ? most : w[i] & 0x7fffffffu;
    else most = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most), __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu)));
  }
}
template <typename T> __device__ __forceinline__ bool seen_odd(unsigned most) {
  if constexpr (sizeof(T) == 4) return most >= 0x7f800000u;
  constexpr unsigned INF = Elem<T>::DTYPE == MJLAB_DTYPE_F16 ? 0x7c00u : 0x7f80u;
  return (most >> 16) >= INF || (most & 0xffffu) >= INF;
}

// How the heads fit the tiles of DA and DC columns: they fill them; they end between two chunks of 16 bytes; or anywhere.
enum { FIT_ANY = 0, FIT_CHUNKS = 1, FIT_FULL = 2 };
// Elements col .. col + VEC - 1 of a row of d, zero from d on.
template <typename T, int FIT> __device__ __forceinline__ Chunk<T> load_row(const T* at, int col, int d) {
  if constexpr (FIT == FIT_FULL) return load_chunk(at);
  else if constexpr (FIT == FIT_CHUNKS) return col < d ? load_chunk(at) : Chunk<T>{};
  else return load_part(at, d - col);
}

// (bf16 128 x 32 heads, 256 sequences of 1024 tokens, forward: 256 threads 90 us, since they need all 256 registers, 512 63.  Chunks of 32 have no eight waves' rows there.)
template <typename T> constexpr int decay_threads(int da, int dc) { return (da >= 64 && dc >= 64) || (da * dc >= 64 * 64 && decay_chunk<T>(false) == 64) ? 512 : 256; }

// 256 or 512 threads per (sequence, head, segment).  STATE: the first pass of a split sequence, the segment's contribution to R alone.
// Products are formed such that an accumulator's four rows are neighbours in memory: P^T and out^T (columns are tokens), R (rows are da).  The rows of a go
// from memory to the matrix cores' registers without LDS, which holds one workgroup of 128 x 128 heads per CU (bf16 155 KB).
// 256 sequences of 1024 tokens, forward with R in the end, us: bf16 128 x 128 116 (2.3 TB/s), 64 x 64 54, 32 x 32 48; fp16 128 x 128 235, 64 x 64 59; float 128 x 128
// 295, 64 x 64 124.  All are bound by the chain of a chunk (stage, pairs, R, with a barrier and LDS reads between): 3 us for a chunk of 64 at 32 x 32, 7 at
// 128 x 128.  More workgroups per CU, where there are more sequences, hide it.
template <typename T, int DA, int DC, int FIT, bool STATE, bool EXACT> __global__ __launch_bounds__(decay_threads<T>(DA, DC), 2) void k_decay_chunks(const DecayPass p) {
  using Cfg = DecayCfg<T, EXACT>;
  using L = typename Cfg::L;
  using S = DecayLds<T, DA, DC, STATE, EXACT>;
  constexpr bool FULL = FIT == FIT_FULL;
  // The scheduler is kept from loading the fragments of every column at once: small heads have the registers for it (float 64 x 64 128 us without, 135 with)
  constexpr bool FENCE = DA * DC > 64 * 64;
  constexpr int C = S::C, KS = Cfg::KS, NA = Cfg::A, PW = Cfg::W, NN = Cfg::N, PR = Cfg::P, LA = S::LA, LC = S::LC, LP = S::LP, V = Elem<T>::VEC, CT = C / 16, KA = DA / KS;
  constexpr int NT = decay_threads<T>(DA, DC), NW = NT / 64, NB = (C * DA / V + NT - 1) / NT, NC = (C * DC / V + NT - 1) / NT;  // 16-byte chunks per thread
  // Waves: of out, OR x OC waves of TR x TC tiles (tokens x dc); of R, RW x NW / RW waves of RR x RC tiles (da x dc)
  constexpr int OC = CT == 4 ? 2 : (DC / 16 < NW ? DC / 16 : NW);
  constexpr int OR = NW / OC, TR = CT / OR, TC = DC / 16 / OC, RW = NW == 8 && DA >= 64 ? 4 : 2, RR = DA / 16 / RW, RC = DC / 16 * RW / NW;
  static_assert(OR * OC == NW && OR * TR == CT && OC * TC == DC / 16 && RR >= 1 && RC >= 1 && RR * RW == DA / 16 && RC * (NW / RW) == DC / 16, "tiles do not cover");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  S& s = *(S*)lds;
  L* const bw = (L*)lds;  // (runs on into s.b where its third plane comes late)
  static_assert(offsetof(S, bw) == 0 && (!S::LATE || offsetof(S, b) == 2 * S::SW * sizeof(L)), "the planes of bw are equally far apart");

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row4 = (lane >> 4) * 4, colx = lane & 15;
  const int t0 = (wave / OC) * TR, c0 = (wave % OC) * TC, r0 = wave / (NW / RW) * RR, rc0 = wave % (NW / RW) * RC;  // this wave's first tiles
  const int segs = STATE ? p.segments - 1 : p.segments;
  const long long sh = blockIdx.x / segs, seq = sh / p.heads;
  const int seg = (int)(blockIdx.x % segs), head = (int)(sh % p.heads);
  // powers of the decay as 2^(n g2); a decay of zero (g2 = -infinity) stays finite here so that its power 0 is 1
  float g2 = p.log_decay[head] * 1.44269504f;
  g2 = g2 < -1e30f ? -1e30f : g2;
  auto power = [&](int n) { return __builtin_amdgcn_exp2f(n * g2); };
  const float decay = power(1);
  long long len = p.length;
  if (p.lengths) { const long long l = p.lengths[seq]; len = l < 0 ? 0 : (l < len ? l : len); }
  const T *ga = (const T*)p.a + seq * p.a_b + head * p.a_h, *gb = (const T*)p.b + seq * p.b_b + head * p.b_h, *gc = (const T*)p.c + seq * p.c_b + head * p.c_h;
  T* go = (T*)p.out + seq * p.o_b + head * p.o_h;
  auto token = [&](long long q) { return p.reverse && q < len ? len - 1 - q : q; };

  // Where this thread's rows of the present chunk lie; one chunk on is `step` tokens on.
  const long long first = (long long)seg * p.seg_chunks * C;
  const long long last = first + (long long)p.seg_chunks * C < p.length ? first + (long long)p.seg_chunks * C : p.length;
  const long long step = p.reverse ? -C : C;
  Chunk<T> xb[NB], xc[NC];
  const T *pb[NB], *pc[NC];
#pragma unroll
  for (int i = 0; i < NB; ++i) pb[i] = gb + token(first + (tid + i * NT) / (DA / V)) * p.b_t + (tid + i * NT) % (DA / V) * V;
#pragma unroll
  for (int i = 0; i < NC; ++i) pc[i] = gc + token(first + (tid + i * NT) / (DC / V)) * p.c_t + (tid + i * NT) % (DC / V) * V;
  auto load = [&](long long q0) {
    const bool all = q0 + C <= len;  // (uniform)
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int row = (tid + i * NT) / (DA / V), col = (tid + i * NT) % (DA / V) * V;
      if ((all && C * DA / V % NT == 0) || (row < C && q0 + row < len)) xb[i] = load_row<T, FIT>(pb[i], col, p.da);
      else xb[i] = Chunk<T>{};
      pb[i] += step * p.b_t;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int row = (tid + i * NT) / (DC / V), col = (tid + i * NT) % (DC / V) * V;
      if ((all && C * DC / V % NT == 0) || (row < C && q0 + row < len)) xc[i] = load_row<T, FIT>(pc[i], col, p.dc);
      else xc[i] = Chunk<T>{};
      pc[i] += step * p.c_t;
    }
  };
  // The rows of a of this wave's tokens.  16 bits: fragments as they are.  float: four k-steps come as 16 bytes, lane group by lane group, so the k order of
  // the fragments is i * 16 + row4 + e, not 4 step + (lane >> 4): the other operand of a product with `a` is read in the same order.
  constexpr bool F32 = sizeof(T) == 4;
  typename std::conditional<F32, f32x4, s16x8>::type fa[TR][F32 ? DA / 16 : KA];
  s16x8 fs[NN > 1 ? KA : 1][NA];  // (fp16) the planes of one tile's
  const T* pa[TR];
  T* po[TR];
#pragma unroll
  for (int t = 0; t < TR; ++t) {
    const long long k = token(first + (t0 + t) * 16 + colx);
    pa[t] = ga + k * p.a_t;
    po[t] = go + k * p.o_t + row4;
  }
  auto load_a = [&](long long q0) {
#pragma unroll
    for (int t = 0; t < TR; ++t) {
      const T* row = pa[t];
      pa[t] += step * p.a_t;
      const bool live = q0 + (t0 + t) * 16 + colx < len;
      if constexpr (!F32) {
#pragma unroll
        for (int k = 0; k < KA; ++k) {
          const int col = k * KS + (lane >> 4) * 8;
          fa[t][k] = live ? __builtin_bit_cast(s16x8, load_row<T, FIT>(row + col, col, p.da)) : s16x8{};
        }
      } else {
#pragma unroll
        for (int i = 0; i < DA / 16; ++i) fa[t][i] = live ? __builtin_bit_cast(f32x4, load_row<T, FIT>(row + i * 16 + row4, i * 16 + row4, p.da)) : f32x4{};
      }
    }
  };
  // (rows row0 .. of b or R, k contiguous) (a's rows of token tile t)^T over all of da.  R, 16 bits: of whole numbers where something is not finite, since a plane of
  // zeros times infinity would be NaN.
  auto with_a = [&](auto of_r, const auto* rows, int row0, int t, bool whole) {
    f32x4 x = {};
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < DA / 16; ++i) {
        const f32x4 o = *(const f32x4*)(rows + (row0 + colx) * LA + i * 16 + row4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x = mma16(o[e], fa[t][i][e], x);
      }
    } else if constexpr (!decltype(of_r)::value) {
#pragma unroll
      for (int k = 0; k < KA; ++k) {
        const s16x8 o = frag_kc(rows, LA, row0, k * KS, lane);
        x = NN == 1 ? mma16(o, fa[t][k], x) : mma16h(o, fa[t][k], x);
      }
    } else if (!whole) {
#pragma unroll
      for (int k = 0; k < KA; ++k) {
        s16x8 o[PR];
#pragma unroll
        for (int i = 0; i < PR; ++i) o[i] = frag_kc(rows + i * S::SR, LA, row0, k * KS, lane);
        x = mma_planes<PR, NA>(o, NN == 1 ? &fa[t][k] : fs[k], x);
      }
    } else {
      for (int k = 0; k < KA; ++k)
        for (int e = 0; e < 8; ++e)
          x = mma16(get<PR>(rows + (row0 + colx) * LA + k * KS + 2 * row4 + e, S::SR), (float)__builtin_bit_cast(Chunk<T>, fa[t][k]).e[e], x);
    }
    return x;
  };

  // R, tile (i, j) of this wave: rows (of da) (r0 + i) * 16 + row4 .. + 3, column (of dc) (rc0 + j) * 16 + colx
  f32x4 acc[RR][RC];
  const float* start = STATE ? nullptr : seg ? p.seg_state + (sh * (p.segments - 1) + seg - 1) * p.da * p.dc : p.state_in ? p.state_in + sh * p.da * p.dc : nullptr;
  const int sr = !seg ? p.in_r : p.seg_given ? 1 : p.dc, sc = !seg ? p.in_c : p.seg_given ? p.da : 1;
#pragma unroll
  for (int i = 0; i < RR; ++i)
#pragma unroll
    for (int j = 0; j < RC; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = (r0 + i) * 16 + row4 + e, c = (rc0 + j) * 16 + colx;
        acc[i][j][e] = start && (FULL || (r < p.da && c < p.dc)) ? start[(long long)r * sr + c * sc] : 0.f;
      }

  float* end = STATE ? p.seg_state + (sh * (p.segments - 1) + seg) * p.da * p.dc : seg == p.segments - 1 && p.state_out ? p.state_out + sh * p.da * p.dc : nullptr;
  float factor = 1.f;
  if (first < last) {
    load(first);
    if constexpr (!STATE) load_a(first);
  }
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
    const bool whole = (cuts >> 1) == 0;  // one episode, but perhaps for the carry
    const int e_last = n ? episode(n - 1) : 0;
    const bool carries = n == 0 || (e_last == 0 && !cut_out);  // R goes through the whole chunk

    __syncthreads();  // the chunk before is done with LDS
    unsigned most = 0;
    float odd = 0.f;  // NaN: R is not finite
    Chunk<L> late[S::LATE ? NB : 1];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int row = (tid + i * NT) / (DA / V), col = (tid + i * NT) % (DA / V) * V;
      if (row >= C) continue;
      const float w = row < n && !cut_out && (whole || episode(row) == e_last) ? p.us * power(n - p.e0 - row) : 0.f;
      put_weighted<PW>(bw + row * LA + col, S::SW, xb[i], w, S::LATE ? late[S::LATE ? i : 0].e : nullptr);
      if constexpr (!STATE) *(Chunk<T>*)(s.b + row * LA + col) = xb[i];
      if constexpr (PW > 1) see(most, xb[i]);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int row = (tid + i * NT) / (DC / V), col = (tid + i * NT) % (DC / V) * V;
      if (row >= C) continue;
      see(most, xc[i]);
      if constexpr (NN == 1) *(Chunk<T>*)(s.c + row * LC + col) = xc[i];
      else put_weighted<NN>(s.c + row * LC + col, S::SC, xc[i], 1.f);
    }
    if (!STATE && tid < C) {
      s.enter[tid] = tid < n && episode(tid) == 0 ? p.is * power(tid + p.e0) : 0.f;
      s.episode[tid] = episode(tid);
    }
    const bool carry = start || q0 > first;  // else R is zero so far
    if (!STATE && carry) {
#pragma unroll
      for (int i = 0; i < RR; ++i)
#pragma unroll
        for (int j = 0; j < RC; ++j) {
          put4<PR>(s.r + ((rc0 + j) * 16 + colx) * LA + (r0 + i) * 16 + row4, S::SR, acc[i][j]);
          if constexpr (PR > 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) odd = __builtin_fmaf(acc[i][j][e], 0.f, odd);
        }
    }
    if constexpr (!STATE && PR > 1)
#pragma unroll
      for (int t = 0; t < TR; ++t)
#pragma unroll
        for (int k = 0; k < KA; ++k) see(most, __builtin_bit_cast(Chunk<T>, fa[t][k]));
    // A zero weight times infinity would be NaN: a chunk whose c holds one goes term by term.  (Planes: any operand, since one may be zero.)
    const bool mine = __ballot(seen_odd<T>(most) || odd != odd) != 0;
    if (lane == 0) s.odd[wave] = mine;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) any |= s.odd[i];
    const bool by_term = __builtin_amdgcn_readfirstlane(any) != 0;
    if (q0 + C < last) load(q0 + C);

    if constexpr (!STATE) {
      // P^T for this wave's tokens; the OC waves that share them take every OC-th tile of the columns
      f32x4 x[TR][TC];
#pragma unroll
      for (int t = 0; t < TR; ++t) {
        const int i = (t0 + t) * 16 + colx, ei = s.episode[i];
        if constexpr (NN > 1) {  // a's rows as planes
#pragma unroll
          for (int k = 0; k < KA; ++k) {
            const h16x8 v = __builtin_bit_cast(h16x8, fa[t][k]);
            typedef float f32x8 __attribute__((ext_vector_type(8)));
            f32x8 left = __builtin_convertvector(v, f32x8);
#pragma unroll
            for (int q = 0; q < NA; ++q) {
              const b16x8 h = __builtin_convertvector(left, b16x8);
              fs[k][q] = __builtin_bit_cast(s16x8, h);
              left -= __builtin_convertvector(h, f32x8);
            }
          }
        }
#pragma unroll
        for (int jj = 0; jj < CT / OC + (CT % OC ? 1 : 0); ++jj) {
          const int tj = jj * OC + wave % OC, j = tj * 16 + row4;
          if (tj >= CT) continue;
          f32x4 y = {};
          if (tj <= t0 + t) {
            y = with_a(std::false_type(), s.b, tj * 16, t, false);
            float w[4];
            if (tj == t0 + t) {
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = j + e <= i ? p.ps * power(i - j - e) : 0.f;
            } else {  // (i > j + 3: neighbours' weights are a decay apart)
              w[3] = p.ps * power(i - j - 3);
#pragma unroll
              for (int e = 2; e >= 0; --e) w[e] = decay * w[e + 1];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (tj < t0 + t || j + e <= i) && i < n && (whole || s.episode[j + e] == ei) ? w[e] * y[e] : 0.f;
          }
          put4<PR>(s.p + i * LP + tj * 16 + row4, S::SP, y);
          if constexpr (FENCE) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int c = 0; c < TC; ++c) {
          x[t][c] = f32x4{};
          if (!carry) continue;
          x[t][c] = with_a(std::true_type(), s.r, (c0 + c) * 16, t, by_term);
          const float f = s.enter[i];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[t][c][e] = f == 0.f ? 0.f : f * x[t][c][e];
          if constexpr (FENCE) __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (q0 + C < last) load_a(q0 + C);
      __syncthreads();
      if constexpr (S::LATE) {  // (the pairs were the last that read b)
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int row = (tid + i * NT) / (DA / V), col = (tid + i * NT) % (DA / V) * V;
          if (row < C) *(Chunk<L>*)(bw + 2 * S::SW + row * LA + col) = late[i];
        }
      }
      if (!by_term) {
#pragma unroll
        for (int t = 0; t < TR; ++t)
          for (int k = 0; k < (t0 + t + 1) * 16; k += KS) {
            decltype(frag_kr(s.c, LC, 0, 0, lane)) fp[PR], fc[NN];
#pragma unroll
            for (int q = 0; q < PR; ++q) fp[q] = frag_kc(s.p + q * S::SP, LP, (t0 + t) * 16, k, lane);
#pragma unroll
            for (int c = 0; c < TC; ++c) {
#pragma unroll
              for (int q = 0; q < NN; ++q) fc[q] = frag_kr(s.c + q * S::SC, LC, (c0 + c) * 16, k, lane);
              x[t][c] = mma_planes<NN, PR>(fc, fp, x[t][c]);
            }
            if constexpr (FENCE) __builtin_amdgcn_sched_barrier(0);
          }
      } else {
#pragma unroll
        for (int t = 0; t < TR; ++t) {
          const int i = (t0 + t) * 16 + colx, ei = s.episode[i];
          for (int j = 0; j <= i && i < n; ++j)
            if (s.episode[j] == ei) {
              const float w = get<PR>(s.p + i * LP + j, S::SP);
#pragma unroll
              for (int c = 0; c < TC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[t][c][e] += w * get<NN>(s.c + j * LC + (c0 + c) * 16 + row4 + e, S::SC);
            }
        }
      }
#pragma unroll
      for (int t = 0; t < TR; ++t) {
        const long long q = q0 + (t0 + t) * 16 + colx;
        // behind the sequence's end x is 0, and the rows there are in order whatever the direction
        T* at = p.reverse && q >= len ? go + q * p.o_t + row4 : po[t];
        po[t] += step * p.o_t;
        if (q >= p.length) continue;
#pragma unroll
        for (int c = 0; c < TC; ++c) {
          const int d = (c0 + c) * 16;
          T o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = (T)x[t][c][e];
          if (FULL || d + row4 + 4 <= p.dc) __builtin_memcpy(at + d, o, sizeof(o));
          else if (FIT == FIT_ANY) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (d + row4 + e < p.dc) at[d + e] = o[e];
          }
        }
      }
    }

    if (!STATE && !end && q0 + C >= last) break;  // nobody wants R any more
    if constexpr (S::LATE) __syncthreads();
    const float through = carries ? power(n) : 0.f;
    factor *= through;
    if (carries) {
#pragma unroll
      for (int i = 0; i < RR; ++i)
#pragma unroll
        for (int j = 0; j < RC; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] *= through;
    } else {  // (whatever it holds)
#pragma unroll
      for (int i = 0; i < RR; ++i)
#pragma unroll
        for (int j = 0; j < RC; ++j) acc[i][j] = f32x4{};
    }
    if (!by_term) {
#pragma unroll 2
      for (int k = 0; k < C; k += KS) {
        decltype(frag_kr(bw, LA, 0, 0, lane)) fb[RR][PW], fc[NN];
#pragma unroll
        for (int i = 0; i < RR; ++i)
#pragma unroll
          for (int q = 0; q < PW; ++q) fb[i][q] = frag_kr(bw + q * S::SW, LA, (r0 + i) * 16, k, lane);
#pragma unroll
        for (int j = 0; j < RC; ++j) {
#pragma unroll
          for (int q = 0; q < NN; ++q) fc[q] = frag_kr(s.c + q * S::SC, LC, (rc0 + j) * 16, k, lane);
#pragma unroll
          for (int i = 0; i < RR; ++i) acc[i][j] = mma_planes<PW, NN>(fb[i], fc, acc[i][j]);
        }
        if constexpr (FENCE) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      for (int t = 0; t < n; ++t) {
        if (cut_out || episode(t) != e_last) continue;
#pragma unroll
        for (int i = 0; i < RR; ++i)
#pragma unroll
          for (int j = 0; j < RC; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = (r0 + i) * 16 + row4 + e;
              if (FULL || r < p.da) acc[i][j][e] += get<PW>(bw + t * LA + r, S::SW) * get<NN>(s.c + t * LC + (rc0 + j) * 16 + colx, S::SC);
            }
      }
    }
  }

  if (end) {
#pragma unroll
    for (int i = 0; i < RR; ++i)
#pragma unroll
      for (int j = 0; j < RC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = (r0 + i) * 16 + row4 + e, c = (rc0 + j) * 16 + colx;
          if (FULL || (r < p.da && c < p.dc)) end[(long long)r * p.dc + c] = acc[i][j][e];
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
