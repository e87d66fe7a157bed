// product.h -- the matrix product of the policy's layers: C[m][n] = sum over k of A[m][k] B[n][k], with what a layer does to C at its end.
//
// One kernel serves the forward product and both products of the backward pass; they differ in which index of an operand is contiguous:
//   y  = x w^T     A = x  (k contiguous)    B = w  (k contiguous)
//   dx = dz w      A = dz (k contiguous)    B = w  (n contiguous)
//   dw = dz^T x    A = dz (m contiguous)    B = x  (n contiguous)
// A k-contiguous tile lies in LDS as rows of 64 or 128 bytes whose 16-byte chunks are exchanged by the row's low bits, so that the 32 rows one
// fragment reads meet all banks evenly; the other kind lies as it is in memory, k rows of m elements, and 16-bit fragments are turned by the
// transposing LDS read (ds_read_b64_tr_b16: four k of one m per lane).  Global loads go through registers one k-tile ahead of the matrix
// instructions.  What lies behind the last m or n may be anything, since its results are not stored: rows behind the last are read from the last,
// and 16 bytes that a row's end cuts are read whole, on into the next row -- but for the last row of all.  So only a k-tile at the end of k pays for bounds.
//
// float: the bf16 matrix cores are sixteen times as fast as those for float.  A float is the sum of three bf16 h + m + l (each the nearest to what is
// left: 3 x 8 bits and their signs hold all 24), so a b = hh + hm + mh + mm + hl + lh and terms below 2^-23 |a b|, which are left out: six products
// of 16 bits, summed in 32, for one of float -- the error of a float product's own rounding, at more than the float instruction's rate (24576 x 1024 x 1024: 190 TFLOP/s; the library's float product
// 128).  A number that has no
// such sum (infinite, NaN, or so large that h overflows) sets a flag, and its workgroup's product is formed again with the float instruction: so do infinities of
// whole operands, since zero times infinity is NaN.
//
// dz, 16 bits: a float in memory, since a gradient may leave fp16's range on both sides where what it is summed to does not, and since its rounding to 16 bits would
// show in the gradients (off by 1.41 times their own rounding).  It is read as two bf16, 2^-16 of it left out, and a float16 that it meets as two, exactly:
// hh + hm + mh, two or three products of 16 bits for one.
#pragma once
#include "policy_common.h"

enum { EPI_LAYER = 0, EPI_GATED = 1, EPI_STORE = 2, EPI_PARTIAL = 3, EPI_SLOPE = 4 };

struct Product {
  const void *A, *B, *B2;      // A: of the kernel's type TA, B and B2 of T.  B2: w_up (EPI_GATED: rows of both in turn; EPI_STORE: the rows k >= kb2 of B)
  long long lda, ldb, ldb2;
  long long M, N, K, kb2;      // kb2: where B's rows end and B2's begin (K where there is no B2)
  long long nb2;               // the same for a k-contiguous B outside EPI_GATED (N where there is no B2)
  long long ksplit;            // k elements per blockIdx.y
  int act;
  const void *b, *b_up, *r;    // the epilogue's
  void* y;
  float *z, *z_up;
  long long ldr, ldy;
  float* partial;              // EPI_PARTIAL: (splits, M, N); EPI_SLOPE: column sums of y, (2 M / BM, 2 N), or NULL
                               // EPI_SLOPE: a gated layer's sums formed again; r = dy, y = [dg | du] as floats
};

__device__ __forceinline__ f32x16 mma(s16x8 a, s16x8 b, f32x16 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(s16x8 a, s16x8 b, f32x16 c, __bf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x4 a, f32x4 b, f32x16 c, float) {
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], c, 0, 0, 0);
  return c;
}

template <typename E> struct Frag { using type = s16x8; };
template <> struct Frag<float> { using type = f32x4; };

// A unit: what one thread loads, keeps and stages at a time, UE neighbouring elements of memory.
template <typename T, int UE> struct alignas(sizeof(T) * UE < 16 ? sizeof(T) * UE : 16) Unit {
  T e[UE];
};
template <typename T, int UE> __device__ __forceinline__ void load_unit(Unit<T, UE>& u, const T* p) { __builtin_memcpy(&u, p, sizeof(u)); }
template <typename T, int UE> __device__ __forceinline__ void load_unit_part(Unit<T, UE>& u, const T* p, long long n) {
  if (n >= UE) { load_unit(u, p); return; }
#pragma unroll
  for (int i = 0; i < UE; ++i) u.e[i] = i < n ? p[i] : (T)0.f;
}

// How an operand is multiplied: memory holds M, the matrix cores read it as the sum of P numbers of E, each the nearest to what is left.
// KB: bytes of k per row and plane of a tile; a k-step of the inner loop is two 16-byte chunks.
template <typename M_, typename E_, int P_> struct Operand {
  using M = M_;
  using E = E_;
  static constexpr int PLANES = P_, UE = 16 / sizeof(E);
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));

// The P bf16 of eight numbers, the first plane's where h points; `odd` becomes NaN if one of them has none (what is left is then infinite or NaN)
template <int P, typename M> __device__ __forceinline__ void put_split(char* h, int plane, const M* x, float& odd) {
  b16x8 part[P];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    f32x2 v = {(float)x[i], (float)x[i + 1]};
#pragma unroll
    for (int q = 0; q < P; ++q) {
      const b16x2 a = __builtin_convertvector(v, b16x2);
      part[q][i] = a[0]; part[q][i + 1] = a[1];
      if (q + 1 == P) break;
      const unsigned u = __builtin_bit_cast(unsigned, a);
      v = f32x2{v[0] - __uint_as_float(u << 16), v[1] - __uint_as_float(u & 0xffff0000u)};
      if (q == 0) odd = __builtin_fmaf(v[1], 0.f, __builtin_fmaf(v[0], 0.f, odd));
    }
  }
#pragma unroll
  for (int q = 0; q < P; ++q) *(b16x8*)(h + q * plane) = part[q];
}

// LDS layout of one operand tile of R rows (m or n)
template <typename O, int KB, bool KC, int R> struct Tile {
  using M = typename O::M;
  using E = typename O::E;
  static constexpr int UE = O::UE, KT = KB / (int)sizeof(E), NU = R * KT / UE / 256;  // units per thread
  static constexpr int STRIDE = KC ? KB : R * (int)sizeof(E) + 32;      // bytes; + 32: the four k rows a transposing read takes lie in other banks
  static constexpr int PLANE = KC ? R * KB : KT * STRIDE, BYTES = O::PLANES * PLANE;
  static constexpr int UPR = KC ? KT / UE : R / UE;                     // units per row of the tile (KC: m rows; else k rows)

  static __device__ __forceinline__ int swizzle(int row, int c) { return KB == 128 ? c ^ ((row >> 1) & 7) : c ^ ((row >> 2) & 3); }
  static __device__ __forceinline__ int row_of(int u) { return u / UPR; }
  static __device__ __forceinline__ int col_of(int u) { return u % UPR * UE; }

  // WATCH: the other operand has several planes, one of which may be zero where this one is infinite
  template <bool WATCH> static __device__ __forceinline__ void put(char* s, int u, const Unit<M, UE>& x, float& odd) {
    const int row = u / UPR, c = u % UPR;
    char* at = s + (KC ? row * KB + (swizzle(row, c) << 4) : row * STRIDE + c * 16);
    if constexpr (O::PLANES > 1) put_split<O::PLANES>(at, PLANE, x.e, odd);
    else if constexpr (sizeof(M) == sizeof(E)) {
      *(Unit<M, UE>*)at = x;
      if constexpr (WATCH)
#pragma unroll
        for (int i = 0; i < UE; ++i) odd = __builtin_fmaf((float)x.e[i], 0.f, odd);
    }
    else *(f32x4*)at = f32x4{(float)x.e[0], (float)x.e[1], (float)x.e[2], (float)x.e[3]};
  }

  // the fragment of rows row0 .. row0 + 31 at k-step kk: lanes 0-31 hold chunk 2 kk, lanes 32-63 chunk 2 kk + 1 of k
  static __device__ __forceinline__ typename Frag<E>::type frag(const char* s, int plane, int row0, int kk, int lane) {
    const int half = lane >> 5;
    s += plane * PLANE;
    if constexpr (KC) {
      const int row = row0 + (lane & 31);
      return *(const typename Frag<E>::type*)(s + row * KB + (swizzle(row, 2 * kk + half) << 4));
    } else if constexpr (sizeof(E) == 2) {
      const int t = lane & 15, k = kk * 16 + half * 8 + (t >> 2), m = row0 + ((lane >> 4) & 1) * 16 + (t & 3) * 4;
      typedef __attribute__((address_space(3))) s16x4 lds_s4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(s + k * STRIDE + m * 2));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(s + (k + 4) * STRIDE + m * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      f32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *(const float*)(s + (kk * 8 + half * 4 + i) * STRIDE + (row0 + (lane & 31)) * 4);
      return v;
    }
  }
};

// The sum over k in [kbeg, kend) for the tile at (m0, n0): 4 waves as 2 x 2, each BM / 2 x BN / 2 in 32 x 32 tiles.  -> true if planes do not multiply as their number does.
template <typename OA, typename OB, int KB, int BUFFERS, bool AK, bool BK, int BM, int BN, bool GATED>
__device__ __forceinline__ bool product_tile(const Product& p, long long m0, long long n0, long long kbeg, long long kend, char* lds, f32x16 (&acc)[BM / 64][BN / 64]) {
  using TA = Tile<OA, KB, AK, BM>;
  using TB = Tile<OB, KB, BK, BN>;
  using E = typename OA::E;
  using MA = typename OA::M;
  using MB = typename OB::M;
  constexpr int UE = OA::UE, KT = TA::KT, WM = BM / 2, WN = BN / 2, MI = WM / 32, NI = WN / 32, HALF = WN / 2, BUF = TA::BYTES + TB::BYTES;
  constexpr int PA = OA::PLANES, PB = OB::PLANES, ORDER = PA > PB ? PA : PB, STEPS = KB / 32;
  static_assert(sizeof(E) == sizeof(typename OB::E), "the matrix cores read both operands alike");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * WM, wn = (wave & 1) * WN;
  const MA* A = (const MA*)p.A;
  const MB *B = (const MB*)p.B, *B2 = (const MB*)p.B2;
  // Row-contiguous operands: no row's end cuts the tile, or rows are at least a unit apart, so that a unit read beyond a row's end stays inside the next row
  const bool in_a = AK || m0 + BM <= p.M, in_b = BK || n0 + BN <= p.N;
  const bool over_a = in_a || p.lda >= UE, over_b = in_b || (p.ldb >= UE && (p.kb2 == p.K || p.ldb2 >= UE));
  auto whole = [&](long long k0) {  // (uniform) the k-tile at k0 can be read without bounds
    const long long k1 = k0 + KT;
    return k1 <= kend && over_a && over_b && (in_a || k1 < p.K) && (in_b || (k1 < p.K && (k1 < p.kb2 || k0 >= p.kb2)));
  };

  Unit<MA, UE> ra[TA::NU];
  Unit<MB, UE> rb[TB::NU];
  const MA* pa[TA::NU];
  const MB* pb[TB::NU];  // where this thread's units lie at the present k-tile
  auto a_at = [&](int i, long long k0) {
    const int u = tid + i * 256, r = TA::row_of(u), c = TA::col_of(u);
    if constexpr (AK) { const long long m = m0 + r < p.M ? m0 + r : p.M - 1; return A + m * p.lda + k0 + c; }
    else return A + (k0 + r) * p.lda + (m0 + c < p.M ? m0 + c : 0);
  };
  auto b_at = [&](int i, long long k0) {
    const int u = tid + i * 256, r = TB::row_of(u), c = TB::col_of(u);
    if constexpr (BK) {
      long long n = GATED ? n0 + r / (2 * HALF) * HALF + r % HALF : n0 + r;
      n = n < p.N ? n : p.N - 1;
      if (!GATED && n >= p.nb2) return B2 + (n - p.nb2) * p.ldb2 + k0 + c;
      return (GATED && (r / HALF & 1) ? B2 + n * p.ldb2 : B + n * p.ldb) + k0 + c;
    } else {
      const long long k = k0 + r;
      return (k < p.kb2 ? B + k * p.ldb : B2 + (k - p.kb2) * p.ldb2) + (n0 + c < p.N ? n0 + c : 0);
    }
  };
  auto aim = [&](long long k0) {
#pragma unroll
    for (int i = 0; i < TA::NU; ++i) pa[i] = a_at(i, k0);
#pragma unroll
    for (int i = 0; i < TB::NU; ++i) pb[i] = b_at(i, k0);
  };
  auto load = [&](long long k0) {
    if (whole(k0)) {
#pragma unroll
      for (int i = 0; i < TA::NU; ++i) load_unit(ra[i], pa[i]);
#pragma unroll
      for (int i = 0; i < TB::NU; ++i) load_unit(rb[i], pb[i]);
    } else {
#pragma unroll
      for (int i = 0; i < TA::NU; ++i) {
        const int u = tid + i * 256, r = TA::row_of(u), c = TA::col_of(u);
        load_unit_part(ra[i], pa[i], AK ? kend - (k0 + c) : k0 + r < kend ? p.M - (m0 + c) : 0);
      }
#pragma unroll
      for (int i = 0; i < TB::NU; ++i) {
        const int u = tid + i * 256, r = TB::row_of(u), c = TB::col_of(u);
        load_unit_part(rb[i], pb[i], BK ? kend - (k0 + c) : k0 + r < kend ? p.N - (n0 + c) : 0);
      }
    }
    // on to the next k-tile; where B's rows change over to B2's, the pointers are formed anew
#pragma unroll
    for (int i = 0; i < TA::NU; ++i) pa[i] += AK ? KT : KT * p.lda;
    if constexpr (BK) {
#pragma unroll
      for (int i = 0; i < TB::NU; ++i) pb[i] += KT;
    } else {
      const bool same = k0 + 2 * KT <= p.kb2 || k0 >= p.kb2;  // (uniform)
#pragma unroll
      for (int i = 0; i < TB::NU; ++i) pb[i] = same ? pb[i] + KT * (k0 < p.kb2 ? p.ldb : p.ldb2) : b_at(i, k0 + KT);
    }
  };
  float odd = 0.f;
  auto stage = [&](char* s) {
#pragma unroll
    for (int i = 0; i < TA::NU; ++i) TA::template put<(PB > 1)>(s, tid + i * 256, ra[i], odd);
#pragma unroll
    for (int i = 0; i < TB::NU; ++i) TB::template put<(PA > 1)>(s + TA::BYTES, tid + i * 256, rb[i], odd);
  };

#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x16{};
  // Fragments of two k-steps: one is multiplied while the next comes from LDS.  (The scheduler would read into the registers of the step before and wait for
  // every read; the barriers keep it from that.)
  constexpr int SETS = ORDER > 1 ? 1 : 2;
  typename Frag<E>::type fa[SETS][MI][PA], fb[SETS][NI][PB];
  auto fetch = [&](const char* sa, int kk) {
#pragma unroll
    for (int q = 0; q < PA; ++q)
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[kk % SETS][i][q] = TA::frag(sa, q, wm + i * 32, kk, lane);
#pragma unroll
    for (int q = 0; q < PB; ++q)
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[kk % SETS][j][q] = TB::frag(sa + TA::BYTES, q, wn + j * 32, kk, lane);
  };
  auto multiply = [&](int kk) {
#pragma unroll
    for (int qa = 0; qa < PA; ++qa)
#pragma unroll
      for (int qb = 0; qb < PB && qa + qb < ORDER; ++qb)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = mma(fa[kk % SETS][i][qa], fb[kk % SETS][j][qb], acc[i][j], E());
  };
  aim(kbeg);
  load(kbeg);
  stage(lds);
  if (BUFFERS == 2 && kbeg + KT < kend) load(kbeg + KT);
  __syncthreads();
  int cur = 0;
  for (long long k0 = kbeg; k0 < kend; k0 += KT) {
    const char* sa = lds + cur * BUF;
    if constexpr (BUFFERS == 2) {
      // The next k-tile, which came while the last was multiplied, goes to the other buffer before this one is multiplied, so that its way to LDS and the
      // one after's way here lie behind the matrix instructions; what the first of those read is asked for ahead of it.
      fetch(sa, 0);
      cur ^= 1;
      if (k0 + KT < kend) stage(lds + cur * BUF);
      if (k0 + 2 * KT < kend) load(k0 + 2 * KT);
    } else {
      if (k0 + KT < kend) load(k0 + KT);
      fetch(sa, 0);
    }
#pragma unroll
    for (int kk = 0; kk < STEPS; ++kk) {
      if constexpr (SETS == 1) {
        if (kk) fetch(sa, kk);
      } else {
        if (kk + 1 < STEPS) fetch(sa, kk + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      multiply(kk);
    }
    if constexpr (BUFFERS == 1) {
      __syncthreads();
      if (k0 + KT < kend) stage(lds);
    }
    __syncthreads();
  }
  return odd != odd;
}

// Sizes of a launch: the tile, and how T is multiplied in it.  16 bits: 256 x 128 needs 48 KB of LDS with two buffers of 32 k, 128 x 128 32 KB with one of 64
// (two and three workgroups per CU).  Other depths were no faster (16384 x 2048 x 2816 bf16, us: two buffers of 32 k 226, one of 64 k 239, registers two tiles
// ahead 235), nor was a loop without bounds checks (220), other orders of its instructions (220 .. 224) or a wave priority (220); 256 x 256 tiles, one workgroup
// per CU, gain where k is long (8192 x 8192 x 8192: 1040 instead of 1140) and lose where it is not, since nothing hides their ends (24576 x 1024 x 1024: 100
// instead of 74).  The library's product takes 190 in the first and 52 in the last.
template <typename TA, typename T, int BM_, int BN_> struct Shape {
  static constexpr int BM = BM_, BN = BN_, KB = BM_ == 256 ? 64 : 128, BUFFERS = BM_ == 128 ? 1 : 2;
  using A = Operand<T, T, 1>;
  using B = Operand<T, T, 1>;
};
template <int BM_, int BN_> struct Shape<float, float, BM_, BN_> {
  static constexpr int BM = BM_, BN = BN_, KB = 64, BUFFERS = BM_ == 64 ? 2 : 1;
  using A = Operand<float, __bf16, 3>;
  using B = Operand<float, __bf16, 3>;
};
// dz: one buffer of 32 k is 4 % slower, one of 64 k 2 % (24576 x 1024 x 1024 bf16 dx with its slope kernel 207, 213, 208 us)
template <typename T, int BM_, int BN_> struct Shape<float, T, BM_, BN_> {
  static constexpr int BM = BM_, BN = BN_, KB = 64, BUFFERS = 2;
  using A = Operand<float, __bf16, 2>;
  using B = Operand<T, __bf16, Elem<T>::DTYPE == MJLAB_DTYPE_BF16 ? 1 : 2>;
};

template <typename TA, typename T, bool AK, bool BK, int BM, int BN, int EPI> struct ProductLds {
  using S = Shape<TA, T, BM, BN>;
  static constexpr int TILES = S::BUFFERS * (Tile<typename S::A, S::KB, AK, BM>::BYTES + Tile<typename S::B, S::KB, BK, BN>::BYTES);
  static constexpr int AGAIN = sizeof(TA) == 4 ? Tile<Operand<TA, float, 1>, 64, AK, BM>::BYTES + Tile<Operand<T, float, 1>, 64, BK, BN>::BYTES : 0;  // (the second try)
  static constexpr int EPILOGUE = 4 * 32 * (BN / 2 + 4) * 4;
  static constexpr int BYTES = TILES > EPILOGUE ? (TILES > AGAIN ? TILES : AGAIN) : (EPILOGUE > AGAIN ? EPILOGUE : AGAIN);
};

// (Three workgroups of 128 x 128 per CU need 168 registers: the activations' branches are held to that, or all pay, 83 -> 94 us at 24576 x 512 x 512 float.)
template <typename TA, typename T, bool AK, bool BK, int BM, int BN, int EPI> __global__ __launch_bounds__(256, BK && BM == 128 ? 3 : 2) void k_product(const Product p) {
  using S = Shape<TA, T, BM, BN>;
  constexpr int V = Elem<T>::VEC, WM = BM / 2, WN = BN / 2, MI = WM / 32, NI = WN / 32;
  constexpr bool SLOPE = EPI == EPI_SLOPE, GATED = EPI == EPI_GATED || SLOPE;
  constexpr int BNO = GATED ? BN / 2 : BN, HALF = WN / 2;  // output columns per workgroup; a gated wave owns HALF columns of both products
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave >> 1) * WM, wn = (wave & 1) * WN;
  // Tiles go through the device in groups of 8 rows of tiles, column after column: neighbours in time share operand rows in L2.
  const long long tm = (p.M + BM - 1) / BM, tn = (p.N + BNO - 1) / BNO, tile = xcd_tile(blockIdx.x, gridDim.x);
  const long long g = tile / (8 * tn), in = tile % (8 * tn), gm = tm - 8 * g < 8 ? tm - 8 * g : 8;
  const long long m0 = (8 * g + in % gm) * BM, n0 = in / gm * BNO;
  const long long kbeg = blockIdx.y * p.ksplit, kend = kbeg + p.ksplit < p.K ? kbeg + p.ksplit : p.K;

  f32x16 acc[MI][NI];
  const bool odd = product_tile<typename S::A, typename S::B, S::KB, S::BUFFERS, AK, BK, BM, BN, GATED>(p, m0, n0, kbeg, kend, lds, acc);
  if constexpr (sizeof(TA) == 4) {
    if (__syncthreads_or(odd)) product_tile<Operand<TA, float, 1>, Operand<T, float, 1>, 64, 1, AK, BK, BM, BN, GATED>(p, m0, n0, kbeg, kend, lds, acc);
  }

  // C leaves through LDS, 32 rows of the wave's own at a time: an accumulator holds one column per lane, memory wants 16 bytes of a row.
  constexpr int LD = WN + 4;
  float* c = (float*)lds + wave * 32 * LD;
  constexpr int OV = EPI == EPI_PARTIAL ? 4 : V, OW = GATED ? HALF : WN, LPR = OW / OV, RPP = 64 / LPR;  // output elements per lane, lanes per row, rows per pass
  const int col = (lane % LPR) * OV;
  float sum[SLOPE ? OV : 1] = {}, sum_up[SLOPE ? OV : 1] = {};  // of this lane's rows
  const long long n = n0 + (GATED ? wn / 2 : wn) + col, left = p.N - n;
  float bias[OV], bias_up[OV];
#pragma unroll
  for (int e = 0; e < OV; ++e) bias[e] = bias_up[e] = 0.f;
  if constexpr (EPI == EPI_LAYER || GATED) {
#pragma unroll
    for (int e = 0; e < OV; ++e) {
      if (p.b && e < left) bias[e] = (float)((const T*)p.b)[n + e];
      if (GATED && p.b_up && e < left) bias_up[e] = (float)((const T*)p.b_up)[n + e];
    }
  }
  constexpr int PASSES = 32 / RPP;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    // the residual's rows are on their way while C goes through LDS
    Chunk<T> res[EPI == EPI_LAYER || SLOPE ? PASSES : 1];
    if constexpr (EPI == EPI_LAYER || SLOPE) {
      if (SLOPE || p.r) {
#pragma unroll
        for (int q = 0; q < PASSES; ++q) {
          const long long m = m0 + wm + i * 32 + q * RPP + lane / LPR;
          res[q] = load_part((const T*)p.r + m * p.ldr + n, m < p.M ? left : 0);
        }
      }
    }
    if (i) __syncthreads();
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) c[(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * LD + j * 32 + (lane & 31)] = acc[i][j][e];
    __syncthreads();
    float v[PASSES][OV], u[GATED ? PASSES : 1][OV];
#pragma unroll
    for (int q = 0; q < PASSES; ++q)
#pragma unroll
      for (int e = 0; e < OV; ++e) {
        v[q][e] = c[(q * RPP + lane / LPR) * LD + col + e] + bias[e];
        if constexpr (GATED) u[q][e] = c[(q * RPP + lane / LPR) * LD + HALF + col + e] + bias_up[e];
      }
    auto rows = [&](auto f) {  // f(pass, row of C) for the rows that there are
#pragma unroll
      for (int q = 0; q < PASSES; ++q) {
        const long long m = m0 + wm + i * 32 + q * RPP + lane / LPR;
        if (m < p.M && left > 0) f(q, m);
      }
    };
    if constexpr (EPI == EPI_PARTIAL) {
      rows([&](int q, long long m) {
        Chunk<float> out;
#pragma unroll
        for (int e = 0; e < OV; ++e) out.e[e] = v[q][e];
        store_part(p.partial + ((long long)blockIdx.y * p.M + m) * p.N + n, out, left);
      });
    } else {
      auto put = [&](void* base, long long ld, int q, long long m, const float (&x)[OV]) {
        Chunk<T> out;
#pragma unroll
        for (int e = 0; e < OV; ++e) out.e[e] = (T)x[e];
        store_part((T*)base + m * ld + n, out, left);
      };
      auto put_float = [&](float* base, long long ld, int q, long long m, const float (&x)[OV]) {
#pragma unroll
        for (int e = 0; e < OV; e += 4) store_part(base + m * ld + n + e, Chunk<float>{{x[e], x[e + 1], x[e + 2], x[e + 3]}}, left - e);
      };
      if constexpr (SLOPE) {
        with_act(p.act, [&](auto act) {
          constexpr int ACT = decltype(act)::value;
#pragma unroll
          for (int q = 0; q < PASSES; ++q)
#pragma unroll
            for (int e = 0; e < OV; ++e) {
              const float d = (float)res[q].e[e], g = v[q][e];  // (d is 0 behind the last row)
              v[q][e] = d * act_slope<ACT, sizeof(T) == 4>(g) * u[q][e];
              u[q][e] = d * act_value<ACT, sizeof(T) == 4>(g);
              const bool there = m0 + wm + i * 32 + q * RPP + lane / LPR < p.M;  // (what stands behind may be infinite)
              sum[e] += there ? v[q][e] : 0.f;
              sum_up[e] += there ? u[q][e] : 0.f;
            }
        });
        rows([&](int q, long long m) {
          put_float((float*)p.y, p.ldy, q, m, v[q]);
          put_float((float*)p.y + p.N, p.ldy, q, m, u[q]);
        });
      } else if constexpr (EPI != EPI_STORE) {
        if (p.z) rows([&](int q, long long m) { put_float(p.z, p.N, q, m, v[q]); });
        with_act(p.act, [&](auto act) {
#pragma unroll
          for (int q = 0; q < PASSES; ++q)
#pragma unroll
            for (int e = 0; e < OV; ++e) v[q][e] = act_value<decltype(act)::value, sizeof(T) == 4>(v[q][e]);
        });
        if constexpr (GATED) {
          if (p.z_up) rows([&](int q, long long m) { put_float(p.z_up, p.N, q, m, u[q]); });
#pragma unroll
          for (int q = 0; q < PASSES; ++q)
#pragma unroll
            for (int e = 0; e < OV; ++e) v[q][e] *= u[q][e];
        } else if (p.r) {
#pragma unroll
          for (int q = 0; q < PASSES; ++q)
#pragma unroll
            for (int e = 0; e < OV; ++e) v[q][e] += (float)res[q].e[e];
        }
      }
      if constexpr (!SLOPE) rows([&](int q, long long m) { put(p.y, p.ldy, q, m, v[q]); });
    }
  }
  if constexpr (SLOPE) {
    if (p.partial) {
#pragma unroll
      for (int e = 0; e < OV; ++e)
#pragma unroll
        for (int x = LPR; x < 64; x *= 2) {
          sum[e] += __shfl_xor(sum[e], x);
          sum_up[e] += __shfl_xor(sum_up[e], x);
        }
      if (lane < LPR) {
        float* to = p.partial + (m0 / BM * 2 + (wave >> 1)) * 2 * p.N + n;
#pragma unroll
        for (int e = 0; e < OV; ++e)
          if (e < left) { to[e] = sum[e]; to[p.N + e] = sum_up[e]; }
      }
    }
  }
}

// out = sum over the splits, in the order of the splits; one element per thread, eight loads in flight
template <typename T> __global__ __launch_bounds__(256) void k_join_splits(const float* partial, T* out, long long n, long long stride, int splits) {
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < splits; ++k) s += partial[k * stride + i];
  out[i] = (T)s;
}

// What EPI_LAYER and EPI_GATED do, on sums that were split: partial (splits, rows, out | 2 out), one output per thread
template <typename T, bool GATED> __global__ __launch_bounds__(256) void k_join_layer(const Product p, int splits) {
  const long long i = blockIdx.x * 256LL + threadIdx.x, n = p.M * p.N;
  if (i >= n) return;
  const long long m = i / p.N, c = i % p.N, width = GATED ? 2 * p.N : p.N;
  float v = 0.f, u = 0.f;
#pragma unroll 8
  for (int k = 0; k < splits; ++k) {
    v += p.partial[(k * p.M + m) * width + c];
    if constexpr (GATED) u += p.partial[(k * p.M + m) * width + p.N + c];
  }
  if (p.b) v += (float)((const T*)p.b)[c];
  if (p.z) p.z[i] = v;
  with_act(p.act, [&](auto act) { v = act_value<decltype(act)::value, sizeof(T) == 4>(v); });
  if constexpr (GATED) {
    if (p.b_up) u += (float)((const T*)p.b_up)[c];
    if (p.z_up) p.z_up[i] = u;
    v *= u;
  } else if (p.r) v += (float)((const T*)p.r)[m * p.ldr + c];
  ((T*)p.y)[m * p.ldy + c] = (T)v;
}

// dz (rows, out | 2 out), floats, from dy and the stored sums, and this row block's column sums for the bias gradient.
// 256 threads: 32 chunk columns x 8 rows, four rows of each thread in flight, over SLOPE_ROWS rows; workgroups: row blocks x `colblocks`.
// dz NULL: column sums of dy alone.  FROM: what is stored is the output of a float layer.  Bound by memory: dense two reads and a write, gated three and two.
#define SLOPE_ROWS 64
template <typename T, bool GATED, bool FROM> __global__ __launch_bounds__(256) void k_layer_slope(const T* dy, long long ld_dy, const float* z, const float* z_up, float* dz, long long pitch,
                                                                                                  float* sums, long long rows, long long out, unsigned colblocks, int act) {
  constexpr int V = Elem<T>::VEC, NS = GATED ? 2 : 1, ROWS = GATED ? 1 : 2;
  __shared__ float part[NS][8][32 * V];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const unsigned bx = blockIdx.x % colblocks, by = blockIdx.x / colblocks;
  const long long n = (bx * 32LL + tx) * V, left = out - n, r0 = by * (long long)SLOPE_ROWS;
  float s[NS][V] = {};
  const bool slope = dz && (GATED || act != MJLAB_ACT_NONE);
  for (int i = ty; i < SLOPE_ROWS && r0 + i < rows; i += 8 * ROWS) {
    Chunk<T> d[ROWS];
    float z0[ROWS][V], z1[GATED ? ROWS : 1][V];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const long long m = r0 + i + 8 * q, have = m < rows ? left : 0;
      d[q] = load_part(dy + m * ld_dy + n, have);
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        const Chunk<float> x = load_part(z + m * out + n + e, slope ? have - e : 0), y = load_part(z_up + m * out + n + e, GATED ? have - e : 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          z0[q][e + k] = x.e[k];
          if constexpr (GATED) z1[q][e + k] = y.e[k];
        }
      }
    }
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const long long m = r0 + i + 8 * q;
      if (slope) {
        float o[V], o_up[GATED ? V : 1];
        with_act(act, [&](auto a) {
          constexpr int ACT = decltype(a)::value;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float x = z0[q][e], t = (float)d[q].e[e];
            o[e] = t * (FROM ? act_slope_out<ACT>(x) : act_slope<ACT, sizeof(T) == 4>(x));
            if constexpr (GATED) {
              o[e] *= z1[q][e];
              o_up[e] = t * act_value<ACT, sizeof(T) == 4>(x);
              s[NS - 1][e] += o_up[e];
            }
            s[0][e] += o[e];
          }
        });
        if (m < rows && left > 0) {
          float* at = dz + m * pitch + n;
#pragma unroll
          for (int e = 0; e < V; e += 4) {
            store_part(at + e, Chunk<float>{{o[e], o[e + 1], o[e + 2], o[e + 3]}}, left - e);
            if constexpr (GATED) store_part(at + out + e, Chunk<float>{{o_up[e], o_up[e + 1], o_up[e + 2], o_up[e + 3]}}, left - e);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) s[0][e] += (float)d[q].e[e];
      }
    }
  }
  if (!sums) return;
#pragma unroll
  for (int q = 0; q < NS; ++q)
#pragma unroll
    for (int e = 0; e < V; ++e) part[q][ty][tx * V + e] = s[q][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256) {
    const long long c = bx * 32LL * V + i;
    if (c >= out) continue;
#pragma unroll
    for (int q = 0; q < NS; ++q) {
      float t = 0.f;
#pragma unroll
      for (int y = 0; y < 8; ++y) t += part[q][y][i];
      sums[by * (NS * out) + q * out + c] = t;
    }
  }
}

// Bias gradients: the row blocks' sums, in order, 16 partial sums per column.
template <typename T> __global__ __launch_bounds__(256) void k_join_sums(const float* sums, T* db, T* db_up, long long out, long long cols, long long blocks) {
  __shared__ float part[16][17];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long long c = blockIdx.x * 16LL + tx;
  float s = 0.f;
  if (c < cols)
#pragma unroll 4
    for (long long b = ty; b < blocks; b += 16) s += sums[b * cols + c];
  part[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < cols) {
    s = 0.f;
#pragma unroll
    for (int y = 0; y < 16; ++y) s += part[y][tx];
    if (c < out) db[c] = (T)s;
    else db_up[c - out] = (T)s;
  }
}
