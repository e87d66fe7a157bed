// product.h -- the matrix product of the policy's layers: C[m][n] = sum over k of A[m][k] B[n][k], with what a layer does to C at its end.
//
// One kernel serves the forward product and both products of the backward pass; they differ in which index of an operand is contiguous:
//   y  = x w^T     A = x  (k contiguous)    B = w  (k contiguous)
//   dx = dz w      A = dz (k contiguous)    B = w  (n contiguous)
//   dw = dz^T x    A = dz (m contiguous)    B = x  (n contiguous)
// A k-contiguous tile lies in LDS as rows of 128 bytes whose eight 16-byte chunks are exchanged by the row's low bits, so that the 32 rows
// one fragment reads meet all banks evenly; the other kind lies as it is in memory, k rows of m elements, and 16-bit fragments are turned by
// the transposing LDS read (ds_read_b64_tr_b16: four k of one m per lane).  Global loads go through registers one k-tile ahead of the
// matrix instructions, two LDS buffers, one barrier per k-tile.
#pragma once
#include "policy_common.h"

enum { EPI_LAYER = 0, EPI_GATED = 1, EPI_STORE = 2, EPI_PARTIAL = 3 };

struct Product {
  const void *A, *B, *B2;      // B2: w_up (EPI_GATED: rows of both in turn; EPI_STORE: the rows k >= kb2 of B)
  long long lda, ldb, ldb2;
  long long M, N, K, kb2;      // kb2: where B's rows end and B2's begin (K where there is no B2)
  long long ksplit;            // k elements per blockIdx.y
  int act;
  const void *b, *b_up, *r;    // the epilogue's
  void *y, *z, *z_up;
  long long ldr, ldy;
  float* partial;              // EPI_PARTIAL: (splits, M, N)
};

template <typename T> struct Frag { using type = s16x8; };
template <> struct Frag<float> { using type = f32x4; };

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

// LDS layout of one operand tile of R rows (m or n) and 128 bytes of k per row
template <typename T, bool KC, int R> struct Tile {
  static constexpr int V = Elem<T>::VEC, KT = 8 * V, NCH = R * 8 / 256;  // k per tile, 16-byte chunks per thread
  static constexpr int STRIDE = KC ? 128 : R * (int)sizeof(T) + 32;      // bytes; + 32: the four k rows a transposing read takes lie in other banks
  static constexpr int BYTES = KC ? R * 128 : KT * STRIDE;

  static __device__ __forceinline__ int address(int idx) {
    if constexpr (KC) { const int row = idx >> 3, c = idx & 7; return row * 128 + ((c ^ (row & 7)) << 4); }
    else { const int row = idx / (R / V), c = idx % (R / V); return row * STRIDE + c * 16; }
  }

  // the fragment of rows row0 .. row0 + 31 for the kk-th eighth-pair of the tile: lanes 0-31 hold chunk 2 kk, lanes 32-63 chunk 2 kk + 1 of k
  static __device__ __forceinline__ typename Frag<T>::type frag(const char* s, int row0, int kk, int lane) {
    const int half = lane >> 5;
    if constexpr (KC) {
      const int row = row0 + (lane & 31), c = 2 * kk + half;
      return *(const typename Frag<T>::type*)(s + row * 128 + ((c ^ (row & 7)) << 4));
    } else if constexpr (sizeof(T) == 2) {
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

// 256 threads = 4 waves as 2 x 2; a wave owns BM / 2 x BN / 2 of C in 32 x 32 tiles.
template <typename T, bool AK, bool BK, int BM, int BN, int EPI> __global__ __launch_bounds__(256, 2) void k_product(const Product p) {
  using TA = Tile<T, AK, BM>;
  using TB = Tile<T, BK, BN>;
  constexpr int V = Elem<T>::VEC, KT = TA::KT, WM = BM / 2, WN = BN / 2, MI = WM / 32, NI = WN / 32;
  constexpr int BUF = TA::BYTES + TB::BYTES;
  constexpr bool GATED = EPI == EPI_GATED;
  constexpr int BNO = GATED ? BN / 2 : BN, HALF = WN / 2;  // output columns per workgroup; a gated wave owns HALF columns of both products
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * WM, wn = (wave & 1) * WN;
  const long long tn = (p.N + BNO - 1) / BNO, tile = xcd_tile(blockIdx.x, gridDim.x);
  const long long m0 = tile / tn * BM, n0 = tile % tn * BNO;
  const long long kbeg = blockIdx.y * p.ksplit, kend = kbeg + p.ksplit < p.K ? kbeg + p.ksplit : p.K;
  const T *A = (const T*)p.A, *B = (const T*)p.B, *B2 = (const T*)p.B2;

  Chunk<T> ra[TA::NCH], rb[TB::NCH];
  auto load = [&](long long k0) {
#pragma unroll
    for (int i = 0; i < TA::NCH; ++i) {
      const int idx = tid + i * 256;
      if constexpr (AK) {
        const long long m = m0 + (idx >> 3), k = k0 + (idx & 7) * V;
        ra[i] = load_part(A + m * p.lda + k, m < p.M ? kend - k : 0);
      } else {
        const long long k = k0 + idx / (BM / V), m = m0 + (idx % (BM / V)) * V;
        ra[i] = load_part(A + k * p.lda + m, k < kend ? p.M - m : 0);
      }
    }
#pragma unroll
    for (int i = 0; i < TB::NCH; ++i) {
      const int idx = tid + i * 256;
      if constexpr (BK) {
        const int row = idx >> 3;
        const long long k = k0 + (idx & 7) * V;
        if constexpr (GATED) {
          const long long n = n0 + row / (2 * HALF) * HALF + row % HALF;
          const bool up = (row / HALF) & 1;
          rb[i] = load_part((up ? B2 + n * p.ldb2 : B + n * p.ldb) + k, n < p.N ? kend - k : 0);
        } else {
          const long long n = n0 + row;
          rb[i] = load_part(B + n * p.ldb + k, n < p.N ? kend - k : 0);
        }
      } else {
        const long long k = k0 + idx / (BN / V), n = n0 + (idx % (BN / V)) * V;
        const T* row = k < p.kb2 ? B + k * p.ldb : B2 + (k - p.kb2) * p.ldb2;
        rb[i] = load_part(row + n, k < kend ? p.N - n : 0);
      }
    }
  };
  auto stage = [&](char* s) {
#pragma unroll
    for (int i = 0; i < TA::NCH; ++i) *(Chunk<T>*)(s + TA::address(tid + i * 256)) = ra[i];
#pragma unroll
    for (int i = 0; i < TB::NCH; ++i) *(Chunk<T>*)(s + TA::BYTES + TB::address(tid + i * 256)) = rb[i];
  };

  f32x16 acc[MI][NI] = {};
  load(kbeg);
  stage(lds);
  __syncthreads();
  int cur = 0;
  for (long long k0 = kbeg; k0 < kend; k0 += KT) {
    const bool more = k0 + KT < kend;
    if (more) load(k0 + KT);
    const char *sa = lds + cur * BUF, *sb = sa + TA::BYTES;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      typename Frag<T>::type fa[MI], fb[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = TA::frag(sa, wm + i * 32, kk, lane);
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[j] = TB::frag(sb, wn + j * 32, kk, lane);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mma(fa[i], fb[j], acc[i][j], T());
    }
    if (more) stage(lds + (cur ^ 1) * BUF);
    __syncthreads();
    cur ^= 1;
  }

  // C leaves through LDS, 32 rows of the wave's own at a time: an accumulator holds one column per lane, memory wants 16 bytes of a row.
  constexpr int LD = WN + 4;
  float* c = (float*)lds + wave * 32 * LD;
  constexpr int OV = EPI == EPI_PARTIAL ? 4 : V, OW = GATED ? HALF : WN, LPR = OW / OV, RPP = 64 / LPR;  // output elements per lane, lanes per row, rows per pass
  const int col = (lane % LPR) * OV;
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
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    if (i) __syncthreads();
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) c[(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * LD + j * 32 + (lane & 31)] = acc[i][j][e];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 32 / RPP; ++q) {
      const int row = q * RPP + lane / LPR;
      const long long m = m0 + wm + i * 32 + row;
      if (m >= p.M || left <= 0) continue;
      float v[OV];
#pragma unroll
      for (int e = 0; e < OV; ++e) v[e] = c[row * LD + col + e];
      if constexpr (EPI == EPI_PARTIAL) {
        Chunk<float> out;
#pragma unroll
        for (int e = 0; e < OV; ++e) out.e[e] = v[e];
        store_part(p.partial + ((long long)blockIdx.y * p.M + m) * p.N + n, out, left);
      } else if constexpr (EPI == EPI_STORE) {
        Chunk<T> out;
#pragma unroll
        for (int e = 0; e < OV; ++e) out.e[e] = (T)v[e];
        store_part((T*)p.y + m * p.ldy + n, out, left);
      } else {
        Chunk<T> out, zs;
#pragma unroll
        for (int e = 0; e < OV; ++e) { v[e] += bias[e]; zs.e[e] = (T)v[e]; v[e] = act_value(v[e], p.act); }
        if (p.z) store_part((T*)p.z + m * p.N + n, zs, left);
        if constexpr (GATED) {
#pragma unroll
          for (int e = 0; e < OV; ++e) { const float u = c[row * LD + HALF + col + e] + bias_up[e]; zs.e[e] = (T)u; v[e] *= u; }
          if (p.z_up) store_part((T*)p.z_up + m * p.N + n, zs, left);
        } else if (p.r) {
          const Chunk<T> r = load_part((const T*)p.r + m * p.ldr + n, left);
#pragma unroll
          for (int e = 0; e < OV; ++e) v[e] += (float)r.e[e];
        }
#pragma unroll
        for (int e = 0; e < OV; ++e) out.e[e] = (T)v[e];
        store_part((T*)p.y + m * p.ldy + n, out, left);
      }
    }
  }
}

// out = sum over the splits, in the order of the splits
template <typename T> __global__ __launch_bounds__(256) void k_join_splits(const float* partial, T* out, long long n, long long stride, int splits) {
  const long long i = (blockIdx.x * 256LL + threadIdx.x) * 4;
  if (i >= n) return;
  const long long left = n - i;
  float s[4] = {};
  for (int k = 0; k < splits; ++k) {
    const Chunk<float> c = load_part(partial + k * stride + i, left);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += c.e[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) out[i + e] = (T)s[e];
}

// dz (rows, out | 2 out) from dy and the stored sums, and this row block's column sums for the bias gradient.
// 256 threads: 32 chunk columns x 8 rows at a time over SLOPE_ROWS rows; workgroups: row blocks x `colblocks`.  dz NULL: column sums of dy alone.
#define SLOPE_ROWS 128
template <typename T, bool GATED> __global__ __launch_bounds__(256) void k_layer_slope(const T* dy, long long ld_dy, const T* z, const T* z_up, T* dz, float* sums,
                                                                                        long long rows, long long out, unsigned colblocks, int act) {
  constexpr int V = Elem<T>::VEC, NS = GATED ? 2 : 1;
  __shared__ float part[NS][8][32 * V];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const unsigned bx = blockIdx.x % colblocks, by = blockIdx.x / colblocks;
  const long long n = (bx * 32LL + tx) * V, left = out - n, r0 = by * (long long)SLOPE_ROWS;
  float s[NS][V] = {};
  if (left > 0)
    for (int i = ty; i < SLOPE_ROWS && r0 + i < rows; i += 8) {
      const long long m = r0 + i;
      const Chunk<T> d = load_part(dy + m * ld_dy + n, left);
      Chunk<T> o, o2;
      if (dz && (GATED || act != MJLAB_ACT_NONE)) {
        const Chunk<T> g = load_part(z + m * out + n, left);
        Chunk<T> u;
        if constexpr (GATED) u = load_part(z_up + m * out + n, left);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float v = (float)d.e[e] * act_slope((float)g.e[e], act);
          if constexpr (GATED) {
            v *= (float)u.e[e];
            const float w = (float)d.e[e] * act_value((float)g.e[e], act);
            s[NS - 1][e] += w;
            o2.e[e] = (T)w;
          }
          s[0][e] += v;
          o.e[e] = (T)v;
        }
        store_part(dz + m * (NS * out) + n, o, left);
        if constexpr (GATED) store_part(dz + m * (NS * out) + out + n, o2, left);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) s[0][e] += (float)d.e[e];
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
