// layer_inst.hip -- the layers' launches for ONE element type: compiled with -DMJLAB_POLICY_DTYPE=<0 f32 | 1 f16 | 2 bf16> (mjlab_amd/native.py).
#include "policy_type.h"
#include "product.h"

namespace {

template <typename TA, bool AK, bool BK, int BM, int BN, int EPI> hipError_t launch_tile(const Product& p, int splits, hipStream_t st) {
  constexpr int BNO = EPI == EPI_GATED || EPI == EPI_SLOPE ? BN / 2 : BN, LDS = ProductLds<TA, T, AK, BK, BM, BN, EPI>::BYTES;
  const long long tiles = ((p.M + BM - 1) / BM) * ((p.N + BNO - 1) / BNO);
  if (tiles > MAX_BLOCKS) return hipErrorInvalidValue;
  auto kern = k_product<TA, T, AK, BK, BM, BN, EPI>;
  static std::atomic<unsigned long long> asked{0};
  if (hipError_t e = allow_lds(kern, LDS, asked); e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles, (unsigned)splits), dim3(256), LDS, st, p);
  return hipGetLastError();
}

// The tile, by an estimate of the time in units of a 256 x 128 tile's share of a CU: `n` tiles of cost `c` for the CU that gets most, of which R run there at
// once; a round with fewer takes up to 0.4 of a tile longer than its share, since nothing hides what it waits for.  Per element of C a smaller tile costs
// more: 128 x 128 12 % (24 % where an operand has to be turned), 64 x 64 60 % (124 %); float, whose matrix instructions take longer, 33 % over 128 x 128.
// Measured (us; 256 x 128 / 128 x 128 / 64 x 64): bf16 y of 16384 x 2048 x 2816 226 / 234 / 351, 24576 x 512 x 1365 71 / 63 / 83,
// 4096 x 1024 x 1024 30 / 20 / 24; dx of a layer without activation, 24576 x 512 x 1365, 66 / 77 / 90; float y of 24576 x 1024 x 1024 - / 278 / 368, 512 x 2048 x 2048 - / 116 / 52.
float tile_cost(long long tiles, float cost, int at_once) {
  const long long n = (tiles + CUS - 1) / CUS, rest = n % at_once;
  return cost * (n + (rest ? 0.4f * (at_once - rest) / (at_once - 1) : 0.f));
}

// A layer's epilogue (BK: the products that have one) is hidden behind the other workgroups of a CU, of which the large tile leaves one: counted as 0.13 of the
// large tile's time at 1024 k (gated bf16 24576 rows, y, us, large / mid: 512 x 1365 122 / 110; 1024 x 2048 264 / 264).
// TA: what memory holds A as: float for dz, also where T has 16 bits.  There 128 x 128 costs a quarter less than 64 x 64, and a 256 x 128 tile has no registers left.
// (dx with its slope kernel, 128 x 128 / 64 x 64, us: bf16 24576 x 1024 x 1024 201 / 239, 4096 x 1024 x 1024 49 / 49, 1024 x 512 x 512 29 / 22;
// fp16 237 / 292, 58 / 59, 33 / 23.)
struct Choice {
  int rows;  // the tile: 64 x 64, 128 x 128 or 256 x 128
  float cost;
};
template <typename TA, bool BK> Choice choose(long long M, long long width, long long K, long long splits) {
  auto tiles = [&](int bm, int bn) { return (M + bm - 1) / bm * ((width + bn - 1) / bn) * splits; };
  constexpr bool F32 = sizeof(T) == 4, MIXED = sizeof(TA) != sizeof(T);
  const float small = tile_cost(tiles(64, 64), F32 ? 0.166f : BK || MIXED ? 0.2f : 0.28f, F32 ? 3 : 5);
  const float mid = tile_cost(tiles(128, 128), F32 ? 0.5f : BK ? 0.56f : 0.62f, BK ? 3 : 2);
  const float large = F32 || MIXED ? 1e30f : tile_cost(tiles(256, 128), BK ? 1.f + 133.f / K : 1.f, 2);
  return large < mid && large < small ? Choice{256, large} : mid < small ? Choice{128, mid} : Choice{64, small};
}

template <typename TA, bool AK, bool BK, int EPI> hipError_t launch_product(const Product& p, int splits, hipStream_t st) {
  const int rows = choose<TA, BK>(p.M, EPI == EPI_GATED || EPI == EPI_SLOPE ? 2 * p.N : p.N, p.K, splits).rows;
  if constexpr (sizeof(TA) == 2)
    if (rows == 256) return launch_tile<TA, AK, BK, 256, 128, EPI>(p, splits, st);
  return rows == 128 ? launch_tile<TA, AK, BK, 128, 128, EPI>(p, splits, st) : launch_tile<TA, AK, BK, 64, 64, EPI>(p, splits, st);
}

// Few rows leave most CUs idle: the sum over k is then split, each part's sums go through memory, and a second launch joins them.  The time of an unsplit unit of
// tile_cost() is about 21 ns per k (float 80 ns, dz in 16 bits 42 ns), the second launch 4 us and what it reads at 3 TB/s.
// (64 rows, 2048 x 2048: float 49 us unsplit, 12 + 4 us split; bf16 17 us, 6 + 3 us.)
template <typename TA, bool BK> int sum_splits(long long M, long long width, long long K) {
  const float per_k = sizeof(T) == 4 ? 0.08f : sizeof(TA) == 4 ? 0.042f : 0.021f;
  int best = 1;
  float time = choose<TA, BK>(M, width, K, 1).cost * K * per_k;
  for (int s = 2; s <= 32 && K / s >= 128; s *= 2) {
    const float t = choose<TA, BK>(M, width, K, s).cost * K / s * per_k + 4.f + 4e-6f * M * width * s * 0.67f;
    if (t < time) { time = t; best = s; }
  }
  return best;
}
long long per_split(long long K, int splits) { return ((K + splits - 1) / splits + 63) / 64 * 64; }
int parts(long long K, int splits) { return (int)((K + per_split(K, splits) - 1) / per_split(K, splits)); }

// How many ways the sum over the rows is split in dw = dz^T x: few tiles, many rows.
int weight_splits(long long out, long long in, long long rows) {
  const long long tiles = ((out + 127) / 128) * ((in + 127) / 128);
  const long long most = (rows + 255) / 256, want = 2 * CUS / tiles;
  const long long s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s);
}

long long up256(long long x) { return (x + 255) & ~255LL; }

struct Plan {
  bool gated, slope, sums, weights, again;
  long long ns, blocks, o_dz, o_sums, o_partial, bytes;
  int splits, x_splits;
};

Plan plan(const mjlab_layer_grad_t* g) {
  const mjlab_layer_t& f = g->f;
  Plan q;
  q.gated = f.w_up != nullptr;
  q.ns = q.gated ? 2 : 1;
  q.slope = q.gated || f.act != MJLAB_ACT_NONE;
  q.sums = g->db != nullptr;
  q.weights = g->dw != nullptr;
  q.again = q.gated && !f.z;
  q.blocks = (f.rows + SLOPE_ROWS - 1) / SLOPE_ROWS;
  if (q.again) {  // two sets of column sums per tile of rows
    const int bm = choose<T, true>(f.rows, 2 * f.out, f.in, 1).rows;
    q.blocks = 2 * ((f.rows + bm - 1) / bm);
  }
  q.splits = weight_splits(q.ns * f.out, f.in, f.rows);
  long long at = 0;
  q.o_dz = at;
  if (q.slope) at += up256(f.rows * q.ns * f.out * 4);
  q.o_sums = at;
  if (q.sums) at += up256(q.blocks * q.ns * f.out * 4);
  const long long k = q.ns * f.out;
  q.x_splits = !g->dx ? 1 : q.slope ? sum_splits<float, false>(f.rows, f.in, k) : sum_splits<T, false>(f.rows, f.in, k);
  q.o_partial = at;  // (dx's sums are joined before dw's are formed)
  const long long w = q.weights && (q.splits > 1 || q.gated) ? q.splits * k * f.in : 0, x = q.x_splits > 1 ? q.x_splits * f.rows * f.in : 0;
  at += up256((w > x ? w : x) * 4);
  q.bytes = at;
  return q;
}

int forward_splits(const mjlab_layer_t* f) { return sum_splits<T, true>(f->rows, f->w_up ? 2 * f->out : f->out, f->in); }

Product forward_product(const mjlab_layer_t* f) {
  Product p = {};
  p.A = f->x; p.lda = f->ldx; p.B = f->w; p.ldb = f->ldw; p.B2 = f->w_up; p.ldb2 = f->ldw_up;
  p.M = f->rows; p.N = p.nb2 = f->out; p.K = p.kb2 = p.ksplit = f->in;
  p.act = f->act; p.b = f->b; p.b_up = f->b_up; p.r = f->r; p.ldr = f->ldr; p.y = f->y; p.ldy = f->ldy; p.z = (float*)f->z; p.z_up = (float*)f->z_up;
  return p;
}

// dx and dw (dw_up) from d, the gradient of the sums before the activation: rows of q.ns out, `ldd` apart
template <typename TA> hipError_t input_gradient(const mjlab_layer_grad_t* g, const Plan& q, const void* d, long long ldd, float* partial, hipStream_t st) {
  const mjlab_layer_t& f = g->f;
  Product p = {};
  p.A = d; p.lda = ldd; p.B = f.w; p.ldb = f.ldw; p.B2 = f.w_up; p.ldb2 = f.ldw_up;
  p.M = f.rows; p.N = p.nb2 = f.in; p.K = p.ksplit = q.ns * f.out; p.kb2 = f.out;
  p.y = g->dx; p.ldy = f.in; p.partial = partial;
  if (q.x_splits == 1) return launch_product<TA, true, false, EPI_STORE>(p, 1, st);
  p.ksplit = per_split(p.K, q.x_splits);
  const int splits = parts(p.K, q.x_splits);
  const long long n = f.rows * f.in;
  if ((n + 255) / 256 > MAX_BLOCKS) return hipErrorInvalidValue;
  if (hipError_t e = launch_product<TA, true, false, EPI_PARTIAL>(p, splits, st); e != hipSuccess) return e;
  hipLaunchKernelGGL(k_join_splits<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, partial, (T*)g->dx, n, n, splits);
  return hipGetLastError();
}

template <typename TA> hipError_t weight_gradient(const mjlab_layer_grad_t* g, const Plan& q, const void* d, long long ldd, float* partial, hipStream_t st) {
  const mjlab_layer_t& f = g->f;
  Product p = {};
  p.A = d; p.lda = ldd; p.B = f.x; p.ldb = f.ldx;
  p.M = q.ns * f.out; p.N = p.nb2 = f.in; p.K = p.kb2 = f.rows;
  p.ksplit = per_split(f.rows, q.splits);
  const int splits = parts(f.rows, q.splits);
  p.y = g->dw; p.ldy = f.in; p.partial = partial;
  if (splits == 1 && !q.gated) return launch_product<TA, false, false, EPI_STORE>(p, 1, st);
  if (hipError_t e = launch_product<TA, false, false, EPI_PARTIAL>(p, splits, st); e != hipSuccess) return e;
  const long long n = f.out * f.in;
  if ((n + 255) / 256 > MAX_BLOCKS) return hipErrorInvalidValue;
  for (int u = 0; u < (q.gated ? 2 : 1); ++u) {
    // (partials: splits x a gated layer's two matrices)
    hipLaunchKernelGGL(k_join_splits<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, partial + u * n, (T*)(u ? g->dw_up : g->dw), n, q.ns * n, splits);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

// 16-bit gated layers up to this many inputs form their sums again in the backward pass, inside the launch that turns dy into [dg | du].
int POLICY_NAME(mjlab_layer_again)(const mjlab_layer_t* f) { return sizeof(T) == 2 && f->w_up && f->in <= 1024; }

hipError_t POLICY_NAME(mjlab_launch_layer_forward)(const mjlab_layer_t* f, hipStream_t st) {
  Product p = forward_product(f);
  const int s = forward_splits(f);
  if (s == 1) return f->w_up ? launch_product<T, true, true, EPI_GATED>(p, 1, st) : launch_product<T, true, true, EPI_LAYER>(p, 1, st);
  Product q = p;
  q.N = f->w_up ? 2 * f->out : f->out;
  q.ksplit = per_split(f->in, s);
  q.partial = p.partial = (float*)f->workspace;
  const int splits = parts(f->in, s);
  if (hipError_t e = launch_product<T, true, true, EPI_PARTIAL>(q, splits, st); e != hipSuccess) return e;
  const long long blocks = (f->rows * f->out + 255) / 256;
  if (blocks > MAX_BLOCKS) return hipErrorInvalidValue;
  auto join = f->w_up ? k_join_layer<T, true> : k_join_layer<T, false>;
  hipLaunchKernelGGL(join, dim3((unsigned)blocks), dim3(256), 0, st, p, splits);
  return hipGetLastError();
}

long long POLICY_NAME(mjlab_layer_forward_bytes)(const mjlab_layer_t* f) {
  const int s = forward_splits(f);
  return s == 1 ? 0 : up256(s * f->rows * (f->w_up ? 2 : 1) * f->out * 4);
}

int POLICY_NAME(mjlab_layer_tile_of)(const mjlab_layer_t* f, int product) {
  mjlab_layer_grad_t g = {};
  g.f = *f; g.dx = g.dw = (void*)1;  // (only asked for being there)
  const Plan q = plan(&g);
  if (product == MJLAB_PRODUCT_FORWARD) {
    const int s = forward_splits(f);
    const int rows = choose<T, true>(f->rows, q.ns * f->out, f->in, s == 1 ? 1 : parts(f->in, s)).rows;
    return s == 1 ? rows : -rows;
  }
  if (product == MJLAB_PRODUCT_INPUT) {
    const long long k = q.ns * f->out, s = q.x_splits == 1 ? 1 : parts(k, q.x_splits);
    const int rows = q.slope ? choose<float, false>(f->rows, f->in, k, s).rows : choose<T, false>(f->rows, f->in, k, s).rows;
    return q.x_splits == 1 ? rows : -rows;
  }
  const int s = parts(f->rows, q.splits);
  const int rows = q.slope ? choose<float, false>(q.ns * f->out, f->in, f->rows, s).rows : choose<T, false>(q.ns * f->out, f->in, f->rows, s).rows;
  return s == 1 && !q.gated ? rows : -rows;
}

long long POLICY_NAME(mjlab_layer_backward_bytes)(const mjlab_layer_grad_t* g) { return plan(g).bytes; }

hipError_t POLICY_NAME(mjlab_launch_layer_backward)(const mjlab_layer_grad_t* g, hipStream_t st) {
  const mjlab_layer_t& f = g->f;
  const Plan q = plan(g);
  char* ws = (char*)g->workspace;
  float* dz = (float*)(ws + q.o_dz);
  float *sums = q.sums ? (float*)(ws + q.o_sums) : nullptr, *partial = (float*)(ws + q.o_partial);
  hipError_t e = hipSuccess;
  if (q.again) {
    if constexpr (sizeof(T) == 2) {
      Product p = forward_product(&f);
      p.r = g->dy; p.ldr = g->ld_dy; p.y = dz; p.ldy = 2 * f.out; p.z = p.z_up = nullptr; p.partial = sums;
      if ((e = launch_product<T, true, true, EPI_SLOPE>(p, 1, st)) != hipSuccess) return e;
    } else return hipErrorInvalidValue;
  } else if (q.slope || q.sums) {
    constexpr int V = Elem<T>::VEC;
    const long long colblocks = (f.out + 32 * V - 1) / (32 * V);
    if (colblocks * q.blocks > MAX_BLOCKS) return hipErrorInvalidValue;
    auto kern = q.gated ? k_layer_slope<T, true, false> : sizeof(T) == 4 && f.z_is_y ? k_layer_slope<T, false, sizeof(T) == 4> : k_layer_slope<T, false, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(colblocks * q.blocks)), dim3(256), 0, st, (const T*)g->dy, g->ld_dy, (const float*)f.z, (const float*)f.z_up, q.slope ? dz : nullptr, q.ns * f.out, sums, f.rows, f.out, (unsigned)colblocks, f.act);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (q.sums) {
    const long long cols = q.ns * f.out;
    hipLaunchKernelGGL(k_join_sums<T>, dim3((unsigned)((cols + 15) / 16)), dim3(256), 0, st, sums, (T*)g->db, (T*)g->db_up, f.out, cols, q.blocks);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (q.slope) {
    if (g->dx && (e = input_gradient<float>(g, q, dz, q.ns * f.out, partial, st)) != hipSuccess) return e;
    return g->dw ? weight_gradient<float>(g, q, dz, q.ns * f.out, partial, st) : hipSuccess;
  }
  if (g->dx && (e = input_gradient<T>(g, q, g->dy, g->ld_dy, partial, st)) != hipSuccess) return e;
  return g->dw ? weight_gradient<T>(g, q, g->dy, g->ld_dy, partial, st) : hipSuccess;
}
