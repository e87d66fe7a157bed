// policy.hip -- C ABI of include/mjlab_policy.h: argument checks and the choice of the element type; the kernels live in layer_inst.hip.
#include "policy_launch.h"

#include <cstdio>

static thread_local char g_error[256] = "";

static int fail(int rc, const char* what) {
  snprintf(g_error, sizeof(g_error), "%s%s%s", what, rc > 0 ? ": " : "", rc > 0 ? hipGetErrorString((hipError_t)rc) : "");
  return rc;
}
static int done(hipError_t e, const char* what) { return e == hipSuccess ? 0 : fail((int)e, what); }

// f(args) of the element type `dtype`
#define BY_TYPE(dtype, f, ...) ((dtype) == MJLAB_DTYPE_F32 ? f##_f32(__VA_ARGS__) : (dtype) == MJLAB_DTYPE_F16 ? f##_f16(__VA_ARGS__) : f##_bf16(__VA_ARGS__))

static bool bad_type(int dtype) { return dtype < MJLAB_DTYPE_F32 || dtype > MJLAB_DTYPE_BF16; }

static int check_layer(const mjlab_layer_t& f) {
  if (bad_type(f.dtype)) return fail(-2, "layer: unknown dtype");
  if (f.act < 0 || f.act >= MJLAB_ACT_COUNT) return fail(-2, "layer: unknown activation");
  // in, out < 2^31 and rows < 2^37 keep every product of two sizes and an element size inside 64 bits with room to spare
  if (f.rows < 1 || f.in < 1 || f.out < 1 || f.in >= (1LL << 30) || f.out >= (1LL << 30) || f.rows >= (1LL << 31)) return fail(-2, "layer: sizes must be positive (in, out below 2^30, rows below 2^31)");
  if (!f.x || !f.w) return fail(-2, "layer: null x or w");
  if ((f.rows > 1 && f.ldx < 0) || (f.out > 1 && f.ldw < 0) || (f.w_up && f.out > 1 && f.ldw_up < 0)) return fail(-2, "layer: negative row stride");
  return 0;
}

extern "C" {

int mjlab_policy_abi_version(void) { return MJLAB_POLICY_ABI_VERSION; }
const char* mjlab_policy_last_error(void) { return g_error; }
int mjlab_sizeof_layer(void) { return (int)sizeof(mjlab_layer_t); }
int mjlab_sizeof_layer_grad(void) { return (int)sizeof(mjlab_layer_grad_t); }

int mjlab_layer_forward(const mjlab_layer_t* f, void* stream) {
  if (!f) return fail(-1, "layer_forward: null argument");
  int rc = check_layer(*f);
  if (rc) return rc;
  if (!f->y) return fail(-2, "layer_forward: null y");
  if (f->rows > 1 && f->ldy < f->out) return fail(-2, "layer_forward: the rows of y overlap");
  if (f->r && f->w_up) return fail(-2, "layer_forward: a gated layer takes no residual");
  if (f->b_up && !f->w_up) return fail(-2, "layer_forward: b_up without w_up");
  if (f->z_up && !f->w_up) return fail(-2, "layer_forward: z_up without w_up");
  return done(BY_TYPE(f->dtype, mjlab_launch_layer_forward, f, (hipStream_t)stream), "layer_forward launch failed");
}

long long mjlab_layer_backward_workspace(const mjlab_layer_grad_t* g) {
  if (!g) return fail(-1, "layer_backward_workspace: null argument");
  if (check_layer(g->f)) return -1;
  return BY_TYPE(g->f.dtype, mjlab_layer_backward_bytes, g);
}

int mjlab_layer_backward(const mjlab_layer_grad_t* g, void* stream) {
  if (!g) return fail(-1, "layer_backward: null argument");
  int rc = check_layer(g->f);
  if (rc) return rc;
  const bool gated = g->f.w_up != nullptr;
  if (!g->dy) return fail(-2, "layer_backward: null dy");
  if ((gated || g->f.act != MJLAB_ACT_NONE) && !g->f.z) return fail(-2, "layer_backward: the sums before the activation (z) are missing");
  if (gated && !g->f.z_up) return fail(-2, "layer_backward: z_up is missing");
  if (gated && ((g->dw != nullptr) != (g->dw_up != nullptr) || (g->db != nullptr) != (g->db_up != nullptr))) return fail(-2, "layer_backward: dw / dw_up and db / db_up come together");
  const long long need = BY_TYPE(g->f.dtype, mjlab_layer_backward_bytes, g);
  if (need > 0 && (!g->workspace || g->workspace_bytes < need)) return fail(-3, "layer_backward: workspace too small");
  return done(BY_TYPE(g->f.dtype, mjlab_launch_layer_backward, g, (hipStream_t)stream), "layer_backward launch failed");
}

}  // extern "C"
