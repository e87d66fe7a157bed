// policy.hip -- C ABI of include/mjlab_policy.h: argument checks and the choice of the element type; the kernels live in layer_inst.hip, decay_inst.hip and short_inst.hip.
#include "policy_common.h"
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
  if (f.rows < 1 || f.in < 1 || f.out < 1 || f.in >= (1LL << 30) || f.out >= (1LL << 27) || f.rows >= (1LL << 31)) return fail(-2, "layer: sizes must be positive (in below 2^30, out below 2^27, rows below 2^31)");
  // 2^44 elements are more than any memory holds: the sizes of workspaces (up to 512 times a matrix of floats) stay inside 64 bits
  if (f.rows * f.in >= (1LL << 44) || f.rows * f.out >= (1LL << 44) || f.in * f.out >= (1LL << 44)) return fail(-2, "layer: the product of two sizes must be below 2^44");
  if (!f.x || !f.w) return fail(-2, "layer: null x or w");
  if ((f.rows > 1 && f.ldx < 0) || (f.out > 1 && f.ldw < 0) || (f.w_up && f.out > 1 && f.ldw_up < 0)) return fail(-2, "layer: negative row stride");
  return 0;
}

extern "C" {

int mjlab_policy_abi_version(void) { return MJLAB_POLICY_ABI_VERSION; }
const char* mjlab_policy_last_error(void) { return g_error; }
int mjlab_sizeof_layer(void) { return (int)sizeof(mjlab_layer_t); }
int mjlab_sizeof_layer_grad(void) { return (int)sizeof(mjlab_layer_grad_t); }

static int check_z(const mjlab_layer_t& f) {
  return (f.z || f.z_up) && f.z_bytes != 4 ? fail(-2, "layer: z_bytes: the sums before the activation are floats") : 0;
}

int mjlab_layer_recomputes(const mjlab_layer_t* f) {
  if (!f || check_layer(*f)) return 0;
  return BY_TYPE(f->dtype, mjlab_layer_again, f);
}

int mjlab_layer_tile(const mjlab_layer_t* f, int product) {
  if (!f || product < MJLAB_PRODUCT_FORWARD || product > MJLAB_PRODUCT_WEIGHT || check_layer(*f)) return 0;
  return BY_TYPE(f->dtype, mjlab_layer_tile_of, f, product);
}

long long mjlab_layer_forward_workspace(const mjlab_layer_t* f) {
  if (!f) return fail(-1, "layer_forward_workspace: null argument");
  if (check_layer(*f)) return -1;
  return BY_TYPE(f->dtype, mjlab_layer_forward_bytes, f);
}

int mjlab_layer_forward(const mjlab_layer_t* f, void* stream) {
  if (!f) return fail(-1, "layer_forward: null argument");
  int rc = check_layer(*f);
  if (rc) return rc;
  if (!f->y) return fail(-2, "layer_forward: null y");
  if (f->rows > 1 && f->ldy < f->out) return fail(-2, "layer_forward: the rows of y overlap");
  if (f->r && f->w_up) return fail(-2, "layer_forward: a gated layer takes no residual");
  if (f->b_up && !f->w_up) return fail(-2, "layer_forward: b_up without w_up");
  if (f->z_up && !f->w_up) return fail(-2, "layer_forward: z_up without w_up");
  if ((rc = check_z(*f))) return rc;
  const long long need = BY_TYPE(f->dtype, mjlab_layer_forward_bytes, f);
  if (need > 0 && (!f->workspace || f->workspace_bytes < need)) return fail(-3, "layer_forward: workspace too small");
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
  const bool again = gated && !g->f.z && !g->f.z_up && mjlab_layer_recomputes(&g->f);
  if (!again && (gated || g->f.act != MJLAB_ACT_NONE) && !g->f.z) return fail(-2, "layer_backward: the sums before the activation (z) are missing");
  if (g->f.z_is_y && (gated || g->f.dtype != MJLAB_DTYPE_F32 || !slope_from_output(g->f.act))) return fail(-2, "layer_backward: z_is_y: the output does not determine this layer's slope");
  if (gated && !again && !g->f.z_up) return fail(-2, "layer_backward: z_up is missing");
  if ((rc = check_z(g->f))) return rc;
  if (gated && ((g->dw != nullptr) != (g->dw_up != nullptr) || (g->db != nullptr) != (g->db_up != nullptr))) return fail(-2, "layer_backward: dw / dw_up and db / db_up come together");
  const long long need = BY_TYPE(g->f.dtype, mjlab_layer_backward_bytes, g);
  if (need > 0 && (!g->workspace || g->workspace_bytes < need)) return fail(-3, "layer_backward: workspace too small");
  return done(BY_TYPE(g->f.dtype, mjlab_launch_layer_backward, g, (hipStream_t)stream), "layer_backward launch failed");
}

static int check_decay(const mjlab_decay_t& d) {
  if (bad_type(d.dtype)) return fail(-2, "decay: unknown dtype");
  if (d.batch < 1 || d.heads < 1 || d.length < 1 || d.batch >= (1LL << 31) || d.length >= (1LL << 31) || d.batch * d.heads >= (1LL << 24)) return fail(-2, "decay: batch, length and heads must be positive (batch x heads below 2^24)");
  if (d.dk < 1 || d.dv < 1 || d.dk > MJLAB_DECAY_MAX_DIM || d.dv > MJLAB_DECAY_MAX_DIM) return fail(-2, "decay: dk and dv must be in [1, MJLAB_DECAY_MAX_DIM]");
  if (!d.q.p || !d.k.p || !d.v.p || !d.log_decay) return fail(-2, "decay: null q, k, v or log_decay");
  if (d.reset && d.reset_bytes != 1 && d.reset_bytes != 4) return fail(-2, "decay: reset_bytes must be 1 or 4");
  return 0;
}

int mjlab_sizeof_decay(void) { return (int)sizeof(mjlab_decay_t); }
int mjlab_sizeof_decay_grad(void) { return (int)sizeof(mjlab_decay_grad_t); }

long long mjlab_decay_workspace(const mjlab_decay_t* d) {
  if (!d) return fail(-1, "decay_workspace: null argument");
  if (check_decay(*d)) return -1;
  return BY_TYPE(d->dtype, mjlab_decay_bytes, d);
}

static int check_decay_workspace(const mjlab_decay_t& d) {
  const long long need = BY_TYPE(d.dtype, mjlab_decay_bytes, &d);
  return need > 0 && (!d.workspace || d.workspace_bytes < need) ? fail(-3, "decay: workspace too small") : 0;
}

int mjlab_decay_forward(const mjlab_decay_t* d, void* stream) {
  if (!d) return fail(-1, "decay_forward: null argument");
  int rc = check_decay(*d);
  if (rc) return rc;
  if (!d->o.p) return fail(-2, "decay_forward: null o");
  if (d->state && d->state == d->state_out) return fail(-2, "decay_forward: state_out must not be state");
  if ((rc = check_decay_workspace(*d))) return rc;
  return done(BY_TYPE(d->dtype, mjlab_launch_decay_forward, d, (hipStream_t)stream), "decay_forward launch failed");
}

int mjlab_decay_backward(const mjlab_decay_grad_t* g, void* stream) {
  if (!g) return fail(-1, "decay_backward: null argument");
  int rc = check_decay(g->f);
  if (rc) return rc;
  if (!g->d_out.p) return fail(-2, "decay_backward: null d_out");
  if (g->d_state && (!g->dv.p || g->d_state == g->d_state_out)) return fail(-2, "decay_backward: d_state comes with dv and must not be d_state_out");
  if ((rc = check_decay_workspace(g->f))) return rc;
  if (g->segments && g->segments == g->f.workspace) return fail(-2, "decay_backward: segments must not be the workspace");
  return done(BY_TYPE(g->f.dtype, mjlab_launch_decay_backward, g, (hipStream_t)stream), "decay_backward launch failed");
}

int mjlab_decay_step(const mjlab_decay_t* d, void* stream) {
  if (!d) return fail(-1, "decay_step: null argument");
  int rc = check_decay(*d);
  if (rc) return rc;
  if (d->length != 1) return fail(-2, "decay_step: length must be 1");
  if (!d->o.p || !d->state || !d->state_out) return fail(-2, "decay_step: null o, state or state_out");
  if (d->lengths) return fail(-2, "decay_step: lengths do not apply to one token");
  return done(BY_TYPE(d->dtype, mjlab_launch_decay_step, d, (hipStream_t)stream), "decay_step launch failed");
}

}  // extern "C"
