/*
 * Autograd nodes of the operators along a sequence: the short causal convolution, the selective state space scan, and the norms
 * around a block.  They follow the matmul nodes (op_matmul.c): RecPulse's Tensor / Meta / GradFn structs in place, strided column
 * blocks read as they lie, gradients written straight into new or added to existing grad tensors, workspaces from the pool in the
 * node stream's order.  What a backward call needs beside its inputs rides along as an extra input without Meta, which RecPulse's
 * tensor_backward skips (core/tensor.c:251, 296) and its free_grad_fn releases (ops/ops.c:7227-7322).
 */
#include <cuda_runtime_api.h>
#include <limits.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "rpb_common.h"

cudaStream_t rpb_current_node_stream(void);     /* op_matmul.c */
int rpb_finish_node(int device_id);
int rpb_attach_node(Tensor* out, BackwardFunction backward, Tensor** in, int n_in);

static bool wanted(const Tensor* t) { return t && t->metadata && t->metadata->requires_grad; }

static bool packed(const Tensor* t) {
    long long s = 1;
    for (int d = t->ndim - 1; d >= 0; d--) { if (t->strides[d] != s) return false; s *= t->shape[d]; }
    return true;
}

static Tensor* refused(const char* op, const char* why) {
    fprintf(stderr, "recpulse_b200: %s: %s\n", op, why);
    return NULL;
}

static bool empty(const Tensor* t) {
    for (int d = 0; t && d < t->ndim; d++)
        if (t->shape[d] <= 0) return true;
    return false;
}

/* [batch, len, cols] with unit stride within a row, on x's device and of its type */
static bool sequence_ok(const Tensor* t, const Tensor* x, int cols) {
    return t && t->ndim == 3 && t->dtype == x->dtype && t->device_id == x->device_id && t->shape[0] == x->shape[0] && t->shape[1] == x->shape[1] &&
           t->shape[2] == cols && (cols == 1 || t->strides[2] == 1) && t->strides[0] >= 0 && t->strides[1] >= 0;
}

static bool vector_ok(const Tensor* t, DType dtype, int device_id, long long elems) {
    return t->dtype == dtype && t->device_id == device_id && (long long)t->size == elems && packed(t);
}

/* A gradient is added to the grad of its input; the same tensor in two places of one node would need two sums into one buffer. */
static bool twice(Tensor** in, int n) {
    for (int i = 0; i < n; i++)
        for (int k = 0; k < i; k++)
            if (in[i] && in[i] == in[k] && wanted(in[i])) return true;
    return false;
}

/* The buffer that an input's gradient goes to: its existing grad (*add = bit) or a new tensor.  NULL in *data: not wanted. */
typedef struct { Tensor* of; Tensor* fresh; } Target;
static int target_of(Tensor* t, Target* target, void** data, int* accumulate, int bit) {
    target->of = t; target->fresh = NULL;
    *data = NULL;
    if (!wanted(t)) return 0;
    Tensor* have = t->metadata->grad;
    if (have) {
        if (!packed(have) || have->size != t->size || have->dtype != t->dtype || have->device_id != t->device_id) {
            fprintf(stderr, "recpulse_b200: existing grad is not a packed tensor of the input's shape\n");
            return -1;
        }
        *accumulate |= bit;
        *data = have->data;
        return 0;
    }
    target->fresh = rpb_tensor_empty(t->dtype, t->ndim, t->shape, t->device_id);
    if (!target->fresh) return -1;
    *data = target->fresh->data;
    return 0;
}
/* New grads become their inputs', or are released when the call failed. */
static void settle(Target* t, int n, int rc) {
    for (int i = 0; i < n; i++) {
        if (!t[i].fresh) continue;
        if (rc == 0) t[i].of->metadata->grad = t[i].fresh;
        else rpb_tensor_release(t[i].fresh);
    }
}

static Tensor* workspace(long long bytes, int device_id) {
    int shape[2] = {0, 1024};
    const long long rows = (bytes + 4095) / 4096;
    if (bytes < 0 || rows > INT_MAX) return NULL;
    shape[0] = rows > 0 ? (int)rows : 1;
    return rpb_tensor_empty(DTYPE_FLOAT32, 2, shape, device_id);
}

/* ------------------------------------------------------------------ causal convolution */

typedef struct { int activation, has_bias; } ConvSaved;

static void conv_geometry(RpbCausalConv* c, const Tensor* x, const Tensor* w, int activation) {
    rpb_causal_conv_packed(c, x->shape[0], x->shape[1], x->shape[2], w->shape[1], activation);
    c->x_batch = x->strides[0]; c->x_row = x->strides[1];
}

Tensor* op_causal_conv(Tensor* x, Tensor* w, Tensor* bias, int activation) {
    const char* op = "op_causal_conv";
    if (!x || !w || x->ndim != 3 || w->ndim != 2) return NULL;
    if (x->device_id < 0) return refused(op, "host tensors: this library has no CPU path");
    if (empty(x) || empty(w)) return refused(op, "a dimension of size 0");
    if (!sequence_ok(x, x, x->shape[2]) || w->shape[0] != x->shape[2]) return refused(op, "x is [batch, len, channels], w [channels, width]");
    if (!vector_ok(w, x->dtype, x->device_id, (long long)w->shape[0] * w->shape[1])) return refused(op, "w must be packed, of x's type and device");
    if (bias && !vector_ok(bias, x->dtype, x->device_id, x->shape[2])) return refused(op, "bias must be packed, of x's type and device");
    Tensor* in[3] = {x, w, bias};
    if (twice(in, 3)) return refused(op, "one tensor in two places");
    RpbCausalConv c;
    conv_geometry(&c, x, w, activation);
    Tensor* out = rpb_tensor_empty(x->dtype, 3, x->shape, x->device_id);
    if (!out) return NULL;
    int rc = rp_causal_conv_ex(out->data, NULL, x->data, w->data, bias ? bias->data : NULL, NULL, NULL, &c, x->dtype, x->device_id,
                               rpb_current_node_stream());
    if (rc == 0) rc = rpb_finish_node(x->device_id);
    if (rc == 0 && (wanted(x) || wanted(w) || wanted(bias))) {
        ConvSaved* saved = (ConvSaved*)malloc(sizeof(ConvSaved));
        if (!saved || rpb_attach_node(out, backward_causal_conv_fn, in, bias ? 3 : 2)) { free(saved); rc = -1; }
        else { saved->activation = activation; saved->has_bias = bias != NULL; out->metadata->grad_fn->saved_data = saved; }
    }
    if (rc != 0) { rpb_tensor_release(out); return NULL; }
    return out;
}

void backward_causal_conv_fn(GradFn* self, Tensor* grad_output) {
    if (!self || !grad_output || !self->inputs || !self->saved_data) return;
    const ConvSaved* saved = (const ConvSaved*)self->saved_data;
    if (self->num_inputs != 2 + saved->has_bias) return;
    Tensor *x = self->inputs[0], *w = self->inputs[1], *bias = saved->has_bias ? self->inputs[2] : NULL;
    if (!x || !w || x->device_id < 0 || !sequence_ok(grad_output, x, x->shape[2])) {
        refused("op_causal_conv backward", "the upstream gradient must be [batch, len, channels] like the output");
        return;
    }
    RpbCausalConv c;
    conv_geometry(&c, x, w, saved->activation);
    c.y_batch = grad_output->strides[0]; c.y_row = grad_output->strides[1];
    Target t[3];
    void *dx = NULL, *dw = NULL, *db = NULL;
    memset(t, 0, sizeof(t));
    int acc = 0;
    int rc = target_of(x, &t[0], &dx, &acc, RPB_CONV_ACC_DX) || target_of(w, &t[1], &dw, &acc, RPB_CONV_ACC_DW) ||
             target_of(bias, &t[2], &db, &acc, RPB_CONV_ACC_DBIAS) ? -1 : 0;
    if (rc == 0 && (dx || dw || db)) {
        Tensor* ws = workspace(rp_causal_conv_ws_bytes(&c, x->dtype), x->device_id);
        rc = ws ? rp_causal_conv_grad_ex(dx, dw, db, NULL, acc, grad_output->data, NULL, x->data, w->data, bias ? bias->data : NULL, NULL, NULL, ws->data,
                                         &c, x->dtype, x->device_id, rpb_current_node_stream()) : -1;
        if (rc == 0) rc = rpb_finish_node(x->device_id);
        rpb_tensor_release(ws);
    }
    settle(t, 3, rc);
}

/* ------------------------------------------------------------------ selective scan */

typedef struct { int softplus, has_D, has_bias, has_z, groups; } ScanSaved;

static void scan_geometry(RpbScan* c, const Tensor* x, const Tensor* dt, const Tensor* A, const Tensor* B, const Tensor* C, const Tensor* z, int groups,
                          int softplus) {
    rpb_scan_packed(c, x->shape[0], x->shape[1], x->shape[2], A->shape[1], groups, softplus);
    c->x_batch = x->strides[0]; c->x_row = x->strides[1];
    c->dt_batch = dt->strides[0]; c->dt_row = dt->strides[1];
    c->b_batch = B->strides[0]; c->b_row = B->strides[1];
    c->c_batch = C->strides[0]; c->c_row = C->strides[1];
    if (z) { c->z_batch = z->strides[0]; c->z_row = z->strides[1]; }
}

Tensor* op_selective_scan(Tensor* x, Tensor* dt, Tensor* A, Tensor* B, Tensor* C, Tensor* D, Tensor* dt_bias, Tensor* z, int softplus) {
    const char* op = "op_selective_scan";
    if (!x || !dt || !A || !B || !C || x->ndim != 3 || A->ndim != 2 || B->ndim != 3) return NULL;
    if (x->device_id < 0) return refused(op, "host tensors: this library has no CPU path");
    if (empty(x) || empty(A) || empty(B)) return refused(op, "a dimension of size 0");
    const int channels = x->shape[2], states = A->shape[1], cols = B->shape[2];
    const DType acc = x->dtype == DTYPE_FLOAT64 ? DTYPE_FLOAT64 : DTYPE_FLOAT32;
    if (!sequence_ok(x, x, channels) || !sequence_ok(dt, x, channels) || (z && !sequence_ok(z, x, channels)))
        return refused(op, "x, dt and z are [batch, len, channels] of one type");
    if (A->shape[0] != channels || !vector_ok(A, acc, x->device_id, (long long)channels * states))
        return refused(op, "A is a packed float32 [channels, states] (float64 for float64)");
    if (cols % states != 0 || !sequence_ok(B, x, cols) || !sequence_ok(C, x, cols)) return refused(op, "B and C are [batch, len, groups * states] of x's type");
    if ((D && !vector_ok(D, acc, x->device_id, channels)) || (dt_bias && !vector_ok(dt_bias, acc, x->device_id, channels)))
        return refused(op, "D and dt_bias are packed float32 [channels] (float64 for float64)");
    Tensor* in[9] = {x, dt, A, B, C};
    int n = 5;
    if (D) in[n++] = D;
    if (dt_bias) in[n++] = dt_bias;
    if (z) in[n++] = z;
    if (twice(in, n)) return refused(op, "one tensor in two places");
    RpbScan c;
    scan_geometry(&c, x, dt, A, B, C, z, cols / states, softplus);
    const long long kept = rp_selective_scan_saved_elems(&c, x->dtype), ws_bytes = rp_selective_scan_ws_bytes(&c, x->dtype, 0);
    if (kept < 0 || ws_bytes < 0) return NULL;
    bool grads = false;
    for (int i = 0; i < n; i++) grads = grads || wanted(in[i]);
    int shape[2] = {0, states};
    if (kept / states > INT_MAX) return refused(op, "too many rows for one node");
    shape[0] = (int)(kept / states);
    Tensor* out = rpb_tensor_empty(x->dtype, 3, x->shape, x->device_id);
    Tensor* saved = grads ? rpb_tensor_empty(acc, 2, shape, x->device_id) : NULL;
    Tensor* ws = ws_bytes ? workspace(ws_bytes, x->device_id) : NULL;
    int rc = out && (!grads || saved) && (!ws_bytes || ws) ? 0 : -1;
    if (rc == 0)
        rc = rp_selective_scan_ex(out->data, NULL, saved ? saved->data : NULL, x->data, dt->data, A->data, B->data, C->data, D ? D->data : NULL,
                                  dt_bias ? dt_bias->data : NULL, z ? z->data : NULL, NULL, NULL, ws ? ws->data : NULL, &c, x->dtype, x->device_id,
                                  rpb_current_node_stream());
    if (rc == 0) rc = rpb_finish_node(x->device_id);
    if (rc == 0 && grads) {
        in[n] = saved;
        ScanSaved* s = (ScanSaved*)malloc(sizeof(ScanSaved));
        if (!s || rpb_attach_node(out, backward_selective_scan_fn, in, n + 1)) { free(s); rc = -1; }
        else {
            s->softplus = softplus; s->has_D = D != NULL; s->has_bias = dt_bias != NULL; s->has_z = z != NULL; s->groups = cols / states;
            out->metadata->grad_fn->saved_data = s;
        }
    }
    rpb_tensor_release(ws);
    rpb_tensor_release(saved);          /* the node (if any) holds its own reference */
    if (rc != 0) { rpb_tensor_release(out); return NULL; }
    return out;
}

void backward_selective_scan_fn(GradFn* self, Tensor* grad_output) {
    if (!self || !grad_output || !self->inputs || !self->saved_data) return;
    const ScanSaved* s = (const ScanSaved*)self->saved_data;
    if (self->num_inputs != 6 + s->has_D + s->has_bias + s->has_z) return;
    Tensor** in = self->inputs;
    Tensor *x = in[0], *dt = in[1], *A = in[2], *B = in[3], *C = in[4];
    int n = 5;
    Tensor* D = s->has_D ? in[n++] : NULL;
    Tensor* bias = s->has_bias ? in[n++] : NULL;
    Tensor* z = s->has_z ? in[n++] : NULL;
    Tensor* saved = in[n];
    if (!x || !dt || !A || !B || !C || !saved || x->device_id < 0 || !sequence_ok(grad_output, x, x->shape[2])) {
        refused("op_selective_scan backward", "the upstream gradient must be [batch, len, channels] like the output");
        return;
    }
    RpbScan c;
    scan_geometry(&c, x, dt, A, B, C, z, s->groups, s->softplus);
    c.y_batch = grad_output->strides[0]; c.y_row = grad_output->strides[1];
    Tensor* of[8] = {x, dt, A, B, C, D, bias, z};
    const int bits[8] = {RPB_SCAN_ACC_DX, RPB_SCAN_ACC_DDT, RPB_SCAN_ACC_DA, RPB_SCAN_ACC_DB, RPB_SCAN_ACC_DC, RPB_SCAN_ACC_DD, RPB_SCAN_ACC_DDT_BIAS,
                         RPB_SCAN_ACC_DZ};
    Target t[8];
    void* to[8] = {NULL};
    memset(t, 0, sizeof(t));
    int acc = 0, rc = 0;
    bool any = false;
    for (int i = 0; i < 8 && rc == 0; i++) { rc = target_of(of[i], &t[i], &to[i], &acc, bits[i]); any = any || to[i]; }
    if (rc == 0 && any) {
        Tensor* ws = workspace(rp_selective_scan_ws_bytes(&c, x->dtype, 1), x->device_id);
        rc = ws ? rp_selective_scan_grad_ex(to[0], to[1], to[2], to[3], to[4], to[5], to[6], to[7], NULL, acc, grad_output->data, NULL, x->data, dt->data,
                                            A->data, B->data, C->data, D ? D->data : NULL, bias ? bias->data : NULL, z ? z->data : NULL, NULL, saved->data,
                                            ws->data, &c, x->dtype, x->device_id, rpb_current_node_stream()) : -1;
        if (rc == 0) rc = rpb_finish_node(x->device_id);
        rpb_tensor_release(ws);
    }
    settle(t, 8, rc);
}

/* ------------------------------------------------------------------ norms around a block */

/* rows of the last dimension at one distance from each other: that distance, or -1.  Dimensions of size 1 have no say. */
static long long row_stride(const Tensor* t) {
    const int n = t->ndim;
    if (t->shape[n - 1] > 1 && t->strides[n - 1] != 1) return -1;
    long long stride = t->shape[n - 1], rows = 1;       /* rows: of the dimensions behind d, which lie `stride` apart */
    for (int d = n - 2; d >= 0; d--) {
        if (t->shape[d] == 1) continue;
        if (rows == 1) stride = t->strides[d];
        else if (t->strides[d] != stride * rows) return -1;
        rows *= t->shape[d];
    }
    return stride < 0 ? -1 : stride;
}
static bool like(const Tensor* t, const Tensor* x) {
    if (t->ndim != x->ndim || t->dtype != x->dtype || t->device_id != x->device_id || row_stride(t) < 0) return false;
    return memcmp(t->shape, x->shape, sizeof(int) * x->ndim) == 0;
}

typedef struct { float eps; int has_z, has_w, has_scale, has_r, before; } NormSaved;

static int norm_geometry(RpbBlockNorm* c, const Tensor* u, const Tensor* z, const Tensor* r, float eps) {
    const int d = u->shape[u->ndim - 1];
    rpb_block_norm_packed(c, (long long)(u->size / (size_t)d), d, eps);
    c->u_row = row_stride(u);
    if (z) c->z_row = row_stride(z);
    if (r) c->r_row = row_stride(r);
    return 0;
}

/* before = 0: r + scale * norm(u silu(z)) w;  before = 1: norm(u) w */
static Tensor* norm_node(const char* op, Tensor* u, Tensor* z, Tensor* w, Tensor* scale, Tensor* r, float eps, int before) {
    if (!u || u->ndim < 1) return NULL;
    if (u->device_id < 0) return refused(op, "host tensors: this library has no CPU path");
    if (empty(u)) return refused(op, "a dimension of size 0");
    const int d = u->shape[u->ndim - 1];
    if (row_stride(u) < 0 || (z && !like(z, u)) || (r && !like(r, u))) return refused(op, "u, z and r have one shape and type, and rows at one distance");
    if ((w && !vector_ok(w, u->dtype, u->device_id, d)) || (scale && !vector_ok(scale, u->dtype, u->device_id, d)))
        return refused(op, "weights must be packed, one per channel, of u's type");
    if (before && !w) return refused(op, "the weight is needed");
    Tensor* in[5] = {u};
    int n = 1;
    if (z) in[n++] = z;
    if (w) in[n++] = w;
    if (scale) in[n++] = scale;
    if (r) in[n++] = r;
    if (twice(in, n)) return refused(op, "one tensor in two places");
    RpbBlockNorm c;
    norm_geometry(&c, u, z, r, eps);
    Tensor* out = rpb_tensor_empty(u->dtype, u->ndim, u->shape, u->device_id);
    if (!out) return NULL;
    int rc = rp_block_norm_ex(before ? NULL : out->data, before ? out->data : NULL, u->data, z ? z->data : NULL, !before && w ? w->data : NULL,
                              scale ? scale->data : NULL, r ? r->data : NULL, before ? w->data : NULL, &c, u->dtype, u->device_id,
                              rpb_current_node_stream());
    if (rc == 0) rc = rpb_finish_node(u->device_id);
    bool grads = false;
    for (int i = 0; i < n; i++) grads = grads || wanted(in[i]);
    if (rc == 0 && grads) {
        NormSaved* s = (NormSaved*)malloc(sizeof(NormSaved));
        if (!s || rpb_attach_node(out, backward_block_norm_fn, in, n)) { free(s); rc = -1; }
        else {
            s->eps = eps; s->has_z = z != NULL; s->has_w = w != NULL; s->has_scale = scale != NULL; s->has_r = r != NULL; s->before = before;
            out->metadata->grad_fn->saved_data = s;
        }
    }
    if (rc != 0) { rpb_tensor_release(out); return NULL; }
    return out;
}

Tensor* op_gated_norm(Tensor* u, Tensor* z, Tensor* w, Tensor* scale, Tensor* r, float eps) {
    return norm_node("op_gated_norm", u, z, w, scale, r, eps, 0);
}
Tensor* op_rms_norm(Tensor* x, Tensor* w, float eps) { return norm_node("op_rms_norm", x, NULL, w, NULL, NULL, eps, 1); }

void backward_block_norm_fn(GradFn* self, Tensor* grad_output) {
    if (!self || !grad_output || !self->inputs || !self->saved_data) return;
    const NormSaved* s = (const NormSaved*)self->saved_data;
    if (self->num_inputs != 1 + s->has_z + s->has_w + s->has_scale + s->has_r) return;
    Tensor** in = self->inputs;
    Tensor* u = in[0];
    int n = 1;
    Tensor* z = s->has_z ? in[n++] : NULL;
    Tensor* w = s->has_w ? in[n++] : NULL;
    Tensor* scale = s->has_scale ? in[n++] : NULL;
    Tensor* r = s->has_r ? in[n++] : NULL;
    if (!u || u->device_id < 0 || !like(grad_output, u)) {
        refused("block norm backward", "the upstream gradient must have the output's shape and rows at one distance");
        return;
    }
    RpbBlockNorm c;
    norm_geometry(&c, u, z, r, s->eps);
    c.out_row = c.y_row = row_stride(grad_output);
    Tensor* of[5] = {u, z, w, scale, r};
    const int bits[5] = {RPB_NORM_ACC_DU, RPB_NORM_ACC_DZ, s->before ? RPB_NORM_ACC_DW_BEFORE : RPB_NORM_ACC_DW_AFTER, RPB_NORM_ACC_DSCALE, RPB_NORM_ACC_DR};
    Target t[5];
    void* to[5] = {NULL};
    memset(t, 0, sizeof(t));
    int acc = 0, rc = 0;
    bool any = false;
    for (int i = 0; i < 5 && rc == 0; i++) { rc = target_of(of[i], &t[i], &to[i], &acc, bits[i]); any = any || to[i]; }
    if (rc == 0 && any) {
        Tensor* ws = workspace(rp_block_norm_ws_bytes(&c, u->dtype), u->device_id);
        const void* g = grad_output->data;
        const void* weight = w ? w->data : NULL;
        rc = ws ? rp_block_norm_grad_ex(to[0], to[1], to[4], s->before ? NULL : to[2], to[3], s->before ? to[2] : NULL, acc, s->before ? NULL : g,
                                        s->before ? g : NULL, u->data, z ? z->data : NULL, s->before ? NULL : weight, scale ? scale->data : NULL,
                                        r ? r->data : NULL, s->before ? weight : NULL, ws->data, &c, u->dtype, u->device_id, rpb_current_node_stream()) : -1;
        if (rc == 0) rc = rpb_finish_node(u->device_id);
        rpb_tensor_release(ws);
    }
    settle(t, 5, rc);
}
