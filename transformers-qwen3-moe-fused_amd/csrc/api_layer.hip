// extern "C" surface of the norm and of the whole expert layer: argument validation and dispatch only.
#include <math.h>

#include "fp8.h"
#include "ops.h"

using namespace mfl;

namespace {

int check_norm(const NormCall &n, bool forward) {
    if (n.R < 0 || n.H <= 0) return MFL_ERR_SHAPE;
    if (n.H > MFL_NORM_WIDTH || (forward && n.R > add_rms_norm_rows(n.H))) return MFL_ERR_LIMIT;
    if (!(n.eps >= 0.0f) || isinf(n.eps)) return MFL_ERR_SHAPE;
    if (!dtype_ok(n.dtype) || (n.weight_dtype != n.dtype && n.weight_dtype != MFL_F32)) return MFL_ERR_DTYPE;
    if (n.R == 0) return MFL_OK;
    if (!n.x || !n.weight || (n.residual && !n.s)) return MFL_ERR_NULL;
    const size_t size = dtype_size(n.dtype);
    if (!aligned(n.x, size) || !aligned(n.residual, size) || !aligned(n.y, size) || !aligned(n.s, size) ||
        !aligned(n.weight, dtype_size(n.weight_dtype)))
        return MFL_ERR_ALIGN;
    return MFL_OK;
}

// (the gated unit's rows, T k of them, are addressed with 32 bits)
bool past_limits(const mfl_moe_layer &p) {
    return p.T > MFL_LAYER_TOKENS || p.E > 1024 || p.k > 64 || p.H > 1 << 24 || p.I > 1 << 24 ||
           p.T * p.k * ((int64_t)p.I + 16) > 1 << 28;
}

}  // namespace

extern "C" {

int mfl_add_rms_norm(const void *x, const void *residual, const void *weight, void *y, void *s, int64_t R, int H, float eps, int dtype,
                     int weight_dtype, void *stream) {
    const NormCall n = {x, residual, weight, y, s, nullptr, nullptr, R, H, eps, dtype, weight_dtype};
    const int rc = check_norm(n, true);
    if (rc) return rc;
    if (R == 0) return MFL_OK;
    if (!y) return MFL_ERR_NULL;
    return add_rms_norm(n, (hipStream_t)stream);
}

int mfl_add_rms_norm_fp8(const void *x, const void *residual, const void *weight, void *q, uint8_t *scale, void *y, void *s, int64_t R,
                         int H, float eps, int dtype, int weight_dtype, void *stream) {
    const NormCall n = {x, residual, weight, y, s, (uint8_t *)q, scale, R, H, eps, dtype, weight_dtype};
    const int rc = check_norm(n, true);
    if (rc) return rc;
    if (R == 0) return MFL_OK;
    if (!q || !scale) return MFL_ERR_NULL;
    if (!aligned(q, 16)) return MFL_ERR_ALIGN;
    return add_rms_norm(n, (hipStream_t)stream);
}

size_t mfl_add_rms_norm_bwd_workspace(int64_t R, int H) {
    return R <= 0 || H <= 0 || H > MFL_NORM_WIDTH ? 0 : add_rms_norm_bwd_workspace(R, H);
}

int mfl_add_rms_norm_bwd(const void *dy, const void *ds, const void *s, const void *weight, void *dx, void *dw, int64_t R, int H,
                         float eps, int dtype, int weight_dtype, void *workspace, size_t ws_bytes, void *stream) {
    const NormCall n = {s, nullptr, weight, nullptr, (void *)s, nullptr, nullptr, R, H, eps, dtype, weight_dtype};
    int rc = check_norm(n, false);
    if (rc) return rc;
    if (!dx && !dw) return MFL_OK;
    const size_t size = dtype_size(dtype);
    if (R > 0 && !dy) return MFL_ERR_NULL;
    if (!aligned(dy, size) || !aligned(ds, size) || !aligned(dx, size) || !aligned(dw, dtype_size(weight_dtype))) return MFL_ERR_ALIGN;
    if (dw && R > 0) {
        if (!workspace || ws_bytes < add_rms_norm_bwd_workspace(R, H)) return MFL_ERR_WORKSPACE;
        if (!aligned(workspace, 16)) return MFL_ERR_ALIGN;
    }
    if (R == 0 && !dw) return MFL_OK;
    return add_rms_norm_bwd(n, dy, ds, dx, dw, (float *)workspace, (hipStream_t)stream);
}

size_t mfl_moe_layer_workspace(const mfl_moe_layer *p) {
    if (!p || p->T <= 0 || p->E <= 0 || p->k <= 0 || p->k > p->E || p->H <= 0 || p->I <= 0) return 0;
    if (past_limits(*p) || !dtype_ok(p->dtype)) return 0;
    return moe_layer_workspace(*p);
}

int mfl_moe_layer_fwd(const mfl_moe_layer *p, void *out, void *logits, void *workspace, size_t ws_bytes, void *stream) {
    if (!p) return MFL_ERR_NULL;
    if (p->T < 0 || p->E <= 0 || p->k <= 0 || p->k > p->E || p->H <= 0 || p->I <= 0) return MFL_ERR_SHAPE;
    if (past_limits(*p)) return MFL_ERR_LIMIT;
    if (!dtype_ok(p->dtype)) return MFL_ERR_DTYPE;
    if (p->norm_weight && (!(p->eps >= 0.0f) || isinf(p->eps))) return MFL_ERR_SHAPE;
    if (p->T == 0) return MFL_OK;
    if (!p->x || !p->router || !p->w_gate || !p->w_up || !p->w_down || !out || !logits) return MFL_ERR_NULL;
    if ((p->s_gate == nullptr) != (p->s_up == nullptr) || (p->s_gate == nullptr) != (p->s_down == nullptr)) return MFL_ERR_NULL;
    if (p->residual && !p->norm_weight) return MFL_ERR_NULL;
    const size_t size = dtype_size(p->dtype), wsize = p->s_gate ? 1 : size;
    if (!aligned(p->x, size) || !aligned(p->residual, size) || !aligned(p->norm_weight, size) || !aligned(p->router, size) ||
        !aligned(out, size) || !aligned(logits, size) || !aligned(p->w_gate, wsize) || !aligned(p->w_up, wsize) ||
        !aligned(p->w_down, wsize) || !aligned(p->s_gate, 4) || !aligned(p->s_up, 4) || !aligned(p->s_down, 4))
        return MFL_ERR_ALIGN;
    if (!workspace || ws_bytes < moe_layer_workspace(*p)) return MFL_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return MFL_ERR_ALIGN;
    return moe_layer_fwd(*p, out, logits, workspace, (hipStream_t)stream);
}

}  // extern "C"
