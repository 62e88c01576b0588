// extern "C" surface of the expert products in 8-bit floating point: argument validation and dispatch only.
#include "fp8.h"

using namespace mfl;

namespace {

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Room for quantised rows in a workspace, and where they lie.
size_t rows_bytes(int64_t rows, int K) { return up256((size_t)rows * fp8_ld(K)) + up256((size_t)rows * fp8_ld_scale(K)); }
struct RowsRoom {
    uint8_t *q, *scale;
    RowsRoom(uint8_t *at, int64_t rows, int K) : q(at), scale(at + up256((size_t)rows * fp8_ld(K))) {}
    Fp8Rows rows() const { return {q, scale}; }
};

// (columns counted in int, rounded up to whole blocks)
bool width_ok(int n) { return n > 0 && n <= 1 << 30; }
bool sizes_ok(int64_t R, int N, int K, int E) { return R >= 0 && R <= 0x7fffffff && width_ok(N) && width_ok(K) && E > 0; }

int check_call(const void *m_sizes, int ms_dtype, int64_t R, int N, int K, int E, int in_dtype, int out_dtype) {
    if (!sizes_ok(R, N, K, E)) return MFL_ERR_SHAPE;
    if (!dtype_ok(in_dtype) || !dtype_ok(out_dtype) || !itype_ok(ms_dtype)) return MFL_ERR_DTYPE;
    if (!m_sizes) return MFL_ERR_NULL;
    if (!aligned(m_sizes, ms_dtype == MFL_I64 ? 8 : 4)) return MFL_ERR_ALIGN;
    return MFL_OK;
}
int check_source(int64_t src_rows, const int32_t *row_idx, int idx_div, int64_t R) {
    if (row_idx != nullptr && (idx_div <= 0 || src_rows <= 0)) return MFL_ERR_SHAPE;
    if (row_idx == nullptr && src_rows < R) return MFL_ERR_SHAPE;
    if (!aligned(row_idx, 4)) return MFL_ERR_ALIGN;
    return MFL_OK;
}
int check_weight(const mfl_fp8_weight *w) {
    if (!w || !w->q || !w->scale) return MFL_ERR_NULL;
    return aligned(w->scale, 4) ? MFL_OK : MFL_ERR_ALIGN;
}
int check_workspace(int op, int64_t src_rows, int64_t R, int N, int K, int E, const void *ws, size_t ws_bytes) {
    const size_t need = mfl_fp8_workspace(op, src_rows, R, N, K, E);
    if (need == 0) return MFL_OK;
    if (!ws || ws_bytes < need) return MFL_ERR_WORKSPACE;
    return aligned(ws, 256) ? MFL_OK : MFL_ERR_ALIGN;
}
Fp8Matrix matrix(const mfl_fp8_weight *w) { return {(const uint8_t *)w->q, w->scale}; }

// the rows of the left operand that a product reads
int64_t source_rows(int64_t src_rows, const int32_t *row_idx, int64_t R) { return row_idx != nullptr ? src_rows : R; }

// Weights whose rows no 16-byte access fits are copied to rows that one does where the call has rows for most experts.  The copy
// reads every expert's, the kernels for any shape only those of experts with rows: us of forward / input gradient with copies,
// and without, 60 experts of 333 x 1001: 30 / 29 and 58 / 73 at one row for every expert, 29 / 29 and 61 / 77 at four, 31 / 31 and
// 63 / 78 at 32; 128 of 768 x 2041: 123 / 122 and 364 / 688, 124 / 124 and 365 / 672, 133 / 144 and 380 / 686.  So they pay where
// a third to a half of the experts have rows; with four rows per expert nearly all do, unless they are very unequal.
int padded_row(int K) { return (K + 15) / 16 * 16; }
size_t padded_bytes(int64_t R, int N, int K, int E) {
    return K % 16 != 0 && R >= (int64_t)4 * E ? up256((size_t)E * N * padded_row(K)) : 0;
}

// One product; `room` holds padded_bytes() for each of its matrices.
int run_product(Fp8Product p, uint8_t *room, hipStream_t stream) {
    const size_t bytes = padded_bytes(p.R, p.N, p.K, p.E);
    if (bytes != 0) {
        Fp8Product padded = p;
        padded.ldw = padded_row(p.K);
        const int matrices = p.glu || p.terms == 2 ? 2 : 1;
        for (int i = 0; i < matrices; ++i) padded.w[i].q = room + i * bytes;
        if (gemm_fp8_tiles(padded)) {
            for (int i = 0; i < matrices; ++i) {
                const int rc = fp8_pad_rows(p.w[i].q, (int64_t)p.E * p.N, p.K, padded.ldw, room + i * bytes, stream);
                if (rc) return rc;
            }
            return gemm_fp8_tile(padded, stream);
        }
    }
    int rc = gemm_fp8_tile(p, stream);
    if (rc != MFL_ERR_UNSUPPORTED) return rc;
    if (p.hq != nullptr && p.h32 == nullptr) return MFL_ERR_WORKSPACE;  // (no such call: mlp_needs_values)
    rc = gemm_fp8_generic(p, stream);
    return rc || p.hq == nullptr ? rc : fp8_quant_rows(p.h32, MFL_F32, p.R, p.N, p.hq, p.hq_scale, stream);
}

// Whether the expert MLP's gated unit leaves fp32 values in the workspace (the tiles write quantised rows, the other kernels do
// not).  `on_grid`: gate, up and the products' outputs lie on the 16-byte grid.
bool mlp_needs_values(int64_t src_rows, int64_t R, int N, int K, int E, bool on_grid) {
    if (R <= (int64_t)kFp8DecodeRowsPerExpert * E || !on_grid) return true;
    static const int32_t gathered = 0;
    Fp8Product p = {};
    p.glu = true, p.terms = 1, p.row_idx = &gathered, p.src_rows = src_rows > 256 ? src_rows : 256, p.out_dtype = MFL_F32;
    p.R = R, p.N = N, p.K = K, p.E = E, p.ldw = padded_bytes(R, N, K, E) != 0 ? padded_row(K) : K;
    return !gemm_fp8_tiles(p);
}
size_t mlp_values_bytes(bool needed, int64_t R, int N) { return needed ? up256((size_t)R * N * 4) : 0; }
// (the down projection's padded copy takes the place of the others')
size_t mlp_bytes(int64_t src_rows, int64_t R, int N, int K, int E, bool on_grid) {
    const size_t front = 2 * padded_bytes(R, N, K, E), back = padded_bytes(R, K, N, E);
    return rows_bytes(src_rows, K) + rows_bytes(R, N) + mlp_values_bytes(mlp_needs_values(src_rows, R, N, K, E, on_grid), R, N) +
           (front > back ? front : back);
}

int mlp_fwd(const void *x, const Fp8Rows *given, int64_t src_rows, const int32_t *row_idx, int idx_div, const mfl_fp8_weight *gate,
                    const mfl_fp8_weight *up, const mfl_fp8_weight *down, const void *m_sizes, int m_sizes_dtype, void *y,
                    void *e_out, void *g_out, int64_t R, int I, int H, int E, int dtype, void *workspace, size_t ws_bytes,
                    void *stream) {
    int rc = check_call(m_sizes, m_sizes_dtype, R, I, H, E, dtype, dtype);
    if (!rc) rc = check_source(src_rows, row_idx, idx_div, R);
    if (rc) return rc;
    if (R == 0) return MFL_OK;
    if (!x || !y) return MFL_ERR_NULL;
    rc = check_weight(gate);
    if (!rc) rc = check_weight(up);
    if (!rc) rc = check_weight(down);
    if (rc) return rc;
    const size_t size = dtype_size(dtype);
    if (!aligned(x, size) || !aligned(y, size) || !aligned(e_out, size) || !aligned(g_out, size)) return MFL_ERR_ALIGN;
    if ((e_out == nullptr) != (g_out == nullptr)) return MFL_ERR_NULL;
    const bool on_grid = aligned(gate->q, 16) && aligned(up->q, 16) && aligned(e_out, 16) && aligned(g_out, 16);
    rc = check_workspace(on_grid ? MFL_FP8_MLP : MFL_FP8_MLP_OFF_GRID, src_rows, R, I, H, E, workspace, ws_bytes);
    if (rc) return rc;
    const size_t values = mlp_values_bytes(mlp_needs_values(src_rows, R, I, H, E, on_grid), R, I);
    const int64_t used = source_rows(src_rows, row_idx, R);
    const RowsRoom room((uint8_t *)workspace, used, H), hidden((uint8_t *)workspace + rows_bytes(src_rows, H), R, I);
    void *const h = (uint8_t *)workspace + rows_bytes(src_rows, H) + rows_bytes(R, I);
    uint8_t *const padding = (uint8_t *)h + values;
    Fp8Product p = {};
    p.glu = true, p.terms = 1, p.a[0] = room.rows(), p.w[0] = matrix(gate), p.w[1] = matrix(up);
    p.row_idx = row_idx, p.idx_div = idx_div, p.src_rows = used;
    p.m_sizes = m_sizes, p.ms_i64 = m_sizes_dtype == MFL_I64;
    p.e_out = e_out, p.g_out = g_out, p.out_dtype = dtype, p.R = R, p.N = I, p.K = p.ldw = H, p.E = E;
    Fp8Product d = p;  // the down projection
    d.glu = false, d.a[0] = hidden.rows(), d.w[0] = matrix(down), d.row_idx = nullptr, d.src_rows = R;
    d.out = y, d.e_out = d.g_out = nullptr, d.N = H, d.K = d.ldw = I;
    if (gemm_fp8_decodes(p) && gemm_fp8_decodes(d) && aligned(x, 16)) {
        // a few rows: both kernels quantise their rows themselves, from the fp32 values between them
        p.h32 = (float *)h;
        rc = gemm_fp8_decode(p, x, dtype, (hipStream_t)stream);
        return rc ? rc : gemm_fp8_decode(d, h, MFL_F32, (hipStream_t)stream);
    }
    if (given != nullptr) p.a[0] = *given;
    else rc = fp8_quant_rows(x, dtype, used, H, room.q, room.scale, (hipStream_t)stream);
    if (rc) return rc;
    p.hq = hidden.q, p.hq_scale = hidden.scale, p.h32 = values != 0 ? (float *)h : nullptr;
    rc = run_product(p, padding, (hipStream_t)stream);
    return rc ? rc : run_product(d, padding, (hipStream_t)stream);
}

}  // namespace

extern "C" {

size_t mfl_fp8_workspace(int op, int64_t src_rows, int64_t R, int N, int K, int E) {
    if (!sizes_ok(R, N, K, E) || src_rows < 0 || R == 0) return 0;
    switch (op) {
        case MFL_FP8_FWD:
            return rows_bytes(src_rows, K) + padded_bytes(R, N, K, E);
        case MFL_FP8_GLU:
            return rows_bytes(src_rows, K) + 2 * padded_bytes(R, N, K, E);
        case MFL_FP8_DX:
            return rows_bytes(R, N) + padded_bytes(R, N, K, E);
        case MFL_FP8_GLU_BWD:
            return 2 * rows_bytes(R, N) + 2 * padded_bytes(R, N, K, E);
        case MFL_FP8_MLP:
            return mlp_bytes(src_rows, R, N, K, E, true);
        case MFL_FP8_MLP_OFF_GRID:
            return mlp_bytes(src_rows, R, N, K, E, false);
        default:
            return 0;
    }
}

int mfl_gemm_fwd_fp8(const void *x, int64_t src_rows, const int32_t *row_idx, int idx_div, const mfl_fp8_weight *w,
                     const void *m_sizes, int m_sizes_dtype, void *y, int64_t R, int N, int K, int E, int in_dtype,
                     int out_dtype, void *workspace, size_t ws_bytes, void *stream) {
    int rc = check_call(m_sizes, m_sizes_dtype, R, N, K, E, in_dtype, out_dtype);
    if (!rc) rc = check_source(src_rows, row_idx, idx_div, R);
    if (rc) return rc;
    if (R == 0) return MFL_OK;
    if (!x || !y) return MFL_ERR_NULL;
    rc = check_weight(w);
    if (rc) return rc;
    if (!aligned(x, dtype_size(in_dtype)) || !aligned(y, dtype_size(out_dtype))) return MFL_ERR_ALIGN;
    const int64_t used = source_rows(src_rows, row_idx, R);
    const RowsRoom room((uint8_t *)workspace, used, K);
    Fp8Product p = {};
    p.terms = 1, p.a[0] = room.rows(), p.w[0] = matrix(w);
    p.row_idx = row_idx, p.idx_div = idx_div, p.src_rows = used;
    p.m_sizes = m_sizes, p.ms_i64 = m_sizes_dtype == MFL_I64;
    p.out = y, p.out_dtype = out_dtype, p.R = R, p.N = N, p.K = p.ldw = K, p.E = E;
    rc = gemm_fp8_decode(p, x, in_dtype, (hipStream_t)stream);
    if (rc != MFL_ERR_UNSUPPORTED) return rc;
    rc = check_workspace(MFL_FP8_FWD, src_rows, R, N, K, E, workspace, ws_bytes);
    if (rc) return rc;
    rc = fp8_quant_rows(x, in_dtype, used, K, room.q, room.scale, (hipStream_t)stream);
    if (rc) return rc;
    return run_product(p, (uint8_t *)workspace + rows_bytes(src_rows, K), (hipStream_t)stream);
}

int mfl_gemm_dx_fp8(const void *dy, const mfl_fp8_weight *w, const void *m_sizes, int m_sizes_dtype, void *dx, int64_t R, int N,
                    int K, int E, int in_dtype, int out_dtype, void *workspace, size_t ws_bytes, void *stream) {
    int rc = check_call(m_sizes, m_sizes_dtype, R, N, K, E, in_dtype, out_dtype);
    if (rc) return rc;
    if (R == 0) return MFL_OK;
    if (!dy || !dx) return MFL_ERR_NULL;
    rc = check_weight(w);
    if (rc) return rc;
    if (!aligned(dy, dtype_size(in_dtype)) || !aligned(dx, dtype_size(out_dtype))) return MFL_ERR_ALIGN;
    rc = check_workspace(MFL_FP8_DX, 0, R, N, K, E, workspace, ws_bytes);
    if (rc) return rc;
    const RowsRoom room((uint8_t *)workspace, R, N);
    rc = fp8_quant_rows(dy, in_dtype, R, N, room.q, room.scale, (hipStream_t)stream);
    if (rc) return rc;
    Fp8Product p = {};
    p.dx = true, p.terms = 1, p.a[0] = room.rows(), p.w[0] = matrix(w);
    p.m_sizes = m_sizes, p.ms_i64 = m_sizes_dtype == MFL_I64;
    p.out = dx, p.out_dtype = out_dtype, p.R = R, p.N = N, p.K = p.ldw = K, p.E = E;
    return run_product(p, (uint8_t *)workspace + rows_bytes(R, N), (hipStream_t)stream);
}

int mfl_glu_fwd_fp8(const void *x, int64_t src_rows, const int32_t *row_idx, int idx_div, const mfl_fp8_weight *gate,
                    const mfl_fp8_weight *up, const void *m_sizes, int m_sizes_dtype, void *h, void *e_out, void *g_out,
                    int64_t R, int N, int K, int E, int dtype, void *workspace, size_t ws_bytes, void *stream) {
    int rc = check_call(m_sizes, m_sizes_dtype, R, N, K, E, dtype, dtype);
    if (!rc) rc = check_source(src_rows, row_idx, idx_div, R);
    if (rc) return rc;
    if (R == 0) return MFL_OK;
    if (!x || !h) return MFL_ERR_NULL;
    rc = check_weight(gate);
    if (!rc) rc = check_weight(up);
    if (rc) return rc;
    const size_t size = dtype_size(dtype);
    if (!aligned(x, size) || !aligned(h, size) || !aligned(e_out, size) || !aligned(g_out, size)) return MFL_ERR_ALIGN;
    const int64_t used = source_rows(src_rows, row_idx, R);
    const RowsRoom room((uint8_t *)workspace, used, K);
    Fp8Product p = {};
    p.glu = true, p.terms = 1, p.a[0] = room.rows(), p.w[0] = matrix(gate), p.w[1] = matrix(up);
    p.row_idx = row_idx, p.idx_div = idx_div, p.src_rows = used;
    p.m_sizes = m_sizes, p.ms_i64 = m_sizes_dtype == MFL_I64;
    p.out = h, p.e_out = e_out, p.g_out = g_out, p.out_dtype = dtype, p.R = R, p.N = N, p.K = p.ldw = K, p.E = E;
    rc = gemm_fp8_decode(p, x, dtype, (hipStream_t)stream);
    if (rc != MFL_ERR_UNSUPPORTED) return rc;
    rc = check_workspace(MFL_FP8_GLU, src_rows, R, N, K, E, workspace, ws_bytes);
    if (rc) return rc;
    rc = fp8_quant_rows(x, dtype, used, K, room.q, room.scale, (hipStream_t)stream);
    if (rc) return rc;
    return run_product(p, (uint8_t *)workspace + rows_bytes(src_rows, K), (hipStream_t)stream);
}

int mfl_glu_bwd_fp8(const void *dh, const void *e, const void *g, const mfl_fp8_weight *gate, const mfl_fp8_weight *up,
                    const void *m_sizes, int m_sizes_dtype, void *dx, int64_t R, int N, int K, int E, int dtype,
                    void *workspace, size_t ws_bytes, void *stream) {
    int rc = check_call(m_sizes, m_sizes_dtype, R, N, K, E, dtype, dtype);
    if (rc) return rc;
    if (R == 0) return MFL_OK;
    if (!dh || !e || !g || !dx) return MFL_ERR_NULL;
    rc = check_weight(gate);
    if (!rc) rc = check_weight(up);
    if (rc) return rc;
    const size_t size = dtype_size(dtype);
    if (!aligned(dh, size) || !aligned(e, size) || !aligned(g, size) || !aligned(dx, size)) return MFL_ERR_ALIGN;
    rc = check_workspace(MFL_FP8_GLU_BWD, 0, R, N, K, E, workspace, ws_bytes);
    if (rc) return rc;
    const RowsRoom de((uint8_t *)workspace, R, N), dg((uint8_t *)workspace + rows_bytes(R, N), R, N);
    rc = fp8_silu_bwd_quant(dh, e, g, dtype, R, N, de.q, de.scale, dg.q, dg.scale, (hipStream_t)stream);
    if (rc) return rc;
    Fp8Product p = {};
    p.dx = true, p.terms = 2, p.a[0] = de.rows(), p.a[1] = dg.rows(), p.w[0] = matrix(gate), p.w[1] = matrix(up);
    p.m_sizes = m_sizes, p.ms_i64 = m_sizes_dtype == MFL_I64;
    p.out = dx, p.out_dtype = dtype, p.R = R, p.N = N, p.K = p.ldw = K, p.E = E;
    return run_product(p, (uint8_t *)workspace + 2 * rows_bytes(R, N), (hipStream_t)stream);
}

int mfl_mlp_fwd_fp8(const void *x, int64_t src_rows, const int32_t *row_idx, int idx_div, const mfl_fp8_weight *gate,
                    const mfl_fp8_weight *up, const mfl_fp8_weight *down, const void *m_sizes, int m_sizes_dtype, void *y,
                    void *e_out, void *g_out, int64_t R, int I, int H, int E, int dtype, void *workspace, size_t ws_bytes,
                    void *stream) {
    return mlp_fwd(x, nullptr, src_rows, row_idx, idx_div, gate, up, down, m_sizes, m_sizes_dtype, y, e_out, g_out, R, I, H, E, dtype,
                   workspace, ws_bytes, stream);
}

int mfl_mlp_fwd_fp8_rows(const void *x, const void *xq, const uint8_t *xq_scale, int64_t src_rows, const int32_t *row_idx, int idx_div,
                         const mfl_fp8_weight *gate, const mfl_fp8_weight *up, const mfl_fp8_weight *down, const void *m_sizes,
                         int m_sizes_dtype, void *y, void *e_out, void *g_out, int64_t R, int I, int H, int E, int dtype,
                         void *workspace, size_t ws_bytes, void *stream) {
    if (R > 0 && (!xq || !xq_scale)) return MFL_ERR_NULL;
    if (!aligned(xq, 16) || !aligned(xq_scale, 4)) return MFL_ERR_ALIGN;
    const Fp8Rows given = {(const uint8_t *)xq, xq_scale};
    return mlp_fwd(x, &given, src_rows, row_idx, idx_div, gate, up, down, m_sizes, m_sizes_dtype, y, e_out, g_out, R, I, H, E, dtype,
                   workspace, ws_bytes, stream);
}

int mfl_fp8_quant_rows(const void *x, int dtype, int64_t R, int K, void *q, uint8_t *scale, void *stream) {
    if (R < 0 || !width_ok(K)) return MFL_ERR_SHAPE;
    if (!dtype_ok(dtype)) return MFL_ERR_DTYPE;
    if (R == 0) return MFL_OK;
    if (!x || !q || !scale) return MFL_ERR_NULL;
    if (!aligned(x, dtype_size(dtype)) || !aligned(q, 16)) return MFL_ERR_ALIGN;
    return fp8_quant_rows(x, dtype, R, K, (uint8_t *)q, scale, (hipStream_t)stream);
}

int mfl_fp8_dequant_rows(const void *q, const uint8_t *scale, int64_t R, int K, void *out, int out_dtype, void *stream) {
    if (R < 0 || !width_ok(K)) return MFL_ERR_SHAPE;
    if (!dtype_ok(out_dtype)) return MFL_ERR_DTYPE;
    if (R == 0) return MFL_OK;
    if (!q || !scale || !out) return MFL_ERR_NULL;
    if (!aligned(out, dtype_size(out_dtype))) return MFL_ERR_ALIGN;
    return fp8_dequant_rows((const uint8_t *)q, scale, R, K, out, out_dtype, (hipStream_t)stream);
}

int mfl_fp8_quant_blocks(const void *w, int dtype, int E, int N, int K, void *q, float *scale, void *stream) {
    if (E <= 0 || !width_ok(N) || !width_ok(K)) return MFL_ERR_SHAPE;
    if (!dtype_ok(dtype)) return MFL_ERR_DTYPE;
    if (!w || !q || !scale) return MFL_ERR_NULL;
    if (!aligned(w, dtype_size(dtype)) || !aligned(scale, 4)) return MFL_ERR_ALIGN;
    return fp8_quant_blocks(w, dtype, E, N, K, (uint8_t *)q, scale, (hipStream_t)stream);
}

int mfl_fp8_dequant_blocks(const void *q, const float *scale, int E, int N, int K, void *out, int out_dtype, void *stream) {
    if (E <= 0 || !width_ok(N) || !width_ok(K)) return MFL_ERR_SHAPE;
    if (!dtype_ok(out_dtype)) return MFL_ERR_DTYPE;
    if (!q || !scale || !out) return MFL_ERR_NULL;
    if (!aligned(scale, 4) || !aligned(out, dtype_size(out_dtype))) return MFL_ERR_ALIGN;
    return fp8_dequant_blocks((const uint8_t *)q, scale, E, N, K, out, out_dtype, (hipStream_t)stream);
}

}  // extern "C"
