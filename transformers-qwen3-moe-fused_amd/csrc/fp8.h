// Expert products in 8-bit floating point: internal interface between the C ABI (api_fp8.hip) and the kernel files, and
// what the kernels share.
//
// Values are e4m3 (OCP: largest 448, no infinity, NaN 0x7f).  Rows (activations, gradients) carry one power-of-two scale per
// row and 128 elements of the reduction, as a biased exponent byte; weights one fp32 scale per 128 x 128 block.  The scale
// of a row block is the smallest power of two, at least 2^-117, that brings the block's largest finite magnitude to 448 or
// below.  A power of two because then x / scale is exact: a value is rounded once, what it is rounded to does not depend on
// how the division is done, and the matrix instruction applies the scale itself.  2^-117 because the smallest value of the
// grid, 2^-9, is a normal float at that scale.  Elements that are no number or infinite become NaN and leave the block's
// scale to the others.
//
// Which matrix instruction.  The 8-bit one (v_mfma_*_fp8_fp8 the same as v_mfma_scale_*_f8f6f4) adds its products in groups of
// eight and cuts them off 2^-13 below the group's largest.  Measured against the sum of magnitudes of 128 products: 1.5e-6 on
// average and 2.2e-5 at most for normal values, 1.8e-5 and 1.7e-4 for bytes of any value (the bf16 instruction 2e-10 and 3e-8,
// 2e-8 and 3e-7).  Against the definition in 64 bits, over the norm, reductions of 256 to 8192, normal values / one channel in
// 64 64 times as large / magnitudes spread evenly over 2^8: fp16 outputs 2.08e-4 / 2.18e-4 / 2.17e-4, where their rounding alone is
// 2.07e-4; bf16 outputs 1.66e-3, their rounding alone, each time.  So 16-bit outputs are multiplied in 8 bits.  fp32 outputs are
// multiplied in bf16, which holds every e4m3 value times its scale, at half the rate.
// The expert MLP's gated unit is quantised from its sums, and a sum that is off by 1e-5 takes an element across a border of the
// 8-bit grid.  With 8-bit products the MLP of 24008 rows, 2048 and 768, is 2.3e-3 from the definition in bf16 (1.66e-3 are its
// rounding) and 1.5e-3 in fp16 (2.07e-4), with bf16 products 1.68e-3 and 2.16e-4.  Either neighbour across a border is as near to
// the unit's real value: against the MLP without the rounding to the grid it is 2.65e-2 either way.  So that unit has bf16 products
// in fp16, which is chosen for its digits (24008 rows 247 -> 301 us), and the gated unit at decode sizes has them in any type (32
// tokens' unit 1 %, bound by the weights' bytes; one token's MLP in a graph 15.2 -> 15.9 us); the tiles of that unit in bf16 have
// 8-bit ones (the MLP of 131072 rows 910 us against 1190).
#pragma once
#include "common.h"
#include "fp8_counts.h"

namespace mfl {

constexpr int kFp8Block = 128;

__host__ __device__ constexpr int fp8_blocks(int n) { return (n + kFp8Block - 1) / kFp8Block; }
// Quantised rows lie `fp8_ld(K)` bytes apart, zeros behind the row's end, and their scales `fp8_ld_scale(K)` bytes apart (whole
// dwords, which the kernels fetch four blocks at a time).
__host__ __device__ constexpr int64_t fp8_ld(int K) { return (int64_t)fp8_blocks(K) * kFp8Block; }
__host__ __device__ constexpr int64_t fp8_ld_scale(int K) { return (fp8_blocks(K) + 3) / 4 * 4; }

struct Fp8Rows {
    const uint8_t *q;
    const uint8_t *scale;
};
struct Fp8Matrix {  // (E, out, in) with (E, ceil(out / 128), ceil(in / 128)) scales
    const uint8_t *q;
    const float *scale;
};

// One product over rows grouped by expert.  Forward: out (R, N) = a (., K) w^T, gathered rows where row_idx is given; gated
// (glu): out = silu(a w[0]^T) * (a w[1]^T), the two products to e_out / g_out where given.  Input gradient (dx): out (R, K) =
// a[0] (R, N) w[0], plus a[1] w[1] where terms is 2.
struct Fp8Product {
    bool dx, glu;
    int terms;
    Fp8Rows a[2];
    Fp8Matrix w[2];
    const int32_t *row_idx;
    int idx_div;
    int64_t src_rows;
    const void *m_sizes;
    int ms_i64;
    void *out, *e_out, *g_out;
    int out_dtype;
    // (glu) where hq is given, `out` is not written: the tiles write quantised rows, made from the fp32 values; the other kernels
    // leave those in h32
    uint8_t *hq, *hq_scale;
    float *h32;
    int64_t R;
    int N, K, E;
    int ldw;  // bytes from one row of the weights to the next: K, or (tiles only) K rounded up to 16 with zeros behind column K
};

// A few rows per expert (kFp8DecodeRowsPerExpert on average), forward and gated, 16-bit outputs, K % 16 == 0: the rows come as
// they are (x, of the output's type or fp32) and are quantised on the way; p.a is not read.  MFL_ERR_UNSUPPORTED for the rest;
// gemm_fp8_decodes: whether it takes the product with an aligned x.
// The line: 128 experts, 2048 to 768, us of a launch with the same rows for every expert, this kernel / tiles behind the
// quantiser, product and gated unit: 42.6 / 50.8 and 75 / 81 at 8 rows per expert, 46.6 / 53.1 and 83 / 86 at 16, 73 / 55 and
// 130 / 90 at 24, where an expert's weights are read twice (16 rows at a time).  The sizes are known on the device only, and
// skewed ones have experts past 16 rows well before: 8 per expert under Zipf(1) 46.6 / 50.0 and 77 / 79, under Zipf(1.5)
// 34 / 29 and 63 / 54, all on one expert 24 / 22 and 36 / 24; 2 per expert there 23 / 22 and 32 / 29, 14 / 21 and 15 / 22.
constexpr int kFp8DecodeRowsPerExpert = MFL_FP8_DECODE_ROWS;
bool gemm_fp8_decodes(const Fp8Product &p);
int gemm_fp8_decode(const Fp8Product &p, const void *x, int x_dtype, hipStream_t stream);
// Tiles in LDS, ldw % 16 == 0, two steps of the reduction at least; MFL_ERR_UNSUPPORTED for the rest.
bool gemm_fp8_tiles(const Fp8Product &p);  // whether it takes the product
int gemm_fp8_tile(const Fp8Product &p, hipStream_t stream);
// Any shape; MFL_OK or a launch error.
int gemm_fp8_generic(const Fp8Product &p, hipStream_t stream);

int fp8_quant_rows(const void *x, int dtype, int64_t R, int K, uint8_t *q, uint8_t *scale, hipStream_t stream);
int fp8_dequant_rows(const uint8_t *q, const uint8_t *scale, int64_t R, int K, void *out, int out_dtype, hipStream_t stream);
// The gated unit's backward, de and dg straight to quantised rows.
int fp8_silu_bwd_quant(const void *dh, const void *e, const void *g, int dtype, int64_t R, int N, uint8_t *de_q,
                       uint8_t *de_scale, uint8_t *dg_q, uint8_t *dg_scale, hipStream_t stream);
int fp8_quant_blocks(const void *w, int dtype, int E, int N, int K, uint8_t *q, float *scale, hipStream_t stream);
// (rows, K) bytes to rows of ldw bytes, zeros behind column K; out 16-byte aligned, ldw a multiple of 16.
int fp8_pad_rows(const uint8_t *w, int64_t rows, int K, int ldw, uint8_t *out, hipStream_t stream);
int fp8_dequant_blocks(const uint8_t *q, const float *scale, int E, int N, int K, void *out, int out_dtype, hipStream_t stream);

typedef __attribute__((ext_vector_type(8))) int intx8;

// Biased exponent byte of the scale for a block whose largest finite magnitude has the bits b: amax = f 2^p with 1 <= f < 2 fits
// 448 2^e = 1.75 2^(8 + e) with e = p - 8 if f <= 1.75, else p - 7.  (amax 0 or subnormal: the least exponent.)
__device__ __forceinline__ int fp8_scale_byte(uint32_t b) {
    const int byte = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return byte < 10 ? 10 : byte;
}
__device__ __forceinline__ float fp8_scale_of(int byte) { return __uint_as_float((uint32_t)byte << 23); }
__device__ __forceinline__ float fp8_inverse_of(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// Largest magnitude of a block.  Magnitudes are compared as whole numbers (their order is that of the values, infinity and then
// NaN above all): fp8_wider takes another value's bits in, fp8_unusual says whether there is one that is no finite number; only
// then do the values have to be looked at one by one (fp8_finite_abs, fp8_finite).
__device__ __forceinline__ uint32_t fp8_wider(uint32_t bits, float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return bits > b ? bits : b;
}
__device__ __forceinline__ bool fp8_unusual(uint32_t bits) { return bits >= 0x7f800000u; }
__device__ __forceinline__ float fp8_finite_abs(float v) {
    const float a = __builtin_fabsf(v);
    return a <= 3.4028234663852886e38f ? a : 0.0f;
}
// v, or NaN where it is infinite
__device__ __forceinline__ float fp8_finite(float v) {
    return __builtin_fabsf(v) <= 3.4028234663852886e38f ? v : __uint_as_float(0x7fc00000u);
}
// Four values times a power of two, rounded to e4m3 (nearest, ties to even): one dword.  None of them infinite.
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d, float inverse) {
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a * inverse, b * inverse, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c * inverse, d * inverse, r, true);
    return (uint32_t)r;
}

// 8 e4m3 values times the power of two `scale`, as bf16 (exact below 2^128)
typedef __attribute__((ext_vector_type(2))) int intx2;
__device__ __forceinline__ bf16x8 fp8_widen(const intx2 v, float scale) {
    union {
        bf16x2 p[4];
        bf16x8 all;
    } u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        u.p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], scale, false);
        u.p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], scale, true);
    }
    return u.all;
}

// The largest of a row of 16 lanes, in all of them.
template <int CTRL>
__device__ __forceinline__ uint32_t fp8_dpp_max(uint32_t x) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
    return x > y ? x : y;
}
__device__ __forceinline__ uint32_t fp8_max16(uint32_t x) {
    x = fp8_dpp_max<0x128>(x);  // row_ror 8, 4, 2, 1
    x = fp8_dpp_max<0x124>(x);
    x = fp8_dpp_max<0x122>(x);
    return fp8_dpp_max<0x121>(x);
}

// The row counts of experts e, e + 64, ..., 0 past the last expert, their loads all in flight together.
template <int N>
__device__ __forceinline__ void fp8_load_counts(const void *m_sizes, int ms_i64, int e, int E, int64_t R, uint32_t (&count)[N]) {
    int64_t size[N];
    if (ms_i64) {
#pragma unroll
        for (int i = 0; i < N; ++i) size[i] = ((const int64_t *)m_sizes)[e + 64 * i < E ? e + 64 * i : E - 1];
    } else {
        int32_t narrow[N];
#pragma unroll
        for (int i = 0; i < N; ++i) narrow[i] = ((const int32_t *)m_sizes)[e + 64 * i < E ? e + 64 * i : E - 1];
#pragma unroll
        for (int i = 0; i < N; ++i) size[i] = narrow[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) count[i] = e + 64 * i < E ? fp8_count_of(size[i], (uint32_t)R) : 0u;
}
// 64 counts, a lane each, cut at `room` rows: the lane's first row, the row behind its last one, and (in every lane) that of the
// last lane.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t fp8_dpp_sum(uint32_t x) {
    return fp8_sum(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROW_MASK, 0xf, true));
}
struct Fp8Counted {
    int begin, end, all;
};
__device__ __forceinline__ Fp8Counted fp8_cut(uint32_t count, uint32_t room) {
    uint32_t x = count;  // (the order of wave_inclusive_scan)
    x = fp8_dpp_sum<0x111, 0xf>(x);
    x = fp8_dpp_sum<0x112, 0xf>(x);
    x = fp8_dpp_sum<0x114, 0xf>(x);
    x = fp8_dpp_sum<0x118, 0xf>(x);
    x = fp8_dpp_sum<0x142, 0xa>(x);
    x = fp8_dpp_sum<0x143, 0xc>(x);
    const int end = (int)fp8_end(x, room);
    return {(int)fp8_begin(x, count, room), end, wave_last(end)};
}
__device__ __forceinline__ int fp8_tiles_of(int rows, int bm) { return (int)(((uint32_t)rows + (uint32_t)bm - 1u) / (uint32_t)bm); }

// Where tile `slot` of the row tiles of BM rows lies: every wave scans the row counts, 64 experts at a time.  False past the last
// tile.
template <int BM>
__device__ __forceinline__ bool fp8_find_tile(const void *m_sizes, int ms_i64, int E, int64_t R, int slot, int lane, int &expert,
                                              int64_t &row0, int &rows) {
    int tiles_before = 0, rows_before = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
        uint32_t count[1];
        fp8_load_counts(m_sizes, ms_i64, e0 + lane, E, R, count);
        const Fp8Counted c = fp8_cut(count[0], (uint32_t)R - (uint32_t)rows_before);
        const int t = fp8_tiles_of(c.end - c.begin, BM), ti = wave_inclusive_scan(t);
        const uint64_t past = __ballot(tiles_before + ti > slot);
        if (past) {
            const int src = __ffsll((unsigned long long)past) - 1;
            const int tile = slot - (tiles_before + __builtin_amdgcn_readlane(ti, src) - __builtin_amdgcn_readlane(t, src));
            const int begin = __builtin_amdgcn_readlane(c.begin, src) + tile * BM, end = __builtin_amdgcn_readlane(c.end, src);
            expert = e0 + src;
            row0 = (int64_t)rows_before + begin;
            rows = end - begin < BM ? end - begin : BM;
            return true;
        }
        rows_before += c.all;
        tiles_before += wave_last(ti);
    }
    return false;
}
// Row tiles that a launch has to provide for (the sizes are known on the device only).
inline int64_t fp8_max_tiles(int64_t R, int E, int bm) { return R / bm + (R < E ? R : E); }

}  // namespace mfl
