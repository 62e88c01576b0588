// Expert products in 8-bit floating point, any shape: 64 x 64 tiles, both operands through registers into LDS, where they lie
// as bf16 (which holds every e4m3 value).  For what the other kernels leave: one step of the reduction, more than 512 experts,
// weights of odd rows for a few rows, weights off the 16-byte grid, offsets past 32 bits.
//
//   forward         out[r, n] = sum_b S[e, n / 128, b] sx[r, b] sum_{k in block b} x[r, k] w[e, n, k]
//   input gradient  out[r, k] = sum_b S[e, b, k / 128] sd[r, b] sum_{n in block b} d[r, n] w[e, n, k]
//
// A step is one block of 128 of the reduction: eight bf16 matrix instructions into fresh accumulators, and a multiply-add by
// both scales into the running fp32 sums (bf16 products for every output: fp8.h).  The weights are the first operand, so that
// a lane's accumulators belong to one row (its scale is the lane's) and to runs of four columns.  For widths that no 16-byte
// access fits the weights are read byte by byte; that, and the plain load-wait-multiply order, is what bounds it: 32768 rows, 128
// experts, 2048 to 768, fp32, weights off the grid 1226 us, its input gradient 2763 (tiles, weights on the grid: 217 and 197).
#include "fp8.h"

namespace mfl {

namespace {

constexpr int kTile = 64, kPitch = 272;  // rows of 128 bf16, 16 bytes apart in the banks

struct Bytes16 {
    uint8_t b[16];
};

// 16 e4m3 values as bf16 to LDS
__device__ __forceinline__ void store16(uint8_t *dst, const uint4_t v) {
    bf16x8 out[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int w = (int)v[i];
        out[i / 2][i % 2 * 4 + 0] = (bf16_t)__builtin_amdgcn_cvt_f32_fp8(w, 0);
        out[i / 2][i % 2 * 4 + 1] = (bf16_t)__builtin_amdgcn_cvt_f32_fp8(w, 1);
        out[i / 2][i % 2 * 4 + 2] = (bf16_t)__builtin_amdgcn_cvt_f32_fp8(w, 2);
        out[i / 2][i % 2 * 4 + 3] = (bf16_t)__builtin_amdgcn_cvt_f32_fp8(w, 3);
    }
    *(bf16x8 *)dst = out[0], *(bf16x8 *)(dst + 16) = out[1];
}

template <bool DX, bool GLU, typename TO>
__global__ __launch_bounds__(256) void fp8_generic_kernel(Fp8Product p) {
    constexpr int CB = GLU ? 2 : 1;
    __shared__ __attribute__((aligned(16))) uint8_t sa[kTile * kPitch];
    __shared__ __attribute__((aligned(16))) uint8_t sw[CB][kTile * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int e, rows;
    int64_t row0;
    if (!fp8_find_tile<kTile>(p.m_sizes, p.ms_i64, p.E, p.R, blockIdx.x, lane, e, row0, rows)) return;
    const int cols = DX ? p.K : p.N, red = DX ? p.N : p.K;
    const int col0 = blockIdx.y * kTile;
    const int64_t ld = fp8_ld(red), ld_scale = fp8_ld_scale(red);
    const int nbn = fp8_blocks(p.N), kbk = fp8_blocks(p.K);
    const int wr = (wave & 1) * 32, wc = (wave >> 1) * 32, l = lane & 31, half = lane >> 5;

    // source row of the rows of the tile that this thread copies (two of every four threads' chunks), and of its lane's row
    auto source = [&](int r) -> int64_t {
        int64_t i = row0 + (r < rows ? r : rows - 1);
        if (!DX && p.row_idx != nullptr) {
            i = p.row_idx[i] / p.idx_div;
            i = i < 0 ? 0 : i >= p.src_rows ? p.src_rows - 1 : i;
        }
        return i;
    };
    const int64_t my_row = source(wr + l);
    const int64_t copy_row[2] = {source(tid >> 3), source(32 + (tid >> 3))};

    floatx16 acc[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c][i] = 0.0f;

    for (int term = 0; term < p.terms; ++term) {
        const Fp8Rows a = p.a[term];
        for (int b = 0; b < fp8_blocks(red); ++b) {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int r = q * 32 + (tid >> 3), ch = tid & 7;
                store16(sa + r * kPitch + ch * 32, *(const uint4_t *)(a.q + copy_row[q] * ld + b * kFp8Block + ch * 16));
            }
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                const uint8_t *w = p.w[DX ? term : c].q + (int64_t)e * p.N * p.K;
                if (!DX) {
                    const bool wide = p.K % 16 == 0 && ((uintptr_t)w & 15) == 0;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int r = q * 32 + (tid >> 3), ch = tid & 7;
                        const int n = col0 + r, k = b * kFp8Block + ch * 16;
                        union {
                            uint4_t v;
                            Bytes16 s;
                        } u;
                        u.v = uint4_t{0u, 0u, 0u, 0u};
                        if (n < p.N) {
                            const uint8_t *src = w + (int64_t)n * p.K + k;
                            if (wide && k < p.K) {
                                u.v = *(const uint4_t *)src;
                            } else if (!wide) {
#pragma unroll
                                for (int j = 0; j < 16; ++j)
                                    if (k + j < p.K) u.s.b[j] = src[j];
                            }
                        }
                        store16(sw[c] + r * kPitch + ch * 32, u.v);
                    }
                } else {
                    // 128 rows of the weights by 64 columns, stored with the reduction contiguous: a thread takes one
                    // column of 32 rows (neighbouring threads neighbouring columns)
                    const int k = col0 + (tid & 63), n0 = b * kFp8Block + (tid >> 6) * 32;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        union {
                            uint4_t v;
                            Bytes16 s;
                        } u;
                        u.v = uint4_t{0u, 0u, 0u, 0u};
                        if (k < p.K) {
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (n0 + q * 16 + j < p.N) u.s.b[j] = w[(int64_t)(n0 + q * 16 + j) * p.K + k];
                        }
                        store16(sw[c] + (tid & 63) * kPitch + (tid >> 6) * 64 + q * 32, u.v);
                    }
                }
            }
            __syncthreads();
            const float row_scale = fp8_scale_of(a.scale[my_row * ld_scale + b]);
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                const Fp8Matrix &m = p.w[DX ? term : c];
                const int64_t at = DX ? ((int64_t)e * nbn + b) * kbk + col0 / kFp8Block : ((int64_t)e * nbn + col0 / kFp8Block) * kbk + b;
                const float scale = m.scale[at];
                floatx16 part;
#pragma unroll
                for (int i = 0; i < 16; ++i) part[i] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const bf16x8 fw = *(const bf16x8 *)(sw[c] + (wc + l) * kPitch + ks * 32 + half * 16);
                    const bf16x8 fa = *(const bf16x8 *)(sa + (wr + l) * kPitch + ks * 32 + half * 16);
                    part = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fw, fa, part, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c][i] = __builtin_fmaf(scale, part[i] * row_scale, acc[c][i]);  // (the product of the two scales may overflow by itself)
            }
        }
    }
    if (wr + l >= rows) return;
    const int64_t at = (row0 + wr + l) * cols;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int n = col0 + wc + 8 * (i / 4) + 4 * half + i % 4;
        if (n >= cols) continue;
        if (GLU) {
            const float ev = acc[0][i], gv = acc[CB - 1][i];
            const float h = ev * sigmoid_f32(ev) * gv;
            if (p.h32 != nullptr)
                p.h32[at + n] = h;
            else
                ((TO *)p.out)[at + n] = from_f32<TO>(h);
            if (p.e_out != nullptr) ((TO *)p.e_out)[at + n] = from_f32<TO>(ev);
            if (p.g_out != nullptr) ((TO *)p.g_out)[at + n] = from_f32<TO>(gv);
        } else {
            ((TO *)p.out)[at + n] = from_f32<TO>(acc[0][i]);
        }
    }
}

}  // namespace

int gemm_fp8_generic(const Fp8Product &p, hipStream_t stream) {
    const int64_t tiles = fp8_max_tiles(p.R, p.E, kTile);
    const dim3 grid((unsigned)tiles, (unsigned)ceil_div(p.dx ? p.K : p.N, kTile));
    if (grid.y > 65535u || tiles > 0xffffff) return MFL_ERR_SHAPE;  // (a launch's threads are counted in 32 bits)
    MFL_DISPATCH_FLOAT(p.out_dtype, TO, {
        if (p.dx)
            fp8_generic_kernel<true, false, TO><<<grid, 256, 0, stream>>>(p);
        else if (p.glu)
            fp8_generic_kernel<false, true, TO><<<grid, 256, 0, stream>>>(p);
        else
            fp8_generic_kernel<false, false, TO><<<grid, 256, 0, stream>>>(p);
    });
    return launch_status();
}

}  // namespace mfl
