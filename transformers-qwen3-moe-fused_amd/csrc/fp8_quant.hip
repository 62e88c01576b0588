// Quantisation to e4m3 blocks and back.
//
// Rows: one scale per row and 128 elements; 16 lanes hold a block, 8 elements each, so the block's largest magnitude is four
// moves between the lanes of a row of 16 and a block's values leave as 16 stores of 8 bytes.  Reads 2 (or 4) bytes and writes
// 1 + 1/128 per element, no reuse: bound by memory.
#include "fp8.h"

namespace mfl {

namespace {

// 8 consecutive elements of a row from column k on as floats, zeros behind column K.  WIDE: the row can be read 16 bytes at a
// time (K a multiple of 8 and the base aligned), so a run of 8 lies inside or outside as a whole.
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T *row, int k, int K, float (&v)[8]) {
    if (WIDE) {
        union {
            uint4_t q[sizeof(T) / 2];
            T t[8];
        } u;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.q[i] = k < K ? ((const uint4_t *)(row + k))[i] : uint4_t{0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(u.t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f32(row[k + i]) : 0.0f;
    }
}

// Blocks of a launch are numbered row by row; a group of 16 lanes takes kPerGroup of them, a workgroup's groups side by side.
constexpr int kGroups = 16, kPerGroup = 4;

template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T *__restrict__ x, int64_t blocks, int K, int kb,
                                                         uint8_t *__restrict__ q, uint8_t *__restrict__ scale) {
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int64_t ld = fp8_ld(K), ld_scale = fp8_ld_scale(K);
    float v[kPerGroup][8];
    int64_t row[kPerGroup];
    int b[kPerGroup];
#pragma unroll
    for (int i = 0; i < kPerGroup; ++i) {
        const int64_t at = ((int64_t)blockIdx.x * kPerGroup + i) * kGroups + group;
        row[i] = at / kb, b[i] = (int)(at - row[i] * kb);
        load8<T, WIDE>(x + row[i] * K, b[i] * kFp8Block + lane * 8, at < blocks ? K : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kPerGroup; ++i) {
        const int64_t at = ((int64_t)blockIdx.x * kPerGroup + i) * kGroups + group;
        if (at < blocks)  // (the same for the 16 lanes of a group)
            fp8_store_block(v[i], q + row[i] * ld + b[i] * kFp8Block + lane * 8, scale + row[i] * ld_scale + b[i], lane == 0);
    }
}

// d/de and d/dg of h = silu(e) g, in fp32 from the three tensors, straight to quantised rows.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void silu_bwd_quant_kernel(const T *__restrict__ dh, const T *__restrict__ e,
                                                             const T *__restrict__ g, int64_t blocks, int N, int nb,
                                                             uint8_t *__restrict__ de_q, uint8_t *__restrict__ de_scale,
                                                             uint8_t *__restrict__ dg_q, uint8_t *__restrict__ dg_scale) {
    const int lane = threadIdx.x & 15;
    const int64_t at = (int64_t)blockIdx.x * kGroups + (threadIdx.x >> 4);
    if (at >= blocks) return;
    const int64_t row = at / nb;
    const int b = (int)(at - row * nb), n = b * kFp8Block + lane * 8;
    float d[8], ev[8], gv[8];
    load8<T, WIDE>(dh + row * N, n, N, d);
    load8<T, WIDE>(e + row * N, n, N, ev);
    load8<T, WIDE>(g + row * N, n, N, gv);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s = sigmoid_f32(ev[i]);
        const float de = d[i] * gv[i] * s * __builtin_fmaf(ev[i], 1.0f - s, 1.0f);
        gv[i] = d[i] * (ev[i] * s);
        ev[i] = de;
    }
    const int64_t out = row * fp8_ld(N) + n, out_scale = row * fp8_ld_scale(N) + b;
    fp8_store_block(ev, de_q + out, de_scale + out_scale, lane == 0);
    fp8_store_block(gv, dg_q + out, dg_scale + out_scale, lane == 0);
}

__device__ __forceinline__ float fp8_value(uint32_t byte) { return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0); }

// Eight elements a thread; out rows may start anywhere (stores of 16 bytes whatever the alignment, the last ones of a row one by one).
// 16384 x 2048 to bf16: 49 us with an element a thread, 21 so.
template <typename T>
__global__ __launch_bounds__(256) void dequant_rows_kernel(const uint8_t *__restrict__ q, const uint8_t *__restrict__ scale,
                                                           int64_t runs, int per_row, int K, T *__restrict__ out) {
    const int64_t ld = fp8_ld(K), ld_scale = fp8_ld_scale(K);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < runs; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row;
        const int k = (int)(i - row * per_row) * 8;
        uint2_t v = {0u, 0u};
        if (k + 8 <= K) {
            __builtin_memcpy(&v, q + row * ld + k, sizeof(v));
        } else {  // (a single row may end with its last column)
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k + u < K) v[u / 4] |= (uint32_t)q[row * ld + k + u] << 8 * (u % 4);
        }
        const float s = fp8_scale_of(scale[row * ld_scale + k / kFp8Block]);
        T o[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) o[u] = from_f32<T>(fp8_value(v[u / 4] >> 8 * (u % 4) & 0xffu) * s);
        T *const to = out + row * K + k;
        if (k + 8 <= K) {
            __builtin_memcpy(to, o, sizeof(o));
        } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k + u < K) to[u] = o[u];
        }
    }
}

// One workgroup per 128 x 128 block of a weight matrix; thread t holds every second row of one column.
template <typename T>
__global__ __launch_bounds__(256) void quant_blocks_kernel(const T *__restrict__ w, int N, int K, uint8_t *__restrict__ q,
                                                           float *__restrict__ scale) {
    __shared__ float part[4];
    const int kb = fp8_blocks(K), nb = fp8_blocks(N);
    const int64_t block = blockIdx.x;
    const int b = (int)(block % kb);
    const int64_t en = block / kb;
    const int64_t e = en / nb;
    const int n0 = (int)(en % nb) * kFp8Block;
    const int k = b * kFp8Block + (threadIdx.x & 127);
    const int rows = N - n0 < kFp8Block ? N - n0 : kFp8Block;
    const int64_t base = (e * N + n0) * K + k;
    float a = 0.0f;
    if (k < K)
        for (int r = threadIdx.x >> 7; r < rows; r += 2) a = __builtin_fmaxf(a, fp8_finite_abs(to_f32(w[base + (int64_t)r * K])));
    for (int d = 32; d; d >>= 1) a = __builtin_fmaxf(a, __shfl_xor(a, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
    __syncthreads();
    a = __builtin_fmaxf(__builtin_fmaxf(part[0], part[1]), __builtin_fmaxf(part[2], part[3]));
    const int byte = fp8_scale_byte(__float_as_uint(a));
    const float inverse = fp8_inverse_of(byte);
    if (threadIdx.x == 0) scale[block] = fp8_scale_of(byte);
    if (k < K)
        for (int r = threadIdx.x >> 7; r < rows; r += 2) {
            const float v = fp8_finite(to_f32(w[base + (int64_t)r * K]));
            q[base + (int64_t)r * K] = (uint8_t)fp8_pack4(v, 0.0f, 0.0f, 0.0f, inverse);
        }
}

template <typename T>
__global__ __launch_bounds__(256) void dequant_blocks_kernel(const uint8_t *__restrict__ q, const float *__restrict__ scale,
                                                             int N, int K, T *__restrict__ out) {
    const int kb = fp8_blocks(K), nb = fp8_blocks(N);
    const int64_t block = blockIdx.x;
    const int b = (int)(block % kb);
    const int64_t en = block / kb;
    const int64_t e = en / nb;
    const int n0 = (int)(en % nb) * kFp8Block;
    const int k = b * kFp8Block + (threadIdx.x & 127);
    const int rows = N - n0 < kFp8Block ? N - n0 : kFp8Block;
    const int64_t base = (e * N + n0) * K + k;
    const float s = scale[block];
    if (k < K)
        for (int r = threadIdx.x >> 7; r < rows; r += 2) out[base + (int64_t)r * K] = from_f32<T>(fp8_value(q[base + (int64_t)r * K]) * s);
}

__global__ __launch_bounds__(256) void pad_rows_kernel(const uint8_t *__restrict__ w, int64_t pieces, int K, int per_row,
                                                       uint8_t *__restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row;
        const int k = (int)(i - row * per_row) * 16;
        union {
            uint4_t v;
            uint64_t q[2];
            uint8_t b[16];
        } u;
        if (K >= 16) {
            // (the row's last piece: its last 16 bytes, moved down; byte by byte they would be a load behind the other)
            const int at = k + 16 <= K ? k : K - 16, moved = (k - at) * 8;
            __builtin_memcpy(&u.v, w + row * K + at, 16);
            if (moved >= 64) u.q[0] = u.q[1] >> (moved - 64), u.q[1] = 0u;
            else if (moved > 0) u.q[0] = u.q[0] >> moved | u.q[1] << (64 - moved), u.q[1] >>= moved;
        } else {
            u.v = uint4_t{0u, 0u, 0u, 0u};
#pragma unroll
            for (int j = 0; j < 15; ++j)
                if (j < K) u.b[j] = w[row * K + j];
        }
        *(uint4_t *)(out + i * 16) = u.v;
    }
}

constexpr int64_t kMaxGroups = 0xffffff;  // a launch's threads are counted in 32 bits

template <typename T>
bool wide_rows(const T *x, int K) {
    return K % 8 == 0 && aligned(x, 16);
}

}  // namespace

int fp8_quant_rows(const void *x, int dtype, int64_t R, int K, uint8_t *q, uint8_t *scale, hipStream_t stream) {
    const int kb = fp8_blocks(K);
    const int64_t blocks = R * kb, grid = (blocks + kGroups * kPerGroup - 1) / (kGroups * kPerGroup);
    if (grid > kMaxGroups) return MFL_ERR_SHAPE;
    MFL_DISPATCH_FLOAT(dtype, T, {
        if (wide_rows((const T *)x, K))
            quant_rows_kernel<T, true><<<(unsigned)grid, 256, 0, stream>>>((const T *)x, blocks, K, kb, q, scale);
        else
            quant_rows_kernel<T, false><<<(unsigned)grid, 256, 0, stream>>>((const T *)x, blocks, K, kb, q, scale);
    });
    return launch_status();
}

int fp8_silu_bwd_quant(const void *dh, const void *e, const void *g, int dtype, int64_t R, int N, uint8_t *de_q,
                       uint8_t *de_scale, uint8_t *dg_q, uint8_t *dg_scale, hipStream_t stream) {
    const int nb = fp8_blocks(N);
    const int64_t blocks = R * nb, grid = (blocks + kGroups - 1) / kGroups;
    if (grid > kMaxGroups) return MFL_ERR_SHAPE;
    MFL_DISPATCH_FLOAT(dtype, T, {
        if (wide_rows((const T *)dh, N) && wide_rows((const T *)e, N) && wide_rows((const T *)g, N))
            silu_bwd_quant_kernel<T, true><<<(unsigned)grid, 256, 0, stream>>>((const T *)dh, (const T *)e, (const T *)g, blocks, N,
                                                                              nb, de_q, de_scale, dg_q, dg_scale);
        else
            silu_bwd_quant_kernel<T, false><<<(unsigned)grid, 256, 0, stream>>>((const T *)dh, (const T *)e, (const T *)g, blocks, N,
                                                                               nb, de_q, de_scale, dg_q, dg_scale);
    });
    return launch_status();
}

int fp8_dequant_rows(const uint8_t *q, const uint8_t *scale, int64_t R, int K, void *out, int out_dtype, hipStream_t stream) {
    const int per_row = ceil_div(K, 8);
    const int64_t runs = R * per_row, want = (runs + 255) / 256;
    const unsigned grid = (unsigned)(want < 65536 ? want : 65536);
    MFL_DISPATCH_FLOAT(out_dtype, T, { dequant_rows_kernel<T><<<grid, 256, 0, stream>>>(q, scale, runs, per_row, K, (T *)out); });
    return launch_status();
}

int fp8_quant_blocks(const void *w, int dtype, int E, int N, int K, uint8_t *q, float *scale, hipStream_t stream) {
    const int64_t blocks = (int64_t)E * fp8_blocks(N) * fp8_blocks(K);
    if (blocks > kMaxGroups) return MFL_ERR_SHAPE;
    MFL_DISPATCH_FLOAT(dtype, T, { quant_blocks_kernel<T><<<(unsigned)blocks, 256, 0, stream>>>((const T *)w, N, K, q, scale); });
    return launch_status();
}

int fp8_pad_rows(const uint8_t *w, int64_t rows, int K, int ldw, uint8_t *out, hipStream_t stream) {
    const int64_t pieces = rows * (ldw / 16), want = (pieces + 255) / 256;
    pad_rows_kernel<<<(unsigned)(want < 65536 ? want : 65536), 256, 0, stream>>>(w, pieces, K, ldw / 16, out);
    return launch_status();
}

int fp8_dequant_blocks(const uint8_t *q, const float *scale, int E, int N, int K, void *out, int out_dtype, hipStream_t stream) {
    const int64_t blocks = (int64_t)E * fp8_blocks(N) * fp8_blocks(K);
    if (blocks > kMaxGroups) return MFL_ERR_SHAPE;
    MFL_DISPATCH_FLOAT(out_dtype, T, { dequant_blocks_kernel<T><<<(unsigned)blocks, 256, 0, stream>>>(q, scale, N, K, (T *)out); });
    return launch_status();
}

}  // namespace mfl
