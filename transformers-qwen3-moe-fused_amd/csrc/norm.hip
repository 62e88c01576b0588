// The residual's addition and the root-mean-square norm behind it, forward and backward, and with rows in 8-bit blocks as the
// result (norm_parts.h has the arithmetic).
#include "fp8.h"
#include "norm_parts.h"
#include "ops.h"

namespace mfl {

namespace {

// ---- forward --------------------------------------------------------------------------------------------------------------
// A row belongs to LANES threads, which hold it in registers, 8 C elements each in C runs of 8: one pass over memory, which is all
// that bounds it where there are rows enough to fill the chip.  bf16 with a residual: 16384 x 2048 44.6 us, 6.0 TB/s of the 2 + 2
// rows that it has to read and write, 4096 x 8192 44.3, 1024 x 32768 52.5; to 8-bit rows 16384 x 2048 50.  y may be x, and s x or
// the residual: what a thread reads of a row it has read before it writes there.
template <typename T, typename TW, int LANES, int C, bool FP8, bool WHOLE>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void norm_fwd_kernel(const T *x, const T *residual, const TW *__restrict__ weight,
                                                                           T *y, T *s, uint8_t *__restrict__ q,
                                                                           uint8_t *__restrict__ scale, int64_t R, int H,
                                                                           double eps) {
    constexpr int ROWS = LANES < 256 ? 256 / LANES : 1, WAVES = LANES / 64;
    __shared__ double part[ROWS * WAVES];
    const int i = threadIdx.x % LANES;
    int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
    const bool in = row < R;
    if (!in) row = R - 1;  // (computed along, not stored)
    x += row * H;
    Eight<T, WHOLE> v[C];
    Eight<TW, WHOLE> w[C];
    constexpr bool EARLY = C == 1;  // the weight is asked for before the sum's end where the registers hold it (1024 x 32768: 92 us, 52 late)
#pragma unroll
    for (int c = 0; c < C; ++c) v[c].load(x, (c * LANES + i) * 8, H);
    if (residual != nullptr) {
        Eight<T, WHOLE> o[C];
#pragma unroll
        for (int c = 0; c < C; ++c) o[c].load(residual + row * H, (c * LANES + i) * 8, H);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            add_rounded(v[c], o[c]);
            if (in) v[c].store(s + row * H, (c * LANES + i) * 8, H);
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c) sum = sum_of_squares(v[c], sum);
    if (EARLY) w[0].load(weight, i * 8, H);
    sum = wave_sum(sum);
    if (LANES > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int u = 0; u < WAVES; ++u) sum += part[threadIdx.x / LANES * WAVES + u];
    }
    const double r = inverse_root(sum / (double)H + eps);
    if (!in) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k = (c * LANES + i) * 8;
        if (!EARLY) w[c].load(weight, k, H);
#pragma unroll
        for (int u = 0; u < 8; ++u) v[c].v[u] = normed(v[c].v[u], r, w[c].v[u]);
        if (y != nullptr) v[c].store(y + row * H, k, H);
        if constexpr (FP8) {
            float f[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) f[u] = k + u < H ? to_f32(v[c].v[u]) : 0.0f;
            if (k < fp8_ld(H))  // (the 16 lanes of a block alike)
                fp8_store_block(f, q + row * fp8_ld(H) + k, scale + row * fp8_ld_scale(H) + k / kFp8Block, (i & 15) == 0);
        }
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------
// With u = s r and g = dy w: dx = r (g - u mean(g u)) + ds, dw = sum over the rows of dy u.  s is read as the forward pass left
// it and its r found again, which costs a sum beside the one that is needed anyway.  A group of LANES threads takes every
// gridDim.x * GROUPS-th row and keeps its columns' share of dw in registers; the groups of a workgroup meet in LDS, the workgroups
// in `partial` (workgroup, H), which a second kernel adds up in order.  Memory bounds it too: bf16 with ds, 16384 x 2048 50 us for
// both kernels, 5.4 TB/s of three rows read and one written (49 with the second sum in 32 bits, which rows near their type's end pass).
// dx may be dy, ds or s, so whatever is to be on its way over a store is asked for in front of it.
// BARE: without eps a row around 2^-127 has an r that 32 bits do not hold: such rows are taken as 2^64 s.  (A kernel of its own: two products
// more an element for every row take 16384 x 2048 from 50 to 59 us, a second copy of the loop behind a question to 56.)
template <typename T, typename TW, int LANES, int C, int THREADS, bool WHOLE, bool BARE>
__global__ __launch_bounds__(THREADS) void norm_bwd_kernel(const T *dy, const T *ds, const T *s, const TW *__restrict__ weight, T *dx,
                                                          float *__restrict__ partial, int64_t R, int H, double eps) {
    constexpr int GROUPS = THREADS / LANES, WAVES = LANES / 64;
    constexpr bool ONE = C == 1;
    // s and dy stay in registers between a row's two passes where they fit; else they are read again, from the caches (1024 x 32768
    // in bf16: 251 us in registers, 153 so, where dw and the rest still spill 47; 2048 x 16384: 81 in registers, 90 so)
    constexpr int HELD = C == 2 ? C : 1;
    constexpr bool AHEAD = WHOLE && ONE;  // the next row is asked for before this one's sums are there (16384 x 2048: 61 -> 50 us)
    __shared__ double squares[2][GROUPS * WAVES];
    __shared__ double alongs[2][GROUPS * WAVES];
    extern __shared__ float shared_dw[];  // (GROUPS - 1, LANES * C * 8) where the groups are many
    const int i = threadIdx.x % LANES, group = threadIdx.x / LANES;
    float dw[C][8];
    Eight<TW, WHOLE> w;
    if (ONE) w.load(weight, i * 8, H);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int u = 0; u < 8; ++u) dw[c][u] = 0.0f;
    int turn = 0;
    Eight<T, WHOLE> sv, g, d, next_s, next_g, next_d, held_s[HELD], held_g[HELD];
    const bool add = ds != nullptr && dx != nullptr;
    auto fetch = [&](int64_t row0, Eight<T, WHOLE> &a, Eight<T, WHOLE> &b, Eight<T, WHOLE> &e) {
        const int64_t at = (row0 + group < R ? row0 + group : R - 1) * H;
        a.load(s + at, i * 8, H);
        b.load(dy + at, i * 8, H);
        if (add) e.load(ds + at, i * 8, H);
    };
    const int64_t first = (int64_t)blockIdx.x * GROUPS, by = (int64_t)gridDim.x * GROUPS;
    if (AHEAD) fetch(first, next_s, next_g, next_d);
    // (every group of a workgroup takes as many turns: the rows' sums wait for one another where a row has several waves)
    for (int64_t row0 = first; row0 < R; row0 += by, turn ^= 1) {
        const int64_t row = row0 + group;
        const bool in = row < R;
        const int64_t at = (in ? row : R - 1) * H;
        if (AHEAD) {
            sv = next_s, g = next_g, d = next_d;
            if (row0 + by < R) fetch(row0 + by, next_s, next_g, next_d);
        } else if (ONE) {
            fetch(row0, sv, g, d);
        }
        double square = 0.0, along = 0.0;  // (32 bits hold no square of a 32-bit or bf16 value past 2^64, nor a sum of many near 2^120)
#pragma unroll HELD
        for (int c = 0; c < C; ++c) {
            if (!ONE) {
                sv.load(s + at, (c * LANES + i) * 8, H);
                g.load(dy + at, (c * LANES + i) * 8, H);
                w.load(weight, (c * LANES + i) * 8, H);
                if (HELD == C) held_s[c] = sv, held_g[c] = g;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float a = to_f32(sv.v[u]);
                square = __builtin_fma((double)a, (double)a, square);
                along = __builtin_fma((double)(to_f32(g.v[u]) * to_f32(w.v[u])), (double)a, along);
            }
        }
        square = wave_sum(square), along = wave_sum(along);
        if (WAVES > 1) {
            if ((threadIdx.x & 63) == 0) squares[turn][threadIdx.x >> 6] = square, alongs[turn][threadIdx.x >> 6] = along;
            __syncthreads();  // (two tables in turn: one barrier a row)
            square = 0.0, along = 0.0;
#pragma unroll
            for (int u = 0; u < WAVES; ++u) square += squares[turn][group * WAVES + u], along += alongs[turn][group * WAVES + u];
        }
        double root = inverse_root(square / (double)H + eps);
        float up = 1.0f;
        if (BARE && root > 0x1p127) up = 0x1p64f, root *= 0x1p-64, along *= 0x1p64;
        const float r = (float)root, back = (float)(along / (double)H * root * root);  // dx = r (g - s back) + ds
        if (!in) continue;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!ONE) {
                if (HELD == C) {
                    sv = held_s[c], g = held_g[c];
                } else {
                    sv.load(s + at, (c * LANES + i) * 8, H);
                    g.load(dy + at, (c * LANES + i) * 8, H);
                }
                w.load(weight, (c * LANES + i) * 8, H);
                if (add) d.load(ds + at, (c * LANES + i) * 8, H);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                float a = to_f32(sv.v[u]);
                if (BARE) a *= up;
                const float b = to_f32(g.v[u]);
                dw[c][u] = __builtin_fmaf(b, a * r, dw[c][u]);
                float o = r * __builtin_fmaf(-a, back, b * to_f32(w.v[u]));
                if (BARE) o *= up;
                if (add) o += to_f32(d.v[u]);
                sv.v[u] = from_f32<T>(o);
            }
            if (dx != nullptr) sv.store(dx + at, (c * LANES + i) * 8, H);
        }
    }
    if (partial == nullptr) return;
    if (GROUPS > 1) {
        constexpr int WIDTH = LANES * C * 8;
        if (group > 0) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int u = 0; u < 8; ++u) shared_dw[(group - 1) * WIDTH + (c * 8 + u) * LANES + i] = dw[c][u];
        }
        __syncthreads();
        if (group > 0) return;
        for (int o = 0; o < GROUPS - 1; ++o)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int u = 0; u < 8; ++u) dw[c][u] += shared_dw[o * WIDTH + (c * 8 + u) * LANES + i];
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k = (c * LANES + i) * 8;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (k + u < H) partial[(int64_t)blockIdx.x * H + k + u] = dw[c][u];
    }
}

// dw (H) = the sum of `parts` rows of partial; 16 columns a workgroup, four of them a thread, 64 threads a column (512 rows of 2048:
// 10.8 us with a column and a load of four bytes a thread, 2.5 so).
template <typename TW>
__global__ __launch_bounds__(256) void norm_dw_kernel(const float *__restrict__ partial, TW *__restrict__ dw, int parts, int H) {
    __shared__ float sums[64][17];
    const int part = threadIdx.x >> 2, k = blockIdx.x * 16 + (threadIdx.x & 3) * 4;
    floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (k + 4 <= H) {
#pragma unroll 8
        for (int p = part; p < parts; p += 64) {
            floatx4 v;
            __builtin_memcpy(&v, partial + (int64_t)p * H + k, 16);
            sum += v;
        }
    } else {
        for (int p = part; p < parts; p += 64)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k + u < H) sum[u] += partial[(int64_t)p * H + k + u];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) sums[part][(threadIdx.x & 3) * 4 + u] = sum[u];
    __syncthreads();
    const int col = threadIdx.x & 15, group = threadIdx.x >> 4;
    float v = sums[group * 4][col] + sums[group * 4 + 1][col] + sums[group * 4 + 2][col] + sums[group * 4 + 3][col];
    __syncthreads();
    sums[group][col] = v;
    __syncthreads();
    if (threadIdx.x >= 16 || blockIdx.x * 16 + col >= H) return;
    v = 0.0f;
#pragma unroll
    for (int p = 0; p < 16; ++p) v += sums[p][col];
    dw[blockIdx.x * 16 + col] = from_f32<TW>(v);
}

static_assert(MFL_NORM_WIDTH == 1024 * 4 * 8, "1024 threads of four runs");
constexpr int kBwdThreads = 512;

// threads of a row, and the backward kernel's workgroups
int lanes_of(int H) { return H <= 512 ? 64 : H <= 1024 ? 128 : H <= 2048 ? 256 : H <= 4096 ? 512 : 1024; }
int bwd_grid(int64_t R, int H) {
    const int lanes = lanes_of(H), groups = lanes < kBwdThreads ? kBwdThreads / lanes : 1;
    // (as many as are resident at once)
    const int64_t want = (R + groups - 1) / groups, most = (lanes < 1024 ? 2 : 1) * device_info().cu_count;
    return (int)(want < most ? want : most);
}

template <typename T, typename TW, bool FP8, bool WHOLE>
int launch_fwd(const NormCall &n, hipStream_t stream) {
#define MFL_NORM(L, C)                                                                                                          \
    norm_fwd_kernel<T, TW, L, C, FP8, WHOLE><<<(unsigned)((n.R + (L < 256 ? 256 / L : 1) - 1) / (L < 256 ? 256 / L : 1)),               \
                                        L < 256 ? 256 : L, 0, stream>>>((const T *)n.x, (const T *)n.residual,                   \
                                                                       (const TW *)n.weight, (T *)n.y, (T *)n.s, n.q, n.scale,   \
                                                                       n.R, n.H, (double)n.eps)
    const int H = n.H;
    if (H <= 512) MFL_NORM(64, 1);
    else if (H <= 1024) MFL_NORM(128, 1);
    else if (H <= 2048) MFL_NORM(256, 1);
    else if (H <= 4096) MFL_NORM(512, 1);
    else if (H <= 8192) MFL_NORM(1024, 1);
    else if (H <= 16384) MFL_NORM(1024, 2);
    else MFL_NORM(1024, 4);
#undef MFL_NORM
    return launch_status();
}

template <typename T, typename TW, bool WHOLE>
int launch_bwd(const NormCall &n, const void *dy, const void *ds, void *dx, void *dw, float *partial, hipStream_t stream) {
    const int grid = bwd_grid(n.R, n.H), H = n.H;
#define MFL_NORM(L, C)                                                                                                         \
    {                                                                                                                          \
        constexpr int threads = L < kBwdThreads ? kBwdThreads : L;                                                             \
        constexpr int room = (threads / L - 1) * L * C * 8 * 4;  /* 14 KB at most */                                           \
        auto kernel = n.eps == 0.0f ? norm_bwd_kernel<T, TW, L, C, threads, WHOLE, true>                                       \
                                    : norm_bwd_kernel<T, TW, L, C, threads, WHOLE, false>;                                     \
        if (grid > 0)                                                                                                          \
            kernel<<<grid, threads, room, stream>>>((const T *)dy, (const T *)ds, (const T *)n.s, (const TW *)n.weight, (T *)dx, \
                                                    dw != nullptr ? partial : nullptr, n.R, H, (double)n.eps);                 \
    }
    if (H <= 512) MFL_NORM(64, 1)
    else if (H <= 1024) MFL_NORM(128, 1)
    else if (H <= 2048) MFL_NORM(256, 1)
    else if (H <= 4096) MFL_NORM(512, 1)
    else if (H <= 8192) MFL_NORM(1024, 1)
    else if (H <= 16384) MFL_NORM(1024, 2)
    else MFL_NORM(1024, 4)
#undef MFL_NORM
    if (dw != nullptr) norm_dw_kernel<TW><<<ceil_div(H, 16), 256, 0, stream>>>(partial, (TW *)dw, grid, H);
    return launch_status();
}

template <typename T, typename TW>
int fwd(const NormCall &n, hipStream_t stream) {
    if (n.H % 8 == 0) return n.q ? launch_fwd<T, TW, true, true>(n, stream) : launch_fwd<T, TW, false, true>(n, stream);
    return n.q ? launch_fwd<T, TW, true, false>(n, stream) : launch_fwd<T, TW, false, false>(n, stream);
}
template <typename T, typename TW>
int bwd(const NormCall &n, const void *dy, const void *ds, void *dx, void *dw, float *partial, hipStream_t stream) {
    if (n.H % 8 == 0) return launch_bwd<T, TW, true>(n, dy, ds, dx, dw, partial, stream);
    return launch_bwd<T, TW, false>(n, dy, ds, dx, dw, partial, stream);
}

}  // namespace

// (a launch's threads are counted in 32 bits: below 2^32 with the last workgroup's, too)
int64_t add_rms_norm_rows(int H) { return (1ll << 32) / lanes_of(H) - 1024; }

int add_rms_norm(const NormCall &n, hipStream_t stream) {
    int rc = MFL_OK;
    MFL_DISPATCH_FLOAT(n.dtype, T, {
        if (n.weight_dtype == n.dtype) rc = fwd<T, T>(n, stream);
        else rc = fwd<T, float>(n, stream);
    });
    return rc;
}

size_t add_rms_norm_bwd_workspace(int64_t R, int H) { return (size_t)bwd_grid(R, H) * H * sizeof(float); }

int add_rms_norm_bwd(const NormCall &n, const void *dy, const void *ds, void *dx, void *dw, float *partial, hipStream_t stream) {
    int rc = MFL_OK;
    MFL_DISPATCH_FLOAT(n.dtype, T, {
        if (n.weight_dtype == n.dtype) rc = bwd<T, T>(n, dy, ds, dx, dw, partial, stream);
        else rc = bwd<T, float>(n, dy, ds, dx, dw, partial, stream);
    });
    return rc;
}

}  // namespace mfl
