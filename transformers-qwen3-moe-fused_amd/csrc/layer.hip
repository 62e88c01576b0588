// The whole sparse expert layer for a few tokens: router, softmax and top-k, gated experts, weighted sum; with the residual's
// addition and the norm in front and the stream's addition behind where asked for.
#include <type_traits>

#include "fp8.h"
#include "norm_parts.h"
#include "ops.h"

namespace mfl {

namespace {

constexpr int kTokens = MFL_LAYER_TOKENS, kMaxExperts = 1024, kMaxChosen = 64;
constexpr int kWaves = 8, kThreads = kWaves * 64;
static_assert(kTokens == 16, "an expert's rows are the 16 columns of one matrix instruction");

struct Layer {
    mfl_moe_layer c;
    void *out, *logits;
    const void *stream;  // (T, H): what is added to out, or null
    void *stream_out;    // where the first kernel leaves it, or null (no residual: it is x)
    const void *rows;    // the rows that the experts read, `ld` apart: normed rows, in 8-bit layers what their blocks stand for in bf16
    void *rows_out;      // where the first kernel leaves them, or null (they are x)
    int64_t ld;
    float *h;  // (T k, ldh): the gated unit's results, a row per (expert, token) in this order
    int64_t ldh;
};

// ---- first kernel: stream, norm, logits -----------------------------------------------------------------------------------
// A workgroup has two experts and all tokens.  It norms the tokens itself (the rows are read once more per workgroup, from the
// caches), so that nothing has to wait for another workgroup; token t is written by workgroup t.
constexpr int kRouterExperts = 2;

template <typename T, int TOKENS, bool FP8, bool WHOLE>
__global__ __launch_bounds__(256) void layer_router_kernel(Layer p) {
    constexpr int SUMS = kRouterExperts * TOKENS;
    __shared__ double root[TOKENS];
    __shared__ double part[4][SUMS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int H = p.c.H, E = p.c.E, tokens = (int)p.c.T;
    const bool norm = p.c.norm_weight != nullptr;
    const T *const x = (const T *)p.c.x, *const residual = (const T *)p.c.residual, *const weight = (const T *)p.c.norm_weight;
    const int e0 = blockIdx.x * kRouterExperts;
    const T *router[kRouterExperts];
#pragma unroll
    for (int j = 0; j < kRouterExperts; ++j) router[j] = (const T *)p.c.router + (int64_t)(e0 + j < E ? e0 + j : E - 1) * H;

    auto stream_of = [&](int t, int k) {
        Eight<T, WHOLE> v;
        v.load(x + (int64_t)t * H, k, H);
        if (residual != nullptr) {
            Eight<T, WHOLE> o;
            o.load(residual + (int64_t)t * H, k, H);
            add_rounded(v, o);
        }
        return v;
    };
    if (norm) {
        for (int t = wave; t < tokens; t += 4) {
            double sum = 0.0;
            for (int k = lane * 8; k < H; k += 512) sum = sum_of_squares(stream_of(t, k), sum);
            sum = wave_sum(sum);
            if (lane == 0) root[t] = inverse_root(sum / (double)H + (double)p.c.eps);
        }
        __syncthreads();
    }
    double acc[kRouterExperts][TOKENS];
#pragma unroll
    for (int j = 0; j < kRouterExperts; ++j)
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) acc[j][t] = 0.0;
    const int padded = FP8 ? (int)fp8_ld(H) : H;  // (8-bit: whole blocks of 128, the same for the 16 lanes of a block)
    for (int k = tid * 8; k < padded; k += 2048) {
        Eight<T, WHOLE> w, r[kRouterExperts];
        if (norm) w.load(weight, k, H);
#pragma unroll
        for (int j = 0; j < kRouterExperts; ++j) r[j].load(router[j], k, H);
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) {
            Eight<T, WHOLE> v = stream_of(t < tokens ? t : tokens - 1, k);
            const bool mine = t < tokens && t % gridDim.x == blockIdx.x;
            if (norm) {
                if (mine && p.stream_out != nullptr) v.store((T *)p.stream_out + (int64_t)t * H, k, H);
                const double length = root[t < tokens ? t : tokens - 1];
#pragma unroll
                for (int i = 0; i < 8; ++i) v.v[i] = normed(v.v[i], length, w.v[i]);
            }
            if (mine && p.rows_out != nullptr) {
                if constexpr (FP8) {
                    float f[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = k + i < H ? to_f32(v.v[i]) : 0.0f;
                    fp8_store_wide(f, (bf16_t *)p.rows_out + t * p.ld + k);
                } else {
                    v.store((T *)p.rows_out + t * p.ld, k, H);
                }
            }
#pragma unroll
            for (int j = 0; j < kRouterExperts; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    // (behind column H the stream, the weight and the router are zeros; a NaN of the token's stays its own)
                    acc[j][t] = __builtin_fma((double)to_f32(v.v[i]), (double)to_f32(r[j].v[i]), acc[j][t]);
        }
    }
#pragma unroll
    for (int j = 0; j < kRouterExperts; ++j)
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) {
            const double sum = wave_sum(acc[j][t]);
            if (lane == 0) part[wave][j * TOKENS + t] = sum;
        }
    __syncthreads();
    if (tid < SUMS) {
        const int e = e0 + tid / TOKENS, t = tid % TOKENS;
        if (e < E && t < tokens)
            ((T *)p.logits)[(int64_t)t * E + e] = from_f32<T>((float)(part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]));
    }
}

// ---- routing, found by every workgroup of the other kernels from the logits -----------------------------------------------
// Lists in LDS: the experts that some token chose, ascending, each with its (token, weight) pairs, tokens ascending.
struct Routing {
    uint32_t mask[kMaxExperts];  // the tokens that chose an expert; then the expert's first pair
    int16_t expert[kMaxExperts];
    int16_t first[kMaxExperts + 1];
    float weight[kTokens * kMaxChosen];
    uint8_t token[kTokens * kMaxChosen];
    float own_weight[kTokens][kMaxChosen];
    int16_t own_expert[kTokens][kMaxChosen];
    int experts;
    uint32_t lost;  // the tokens that choose none
};

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_max_step(int x) {
    const int y = __builtin_amdgcn_update_dpp(x, x, CTRL, ROW_MASK, 0xf, false);
    return x > y ? x : y;
}
__device__ __forceinline__ int wave_max(int x) {
    x = dpp_max_step<0x111, 0xf>(x);  // (the order of wave_inclusive_scan)
    x = dpp_max_step<0x112, 0xf>(x);
    x = dpp_max_step<0x114, 0xf>(x);
    x = dpp_max_step<0x118, 0xf>(x);
    x = dpp_max_step<0x142, 0xa>(x);
    x = dpp_max_step<0x143, 0xc>(x);
    return wave_last(x);
}

// One token by one wave; PER_LANE: experts lane, lane + 64, ...
template <typename T, int PER_LANE>
__device__ __forceinline__ void choose(const T *logits, int t, int E, int k, int renorm, Routing &r, int lane) {
    constexpr int kNone = -0x7fffffff - 1;
    float v[PER_LANE];
    int key[PER_LANE];  // the order of the values as whole numbers (-0 as 0)
    int top = kNone;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        const int e = lane + 64 * i;
        v[i] = e < E ? to_f32(logits[(int64_t)t * E + e]) + 0.0f : -INFINITY;
        nan |= v[i] != v[i];
        const int bits = __float_as_int(v[i]);
        key[i] = e < E ? bits ^ ((bits >> 31) & 0x7fffffff) : kNone;
        top = top > key[i] ? top : key[i];
    }
    top = wave_max(top);
    const float largest = __int_as_float(top ^ ((top >> 31) & 0x7fffffff));
    if (__any(nan) || __builtin_isinf(largest)) {
        if (lane == 0) atomicOr(&r.lost, 1u << t);
        for (int j = lane; j < k; j += 64) r.own_expert[t][j] = -1;
        return;
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) sum += expf(v[i] - largest);  // (0 past the last expert)
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    float mine = 0.0f, chosen = 0.0f;
    int mine_e = 0;
    for (int j = 0; j < k; ++j) {
        int best = kNone, at = 0;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (key[i] > best) best = key[i], at = i;  // (ascending ids: the lower of equals)
        const int m = j == 0 ? top : wave_max(best);
        // of the lanes with that value the lowest expert id: the least i, then the least lane
        const uint64_t owners = __ballot(best == m);
        int e;
        if (__popcll(owners) == 1) {
            const int o = __ffsll((unsigned long long)owners) - 1;
            e = __builtin_amdgcn_readlane(at, o) * 64 + o;
        } else {
            e = -wave_max(best == m ? -(at * 64 + lane) : kNone);
        }
        const float p = expf(__int_as_float(m ^ ((m >> 31) & 0x7fffffff)) - largest) / sum;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (e == lane + 64 * i) key[i] = kNone;
        if (lane == j) mine = p, mine_e = e;
        chosen += p;
    }
    if (lane < k) {
        r.own_expert[t][lane] = (int16_t)mine_e;
        r.own_weight[t][lane] = renorm ? mine / chosen : mine;
        atomicOr(&r.mask[mine_e], 1u << t);
    }
}

template <typename T>
__device__ __forceinline__ void find_routing(const Layer &p, Routing &r) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int E = p.c.E, k = p.c.k, tokens = (int)p.c.T;
    for (int e = tid; e < E; e += kThreads) r.mask[e] = 0u;
    if (tid == 0) r.lost = 0u;
    __syncthreads();
    for (int t = wave; t < tokens; t += kWaves) {
        const T *const logits = (const T *)p.logits;
        if (E <= 128) choose<T, 2>(logits, t, E, k, p.c.renorm, r, lane);
        else if (E <= 256) choose<T, 4>(logits, t, E, k, p.c.renorm, r, lane);
        else choose<T, 16>(logits, t, E, k, p.c.renorm, r, lane);
    }
    __syncthreads();
    if (wave == 0) {
        int experts = 0, pairs = 0;
        for (int e0 = 0; e0 < E; e0 += 64) {
            const uint32_t mask = e0 + lane < E ? r.mask[e0 + lane] : 0u;
            const uint64_t hit = __ballot(mask != 0u);
            const int n = __popc(mask), upto = wave_inclusive_scan(n);
            if (mask != 0u) {
                const int at = experts + __popcll(hit & ((1ull << lane) - 1));
                r.expert[at] = (int16_t)(e0 + lane);
                r.first[at] = (int16_t)(pairs + upto - n);
            }
            if (e0 + lane < E) r.mask[e0 + lane] = mask | (uint32_t)(pairs + upto - n) << 16;
            experts += __popcll(hit);
            pairs += wave_last(upto);
        }
        if (lane == 0) r.experts = experts, r.first[experts] = (int16_t)pairs;
    }
    __syncthreads();
    for (int i = tid; i < tokens * k; i += kThreads) {
        const int t = i / k, j = i - t * k, e = r.own_expert[t][j];
        if (e < 0) continue;
        const uint32_t m = r.mask[e];
        const int at = (int)(m >> 16) + __popc(m & ((1u << t) - 1u));
        r.token[at] = (uint8_t)t;
        r.weight[at] = r.own_weight[t][j];
    }
    __syncthreads();
}

// ---- operands ---------------------------------------------------------------------------------------------------------------
// A load is 16 bytes of a weight's row, `kRun` elements; the four quarters of a wave hold neighbouring runs, so that a step is
// 4 kRun elements of 16 rows.  Which elements a matrix instruction's lanes hold does not matter as long as both operands agree.
template <typename T, bool FP8>
struct Weights {
    typedef typename std::conditional<FP8, uint8_t, T>::type Element;
    static constexpr int kRun = 16 / (int)sizeof(Element), kStep = 4 * kRun;
};

// `count` (a constant) elements of a row from k on; zeros from column K on.  WHOLE: K is a multiple of count.
template <bool WHOLE, int BYTES, typename E>
__device__ __forceinline__ void load_run(const E *row, int k, int K, void *to) {
    constexpr int count = BYTES / (int)sizeof(E);
    if (WHOLE ? k < K : k + count <= K) {
        __builtin_memcpy(to, row + k, BYTES);
    } else {
#pragma unroll
        for (int i = 0; i < count; ++i) ((E *)to)[i] = !WHOLE && k + i < K ? row[k + i] : (E)0;
    }
}

struct alignas(16) Run {
    uint4_t v;
};

__device__ __forceinline__ floatx4 mfma_f32(const float (&a)[4], const float (&b)[4], floatx4 acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
    return acc;
}
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// ---- gate and up --------------------------------------------------------------------------------------------------------------
// An item is an expert's eight columns of either matrix, side by side as the 16 rows of one tile, times the expert's tokens as its
// 16 columns; the eight waves share the reduction and meet in LDS.  Weights straight from memory into the matrix unit's registers.
typedef floatx4 Parts[2][kWaves][64];

template <typename T, bool FP8, bool WHOLE>
__device__ __forceinline__ void gate_up_item(const Layer &p, const Routing &r, int at, int tile, floatx4 (*part)[64], int finisher) {
    typedef Weights<T, FP8> W;
    typedef typename W::Element Element;
    typedef typename std::conditional<FP8, bf16_t, T>::type X;
    constexpr int kRun = W::kRun, kStep = W::kStep, kRowBytes = kRun * (int)sizeof(X);
    constexpr int U = FP8 ? 4 : 8;  // steps whose loads are in flight together
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int H = p.c.H, I = p.c.I;
    const int e = __builtin_amdgcn_readfirstlane(r.expert[at]);
    const int first = __builtin_amdgcn_readfirstlane(r.first[at]);
    const int rows = __builtin_amdgcn_readfirstlane(r.first[at + 1]) - first;
    const int col = tile * 8 + (n & 7);
    const Element *const w = (const Element *)(n < 8 ? p.c.w_gate : p.c.w_up) + ((int64_t)e * I + (col < I ? col : I - 1)) * H;
    const X *const x = (const X *)p.rows + r.token[first + (n < rows ? n : rows - 1)] * p.ld;
    // whole blocks of 128 a wave where weights have scales
    constexpr int kUnit = FP8 ? 2 : 1;
    const int steps = (H + kStep - 1) / kStep, share = ((steps + kWaves - 1) / kWaves + kUnit - 1) / kUnit * kUnit;
    const int begin = wave * share, end = begin + share < steps ? begin + share : steps;
    const int nb = fp8_blocks(I), kb = fp8_blocks(H);
    const float *scale = nullptr;
    if (FP8) {
        const int64_t block = ((int64_t)e * nb + tile * 8 / kFp8Block) * kb;
        scale = (g < 2 ? p.c.s_gate : p.c.s_up) + block;  // (of the results that the lane holds, not of the rows that it loads)
    }
    floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = begin; s0 < end; s0 += U) {
        Run a[U];
        struct alignas(16) {
            X v[kRun];
        } b[U];
        float block_scale[U / 2];
#pragma unroll
        for (int u = 0; u < U; ++u) load_run<WHOLE, 16>(w, s0 + u < end ? (s0 + u) * kStep + g * kRun : H, H, &a[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = s0 + u < end ? (s0 + u) * kStep + g * kRun : H;
            if (FP8) {  // (rows of whole blocks)
                if (s0 + u < end) __builtin_memcpy(b[u].v, x + k, kRowBytes);
                else __builtin_memset(b[u].v, 0, kRowBytes);
            } else {
                load_run<WHOLE, kRowBytes>(x, k, H, b[u].v);
            }
        }
        if (FP8) {
#pragma unroll
            for (int u = 0; u < U / 2; ++u) block_scale[u] = s0 + 2 * u < end ? scale[(s0 + 2 * u) / 2] : 0.0f;
        }
        if constexpr (FP8) {
#pragma unroll
            for (int u = 0; u < U / 2; ++u) {
                floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    union {
                        Run r;
                        intx2 t[2];
                    } f = {a[2 * u + q]};
#pragma unroll
                    for (int o = 0; o < 2; ++o) {
                        bf16x8 bv;
                        __builtin_memcpy(&bv, b[2 * u + q].v + 8 * o, 16);
                        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_widen(f.t[o], 1.0f), bv, sum, 0, 0, 0);
                    }
                }
                if (s0 + 2 * u < end)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(block_scale[u], sum[i], acc[i]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if constexpr (std::is_same<T, bf16_t>::value) {
                    bf16x8 av, bv;
                    __builtin_memcpy(&av, &a[u], 16);
                    __builtin_memcpy(&bv, &b[u], 16);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bv, acc, 0, 0, 0);
                } else if constexpr (std::is_same<T, f16_t>::value) {
                    f16x8 av, bv;
                    __builtin_memcpy(&av, &a[u], 16);
                    __builtin_memcpy(&bv, &b[u], 16);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, bv, acc, 0, 0, 0);
                } else {
                    float av[4], bv[4];
                    __builtin_memcpy(av, &a[u], 16);
                    __builtin_memcpy(bv, &b[u], 16);
                    acc = mfma_f32(av, bv, acc);
                }
            }
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave != finisher) return;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) acc = v == 0 ? part[0][lane] : acc + part[v][lane];
    // lane (token n, g): gate of columns 4 g ... where g < 2, up of columns 4 (g - 2) ... else
    floatx4 up;
#pragma unroll
    for (int i = 0; i < 4; ++i) up[i] = __shfl_xor(acc[i], 32);
    if (g < 2 && n < rows) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float h = acc[i] * sigmoid_f32(acc[i]) * up[i];
            acc[i] = tile * 8 + 4 * g + i < I ? h : 0.0f;
        }
        *(floatx4 *)(p.h + (int64_t)(first + n) * p.ldh + tile * 8 + 4 * g) = acc;
    }
}

// ---- down and sum ---------------------------------------------------------------------------------------------------------------
// An item is four columns of the output, all chosen experts: a wave takes every eighth of them.  A tile's 16 rows are the four
// columns' weights times four parts of the reduction, its 16 columns four tokens times the same four parts; where the parts agree
// the result counts, and the four are added.  (With 16 columns an item there would be too few to fill the chip; three quarters of
// the matrix unit's work are for nothing, but it has a thirtieth of its time to do.)
typedef float Sums[kWaves][kTokens][4];

template <typename T, bool FP8, bool WHOLE>
__device__ __forceinline__ void down_item(const Layer &p, const Routing &r, int tile, float (*sums)[kTokens][4]) {
    typedef Weights<T, FP8> W;
    typedef typename W::Element Element;
    constexpr int kRun = W::kRun, kStep = W::kStep;
    constexpr int U = FP8 ? 4 : 6;
    constexpr int kUnit = FP8 ? kFp8Block : kRun;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int H = p.c.H, I = p.c.I;
    const int length = ((I + 3) / 4 + kUnit - 1) / kUnit * kUnit;  // of a part
    const int steps = (length + kStep - 1) / kStep;
    const int row = tile * 4 + (n >> 2), from = (n & 3) * length;
    const int left = I - from < length ? (I - from < 0 ? 0 : I - from) : length;  // of the lane's part, both as row and as column
    const int nb = fp8_blocks(H), kb = fp8_blocks(I);
    sums[wave][lane >> 2][lane & 3] = 0.0f;  // (a wave's own: its LDS operations keep their order)
    const int experts = r.experts;
    for (int at = wave; at < experts; at += kWaves) {
        const int e = __builtin_amdgcn_readfirstlane(r.expert[at]);
        const int first = __builtin_amdgcn_readfirstlane(r.first[at]);
        const int rows = __builtin_amdgcn_readfirstlane(r.first[at + 1]) - first;
        const Element *const w = (const Element *)p.c.w_down + ((int64_t)e * H + (row < H ? row : H - 1)) * I + from;
        const float *const scale = FP8 ? p.c.s_down + ((int64_t)e * nb + tile * 4 / kFp8Block) * kb : nullptr;
        floatx4 acc[4];
        float total[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q] = floatx4{0.0f, 0.0f, 0.0f, 0.0f}, total[q] = 0.0f;
        for (int s0 = 0; s0 < steps; s0 += U) {
            Run a[U];
#pragma unroll
            for (int u = 0; u < U; ++u) load_run<WHOLE, 16>(w, s0 + u < steps ? (s0 + u) * kStep + g * kRun : left, left, &a[u]);
            float block_scale[U];
            if (FP8) {
#pragma unroll
                for (int u = 0; u < U / 2; ++u) {
                    const int b = from / kFp8Block + s0 / 2 + u;
                    block_scale[u] = (s0 + 2 * u) * kStep < left ? scale[b] : 0.0f;
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q * 4 >= rows) break;
                const int mine = q * 4 + (n >> 2);
                const float *const h = p.h + (int64_t)(first + (mine < rows ? mine : rows - 1)) * p.ldh + from;
#pragma unroll
                for (int u0 = 0; u0 < U; u0 += 2) {
                    if (s0 + u0 >= steps) break;
                    struct alignas(16) {
                        float v[kRun];
                    } b[2];
#pragma unroll
                    for (int o = 0; o < 2; ++o) {
                        // (rows of h are whole runs long, zeros behind column I)
                        const int k = (s0 + u0 + o) * kStep + g * kRun;
                        if (s0 + u0 + o < steps && k < left) __builtin_memcpy(b[o].v, h + k, sizeof(b[o].v));
                        else __builtin_memset(b[o].v, 0, sizeof(b[o].v));
                    }
                    if constexpr (FP8) {
                        // the block's 128 values: 32 here, the others in the other quarters of the wave
                        uint32_t top = 0u;
#pragma unroll
                        for (int o = 0; o < 2; ++o)
#pragma unroll
                            for (int i = 0; i < 16; ++i) top = fp8_wider(top, b[o].v[i]);
                        top = fp8_over_quarters(top);
                        if (__builtin_expect(__any(fp8_unusual(top)), 0)) {
                            top = 0u;
#pragma unroll
                            for (int o = 0; o < 2; ++o)
#pragma unroll
                                for (int i = 0; i < 16; ++i) top = fp8_wider(top, fp8_finite_abs(b[o].v[i])), b[o].v[i] = fp8_finite(b[o].v[i]);
                            top = fp8_over_quarters(top);
                        }
                        const int byte = fp8_scale_byte(top);
                        const float inverse = fp8_inverse_of(byte), back = fp8_scale_of(byte);
                        floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            union {
                                Run r;
                                intx2 t[2];
                            } f = {a[u0 + o]};
#pragma unroll
                            for (int z = 0; z < 2; ++z) {
                                const float *const c = b[o].v + 8 * z;
                                const intx2 packed = {(int)fp8_pack4(c[0], c[1], c[2], c[3], inverse), (int)fp8_pack4(c[4], c[5], c[6], c[7], inverse)};
                                sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_widen(f.t[z], 1.0f), fp8_widen(packed, back), sum, 0, 0, 0);
                            }
                        }
                        const float lo = n & 1 ? sum[1] : sum[0], hi = n & 1 ? sum[3] : sum[2];
                        total[q] = __builtin_fmaf(block_scale[u0 / 2], n & 2 ? hi : lo, total[q]);
                    } else {
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            if constexpr (std::is_same<T, bf16_t>::value) {
                                // the fp32 value as the sum of two bf16 ones: 2^-17 of it is lost at most, the output's own rounding is 2^-9
                                bf16x8 av, high, low;
                                __builtin_memcpy(&av, &a[u0 + o], 16);
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    high[i] = (bf16_t)b[o].v[i];
                                    low[i] = (bf16_t)(b[o].v[i] - (float)high[i]);
                                }
                                acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, low, acc[q], 0, 0, 0);
                                acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, high, acc[q], 0, 0, 0);
                            } else {
                                // (fp16: widened, since the unit's values need not fit the type)
                                T narrow[kRun];
                                __builtin_memcpy(narrow, &a[u0 + o], 16);
#pragma unroll
                                for (int z = 0; z < kRun; z += 4) {
                                    const float av[4] = {to_f32(narrow[z]), to_f32(narrow[z + 1]), to_f32(narrow[z + 2]), to_f32(narrow[z + 3])};
                                    const float bv[4] = {b[o].v[z], b[o].v[z + 1], b[o].v[z + 2], b[o].v[z + 3]};
                                    acc[q] = mfma_f32(av, bv, acc[q]);
                                }
                            }
                        }
                    }
                }
            }
        }
        // lane (n, g): column g's sum of part i for the token and part of n, in acc[.][i]
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (q * 4 >= rows) break;
            if (!FP8) {
                const float lo = n & 1 ? acc[q][1] : acc[q][0], hi = n & 1 ? acc[q][3] : acc[q][2];
                total[q] = n & 2 ? hi : lo;
            }
            float v = total[q];
            v += __shfl_xor(v, 1);
            v += __shfl_xor(v, 2);
            const int mine = q * 4 + (n >> 2);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if ((n & 3) == 0 && mine < rows) sums[wave][r.token[first + mine]][g] += r.weight[first + mine] * v;
        }
    }
    __syncthreads();
    const int t = threadIdx.x >> 2, c = tile * 4 + (threadIdx.x & 3);
    if (t < (int)p.c.T && c < H) {
        float v = 0.0f;
#pragma unroll
        for (int u = 0; u < kWaves; ++u) v += sums[u][t][threadIdx.x & 3];
        if (p.stream != nullptr) v += to_f32(((const T *)p.stream)[(int64_t)t * H + c]);
        if (r.lost >> t & 1u) v = __builtin_nanf("");
        ((T *)p.out)[(int64_t)t * H + c] = from_f32<T>(v);
    }
}

template <typename T, bool FP8, bool WHOLE>
__global__ __launch_bounds__(kThreads, 4) void layer_gate_up_kernel(Layer p) {
    __shared__ Routing r;
    __shared__ Parts part;
    find_routing<T>(p, r);
    const int tiles = (int)(p.ldh / 8), items = r.experts * tiles;
    int turn = 0;
    for (int i = blockIdx.x; i < items; i += gridDim.x, ++turn)
        gate_up_item<T, FP8, WHOLE>(p, r, i / tiles, i % tiles, part[turn & 1], turn & (kWaves - 1));
}

template <typename T, bool FP8, bool WHOLE>
__global__ __launch_bounds__(kThreads, 4) void layer_down_kernel(Layer p) {
    __shared__ Routing r;
    __shared__ Sums sums[2];
    find_routing<T>(p, r);
    const int items = ceil_div(p.c.H, 4);
    int turn = 0;
    for (int i = blockIdx.x; i < items; i += gridDim.x, ++turn) down_item<T, FP8, WHOLE>(p, r, i, sums[turn & 1]);
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct Room {
    size_t stream, rows, h;  // bytes
    int64_t ld, ldh;
    explicit Room(const mfl_moe_layer &c) {
        const bool fp8 = c.s_gate != nullptr, norm = c.norm_weight != nullptr;
        ld = fp8 ? fp8_ld(c.H) : c.H;
        ldh = (c.I + 15) / 16 * 16;
        stream = c.residual != nullptr ? up256((size_t)c.T * c.H * dtype_size(c.dtype)) : 0;
        rows = fp8 ? up256((size_t)c.T * ld * 2) : norm ? up256((size_t)c.T * ld * dtype_size(c.dtype)) : 0;
        h = up256((size_t)c.T * c.k * ldh * 4);
    }
};

template <typename T, bool FP8, bool WHOLE>
int launch(const Layer &p, hipStream_t stream) {
    const int tokens = (int)p.c.T;
    const unsigned routers = (unsigned)ceil_div(p.c.E, kRouterExperts);
    const bool whole8 = p.c.H % 8 == 0;
#define MFL_LAYER_ROUTER(N)                                                                             \
    if (whole8) layer_router_kernel<T, N, FP8, true><<<routers, 256, 0, stream>>>(p);                    \
    else layer_router_kernel<T, N, FP8, false><<<routers, 256, 0, stream>>>(p);
    if (tokens == 1) { MFL_LAYER_ROUTER(1) }
    else if (tokens <= 4) { MFL_LAYER_ROUTER(4) }
    else if (tokens <= 8) { MFL_LAYER_ROUTER(8) }
    else { MFL_LAYER_ROUTER(16) }
#undef MFL_LAYER_ROUTER
    const int most = 2 * device_info().cu_count;
    const int hits = p.c.T * p.c.k < p.c.E ? (int)p.c.T * p.c.k : p.c.E;
    const int64_t front = hits * (p.ldh / 8), back = ceil_div(p.c.H, 4);
    layer_gate_up_kernel<T, FP8, WHOLE><<<(unsigned)(front < most ? front : most), kThreads, 0, stream>>>(p);
    layer_down_kernel<T, FP8, WHOLE><<<(unsigned)(back < most ? back : most), kThreads, 0, stream>>>(p);
    return launch_status();
}

template <typename T>
int launch_type(const Layer &p, hipStream_t stream) {
    constexpr int run = 16 / (int)sizeof(T);
    if (p.c.s_gate != nullptr) {
        if (p.c.H % 16 == 0 && p.c.I % 16 == 0) return launch<T, true, true>(p, stream);
        return launch<T, true, false>(p, stream);
    }
    if (p.c.H % run == 0 && p.c.I % run == 0) return launch<T, false, true>(p, stream);
    return launch<T, false, false>(p, stream);
}

}  // namespace

size_t moe_layer_workspace(const mfl_moe_layer &c) {
    const Room room(c);
    return room.stream + room.rows + room.h;
}

int moe_layer_fwd(const mfl_moe_layer &c, void *out, void *logits, void *workspace, hipStream_t stream) {
    const Room room(c);
    uint8_t *const ws = (uint8_t *)workspace;
    Layer p = {};
    p.c = c, p.out = out, p.logits = logits;
    p.ld = room.ld, p.ldh = room.ldh;
    p.stream_out = room.stream ? ws : nullptr;
    p.stream = c.norm_weight == nullptr ? nullptr : room.stream ? p.stream_out : c.x;
    p.rows_out = room.rows ? ws + room.stream : nullptr;
    p.rows = room.rows ? p.rows_out : c.x;
    p.h = (float *)(ws + room.stream + room.rows);
    int rc = MFL_OK;
    MFL_DISPATCH_FLOAT(c.dtype, T, { rc = launch_type<T>(p, stream); });
    return rc;
}

}  // namespace mfl
