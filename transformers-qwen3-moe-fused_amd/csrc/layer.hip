// The whole sparse expert layer for a few tokens: router, softmax and top-k, gated experts, weighted sum; with the residual's
// addition and the norm in front and the stream's addition behind where asked for.
//
// Two launches: the logits (and the stream and the normed rows), then everything behind them, the routing found again by every
// workgroup.  An expert's weights are read once, straight from memory into the matrix unit's operands, for all tokens that chose it.
// With 128 experts of 2048 x 768, 8 a token, in bf16: 16 tokens 140 us, of which the router is 6: the weights of the 82 experts that
// are hit on average (780 MB) at 5.8 TB/s, which is what the memory gives.  One token 25 us, where its 8 experts' 75 MB take 14: a chain of
// round trips, the router 3.6, the routing 3.4, gate and up 9, the meeting of the workgroups 3.5, down 4.5 (8-bit weights, with addition and
// norm: 25.5, and 13 tokens 65).  In three launches, with the gated unit and the down projection as kernels of their own, one token took 33 us
// and 16 tokens 226.
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
    float *h;  // (T k, ldh): the gated unit's results, a row per (expert, token) in this order; bf16: eight columns at a time as eight
               // high and eight low halves (Halves)
    int64_t ldh;
    uint32_t *widest;  // 8-bit layers: (T k, blocks of 128) largest finite magnitudes of h, as bits
    uint32_t *units;   // a word per unit of the second kernel's work
    uint32_t *zeros;           // what the first kernel clears of all these, and how many words
    int zero_words;
};

// ---- first kernel: stream, norm, logits -----------------------------------------------------------------------------------
// A workgroup has a token and EXPERTS experts.  It norms the token itself (the row is read once more per workgroup, from the
// caches), so that nothing has to wait for another workgroup; the first one of a token writes its rows.  ONE: a row is one run of
// eight elements a thread, and stays in registers.
constexpr int kRouterExperts = 2;

template <typename T, int EXPERTS, bool FP8, bool WHOLE, bool ONE>
__global__ __launch_bounds__(256) void layer_router_kernel(Layer p) {
    __shared__ double squares[4];
    __shared__ double part[4][EXPERTS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int H = p.c.H, E = p.c.E, t = blockIdx.y, e0 = blockIdx.x * EXPERTS;
    const bool norm = p.c.norm_weight != nullptr, writes = blockIdx.x == 0;
    const T *const x = (const T *)p.c.x + (int64_t)t * H;
    const T *const residual = p.c.residual != nullptr ? (const T *)p.c.residual + (int64_t)t * H : nullptr;
    for (int i = (blockIdx.y * gridDim.x + blockIdx.x) * 256 + tid; i < p.zero_words; i += gridDim.x * gridDim.y * 256) p.zeros[i] = 0u;

    auto stream_of = [&](int k) {
        Eight<T, WHOLE> v;
        v.load(x, k, H);
        if (residual != nullptr) {
            Eight<T, WHOLE> o;
            o.load(residual, k, H);
            add_rounded(v, o);
        }
        return v;
    };
    Eight<T, WHOLE> w, r[EXPERTS], s;
    auto load_weights = [&](int k) {
        if (norm) w.load((const T *)p.c.norm_weight, k, H);
#pragma unroll
        for (int j = 0; j < EXPERTS; ++j) r[j].load((const T *)p.c.router + (int64_t)(e0 + j < E ? e0 + j : E - 1) * H, k, H);
    };
    if (ONE) s = stream_of(tid * 8), load_weights(tid * 8);
    double length = 0.0;
    if (norm) {
        double sum = 0.0;
        if (ONE) sum = sum_of_squares(s, sum);
        else
            for (int k = tid * 8; k < H; k += 2048) sum = sum_of_squares(stream_of(k), sum);
        sum = wave_sum(sum);
        if (lane == 0) squares[wave] = sum;
        __syncthreads();
        length = inverse_root((squares[0] + squares[1] + squares[2] + squares[3]) / (double)H + (double)p.c.eps);
    }
    double acc[EXPERTS];
#pragma unroll
    for (int j = 0; j < EXPERTS; ++j) acc[j] = 0.0;
    const int padded = FP8 ? (int)fp8_ld(H) : H;  // (8-bit: whole blocks of 128, the same for the 16 lanes of a block)
    for (int k = tid * 8; k < padded; k += 2048) {
        if (!ONE) s = stream_of(k), load_weights(k);
        Eight<T, WHOLE> v = s;
        if (norm) {
            if (writes && p.stream_out != nullptr) s.store((T *)p.stream_out + (int64_t)t * H, k, H);
#pragma unroll
            for (int i = 0; i < 8; ++i) v.v[i] = normed(s.v[i], length, w.v[i]);
        }
        if (writes && p.rows_out != nullptr) {
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
        for (int i = 0; i < 8; ++i) {
            const double a = (double)to_f32(v.v[i]);
#pragma unroll
            for (int j = 0; j < EXPERTS; ++j)
                // (behind column H the stream, the weight and the router are zeros)
                acc[j] = __builtin_fma(a, (double)to_f32(r[j].v[i]), acc[j]);
        }
    }
    // every step halves the sums that a lane holds: EXPERTS - 1 exchanges and one a step for the rest
    int step = 32, mine = 0;
#pragma unroll
    for (int half = EXPERTS / 2; half; half /= 2, step /= 2) {
        const bool upper = lane & step;
        if (upper) mine += half;
#pragma unroll
        for (int j = 0; j < half; ++j) {
            const double keep = upper ? acc[j + half] : acc[j], give = upper ? acc[j] : acc[j + half];
            acc[j] = keep + __shfl_xor(give, step);
        }
    }
    const int last = step;
    for (; step; step /= 2) acc[0] += __shfl_xor(acc[0], step);
    if ((lane & (2 * last - 1)) == 0) part[wave][mine] = acc[0];
    __syncthreads();
    if (tid < EXPERTS && e0 + tid < E)
        ((T *)p.logits)[(int64_t)t * E + e0 + tid] = from_f32<T>((float)(part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]));
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

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ float dpp_sum_step(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROW_MASK, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float x) {
    x = dpp_sum_step<0x111, 0xf>(x);
    x = dpp_sum_step<0x112, 0xf>(x);
    x = dpp_sum_step<0x114, 0xf>(x);
    x = dpp_sum_step<0x118, 0xf>(x);
    x = dpp_sum_step<0x142, 0xa>(x);
    x = dpp_sum_step<0x143, 0xc>(x);
    return __int_as_float(wave_last(__float_as_int(x)));
}

// TOKENS tokens t, t + 8, ... by one wave, side by side (each is a chain of dependent steps); PER_LANE: experts lane, lane + 64, ...
// `ready` is called when the logits are on their way.
template <typename T, int PER_LANE, int TOKENS, typename F>
__device__ __forceinline__ void choose(const Layer &p, int t, Routing &r, int lane, F &&ready) {
    constexpr int kNone = -0x7fffffff - 1;
    const int E = p.c.E, k = p.c.k;
    T raw[TOKENS][PER_LANE];
#pragma unroll
    for (int o = 0; o < TOKENS; ++o) {
        const int at = t + o * kWaves < (int)p.c.T ? t + o * kWaves : (int)p.c.T - 1;  // (a wave without a token looks at the last one)
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) raw[o][i] = ((const T *)p.logits)[(int64_t)at * E + (lane + 64 * i < E ? lane + 64 * i : E - 1)];
    }
    ready();
    float share[TOKENS][PER_LANE], sum[TOKENS], chosen[TOKENS], mine[TOKENS];
    int key[TOKENS][PER_LANE], top[TOKENS], mine_e[TOKENS];
    bool lost[TOKENS];
#pragma unroll
    for (int o = 0; o < TOKENS; ++o) {
        top[o] = kNone;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            const bool in = lane + 64 * i < E;
            share[o][i] = in ? to_f32(raw[o][i]) + 0.0f : -INFINITY;
            nan |= share[o][i] != share[o][i];
            const int bits = __float_as_int(share[o][i]);
            key[o][i] = in ? bits ^ ((bits >> 31) & 0x7fffffff) : kNone;  // the order of the values as whole numbers (-0 as 0)
            top[o] = top[o] > key[o][i] ? top[o] : key[o][i];
        }
        top[o] = wave_max(top[o]);
        const float largest = __int_as_float(top[o] ^ ((top[o] >> 31) & 0x7fffffff));
        lost[o] = __any(nan) || __builtin_isinf(largest);
        sum[o] = chosen[o] = mine[o] = 0.0f, mine_e[o] = 0;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) share[o][i] = expf(share[o][i] - largest), sum[o] += share[o][i];  // (0 past the last expert)
        sum[o] = wave_sum(sum[o]);
    }
    for (int j = 0; j < k; ++j) {
#pragma unroll
        for (int o = 0; o < TOKENS; ++o) {
            int best = kNone, at = 0;
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i)
                if (key[o][i] > best) best = key[o][i], at = i, s = share[o][i];  // (ascending ids: the lower of equals)
            const int m = j == 0 ? top[o] : wave_max(best);
            // of the lanes with that value the lowest expert id: the least i, then the least lane
            const uint64_t owners = __ballot(best == m);
            int e;
            if (__popcll(owners) == 1) {
                const int owner = __ffsll((unsigned long long)owners) - 1;
                e = __builtin_amdgcn_readlane(at, owner) * 64 + owner;
            } else {
                e = -wave_max(best == m ? -(at * 64 + lane) : kNone);
            }
            const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s), e & 63));
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i)
                if (e == lane + 64 * i) key[o][i] = kNone;
            if (lane == j) mine[o] = w, mine_e[o] = e;
            chosen[o] += w;
        }
    }
#pragma unroll
    for (int o = 0; o < TOKENS; ++o) {
        const int at = t + o * kWaves;
        if (at >= (int)p.c.T || lane >= k) continue;
        r.own_expert[at][lane] = lost[o] ? -1 : (int16_t)mine_e[o];
        if (lost[o]) {
            if (lane == 0) atomicOr(&r.lost, 1u << at);
            continue;
        }
        r.own_weight[at][lane] = mine[o] / (p.c.renorm ? chosen[o] : sum[o]);
        atomicOr(&r.mask[mine_e[o]], 1u << at);
    }
}

template <typename T>
__device__ __forceinline__ void find_routing(const Layer &p, Routing &r) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int E = p.c.E, k = p.c.k, tokens = (int)p.c.T;
    auto clear = [&] {
        for (int e = tid; e < E; e += kThreads) r.mask[e] = 0u;
        if (tid == 0) r.lost = 0u;
        __syncthreads();
    };
    if (E > 128) {
        choose<T, 16, 1>(p, wave, r, lane, clear);
        if (tokens > kWaves) choose<T, 16, 1>(p, wave + kWaves, r, lane, [] {});
    } else if (tokens > kWaves) {
        choose<T, 2, 2>(p, wave, r, lane, clear);
    } else {
        choose<T, 2, 1>(p, wave, r, lane, clear);
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

struct alignas(16) Run {
    uint64_t v[2];
};

// How the sizes fit the loads.  kExact: every load of every wave lies in its row (rows of whole chunks for all waves): nothing
// is asked (16 tokens of the sizes above 150 -> 142 us, one 27.8 -> 25.9); kWhole: rows are whole loads long; kRagged: any.
enum Fit { kRagged, kWhole, kExact };

// 16 bytes of a row from element k on, zeros from element K on.  In two steps: `fetch` loads, always and without a branch, so that the
// compiler can count what is on its way behind what it waits for; `settle`, called where the values are needed, puts zeros in the place of
// what lies behind the row's end (ragged: fetch loads the row's last 16 bytes where the end cuts the run, and settle moves them down).
template <int FIT, typename E>
__device__ __forceinline__ Run fetch(const E *row, int k, int K) {
    constexpr int count = 16 / (int)sizeof(E);
    Run run;
    if (FIT == kExact) {
        __builtin_memcpy(&run, row + k, 16);
    } else if (FIT == kWhole || K >= count) {
        __builtin_memcpy(&run, row + (k + count <= K ? k : K - count), 16);
    } else {
        run.v[0] = run.v[1] = 0u;
#pragma unroll 1
        for (int i = 0; i < count && k + i < K; ++i) {
            uint64_t bits = 0u;
            __builtin_memcpy(&bits, row + k + i, sizeof(E));
            const int at = i * 8 * (int)sizeof(E);
            if (at < 64) run.v[0] |= bits << at;
            else run.v[1] |= bits << (at - 64);
        }
    }
    return run;
}
template <int FIT, typename E>
__device__ __forceinline__ Run settle(Run run, int k, int K) {
    constexpr int count = 16 / (int)sizeof(E);
    if (FIT == kExact) return run;
    if (FIT == kWhole) {
        run.v[0] = k < K ? run.v[0] : 0u;
        run.v[1] = k < K ? run.v[1] : 0u;
        return run;
    }
    if (K < count) return run;
    const int moved = k + count <= K ? 0 : (k + count - K) * 8 * (int)sizeof(E);
    const uint64_t lo = run.v[0], hi = run.v[1];
    run.v[0] = moved == 0 ? lo : moved < 64 ? lo >> moved | hi << (64 - moved) : moved < 128 ? hi >> (moved - 64) : 0u;
    run.v[1] = moved < 64 ? hi >> moved : 0u;
    return run;
}

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// bf16 layers keep a value h of the gated unit as two bf16 ones, h as rounded and what that leaves, as rounded: 2^-17 of it is lost at
// most, where the output's own rounding is 2^-9.  The first is no further from zero than the type's largest value (past that h rounds
// to an infinity, and what is left would be the other one): the second has what lies behind, an infinity or no number too.  fp16 weights are widened for h in 32 bits (it need not fit the type), and in 8-bit
// layers h is quantised where it is read, by which time its blocks' largest magnitudes are known.
template <typename T, bool FP8>
constexpr bool kHalves = std::is_same<T, bf16_t>::value && !FP8;
constexpr float kLargest = 3.3895313892515355e38f;  // of bf16: 2^128 (1 - 2^-8)

// What workgroups hand to one another within a kernel goes past the L2s of the XCDs, both ways: stores and loads of the device's
// scope.  (Ordinary ones with a fence before the word that says so write back and invalidate a whole L2 for every wave: 120 us.)
__device__ __forceinline__ void publish(void *to, uint64_t v) {
    __hip_atomic_store((uint64_t *)to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t peek(const uint32_t *word) {
    return __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr int kDeviceScope = 16;  // a buffer load's sc1 bit

// ---- gate and up --------------------------------------------------------------------------------------------------------------
// An item is an expert's eight columns of either matrix, side by side as the 16 rows of one tile, times the expert's tokens as its
// 16 columns; the eight waves share the reduction and meet in LDS.  Weights straight from memory into the matrix unit's registers.
// A column is a token, whether it chose the expert or not: what a wave needs of the tokens is the same for every item, and stays in
// registers where its share of the reduction is one chunk.  The next item's weights are asked for before the waves meet.
typedef floatx4 Parts[2][2][kWaves][64];

// NARROW: rows of which a wave's share is half a chunk or less (1024 elements, 512 in 32 bits) are taken in chunks of half as many
// steps, with twice as many items ahead: what is loaded behind a share is loaded for nothing, and where rows have to be moved down
// its registers are short (5 tokens, 60 experts of 1001 x 333 in fp16 44 -> 34 us, of 1008 x 336 25.9 -> 24.3).
template <typename T, bool FP8, int FIT, bool NARROW>
struct GateUp {
    typedef Weights<T, FP8> W;
    typedef typename W::Element Element;
    typedef typename std::conditional<FP8, bf16_t, T>::type X;
    static constexpr int kRun = W::kRun, kStep = W::kStep, kPieces = kRun * (int)sizeof(X) / 16;
    static constexpr int U = (FP8 ? 4 : 8) / (NARROW ? 2 : 1);  // steps of a chunk: their loads are in flight together
    static constexpr int D = (FP8 ? 4 : 2) * (NARROW ? 2 : 1);  // items whose first chunks are
    static constexpr int kGroup = FP8 ? 2 : 1;
    static constexpr int kUnit = FP8 ? 2 : 1;  // (whole blocks of 128 a wave where weights have scales)
    const Layer &p;
    const Routing &r;
    const int lane, n, g, wave, tiles, begin, end, chunks;
    struct Weight {
        Run a[U];
        float scale[U / 2];
    };
    Weight w[D];
    Run b[U][kPieces];

    static __device__ __forceinline__ int share(int H) {
        const int steps = (H + kStep - 1) / kStep;
        return ((steps + kWaves - 1) / kWaves + kUnit - 1) / kUnit * kUnit;
    }
    __device__ __forceinline__ GateUp(const Layer &p, const Routing &r)
        : p(p), r(r), lane(threadIdx.x & 63), n(lane & 15), g(lane >> 4), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
          tiles((int)(p.ldh / 8)), begin(wave * share(p.c.H)),
          end(begin + share(p.c.H) < (p.c.H + kStep - 1) / kStep ? begin + share(p.c.H) : (p.c.H + kStep - 1) / kStep),
          chunks((share(p.c.H) + U - 1) / U) {
        if (chunks == 1) load_rows(begin);
    }

    // the first element of the lane's run of a step; H behind the wave's share
    __device__ __forceinline__ int element(int step) const { return FIT == kExact || step < end ? step * kStep + g * kRun : p.c.H; }
    __device__ __forceinline__ void load_weights(Weight &to, int item, int s0) const {
        const int H = p.c.H, I = p.c.I, tile = item % tiles, col = tile * 8 + (n & 7);
        const int e = __builtin_amdgcn_readfirstlane(r.expert[item / tiles]);
        const Element *const w = (const Element *)(n < 8 ? p.c.w_gate : p.c.w_up) + ((int64_t)e * I + (col < I ? col : I - 1)) * H;
#pragma unroll
        for (int u = 0; u < U; ++u) to.a[u] = fetch<FIT>(w, element(s0 + u), H);
        if (FP8) {
            const int64_t block = ((int64_t)e * fp8_blocks(I) + tile * 8 / kFp8Block) * fp8_blocks(H);
            // (of the results that the lane holds, not of the rows that it loads)
            const float *const scales = (g < 2 ? p.c.s_gate : p.c.s_up) + block;
#pragma unroll
            for (int u = 0; u < U / 2; ++u) to.scale[u] = s0 + 2 * u < end ? scales[(s0 + 2 * u) / 2] : 0.0f;
        }
    }
    __device__ __forceinline__ void load_rows(int s0) {
        const X *const x = (const X *)p.rows + (n < (int)p.c.T ? n : (int)p.c.T - 1) * p.ld;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // (8-bit layers: rows of whole blocks, zeros behind column H)
            if constexpr (FP8) __builtin_memcpy(b[u], s0 + u < end ? x + (s0 + u) * kStep + g * kRun : x, sizeof(b[u]));
            else b[u][0] = settle<FIT, X>(fetch<FIT>(x, element(s0 + u), p.c.H), element(s0 + u), p.c.H);
        }
    }
    __device__ __forceinline__ void multiply(const Weight &weight, int s0, floatx4 &acc) const {
        Run a[U];
#pragma unroll
        for (int u = 0; u < U; ++u) a[u] = settle<FIT, Element>(weight.a[u], element(s0 + u), p.c.H);
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
                    for (int o = 0; o < 2; ++o)
                        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_widen(f.t[o], 1.0f), __builtin_bit_cast(bf16x8, b[2 * u + q][o]), sum, 0, 0, 0);
                }
                // (behind the wave's share the weights are zeros, and so is the scale)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(weight.scale[u], sum[i], acc[i]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if constexpr (std::is_same<T, bf16_t>::value) {
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[u]), __builtin_bit_cast(bf16x8, b[u][0]), acc, 0, 0, 0);
                } else if constexpr (std::is_same<T, f16_t>::value) {
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a[u]), __builtin_bit_cast(f16x8, b[u][0]), acc, 0, 0, 0);
                } else {
                    const floatx4 av = __builtin_bit_cast(floatx4, a[u]), bv = __builtin_bit_cast(floatx4, b[u][0]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(av[i], bv[i], acc, 0, 0, 0);
                }
            }
        }
    }

    // One meeting of the waves: items item, item + by, ... (kGroup of them, as far as they are below to) from w[d], w[d + 1], ..., which are
    // loaded again, with the items D on: ALL, or as far as there are any.
    template <bool ALL>
    __device__ __forceinline__ void meet(int d, int item, int to, int by, Parts &parts, int turn) {
        floatx4 acc[kGroup];
#pragma unroll
        for (int o = 0; o < kGroup; ++o) acc[o] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = 0; c < chunks; ++c) {
            if (c != 0) {
#pragma unroll
                for (int o = 0; o < kGroup; ++o)
                    if (ALL || item + o * by < to) load_weights(w[d + o], item + o * by, begin + c * U);
            }
            if (chunks != 1) load_rows(begin + c * U);
#pragma unroll
            for (int o = 0; o < kGroup; ++o)
                if (ALL || item + o * by < to) multiply(w[d + o], begin + c * U, acc[o]);
        }
        floatx4(*const part)[kWaves][64] = parts[turn & 1];
#pragma unroll
        for (int o = 0; o < kGroup; ++o) {
            if (ALL || item + (D + o) * by < to) load_weights(w[d + o], item + (D + o) * by, begin);
            if (ALL || item + o * by < to) part[o][wave][lane] = acc[o];
        }
        __syncthreads();
        // as many waves finish an item each, others every time
        const int mine = (wave - kGroup * turn) & (kWaves - 1);
        if (mine >= kGroup || (!ALL && item + mine * by >= to)) return;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) acc[0] = v == 0 ? part[mine][0][lane] : acc[0] + part[mine][v][lane];
        finish(item + mine * by, acc[0]);
    }
    // Items from, from + by, ... below to; `turn` counts a workgroup's meetings.
    __device__ __forceinline__ void run(int from, int to, int by, Parts &parts, int &turn) {
        int i = from;
        // (A loop in which nothing is loaded or not: else the compiler waits for all that might be the last.  Four items of 4 KB a wave
        // need it, 13 tokens in 8 bits 84 -> 70 us; two of 8 KB fill the memory without, and lose what its registers cost.)
        if (FP8 && i + (2 * D - 1) * by < to) {
#pragma unroll
            for (int d = 0; d < D; ++d) load_weights(w[d], i + d * by, begin);
            for (; i + (2 * D - 1) * by < to; i += D * by) {
#pragma unroll
                for (int d = 0; d < D; d += kGroup, ++turn) meet<true>(d, i + d * by, to, by, parts, turn);
            }
        } else {
#pragma unroll
            for (int d = 0; d < D; ++d)
                if (i + d * by < to) load_weights(w[d], i + d * by, begin);
        }
        for (; i < to; i += D * by) {
#pragma unroll
            for (int d = 0; d < D; d += kGroup, ++turn) {
                if (i + d * by >= to) break;
                meet<false>(d, i + d * by, to, by, parts, turn);
            }
        }
    }
    // lane (token n, g): gate of columns 4 g ... where g < 2, up of columns 4 (g - 2) ... else
    __device__ __forceinline__ void finish(int item, floatx4 acc) const {
        const int tile = item % tiles, e = r.expert[item / tiles];
        const uint32_t mask = r.mask[e];
        const bool chosen = mask >> n & 1u;
        const int pair = (int)(mask >> 16) + __popc(mask & ((1u << n) - 1u));
        floatx4 up;
#pragma unroll
        for (int i = 0; i < 4; ++i) up[i] = __shfl_xor(acc[i], 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float h = acc[i] * sigmoid_f32(acc[i]) * up[i];
            acc[i] = tile * 8 + 4 * g + i < p.c.I ? h : 0.0f;
        }
        if (g < 2 && chosen) {
            float *const to = p.h + (int64_t)pair * p.ldh + tile * 8;
            if constexpr (kHalves<T, FP8>) {
                bf16x4 high, low;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    high[i] = (bf16_t)__builtin_amdgcn_fmed3f(acc[i], -kLargest, kLargest);
                    low[i] = (bf16_t)(acc[i] - (float)high[i]);
                }
                publish((bf16_t *)to + 4 * g, __builtin_bit_cast(uint64_t, high));
                publish((bf16_t *)to + 8 + 4 * g, __builtin_bit_cast(uint64_t, low));
            } else {
                publish(to + 4 * g, __builtin_bit_cast(uint64_t, floatx2{acc[0], acc[1]}));
                publish(to + 4 * g + 2, __builtin_bit_cast(uint64_t, floatx2{acc[2], acc[3]}));
            }
        }
        if constexpr (FP8) {
            // the blocks' largest magnitudes: their order is that of the bits, and whoever comes last, the result is the same
            uint32_t top = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fp8_wider(top, fp8_finite_abs(acc[i]));
            const uint32_t other = (uint32_t)__shfl_xor((int)top, 16);
            if (g == 0 && chosen)
                __hip_atomic_fetch_max(p.widest + (int64_t)pair * fp8_blocks(p.c.I) + tile * 8 / kFp8Block, top > other ? top : other,
                                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
};

// ---- down and sum ---------------------------------------------------------------------------------------------------------------
// An item is eight columns of the output, all chosen experts: a wave takes every eighth of them.  A tile's 16 rows are the eight
// columns' weights times two parts of the reduction, its 16 columns eight tokens times the same two parts; where the parts agree the
// result counts, and the two are added.  (With 16 columns an item there would be too few to fill the chip; half of the matrix unit's
// work is for nothing, but it has a thirtieth of its time to do.)
constexpr int kParts = 2, kColumns = 16 / kParts;
typedef float Sums[kWaves][kTokens][kColumns];
constexpr int kStageBytes = 12544;  // of LDS for a wave's rows of h

// A chunk of an expert's weights for an item: U steps of the lane's row and part.
// (Six where more would not fit the registers: rows that have to be moved down, and fp16, which is widened: 61 -> 44 us at 5 tokens of
// 1001 x 333.)
template <typename T, bool FP8, int FIT>
struct Chunk {
    static constexpr int U = FP8 || FIT == kRagged || std::is_same<T, f16_t>::value ? 6 : 12;
    Run a[U];
    float scale[U / 2];
};

template <typename T, bool FP8, int FIT>
struct Down {
    typedef Weights<T, FP8> W;
    typedef typename W::Element Element;
    static constexpr int kRun = W::kRun, kStep = W::kStep, U = Chunk<T, FP8, FIT>::U;
    static constexpr int kUnit = FP8 ? kFp8Block : kRun;
    const Layer &p;
    const Routing &r;
    const int lane, n, g, wave, length, steps, from, left, nb, kb;
    const uint32_t h_bytes;
    const __amdgpu_buffer_rsrc_t h;

    __device__ __forceinline__ Down(const Layer &p, const Routing &r)
        : p(p), r(r), lane(threadIdx.x & 63), n(lane & 15), g(lane >> 4), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
          length(((p.c.I + kParts - 1) / kParts + kUnit - 1) / kUnit * kUnit),  // of a part
          steps((length + kStep - 1) / kStep), from((n & (kParts - 1)) * length),
          // (of the lane's part, as a row of the weights and as a column of the rows)
          left(p.c.I - from < length ? (p.c.I - from < 0 ? 0 : p.c.I - from) : length), nb(fp8_blocks(p.c.H)), kb(fp8_blocks(p.c.I)),
          h_bytes((uint32_t)(p.c.T * p.c.k * p.ldh * 4)), h(__builtin_amdgcn_make_buffer_rsrc(p.h, 0, (int)h_bytes, 0x00020000)) {}

    __device__ __forceinline__ void load(Chunk<T, FP8, FIT> &c, int tile, int at, int s0) const {
        const int row = tile * kColumns + n / kParts, H = p.c.H, e = __builtin_amdgcn_readfirstlane(r.expert[at]);
        const Element *const w = (const Element *)p.c.w_down + ((int64_t)e * H + (row < H ? row : H - 1)) * p.c.I;
        // (the lane's part ends where the next begins, or with the row: a run that the row's end cuts is the last one of all)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (s0 + u) * kStep + g * kRun;
            c.a[u] = fetch<FIT>(w, FIT == kExact || (s0 + u < steps && k < length) ? from + k : p.c.I, p.c.I);
        }
        if (FP8) {
            const float *const scale = p.c.s_down + ((int64_t)e * nb + tile * kColumns / kFp8Block) * kb;
#pragma unroll
            for (int u = 0; u < U / 2; ++u) c.scale[u] = (s0 + 2 * u) * kStep < left ? scale[from / kFp8Block + s0 / 2 + u] : 0.0f;
        }
    }

    __device__ __forceinline__ Run weight(const Chunk<T, FP8, FIT> &c, int s0, int u) const {
        const int k = (s0 + u) * kStep + g * kRun;
        return settle<FIT, Element>(c.a[u], s0 + u < steps && k < length ? from + k : p.c.I, p.c.I);
    }

    // The rows of h for a chunk go through LDS, a part of it for every wave: loaded by the whole wave, each value once (in registers the
    // lanes that multiply the same one would each load it, twice the bytes of the weights), and in 8-bit layers rounded on the way, to what
    // the rounded values stand for.  The next chunk's first rows are on their way while this one is multiplied.
    static constexpr int kSize = FP8 ? 2 : 4, kSlots = FP8 ? kColumns : 4;  // bytes of an element, rows
    static constexpr int kPart = U * kStep, kStaged = kParts * kPart;         // elements of a part and of both
    static constexpr int kPartBytes = kPart * kSize + 16, kRowBytes = kParts * kPartBytes;  // (16 bytes more: other banks for every part)
    static constexpr int kTurns = (kStaged + 255) / 256, kAhead = 2;
    static_assert(kSlots * kRowBytes <= kStageBytes, "room for a wave's rows");
    struct Staged {
        floatx4 v[kTurns];
        uint32_t top[kTurns];
    };
    // (rows of h are whole runs long, zeros behind column I; behind the last row the loads return zeros)
    __device__ __forceinline__ void stage_load(Staged &s, int s0, int pair) const {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int x = i * 256 + lane * 4, part = x / kPart, k = s0 * kStep + x - part * kPart, at = part * length + k;
            const bool in = part < kParts && k < length && at < (int)p.ldh;
            const auto v = __builtin_amdgcn_raw_buffer_load_b128(h, (int)(in ? ((uint32_t)pair * (uint32_t)p.ldh + (uint32_t)at) * 4u : h_bytes), 0, kDeviceScope);
            s.v[i] = __builtin_bit_cast(floatx4, v);
            if constexpr (FP8) {
                s.top[i] = 0u;
                if (in && at < p.c.I) s.top[i] = peek(p.widest + (int64_t)pair * kb + at / kFp8Block);
            }
        }
    }
    __device__ __forceinline__ void stage_store(const Staged &s, unsigned char *row) const {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int x = i * 256 + lane * 4, part = x / kPart;
            unsigned char *const to = row + x * kSize + part * 16;
            if (kStaged % 256 != 0 && part >= kParts) continue;
            if constexpr (FP8) {
                typedef __attribute__((ext_vector_type(2))) short shortx2;
                const float scale = fp8_scale_of(fp8_scale_byte(s.top[i]));
                shortx2 q = {};
                q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q, s.v[i][0], s.v[i][1], scale, false);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q, s.v[i][2], s.v[i][3], scale, true);
                union {
                    bf16x2 p[2];
                    uint2_t d;
                } o;
                o.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(__builtin_bit_cast(int, q), scale, false);
                o.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(__builtin_bit_cast(int, q), scale, true);
                *(uint2_t *)to = o.d;
            } else {
                *(floatx4 *)to = s.v[i];
            }
        }
    }

    // acc += the chunk times the lane's row (8-bit: total, block by block)
    __device__ __forceinline__ void multiply(const Chunk<T, FP8, FIT> &c, const unsigned char *staged, int s0, floatx4 &acc, floatx2 &total) const {
        const unsigned char *const row = staged + n / kParts % kSlots * kRowBytes + n % kParts * kPartBytes + g * kRun * kSize;
        if constexpr (FP8) {
#pragma unroll
            for (int u = 0; u < U; u += 2) {
                floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    union {
                        Run r;
                        intx2 t[2];
                    } f = {weight(c, s0, u + o)};
#pragma unroll
                    for (int z = 0; z < 2; ++z)
                        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_widen(f.t[z], 1.0f), *(const bf16x8 *)(row + (u + o) * kStep * kSize + 16 * z), sum, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) total[i] = __builtin_fmaf(c.scale[u / 2], n & 1 ? sum[2 * i + 1] : sum[2 * i], total[i]);
            }
        } else {
            floatx4 less = {0.0f, 0.0f, 0.0f, 0.0f};  // (a chain of its own)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const Run run = weight(c, s0, u);
                const unsigned char *const b = row + u * kStep * kSize;
                if constexpr (kHalves<T, FP8>) {
                    less = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, run), *(const bf16x8 *)(b + 16), less, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, run), *(const bf16x8 *)b, acc, 0, 0, 0);
                } else {
                    T narrow[kRun];
                    __builtin_memcpy(narrow, &run, 16);
#pragma unroll
                    for (int z = 0; z < kRun; z += 4) {
                        const floatx4 v = *(const floatx4 *)(b + 4 * z);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(narrow[z + i]), v[i], acc, 0, 0, 0);
                    }
                }
            }
            acc += less;
        }
    }

    // What a wave multiplies of an item, one after the other: experts, kSlots tokens at a time (hardly any expert has more: its weights
    // are read again then, from the caches), chunks of the reduction.
    struct Place {
        int at, q, s0;
    };
    __device__ __forceinline__ int rows_of(int at) const { return __builtin_amdgcn_readfirstlane(r.first[at + 1]) - __builtin_amdgcn_readfirstlane(r.first[at]); }
    __device__ __forceinline__ Place after(Place x) const {
        x.s0 += U;
        if (x.s0 < steps) return x;
        x.s0 = 0, x.q += kSlots;
        if (x.q < rows_of(x.at)) return x;
        x.q = 0, x.at += kWaves;
        return x;
    }
    __device__ __forceinline__ void rows_ahead(Staged (&s)[kAhead], Place x) const {
        const int first = __builtin_amdgcn_readfirstlane(r.first[x.at]), count = rows_of(x.at) - x.q;
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (j < count) stage_load(s[j], x.s0, first + x.q + j);
    }
    // Place x with its weights in c and its first rows in s; those of y, if there is one, are asked for before it is multiplied, the rows
    // first: loads come back in order.
    __device__ __forceinline__ void one(const Chunk<T, FP8, FIT> &c, Place x, Chunk<T, FP8, FIT> &d, Place y, Staged (&s)[kAhead], int tile,
                                        floatx4 &acc, floatx2 &total, float (*sums)[kTokens][kColumns], unsigned char *staged) const {
        const int first = __builtin_amdgcn_readfirstlane(r.first[x.at]), rows = rows_of(x.at);
        const int slot = n / kParts, mine = x.q + slot, count = rows - x.q < kSlots ? rows - x.q : kSlots;
        if (x.s0 == 0) acc = floatx4{0.0f, 0.0f, 0.0f, 0.0f}, total = floatx2{0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (j < count) stage_store(s[j], staged + j * kRowBytes);
        for (int j = kAhead; j < count; ++j) {
            stage_load(s[0], x.s0, first + x.q + j);
            stage_store(s[0], staged + j * kRowBytes);
        }
        if (y.at < r.experts) {
            rows_ahead(s, y);
            load(d, tile, y.at, y.s0);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        multiply(c, staged, x.s0, acc, total);
        if (x.s0 + U < steps) return;
        // lane (n, g): columns 2 g and 2 g + 1, part i % 2 in acc[i], for the token and the part of n
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float v = FP8 ? total[i] : n & 1 ? acc[2 * i + 1] : acc[2 * i];
            v += __shfl_xor(v, 1);
            if ((n & 1) == 0 && slot < count) sums[wave][r.token[first + mine]][2 * g + i] += r.weight[first + mine] * v;
        }
    }

    // `c`: the wave's first chunk of the item, loaded already where it has one.  What comes next is asked for before a chunk is multiplied.
    __device__ __forceinline__ void item(Chunk<T, FP8, FIT> &c, int tile, float (*sums)[kTokens][kColumns], unsigned char *staged) const {
        static_assert(kTokens * kColumns == 128, "two sums a lane");
        (&sums[wave][0][0])[lane] = 0.0f;  // (a wave's own: its LDS operations keep their order)
        (&sums[wave][0][0])[lane + 64] = 0.0f;
        floatx4 acc;
        floatx2 total;
        Chunk<T, FP8, FIT> d;
        Staged s[kAhead];
        if (wave < r.experts) rows_ahead(s, {wave, 0, 0});
        __builtin_amdgcn_s_waitcnt(0x0f70);  // (vmcnt(0): in the loop the rows are waited for with the weights behind them on their way)
        for (Place x = {wave, 0, 0}; x.at < r.experts;) {
            const Place y = after(x);
            one(c, x, d, y, s, tile, acc, total, sums, staged);
            if (y.at >= r.experts) break;
            x = after(y);
            one(d, y, c, x, s, tile, acc, total, sums, staged);
        }
        __syncthreads();
        const int t = threadIdx.x / kColumns, col = tile * kColumns + threadIdx.x % kColumns;
        if (t < (int)p.c.T && col < p.c.H) {
            float v = 0.0f;
#pragma unroll
            for (int u = 0; u < kWaves; ++u) v += sums[u][t][threadIdx.x % kColumns];
            if (p.stream != nullptr) v += to_f32(((const T *)p.stream)[(int64_t)t * p.c.H + col]);
            if (r.lost >> t & 1u) v = __builtin_nanf("");
            ((T *)p.out)[(int64_t)t * p.c.H + col] = from_f32<T>(v);
        }
    }
};

// ---- second kernel: both, with one meeting of all workgroups between them -------------------------------------------------------
// The gated unit's items are dealt out in as many units as there are workgroups: unit b is items b, b + G, ...; each unit has a word: 0
// free, 1 claimed, 2 done.  A workgroup claims its own unit; before it waits for anything it looks whether there is one that nobody has
// claimed (of a workgroup that has not started yet) and does it in the other's place.  Whoever claims a unit is running, and waits for
// nothing before the unit is done: every wait ends, however many of the workgroups are there at once.
template <typename T, bool FP8, int FIT, bool NARROW>
__global__ __launch_bounds__(kThreads, 2) void layer_experts_kernel(Layer p) {
    __shared__ Routing r;
    __shared__ union {
        Parts parts;
        struct {
            Sums sums[2];
            alignas(16) unsigned char staged[kWaves][kStageBytes];
        } back;
    } room;
    __shared__ int found;
    const int tid = threadIdx.x, G = (int)gridDim.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto claim = [&](int unit) { return __hip_atomic_fetch_max(p.units + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0u ? unit : -1; };
    int unit = -1;
    if (tid == 0) unit = claim((int)blockIdx.x);  // (asked for before the routing is known: the answer is there by then)
    find_routing<T>(p, r);
    const int tiles = (int)(p.ldh / 8), items = r.experts * tiles, units = items < G ? items : G;
    const int last = ceil_div(p.c.H, kColumns);
    int turn = 0;
    const Down<T, FP8, FIT> down(p, r);
    Chunk<T, FP8, FIT> c;
    if ((int)blockIdx.x >= units) unit = -1;
    for (;;) {
        // (of thread 0: the unit that it claimed)
        if (tid == 0) found = unit;
        __syncthreads();
        const int got = found;
        if (got >= 0) {
            GateUp<T, FP8, FIT, NARROW> front(p, r);
            front.run(got, items, G, room.parts, turn);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every wave's rows of h are there, before the word that says so
            __syncthreads();
            if (tid == 0) __hip_atomic_store(p.units + got, 2u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if ((int)blockIdx.x < last && wave < r.experts) down.load(c, blockIdx.x, wave, 0);
        bool all;
        int any;
        for (;;) {
            int least = 2, free = -1;
            for (int b = tid; b < units; b += kThreads) {
                const int state = (int)peek(p.units + b);
                if (state < least) least = state;
                if (state == 0) free = b;
            }
            any = free;
            all = __syncthreads_and(least == 2);
            if (all || __syncthreads_or(free >= 0)) break;
            __builtin_amdgcn_s_sleep(1);
        }
        if (all) break;
        if (tid == 0) found = -1;
        __syncthreads();
        if (any >= 0) atomicMax(&found, any);  // (any of them)
        __syncthreads();
        if (tid == 0) unit = claim(found);
        __syncthreads();
    }
    turn = 0;
    for (int i = blockIdx.x; i < last; i += G, ++turn) {
        if (turn != 0 && wave < r.experts) down.load(c, i, wave, 0);
        down.item(c, i, room.back.sums[turn & 1], room.back.staged[wave]);
    }
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// one a CU; and a thread of each for every other's word
int most_workgroups() { return device_info().cu_count < kThreads ? device_info().cu_count : kThreads; }

struct Room {
    size_t stream, rows, h, widest, flags;  // bytes
    int64_t ld, ldh;
    explicit Room(const mfl_moe_layer &c) {
        const bool fp8 = c.s_gate != nullptr, norm = c.norm_weight != nullptr;
        ld = fp8 ? fp8_ld(c.H) : c.H;
        ldh = (c.I + 15) / 16 * 16;
        stream = c.residual != nullptr ? up256((size_t)c.T * c.H * dtype_size(c.dtype)) : 0;
        rows = fp8 ? up256((size_t)c.T * ld * 2) : norm ? up256((size_t)c.T * ld * dtype_size(c.dtype)) : 0;
        h = up256((size_t)c.T * c.k * ldh * 4);
        widest = fp8 ? up256((size_t)c.T * c.k * fp8_blocks(c.I) * 4) : 0;
        flags = up256((size_t)most_workgroups() * 4);
    }
    size_t all() const { return stream + rows + h + widest + flags; }
};

template <typename T, bool FP8, int FIT, bool NARROW>
int launch(const Layer &p, hipStream_t stream) {
    const int tokens = (int)p.c.T;
    // (two experts a workgroup: with eight the call takes 2 us more at 13 to 16 tokens of 128 experts; with one the same at one token)
    const dim3 grid(ceil_div(p.c.E, kRouterExperts), tokens);
    if (p.c.H % 8 != 0) layer_router_kernel<T, kRouterExperts, FP8, false, false><<<grid, 256, 0, stream>>>(p);
    else if (p.c.H <= 2048) layer_router_kernel<T, kRouterExperts, FP8, true, true><<<grid, 256, 0, stream>>>(p);
    else layer_router_kernel<T, kRouterExperts, FP8, true, false><<<grid, 256, 0, stream>>>(p);
    const int hits = p.c.T * p.c.k < p.c.E ? (int)p.c.T * p.c.k : p.c.E;
    const int64_t front = hits * (p.ldh / 8), back = ceil_div(p.c.H, kColumns), want = front > back ? front : back;
    const unsigned most = (unsigned)most_workgroups();
    layer_experts_kernel<T, FP8, FIT, NARROW><<<want < most ? (unsigned)want : most, kThreads, 0, stream>>>(p);
    return launch_status();
}

template <typename T, bool FP8, bool NARROW>
int launch_fit(const Layer &p, hipStream_t stream) {
    typedef GateUp<T, FP8, kExact, NARROW> Front;
    typedef Down<T, FP8, kExact> Back;
    const int H = p.c.H, I = p.c.I;
    if (H % (kWaves * Front::U * Front::kStep) == 0 && I % Back::kStaged == 0) return launch<T, FP8, kExact, NARROW>(p, stream);
    if (H % Front::kRun == 0 && I % Front::kRun == 0) return launch<T, FP8, kWhole, NARROW>(p, stream);
    return launch<T, FP8, kRagged, NARROW>(p, stream);
}

template <typename T, bool FP8>
int launch_width(const Layer &p, hipStream_t stream) {
    typedef GateUp<T, FP8, kWhole, true> Narrow;
    return p.c.H <= kWaves * Narrow::U * Narrow::kStep ? launch_fit<T, FP8, true>(p, stream) : launch_fit<T, FP8, false>(p, stream);
}

template <typename T>
int launch_type(const Layer &p, hipStream_t stream) {
    return p.c.s_gate != nullptr ? launch_width<T, true>(p, stream) : launch_width<T, false>(p, stream);
}

}  // namespace

size_t moe_layer_workspace(const mfl_moe_layer &c) { return Room(c).all(); }

int moe_layer_fwd(const mfl_moe_layer &c, void *out, void *logits, void *workspace, hipStream_t stream) {
    const Room room(c);
    uint8_t *at = (uint8_t *)workspace;
    auto take = [&](size_t bytes) {
        uint8_t *const here = bytes ? at : nullptr;
        at += bytes;
        return here;
    };
    Layer p = {};
    p.c = c, p.out = out, p.logits = logits;
    p.ld = room.ld, p.ldh = room.ldh;
    p.stream_out = take(room.stream);
    p.stream = c.norm_weight == nullptr ? nullptr : p.stream_out != nullptr ? p.stream_out : c.x;
    p.rows_out = take(room.rows);
    p.rows = p.rows_out != nullptr ? p.rows_out : c.x;
    p.h = (float *)take(room.h);
    p.zeros = (uint32_t *)at;
    p.zero_words = (int)((room.widest + room.flags) / 4);
    p.widest = (uint32_t *)take(room.widest);
    p.units = (uint32_t *)take(room.flags);
    int rc = MFL_OK;
    MFL_DISPATCH_FLOAT(c.dtype, T, { rc = launch_type<T>(p, stream); });
    return rc;
}

}  // namespace mfl
