// Expert products in 8-bit floating point for a few rows per expert: the forward product and the gated unit in one launch,
// the rows quantised on the way.
//
// The weights are all the traffic.  A workgroup (four waves) owns 16 rows of an expert and PIECES blocks of 16 columns (gated:
// half of them of either matrix); its waves share the reduction, wave w taking the blocks of 128 number w, w + 4, ...  A block
// of 16 columns is one v_mfma_scale_f32_16x16x128_f8f6f4, whose operands come straight from memory into registers: nothing is
// shared between waves, so nothing goes through LDS, and the next two pieces' weights are on their way while one is
// multiplied.  A lane holds bytes 16 g .. 16 g + 15 and 64 + 16 g .. of a row of the block (g: its quarter of the wave), so that
// four lanes read 64 bytes of a row together; the rows are loaded in the same order, their largest magnitude found over the
// four lanes, and rounded to e4m3 in registers (the order within the block does not matter as long as both operands agree).
// The waves' sums meet in LDS.  The gated unit's operands are widened to bf16 and multiplied by v_mfma_f32_16x16x32_bf16 (fp8.h
// says why): in a graph 32 tokens' unit 63.9 against 63.5 us, one token's MLP 15.9 against 15.2.
//
// Bound by the weights' bytes: 32 tokens of 8 of 128 experts, 2048 to 2 x 768, 66 us for 349 MB, 5.3 TB/s.  Of a single token's
// 10 us (25 MB) a wave spends 0.8 finding its rows, 3 (weights in the caches) to 7 until weights and rows are there and quantised, 0.8
// multiplying and joining; instructions fetched for the first time count too, which is why the conversions are the packed ones (16
// for a block's 32 elements) and a chunk that is whole asks nothing: 12.4 us with conversions one by one.
#include <type_traits>

#include "fp8.h"

namespace mfl {

namespace {

constexpr int kRows = 16, kWaves = 4;
constexpr int kBuffers = 3;  // pieces of weights in registers

// 16 elements of a row.  `widest`: the largest magnitude's bits as of a float, in `bits` and these (16-bit types: compared as
// they are, two at a time).  `finite`: the same of the finite ones.  `pack`: four of them by the power of two `scale` as e4m3,
// infinities as NaN: v_cvt_scalef32_pk_fp8_* give what dividing and rounding gives (all values of the 16-bit types, at 13 scales).
template <typename T>
struct Piece {
    static constexpr int kDwords = 4 * sizeof(T);
    union {
        uint4_t q[sizeof(T)];
        uint32_t d[kDwords];
        T e[16];
    };
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) q[i] = ((const uint4_t *)p)[i];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) q[i] = uint4_t{0u, 0u, 0u, 0u};
    }
    __device__ __forceinline__ uint32_t widest(uint32_t bits) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; ++i) bits = fp8_wider(bits, e[i]);
            return bits;
        } else {
            typedef __attribute__((ext_vector_type(2))) uint16_t ushortx2;
            ushortx2 m = {0, 0};
#pragma unroll
            for (int i = 0; i < kDwords; ++i) {
                const uint32_t w = d[i] & 0x7fff7fffu;
                m = __builtin_elementwise_max(m, __builtin_bit_cast(ushortx2, w));
            }
            const uint16_t top = m[0] > m[1] ? m[0] : m[1];
            return fp8_wider(bits, to_f32(__builtin_bit_cast(T, top)));
        }
    }
    __device__ __forceinline__ uint32_t finite(uint32_t bits) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) bits = fp8_wider(bits, fp8_finite_abs(to_f32(e[i])));
        return bits;
    }
    // (all first halves of the results, then all second ones: a half behind the other half of the same register has to wait)
    __device__ __forceinline__ void pack(int (&out)[4], float scale) const {
        typedef __attribute__((ext_vector_type(2))) short shortx2;
        typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
        typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
        shortx2 r[4] = {};
        auto half = [&](auto second) {
            constexpr bool S = decltype(second)::value;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4)
                    r[i] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r[i], e[4 * i + 2 * S], e[4 * i + 2 * S + 1], scale, S);
                else if constexpr (std::is_same<T, bf16_t>::value)
                    r[i] = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r[i], __builtin_bit_cast(bf16x2, d[2 * i + S]), scale, S);
                else
                    r[i] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r[i], __builtin_bit_cast(f16x2, d[2 * i + S]), scale, S);
            }
        };
        half(std::false_type{});
        half(std::true_type{});
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = __builtin_bit_cast(int, r[i]);
    }
};

// The largest of the four lanes that hold a row's block, in all of them.
__device__ __forceinline__ uint32_t over_block(uint32_t a) {
    const auto x = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    a = x[0] > x[1] ? x[0] : x[1];
    const auto y = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    return y[0] > y[1] ? y[0] : y[1];
}

// The row counts of up to 256 experts at once (their loads in flight together), then 64 at a time.  A launch has at most 2^16
// tiles and so fewer than 2^20 rows: 64 counts of no more than that each sum to less than 2^31, and the two sums, which need not
// wait for each other, are never taken past the first expert whose tiles pass `slot`.
__device__ __forceinline__ bool find_rows(const Fp8Product &p, int slot, int lane, int &expert, int64_t &row0, int &rows) {
    int tiles_before = 0, rows_before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 256) {
        uint32_t count[4];
        fp8_load_counts(p.m_sizes, p.ms_i64, e0 + lane, p.E, p.R, count);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = (int)count[i], t = ceil_div(m, kRows);
            const int mi = wave_inclusive_scan(m), ti = wave_inclusive_scan(t);
            const uint64_t past = __ballot(tiles_before + ti > slot);
            if (past) {
                const int src = __ffsll((unsigned long long)past) - 1;
                const int m_e = __builtin_amdgcn_readlane(m, src);
                const int tile = slot - (tiles_before + __builtin_amdgcn_readlane(ti, src) - __builtin_amdgcn_readlane(t, src));
                const int first = rows_before + __builtin_amdgcn_readlane(mi, src) - m_e + tile * kRows;
                const int left = m_e - tile * kRows, room = (int)p.R - first;  // (counts that sum to more than the rows are cut there)
                expert = e0 + 64 * i + src;
                row0 = first;
                rows = left < kRows ? left : kRows;
                if (rows > room) rows = room;
                return rows > 0;
            }
            rows_before += wave_last(mi);
            tiles_before += wave_last(ti);
        }
    }
    return false;
}

// AHEAD: blocks of the reduction that a wave holds of the rows, and of every piece, at a time.  Gated: bf16 products.
template <bool GLU, int PIECES, int AHEAD, typename TX, typename TO>
__global__ __launch_bounds__(kWaves * 64, 2) void fp8_decode_kernel(Fp8Product p, const TX *__restrict__ x) {
    static_assert(!GLU || PIECES % 2 == 0, "gated: blocks of columns of both matrices");
    constexpr int TILES = GLU ? PIECES / 2 : PIECES;  // blocks of output columns
    __shared__ floatx4 sums[kWaves][PIECES][64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    int e, rows;
    int64_t row0;
    // (up to 64 rows, the whole index is read along with the row counts: what a call of a few rows takes is the number of loads
    // one behind the other)
    const bool early = p.row_idx != nullptr && p.R <= 64;
    int index = 0;
    if (early) index = p.row_idx[lane < p.R ? lane : 0];
    if (!find_rows(p, blockIdx.y, lane, e, row0, rows)) return;
    const int n0 = blockIdx.x * 16 * TILES;
    const int blocks = fp8_blocks(p.K), nbn = fp8_blocks(p.N), full = p.K / kFp8Block;

    int64_t src = row0 + (c < rows ? c : rows - 1);
    int looked_up = 0;
    if (early) looked_up = __shfl(index, (int)src);
    else if (p.row_idx != nullptr) looked_up = p.row_idx[src];

    union Frag {
        uint4_t v[2];
        intx2 t[4];
        intx8 i;
    };
    // A chunk of the reduction, blocks b0, b0 + 4, ...  Whole: all of them are there to the end, and nothing is asked about them (a
    // short call takes as long as its instructions take to arrive).
    // Piece t: columns n0 + 16 (t / 2) of matrix t % 2 where gated, else n0 + 16 t.  Columns past the last are not stored.
    floatx4 acc[PIECES];
#pragma unroll
    for (int t = 0; t < PIECES; ++t) acc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    auto chunk = [&](int b0, auto whole) {
        constexpr bool W = decltype(whole)::value;
        Frag fw[kBuffers][AHEAD];
        auto load = [&](int t) {
            const Fp8Matrix &m = p.w[GLU ? t & 1 : 0];
            int n = n0 + 16 * (GLU ? t / 2 : t) + c;
            if (n >= p.N) n = p.N - 1;
            const uint8_t *const w = m.q + (int64_t)e * p.N * p.K;
            const uint32_t at = (uint32_t)n * (uint32_t)p.K + 16 * g;
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = (b0 + kWaves * u) * kFp8Block + 64 * h;
                    if (W || k + 16 * g < p.K) fw[t % kBuffers][u].v[h] = *(const uint4_t *)(w + k + at);  // (K is a multiple of 16)
                    else fw[t % kBuffers][u].v[h] = uint4_t{0u, 0u, 0u, 0u};
                }
        };
        // the weights' scales of the chunk: lane t AHEAD + u that of piece t in block b0 + 4 u
        static_assert(PIECES * AHEAD <= 64, "one scale a lane");
        float scales = 0.0f;
        {
            const int t = lane / AHEAD, b = b0 + kWaves * (lane % AHEAD);
            int nb = (n0 + 16 * (GLU ? t / 2 : t)) / kFp8Block;
            if (nb >= nbn) nb = nbn - 1;
            if (t < PIECES && b < blocks)
                scales = (GLU && t & 1 ? p.w[1].scale : p.w[0].scale)[((int64_t)e * nbn + nb) * blocks + b];
        }
#pragma unroll
        for (int t = 0; t < kBuffers - 1 && t < PIECES; ++t) load(t);
        // the rows' blocks, quantised
        Frag q[AHEAD];
        bf16x8 wide[AHEAD][4];  // (gated)
        int byte[AHEAD];
        {
            int64_t row = src;
            if (p.row_idx != nullptr) {
                const int i = looked_up / p.idx_div;
                row = i < 0 ? 0 : i >= p.src_rows ? p.src_rows - 1 : i;
            }
            const TX *const xr = x + row * p.K + 16 * g;
            Piece<TX> fx[AHEAD][2];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = (b0 + kWaves * u) * kFp8Block + 64 * h;
                    if (W || k + 16 * g < p.K) fx[u][h].load(xr + k);
                    else fx[u][h].clear();
                }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                uint32_t a = over_block(fx[u][1].widest(fx[u][0].widest(0u)));
                if (__builtin_expect(__any(fp8_unusual(a)), 0)) a = over_block(fx[u][1].finite(fx[u][0].finite(0u)));
                byte[u] = fp8_scale_byte(a);
                const float scale = fp8_scale_of(byte[u]);
                int lo[4], hi[4];
                fx[u][0].pack(lo, scale);
                fx[u][1].pack(hi, scale);
                q[u].i = intx8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                if constexpr (GLU) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) wide[u][i] = fp8_widen(q[u].t[i], scale);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < PIECES; ++t) {
            if (t + kBuffers - 1 < PIECES) load(t + kBuffers - 1);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (!W && b0 + kWaves * u >= blocks) break;
                const Frag &w = fw[t % kBuffers][u];
                floatx4 part = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (GLU) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_widen(w.t[i], 1.0f), wide[u][i], part, 0, 0, 0);
                } else {
                    part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.i, q[u].i, part, 0, 0, 0, 127, 0, byte[u]);
                }
                const float s = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scales), t * AHEAD + u));
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_fmaf(s, part[i], acc[t][i]);
            }
        }
    };
    int b0 = wave;
    for (; b0 + kWaves * (AHEAD - 1) < full; b0 += kWaves * AHEAD) chunk(b0, std::true_type{});
    if (b0 < blocks) chunk(b0, std::false_type{});
#pragma unroll
    for (int t = 0; t < PIECES; ++t) sums[wave][t][lane] = acc[t];
    __syncthreads();
    if (c >= rows) return;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        if (t % kWaves != wave) continue;
        floatx4 v[GLU ? 2 : 1];
#pragma unroll
        for (int m = 0; m < (GLU ? 2 : 1); ++m) {
            v[m] = sums[0][GLU ? 2 * t + m : t][lane];
#pragma unroll
            for (int s = 1; s < kWaves; ++s) v[m] += sums[s][GLU ? 2 * t + m : t][lane];
        }
        // four columns of row c
        const int n = n0 + 16 * t + 4 * g;
        const int64_t at = (row0 + c) * p.N + n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (n + i >= p.N) continue;
            if (!GLU) {
                ((TO *)p.out)[at + i] = from_f32<TO>(v[0][i]);
            } else {
                const float ev = v[0][i], gv = v[GLU ? 1 : 0][i];
                const float h = ev * sigmoid_f32(ev) * gv;
                if (p.h32 != nullptr)
                    p.h32[at + i] = h;
                else
                    ((TO *)p.out)[at + i] = from_f32<TO>(h);
                if (p.e_out != nullptr) ((TO *)p.e_out)[at + i] = from_f32<TO>(ev);
                if (p.g_out != nullptr) ((TO *)p.g_out)[at + i] = from_f32<TO>(gv);
            }
        }
    }
}

template <int PIECES, int AHEAD, typename TX, typename TO>
int launch_as(const Fp8Product &p, const TX *x, hipStream_t stream) {
    const unsigned slots = (unsigned)fp8_max_tiles(p.R, p.E, kRows);
    if (p.glu)
        fp8_decode_kernel<true, PIECES, AHEAD, TX, TO><<<dim3(ceil_div(p.N, 8 * PIECES), slots), kWaves * 64, 0, stream>>>(p, x);
    else
        fp8_decode_kernel<false, PIECES, AHEAD, TX, TO><<<dim3(ceil_div(p.N, 16 * PIECES), slots), kWaves * 64, 0, stream>>>(p, x);
    return launch_status();
}

template <typename TX, typename TO>
int launch(const Fp8Product &p, const TX *x, hipStream_t stream) {
    // Pieces of a workgroup: two where there are few (latency counts: as many workgroups as there can be), else eight, two
    // workgroups a CU.
    const int64_t row_tiles = p.R < p.E ? p.R : p.E;
    const bool few = row_tiles * ceil_div(p.N, 16) * (p.glu ? 2 : 1) < (int64_t)8 * 2 * device_info().cu_count;
    // (fp32 rows of four blocks and eight pieces do not fit the registers)
    if (fp8_blocks(p.K) <= 2 * kWaves || sizeof(TX) == 4) return few ? launch_as<2, 2, TX, TO>(p, x, stream) : launch_as<8, 2, TX, TO>(p, x, stream);
    return few ? launch_as<2, 4, TX, TO>(p, x, stream) : launch_as<8, 4, TX, TO>(p, x, stream);
}

}  // namespace

bool gemm_fp8_decodes(const Fp8Product &p) {
    if (p.dx || p.out_dtype == MFL_F32 || p.K % 16 != 0 || p.R > (int64_t)kFp8DecodeRowsPerExpert * p.E) return false;
    if (fp8_max_tiles(p.R, p.E, kRows) > 65535 || (int64_t)p.N * p.K > 0xffffffffll) return false;  // (32-bit offsets in a matrix)
    return aligned(p.w[0].q, 16) && (!p.glu || aligned(p.w[1].q, 16));
}

int gemm_fp8_decode(const Fp8Product &p, const void *x, int x_dtype, hipStream_t stream) {
    if (!gemm_fp8_decodes(p) || !aligned(x, 16)) return MFL_ERR_UNSUPPORTED;
    if (x_dtype == MFL_F32)
        return p.out_dtype == MFL_BF16 ? launch<float, bf16_t>(p, (const float *)x, stream) : launch<float, f16_t>(p, (const float *)x, stream);
    if (x_dtype != p.out_dtype) return MFL_ERR_UNSUPPORTED;
    return p.out_dtype == MFL_BF16 ? launch<bf16_t, bf16_t>(p, (const bf16_t *)x, stream) : launch<f16_t, f16_t>(p, (const f16_t *)x, stream);
}

}  // namespace mfl
