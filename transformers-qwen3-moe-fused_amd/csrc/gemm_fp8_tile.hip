// Expert products in 8-bit floating point on LDS tiles: 16-bit outputs, rows of whole 16-byte pieces (K % 16 == 0).
//
//   forward         out[r, n] = sum_b S[e, n / 128, b] sx[r, b] sum_{k in block b} x[r, k] w[e, n, k]
//   gated           the same for two matrices, out = silu(gate) * up
//   input gradient  out[r, k] = sum_b S[e, b, k / 128] sd[r, b] sum_{n in block b} d[r, n] w[e, n, k], of one or two terms
//
// A workgroup of eight waves owns a tile of BM rows and BN columns of one expert and walks the reduction in steps of one scale
// block, 128 bytes of every row.  A stage in LDS is one such step: BM x 128 row bytes, BN x 128 weight bytes, and the dwords
// that hold the rows' scale bytes.  Everything arrives by direct copies (global_load_lds) that the wave counts itself; one
// barrier a step publishes the stage that has landed and frees the one before.  The tiles of a workgroup are one stream of
// steps: the first copies of the next tile go out under the last step of this one.
//
//   v_mfma_scale_f32_32x32x64_f8f6f4, weights first: a lane's 16 accumulators of a 32 x 32 block belong to one row (whose
//   scale it hands to the instruction) and to runs of four columns.  Two instructions make a block's partial sum over a step,
//   16 multiply-adds by the weights' scale (uniform: 128 x 128) add it to the running fp32 sum.
//
// The instruction adds its products in groups of eight and cuts them off 2^-13 below the group's largest (measured): 3e-6 of
// the sum of magnitudes on average, where the rounding of a 16-bit output is 2e-4 or 2e-3 of the sum itself.  fp32 outputs
// are not taken here.
//
// LDS layouts.  Rows of 128 bytes along the reduction: 16-byte chunk c of row r at c ^ ((r >> 1) & 7).  A lane's 32 bytes of a
// 64-wide sub-step are chunks 4 s + h and 4 s + 2 + h (h: its half of the wave); which reduction element sits where in the
// instruction does not matter as long as both operands agree.  Input gradient: the weights lie as in memory, 128 rows of the
// reduction by BN columns, chunk c of row n at c ^ ((n & 7) << 1), and are read with ds_read_b64_tr_b8 (a group of 16 lanes
// reads 8 rows of 16 bytes and gets 8 rows of one column each), four of them for the same 32 elements.
#include <type_traits>

#include "fp8.h"

namespace mfl {

namespace {

typedef __attribute__((address_space(3))) void *lds_void_ptr;
typedef __attribute__((ext_vector_type(2))) int intx2;
typedef __attribute__((address_space(3))) intx2 *lds_intx2_ptr;
typedef const __attribute__((address_space(3))) uint4_t *lds_uint4_ptr;
typedef const __attribute__((address_space(3))) uint32_t *lds_uint32_ptr;
typedef const __attribute__((address_space(3))) float *lds_float_ptr;

constexpr int kXcd = 8;
constexpr int kMaxExperts = 512;  // prefix tables in LDS
constexpr int kWaves = 8, kThreads = kWaves * 64;

__device__ uint4_t g_fp8_zeros = {0u, 0u, 0u, 0u};

// Copies of 16 and 4 bytes per active lane to LDS address lds_addr + lane * size.  Written out by hand: the compiler orders
// LDS reads behind every copy it knows of; the kernel waits for its copies itself.  M0 is used by nothing else here.
__device__ __forceinline__ void copy16(const void *src, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds_addr) : "memory");
}
// (the same from a scalar base and a 32-bit offset of the lane)
__device__ __forceinline__ void copy16(const uint8_t *base, uint32_t offset, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds_addr) : "memory");
}
__device__ __forceinline__ void copy4(const void *src, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(src), "s"(lds_addr) : "memory");
}

// What the wave has read from LDS is in its registers, at most N of its copies are on their way; then the barrier.
template <int N>
__device__ __forceinline__ void publish() {
    static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// WM x WN waves of MI x NI blocks of 32 x 32.
template <int WM, int WN, int MI, int NI, int STAGES>
struct Shape {
    static_assert(WM * WN == kWaves, "eight waves");
    static constexpr int BM = WM * MI * 32, BN = WN * NI * 32;
    static constexpr int kSLanes = BM / kWaves;                    // rows whose scale dwords a wave copies,
    static constexpr int kSWave = (kSLanes + 2) * 4;               // and behind them the weights' scales of its columns
    static constexpr int kA = BM * 128, kB = BN * 128, kS = kWaves * kSWave;
    static constexpr int kStage = (kA + kB + kS + 1023) / 1024 * 1024;
    static constexpr int kACopies = kA / 1024 / kWaves, kBCopies = kB / 1024 / kWaves;
    static constexpr int kOps = kACopies + kBCopies + 1;  // vector-memory operations a wave issues for a stage
    static constexpr int kTables = 2 * (kMaxExperts + 1) * 4;
    static constexpr int kLds = STAGES * kStage + kTables;
    static_assert(kA % (1024 * kWaves) == 0 && kB % (1024 * kWaves) == 0 && kSLanes + 2 <= 64, "whole copies");
};

// HQ: the gated unit's result leaves as quantised rows.
template <bool DX, bool GLU, bool HQ, int WM, int WN, int MI, int NI, int STAGES, typename TO>
__global__ __launch_bounds__(kThreads) void fp8_tile_kernel(Fp8Product p) {
    using S = Shape<WM, WN, MI, NI, STAGES>;
    constexpr int BM = S::BM, BN = S::BN;
    constexpr int BNC = GLU ? BN / 2 : BN;  // output columns of a tile
    static_assert(!GLU || NI == 2, "gated: a wave holds one block of either matrix");
    static_assert(!HQ || (GLU && BNC == kFp8Block), "quantised output: a tile's columns are one scale block");
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    int *const tab_rows = (int *)(smem + STAGES * S::kStage);
    int *const tab_tiles = tab_rows + kMaxExperts + 1;
    float *const amax = (float *)(tab_tiles + kMaxExperts + 1);  // (HQ) per row and wave column
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    const int l = lane & 31, half = lane >> 5;
    const int cols = DX ? p.K : p.N, red = DX ? p.N : p.K;
    const int col_tiles = ceil_div(cols, BNC);
    const int steps_of_term = fp8_blocks(red), KT = DX ? steps_of_term * p.terms : steps_of_term;
    const int nbn = fp8_blocks(p.N), kbk = fp8_blocks(p.K);
    const int64_t lda = fp8_ld(red);
    const int lds_ = (int)fp8_ld_scale(red);

    // ---- rows and row tiles before every expert; an expert's rows are cut into tiles of equal height, a multiple of 32
    {
        int row_carry = 0, tile_carry = 0;
        for (int e0 = 0; e0 < p.E; e0 += 64) {
            const int e = e0 + lane;
            int m = e < p.E ? load_msize(p.m_sizes, p.ms_i64, e) : 0;
            if (m < 0) m = 0;
            const int64_t room = p.R - row_carry;  // sizes that sum to more than R rows are cut there
            const int before = wave_inclusive_scan(m) - m;
            if (before >= room) m = 0;
            else if (before + m > room) m = (int)(room - before);
            const int t = ceil_div(m, BM);
            const int mi = wave_inclusive_scan(m), ti = wave_inclusive_scan(t);
            if (wave == 0 && e < p.E) tab_rows[e] = row_carry + mi - m, tab_tiles[e] = tile_carry + ti - t;
            row_carry += wave_last(mi), tile_carry += wave_last(ti);
        }
        if (tid == 0) tab_rows[p.E] = row_carry, tab_tiles[p.E] = tile_carry;
        __syncthreads();
    }
    const int total = __builtin_amdgcn_readfirstlane(tab_tiles[p.E]) * col_tiles;
    const int per_xcd = ceil_div(total, kXcd);
    const int last = ((int)blockIdx.x % kXcd + 1) * per_xcd < total ? ((int)blockIdx.x % kXcd + 1) * per_xcd : total;
    const int stride = (int)gridDim.x / kXcd;

    struct Tile {
        int index, expert, row0, rows, col0;
    };
    auto decode = [&](Tile &t) {
        const int v = t.index / col_tiles;
        int e = 0;
        for (int e0 = 0; e0 < p.E; e0 += 64) {
            const int i = e0 + lane < p.E ? e0 + lane : p.E - 1;
            const uint64_t hits = __ballot(e0 + lane < p.E && v >= tab_tiles[i] && v < tab_tiles[i + 1]);
            if (hits) {
                e = e0 + __ffsll((unsigned long long)hits) - 1;
                break;
            }
        }
        e = __builtin_amdgcn_readfirstlane(e);
        const int first = __builtin_amdgcn_readfirstlane(tab_tiles[e]), n = __builtin_amdgcn_readfirstlane(tab_tiles[e + 1]) - first;
        const int r0 = __builtin_amdgcn_readfirstlane(tab_rows[e]), m = __builtin_amdgcn_readfirstlane(tab_rows[e + 1]) - r0;
        const int local = t.index - first * col_tiles;
        const int height = ceil_div(ceil_div(m, n), 32) * 32;
        t.expert = e;
        t.row0 = r0 + local % n * height;
        t.rows = m - local % n * height;
        if (t.rows > height) t.rows = height;
        t.col0 = local / n * BNC;
    };
    Tile cur;
    cur.index = (int)blockIdx.x % kXcd * per_xcd + (int)blockIdx.x / kXcd;
    if (cur.index >= last) return;
    decode(cur);

    // ---- the producer's side: per-lane sources of the copies of the tile whose steps it is issuing
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_ptr)smem;
    Tile pt = cur;
    int pstep = 0, pstage = 0;
    bool more = true;
    // (rows that are not gathered are addressed from the tile's first one; gathered ones from the first of all, within 32 bits)
    const bool gathered = !DX && p.row_idx != nullptr;
    uint32_t aoff[S::kACopies], boff[S::kBCopies];
    const uint8_t *sptr;  // the lane's scale dword: of a row, or of the weights
    const uint8_t *abase, *bbase;
    auto source = [&](int r) -> int {
        const int i = r < pt.rows ? r : pt.rows - 1;
        if (!gathered) return i;
        const int at = p.row_idx[pt.row0 + i] / p.idx_div;
        return at < 0 ? 0 : at >= (int)p.src_rows ? (int)p.src_rows - 1 : at;
    };
    // column block of the weights' scales of the wave's columns (which lie in one: 64 or 32 columns from a multiple of that)
    auto scale_block = [&](const Tile &t) {
        const int at = (t.col0 + (GLU ? wn * 32 : wn * NI * 32)) / kFp8Block, end = DX ? kbk : nbn;
        return at < end ? at : end - 1;
    };
    auto start_term = [&](int term) {
        const Fp8Rows a = term ? p.a[1] : p.a[0];
        const uint8_t *w = (term ? p.w[1].q : p.w[0].q) + (int64_t)pt.expert * p.N * p.K;
        const int64_t first = gathered ? 0 : pt.row0;
        abase = a.q + first * lda;
        bbase = DX ? w + pt.col0 : w + (int64_t)pt.col0 * p.K;
        const int sl = lane < S::kSLanes ? lane : 0;
        const uint8_t *row = a.scale + (first + source(wave * S::kSLanes + sl)) * lds_;
        const float *ws = (term || (GLU && lane > S::kSLanes) ? p.w[1].scale : p.w[0].scale) + (int64_t)pt.expert * nbn * kbk;
        ws += DX ? scale_block(pt) : (int64_t)scale_block(pt) * kbk;
        sptr = lane < S::kSLanes ? row : (const uint8_t *)ws;
    };
    auto start_tile = [&]() {
#pragma unroll
        for (int c = 0; c < S::kACopies; ++c) {
            const int r = (wave * S::kACopies + c) * 8 + (lane >> 3);
            aoff[c] = (uint32_t)source(r) * (uint32_t)lda + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
        }
#pragma unroll
        for (int c = 0; c < S::kBCopies; ++c) {
            const int load = wave * S::kBCopies + c;
            if (!DX) {
                const int r = load * 8 + (lane >> 3);
                int n = GLU ? r % BNC : r;
                if (pt.col0 + n >= p.N) n = p.N - 1 - pt.col0;  // (columns that are not stored)
                boff[c] = (uint32_t)n * (uint32_t)p.K + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
            } else {
                constexpr int CPR = BN / 16;  // chunks of a row of the reduction
                const int r = (load * 64 + lane) / CPR;
                int k = ((lane % CPR) ^ ((r & 7) << 1)) * 16;
                if (pt.col0 + k >= p.K) k = p.K - 16 - pt.col0;  // (columns that are not stored)
                boff[c] = (uint32_t)r * (uint32_t)p.K + k;
            }
        }
        start_term(0);
    };
    start_tile();

    // The copies of one step.
    auto issue = [&]() {
        if (DX && pstep == steps_of_term) start_term(1);
        const int b = DX && pstep >= steps_of_term ? pstep - steps_of_term : pstep;
        const uint32_t st = lds0 + pstage * S::kStage;
#pragma unroll
        for (int c = 0; c < S::kACopies; ++c) copy16(abase, aoff[c], st + (wave * S::kACopies + c) * 1024);
        abase += 128;
        // (gated: the upper half of the waves copies the second matrix)
        const uint8_t *bb = bbase;
        if (GLU && wave >= kWaves / 2) bb += p.w[1].q - p.w[0].q;
        const bool partial = red % kFp8Block != 0 && b == steps_of_term - 1;
        if (!partial) {
#pragma unroll
            for (int c = 0; c < S::kBCopies; ++c) copy16(bb, boff[c], st + S::kA + (wave * S::kBCopies + c) * 1024);
        } else {
            // the last, partial block of the reduction: zeros behind its end (the rows have zeros there, but 0 * NaN is NaN)
#pragma unroll
            for (int c = 0; c < S::kBCopies; ++c) {
                const int load = wave * S::kBCopies + c;
                const int r = DX ? (load * 64 + lane) / (BN / 16) : load * 8 + (lane >> 3);
                const int at = b * kFp8Block + (DX ? r : ((lane & 7) ^ ((r >> 1) & 7)) * 16);
                copy16(at < red ? bb + boff[c] : (const uint8_t *)&g_fp8_zeros, st + S::kA + load * 1024);
            }
        }
        bbase += DX ? (int64_t)128 * p.K : 128;
        if (lane < S::kSLanes + (GLU ? 2 : 1)) copy4(sptr, st + S::kA + S::kB + wave * S::kSWave);
        sptr += lane >= S::kSLanes ? (DX ? kbk * 4 : 4) : (b & 3) == 3 ? 4 : 0;
        if (++pstage == STAGES) pstage = 0;
        if (++pstep == KT) {
            pstep = 0;
            pt.index += stride;
            if (pt.index < last) {
                decode(pt);
                start_tile();
            } else {
                more = false;
            }
        }
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        if (more) issue();

    // ---- the consumer's side
    // (a wave's row blocks are dealt in turn, so that a tile of few blocks keeps all rows of waves at work)
    const int acol0 = GLU ? wn * 32 : wn * NI * 32;
    static_assert(32 % S::kSLanes == 0 || S::kSLanes % 32 == 0, "a row block's scales: whole regions, or one part");
    // Where the lane's fragments lie in a stage; sub-steps and pieces are an exclusive or of the address's chunk bits away,
    // blocks of rows and columns a constant.
    const uint32_t swizzled = (half ^ ((l >> 1) & 7)) * 16;
    const uint32_t xoff = (wm * 32 + l) * 128 + swizzled;
    const int first_row = wm * 32 + l;
    const uint32_t soff = S::kA + S::kB + first_row / S::kSLanes * S::kSWave + first_row % S::kSLanes * 4;
    uint32_t woff;
    if (!DX) {
        woff = S::kA + (acol0 + l) * 128 + swizzled;
    } else {
        const int g = lane >> 4, il = lane & 15;
        woff = S::kA + ((g >> 1) * 16 + (il >> 1)) * BN + (((acol0 >> 4) + (g & 1)) ^ ((il >> 1) << 1)) * 16 + (il & 1) * 8;
    }
    int cstage = 0;
    while (true) {
        floatx16 acc[MI][NI];
        const int blocks = (cur.rows + 31) / 32;
        // the steps of a tile whose waves have `rb` row blocks each (the last wave row one less)
        auto steps = [&](auto rb) {
        constexpr int RB = decltype(rb)::value;
#pragma unroll
        for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;
        for (int step = 0; step < KT; ++step) {
            const int b = DX && step >= steps_of_term ? step - steps_of_term : step;
            if (more || step + STAGES - 2 < KT - 1) publish<(STAGES - 2) * S::kOps>();
            else publish<0>();
            if (more) issue();
            const uint32_t st = lds0 + cstage * S::kStage;
            float wscale[2];
#pragma unroll
            for (int j = 0; j < (GLU ? 2 : 1); ++j) wscale[j] = *(lds_float_ptr)(uintptr_t)(st + S::kA + S::kB + wave * S::kSWave + (S::kSLanes + j) * 4);
            union Frag {
                uint4_t v[2];
                intx2 t[4];
                intx8 i;
            };
            Frag fw[NI][2];
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (!DX) {
                        constexpr int kNext = GLU ? BNC * 128 : 32 * 128;  // to the wave's next block of columns
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            fw[j][s].v[u] = *(lds_uint4_ptr)(uintptr_t)(((st + woff) ^ (64 * s + 32 * u)) + j * kNext);
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            fw[j][s].t[q] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                (lds_intx2_ptr)(uintptr_t)(((st + woff) ^ (32 * j)) + (s * 64 + (q >> 1) * 32 + (q & 1) * 8) * BN));
                    }
                }
            // The matrix unit never waits for the additions: a block's partial sum is added to its running sum while the next
            // block's second half, or the next row block's first, is multiplied.  A row block's fragments of a sub-step are
            // asked for as soon as those of the row block before have gone into the unit.
            Frag fa[2];
            int xscale[2];
            auto fetch = [&](int i, int s) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    fa[s].v[u] = *(lds_uint4_ptr)(uintptr_t)(((st + xoff) ^ (64 * s + 32 * u)) + i * WM * 32 * 128);
            };
            auto fetch_scale = [&](int i) {
                xscale[i & 1] = (int)(*(lds_uint32_ptr)(uintptr_t)(st + soff + i * WM * 32 / S::kSLanes * S::kSWave) >> ((b & 3) * 8));
            };
            floatx16 part[NI];
            auto multiply = [&](int i, int s, int j) {
                if (s == 0) {
#pragma unroll
                    for (int q = 0; q < 16; ++q) part[j][q] = 0.0f;
                }
                part[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[j][s].i, fa[s].i, part[j], 0, 0, 0, 127, 0, xscale[i & 1]);
            };
            auto add = [&](int i, int j) {
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[i][j][q] = __builtin_fmaf(wscale[GLU ? j : 0], part[j][q], acc[i][j][q]);
            };
            fetch(0, 0);
            fetch_scale(0);
            fetch(0, 1);
#pragma unroll
            for (int i = 0; i < RB; ++i) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
#pragma unroll
                    for (int j = 0; j < NI; ++j) {
                        multiply(i, s, j);
                        __builtin_amdgcn_sched_barrier(0);
                        if (s == 0 && j == 0 && i > 0) {
                            add(i - 1, NI - 1);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                    if (i + 1 < RB) {
                        fetch(i + 1, s);
                        if (s == 0) fetch_scale(i + 1);
                    }
                }
#pragma unroll
                for (int j = 0; j < NI - 1; ++j) add(i, j);
                __builtin_amdgcn_sched_barrier(0);
            }
            add(RB - 1, NI - 1);
            if (++cstage == STAGES) cstage = 0;
        }
        };
        const int mine = (blocks + WM - 1) / WM;
        if constexpr (MI >= 4)
            if (mine == 4) steps(std::integral_constant<int, 4>{});
        if constexpr (MI >= 3)
            if (mine == 3) steps(std::integral_constant<int, 3>{});
        if constexpr (MI >= 2)
            if (mine == 2) steps(std::integral_constant<int, 2>{});
        if (mine == 1) steps(std::integral_constant<int, 1>{});

        // ---- output: a lane's runs of four columns, joined to eight with the other half of the wave
        auto store = [&](void *base, int64_t at, const float (&v)[16], int n0) {
#pragma unroll
            for (int t = 0; t < 4; t += 2) {
                union {
                    TO e[4];
                    uint32_t u[2];
                } a, bq;
#pragma unroll
                for (int q = 0; q < 4; ++q) a.e[q] = from_f32<TO>(v[4 * t + q]), bq.e[q] = from_f32<TO>(v[4 * t + 4 + q]);
                const auto x0 = __builtin_amdgcn_permlane32_swap(a.u[0], bq.u[0], false, false);
                const auto x1 = __builtin_amdgcn_permlane32_swap(a.u[1], bq.u[1], false, false);
                const int n = n0 + 8 * (t + half);
                TO *dst = (TO *)base + at + n;
                const uint4_t out = {x0[0], x1[0], x0[1], x1[1]};
                if (cols % 8 == 0) {
                    if (n < cols) *(uint4_t *)dst = out;
                } else {
                    union {
                        uint4_t v;
                        TO e[8];
                    } u;
                    u.v = out;
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (n + q < cols) dst[q] = u.e[q];
                }
            }
        };
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int r = (i * WM + wm) * 32 + l;
            if (i * WM + wm < blocks) {
                const bool live = r < cur.rows;
                const int64_t at = (int64_t)(cur.row0 + r) * cols;
                if (GLU) {
                    const int n0 = cur.col0 + acol0;
                    float e[16], g[16], v[16];
#pragma unroll
                    for (int q = 0; q < 16; ++q) {
                        e[q] = acc[i][0][q], g[q] = acc[i][NI - 1][q];
                        v[q] = e[q] * sigmoid_f32(e[q]) * g[q];
                    }
                    if (p.e_out != nullptr && live) store(p.e_out, at, e, n0);
                    if (p.g_out != nullptr && live) store(p.g_out, at, g, n0);
                    if (!HQ) {
                        if (live) store(p.out, at, v, n0);
                    } else {
                        float a = 0.0f;
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            if (n0 + 8 * (q / 4) + 4 * half + q % 4 >= cols) v[q] = 0.0f;  // (the padding of the rows)
                            a = __builtin_fmaxf(a, fp8_finite_abs(v[q]));
                            acc[i][0][q] = v[q];
                        }
                        a = __builtin_fmaxf(a, __shfl_xor(a, 32));
                        if (half == 0) amax[r * WN + wn] = a;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < NI; ++j) {
                        float v[16];
#pragma unroll
                        for (int q = 0; q < 16; ++q) v[q] = acc[i][j][q];
                        if (live) store(p.out, at, v, cur.col0 + acol0 + j * 32);
                    }
                }
            }
        }
        if (HQ) {
            // a row's 128 columns are with the WN waves of its wave row: the largest magnitude goes through LDS
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
            const int64_t ldh = fp8_ld(cols), ldh_scale = fp8_ld_scale(cols);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int r = (i * WM + wm) * 32 + l;
                if (i * WM + wm < blocks && r < cur.rows) {
                    float a = 0.0f;
#pragma unroll
                    for (int w = 0; w < WN; ++w) a = __builtin_fmaxf(a, amax[r * WN + w]);
                    const int byte = fp8_scale_byte(a);
                    const float inverse = fp8_inverse_of(byte);
                    uint8_t *dst = p.hq + (cur.row0 + r) * ldh + cur.col0 + acol0;
                    if (wn == 0 && half == 0) p.hq_scale[(cur.row0 + r) * ldh_scale + cur.col0 / kFp8Block] = (uint8_t)byte;
#pragma unroll
                    for (int t = 0; t < 4; t += 2) {
                        const floatx16 &v = acc[i][0];
                        const uint32_t x = fp8_pack4(v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3], inverse);
                        const uint32_t y = fp8_pack4(v[4 * t + 4], v[4 * t + 5], v[4 * t + 6], v[4 * t + 7], inverse);
                        const auto z = __builtin_amdgcn_permlane32_swap(x, y, false, false);
                        *(uint2_t *)(dst + 8 * (t + half)) = uint2_t{z[0], z[1]};
                    }
                }
            }
        }
        cur.index += stride;
        if (cur.index >= last) break;
        decode(cur);
    }
}

template <bool DX, bool GLU, bool HQ, int WM, int WN, int MI, int NI, int STAGES, typename TO>
int launch(const Fp8Product &p, hipStream_t stream) {
    using S = Shape<WM, WN, MI, NI, STAGES>;
    constexpr int kLds = S::kLds + (HQ ? S::BM * WN * 4 : 0);
    static_assert(kLds <= 160 * 1024, "a CU's LDS");
    constexpr int kPerCu = 160 * 1024 / kLds < 2 ? 1 : 2;
    auto kern = fp8_tile_kernel<DX, GLU, HQ, WM, WN, MI, NI, STAGES, TO>;
    static PerDeviceOnce once;
    const hipError_t e = once.run([&] {
        return hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    });
    if (e != hipSuccess) return (int)e;
    const int grid = device_info().cu_count / kXcd * kXcd * kPerCu;
    kern<<<grid, kThreads, kLds, stream>>>(p);
    return launch_status();
}

template <int WM, int WN, int MI, int NI, int STAGES, typename TO>
int launch_mode(const Fp8Product &p, hipStream_t stream) {
    if (p.dx) return launch<true, false, false, WM, WN, MI, NI, STAGES, TO>(p, stream);
    if (p.glu) return p.hq != nullptr ? launch<false, true, true, WM, WN, MI, NI, STAGES, TO>(p, stream)
                                        : launch<false, true, false, WM, WN, MI, NI, STAGES, TO>(p, stream);
    return launch<false, false, false, WM, WN, MI, NI, STAGES, TO>(p, stream);
}

template <typename TO>
int launch_shape(const Fp8Product &p, hipStream_t stream) {
    return launch_mode<2, 4, 4, 2, 2, TO>(p, stream);
}

}  // namespace

int gemm_fp8_tile(const Fp8Product &p, hipStream_t stream) {
    if (p.out_dtype == MFL_F32 || p.K % 16 != 0 || p.E > kMaxExperts) return MFL_ERR_UNSUPPORTED;
    const int cols = p.dx ? p.K : p.N, red = p.dx ? p.N : p.K;
    for (int i = 0; i < (p.glu || p.terms == 2 ? 2 : 1); ++i)
        if (!aligned(p.w[i].q, 16)) return MFL_ERR_UNSUPPORTED;
    if (cols % 8 == 0 && (!aligned(p.out, 16) || !aligned(p.e_out, 16) || !aligned(p.g_out, 16))) return MFL_ERR_UNSUPPORTED;
    // 32-bit offsets of a lane: 256 rows (or all, gathered) of the left operand, 256 of the weights; 32-bit counts of tiles
    if ((p.row_idx != nullptr ? p.src_rows : 256) * fp8_ld(red) > 0xffffffffll || (int64_t)256 * p.K > 0xffffffffll)
        return MFL_ERR_UNSUPPORTED;
    if ((p.R / 64 + p.E) * (int64_t)ceil_div(cols, 64) > 0x3fffffff) return MFL_ERR_UNSUPPORTED;
    return p.out_dtype == MFL_BF16 ? launch_shape<bf16_t>(p, stream) : launch_shape<f16_t>(p, stream);
}

}  // namespace mfl
