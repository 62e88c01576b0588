// Expert products in 8-bit floating point on LDS tiles: weights in rows of whole 16-byte pieces.
//
//   forward         out[r, n] = sum_b S[e, n / 128, b] sx[r, b] sum_{k in block b} x[r, k] w[e, n, k]
//   gated           the same for two matrices, out = silu(gate) * up
//   input gradient  out[r, k] = sum_b S[e, b, k / 128] sd[r, b] sum_{n in block b} d[r, n] w[e, n, k], of one or two terms
//
// A workgroup of four or eight waves owns a tile of BM rows and BN columns of one expert and walks the reduction in steps of one scale
// block, 128 bytes of every row.  A stage in LDS is one such step: BM x 128 row bytes, BN x 128 weight bytes, and the dwords
// that hold the rows' scale bytes.  Everything arrives by direct copies (global_load_lds) that the wave counts itself; one
// barrier a step publishes the stage that has landed and frees the one before.  The tiles of a workgroup are one stream of
// steps: the first copies of the next tile go out under the last step of this one.
//
//   v_mfma_scale_f32_32x32x64_f8f6f4, weights first: a lane's 16 accumulators of a 32 x 32 block belong to one row (whose
//   scale it hands to the instruction) and to runs of four columns.  Two instructions make a block's partial sum over a step,
//   16 multiply-adds by the weights' scale (uniform: 128 x 128) add it to the running fp32 sum.
//
// For fp32 outputs and the quantised gated unit in fp16 the fragments are widened to bf16 in registers and multiplied by
// v_mfma_f32_32x32x16_bf16: half the rate, and 16 conversions a fragment (fp8.h says why).
//
// LDS layouts.  Rows of 128 bytes along the reduction: 16-byte chunk c of row r at c ^ ((r >> 1) & 7).  A lane's 32 bytes of a
// 64-wide sub-step are chunks 4 s + h and 4 s + 2 + h (h: its half of the wave); which reduction element sits where in the
// instruction does not matter as long as both operands agree.  Input gradient: the weights lie as in memory, 128 rows of the
// reduction by BN columns, chunk c of row n at c ^ ((n & 7) << 1) (BN 128: c ^ (n & 6)), and are read with ds_read_b64_tr_b8 (a group of 16 lanes
// reads 8 rows of 16 bytes and gets 8 rows of one column each), four of them for the same 32 elements.
#include <type_traits>

#include "fp8.h"

namespace mfl {

namespace {

typedef __attribute__((address_space(3))) void *lds_void_ptr;
typedef __attribute__((address_space(3))) intx2 *lds_intx2_ptr;
typedef const __attribute__((address_space(3))) uint4_t *lds_uint4_ptr;
typedef const __attribute__((address_space(3))) uint32_t *lds_uint32_ptr;
typedef const __attribute__((address_space(3))) float *lds_float_ptr;

constexpr int kXcd = 8;
constexpr int kMaxExperts = 512;  // prefix tables in LDS

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

// The same behind a tile's output: the `newer` stores that the wave has issued since the copies it waits for need not have
// landed (the counter retires in order).
template <int N>
__device__ __forceinline__ void publish_past(int newer) {
    static_assert(N >= 0 && N + 16 < 64, "vmcnt is a 6-bit counter");
    asm volatile(
        "s_cmp_ge_u32 %0, 16\n\ts_cbranch_scc1 1f\n\ts_cmp_ge_u32 %0, 8\n\ts_cbranch_scc1 2f\n\ts_cmp_ge_u32 %0, 4\n\ts_cbranch_scc1 3f\n\t"
        "s_waitcnt vmcnt(%1) lgkmcnt(0)\n\ts_branch 4f\n"
        "1:\n\ts_waitcnt vmcnt(%2) lgkmcnt(0)\n\ts_branch 4f\n"
        "2:\n\ts_waitcnt vmcnt(%3) lgkmcnt(0)\n\ts_branch 4f\n"
        "3:\n\ts_waitcnt vmcnt(%4) lgkmcnt(0)\n"
        "4:\n\ts_barrier"
        :
        : "s"(__builtin_amdgcn_readfirstlane(newer)), "n"(N), "n"(N + 16), "n"(N + 8), "n"(N + 4)
        : "memory", "scc");
}

// WM x WN waves of MI x NI blocks of 32 x 32.
template <int WM, int WN, int MI, int NI, int STAGES>
struct Shape {
    static constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
    static constexpr int BM = WM * MI * 32, BN = WN * NI * 32;
    static constexpr int kSLanes = BM / kWaves;                    // rows whose scale dwords a wave copies,
    static constexpr int kSWave = 64 * 4;                          // and behind them the weights' scales of its columns
    static constexpr int kA = BM * 128, kB = BN * 128, kS = kWaves * kSWave;
    static constexpr int kStage = (kA + kB + kS + 1023) / 1024 * 1024;
    static constexpr int kACopies = kA / 1024 / kWaves, kBCopies = kB / 1024 / kWaves;
    static constexpr int kOps = kACopies + kBCopies + 1;  // vector-memory operations a wave issues for a stage
    static constexpr int kTables = (2 * (kMaxExperts + 1) * 4 + 127) / 128 * 128;
    static constexpr int kLds = STAGES * kStage + kTables;
    static_assert(kA % (1024 * kWaves) == 0 && kB % (1024 * kWaves) == 0 && kSLanes + 2 <= 64, "whole copies");
};

// HQ: the gated unit's result leaves as quantised rows.  PARTIAL: the reduction ends inside a block of 128.
template <bool DX, bool GLU, bool HQ, bool PARTIAL, int WM, int WN, int MI, int NI, int STAGES, typename TO>
__global__ __launch_bounds__(WM * WN * 64, 2) void fp8_tile_kernel(Fp8Product p) {
    using S = Shape<WM, WN, MI, NI, STAGES>;
    constexpr int BM = S::BM, BN = S::BN, kWaves = S::kWaves;
    constexpr int BNC = GLU ? BN / 2 : BN;  // output columns of a tile
    constexpr bool kF32 = sizeof(TO) == 4;
    constexpr bool kBf16 = kF32 || (HQ && std::is_same<TO, f16_t>::value);  // bf16 products
    static_assert(!GLU || NI == 2, "gated: a wave holds one block of either matrix");
    static_assert(!HQ || (GLU && BNC == kFp8Block), "quantised output: a tile's columns are one scale block");
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    int *const tab_rows = (int *)(smem + STAGES * S::kStage);
    int *const tab_tiles = tab_rows + kMaxExperts + 1;
    uint32_t *const amax = (uint32_t *)(smem + S::kLds);  // (HQ) per row and wave column
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

    // (DX) which chunks of a row of the reduction are exchanged, by its number: eight rows' pieces of 32 bytes in all 64 banks
    static_assert(!DX || BN == 128 || BN == 256, "rows of half or all of the banks");
    auto spread = [](int n) { return BN == 128 ? ((n >> 1) & 3) << 1 : (n & 7) << 1; };

    // ---- rows and row tiles before every expert, cut at row R; an expert's rows come in tiles of equal height, a multiple of 32
    {
        int row_carry = 0, tile_carry = 0;
        for (int e0 = 0; e0 < p.E; e0 += 64) {
            const int e = e0 + lane;
            uint32_t count[1];
            fp8_load_counts(p.m_sizes, p.ms_i64, e, p.E, p.R, count);
            const Fp8Counted c = fp8_cut(count[0], (uint32_t)p.R - (uint32_t)row_carry);
            const int t = fp8_tiles_of(c.end - c.begin, BM), ti = wave_inclusive_scan(t);
            if (wave == 0 && e < p.E) tab_rows[e] = row_carry + c.begin, tab_tiles[e] = tile_carry + ti - t;
            row_carry += c.all, tile_carry += wave_last(ti);
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
    // The lane, for what is computed once a tile: taken from here, its terms are not kept in registers through the steps.
    auto lane_now = [&]() {
        int now = lane;
        asm volatile("" : "+v"(now));
        return now;
    };
    auto decode = [&](Tile &t) {
        const int lane = lane_now();
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
    Tile pt = cur, nt = cur;  // the producer's tile, and the one it takes up next
    int pstep = 0, pstage = 0;
    // (rows that are not gathered are addressed from the tile's first one; gathered ones from the first of all, within 32 bits)
    const bool gathered = !DX && p.row_idx != nullptr;
    uint32_t aoff[S::kACopies], boff[S::kBCopies];
    const uint8_t *sptr;  // the lane's scale dword: of a row, or of the weights
    int src_row = 0;
    const uint8_t *abase, *bbase;
    // Lane i of a wave looks up the source of row i of the wave's BM / 8 rows when the tile is known, several steps before
    // its first copies.
    int looked_up = 0;
    auto look_up = [&]() {
        const int lane = lane_now();
        const int r = wave * S::kSLanes + (S::kSLanes >= 64 ? lane : lane % S::kSLanes);
        looked_up = r < nt.rows ? r : nt.rows - 1;
        if (gathered) looked_up = p.row_idx[nt.row0 + looked_up];
    };
    // column block of the weights' scales of the wave's columns (which lie in one: 64 or 32 columns from a multiple of that)
    auto scale_block = [&](const Tile &t) {
        const int at = (t.col0 + (GLU ? wn * 32 : wn * NI * 32)) / kFp8Block, end = DX ? kbk : nbn;
        return at < end ? at : end - 1;
    };
    auto start_tile = [&]() {
        const int lane = lane_now();
        pt = nt, pstep = 0;
        src_row = looked_up;
        if (gathered) {
            src_row /= p.idx_div;
            src_row = src_row < 0 ? 0 : src_row >= (int)p.src_rows ? (int)p.src_rows - 1 : src_row;
        }
#pragma unroll
        for (int c = 0; c < S::kACopies; ++c) {
            const int r = (wave * S::kACopies + c) * 8 + (lane >> 3);
            aoff[c] = (uint32_t)__shfl(src_row, c * 8 + (lane >> 3)) * (uint32_t)lda + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
        }
#pragma unroll
        for (int c = 0; c < S::kBCopies; ++c) {
            const int load = wave * S::kBCopies + c;
            if (!DX) {
                const int r = load * 8 + (lane >> 3);
                int n = GLU ? r % BNC : r;
                if (pt.col0 + n >= p.N) n = p.N - 1 - pt.col0;  // (columns that are not stored)
                boff[c] = (uint32_t)n * (uint32_t)p.ldw + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
            } else {
                constexpr int CPR = BN / 16;  // chunks of a row of the reduction
                const int r = (load * 64 + lane) / CPR;
                int k = ((lane % CPR) ^ spread(r)) * 16;
                if (pt.col0 + k >= p.ldw) k = p.ldw - 16 - pt.col0;  // (columns that are not stored)
                boff[c] = (uint32_t)r * (uint32_t)p.ldw + k;
            }
        }
        const Fp8Rows a = p.a[0];
        const int64_t first = gathered ? 0 : pt.row0, mat = (int64_t)pt.expert * p.N * p.ldw;
        abase = a.q + first * lda;
        bbase = p.w[0].q + mat + (DX ? pt.col0 : (int64_t)pt.col0 * p.ldw);
        const float *ws = (GLU && lane > S::kSLanes ? p.w[1].scale : p.w[0].scale) + (int64_t)pt.expert * nbn * kbk;
        ws += DX ? scale_block(pt) : (int64_t)scale_block(pt) * kbk;
        sptr = lane < S::kSLanes ? a.scale + (first + src_row) * lds_ : (const uint8_t *)ws;
    };
    // The copies of one step.  Without a branch, so that the compiler leaves the order of the steps' arithmetic alone.
    auto issue = [&]() {
        const int b = DX && pstep >= steps_of_term ? pstep - steps_of_term : pstep;
        const uint32_t st = lds0 + pstage * S::kStage;
#pragma unroll
        for (int c = 0; c < S::kACopies; ++c) copy16(abase, aoff[c], st + (wave * S::kACopies + c) * 1024);
        // (gated: the upper half of the waves copies the second matrix)
        const uint8_t *bb = bbase;
        if (GLU) bb += wave >= kWaves / 2 ? p.w[1].q - p.w[0].q : 0;
#pragma unroll
        for (int c = 0; c < S::kBCopies; ++c) {
            const int load = wave * S::kBCopies + c;
            if (!PARTIAL) {
                copy16(bb, boff[c], st + S::kA + load * 1024);
            } else {
                // zeros behind the end of the reduction (the rows have zeros there, but 0 * NaN is NaN)
                const int r = DX ? (load * 64 + lane) / (BN / 16) : load * 8 + (lane >> 3);
                const int at = b * kFp8Block + (DX ? r : ((lane & 7) ^ ((r >> 1) & 7)) * 16);
                copy16(at < red ? bb + boff[c] : (const uint8_t *)&g_fp8_zeros, st + S::kA + load * 1024);
            }
        }
        copy4(sptr, st + S::kA + S::kB + wave * S::kSWave);
        int64_t a_step = 128, b_step = DX ? (int64_t)128 * p.ldw : 128, row_step = (b & 3) == 3 ? 4 : 0, w_step = DX ? kbk * 4 : 4;
        if (DX) {
            // to the second term's operands
            const bool jump = pstep + 1 == steps_of_term && p.terms == 2;
            a_step = jump ? p.a[1].q - p.a[0].q - (int64_t)(steps_of_term - 1) * 128 : a_step;
            b_step = jump ? p.w[1].q - p.w[0].q - (int64_t)(steps_of_term - 1) * 128 * p.ldw : b_step;
            row_step = jump ? p.a[1].scale - p.a[0].scale - (steps_of_term - 1) / 4 * 4 : row_step;
            w_step = jump ? (const uint8_t *)p.w[1].scale - (const uint8_t *)p.w[0].scale - (int64_t)(steps_of_term - 1) * kbk * 4 : w_step;
        }
        abase += a_step, bbase += b_step;
        sptr += lane >= S::kSLanes ? w_step : row_step;
        pstage = pstage + 1 == STAGES ? 0 : pstage + 1;
        ++pstep;
    };
    // (a tile has at least as many steps as there are stages)
    look_up();
    start_tile();
#pragma unroll
    for (int i = 0; i < STAGES; ++i) issue();
    publish<(STAGES - 1) * S::kOps>();

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
        woff = S::kA + ((g >> 1) * 16 + (il >> 1)) * BN + (((acol0 >> 4) + (g & 1)) ^ spread(il >> 1)) * 16 + (il & 1) * 8;
    }
    int cstage = 0, newer = 0;
    while (true) {
        floatx16 acc[MI][NI];
        const int blocks = (cur.rows + 31) / 32;
        nt.index = cur.index + stride;
        const bool follows = nt.index < last;
        if (follows) decode(nt);
        else nt = cur;
        look_up();
        // the steps of a tile of which this wave has `rb` row blocks (others may have one less: what the waves of a workgroup have
        // to agree in is the number of barriers, one a step)
        auto steps = [&](auto rb) {
            constexpr int RB = decltype(rb)::value;
#pragma unroll
            for (int i = 0; i < RB; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
#pragma unroll
                    for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;
            union Frag {
                uint4_t v[2];
                intx2 t[4];
                intx8 i;
            };
            Frag fw[NI][2], fa[2];
            int xscale[2];
            float wscale[2], wlast = 0.0f;  // the weights' scales of this step, and of the last one's last block
            floatx16 part[NI];
            uint32_t st = lds0 + cstage * S::kStage;
            auto fetch_w = [&](int s) {
#pragma unroll
                for (int j = 0; j < NI; ++j) {
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
            };
            auto fetch_scales = [&]() {
#pragma unroll
                for (int j = 0; j < (GLU ? 2 : 1); ++j)
                    wscale[j] = *(lds_float_ptr)(uintptr_t)(st + S::kA + S::kB + wave * S::kSWave + (S::kSLanes + j) * 4);
            };
            auto fetch = [&](int i, int s) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    fa[s].v[u] = *(lds_uint4_ptr)(uintptr_t)(((st + xoff) ^ (64 * s + 32 * u)) + i * WM * 32 * 128);
            };
            auto fetch_scale = [&](int i, int b) {
                xscale[i & 1] = (int)(*(lds_uint32_ptr)(uintptr_t)(st + soff + i * WM * 32 / S::kSLanes * S::kSWave) >> ((b & 3) * 8));
            };
            auto multiply = [&](int i, int s, int j) {
                if (s == 0) {
#pragma unroll
                    for (int q = 0; q < 16; ++q) part[j][q] = 0.0f;
                }
                if constexpr (!kBf16) {
                    part[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[j][s].i, fa[s].i, part[j], 0, 0, 0, 127, 0, xscale[i & 1]);
                } else {
                    const float row_scale = fp8_scale_of(xscale[i & 1] & 255);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        part[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fp8_widen(fw[j][s].t[q], 1.0f), fp8_widen(fa[s].t[q], row_scale), part[j], 0, 0, 0);
                }
            };
            auto add = [&](int i, int j, float scale) {
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[i][j][q] = __builtin_fmaf(scale, part[j][q], acc[i][j][q]);
            };
            // The matrix unit never waits for the additions: a block's partial sum is added to its running sum while the next block's
            // second half, or the next row block's first, is multiplied.  A row block's fragments of a sub-step are asked for as soon
            // as those of the row block before have gone into the unit, those of the next step behind the barrier, which lies before
            // the step's last sub-step.
#pragma unroll
            for (int q = 0; q < 16; ++q) part[NI - 1][q] = 0.0f;
            fetch_w(0);
            fetch(0, 0);
            fetch_scale(0, 0);
            fetch_scales();
            fetch_w(1);
            fetch(0, 1);
            // (the last steps' copies are the next tile's first; behind the last tile this one's again, which nobody reads)
            int step = 0;
            for (int end = KT - STAGES; step < KT; end = KT) {
                if (step == KT - STAGES) start_tile();
                for (; step < end; ++step) {
                    const int b = DX && step >= steps_of_term ? step - steps_of_term : step;
#pragma unroll
                    for (int i = 0; i < RB; ++i) {
                        multiply(i, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                        if (i == 0) add(RB - 1, NI - 1, wlast);
                        else add(i - 1, NI - 1, wscale[GLU ? NI - 1 : 0]);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int j = 1; j < NI; ++j) multiply(i, 0, j);
                        __builtin_amdgcn_sched_barrier(0);
                        const int bn = DX && step + 1 >= steps_of_term ? step + 1 - steps_of_term : step + 1;
                        if (i + 1 < RB) {
                            fetch(i + 1, 0);
                            fetch_scale(i + 1, b);
                        } else {
                            wlast = wscale[GLU ? NI - 1 : 0];
                            publish_past<(STAGES - 2) * S::kOps>(newer);
                            newer = 0;
                            cstage = cstage + 1 == STAGES ? 0 : cstage + 1;
                            st = lds0 + cstage * S::kStage;
                            fetch_w(0);  // (behind the last step: of the next tile, or stale; not used)
                        }
#pragma unroll
                        for (int j = 0; j < NI; ++j) multiply(i, 1, j);
                        __builtin_amdgcn_sched_barrier(0);
                        if (i + 1 < RB) {
                            fetch(i + 1, 1);
#pragma unroll
                            for (int j = 0; j < NI - 1; ++j) add(i, j, wscale[GLU ? j : 0]);
                        } else {
                            issue();
#pragma unroll
                            for (int j = 0; j < NI - 1; ++j) add(i, j, wscale[GLU ? j : 0]);
                            fetch(0, 0);
                            fetch_scale(0, bn);
                            fetch_w(1);
                            fetch(0, 1);
                            fetch_scales();
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            add(RB - 1, NI - 1, wlast);
        };
        // a wave without row blocks in this tile: its part of the copies, and the barriers
        auto no_steps = [&]() {
            int step = 0;
            for (int end = KT - STAGES; step < KT; end = KT) {
                if (step == KT - STAGES) start_tile();
                for (; step < end; ++step) {
                    publish_past<(STAGES - 2) * S::kOps>(newer);
                    newer = 0;
                    cstage = cstage + 1 == STAGES ? 0 : cstage + 1;
                    issue();
                }
            }
        };
        const int mine = (blocks - wm + WM - 1) / WM;
        if constexpr (MI >= 4)
            if (mine == 4) steps(std::integral_constant<int, 4>{});
        if constexpr (MI >= 3)
            if (mine == 3) steps(std::integral_constant<int, 3>{});
        if constexpr (MI >= 2)
            if (mine == 2) steps(std::integral_constant<int, 2>{});
        if (mine == 1) steps(std::integral_constant<int, 1>{});
        if (mine == 0) no_steps();

        // ---- output.  A lane holds runs of four columns of one row, joined to eight with the other half of the wave.  (Turned in
        // LDS first, so that whole lines of a row leave at once, the output took as long or longer: 43 against 39 thousand
        // clocks for a tile of six steps.  Streaming stores: 159 against 148 us for the forward product of 32768 rows.)
        auto store16 = [&](void *base, int64_t row, int n, const uint4_t v) {
            TO *dst = (TO *)base + row * cols + n;
            if (cols % 8 == 0) {
                if (n < cols) *(uint4_t *)dst = v;
            } else {
                union {
                    uint4_t v;
                    TO e[8];
                } u;
                u.v = v;
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (n + q < cols) dst[q] = u.e[q];
            }
        };
        auto pack = [&](const float (&v)[4]) {
            union {
                TO e[4];
                uint2_t u;
            } a;
#pragma unroll
            for (int q = 0; q < 4; ++q) a.e[q] = from_f32<TO>(v[q]);
            return a.u;
        };
        // 32 columns of a row block from the wave's column n0 on, from f(q), the lane's q-th value
        auto store_block = [&](void *base, int i, auto f, int n0) {
            const int r = (i * WM + wm) * 32 + l;
            if constexpr (kF32) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int n = cur.col0 + acol0 + n0 + 8 * t + 4 * half;
                    float *dst = (float *)base + (int64_t)(cur.row0 + r) * cols + n;
                    const floatx4 v = {f(4 * t), f(4 * t + 1), f(4 * t + 2), f(4 * t + 3)};
                    if (r >= cur.rows) continue;
                    if (cols % 4 == 0) {
                        if (n < cols) *(floatx4 *)dst = v;
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (n + q < cols) dst[q] = v[q];
                    }
                }
                return;
            }
#pragma unroll
            for (int t = 0; t < 4; t += 2) {
                const float va[4] = {f(4 * t), f(4 * t + 1), f(4 * t + 2), f(4 * t + 3)};
                const float vb[4] = {f(4 * t + 4), f(4 * t + 5), f(4 * t + 6), f(4 * t + 7)};
                const uint2_t a = pack(va), b = pack(vb);
                const auto x0 = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
                const auto x1 = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
                if (r < cur.rows) store16(base, cur.row0 + r, cur.col0 + acol0 + n0 + 8 * (t + half), uint4_t{x0[0], x1[0], x0[1], x1[1]});
            }
        };
        // (whole row blocks only: what is issued for certain)
        int whole = (cur.rows / 32 - wm + WM - 1) / WM;
        if (whole < 0 || cols % BNC != 0) whole = 0;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            if (i * WM + wm < blocks) {
                if (GLU) {
                    if (p.e_out != nullptr) store_block(p.e_out, i, [&](int q) { return acc[i][0][q]; }, 0);
                    if (p.g_out != nullptr) store_block(p.g_out, i, [&](int q) { return acc[i][NI - 1][q]; }, 0);
#pragma unroll
                    for (int q = 0; q < 16; ++q) acc[i][0][q] = acc[i][0][q] * sigmoid_f32(acc[i][0][q]) * acc[i][NI - 1][q];
                    if (!HQ) {
                        store_block(p.out, i, [&](int q) { return acc[i][0][q]; }, 0);
                    } else {
                        uint32_t a = 0u;
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            if (cols % kFp8Block != 0 && cur.col0 + acol0 + 8 * (q / 4) + 4 * half + q % 4 >= cols) acc[i][0][q] = 0.0f;  // (the rows' padding)
                            a = fp8_wider(a, acc[i][0][q]);
                        }
                        if (__any(fp8_unusual(a))) {
                            a = 0u;
#pragma unroll
                            for (int q = 0; q < 16; ++q) a = fp8_wider(a, fp8_finite_abs(acc[i][0][q])), acc[i][0][q] = fp8_finite(acc[i][0][q]);
                        }
                        const uint32_t other = (uint32_t)__shfl_xor((int)a, 32);
                        if (half == 0) amax[((i * WM + wm) * 32 + l) * WN + wn] = a > other ? a : other;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < NI; ++j) store_block(p.out, i, [&](int q) { return acc[i][j][q]; }, j * 32);
                }
            }
        }
        newer = GLU ? whole * 2 * ((HQ ? 0 : 1) + (p.e_out != nullptr) + (p.g_out != nullptr)) : whole * 4;
        if (kF32) newer *= 2;
        if (HQ) {
            // a row's 128 columns are with the WN waves of its wave row: the largest magnitude goes through LDS
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
            const int64_t ldh = fp8_ld(cols), ldh_scale = fp8_ld_scale(cols);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int r = (i * WM + wm) * 32 + l;
                if (i * WM + wm < blocks && r < cur.rows) {
                    uint32_t a = 0u;
#pragma unroll
                    for (int w = 0; w < WN; ++w) a = a > amax[r * WN + w] ? a : amax[r * WN + w];
                    const int byte = fp8_scale_byte(a);
                    const float inverse = fp8_inverse_of(byte);
                    uint8_t *const dst = p.hq + (cur.row0 + r) * ldh + cur.col0 + acol0;
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
        if (!follows) break;
        cur = nt;
    }
    publish<0>();  // (no copy is on its way into this LDS when the workgroup ends)
}

template <bool DX, bool GLU, bool HQ, bool PARTIAL, int WM, int WN, int MI, int NI, int STAGES, typename TO>
int launch(const Fp8Product &p, hipStream_t stream) {
    using S = Shape<WM, WN, MI, NI, STAGES>;
    constexpr int kLds = S::kLds + (HQ ? S::BM * WN * 4 : 0);
    static_assert(kLds <= 160 * 1024, "a CU's LDS");
    constexpr int kPerCu = 160 * 1024 / kLds < 2 ? 1 : 2;
    auto kern = fp8_tile_kernel<DX, GLU, HQ, PARTIAL, WM, WN, MI, NI, STAGES, TO>;
    static PerDeviceOnce once;
    const hipError_t e = once.run([&] {
        return hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    });
    if (e != hipSuccess) return (int)e;
    const int grid = device_info().cu_count / kXcd * kXcd * kPerCu;
    kern<<<grid, S::kThreads, kLds, stream>>>(p);
    return launch_status();
}

template <bool PARTIAL, int WM, int WN, int MI, int NI, int STAGES, typename TO>
int launch_mode(const Fp8Product &p, hipStream_t stream) {
    if (p.dx) return launch<true, false, false, PARTIAL, WM, WN, MI, NI, STAGES, TO>(p, stream);
    if (p.glu) return launch<false, true, false, PARTIAL, WM, WN, MI, NI, STAGES, TO>(p, stream);
    return launch<false, false, false, PARTIAL, WM, WN, MI, NI, STAGES, TO>(p, stream);
}

template <typename TO>
int launch_shape(const Fp8Product &p, hipStream_t stream) {
    const int cols = p.dx ? p.K : p.N, red = p.dx ? p.N : p.K;
    const int steps = fp8_blocks(red) * (p.dx ? p.terms : 1);
    const bool partial = red % kFp8Block != 0;
    // Quantised output: the 128 columns of a scale block, of both matrices, are one tile.  Three stages of 128 rows against two of
    // 256: the expert MLP of 131072 rows 947 against 1054 us, of 24008 under Zipf(1) 289 against 330.
    if (p.hq != nullptr) {
        if (steps < 3) return partial ? launch<false, true, true, true, 2, 4, 2, 2, 2, TO>(p, stream) : launch<false, true, true, false, 2, 4, 2, 2, 2, TO>(p, stream);
        return partial ? launch<false, true, true, true, 2, 4, 2, 2, 3, TO>(p, stream) : launch<false, true, true, false, 2, 4, 2, 2, 3, TO>(p, stream);
    }
    // 256 x 256 tiles, one workgroup a CU, where experts have many rows and there are tiles for two rounds; else 128 x 128, two
    // workgroups a CU, whose output and waiting lie under each other's steps.  128 experts, hidden 2048, inner 768, us for
    // 128 / 256, quantisation included: gated unit with products 352 / 343 at 512 rows per expert, 673 / 617 at 1024, its backward
    // pass 376 / 345, 704 / 642, forward product 233 / 226, 440 / 420; but 129 / 141 at 256 rows and 43 / 55 at 32; 8 experts of
    // 1024 rows 35 / 49.
    // (fp32 outputs: 128 x 128)
    const int64_t large = (p.R / 256) * ceil_div(cols, p.glu ? 128 : 256);
    if constexpr (sizeof(TO) == 2)
        if (p.R >= (int64_t)448 * p.E && large >= (int64_t)2 * device_info().cu_count)
            return partial ? launch_mode<true, 2, 4, 4, 2, 2, TO>(p, stream) : launch_mode<false, 2, 4, 4, 2, 2, TO>(p, stream);
    return partial ? launch_mode<true, 2, 2, 2, 2, 2, TO>(p, stream) : launch_mode<false, 2, 2, 2, 2, 2, TO>(p, stream);
}

}  // namespace

bool gemm_fp8_tiles(const Fp8Product &p) {
    if (p.ldw % 16 != 0 || p.E > kMaxExperts) return false;
    const int cols = p.dx ? p.K : p.N, red = p.dx ? p.N : p.K;
    if (fp8_blocks(red) * (p.dx ? p.terms : 1) < 2) return false;  // (a tile has at least as many steps as there are stages)
    for (int i = 0; i < (p.glu || p.terms == 2 ? 2 : 1); ++i)
        if (!aligned(p.w[i].q, 16)) return false;
    if (cols % (p.out_dtype == MFL_F32 ? 4 : 8) == 0 && (!aligned(p.out, 16) || !aligned(p.e_out, 16) || !aligned(p.g_out, 16))) return false;
    // 32-bit offsets of a lane: 256 rows (or all, gathered) of the left operand, 256 of the weights; 32-bit counts of tiles
    if ((p.row_idx != nullptr ? p.src_rows : 256) * fp8_ld(red) > 0xffffffffll || (int64_t)256 * p.ldw > 0xffffffffll) return false;
    return (p.R / 64 + p.E) * (int64_t)ceil_div(cols, 64) <= 0x3fffffff;
}

int gemm_fp8_tile(const Fp8Product &p, hipStream_t stream) {
    if (!gemm_fp8_tiles(p)) return MFL_ERR_UNSUPPORTED;
    MFL_DISPATCH_FLOAT(p.out_dtype, TO, { return launch_shape<TO>(p, stream); });
    return MFL_ERR_DTYPE;
}

}  // namespace mfl
