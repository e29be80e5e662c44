// experts_gemm.hpp -- products grouped by expert with ragged numbers of rows, on the matrix cores:
//   C[r, :] = x[r] W[e]^T  or  C[r, :] = silu(x[r] G[e]^T) * (x[r] U[e]^T),  r in [offsets[e], offsets[e + 1]).
//
// The mathematics.  fp32 rows are taken as 2^e (hi + lo), two fp16 parts under a power of two per row (hi the nearest half,
// lo the nearest half of the rest: 22 bits), weights as the exact integers of experts_formats.hpp, so the products are exact
// in the fp32 accumulators and a result is as good as an fp32 product's.  Two MFMAs per operand pair instead of one, against
// 16 times slower fp32 MFMAs.
//
// Two kernels, one file per weight format.
//
// rows_kernel: a workgroup of four waves takes MT * 32 rows of an expert (16 with PAIR) and, per wave, two tiles of 32
// columns: two column tiles of W, or the same tile of G and U (SiLU * up is then arithmetic on a lane's own registers).
//   * Rows come from the planes that planes_kernel leaves in the workspace (per 64 k: 64 hi, 64 lo), gathered by their
//     token as they are copied to LDS (global_load_lds, one stage of 64 k ahead, one barrier a stage).  Chunk c of 16
//     bytes of row r lies in slot c ^ (r & 15): the reads of 32 rows' operands meet no bank twice.
//   * Weights go from memory to the registers of the one wave that multiplies them, two stages ahead, and are decoded there:
//     nothing of a weight is shared between waves, so LDS would only cost.
//   * Each decoded operand meets MT * 2 MFMAs and each operand read from LDS two.
//   * PAIR (at most 16 rows): lane rows 0 .. 15 hold hi, 16 .. 31 lo of the same rows; one MFMA does both parts, and the
//     two halves of the output are added at the end.
//   * Where workgroups are few and k is long, k goes to several of them, whose products are added up in order afterwards.
// few_kernel: for calls of few tokens, where what counts is how many waves read weights at once: a workgroup takes up to 8
// rows of an expert and one tile of 32 columns, its waves the units along k, each converting the activations of its own
// units to an LDS area of its own (a power of two per row and unit), no barrier before the sum over the waves.
#pragma once

#include <algorithm>
#include <type_traits>

#include "act.hpp"
#include "experts_formats.hpp"

namespace cri {
namespace dev {

typedef _Float16 eh8 __attribute__((ext_vector_type(8)));
typedef float ef16 __attribute__((ext_vector_type(16)));

// first (most significant) operand A: 32 rows, B: 32 columns
__device__ __forceinline__ ef16 e_mfma(eh8 a, const uint32_t (&b)[4], const ef16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, __builtin_bit_cast(eh8, u32x4{b[0], b[1], b[2], b[3]}), c, 0, 0, 0);
}
// 16 bytes per lane from global memory to LDS (lane l at byte 16 l of the wave-uniform lds; below 64 KB).  Not the builtin:
// behind one of those the compiler has every read of LDS wait for the copy, whatever buffer it goes to.  Here the barrier of
// a stage waits; the s_nop is the wait state after writing M0.
__device__ __forceinline__ void e_dma16(const uint8_t* g, uint32_t lds) {
    uint32_t m0;  // kept as the compiler has it
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "v"(g), "s"(lds)
                 : "memory");
}

typedef __attribute__((address_space(3))) char* Lds;
typedef __attribute__((address_space(3))) const eh8* LdsEight;

// output row of register i for lanes below 32 (4 more above)
__device__ __forceinline__ constexpr int e_row(int i) { return (i & 3) + 8 * (i >> 2); }

// the source row of grouped row r
__device__ __forceinline__ long source_row(const ProductArgs& a, int r) {
    return a.gather ? token_of(clamp_int(a.g.rows[r], 0, a.g.R - 1), a.over_k) : r;
}

template <int I>
using Int = std::integral_constant<int, I>;

// Q4_K: acc -= 64 dmin (minimums . sums); sums(m) the operand of the rows' sums
template <int NT, int MT, class X>
__device__ __forceinline__ void subtract_minimums(const typename ExpertFmt<kFmtQ4_K>::Scale (&s)[NT], ef16 (&acc)[NT][MT],
                                                  X&& sums) {
    typedef ExpertFmt<kFmtQ4_K> F;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        uint32_t b[4];
        F::min_operand(s[n], b);
        const float dmin = F::min_scale(s[n]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const ef16 t = e_mfma(sums(m), b, ef16{});
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[n][m][i] = __builtin_fmaf(dmin, t[i], acc[n][m][i]);
            asm volatile("" : "+v"(acc[n][m]));
        }
    }
}

// this wave's loads and copies but the latest LATER have arrived, and every wave is here
template <int LATER>
__device__ __forceinline__ void stage_barrier() { asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(LATER) : "memory"); }

// The loop is laid out so that a wave alone keeps its matrix unit busy, two of them share a SIMD.  A block is two steps (32 k; Q6_K one);
// its NT * MT tiles are slots of 4 MFMAs (half with PAIR and Q6_K), column tile by column tile, and beside the MFMAs of a slot run
//   * the 16 scalings of the slot before, whose sums are whole by then;
//   * decoding: the second column tile of this block in the first half of its slots, the first one of the next block in the other;
//   * the reads of the next block's activations into the registers of a row tile that no later slot of this block needs (MT 2),
//     or into a second set (MT 1).
// The barrier of a stage stands before the last block of the stage before it, when this stage's copies, asked for a stage
// earlier, and its quants, two stages earlier (RING 2: one), have arrived; four buffers of LDS make every buffer's place a constant.
template <int FMT, int MT, bool PAIR, bool SWIGLU>
__global__ __launch_bounds__(256, 2) void rows_kernel(const ProductArgs a) {
    typedef ExpertFmt<FMT> F;
    constexpr int BM = PAIR ? 16 : 32 * MT, LG = PAIR ? 4 : MT == 1 ? 5 : 6, NT = 2, PARTS = PAIR ? 1 : 2;
    constexpr int kStage = BM * 256, kShare = BM / 4, kCopies = kShare / 4;  // bytes of a stage; a wave's rows of it, its copies
    constexpr int kUnit = unit_bytes(FMT);
    // stages of quants in registers, this one's and those on their way (more of Q8_0's spill: 597 us became 636), and the loads that
    // a stage's barrier leaves on their way
    constexpr int RING = FMT == kFmtQ8_0 && MT == 2 ? 2 : 4, kLater = RING == 2 ? 0 : NT * F::kLoads;
    static_assert(!PAIR || MT == 1, "a pair is one tile");
    __shared__ __attribute__((aligned(256))) char ring[4 * kStage + 4 * BM];  // the copies' buffers first: they are below 64 KB
    int* const exps = reinterpret_cast<int*>(ring + 4 * kStage);

    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile t;
    if (!find_tile(a.g, LG, rows_blocks(a.tiles, SWIGLU) * a.splits, blockIdx.x, t)) return;
    const int block = a.splits == 1 ? t.block : t.block / a.splits, split = t.block - block * a.splits;
    const int u0 = a.splits == 1 ? 0 : split * a.depth / a.splits, u1 = a.splits == 1 ? a.depth : (split + 1) * a.depth / a.splits;

    // this wave's column tiles; one past the last is computed again as the last and not stored
    int tile[NT];
    const uint8_t* unit[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        tile[n] = SWIGLU ? block * 4 + wave : block * 8 + wave * 2 + n;
        unit[n] = a.w[SWIGLU ? n : 0] +
                  (static_cast<long>(t.expert) * a.tiles + min(tile[n], a.tiles - 1)) * a.depth * static_cast<long>(kUnit);
    }
    const int stages = (a.K + 63) >> 6;  // a unit's last ones may be nothing but zeros
    // copies: lane l takes slot l & 15 of row l >> 4 of the four rows of a copy
    uint32_t from[kCopies];  // the rows
    const uint32_t row_bytes = a.depth * 1024;
#pragma unroll
    for (int i = 0; i < kCopies; ++i)
        from[i] = source_row(a, t.first + min(wave * kShare + 4 * i + (lane >> 4), t.count - 1));
    const uint32_t ring_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((Lds)ring));
    auto copy = [&](int stage) {  // (past the end: the last stage again, unused)
        const uint8_t* at = a.planes + 256L * min(stage, stages - 1);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int r = wave * kShare + 4 * i + (lane >> 4);
            uint32_t row = from[i];
            asm volatile("" : "+v"(row));  // the address is made here: kept for all rows it would take twice the registers
            e_dma16(at + static_cast<uint64_t>(row) * row_bytes + 16 * ((lane & 15) ^ (r & 15)),
                    ring_at + (stage & 3) * kStage + wave * kShare * 256 + 1024 * i);
        }
    };
    // operands: lane row, and the place of its chunk 2 step + h (hi) or 8 more (lo)
    const int row = PAIR ? lane & 15 : lane & 31, part = PAIR ? 8 * ((lane >> 4) & 1) : 0;
    uint32_t at[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) at[s] = ring_at + row * 256 + 16 * ((2 * s + h + part) ^ (row & 15));
    uint32_t sums[MT];  // the rows' sums: row * depth
    if constexpr (FMT == kFmtQ4_K) {
#pragma unroll
        for (int m = 0; m < MT; ++m) sums[m] = source_row(a, t.first + min(32 * m + row, t.count - 1)) * a.depth;
    }

    ef16 acc[NT][MT] = {};
    typename F::Quant q[RING][NT];  // of stage % RING
    typename F::Scale sc[2][NT];  // this unit's and the next one's
    auto load_quants = [&](typename F::Quant& d, int stage, int n) {
        const int st = min(stage, stages - 1);
        F::load(d, unit[n] + (st >> 2) * static_cast<long>(kUnit), st & 3, lane);
    };
    auto load_scales = [&](typename F::Scale(&d)[NT], int u) {
        const int v = min(u, a.depth - 1);
#pragma unroll
        for (int n = 0; n < NT; ++n) F::load(d[n], unit[n] + v * static_cast<long>(kUnit), lane);
    };
    constexpr int kSets = MT == 1 ? 2 : 1;
    constexpr bool kRagged = FMT != kFmtQ4_K && FMT != kFmtQ6_K;  // K may end inside a unit
    constexpr int STEPS = F::kScaled == kPerStep ? 1 : 2, BLOCKS = 4 / STEPS;  // of a block, of a stage
    eh8 x[kSets][STEPS][PARTS][MT];  // activations: [set][step][part][row tile]
    uint32_t b[NT][STEPS][4];
    eh8 sum[MT];
    // reads of block I of stage J (its buffer: J)
    auto read = [&](auto stage, auto blk, int set, int m) {
        constexpr int J = decltype(stage)::value, I = decltype(blk)::value;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                x[set][s][p][m] = *reinterpret_cast<LdsEight>((at[STEPS * I + s] ^ (128 * p)) + J * kStage + m * 32 * 256);
    };
    auto decode = [&](auto stage, auto step, int n, const typename F::Scale(&scales)[NT]) {
        if constexpr (FMT == kFmtF16) return;
        constexpr int J = decltype(stage)::value, S = decltype(step)::value;
        uint32_t(&to)[4] = b[n][S % STEPS];
        F::template operand<J, S>(q[J % RING][n], scales[n], to);
        asm volatile("" : "+v"(to[0]), "+v"(to[1]), "+v"(to[2]), "+v"(to[3]));
    };
    // step s of block I of stage J, slot (n, m): its MFMAs onto d
    auto multiply = [&](auto stage, auto blk, int set, int s, int n, int m, ef16& d) {
        constexpr int J = decltype(stage)::value, I = decltype(blk)::value;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            if constexpr (FMT == kFmtF16) {  // the quants are the operands
                const u32x4& w = q[J % RING][n].q[STEPS * I + s];
                const uint32_t v[4] = {w.x, w.y, w.z, w.w};
                d = e_mfma(x[set][s][p][m], v, d);
            } else {
                d = e_mfma(x[set][s][p][m], b[n][s], d);
            }
        }
    };
    // kPerBlock, kPerStep: this slot's sums and those of the one before, whose scale is scale_of
    constexpr bool kParts = F::kScaled == kPerBlock || F::kScaled == kPerStep;
    ef16 sums_of[2];
    float scale_of = 0.0f;
    auto scale = [&](int n, int m, const ef16& d) {
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][m][i] = __builtin_fmaf(scale_of, d[i], acc[n][m][i]);
        asm volatile("" : "+v"(acc[n][m]));  // here, not where acc is used next: the sums would live until then
    };
    // block I of stage J; `next` the scales of the block after it; TAIL: of the stages behind the last whole unit
    auto run_block = [&](auto stage, auto blk, auto tail, int u, const typename F::Scale(&now)[NT], const typename F::Scale(&next)[NT]) {
        constexpr int J = decltype(stage)::value, I = decltype(blk)::value;
        constexpr bool TAIL = decltype(tail)::value != 0;
        constexpr int In = (I + 1) % BLOCKS, Jn = (J + (In == 0)) & 3;  // the next block
        constexpr int set = MT == 1 ? I & 1 : 0, other = MT == 1 ? set ^ 1 : 0;
        constexpr int SLOTS = NT * MT;
#pragma unroll
        for (int slot = 0; slot < SLOTS; ++slot) {
            const int n = slot / MT, m = slot % MT;
            __builtin_amdgcn_sched_barrier(0);
            // a column tile's quants of this stage (RING 4: of the one before) are decoded: a later stage's in their place
            constexpr int kNew = RING == 2 ? 2 : 3;
            constexpr bool kLoad = I == BLOCKS - 1 && (!TAIL || J + kNew < 3);  // (the tail has up to three stages)
            if (kLoad && slot == 0) load_quants(q[(J + kNew) % RING][0], 4 * u + J + kNew, 0);
            if (kLoad && slot == SLOTS / 2) load_quants(q[(J + kNew) % RING][1], 4 * u + J + kNew, 1);
            // the next block's activations, or this one's of the last row tile
            if constexpr (MT == 1) {
                if (slot == 0) read(Int<Jn>{}, Int<In>{}, other, 0);
            } else {
                if (slot == 0) read(Int<J>{}, Int<I>{}, 0, 1);
                if (slot == SLOTS - 1) read(Int<Jn>{}, Int<In>{}, 0, 0);
            }
            if constexpr (kParts) sums_of[slot & 1] = ef16{};
#pragma unroll
            for (int s = 0; s < STEPS; ++s) multiply(stage, blk, set, s, n, m, kParts ? sums_of[slot & 1] : acc[n][m]);
            // the second column tile of this block in the first half of the slots, the first one of the next block in the other
            auto decode_block = [&](auto j, auto i, int tile, int share, const typename F::Scale(&scales)[NT]) {
                constexpr int S0 = STEPS * decltype(i)::value;
                if (MT == 1 || share == 0) decode(j, Int<S0>{}, tile, scales);
                if constexpr (STEPS == 2)
                    if (MT == 1 || share == 1) decode(j, Int<S0 + 1>{}, tile, scales);
            };
            if (slot < SLOTS / 2) decode_block(Int<J>{}, Int<I>{}, 1, slot, now);
            else decode_block(Int<Jn>{}, Int<In>{}, 0, slot - SLOTS / 2, next);
            if constexpr (kParts) {  // the slot before: this block's, or the last block's last
                const int before = (slot + SLOTS - 1) % SLOTS;
                scale(before / MT, before % MT, sums_of[before & 1]);
                scale_of = F::template part_scale<BLOCKS * J + I>(now[n]);
            }
            if (MT == 1 ? slot == 0 : slot == 0 || slot == SLOTS - 1) __builtin_amdgcn_sched_group_barrier(0x100, STEPS * PARTS, 0);
#pragma unroll
            for (int i = 0; i < STEPS * PARTS; ++i) {  // an MFMA's time is eight instructions
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, STEPS == 1 ? 12 : 7, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto run_stage = [&](auto stage, auto tail, int u, const typename F::Scale(&s)[NT], typename F::Scale(&next)[NT]) {
        constexpr int J = decltype(stage)::value;
        run_block(stage, Int<0>{}, tail, u, s, s);
        if constexpr (BLOCKS == 4) {
            run_block(stage, Int<1>{}, tail, u, s, s);
            run_block(stage, Int<2>{}, tail, u, s, s);
        }
        // the next stage is in LDS and in registers, and the buffer after it free; behind the next stage's copies come the quants of
        // one stage, which may be on their way still
        stage_barrier<decltype(tail)::value != 0 ? 0 : kLater>();
#pragma unroll
        for (int n = 0; n < NT; ++n) q[(J + 1) % RING][n].settle();  // the compiler's wait, before it would count the next loads
        if constexpr (J == 0) load_scales(next, u + 1);
        if constexpr (J == 2 && FMT == kFmtQ4_K) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                uint32_t row = sums[m];
                asm volatile("" : "+v"(row));
                sum[m] = *reinterpret_cast<const eh8*>(a.sums + 32 * static_cast<uint64_t>(row + u) + 16 * h);
            }
        }
        copy(4 * u + J + 2);
        run_block(stage, Int<BLOCKS - 1>{}, tail, u, s, J == 3 ? next : s);
    };

    load_scales(sc[0], u0);
#pragma unroll
    for (int n = 0; n < NT; ++n) load_quants(q[0][n], 4 * u0, n), load_quants(q[1][n], 4 * u0 + 1, n);
    const int my_exp = a.exps[source_row(a, t.first + min(static_cast<int>(threadIdx.x), t.count - 1))];
    copy(4 * u0);
    copy(4 * u0 + 1);
    if constexpr (RING == 4) {
#pragma unroll
        for (int n = 0; n < NT; ++n) load_quants(q[2][n], 4 * u0 + 2, n);
    }
    if (threadIdx.x < BM) exps[threadIdx.x] = my_exp;  // (seen behind the stages' barriers)
    stage_barrier<kLater>();
    read(Int<0>{}, Int<0>{}, 0, 0);
    decode(Int<0>{}, Int<0>{}, 0, sc[0]);
    if constexpr (STEPS == 2) decode(Int<0>{}, Int<1>{}, 0, sc[0]);
    sums_of[1] = ef16{};
    const int whole = kRagged ? min(stages >> 2, u1) : u1;
#pragma unroll 1  // (a last round of its own would leave out loads that the barriers count on)
    for (int u = u0; u < whole; ++u) {
        run_stage(Int<0>{}, Int<0>{}, u, sc[0], sc[1]);
        run_stage(Int<1>{}, Int<0>{}, u, sc[0], sc[1]);
        run_stage(Int<2>{}, Int<0>{}, u, sc[0], sc[1]);
        run_stage(Int<3>{}, Int<0>{}, u, sc[0], sc[1]);
        if constexpr (FMT == kFmtQ4_K) {
            if (PAIR && part) sum[0] = eh8{};  // both parts of the sums go with the rows of hi
            subtract_minimums<NT, MT>(sc[0], acc, [&](int m) { return sum[m]; });
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[0][n] = sc[1][n];
    }
    if constexpr (kRagged) {
        const int rest = whole < u1 ? stages & 3 : 0;
        if (rest > 0) {
            run_stage(Int<0>{}, Int<1>{}, whole, sc[0], sc[1]);
            if (rest > 1) {
                run_stage(Int<1>{}, Int<1>{}, whole, sc[0], sc[1]);
                if (rest > 2) run_stage(Int<2>{}, Int<1>{}, whole, sc[0], sc[1]);
            }
        }
    }
    if constexpr (kParts) scale(NT - 1, MT - 1, sums_of[(NT * MT - 1) & 1]);
    stage_barrier<0>();  // the last copies have arrived

    // lanes of a half have rows 32 m + e_row(i) + 4 h; what is the same in all lanes of these is kept out of the addresses
    const int col = tile[0] * kUnitCols + (lane & 31), rows = t.count - 4 * h;
    const bool parts = SWIGLU && a.splits > 1;  // SwiGLU's two products apart
    float* const first = a.out + (static_cast<long>(split) * (parts ? 2 : 1) * a.g.R + t.first + 4 * h) * a.ldo + col;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int q4 = 0; q4 < (PAIR ? 2 : 4); ++q4) {
            typedef int int4_t __attribute__((ext_vector_type(4)));
            const int4_t e = *reinterpret_cast<const int4_t*>(exps + 32 * m + 8 * q4 + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = 4 * q4 + j, r = 32 * m + e_row(i);
                float v[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) v[n] = ldexpf(PAIR ? acc[n][m][i] + acc[n][m][i + 8] : acc[n][m][i], e[j]);
                if (r >= rows) continue;
                float* const o = first + r * a.ldo;
                if constexpr (SWIGLU) {
                    if (col < a.N) {
                        if (parts) {
                            o[0] = v[0];
                            o[a.g.R * a.ldo] = v[NT - 1];
                        } else {
                            o[0] = silu_f(v[0]) * v[NT - 1];
                        }
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        if (col + n * kUnitCols < a.N) o[n * kUnitCols] = v[n];
                }
            }
        }
    }
}

// ---- few tokens ---------------------------------------------------------------

constexpr int kFewWaves = 8;
// what few_kernel needs after its first loads
struct FewRest {
    float* out;
    long ldx, ldo;
    int N, K;
};
// LDS of a wave: rows of 1024 bytes (a unit's hi and lo, in the ring's order), 32 of sums and 4 of exponent
__device__ __host__ constexpr int few_wave_bytes(int bm) { return bm * (1024 + 32) + 64; }

// Eight activations of a row's unit (lane group of 32: one row) to their chunk of hi and lo, the row's sums over 32 and
// its exponent (not the power of two itself, which fp32 may not hold: down to 2^-163); the whole wave calls it.
__device__ __forceinline__ void few_convert(const f32x4& x, const f32x4& y, bool live, int r, char* area, char* sums, int* exps) {
    float mx = fmaxf(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))),
                     fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
    mx = fmaxf(mx, dpp<kQuadPerm1032>(mx));
    mx = fmaxf(mx, dpp<kQuadPerm2301>(mx));
    mx = fmaxf(mx, dpp<kRowHalfMirror>(mx));
    mx = fmaxf(mx, dpp<kRowMirror>(mx));
    mx = fmaxf(mx, swizzle_xor16(mx));
    int ex = 0;
    if (mx > 0.0f) {
        frexpf(mx, &ex);
        ex -= 15;  // the largest just below 2^15
    }
    const int c = threadIdx.x & 31;  // chunk of the unit: 64-wide group c >> 3, chunk c & 7 of it
    eh8 hi, lo;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = ldexpf(i < 4 ? x[i] : y[i - 4], -ex);
        sum += v;
        hi[i] = static_cast<_Float16>(v);
        lo[i] = static_cast<_Float16>(v - static_cast<float>(hi[i]));
    }
    sum += dpp<kQuadPerm1032>(sum);
    sum += dpp<kQuadPerm2301>(sum);
    if (!live) return;
    char* at = area + r * 1024 + 256 * (c >> 3);
    *reinterpret_cast<eh8*>(at + 16 * ((c & 7) ^ (r & 15))) = hi;
    *reinterpret_cast<eh8*>(at + 16 * (((c & 7) + 8) ^ (r & 15))) = lo;
    if ((c & 3) == 0) {
        sum *= 0.015625f;
        const _Float16 s = static_cast<_Float16>(sum);
        _Float16* o = reinterpret_cast<_Float16*>(sums + r * 32) + (c >> 2);
        o[0] = s;
        o[8] = static_cast<_Float16>(sum - static_cast<float>(s));
    }
    if (c == 0) exps[r] = ex;
}

// A stage (64 k) of NT column tiles against paired rows, of which lanes keep the first KEEP of registers 0 .. 3 (rows e_row(i) + 4 h;
// the second part's are 8 registers on): r += the scaled sums, with kNoScale t += the sums.  a(step): an activation operand.
template <class F, int J, int NT, int KEEP, class A>
__device__ __forceinline__ void few_stage(const typename F::Quant (&q)[NT], const typename F::Scale (&s)[NT], float (&r)[NT][KEEP],
                                          ef16 (&whole)[NT], A&& a) {
    auto block = [&](auto blk) {
        constexpr int I = decltype(blk)::value;  // of the stage
        const eh8 x[2] = {a(2 * I), a(2 * I + 1)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            uint32_t b[2][4];
            F::template operand<J, 2 * I>(q[n], s[n], b[0]);
            F::template operand<J, 2 * I + 1>(q[n], s[n], b[1]);
            auto scale = [&](float d, const ef16& t) {
#pragma unroll
                for (int i = 0; i < KEEP; ++i) r[n][i] = __builtin_fmaf(d, t[i] + t[i + 8], r[n][i]);
                if constexpr (KEEP == 1) asm volatile("" : "+v"(r[n][0]));  // the next step's sums not before: together they spill
            };
            if constexpr (F::kScaled == kPerBlock) {
                scale(F::template part_scale<2 * J + I>(s[n]), e_mfma(x[1], b[1], e_mfma(x[0], b[0], ef16{})));
            } else if constexpr (F::kScaled == kPerStep) {
                scale(F::template part_scale<4 * J + 2 * I>(s[n]), e_mfma(x[0], b[0], ef16{}));
                scale(F::template part_scale<4 * J + 2 * I + 1>(s[n]), e_mfma(x[1], b[1], ef16{}));
            } else {
                whole[n] = e_mfma(x[1], b[1], e_mfma(x[0], b[0], whole[n]));
            }
        }
    };
    block(Int<0>{});
    block(Int<1>{});
}

// A unit of NT column tiles times the rows that few_convert has left in the wave's area, up to 8 (lane rows from `count` on: the
// last again, unused): r[n][i], times two to the row's exponent, is the product of row i + 4 h.
template <int FMT, int NT, int KEEP>
__device__ __forceinline__ void few_multiply(const typename ExpertFmt<FMT>::Quant (&q)[4][NT],
                                             const typename ExpertFmt<FMT>::Scale (&sc)[NT], const char* area,
                                             const char* sums, int count, float (&r)[NT][KEEP]) {
    typedef ExpertFmt<FMT> F;
    const int lane = threadIdx.x & 63, h = lane >> 5, part = 8 * ((lane >> 4) & 1), row = min(lane & 15, count - 1);
    auto reader = [&](int j) {
        const char* at = area + row * 1024 + 256 * j;
        return [=](int s) { return *reinterpret_cast<const eh8*>(at + 16 * ((2 * s + h + part) ^ (row & 15))); };
    };
    ef16 whole[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if constexpr (F::kScaled == kNoScale) whole[n] = ef16{};
#pragma unroll
        for (int i = 0; i < KEEP; ++i) r[n][i] = 0.0f;
    }
    few_stage<F, 0, NT, KEEP>(q[0], sc, r, whole, reader(0));
    few_stage<F, 1, NT, KEEP>(q[1], sc, r, whole, reader(1));
    few_stage<F, 2, NT, KEEP>(q[2], sc, r, whole, reader(2));
    few_stage<F, 3, NT, KEEP>(q[3], sc, r, whole, reader(3));
    if constexpr (F::kScaled == kNoScale) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < KEEP; ++i) r[n][i] = whole[n][i] + whole[n][i + 8];
    }
    if constexpr (FMT == kFmtQ4_K) {
        eh8 x = *reinterpret_cast<const eh8*>(sums + row * 32 + 16 * h);
        if (part) x = eh8{};  // both parts of the sums go with the rows of hi
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            uint32_t b[4];
            F::min_operand(sc[n], b);
            const ef16 t = e_mfma(x, b, ef16{});
            const float dmin = F::min_scale(sc[n]);
#pragma unroll
            for (int i = 0; i < KEEP; ++i) r[n][i] = __builtin_fmaf(dmin, t[i], r[n][i]);
        }
    }
}

// what one lane wrote to the wave's LDS, others read: in order, and not to be reordered
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Workgroup of `waves` waves; wave w takes units w, w + waves, ...; up to 2^lg rows a tile (KEEP 1:
// one, 4: 1 .. 8).  The arguments that the
// first loads need come first and plain: those are preloaded into SGPRs.
template <int FMT, bool SWIGLU, int KEEP>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(const int* offsets, const int* rows, const uint8_t* w0, const uint8_t* w1,
                                                             const float* x, int E, int R, uint32_t over_k, int lg_waves, int tiles, int depth,
                                                             const FewRest rest) {
    typedef ExpertFmt<FMT> F;
    constexpr int NT = SWIGLU ? 2 : 1, kUnit = unit_bytes(FMT);
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, h = lane >> 5, lg = lg_waves & 3, waves = lg_waves >> 2;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile t;
    if (!find_tile(Groups{offsets, nullptr, nullptr, E, 1, R}, lg, tiles, blockIdx.x, t)) return;
    // a row for each half of the wave and pass, eight of its activations a lane
    constexpr int PASSES = KEEP;
    int source[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = t.first + min(2 * i + h, t.count - 1);
        source[i] = over_k != 0 ? rows[r] : r;  // (0: rows of x in grouped order)
    }
    const long first_unit = (static_cast<long>(t.expert) * tiles + t.block) * depth;
    char* const area = lds + wave * few_wave_bytes(1 << lg);
    char* const sums = area + (1024 << lg);
    int* const exps = reinterpret_cast<int*>(sums + (32 << lg));
    float acc[NT][KEEP] = {};
    for (int u = wave; u < depth; u += waves) {
        // Loads arrive in order: half of the weights, the activations (whose rows had to be looked up), the other half, so that
        // the activations are converted while weights are on their way.
        typename F::Quant q[4][NT];
        typename F::Scale sc[NT];
        f32x4 lo[PASSES], hi[PASSES];
        const uint8_t* const unit[2] = {w0 + (first_unit + u) * kUnit, w1 + (first_unit + u) * kUnit};
#pragma unroll
        for (int n = 0; n < NT; ++n) F::load(sc[n], unit[n], lane);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) F::load(q[j][n], unit[n], j, lane);
        const int c = u * kUnitK + 8 * (lane & 31);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            lo[i] = hi[i] = f32x4{0, 0, 0, 0};
            if (2 * i < t.count && c < rest.K) {
                const float* p = x + (over_k != 0 ? token_of(clamp_int(source[i], 0, R - 1), over_k) : source[i]) * rest.ldx + c;
                lo[i] = ld_f32x4(p);
                hi[i] = ld_f32x4(p + 4);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 2; j < 4; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) F::load(q[j][n], unit[n], j, lane);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
            if (2 * i < t.count) few_convert(lo[i], hi[i], 2 * i + h < t.count, 2 * i + h, area, sums, exps);
        wave_order();
        float p[NT][KEEP];
        few_multiply<FMT, NT, KEEP>(q, sc, area, sums, t.count, p);
#pragma unroll
        for (int i = 0; i < KEEP; ++i) {
            const int e = exps[min(i + 4 * h, t.count - 1)];
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][i] += ldexpf(p[n][i], e);
        }
        wave_order();
    }
    // the waves' sums, in their order
    __syncthreads();
    float* red = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < KEEP; ++i) red[((wave * NT + n) * 8 + i + 4 * h) * 32 + (lane & 31)] = acc[n][i];
    __syncthreads();
    for (int o = threadIdx.x; o < t.count * 32; o += 64 * waves) {
        float v[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            v[n] = red[n * 256 + o];
            for (int w = 1; w < waves; ++w) v[n] += red[(w * NT + n) * 256 + o];
        }
        const int col = t.block * kUnitCols + (o & 31);
        if (col < rest.N) rest.out[static_cast<long>(t.first + (o >> 5)) * rest.ldo + col] = SWIGLU ? silu_f(v[0]) * v[NT - 1] : v[0];
    }
}

// The weighted sums of few tokens in one launch: a workgroup of 16 waves takes a token and 16 columns, its waves the units of
// all of the token's choices (unit i: choice i / depth), each unit's products times the choice's weight.  Decoding is what
// counts, and a multiplication has 32 columns: a wave takes two units at once, lanes 0 .. 15 and 32 .. 47 the first one's 16
// columns, the others the second one's, against two rows of activations; of the four blocks of the result two are used.  (One
// unit of 32 columns a wave, on half as many CUs: 10.6 us instead of 7.6 for a token of 8 experts, 1024 -> 2048 Q6_K.)  All that
// lookups need is asked for at once and kept.
template <int FMT>
__global__ __launch_bounds__(1024) void token_kernel(const ProductArgs a, const TokenArgs b) {
    typedef ExpertFmt<FMT> F;
    constexpr int WAVES = 16, HELD = 4;
    constexpr long kUnit = unit_bytes(FMT);
    __shared__ __attribute__((aligned(16))) char lds[WAVES * few_wave_bytes(2)];
    __shared__ float red[WAVES][32];
    const int lane = threadIdx.x & 63, h = lane >> 5, k = a.g.k, E = a.g.E;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = blockIdx.x >> 1, t = blockIdx.y;
    const bool second = (lane & 16) != 0;                                  // whose weights the lane multiplies
    const uint32_t from = (lane & 47) | (blockIdx.x & 1) << 4;             // and which of a unit's lanes they were laid out for
    const int choice = t * k + min(lane, k - 1);
    const int slots = a.g.slots[choice];
    const float weights = b.weights[choice];
    int ends[HELD];  // of experts lane, 64 + lane, ...
#pragma unroll
    for (int i = 0; i < HELD; ++i) ends[i] = a.g.offsets[min(64 * i + lane + 1, E)];
    const int col = blockIdx.x * 16 + (threadIdx.x & 15);
    float first = 0.0f;
    if (b.residual != nullptr && threadIdx.x < 16 && col < a.N) first = b.residual[t * b.ldr + col];
    char* const area = lds + wave * few_wave_bytes(2);
    char* const sums = area + 2 * 1024;
    int* const exps = reinterpret_cast<int*>(sums + 2 * 32);
    float acc = 0.0f;  // lanes 0 .. 15 of the first units, lanes 48 .. 63 of the second ones
    const int units = k * a.depth;
    for (int i0 = wave; i0 < units; i0 += 2 * WAVES) {
        bool live[2];
        int slot[2], u[2];
        float weight[2];
        long at[2];  // the unit's place
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int i = min(i0 + n * WAVES, units - 1), j = i / a.depth;
            u[n] = i - j * a.depth;
            slot[n] = __builtin_amdgcn_readlane(slots, j);
            weight[n] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weights), j));
            live[n] = i0 + n * WAVES < units && slot[n] >= 0 && slot[n] < a.g.R;
            slot[n] = clamp_int(slot[n], 0, a.g.R - 1);
            int e = 0;  // the slot's expert: how many end at or before it
#pragma unroll
            for (int m = 0; m < HELD; ++m) e += __popcll(__ballot(64 * m + lane < E && ends[m] <= slot[n]));
            for (int e0 = 64 * HELD; e0 < E; e0 += 64) e += __popcll(__ballot(e0 + lane < E && a.g.offsets[e0 + lane + 1] <= slot[n]));
            at[n] = ((static_cast<long>(min(e, E - 1)) * a.tiles + tile) * a.depth + u[n]) * kUnit;
        }
        if (!live[0] && !live[1]) continue;
        if (!live[1]) slot[1] = slot[0], u[1] = u[0], at[1] = at[0];  // read twice, used once
        if (!live[0]) slot[0] = slot[1], u[0] = u[1], at[0] = at[1];
        const int c = (h ? u[1] : u[0]) * kUnitK + 8 * (lane & 31);
        f32x4 lo = f32x4{0, 0, 0, 0}, hi = lo;
        if (c < a.K) {
            const float* p = a.x + (h ? slot[1] : slot[0]) * a.ldx + c;
            lo = ld_f32x4(p);
            hi = ld_f32x4(p + 4);
        }
        const uint8_t* const unit = a.w[0] + (second ? at[1] : at[0]);
        typename F::Quant q[4][1];
        typename F::Scale sc[1];
        F::load(sc[0], unit, from);
#pragma unroll
        for (int s = 0; s < 4; ++s) F::load(q[s][0], unit, s, from);
        few_convert(lo, hi, true, h, area, sums, exps);
        wave_order();
        float p[1][1];  // of row 0, or row 4: the last one again, the second unit's
        few_multiply<FMT, 1, 1>(q, sc, area, sums, 2, p);
        // the weight meets the product, not the power of two: their product may leave fp32's range where the result does not
        if (h ? live[1] : live[0]) acc = __builtin_fmaf(h ? weight[1] : weight[0], ldexpf(p[0][0], exps[h]), acc);
        wave_order();
    }
    if (second == (h != 0)) red[wave][lane & 31] = acc;  // (lanes 0 .. 15, and 48 .. 63 as 16 .. 31)
    __syncthreads();
    if (threadIdx.x < 16 && col < a.N) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += red[w][threadIdx.x] + red[w][threadIdx.x + 16];
        a.out[t * a.ldo + col] = v + first;
    }
}

template <int FMT>
void expert_rows(const ProductArgs& a, bool swiglu, int bm, long workgroups, hipStream_t stream) {
    const auto run = swiglu ? (bm == 16   ? rows_kernel<FMT, 1, true, true>
                               : bm == 32 ? rows_kernel<FMT, 1, false, true>
                                          : rows_kernel<FMT, 2, false, true>)
                            : (bm == 16   ? rows_kernel<FMT, 1, true, false>
                               : bm == 32 ? rows_kernel<FMT, 1, false, false>
                                          : rows_kernel<FMT, 2, false, false>);
    hipLaunchKernelGGL(run, dim3(static_cast<unsigned>(workgroups)), dim3(256), 0, stream, a);
}

template <int FMT>
void expert_few(const ProductArgs& a, bool swiglu, int lg, int waves, long workgroups, hipStream_t stream) {
    const int lds = std::max(waves * few_wave_bytes(1 << lg), waves * (swiglu ? 2 : 1) * 1024);
    const bool one = a.gather && a.g.R == a.g.k;  // one token: whatever a row's number is, x has that row
    const FewRest rest{a.out, one ? 0 : a.ldx, a.ldo, a.N, a.K};
    const auto run = swiglu ? (lg == 0 ? few_kernel<FMT, true, 1> : few_kernel<FMT, true, 4>)
                            : (lg == 0 ? few_kernel<FMT, false, 1> : few_kernel<FMT, false, 4>);
    hipLaunchKernelGGL(run, dim3(static_cast<unsigned>(workgroups)),
                       dim3(64 * waves), lds, stream, a.g.offsets, a.g.rows, a.w[0], a.w[1], a.x, a.g.E, a.g.R,
                       a.gather && !one ? a.over_k : 0u, lg | waves << 2, a.tiles, a.depth, rest);
}

template <int FMT>
void expert_token(const ProductArgs& a, const TokenArgs& b, int tokens, hipStream_t stream) {
    hipLaunchKernelGGL(token_kernel<FMT>, dim3(2 * a.tiles, tokens), dim3(1024), 0, stream, a, b);
}

}  // namespace dev
}  // namespace cri
