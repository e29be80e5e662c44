// experts.hpp -- what the kernels of a layer of experts share: how a matrix per expert lies once it is laid out
// (cri_expert_pack), and which rows a workgroup works on.
//
// A matrix W [N, K] becomes units of 32 rows (output columns of the product) x 256 k, zero beyond N and K: expert, then
// column tile, then k, so a wave that walks along k reads consecutive memory.  v_mfma_f32_32x32x16_f16 wants of lane
// (n = lane & 31, h = lane >> 5) the eight weights k = 16 i + 8 h .. + 7 of column n at step i, so a unit holds for every
// lane its own bytes of all 16 steps, 16 bytes at a time for 64 lanes: each load of a wave is 1 KB in a row, whatever the
// file's format, and nothing has to be shifted into place.  Sections of a unit, one after the other:
//
//   format  quants                     further bits             scales of column n                         bytes (the file's)
//   Q8_0    [8][64 lanes][16] q + 128  -                        [32][16]: 8 fp16 d                         8704 (8704)
//   Q4_0    [4][64][16] nibbles        -                        [32][16]: 8 fp16 d                         4608 (4608)
//   Q5_0    [4][64][16] nibbles        [64][16] a bit each      [32][16]: 8 fp16 d                         5632 (5632)
//   Q4_K    [4][64][16] nibbles        -                        [32][16]: 8 sc, 8 mn; [32][4]: d, dmin     4736 (4608)
//   Q6_K    [4][64][16] nibbles        [2][64][16] 2 bits each  [32][16]: 16 int8 sc; [32] fp16 d          6720 (6720)
//   FP16    [16][64][16]               -                        -                                         16384 (16384)
//
// A dword of nibbles is one step: weights 0 .. 7 at bits 0, 16, 4, 20, 8, 24, 12, 28, so that one mask gives a pair in the
// low bits of two halves.  Or-ed into 0x6400 (1024 in fp16) an integer below 1024 is exact, and a packed addition takes the
// 1024 and the format's zero point off: five VALU instructions for four weights.  Bytes: weights 0 .. 3 at bits 0, 16, 8,
// 24 of a step's first dword.  Bits of Q5_0: dword j has steps 4 j .. 4 j + 3, pair p of step s at bits 4 s + p and
// 16 + 4 s + p; Q6_K: dword j has steps 2 j and 2 j + 1, two bits at 2 (4 s + p) and 16 + 2 (4 s + p).
#pragma once

#include "common.hpp"
#include "internal.hpp"

namespace cri {
namespace dev {

constexpr int kUnitCols = 32, kUnitK = 256;

__device__ __host__ constexpr int unit_bytes(int fmt) {
    return fmt == kFmtQ8_0 ? 8704 : fmt == kFmtQ4_0 ? 4608 : fmt == kFmtQ5_0 ? 5632 : fmt == kFmtQ4_K ? 4736 : fmt == kFmtQ6_K ? 6720 : 16384;
}

// the grouped rows of a call, as the kernels take them; what the arrays hold is never trusted with an address
struct Groups {
    const int* offsets;  // [E + 1]
    const int* rows;     // [R]: pairs token * k + choice
    const int* slots;    // [R]: a pair's grouped row, or -1
    int E, k, R;         // R = tokens * k
};

// Rows [first, first + count) of an expert, a tile of them, and its block of columns.
struct Tile {
    int expert, first, count, block;
};

__device__ __forceinline__ int wave_scan_add(int v) {  // inclusive sum over the lanes below
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8 within 16 lanes
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return v;
}

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
// tiles of 2^lg rows
__device__ __forceinline__ int tiles_of(int lo, int hi, int lg) { return (max(hi - lo, 0) + (1 << lg) - 1) >> lg; }

// Work item number of workgroup b, out of every expert's tiles of up to 2^lg rows x blocks, or no such item.  Experts come in
// order, then blocks, then tiles: the tiles that share an expert's block of weights are neighbours, and each of the eight
// XCDs (workgroup b runs on XCD b mod 8, with an L2 of its own) gets consecutive items.  The whole wave calls it.  Up to 256
// experts a lane holds four in registers: one trip to memory, then a few dozen instructions.
__device__ __forceinline__ bool find_tile(const Groups& g, int lg, int blocks, int b, Tile& t) {
    constexpr int HELD = 4;
    const int lane = __lane_id(), per = g.E <= 64 ? 1 : g.E <= 64 * HELD ? HELD : (g.E + 63) >> 6;
    const int e0 = lane * per;
    int off[HELD + 1], n[HELD], tiles = 0;
    if (per <= HELD) {
#pragma unroll
        for (int i = 0; i <= HELD; ++i) off[i] = g.offsets[min(e0 + i, g.E)];  // (all asked for at once)
#pragma unroll
        for (int i = 0; i <= HELD; ++i) off[i] = clamp_int(off[i], 0, g.R);
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            n[i] = i < per ? tiles_of(off[i], off[i + 1], lg) : 0;  // (past the last expert nothing: the same offset)
            tiles += n[i];
        }
    } else {
        for (int e = e0; e < min(e0 + per, g.E); ++e)
            tiles += tiles_of(clamp_int(g.offsets[e], 0, g.R), clamp_int(g.offsets[e + 1], 0, g.R), lg);
    }
    const int up = wave_scan_add(tiles);
    const long total = static_cast<long>(__builtin_amdgcn_readlane(up, 63)) * blocks;
    const long share = (total + 7) >> 3;
    const long item = (b & 7) * share + (b >> 3);
    if ((b >> 3) >= share || item >= total) return false;
    const int who = __builtin_ctzl(__ballot(static_cast<long>(up) * blocks > item));
    long before = static_cast<long>(__builtin_amdgcn_readlane(up - tiles, who)) * blocks;
    int lo = 0, hi = 0, count = 0;
    t.expert = who * per;
    if (per <= HELD) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int ni = __builtin_amdgcn_readlane(n[i], who);
            if (count == 0 && item < before + static_cast<long>(ni) * blocks) {
                count = ni;
                lo = __builtin_amdgcn_readlane(off[i], who);
                hi = __builtin_amdgcn_readlane(off[i + 1], who);
                t.expert += i;
            } else if (count == 0) {
                before += static_cast<long>(ni) * blocks;
            }
        }
    } else {  // one of that lane's experts to a lane
        const int mine = min(t.expert + lane, g.E - 1);
        const int from = clamp_int(g.offsets[mine], 0, g.R), to = clamp_int(g.offsets[mine + 1], 0, g.R);
        const int some = lane < per && t.expert + lane < g.E ? tiles_of(from, to, lg) : 0;
        const int sum = wave_scan_add(some);
        const unsigned long hit = __ballot(before + static_cast<long>(sum) * blocks > item);
        if (hit == 0) return false;  // (the offsets changed meanwhile)
        const int at = __builtin_ctzl(hit);
        before += static_cast<long>(__builtin_amdgcn_readlane(sum - some, at)) * blocks;
        count = __builtin_amdgcn_readlane(some, at);
        lo = __builtin_amdgcn_readlane(from, at);
        hi = __builtin_amdgcn_readlane(to, at);
        t.expert += at;
    }
    if (count == 0) return false;
    const int rest = static_cast<int>(item - before);
    t.block = count == 1 ? rest : rest / count;
    t.first = lo + ((rest - t.block * count) << lg);
    t.count = min(1 << lg, hi - t.first);
    return true;
}

// workgroups that find_tile needs whatever the groups hold: an expert's tiles are at most its rows, and all but one of
// its tiles are full
__host__ inline long most_tiles(long R, int E, int bm) {
    const long some = R < E ? R : E;
    const long bound = R / bm + some;
    return bound < R ? bound : R;
}

// pair / k: over_k is 2^31 / k rounded up, off by less than 1, so the product by less than 2^-7 (pairs are below 2^23), and a quotient
// is at least 1 / 64 below the next whole number
__device__ __forceinline__ int token_of(int pair, uint32_t over_k) {
    return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(pair), over_k));
}

struct ProductArgs {
    const uint8_t* w[2];  // W, or G and U
    Groups g;
    const float* x;       // few_kernel: the activations, row t of token t (gather) or grouped row t
    long ldx;
    const uint8_t* planes;  // rows_kernel: [rows][depth][1024] hi and lo
    const uint8_t* sums;    // [rows][depth][32]: sums over 32 k, times 2^-6, 8 hi and 8 lo (Q4_K)
    const int* exps;        // [rows]: the row is 2^exps times its planes
    float* out;
    long ldo;
    int N, K, tiles, depth;  // tiles: columns / 32, depth: k / 256
    bool gather;             // the row of grouped row r is rows[r] / k, else r
    uint32_t over_k;         // of token_of
    int splits;              // rows_kernel: parts of k; with more than one, out is [splits][R][ldo] (SwiGLU: [splits][2][R][ldo])
};

// column blocks of rows_kernel: a wave takes a tile of G and U, or two tiles
__device__ __host__ inline int rows_blocks(int tiles, bool swiglu) { return swiglu ? (tiles + 3) >> 2 : (tiles + 7) >> 3; }

struct TokenArgs {
    const float* weights;   // [tokens, k]
    const float* residual;  // or null
    long ldr;
};

// the kernels of experts_gemm.hpp, instantiated in one file per format (experts_q4_k.hip, ...).  expert_rows: tiles of bm = 16, 32
// or 64 rows, workgroups of 4 waves; expert_few: tiles of up to 2^lg rows, lg 0 .. 3, workgroups of `waves` waves, up
// to 8 (lg 3: 4, for its LDS); expert_token: the weighted sums of so many tokens, x in grouped order
template <int FMT>
void expert_rows(const ProductArgs& a, bool swiglu, int bm, long workgroups, hipStream_t stream);
template <int FMT>
void expert_few(const ProductArgs& a, bool swiglu, int lg, int waves, long workgroups, hipStream_t stream);
template <int FMT>
void expert_token(const ProductArgs& a, const TokenArgs& b, int tokens, hipStream_t stream);

}  // namespace dev
}  // namespace cri
