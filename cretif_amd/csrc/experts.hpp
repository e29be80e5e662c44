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

// Rows [first, first + count) of an expert, a tile of at most BM of them, and its block of columns.
struct Tile {
    int expert, first, count, block;
};

__device__ __forceinline__ int wave_scan_add(int v) {  // inclusive sum over the lanes below
    const int lane = __lane_id();
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __builtin_amdgcn_ds_bpermute((lane - d) << 2, v);
        v += lane >= d ? o : 0;
    }
    return v;
}

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Work item number of workgroup b, out of every expert's ceil(rows / BM) tiles x blocks, or no such item.  Experts come in
// order, then blocks, then tiles: the tiles that share an expert's block of weights are neighbours, and each of the eight
// XCDs (workgroup b runs on XCD b mod 8, with an L2 of its own) gets consecutive items.  The whole wave calls it.
__device__ __forceinline__ bool find_tile(const Groups& g, int bm, int blocks, int b, Tile& t) {
    const int lane = __lane_id(), per = (g.E + 63) >> 6;
    const int e0 = lane * per, e1 = min(e0 + per, g.E);
    int tiles = 0;
    if (per == 1) {
        if (e0 < g.E) {
            const int lo = clamp_int(g.offsets[e0], 0, g.R), hi = clamp_int(g.offsets[e0 + 1], 0, g.R);
            tiles = hi > lo ? (hi - lo + bm - 1) / bm : 0;
        }
    } else {
        int lo = e0 < g.E ? clamp_int(g.offsets[e0], 0, g.R) : 0;
        for (int e = e0; e < e1; ++e) {
            const int hi = clamp_int(g.offsets[e + 1], 0, g.R);
            tiles += hi > lo ? (hi - lo + bm - 1) / bm : 0;
            lo = hi;
        }
    }
    const int up = wave_scan_add(tiles);
    const long total = static_cast<long>(__builtin_amdgcn_readlane(up, 63)) * blocks;
    const long share = (total + 7) >> 3;
    const long item = (b & 7) * share + (b >> 3);
    if ((b >> 3) >= share || item >= total) return false;
    const unsigned long hit = __ballot(static_cast<long>(up) * blocks > item);
    const int who = __builtin_ctzl(hit);
    int before = __builtin_amdgcn_readlane(up - tiles, who), e = who * per;
    if (per > 1) {  // which of that lane's experts: one of them a lane
        const int mine = min(e + lane, g.E - 1);
        const int lo = clamp_int(g.offsets[mine], 0, g.R), hi = clamp_int(g.offsets[mine + 1], 0, g.R);
        const int n = lane < per && e + lane < g.E && hi > lo ? (hi - lo + bm - 1) / bm : 0;
        const int sum = wave_scan_add(n);
        const int at = __builtin_ctzl(__ballot(static_cast<long>(before + sum) * blocks > item));
        before += __builtin_amdgcn_readlane(sum - n, at);
        e = min(e + at, g.E - 1);  // (as it was found, unless the offsets change meanwhile)
    }
    const int lo = clamp_int(g.offsets[e], 0, g.R), hi = clamp_int(g.offsets[e + 1], 0, g.R);
    const int n = max((hi - lo + bm - 1) / bm, 1), rest = static_cast<int>(item - static_cast<long>(before) * blocks);
    t.expert = e;
    t.block = rest / n;
    t.first = lo + (rest - t.block * n) * bm;
    t.count = min(bm, hi - t.first);
    return t.count > 0 && t.block < blocks;
}

// workgroups that find_tile needs whatever the groups hold: an expert's tiles are at most its rows, and all but one of
// its tiles are full
__host__ inline long most_tiles(long R, int E, int bm) {
    const long some = R < E ? R : E;
    const long bound = R / bm + some;
    return bound < R ? bound : R;
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
};

// the kernels of experts_gemm.hpp, instantiated in one file per format (experts_q4_k.hip, ...).  bm: rows of a tile, 16, 32
// or 64 for expert_rows, 1 .. 16 for expert_few, whose workgroups have `waves` waves; expert_few returns a launcher status
template <int FMT>
void expert_rows(const ProductArgs& a, bool swiglu, int bm, long workgroups, hipStream_t stream);
template <int FMT>
int expert_few(const ProductArgs& a, bool swiglu, int bm, int waves, long workgroups, hipStream_t stream);

}  // namespace dev
}  // namespace cri
