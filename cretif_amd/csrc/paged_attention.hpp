// paged_attention.hpp -- attention of a ragged batch over a paged cache whose first positions every sequence shares.
//
// out[row] = sum_j softmax_j(scale q . k_j) v_j over the positions j the row sees.  The shared prefix is multiplied
// with the rows of all sequences at once, so its K and V are read once for the batch; each sequence's own
// positions are multiplied with its own rows.  Both leave (max, sum, acc) records that a second kernel joins.
//
// One wave takes 16 NC query rows ("columns": query q = token x G + g of the heads g that share a KV head) and a
// tile of positions at a time, straight from the pool into registers:
//   * S^T = K Q^T: K is the A operand, whose 16 bytes per lane are consecutive dims of a position's row.
//   * O^T += V^T P^T: a lane owns one column, and the positions of its scores are the positions whose
//     probabilities it supplies, so P never leaves the registers.  V^T's operand is put together in registers from
//     row loads (16-bit types: byte permutations; fp32: none are needed).
//   * 16-bit caches, v_mfma_f32_16x16x32: cached numbers are exact operands.  The fp32 queries and probabilities
//     are taken in parts whose sum is good to fp32: two fp16 parts (queries scaled per row into fp16's upper range,
//     probabilities by 2^12), three bf16 parts.  fp32 caches: v_mfma_f32_16x16x4.
//   * The running maximum is raised, and the accumulators rescaled, only when a score exceeds it by kSlack.
//   * A tile that some column does not see as a whole is multiplied once per limit that its columns have, V zeroed
//     from the limit on: what lies behind a row's last position (stale pages, infinities) never meets it, not even
//     times zero.
#pragma once

#include <algorithm>

#include "paged.hpp"

namespace cri {
namespace dev {

struct PagedAttnArgs {
    const float* q;
    float* out;
    float* rec;  // [rows][H][nrec] records of D + 4 floats (max, sum, 2 pad, acc); unused when nrec is 1
    long ldq, ldo;
    PagePool P;
    PageBatch B;
    const int* prefix_pages;
    int prefix_len, H, G, nrec;
    int pre_wq, pre_tiles, pre_chunks, pre_blocks;  // the prefix's workgroups: [stream / 8][tile][stream % 8]
    int own_wq, own_tiles, own_chunks;              // the sequences': [tile][chunk][KV head]
    float qscale;                                   // scale * log2 e: scores are in base 2
};

constexpr int kPagedWaves = 4;
constexpr int kPagedXcds = 8;

template <int TYPE, int DP>
struct PagedShape {
    static constexpr bool kWide = TYPE == kKvF32;              // 4-byte elements
    static constexpr int kTile = kWide ? 16 : 32;              // positions of a tile
    static constexpr int kT = kTile / 16;                      // MFMA row blocks of a tile
    static constexpr int kKs = kWide ? DP / 16 : DP / 32;      // 16-byte loads of a K row per lane
    static constexpr int kVe = kWide ? 4 : (DP >= 128 ? 8 : 4);  // elements of a V load
    static constexpr int kNh = DP / (16 * kVe);                // V loads of a position per lane
    static constexpr int kAcc = DP / 16;                       // accumulator blocks of a column block
    static constexpr int kParts = TYPE == kKvF16 ? 2 : TYPE == kKvBF16 ? 3 : 1;
    static constexpr float kShift = TYPE == kKvF16 ? 12.0f : 0.0f;  // probabilities enter O times 2^kShift
    static constexpr float kSlack = 3.0f;  // 2^(12 + 3) is inside fp16
};

__device__ __forceinline__ f32x4 mma16(const u32x4& a, const u32x4& b, const f32x4& c, std::integral_constant<int, kKvF16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const u32x4& a, const u32x4& b, const f32x4& c, std::integral_constant<int, kKvBF16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}

// the parts of eight floats (times f for fp16): x = p[0] + p[1] (+ p[2]), each the rest's rounding
template <int TYPE, int PARTS>
__device__ __forceinline__ void split8(const float (&x)[8], u32x4 (&p)[PARTS]) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f32x2 v = {r[2 * e], r[2 * e + 1]};
            if constexpr (TYPE == kKvF16) {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2 w = __builtin_convertvector(v, h2);
                p[k][e] = __builtin_bit_cast(uint32_t, w);
                r[2 * e] -= static_cast<float>(w.x);
                r[2 * e + 1] -= static_cast<float>(w.y);
            } else {
                typedef __bf16 b2 __attribute__((ext_vector_type(2)));
                const b2 w = __builtin_convertvector(v, b2);
                const uint32_t u = __builtin_bit_cast(uint32_t, w);
                p[k][e] = u;
                r[2 * e] -= __builtin_bit_cast(float, u << 16);
                r[2 * e + 1] -= __builtin_bit_cast(float, u & 0xFFFF0000u);
            }
        }
    }
}

__device__ __forceinline__ float col_max(float v) { return swap_max32(swap_max16(v, v), swap_max16(v, v)); }
__device__ __forceinline__ float col_sum(float v) {
    const float s = swap_add16(v, v);
    return swap_add32(s, s);
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = max(v, __shfl_xor(v, m));
    return v;
}
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = min(v, __shfl_xor(v, m));
    return v;
}

// the sequence of row t by bisection, one search per lane; -1 for a row of none
__device__ __forceinline__ int sequence_of(const PageBatch& B, int t) {
    int lo = 0, hi = B.n_seqs;  // the first s with offsets[s + 1] > t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (B.offsets[mid + 1] > t)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo < B.n_seqs && B.offsets[lo] <= t ? lo : -1;
}

// EVEN: head_dim is DP and the page size a multiple of 16, so the 16 positions of a tile's row block lie in one page
template <int TYPE, int DP, int NC, bool EVEN>
__global__ __launch_bounds__(64 * kPagedWaves) void paged_attn_kernel(const PagedAttnArgs a) {
    typedef PagedShape<TYPE, DP> S;
    typedef typename KvType<TYPE>::elem elem;
    typedef std::integral_constant<int, TYPE> Type;
    constexpr int kTile = S::kTile, kT = S::kT, kKs = S::kKs, kVe = S::kVe, kNh = S::kNh, kAcc = S::kAcc;
    constexpr int kRowF = DP + 4;                // floats of a column's record in LDS
    constexpr int kNs = 4 * kT;                  // scores of a lane and column
    extern __shared__ __attribute__((aligned(16))) float lds[];  // 3 waves' records

    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int D = EVEN ? DP : a.P.head_dim;
    const int Hkv = a.P.n_kv_heads, G = a.G;
    const long row_elems = static_cast<long>(Hkv) * D;
    const int cap = static_cast<int>(min(static_cast<long>(a.B.max_pages) * a.P.page_size, 0x7FFFFFFFL));

    // ---- what this workgroup does: a KV head, a tile of rows, a range of positions
    const bool prefix = static_cast<int>(blockIdx.x) < a.pre_blocks;
    int kvh, wq, row0, nrows, tok0, pos0 = 0, rec_at, p_lo, p_hi;
    const int* table;
    int table_len;
    if (prefix) {
        const int b = blockIdx.x, grp = kPagedXcds * a.pre_tiles;
        const int stream = b / grp * kPagedXcds + b % kPagedXcds, tile = b % grp / kPagedXcds;
        if (stream >= Hkv * a.pre_chunks) return;
        kvh = stream % Hkv;
        const int chunk = stream / Hkv;
        wq = a.pre_wq;
        row0 = tile * 16 * NC * wq;
        nrows = a.B.n_rows * G;
        tok0 = 0;
        rec_at = chunk;
        const int ntiles = (a.prefix_len + kTile - 1) / kTile, per = (ntiles + a.pre_chunks - 1) / a.pre_chunks;
        p_lo = min(chunk * per * kTile, a.prefix_len);
        p_hi = min(p_lo + per * kTile, a.prefix_len);
        table = a.prefix_pages;
        table_len = (a.prefix_len + a.P.page_size - 1) / a.P.page_size;
    } else {
        int b = static_cast<int>(blockIdx.x) - a.pre_blocks;
        kvh = b % Hkv;
        b /= Hkv;
        const int chunk = b % a.own_chunks;
        int tile = b / a.own_chunks;
        wq = a.own_wq;
        // the tile-th tile of rows of the batch: 64 sequences' tile counts summed at a time
        const int rt = 16 * NC * wq;
        int seq = -1;
        for (int base = 0; base < a.B.n_seqs; base += 64) {
            const int i = base + lane;
            int n = 0;
            if (i < a.B.n_seqs) n = min(max(a.B.offsets[i + 1] - a.B.offsets[i], 0), a.B.n_rows);
            n = (n * G + rt - 1) / rt;
            int sum = n;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const int o = __shfl_up(sum, m);
                if (lane >= m) sum += o;
            }
            const int before = __popcll(__ballot(sum <= tile));
            if (before < 64) {
                seq = base + before;
                if (before > 0) tile -= __shfl(sum, before - 1);
                break;
            }
            tile -= __shfl(sum, 63);
        }
        if (seq < 0 || seq >= a.B.n_seqs) return;
        seq = __builtin_amdgcn_readfirstlane(seq);
        tile = __builtin_amdgcn_readfirstlane(tile);
        tok0 = a.B.offsets[seq];
        const int n = min(max(a.B.offsets[seq + 1] - tok0, 0), a.B.n_rows);
        row0 = tile * rt;
        nrows = n * G;
        const int len = a.B.lens[seq];
        pos0 = len - n;  // position of the sequence's first row
        rec_at = a.pre_chunks + chunk;
        const int end = min(len, cap), start = a.prefix_len / kTile * kTile;
        const int ntiles = (max(end - start, 0) + kTile - 1) / kTile, per = (ntiles + a.own_chunks - 1) / a.own_chunks;
        p_lo = min(start + chunk * per * kTile, end);
        p_hi = min(p_lo + per * kTile, end);
        p_lo = max(p_lo, min(a.prefix_len, end));
        table = a.B.pages + static_cast<long>(seq) * a.B.max_pages;
        table_len = a.B.max_pages;
    }
    const int wk = kPagedWaves / wq;  // waves that share rows and split positions
    const int wrow = row0 + w / wk * 16 * NC, wpos = w % wk;

    // ---- the wave's columns: row, limit (positions it sees), query operand
    int lim[NC], tok[NC], head[NC];
    int most = 0, least = 0x7FFFFFFF;
    int ncols = 0;  // column blocks with a row
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int r = wrow + 16 * n + c;
        if (wrow + 16 * n < nrows) ncols = n + 1;
        tok[n] = -1;
        lim[n] = 0x7FFFFFFF;  // no row: sees everything, is stored nowhere
        head[n] = 0;
        if (r < nrows) {
            const int i = r / G, t = tok0 + i;
            int p = pos0 + i;
            bool ok = t >= 0 && t < a.B.n_rows;
            if (prefix && ok) {
                const int s = sequence_of(a.B, t);
                ok = s >= 0;
                if (ok) p = a.B.lens[s] - (a.B.offsets[s + 1] - t);
            }
            if (ok) {
                tok[n] = t;
                head[n] = kvh * G + r % G;
                lim[n] = min(max(p + 1, 0), prefix ? a.prefix_len : cap);
                most = max(most, lim[n]);
                least = min(least, lim[n]);
            }
        }
    }
    most = __builtin_amdgcn_readfirstlane(wave_max_i(most));
    least = __builtin_amdgcn_readfirstlane(wave_min_i(least));

    float kf[NC], qmax[NC];
    u32x4 q[NC][S::kWide ? 1 : kKs][S::kParts];
    f32x4 q32[NC][S::kWide ? kKs : 1];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        kf[n] = a.qscale;
        const float* src = a.q + static_cast<long>(max(tok[n], 0)) * a.ldq + static_cast<long>(head[n]) * D;
        const bool ok = tok[n] >= 0;
        if constexpr (S::kWide) {
#pragma unroll
            for (int j = 0; j < kKs; ++j) {
                const int d = 16 * j + 4 * g;
                q32[n][j] = ok && d < D ? ld_f32x4(src + d) : f32x4{0, 0, 0, 0};
            }
        } else {
            float x[kKs][8];
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < kKs; ++j) {
                const int d = 32 * j + 8 * g;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 v = ok && d < D ? ld_f32x4(src + d + 4 * h) : f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[j][4 * h + e] = v[e];
                        m = fmaxf(m, fabsf(v[e]));
                    }
                }
            }
            float f = 1.0f;
            if constexpr (TYPE == kKvF16) {
                // the row's largest magnitude goes to [2^13, 2^14): the parts are off by 2^-23 of an element or
                // 2^-39 of the largest
                qmax[n] = col_max(m);
                const int ex = static_cast<int>(__builtin_bit_cast(uint32_t, qmax[n]) >> 23) - 127;
                const int sh = min(13 - ex, 126);
                f = __builtin_bit_cast(float, (sh + 127) << 23);
                kf[n] = a.qscale * __builtin_bit_cast(float, (127 - max(sh, -126)) << 23);
            }
#pragma unroll
            for (int j = 0; j < kKs; ++j) {
                if constexpr (TYPE == kKvF16) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[j][e] *= f;
                }
                split8<TYPE, S::kParts>(x[j], q[n][j]);
            }
        }
    }

    f32x4 acc[NC][kAcc];
    float mx[NC], sum[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        mx[n] = -INFINITY;
        sum[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < kAcc; ++i) acc[n][i] = f32x4{0, 0, 0, 0};
    }

    // ---- the tiles
    const elem* const kbase = static_cast<const elem*>(a.P.k) + static_cast<long>(kvh) * D;
    const elem* const vbase = static_cast<const elem*>(a.P.v) + static_cast<long>(kvh) * D;
    auto page_of = [&](int pi) {
        const int pg = table[min(pi, table_len - 1)];
        return static_cast<unsigned>(pg) < static_cast<unsigned>(a.P.n_pages) ? pg : 0;
    };
    auto row_at = [&](int pos) {  // element offset of a position's row
        const int pi = page_index(a.P, pos);
        return page_of(pi) * a.P.stride + (pos - pi * a.P.page_size) * row_elems;
    };
    // first row of each 16-position block of a tile (EVEN)
    auto block_rows = [&](int p0, long (&at)[kT]) {
#pragma unroll
        for (int t = 0; t < kT; ++t) at[t] = row_at(p0 + 16 * t);
    };
    auto load_k = [&](int p0, const long (&at)[kT], u32x4 (&k)[kT][kKs]) {
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const elem* row = kbase + (EVEN ? at[t] + c * row_elems : row_at(p0 + 16 * t + c));
#pragma unroll
            for (int j = 0; j < kKs; ++j) {
                const int d = S::kWide ? 16 * j + 4 * g : 32 * j + 8 * g;
                if constexpr (EVEN) {
                    k[t][j] = *reinterpret_cast<const u32x4*>(row + d);
                } else {
                    k[t][j] = *reinterpret_cast<const u32x4*>(row + (d < D ? d : 0));
                    if (d >= D) k[t][j] = u32x4{0, 0, 0, 0};
                }
            }
        }
    };
    typedef uint32_t vreg __attribute__((ext_vector_type(S::kWide ? 4 : kVe / 2)));
    auto load_v = [&](int p0, const long (&at)[kT], vreg (&v)[kT][4][kNh]) {
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const elem* row = vbase + (EVEN ? at[t] + (4 * g + i) * row_elems : row_at(p0 + 16 * t + 4 * g + i));
#pragma unroll
                for (int h = 0; h < kNh; ++h) {
                    const int d = 16 * kVe * h + kVe * c;
                    v[t][i][h] = *reinterpret_cast<const vreg*>(row + (EVEN || d < D ? d : 0));
                }
            }
    };
    const int first = p_lo / kTile + wpos;
    const int last = (min(p_hi, most) + kTile - 1) / kTile;  // tiles [first, last) in steps of wk

    u32x4 k[kT][kKs];
    long at[kT] = {};
    if (first < last) {
        if constexpr (EVEN) block_rows(first * kTile, at);
        load_k(first * kTile, at, k);
    }
    for (int tile = first; tile < last; tile += wk) {
        const int p0 = tile * kTile;
        vreg v[kT][4][kNh];
        load_v(p0, at, v);
        const bool whole = p0 >= p_lo && p0 + kTile <= min(p_hi, least);
        float s[NC][kNs];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if (n > 0 && n >= ncols) continue;
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                f32x4 x = {0, 0, 0, 0};
                if constexpr (S::kWide) {
#pragma unroll
                    for (int j = 0; j < kKs; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            x = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, static_cast<uint32_t>(k[t][j][e])), q32[n][j][e], x,
                                                                     0, 0, 0);
                } else {
#pragma unroll
                    for (int p = S::kParts - 1; p >= 0; --p)
#pragma unroll
                        for (int j = 0; j < kKs; ++j) x = mma16(k[t][j], q[n][j][p], x, Type{});
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][4 * t + i] = x[i] * kf[n];
            }
        }
        if (tile + wk < last) {  // the next tile's keys, in flight during the softmax and the second product
            long nat[kT] = {};
            if constexpr (EVEN) block_rows(p0 + wk * kTile, nat);
            load_k(p0 + wk * kTile, nat, k);
#pragma unroll
            for (int t = 0; t < kT; ++t) at[t] = nat[t];
        }
        u32x4 pb[NC][S::kParts];
        float p32[NC][4];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if (n > 0 && n >= ncols) continue;
            if (!whole) {
                const int hi = min(p_hi, lim[n]);
#pragma unroll
                for (int t = 0; t < kT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int p = p0 + 16 * t + 4 * g + i;
                        if (p < p_lo || p >= hi) s[n][4 * t + i] = -INFINITY;
                    }
            }
            float m = s[n][0];
#pragma unroll
            for (int i = 1; i < kNs; ++i) m = fmaxf(m, s[n][i]);
            m = col_max(m);
            const bool raise = m > mx[n] + S::kSlack;
            if (__ballot(raise) != 0) {
                const float f = raise ? __builtin_amdgcn_exp2f(mx[n] - m) : 1.0f;
                if (raise) mx[n] = m;
                sum[n] *= f;
#pragma unroll
                for (int i = 0; i < kAcc; ++i) acc[n][i] *= f;
            }
            const float base = (mx[n] == -INFINITY ? 0.0f : mx[n]) - S::kShift;
            float p[8] = {};
            float l = 0.0f;
#pragma unroll
            for (int i = 0; i < kNs; ++i) {
                p[i] = __builtin_amdgcn_exp2f(s[n][i] - base);
                l += p[i];
            }
            sum[n] += l;
            if constexpr (S::kWide) {
#pragma unroll
                for (int i = 0; i < 4; ++i) p32[n][i] = p[i];
            } else {
                split8<TYPE, S::kParts>(p, pb[n]);
            }
        }
        // O^T += V^T P^T; `from` zeroes the positions from there on (an index into the tile) and those before p_lo
        auto multiply = [&](auto masked, int from, const int (&rel)[NC]) {
            constexpr bool kMask = decltype(masked)::value;
            const int lo = kMask ? p_lo - p0 : 0;
#pragma unroll
            for (int h = 0; h < kNh; ++h)
#pragma unroll
                for (int e = 0; e < kVe; ++e) {
                    if constexpr (S::kWide) {
#pragma unroll
                        for (int n = 0; n < NC; ++n) {
                            if (n > 0 && n >= ncols) continue;
                            f32x4 x = acc[n][h * kVe + e];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float u = __builtin_bit_cast(float, static_cast<uint32_t>(v[0][i][h][e]));
                                if (kMask && (4 * g + i < lo || 4 * g + i >= from)) u = 0.0f;
                                x = __builtin_amdgcn_mfma_f32_16x16x4f32(u, p32[n][i], x, 0, 0, 0);
                            }
                            if (!kMask || rel[n] == from) acc[n][h * kVe + e] = x;
                        }
                    } else {
                        // dim e of the lane's eight positions: halves of two rows' dwords
                        u32x4 f;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int t = j >> 1, i = 2 * (j & 1);
                            const uint32_t x = v[t][i][h][e >> 1], y = v[t][i + 1][h][e >> 1];
                            f[j] = __builtin_amdgcn_perm(y, x, e & 1 ? 0x07060302u : 0x05040100u);
                            if (kMask) {
                                const int at0 = 16 * t + 4 * g + i;
                                if (at0 < lo || at0 >= from) f[j] &= 0xFFFF0000u;
                                if (at0 + 1 < lo || at0 + 1 >= from) f[j] &= 0x0000FFFFu;
                            }
                        }
#pragma unroll
                        for (int n = 0; n < NC; ++n) {
                            if (n > 0 && n >= ncols) continue;
                            f32x4 x = acc[n][h * kVe + e];
#pragma unroll
                            for (int p = S::kParts - 1; p >= 0; --p) x = mma16(f, pb[n][p], x, Type{});
                            if (!kMask || rel[n] == from) acc[n][h * kVe + e] = x;
                        }
                    }
                }
        };
        int rel[NC];
        if (whole) {
            multiply(std::false_type{}, 0, rel);
        } else {
#pragma unroll
            for (int n = 0; n < NC; ++n) rel[n] = min(max(min(p_hi, lim[n]) - p0, 0), kTile);
            for (int from = kTile; from > 0; --from) {
                bool any = false;
#pragma unroll
                for (int n = 0; n < NC; ++n) any = any || rel[n] == from;
                if (__ballot(any) != 0) multiply(std::true_type{}, from, rel);
            }
        }
    }

    // ---- a column's waves meet in LDS, the first of them has the result
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        sum[n] = col_sum(sum[n]);
        if (sum[n] != sum[n]) mx[n] = INFINITY;  // NaN scores leave no maximum: keep the record from being skipped
    }
    auto dim_of = [&](int h, int i) { return 16 * kVe * h + kVe * (4 * g + i); };  // of accumulators h kVe .., element i
    if (wk > 1) {
        const int slot = wpos - 1 + w / wk * (wk - 1);  // of kPagedWaves - wq
        if (wpos > 0) {
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                float* r = lds + (slot * NC * 16 + n * 16 + c) * kRowF;
                if (g == 0) {
                    r[DP] = mx[n];
                    r[DP + 1] = sum[n];
                }
#pragma unroll
                for (int h = 0; h < kNh; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < kVe; e += 4)
                            *reinterpret_cast<f32x4*>(r + dim_of(h, i) + e) =
                                f32x4{acc[n][h * kVe + e][i], acc[n][h * kVe + e + 1][i], acc[n][h * kVe + e + 2][i],
                                      acc[n][h * kVe + e + 3][i]};
            }
        }
        __syncthreads();
        if (wpos > 0) return;
        for (int o = 0; o < wk - 1; ++o) {
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const float* r = lds + ((o + w / wk * (wk - 1)) * NC * 16 + n * 16 + c) * kRowF;
                const float m2 = r[DP], l2 = r[DP + 1], m = fmaxf(mx[n], m2);
                const float f1 = mx[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx[n] - m);
                const float f2 = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m2 - m);
                mx[n] = m;
                sum[n] = sum[n] * f1 + l2 * f2;
#pragma unroll
                for (int h = 0; h < kNh; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < kVe; e += 4) {
                            const f32x4 x = *reinterpret_cast<const f32x4*>(r + dim_of(h, i) + e);
#pragma unroll
                            for (int d = 0; d < 4; ++d)
                                acc[n][h * kVe + e + d][i] = acc[n][h * kVe + e + d][i] * f1 + x[d] * f2;
                        }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        if (tok[n] < 0) continue;
        float* dst;
        float f = 1.0f;
        if (a.nrec == 1) {
            dst = a.out + tok[n] * a.ldo + static_cast<long>(head[n]) * D;
            f = sum[n] == 0.0f ? 0.0f : 1.0f / sum[n];  // a row that sees nothing: zeros
        } else {
            dst = a.rec + ((static_cast<long>(tok[n]) * a.H + head[n]) * a.nrec + rec_at) * (D + 4);
            if (g == 0) *reinterpret_cast<f32x2*>(dst) = f32x2{mx[n], sum[n]};
            dst += 4;
            if (mx[n] == -INFINITY) continue;
        }
#pragma unroll
        for (int h = 0; h < kNh; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < kVe; e += 4) {
                    const int d = dim_of(h, i) + e;
                    if (EVEN || d < D)
                        *reinterpret_cast<f32x4_a4*>(dst + d) =
                            f32x4_a4{acc[n][h * kVe + e][i] * f, acc[n][h * kVe + e + 1][i] * f,
                                     acc[n][h * kVe + e + 2][i] * f, acc[n][h * kVe + e + 3][i] * f};
                }
    }
}

template <int TYPE, int DP, int NC, bool EVEN>
void run_paged_attn(const PagedAttnArgs& a, int blocks, hipStream_t stream) {
    const int lds = (kPagedWaves - 1) * NC * 16 * (DP + 4) * 4;
    hipLaunchKernelGGL((paged_attn_kernel<TYPE, DP, NC, EVEN>), dim3(blocks), dim3(64 * kPagedWaves), lds, stream, a);
}

template <int TYPE>
void run_paged_attn_type(const PagedAttnArgs& a, bool even, int nc, int blocks, hipStream_t stream) {
    const int D = a.P.head_dim;
    if (even) {
        if (D == 64)
            nc == 2 ? run_paged_attn<TYPE, 64, 2, true>(a, blocks, stream) : run_paged_attn<TYPE, 64, 1, true>(a, blocks, stream);
        else if (D == 128)
            nc == 2 ? run_paged_attn<TYPE, 128, 2, true>(a, blocks, stream) : run_paged_attn<TYPE, 128, 1, true>(a, blocks, stream);
        else
            run_paged_attn<TYPE, 256, 1, true>(a, blocks, stream);
    } else {
        if (D <= 64)
            run_paged_attn<TYPE, 64, 1, false>(a, blocks, stream);
        else if (D <= 128)
            run_paged_attn<TYPE, 128, 1, false>(a, blocks, stream);
        else
            run_paged_attn<TYPE, 256, 1, false>(a, blocks, stream);
    }
}

void run_paged_attn_f32(const PagedAttnArgs& a, bool even, int nc, int blocks, hipStream_t stream);
void run_paged_attn_f16(const PagedAttnArgs& a, bool even, int nc, int blocks, hipStream_t stream);
void run_paged_attn_bf16(const PagedAttnArgs& a, bool even, int nc, int blocks, hipStream_t stream);

}  // namespace dev
}  // namespace cri
