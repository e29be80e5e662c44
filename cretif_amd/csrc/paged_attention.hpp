// paged_attention.hpp -- attention of a ragged batch over a paged cache whose first positions every sequence shares.
//
// out[row] = sum_j softmax_j(scale q . k_j) v_j over the positions j the row sees.  The shared prefix is multiplied
// with the rows of all sequences at once, so its K and V are read once for the batch; each sequence's own
// positions are multiplied with its own rows.  Both leave (max, sum, acc) records that a second kernel joins.
//
// rows_body: a wave takes 16 query rows ("columns": query q = token x G + g of the heads g that share a KV head), a
// range of positions and a tile of them at a time, straight from the pool into registers, without LDS or barriers.  It
// is bound by memory: 64 sequences of 1500 own positions, 32/8 heads of 128, read their 393 MB of fp16 in 79 us (5.0
// TB/s; a large copy moves 4.7), fp32 786 MB in 140 us (5.6); a range of 256 positions, half that or a third took the
// same within a tenth, 512 left waves idle where lengths differ.  Two waves per SIMD (216 registers): three spilled, and
// were slower (99 -> 130 us before the waves were made independent).
//   * S^T = K Q^T: K is the A operand, whose 16 bytes per lane are consecutive dims of a position's row.
//   * O^T += V^T P^T: a lane owns one column, and the positions of its scores are the positions whose
//     probabilities it supplies, so P never leaves the registers.  V^T's operand is put together in registers from
//     row loads (16-bit types: byte permutations; fp32: none are needed).
//   * 16-bit caches, v_mfma_f32_16x16x32: cached numbers are exact operands.  The fp32 queries and probabilities
//     are taken in parts whose sum is good to fp32: two fp16 parts (queries scaled per row into fp16's upper range,
//     probabilities by 2^12; kSafe says what that leaves), three bf16 parts.  fp32 caches: v_mfma_f32_16x16x4, which keeps up with memory.
//   * The running maximum is raised, and the accumulators rescaled, only when a score exceeds it by kSlack.
//   * A tile that some column does not see as a whole is multiplied once per limit that its columns have, V zeroed
//     from the limit on: what lies behind a row's last position (stale pages, infinities) never meets it, not even
//     times zero.
// prefix_body, below, takes the prefix where many rows share it.
#pragma once

#include <algorithm>

#include "paged.hpp"

namespace cri {
namespace dev {

// n / d for 0 <= n < 2^31 by a host-made multiplier (page_index says why it is exact)
struct FastDiv {
    uint32_t magic;
    int shift;
};
inline FastDiv fast_div(int d) {
    int l = 0;
    while ((1L << l) < d) ++l;
    return FastDiv{static_cast<uint32_t>((1UL << (31 + l)) / d + 1), 31 + l};
}
__device__ __forceinline__ int div_by(int n, FastDiv d) {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * d.magic) >> d.shift);
}

struct PagedAttnArgs {
    const float* q;
    float* out;
    float* rec;  // [rows][H][nrec] records of D + 4 floats (max, sum, 2 pad, acc); unused when nrec is 1
    long ldq, ldo;
    PagePool P;
    PageBatch B;
    const int* prefix_pages;
    int prefix_len, H, G, nrec;
    // work of the prefix, by XCD: [chunk][KV head][row tile], an item per workgroup (staged) or wave; and of the
    // sequences, an item per wave: their first row tiles [chunk][sequence][KV head], then the others [chunk][KV head][tile]
    int pre_tiles, pre_chunks, pre_per, pre_blocks;
    int own_more, own_chunks, own_per, own_first;  // own_first: items of first tiles, own_more: other tiles at most
    FastDiv by_G, by_Hkv, by_pre_tiles, by_seqs, by_more;
    float qscale;  // scale * log2 e: scores are in base 2
    bool staged;   // the prefix is prefix_body's
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

// Probabilities in two fp16 parts.  One of 2^-15 of the running maximum and more keeps 22 bits.  Below, the parts reach fp16's
// smallest step, and what they leave is up to 2^-25 (in accumulators of 2^kShift times the sum) whatever the probability: over
// n positions an accumulator is off by up to n 2^-25 of the largest value.  That counts where the result is small against
// the values, as where a position of weight whose value is next to nothing stands before many others (an attention sink).  So
// a wave keeps the largest value that a row sees, and a row whose accumulators all are below 2^kSafe of that bound is done again
// with the probabilities as they are, by fp32 matrix instructions (rows_body with EXACT): it and no other row, or what
// a row does not see would reach its bits.  Rows that pass
// are within 2^-kSafe of their largest element, by this bound; as rounding goes they are at 2^-22.  Ordinary rows pass: a
// position of weight 1 puts 2^12 of its value into them, and the bar is 2^6 of the largest value over 8192 positions.
// Measured: the watch costs 1.5% (480 rows x 32 heads of 128 on 32768 positions 492 -> 500 us; 64 sequences of 1500 own
// positions 64.4 -> 64.7), 3 to 4% where it is not EVEN, 11% of a prefix of heads of 256 (567 -> 628).  Where every row has such
// a position in the prefix's first chunk, that chunk is done again by waves of their own: 496 -> 2228 us, 64 conversations
// on 8192 positions 60 -> 216; own positions 52 -> 59.
constexpr int kSafe = 18;
struct Largest {  // of fp16 numbers of either sign; a NaN stays one
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    h2 top = {0, 0}, low = {0, 0};
    __device__ __forceinline__ void add(uint32_t a, uint32_t b) {  // (two v_pk_maximum3 for four numbers)
        const h2 x = __builtin_bit_cast(h2, a), y = __builtin_bit_cast(h2, b);
        top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, x), y);
        low = __builtin_elementwise_minimum(__builtin_elementwise_minimum(low, x), y);
    }
    // the wave's largest magnitude, infinity where there are NaN
    __device__ __forceinline__ float of_wave() const {
        const h2 m = __builtin_elementwise_maximum(top, -low);
        const _Float16 most = __builtin_elementwise_maximum(m.x, m.y);
        return wave_max(most == most ? static_cast<float>(most) : INFINITY);
    }
};
// whether accumulators of largest magnitude `most` may be off by more than their share, n positions with values up to `value`
__device__ __forceinline__ bool too_small(float most, int n, float value) {
    constexpr float kStep = 1.0f / (1 << (25 - kSafe));
    return !(most >= static_cast<float>(n) * kStep * value);
}

__device__ __forceinline__ f32x4 mma16(const u32x4& a, const u32x4& b, const f32x4& c, std::integral_constant<int, kKvF16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const u32x4& a, const u32x4& b, const f32x4& c, std::integral_constant<int, kKvBF16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}

// the parts of eight floats (times f for fp16): x = p[0] + p[1] (+ p[2]), each the rest's rounding
template <int TYPE, int PARTS>
__device__ __forceinline__ void split8(const float (&x)[8], u32x4 (&p)[PARTS]) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    float r[8], one = 1.0f;
    h2 hi[4];
    if (TYPE == kKvF16) asm("" : "+s"(one));  // (opaque: a product by 1 would be folded away, and with it the v_fma_mix)
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f32x2 v = {r[2 * e], r[2 * e + 1]};
            if constexpr (TYPE == kKvF16) {
                h2 w;
                if (k == 0) {
                    w = __builtin_convertvector(v, h2);
                    hi[e] = w;
                } else {  // the rest and its rounding in one v_fma_mix each
                    w = h2{static_cast<_Float16>(fmaf(v.x, one, -static_cast<float>(hi[e].x))),
                           static_cast<_Float16>(fmaf(v.y, one, -static_cast<float>(hi[e].y)))};
                }
                p[k][e] = __builtin_bit_cast(uint32_t, w);
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

// The factors of a query row of largest magnitude m and of its raw scores: f before the products, kf within the
// exponential's fma, f kf = qscale.  kf is positive (f has the sign, and is 0 for a scale of 0), so the raw scores' maximum
// is the scaled ones' and a masked score of -infinity stays one.  For fp16 parts f also takes m to [2^13, 2^14): the parts
// are then off by 2^-23 of an element or 2^-39 of the largest.
template <int TYPE>
__device__ __forceinline__ void row_factors(float qscale, float m, float& f, float& kf) {
    constexpr float kTiny = 1.17549435e-38f;
    f = 1.0f;
    kf = fabsf(qscale);
    if constexpr (TYPE == kKvF16) {
        const int sh = min(13 + 127 - static_cast<int>(__builtin_bit_cast(uint32_t, m) >> 23), 126);
        f = __builtin_bit_cast(float, (127 + sh) << 23);
        kf *= __builtin_bit_cast(float, (127 - sh) << 23);
    }
    kf = fmaxf(kf, kTiny);
    f = qscale == 0.0f ? 0.0f : __builtin_copysignf(f, qscale);
}
// A sum of many small terms beside a large one: in one float a chunk's 8192 weights of 2^-24 beside one of 1 are lost, each in
// its rounding and all the same way, 1.5e-4 of the row as measured; so a tile's are added first, and what their addition
// rounds away is kept beside the sum (2e-6; under 1% of the time, 3% with heads of 256).  The accumulators, which add 16 or more
// terms at a time inside the matrix instructions, are left to fp32.
struct Sum {
    float hi = 0.0f, lo = 0.0f;
    __device__ __forceinline__ void add(float t) {
        const float s = hi + t;
        lo += t - (s - hi);  // (exact where hi is the larger; else off by an ulp of t, once per rise of the maximum)
        hi = s;
    }
    __device__ __forceinline__ void scale(float f) {
        hi *= f;
        lo *= f;
    }
    __device__ __forceinline__ float value() const { return hi + lo; }
};
__device__ __forceinline__ float col_max(float v) { return swap_max32(swap_max16(v, v), swap_max16(v, v)); }
__device__ __forceinline__ float col_sum(float v) {
    const float s = swap_add16(v, v);
    return swap_add32(s, s);
}
template <int CTRL>
__device__ __forceinline__ int dpp_i(int old, int v) {
    return __builtin_amdgcn_update_dpp(old, v, CTRL, 0xF, 0xF, false);
}
// the largest of the first 16 lanes (all rows of 16 hold the same values), in a scalar register
__device__ __forceinline__ int row_max_i(int v) {
    v = max(v, dpp_i<kQuadPerm1032>(v, v));
    v = max(v, dpp_i<kQuadPerm2301>(v, v));
    v = max(v, dpp_i<kRowHalfMirror>(v, v));
    v = max(v, dpp_i<kRowMirror>(v, v));
    return __builtin_amdgcn_readfirstlane(v);
}
// sums over the lanes up to and with each
__device__ __forceinline__ int wave_scan_i(int v) {
    v += dpp_i<0x111>(0, v);  // row_shr 1, 2, 4, 8: within 16 lanes, zeros from outside
    v += dpp_i<0x112>(0, v);
    v += dpp_i<0x114>(0, v);
    v += dpp_i<0x118>(0, v);
    const int lane = threadIdx.x & 63;
    const int a = __builtin_amdgcn_readlane(v, 15), b = __builtin_amdgcn_readlane(v, 31), c = __builtin_amdgcn_readlane(v, 47);
    return v + (lane >= 16 ? a : 0) + (lane >= 32 ? b : 0) + (lane >= 48 ? c : 0);
}
// int arrays that no kernel here writes, read at uniform places with scalar loads
typedef const __attribute__((address_space(4))) int* UniformInts;
__device__ __forceinline__ UniformInts uniform(const int* p) { return (UniformInts)p; }

// The sequences of up to 64 consecutive tokens t0 .. t0 + n - 1, lane l's being t0 + l's k: 64 offsets are read at a time
// and compared with every token, so that the searches of a wave cost one trip to memory.  Returns the position of token
// t0 + k in its sequence, or a negative number for a token of none (any below 0 is "before all positions").
__device__ __forceinline__ int position_of(const PageBatch& B, int t0, int n, int k, bool& found) {
    const int lane = threadIdx.x & 63;
    int s = 0;
    for (int base = 0; base < B.n_seqs; base += 64) {
        const int i = base + lane;
        const int end = i < B.n_seqs ? B.offsets[i + 1] : 0x7FFFFFFF;
        bool all = true;
        for (int j = 0; j < n; ++j) {
            const int before = __popcll(__ballot(end <= t0 + j));
            if (j == k) s += before;
            all = all && before < 64;
        }
        if (all) break;
    }
    found = false;
    if (k < n && s < B.n_seqs) {
        const int t = t0 + k, lo = B.offsets[s], hi = B.offsets[s + 1], len = max(B.lens[s], 0);
        found = t >= lo && t < hi;
        return len - (hi - t);
    }
    return -1;
}

// Work item i of the prefix.  The caller's items are consecutive on an XCD, so the row tiles of one chunk and KV head,
// which read the same K and V, meet in its L2.
__device__ __forceinline__ bool prefix_item(const PagedAttnArgs& a, int i, int Hkv, int& chunk, int& kvh, int& tile) {
    const int stream = div_by(i, a.by_pre_tiles);
    tile = i - stream * a.pre_tiles;
    chunk = div_by(stream, a.by_Hkv);
    kvh = stream - chunk * Hkv;
    return chunk < a.pre_chunks;
}
// workgroup b of n in the order of the XCDs that get them: b mod 8's first, n a multiple of 8
__device__ __forceinline__ int by_xcd(int b, int n) { return b % kPagedXcds * (n / kPagedXcds) + b / kPagedXcds; }

constexpr int kPrefixRows = 128;  // rows of a workgroup of prefix_body

// EVEN: head_dim is DP and the page size a multiple of 16, so the 16 positions of a tile's row block lie in one page.
// block: of pre_blocks workgroups of the prefix, then the sequences'.  Returns the columns that have to be done again (bit c),
// which are stored nowhere; EXACT (fp16) does columns `these` again with probabilities in fp32, of the item or of a half of
// a wave's rows in prefix_body.
template <int TYPE, int DP, bool EVEN, bool EXACT = false>
__device__ __forceinline__ uint32_t rows_body(const PagedAttnArgs& a, const int block, const int half = 0, const uint32_t these = 0) {
    typedef PagedShape<TYPE, DP> S;
    typedef typename KvType<TYPE>::elem elem;
    typedef std::integral_constant<int, TYPE> Type;
    constexpr int kTile = S::kTile, kT = S::kT, kKs = S::kKs, kVe = S::kVe, kNh = S::kNh, kAcc = S::kAcc;
    constexpr int kEs = sizeof(elem), kNs = 4 * kT;  // scores of a lane
    constexpr bool kWatch = TYPE == kKvF16 && !EXACT;

    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int D = EVEN ? DP : a.P.head_dim;
    const int Hkv = a.P.n_kv_heads, G = a.G;
    const uint32_t row_bytes = static_cast<uint32_t>(Hkv * D * kEs);
    const int cap = a.B.max_pages * a.P.page_size;
    const UniformInts offsets = uniform(a.B.offsets), lens = uniform(a.B.lens);

    // ---- what this wave does: a KV head, 16 rows, a range of positions
    const bool prefix = block < a.pre_blocks;
    int kvh, row0, nrows, tok0, pos0 = 0, rec_at, own_lo, own_hi;
    UniformInts own_table;
    int own_len, before_lo = 0, before_hi = 0;  // (before: the prefix's positions for rows that do not see all of it)
    const int prefix_pages = (a.prefix_len + a.P.page_size - 1) / a.P.page_size;
    if (prefix) {
        int chunk, tile;
        const int at = by_xcd(block, a.pre_blocks);
        const bool shared = EXACT && a.staged;
        if (!prefix_item(a, shared ? at : 4 * at + w, Hkv, chunk, kvh, tile)) return 0;
        row0 = shared ? tile * kPrefixRows + 32 * w + 16 * half : tile * 16;
        nrows = a.B.n_rows * G;
        tok0 = 0;
        rec_at = chunk;
        own_lo = chunk * a.pre_per;
        own_hi = min(own_lo + a.pre_per, a.prefix_len);
        own_table = uniform(a.prefix_pages);
        own_len = prefix_pages;
    } else {
        int item = 4 * (block - a.pre_blocks) + w, chunk, seq, tile = 0;
        if (item < a.own_first) {
            const int rest = div_by(item, a.by_Hkv);
            kvh = item - rest * Hkv;
            chunk = div_by(rest, a.by_seqs);
            seq = rest - chunk * a.B.n_seqs;
        } else {
            item -= a.own_first;
            const int rest = div_by(item, a.by_more);
            int more = item - rest * a.own_more;
            chunk = div_by(rest, a.by_Hkv);
            kvh = rest - chunk * Hkv;
            if (chunk >= a.own_chunks) return 0;
            // the more-th of the tiles behind the sequences' first ones: 64 sequences' counts summed at a time
            seq = -1;
            for (int base = 0; base < a.B.n_seqs; base += 64) {
                const int i = base + lane;
                int n = 0;
                if (i < a.B.n_seqs) n = min(max(a.B.offsets[i + 1] - a.B.offsets[i], 0), a.B.n_rows);
                const int tiles = max((n * G + 15) / 16 - 1, 0), sum = wave_scan_i(tiles);
                const int before = __popcll(__ballot(sum <= more));
                if (before < 64) {
                    seq = base + before;
                    tile = 1 + more - (before > 0 ? __builtin_amdgcn_readlane(sum, before - 1) : 0);
                    break;
                }
                more -= __builtin_amdgcn_readlane(sum, 63);
            }
            if (seq < 0 || seq >= a.B.n_seqs) return 0;
        }
        tok0 = offsets[seq];
        const int n = min(max(offsets[seq + 1] - tok0, 0), a.B.n_rows);
        if (n == 0) return 0;
        const int len = max(lens[seq], 0);
        row0 = tile * 16;
        nrows = n * G;
        pos0 = len - n;  // position of the sequence's first row
        rec_at = a.pre_chunks + chunk;
        const int end = min(len, cap), start = a.prefix_len / kTile * kTile;
        own_lo = min(start + chunk * a.own_per, end);
        own_hi = min(own_lo + a.own_per, end);
        own_lo = max(own_lo, min(a.prefix_len, end));
        own_table = uniform(a.B.pages + static_cast<long>(seq) * a.B.max_pages);
        own_len = a.B.max_pages;
        if (a.staged && pos0 + div_by(row0, a.by_G) + 1 < a.prefix_len) {
            const int hi = min(a.prefix_len, len);
            const int per = ((hi + a.own_chunks - 1) / a.own_chunks + kTile - 1) / kTile * kTile;
            before_lo = min(chunk * per, hi);
            before_hi = min(before_lo + per, hi);
        }
    }

    // ---- the lane's column: its row, the positions up to and with the row's own, its query operand
    int tok = -1, head = 0, sees = 0;
    {
        const int r = row0 + c, i0 = div_by(row0, a.by_G), i = div_by(r, a.by_G), t = tok0 + i;
        bool ok = r < nrows && t >= 0 && t < a.B.n_rows;
        int p = pos0 + i;
        if (prefix) {
            bool found;
            p = position_of(a.B, i0, min(div_by(row0 + 15, a.by_G), a.B.n_rows - 1) - i0 + 1, i - i0, found);
            ok = ok && found;
        }
        if (EXACT) ok = ok && (these >> c & 1) != 0;
        if (ok) {
            tok = t;
            head = kvh * G + r - i * G;
            sees = max(p + 1, 0);
        }
    }
    if (own_lo >= own_hi && before_lo >= before_hi && a.nrec > 1) {  // no positions: an empty record
        if (g == 0 && tok >= 0)
            *reinterpret_cast<f32x2*>(a.rec + ((static_cast<long>(tok) * a.H + head) * a.nrec + rec_at) * (D + 4)) =
                f32x2{-INFINITY, 0.0f};
        return 0;
    }
    // the query's row, under way while the first tile is looked up
    f32x4 raw[S::kWide ? kKs : 2 * kKs];
    {
        const float* src = a.q + static_cast<long>(max(tok, 0)) * a.ldq + static_cast<long>(head) * D;
#pragma unroll
        for (int j = 0; j < (S::kWide ? kKs : 2 * kKs); ++j) {
            const int d = S::kWide ? 16 * j + 4 * g : 32 * (j >> 1) + 8 * g + 4 * (j & 1);
            raw[j] = tok >= 0 && (EVEN || d < D) ? ld_f32x4(src + d) : f32x4{0, 0, 0, 0};
        }
    }

    // ---- the tiles
    const char* const kbase = static_cast<const char*>(a.P.k) + static_cast<long>(kvh) * D * kEs;
    const char* const vbase = static_cast<const char*>(a.P.v) + static_cast<long>(kvh) * D * kEs;
    // EVEN: a lane's bytes from the first row of a 16-position block; its address is that row's and these
    const uint32_t k_off = c * row_bytes + 16 * g, v_off = 4 * g * row_bytes + kVe * kEs * c;
    typedef uint32_t vreg __attribute__((ext_vector_type(S::kWide ? 4 : kVe / 2)));

    // A sequence's wave may have two ranges: where the prefix is left to prefix_body, first that part of it
    // that rows see which do not see it whole.
    int part = before_lo < before_hi ? 0 : 1, p_lo, p_hi, table_len, lim, least, first, last;
    UniformInts table;
    auto set_part = [&]() {
        p_lo = part ? own_lo : before_lo;
        p_hi = part ? own_hi : before_hi;
        table = part ? own_table : uniform(a.prefix_pages);
        table_len = part ? own_len : prefix_pages;
        // the positions the column sees; no row: everything, it is stored nowhere
        lim = tok < 0   ? 0x7FFFFFFF
              : prefix  ? min(sees, a.prefix_len)
              : part    ? min(sees, cap)
                        : sees < a.prefix_len ? sees : 0;
        least = -row_max_i(-lim);
        first = p_lo / kTile;
        last = (min(p_hi, row_max_i(tok < 0 ? 0 : lim)) + kTile - 1) / kTile;  // tiles [first, last)
    };
    auto page_at = [&](int pi) {
        const int pg = table[min(pi, table_len - 1)];
        return (static_cast<unsigned>(pg) < static_cast<unsigned>(a.P.n_pages) ? pg : 0) * a.P.stride * kEs;
    };
    auto row_at = [&](int pos) {  // byte offset of a position's row; uniform positions only where EVEN
        const int pi = page_index(a.P, pos);
        return page_at(pi) + static_cast<long>(pos - pi * a.P.page_size) * row_bytes;
    };
    auto lane_row = [&](int pos) {  // the same for a position of the lane's own
        const int pi = page_index(a.P, pos);
        const int pg = ((const int*)table)[min(pi, table_len - 1)];
        return (static_cast<unsigned>(pg) < static_cast<unsigned>(a.P.n_pages) ? pg : 0) * a.P.stride * kEs +
               static_cast<long>(pos - pi * a.P.page_size) * row_bytes;
    };
    auto load_k = [&](int p0, const long (&at)[kT], u32x4 (&k)[kT][kKs]) {
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            if constexpr (EVEN) {
                const char* row = kbase + at[t];
#pragma unroll
                for (int j = 0; j < kKs; ++j) k[t][j] = *reinterpret_cast<const u32x4*>(row + k_off + 64 * j);
            } else {
                const char* row = kbase + lane_row(p0 + 16 * t + c);
#pragma unroll
                for (int j = 0; j < kKs; ++j) {
                    const int d = 64 * j + 16 * g;  // bytes
                    const bool in = d < D * kEs;
                    k[t][j] = *reinterpret_cast<const u32x4*>(row + (in ? d : 0));
                    if (!in) k[t][j] = u32x4{0, 0, 0, 0};
                }
            }
        }
    };
    auto load_v = [&](int p0, const long (&at)[kT], vreg (&v)[kT][4][kNh]) {
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (EVEN) {
                    const char* row = vbase + at[t] + static_cast<long>(i) * row_bytes;
#pragma unroll
                    for (int h = 0; h < kNh; ++h)
                        v[t][i][h] = *reinterpret_cast<const vreg*>(row + v_off + 16 * kVe * kEs * h);
                } else {
                    const char* row = vbase + lane_row(p0 + 16 * t + 4 * g + i);
#pragma unroll
                    for (int h = 0; h < kNh; ++h) {
                        const int d = (16 * h + c) * kVe;
                        v[t][i][h] = *reinterpret_cast<const vreg*>(row + (d < D ? d * kEs : 0));
                    }
                }
            }
    };
    u32x4 k[kT][kKs];
    vreg v[kT][4][kNh];
    long at[kT] = {};
    auto load_tile = [&](int tile) {
        if constexpr (EVEN) {
#pragma unroll
            for (int t = 0; t < kT; ++t) at[t] = row_at(tile * kTile + 16 * t);
        }
        load_k(tile * kTile, at, k);
        load_v(tile * kTile, at, v);
    };
    set_part();
    if (first < last) load_tile(first);

    float kf, f;
    u32x4 q[S::kWide ? 1 : kKs][S::kParts];
    f32x4 q32[S::kWide ? kKs : 1];
    if constexpr (S::kWide) {
        row_factors<TYPE>(a.qscale, 0.0f, f, kf);
#pragma unroll
        for (int j = 0; j < kKs; ++j) q32[j] = raw[j] * f;
    } else {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * kKs; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(raw[j][e]));
        row_factors<TYPE>(a.qscale, col_max(m), f, kf);
#pragma unroll
        for (int j = 0; j < kKs; ++j) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = raw[2 * j + (e >> 2)][e & 3] * f;
            split8<TYPE, S::kParts>(x, q[j]);
        }
    }

    f32x4 acc[kAcc];
    float mx = -INFINITY;
    Sum weights;
    Largest values;      // of the tiles that every column sees as a whole
    float value = 0.0f;  // of the others, as far as this column sees them
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[i] = f32x4{0, 0, 0, 0};

#pragma unroll 1
    for (;;) {
#pragma unroll 1
        for (int tile = first; tile < last; ++tile) {
            const int p0 = tile * kTile;
            float s[kNs];
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                f32x4 x = {0, 0, 0, 0};
                if constexpr (S::kWide) {
#pragma unroll
                    for (int j = 0; j < kKs; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            x = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __builtin_bit_cast(float, static_cast<uint32_t>(k[t][j][e])), q32[j][e], x, 0, 0, 0);
                } else {
#pragma unroll
                    for (int p = S::kParts - 1; p >= 0; --p)
#pragma unroll
                        for (int j = 0; j < kKs; ++j) x = mma16(k[t][j], q[j][p], x, Type{});
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * t + i] = x[i];  // (raw: the factor comes with the exponential)
            }
            const int next = p0 + kTile;
            const bool more = tile + 1 < last;
            if (more) {  // the next tile's keys, in flight during the softmax and the second product
                if constexpr (EVEN) {
#pragma unroll
                    for (int t = 0; t < kT; ++t) at[t] = row_at(next + 16 * t);
                }
                load_k(next, at, k);
            }
            const bool whole = p0 >= p_lo && p0 + kTile <= min(p_hi, least);
            if (!whole) {
                const int hi = min(p_hi, lim);
#pragma unroll
                for (int t = 0; t < kT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int p = p0 + 16 * t + 4 * g + i;
                        if (p < p_lo || p >= hi) s[4 * t + i] = -INFINITY;
                    }
            }
            float m = s[0];
#pragma unroll
            for (int i = 1; i < kNs; ++i) m = fmaxf(m, s[i]);
            m = col_max(m) * kf;
            const bool raise = m > mx + S::kSlack;
            if (__ballot(raise) != 0) {
                const float f = raise ? __builtin_amdgcn_exp2f(mx - m) : 1.0f;
                if (raise) mx = m;
                weights.scale(f);
#pragma unroll
                for (int i = 0; i < kAcc; ++i) acc[i] *= f;
            }
            const float base = (mx == -INFINITY ? 0.0f : mx) - S::kShift;
            float p[8] = {}, tile_sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kNs; ++i) {
                p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], kf, -base));
                tile_sum += p[i];
            }
            weights.add(tile_sum);
            u32x4 pb[S::kParts];
            if constexpr (!S::kWide && !EXACT) split8<TYPE, S::kParts>(p, pb);
            // the tile's values, if masked those of its positions [lo, hi)
            auto watch = [&](auto masked, Largest& l, int lo, int hi) {
#pragma unroll
                for (int t = 0; t < kT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = 16 * t + 4 * g + i;
                        const uint32_t on = !decltype(masked)::value || (at >= lo && at < hi) ? 0xFFFFFFFFu : 0u;
#pragma unroll
                        for (int h = 0; h < kNh; ++h)
#pragma unroll
                            for (int e = 0; e < kVe / 2; e += 2) l.add(v[t][i][h][e] & on, v[t][i][h][e + 1] & on);
                    }
            };
            // O^T += V^T P^T; `from` zeroes the positions from there on (an index into the tile) and those before p_lo
            auto multiply = [&](auto masked, int from, bool mine) {
                constexpr bool kMask = decltype(masked)::value;
                const int lo = kMask ? p_lo - p0 : 0;
                uint32_t low = 0x05040100u, high = 0x07060302u;  // byte permutations: the rows' low or high halves
                // (opaque, or the permuted rows of every limit's round would be kept in registers across the rounds)
                if (kMask) asm volatile("" : "+s"(low), "+s"(high));
#pragma unroll
                for (int h = 0; h < kNh; ++h)
#pragma unroll
                    for (int e = 0; e < kVe; ++e) {
                        f32x4 x = acc[h * kVe + e];
                        if constexpr (S::kWide) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float u = __builtin_bit_cast(float, static_cast<uint32_t>(v[0][i][h][e]));
                                if (kMask && (4 * g + i < lo || 4 * g + i >= from)) u = 0.0f;
                                x = __builtin_amdgcn_mfma_f32_16x16x4f32(u, p[i], x, 0, 0, 0);
                            }
                        } else if constexpr (EXACT) {
                            __builtin_amdgcn_sched_barrier(0);  // (registers before speed: one element of V at a time)
#pragma unroll
                            for (int t = 0; t < kT; ++t)
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const int at = 16 * t + 4 * g + i;
                                    const uint32_t r = v[t][i][h][e >> 1];
                                    float u = static_cast<float>(
                                        __builtin_bit_cast(_Float16, static_cast<uint16_t>(e & 1 ? r >> 16 : r)));
                                    if (kMask && (at < lo || at >= from)) u = 0.0f;
                                    x = __builtin_amdgcn_mfma_f32_16x16x4f32(u, p[4 * t + i], x, 0, 0, 0);
                                }
                        } else {
                            // dim e of the lane's eight positions: halves of two rows' dwords
                            u32x4 f;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int t = j >> 1, i = 2 * (j & 1);
                                const uint32_t lo16 = v[t][i][h][e >> 1], hi16 = v[t][i + 1][h][e >> 1];
                                f[j] = __builtin_amdgcn_perm(hi16, lo16, e & 1 ? high : low);
                                if (kMask) {
                                    const int at0 = 16 * t + 4 * g + i;
                                    if (at0 < lo || at0 >= from) f[j] &= 0xFFFF0000u;
                                    if (at0 + 1 < lo || at0 + 1 >= from) f[j] &= 0x0000FFFFu;
                                }
                            }
#pragma unroll
                            for (int k = S::kParts - 1; k >= 0; --k) x = mma16(f, pb[k], x, Type{});
                        }
                        if constexpr (kMask) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[h * kVe + e][i] = mine ? x[i] : acc[h * kVe + e][i];
                        } else {
                            acc[h * kVe + e] = x;
                        }
                    }
            };
            if (!EXACT && whole) {
                multiply(std::false_type{}, 0, true);
                if constexpr (kWatch) {
                    __builtin_amdgcn_sched_barrier(0);
                    watch(std::false_type{}, values, 0, 0);
                }
            } else {  // once per limit that the tile's columns have
                const int rel = min(max(min(p_hi, lim) - p0, 0), kTile);
                for (unsigned long left = __ballot(rel > 0); left != 0;) {
                    const int from = __builtin_amdgcn_readlane(rel, __builtin_ctzl(left));
                    multiply(std::true_type{}, from, rel == from);
                    if constexpr (kWatch) {
                        __builtin_amdgcn_sched_barrier(0);
                        Largest some;
                        watch(std::true_type{}, some, p_lo - p0, from);
                        const float most = some.of_wave();
                        if (rel == from) value = fmaxf(value, most);
                    }
                    left &= ~__ballot(rel == from);
                }
            }
            if (more) load_v(next, at, v);
        }
        if (part == 1) break;
        part = 1;
        set_part();
        if (first < last) load_tile(first);
    }

    // ---- the record, or the output
    uint32_t again = 0;
    if constexpr (kWatch) {
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < kAcc; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(acc[i][e]));
        big = col_max(big);
        value = fmaxf(value, values.of_wave());
        const int n = own_hi - own_lo + before_hi - before_lo;
        again = __ballot(tok >= 0 && mx != -INFINITY && too_small(big, n, value)) & 0xFFFF;
        if ((again >> c & 1) != 0) tok = -1;
    }
    const float sum = col_sum(weights.value());
    if (sum != sum) mx = INFINITY;  // NaN scores leave no maximum: keep the record from being skipped
    if (tok < 0) return again;
    float* dst;
    float back = 1.0f;
    if (a.nrec == 1) {
        dst = a.out + tok * a.ldo + static_cast<long>(head) * D;
        back = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees nothing: zeros
    } else {
        dst = a.rec + ((static_cast<long>(tok) * a.H + head) * a.nrec + rec_at) * (D + 4);
        if (g == 0) *reinterpret_cast<f32x2*>(dst) = f32x2{mx, sum};
        dst += 4;
        if (mx == -INFINITY) return again;
    }
#pragma unroll
    for (int h = 0; h < kNh; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < kVe; e += 4) {
                const int d = 16 * kVe * h + kVe * (4 * g + i) + e;  // of acc[h kVe + e ..][i]
                if (EVEN || d < D)
                    *reinterpret_cast<f32x4_a4*>(dst + d) =
                        f32x4_a4{acc[h * kVe + e][i] * back, acc[h * kVe + e + 1][i] * back, acc[h * kVe + e + 2][i] * back,
                                 acc[h * kVe + e + 3][i] * back};
            }
    return again;
}

// The shared prefix against many rows.  A workgroup of four waves takes 128 rows, 32 to a wave, and a chunk of the
// prefix in tiles of 32 positions that all its waves read from LDS: straight from the pool every wave would load 16 KB
// for the 2 x 0.5 MFLOP it does with a tile, more than the L1 delivers beside the matrix instructions.
// v_mfma_f32_32x32x16: half the instructions of 16x16x32 for the same product.
//   * 16-bit tiles go to LDS with global_load_lds, whole rows at a time, into rings of four, three tiles ahead; one barrier per
//     tile.  The 16-byte pieces of a row are exchanged within it: K's so that the 32 rows of an operand fetch lie in
//     different banks, V's so that the four rows that ds_read_b64_tr_b16 takes apart do (16 lanes read 4 positions x 16
//     dims and get a dim's 4 positions each: V^T's operand without a byte permutation).  No bank conflicts are counted.
//   * fp32 tiles go through registers, where K and V are cut into three bf16 parts, 8 bits of the significand each (exact, and
//     of fp32's range); a product is the six of parts down to 2^-16, each exact in fp32.  v_mfma_f32_32x32x16_bf16 does 16
//     times the multiply-adds per cycle of the fp32 instructions, so the six cost 0.38 of their cycles (512 rows of a KV
//     head on 8192 positions 222 -> 115 us, 256 rows 118 -> 73), at the same distance from float64.
// 480 rows x 32 heads of 128 on 32768 positions of fp16: 493 us, 1045 TFLOP/s of fp16 products, two for each of the
// formula's, where a large library product runs at 1150 (bf16, three: 620 us, 1247 against 1207).  The matrix units are busy
// for half the cycles at 1.9 GHz (the clock under this load; nothing but these instructions on random numbers reach 1600
// TFLOP/s), the rest is the exponentials and parts, about 110 vector instructions and 16 exponentials per wave and tile to
// 32 products.  Issuing the next tile's scores between them, and operands read ahead, were measured at 562 to 585 us against
// 541: more registers, the same power.
constexpr int kPrefixTile = 32, kRing = 4;
constexpr int prefix_lds(int type, int dp) { return 2 * (type == kKvF32 ? 3 : kRing) * kPrefixTile * dp * 2; }

typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f32x16 mma32(const u32x4& a, const u32x4& b, const f32x16& c, std::integral_constant<int, kKvF16>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(const u32x4& a, const u32x4& b, const f32x16& c, std::integral_constant<int, kKvBF16>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
// 16 bytes per lane from global memory into LDS (lane l at byte 16 l of the wave-uniform lds)
__device__ __forceinline__ void dma16(const void* g, char* lds) { __builtin_amdgcn_global_load_lds(g, lds, 16, 0, 0); }
// lanes 4 k + a of each 16 give the address of row k's 4 a-th element, lane i gets element i of rows 0 .. 3
__device__ __forceinline__ u32x2 read_transposed(const char* p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* Ptr;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(p)));
}
// eight floats as three bf16 parts each, the 8 bits of the significand that remain at a time: exact
__device__ __forceinline__ void cut8(const f32x4 (&x)[2], u32x4 (&p)[3]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a = x[e >> 1][2 * (e & 1)], b = x[e >> 1][2 * (e & 1) + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const uint32_t u = __builtin_bit_cast(uint32_t, a), v = __builtin_bit_cast(uint32_t, b);
            p[k][e] = __builtin_amdgcn_perm(v, u, 0x07060302u);
            a -= __builtin_bit_cast(float, u & 0xFFFF0000u);
            b -= __builtin_bit_cast(float, v & 0xFFFF0000u);
        }
    }
}
template <int N>
__device__ __forceinline__ void wait_copies() {  // all but the last N copies of this wave have arrived
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// EVEN: head_dim is DP and the page size a multiple of 16.  Else every lane looks up the page of its own row (a tile ahead of
// the copy that needs it), pieces behind head_dim are the row's first one again (the query is zero there) and blocks of dims
// behind it are not multiplied: 480 rows x 32 heads on 32768 positions, pages of 20 538 us (waves of their own 1437), heads of
// 80 432 (1347), 40 309 (996).
// Returns the wave's rows that have to be done again (bit i), which are stored nowhere.
template <int TYPE, int DP, bool EVEN>
__device__ __forceinline__ uint32_t prefix_body(const PagedAttnArgs& a, const int block, char* const ring) {
    constexpr bool kWide = TYPE == kKvF32;                        // K and V, too, are taken in three bf16 parts
    constexpr int kMath = kWide ? kKvBF16 : TYPE, kKv = kWide ? 3 : 1;
    typedef PagedShape<kMath, DP> S;
    typedef std::integral_constant<int, kMath> Type;
    constexpr int kParts = S::kParts, kKs = DP / 16, kDb = DP / 32, kRowB = 2 * DP, kPieces = kRowB / 16;
    // bytes of (a part of) a tile's K or V; ring: K's tiles or parts, then V's
    constexpr int kTileB = kPrefixTile * kRowB, kValues = (kWide ? kKv : kRing) * kTileB;
    constexpr int kCopies = kTileB / 1024 / 4;  // of a wave, of a tile's K or V

    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int Hkv = a.P.n_kv_heads, G = a.G, nrows = a.B.n_rows * G, D = EVEN ? DP : a.P.head_dim;
    constexpr int kEs = kWide ? 4 : 2;
    const uint32_t row_bytes = static_cast<uint32_t>(Hkv) * D * kEs;
    int chunk, kvh, tile;
    if (!prefix_item(a, by_xcd(block, a.pre_blocks), Hkv, chunk, kvh, tile)) return 0;
    const int p_lo = chunk * a.pre_per, p_hi = min(p_lo + a.pre_per, a.prefix_len);
    const int ntiles = (p_hi - p_lo + kPrefixTile - 1) / kPrefixTile;
    const int table_len = (a.prefix_len + a.P.page_size - 1) / a.P.page_size;

    // ---- the copies: a wave's rows of a tile lie in one page (8 rows each; 16 share a page)
    const char* const kbase = static_cast<const char*>(a.P.k) + static_cast<long>(kvh) * D * kEs;
    const char* const vbase = static_cast<const char*>(a.P.v) + static_cast<long>(kvh) * D * kEs;
    auto k_mix = [&](int row) { return DP >= 128 ? row & 15 : (row >> 1) & 7; };
    auto v_mix = [&](int row) { return DP >= 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; };
    auto real = [&](int piece) { return EVEN || 8 * piece < D ? piece : 0; };
    constexpr int kCopyRows = 64 / kPieces;
    uint32_t k_off[kCopies], v_off[kCopies];  // bytes of the lane's pieces from the wave's first row (not EVEN: from their own)
#pragma unroll
    for (int n = 0; n < kCopies; ++n) {
        const int r = n * kCopyRows + lane / kPieces, row = 8 * w + r;
        k_off[n] = (EVEN ? r * row_bytes : 0) + 16 * real(lane % kPieces ^ k_mix(row));
        v_off[n] = (EVEN ? r * row_bytes : 0) + 16 * real(lane % kPieces ^ v_mix(row));
    }
    auto row_at = [&](int pos) {  // byte offset of a (uniform) position's row
        const int pi = page_index(a.P, pos);
        const int pg = uniform(a.prefix_pages)[min(pi, table_len - 1)];
        return (static_cast<unsigned>(pg) < static_cast<unsigned>(a.P.n_pages) ? pg : 0) * a.P.stride * kEs +
               static_cast<long>(pos - pi * a.P.page_size) * row_bytes;
    };
    // fp32: a thread's pieces, eight elements of a row each, through registers, cut into parts on their way to LDS
    constexpr int kMine = kWide ? kPrefixTile * kPieces / 256 : 1;
    constexpr int kIds = kWide ? kMine : kCopies;  // rows of a tile that a lane has pieces of
    auto lane_pos = [&](int t, int n) {
        const int row = kWide ? (256 * n + static_cast<int>(threadIdx.x)) / kPieces : 8 * w + n * kCopyRows + lane / kPieces;
        return p_lo + min(t, ntiles - 1) * kPrefixTile + row;
    };
    int ids[kIds] = {};  // their pages, of the tile that is copied next
    auto look_up = [&](int t, int (&ids)[kIds]) {
#pragma unroll
        for (int n = 0; n < kIds; ++n) ids[n] = a.prefix_pages[min(page_index(a.P, lane_pos(t, n)), table_len - 1)];
    };
    auto lane_row = [&](int t, int n, int pg) {  // byte offset of a lane's row
        const int pos = lane_pos(t, n);
        return (static_cast<unsigned>(pg) < static_cast<unsigned>(a.P.n_pages) ? pg : 0) * a.P.stride * kEs +
               static_cast<long>(pos - page_index(a.P, pos) * a.P.page_size) * row_bytes;
    };
    // tile t (past the last one: that one again, so that every turn issues as many), its lanes' pages in ids, which get those
    // of tile t + ahead
    auto copy = [&](int t, int (&ids)[kIds], int ahead) {
        char* const dst = ring + t % kRing * kTileB + 8 * w * kRowB;
        if constexpr (EVEN) {
            const long at = row_at(p_lo + min(t, ntiles - 1) * kPrefixTile + 8 * w);
#pragma unroll
            for (int n = 0; n < kCopies; ++n) dma16(kbase + at + k_off[n], dst + n * 1024);
#pragma unroll
            for (int n = 0; n < kCopies; ++n) dma16(vbase + at + v_off[n], dst + kValues + n * 1024);
        } else {
            long at[kCopies];
#pragma unroll
            for (int n = 0; n < kCopies; ++n) at[n] = lane_row(t, n, ids[n]);
            if (ahead > 0) look_up(t + ahead, ids);
#pragma unroll
            for (int n = 0; n < kCopies; ++n) dma16(kbase + at[n] + k_off[n], dst + n * 1024);
#pragma unroll
            for (int n = 0; n < kCopies; ++n) dma16(vbase + at[n] + v_off[n], dst + kValues + n * 1024);
        }
    };
    f32x4 kr[kMine][2], vr[kMine][2];
    auto load = [&](int t) {
#pragma unroll
        for (int n = 0; n < kMine; ++n) {
            const int row = (256 * n + static_cast<int>(threadIdx.x)) / kPieces, row0 = (256 * n + 64 * w) / kPieces;
            const long at = EVEN ? row_at(p_lo + min(t, ntiles - 1) * kPrefixTile + row0) : lane_row(t, n, ids[n]);
            const uint32_t off = (EVEN ? (row - row0) * row_bytes : 0) + 32 * real(threadIdx.x % kPieces);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                kr[n][x] = *reinterpret_cast<const f32x4*>(kbase + at + off + 16 * x);
                vr[n][x] = *reinterpret_cast<const f32x4*>(vbase + at + off + 16 * x);
            }
        }
        if constexpr (!EVEN) look_up(t + 1, ids);
    };
    auto store = [&](int t) {
#pragma unroll
        for (int n = 0; n < kMine; ++n) {
            const int row = (256 * n + static_cast<int>(threadIdx.x)) / kPieces, piece = threadIdx.x % kPieces;
            if (t * kPrefixTile + row >= p_hi - p_lo)  // past the prefix: zeros, whatever the page holds
                kr[n][0] = kr[n][1] = vr[n][0] = vr[n][1] = f32x4{0, 0, 0, 0};
            u32x4 p[3];
            cut8(kr[n], p);
#pragma unroll
            for (int x = 0; x < 3; ++x)
                *reinterpret_cast<u32x4*>(ring + x * kTileB + row * kRowB + 16 * (piece ^ k_mix(row))) = p[x];
            cut8(vr[n], p);
#pragma unroll
            for (int x = 0; x < 3; ++x)
                *reinterpret_cast<u32x4*>(ring + kValues + x * kTileB + row * kRowB + 16 * (piece ^ v_mix(row))) = p[x];
        }
    };
    if constexpr (kWide) {
        if constexpr (!EVEN) look_up(0, ids);
        load(0);
    } else {
        int ids1[kIds] = {}, ids2[kIds] = {};
        if constexpr (!EVEN) {
            look_up(0, ids);
            look_up(1, ids1);
            look_up(2, ids2);
        }
        copy(0, ids, 3);
        copy(1, ids1, 0);
        copy(2, ids2, 0);
    }

    // ---- the lane's row and query operand.  Rows that do not see the whole prefix are left to the workgroups of their
    // sequences: here they get empty records.
    const int row0 = tile * kPrefixRows + 32 * w, r = row0 + i, t0 = div_by(row0, a.by_G), t = div_by(r, a.by_G);
    bool found;
    const int pos = position_of(a.B, t0, min(div_by(row0 + 31, a.by_G), a.B.n_rows - 1) - t0 + 1, t - t0, found);
    const int tok = found && r < nrows ? t : -1, head = kvh * G + r - t * G;
    const bool sees = tok >= 0 && pos + 1 >= a.prefix_len;
    u32x4 q[kKs][kParts];
    float kf;
    {
        const float* src = a.q + static_cast<long>(max(tok, 0)) * a.ldq + static_cast<long>(head) * D + 8 * h;
        float x[kKs][8], m = 0.0f;
#pragma unroll
        for (int j = 0; j < kKs; ++j)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const f32x4 v = sees && (EVEN || 16 * j + 8 * h + e < D) ? ld_f32x4(src + 16 * j + e) : f32x4{0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    x[j][e + d] = v[d];
                    m = fmaxf(m, fabsf(v[d]));
                }
            }
        float f;
        row_factors<kMath>(a.qscale, swap_max32(m, m), f, kf);
#pragma unroll
        for (int j = 0; j < kKs; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[j][e] *= f;
            split8<kMath, kParts>(x[j], q[j]);
        }
    }

    const bool active = __ballot(sees) != 0;  // (a wave without rows copies and waits with the others)
    f32x16 o[kDb];
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
    float mx = -INFINITY;
    Sum weights;

    // the raw scores of tile t, a lane's 16: positions 8 (v >> 2) + 4 h + (v & 3)
    const char* const k_at = ring + i * kRowB;
    // (parts: products of the small ones first, those of a K part and a query part below 2^-24 of the whole left out)
    auto scores = [&](int t, f32x16& s) {
        const char* const kt = k_at + (kWide ? 0 : t % kRing * kTileB);
        const f32x16 zero = {};
        bool first = true;
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) {
            if (!EVEN && 16 * ks >= D) break;
#pragma unroll
            for (int x = kKv - 1; x >= 0; --x) {
                const u32x4 k = *reinterpret_cast<const u32x4*>(kt + x * kTileB + 16 * ((2 * ks + h) ^ k_mix(i)));
#pragma unroll
                for (int p = kParts - 1 - x; p >= 0; --p) {
                    s = mma32(k, q[ks][p], first ? zero : s, Type{});
                    first = false;
                }
            }
        }
    };
    auto largest = [&](int t, f32x16& s) {
        const int left = p_hi - p_lo - t * kPrefixTile;
        if (left < kPrefixTile) {  // the prefix ends in this tile
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if (8 * (v >> 2) + 4 * h + (v & 3) >= left) s[v] = -INFINITY;
        }
        float m = s[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) m = fmaxf(m, s[v]);
        return swap_max32(m, m) * kf;
    };
    // V^T's operand of dim block d and positions 16 b .. : two reads of 4 x 16
    Largest values;  // of the wave's quarter of every tile
    const int v_row = 4 * h + ((lane >> 2) & 3), v_col = 32 * ((lane >> 4) & 1) + 8 * (lane & 3);  // row, byte in 64
    for (int tl = 0; tl < ntiles; ++tl) {
        if constexpr (kWide) {
            store(tl);
            __syncthreads();
            load(tl + 1);
        } else {
            wait_copies<4 * kCopies>();  // tile tl
            __syncthreads();
            copy(tl + 3, ids, 1);
        }
        if (!kWide && p_hi - p_lo - tl * kPrefixTile < kPrefixTile) {  // past the prefix: zeros, whatever the page holds
            const int left = p_hi - p_lo - tl * kPrefixTile;
            for (int x = threadIdx.x; x < (kPrefixTile - left) * kPieces; x += 256)
                *reinterpret_cast<u32x4*>(ring + kValues + tl % kRing * kTileB + left * kRowB + 16 * x) = u32x4{0, 0, 0, 0};
            __syncthreads();
        }
        if constexpr (TYPE == kKvF16) {  // (a block of its own: among the products its reads cost 14 to 140 spilled registers)
            const char* const at = ring + kValues + tl % kRing * kTileB + w * (kTileB / 4) + 16 * lane;
#pragma unroll
            for (int x = 0; x < kTileB / 4; x += 1024) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(at + x);
                values.add(v[0], v[1]);
                values.add(v[2], v[3]);
            }
        }
        if (active) {
            f32x16 s;
            scores(tl, s);
            const float m = largest(tl, s);
            const bool raise = m > mx + S::kSlack;
            if (__ballot(raise) != 0) {
                const float f = raise ? __builtin_amdgcn_exp2f(mx - m) : 1.0f;
                if (raise) mx = m;
                weights.scale(f);
#pragma unroll
                for (int d = 0; d < kDb; ++d) o[d] *= f;
            }
            const float base = (mx == -INFINITY ? 0.0f : mx) - S::kShift;
            u32x4 pb[2][kParts];
            float tile_sum = 0.0f;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(fmaf(s[8 * b + e], kf, -base));
                    tile_sum += p[e];
                }
                split8<kMath, kParts>(p, pb[b]);
            }
            weights.add(tile_sum);
            const char* const vt = ring + kValues + (kWide ? 0 : tl % kRing * kTileB);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int d = 0; d < kDb; ++d) {
                    if (!EVEN && 32 * d >= D) break;
#pragma unroll
                    for (int y = kKv - 1; y >= 0; --y) {
                        u32x4 v;
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int row = 16 * b + 8 * x + v_row;  // row & 3 and (row >> 1) & 1 are the lane's own
                            const u32x2 z =
                                read_transposed(vt + y * kTileB + row * kRowB + ((64 * d) ^ (16 * v_mix(v_row))) + v_col);
                            v[2 * x] = z.x;
                            v[2 * x + 1] = z.y;
                        }
#pragma unroll
                        for (int p = kParts - 1 - y; p >= 0; --p) o[d] = mma32(v, pb[b][p], o[d], Type{});
                    }
                }
        }
        if constexpr (kWide) __syncthreads();  // the parts have been read
    }
    if constexpr (!kWide) wait_copies<0>();
    uint32_t again = 0;
    if constexpr (TYPE == kKvF16) {
        float big = 0.0f;
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) big = fmaxf(big, fabsf(o[d][v]));
        big = swap_max32(big, big);
        const float mine = values.of_wave();
        float* const quarters = reinterpret_cast<float*>(ring);
        __syncthreads();  // the ring has been read, and no copy is under way
        if (lane == 0) quarters[w] = mine;
        __syncthreads();
        const float value = fmaxf(fmaxf(quarters[0], quarters[1]), fmaxf(quarters[2], quarters[3]));
        again = static_cast<uint32_t>(__ballot(sees && mx != -INFINITY && too_small(big, p_hi - p_lo, value)));
    }
    float sum = weights.value();
    sum = swap_add32(sum, sum);
    if (sum != sum) mx = INFINITY;  // NaN scores leave no maximum: keep the record from being skipped
    if (!sees) mx = -INFINITY;
    if (tok < 0 || (again >> i & 1) != 0) return again;
    float* dst = a.rec + ((static_cast<long>(tok) * a.H + head) * a.nrec + chunk) * (D + 4);
    if (h == 0) *reinterpret_cast<f32x2*>(dst) = f32x2{mx, sees ? sum : 0.0f};
    if (mx == -INFINITY) return again;
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
        for (int v = 0; v < 16; v += 4)
            if (EVEN || 32 * d + 2 * v + 4 * h < D)
                *reinterpret_cast<f32x4*>(dst + 4 + 32 * d + 2 * v + 4 * h) = f32x4{o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]};
    return again;
}

// The columns that a body has left (rows of prefix_body: 16 and 16), with exact probabilities.
// The kernel's arguments (its only one: a PagedAttnArgs) are loaded again, from where the compiler cannot know them: or it
// would keep them, and what it computed of them, in registers over the bodies' loops for the sake of this rare path.
template <int TYPE, int DP, bool EVEN>
__device__ __forceinline__ void rows_again(const int block, const uint32_t left) {
    if constexpr (TYPE == kKvF16) {
        const uint32_t columns = __builtin_amdgcn_readfirstlane(left);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            const uint32_t these = columns >> 16 * half & 0xFFFF;
            if (these == 0) continue;
            auto args = (const __attribute__((address_space(4))) PagedAttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
            asm volatile("" : "+s"(args));
            rows_body<TYPE, DP, EVEN, true>(*(const PagedAttnArgs*)args, block, half, these);
        }
    }
}

template <int TYPE, int DP, bool EVEN>
__global__ __launch_bounds__(64 * kPagedWaves, DP <= 128 ? 2 : 1) void paged_attn_kernel(const PagedAttnArgs a) {
    const int block = blockIdx.x + (a.staged ? a.pre_blocks : 0);
    rows_again<TYPE, DP, EVEN>(block, rows_body<TYPE, DP, EVEN>(a, block));
}
// The prefix's workgroups and behind them the sequences', in one launch: the former are bound by the matrix instructions,
// the latter by memory and by the trips to it before their first tile, and a CU holds one of each (64 conversations on
// 8192 tokens: 67 us, 90 in two launches; 480 rows on 32768: 487 and 510, both before kSafe's watch).
template <int TYPE, int DP, bool EVEN>
__global__ __launch_bounds__(64 * kPagedWaves, 2) void paged_mixed_kernel(const PagedAttnArgs a) {
    __shared__ __attribute__((aligned(16))) char ring[prefix_lds(TYPE, DP)];
    uint32_t left;
    if (static_cast<int>(blockIdx.x) < a.pre_blocks)
        left = prefix_body<TYPE, DP, EVEN>(a, blockIdx.x, ring);
    else
        left = rows_body<TYPE, DP, EVEN>(a, blockIdx.x);
    rows_again<TYPE, DP, EVEN>(blockIdx.x, left);
}
// Heads over 128: the queries and accumulators alone take more than half of a SIMD's registers and the ring 128 KB, one
// workgroup to a CU, so the sequences' workgroups have a launch of their own.  16 heads of 256, 480 rows on 32768
// positions of fp16: 655 us (waves of their own 1316); bf16's third part spills 40 registers, 1048 (1399).
template <int TYPE, bool EVEN>
__global__ __launch_bounds__(64 * kPagedWaves, 1) void paged_prefix_kernel(const PagedAttnArgs a) {
    __shared__ __attribute__((aligned(16))) char ring[prefix_lds(TYPE, 256)];
    rows_again<TYPE, 256, EVEN>(blockIdx.x, prefix_body<TYPE, 256, EVEN>(a, blockIdx.x, ring));
}

template <int TYPE, int DP, bool EVEN>
void run_paged_attn(const PagedAttnArgs& a, int blocks, hipStream_t stream) {
    hipLaunchKernelGGL((paged_attn_kernel<TYPE, DP, EVEN>), dim3(blocks), dim3(64 * kPagedWaves), 0, stream, a);
}

template <int TYPE>
void run_paged_attn_type(const PagedAttnArgs& a, bool even, int blocks, hipStream_t stream) {
    const int D = a.P.head_dim;
    if (D <= 64)
        even ? run_paged_attn<TYPE, 64, true>(a, blocks, stream) : run_paged_attn<TYPE, 64, false>(a, blocks, stream);
    else if (D <= 128)
        even ? run_paged_attn<TYPE, 128, true>(a, blocks, stream) : run_paged_attn<TYPE, 128, false>(a, blocks, stream);
    else
        even ? run_paged_attn<TYPE, 256, true>(a, blocks, stream) : run_paged_attn<TYPE, 256, false>(a, blocks, stream);
}

template <int TYPE>
void run_paged_mixed_type(const PagedAttnArgs& a, bool even, int own_blocks, hipStream_t stream) {
    const int D = a.P.head_dim;
    if (D > 128) {
        if constexpr (TYPE != kKvF32)  // (three parts of both, and of 256 dims, do not fit the registers)
            hipLaunchKernelGGL((even ? paged_prefix_kernel<TYPE, true> : paged_prefix_kernel<TYPE, false>), dim3(a.pre_blocks),
                               dim3(64 * kPagedWaves), 0, stream, a);
        return run_paged_attn_type<TYPE>(a, even, own_blocks, stream);
    }
    const auto run = D <= 64 ? (even ? paged_mixed_kernel<TYPE, 64, true> : paged_mixed_kernel<TYPE, 64, false>)
                             : (even ? paged_mixed_kernel<TYPE, 128, true> : paged_mixed_kernel<TYPE, 128, false>);
    hipLaunchKernelGGL(run, dim3(a.pre_blocks + own_blocks), dim3(64 * kPagedWaves), 0, stream, a);
}

void run_paged_mixed_f32(const PagedAttnArgs& a, bool even, int own_blocks, hipStream_t stream);
void run_paged_mixed_f16(const PagedAttnArgs& a, bool even, int own_blocks, hipStream_t stream);
void run_paged_mixed_bf16(const PagedAttnArgs& a, bool even, int own_blocks, hipStream_t stream);
void run_paged_attn_f32(const PagedAttnArgs& a, bool even, int blocks, hipStream_t stream);
void run_paged_attn_f16(const PagedAttnArgs& a, bool even, int blocks, hipStream_t stream);
void run_paged_attn_bf16(const PagedAttnArgs& a, bool even, int blocks, hipStream_t stream);

}  // namespace dev
}  // namespace cri
