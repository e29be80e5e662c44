// paged_attention.hip -- how a call of the paged attention is cut into workgroups, and the kernel that joins their
// records.
#include <numeric>

#include "paged_attention.hpp"

namespace cri {
namespace dev {
namespace {

// The records of a (row, head) joined: their maxima and sums weigh the accumulators.  W waves share one (row, head), each
// with a W-th of its records, and meet in LDS; 2^lg lanes hold a record's accumulators, the 64 >> lg groups of a wave's
// lanes take records in turn.  Bound by the records' bytes.
template <int W>
__global__ __launch_bounds__(256) void paged_join_kernel(const float* __restrict__ rec, float* __restrict__ out, long ldo,
                                                         const int* __restrict__ offsets, int n_seqs, int n_rows, int H,
                                                         FastDiv by_H, int D, int lg, int nrec) {
    __shared__ float part[W > 1 ? W : 1][256 + 2];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = blockIdx.x * (4 / W) + w / W, mine = w % W;
    const int t = div_by(id, by_H), h = id - t * H;
    // rows of no sequence stay as they were
    const bool on = t < n_rows && t >= offsets[0] && t < offsets[n_seqs];
    if (W == 1 && !on) return;
    const float* r = rec + static_cast<long>(id) * nrec * (D + 4);
    const int per = (nrec + W - 1) / W, lo = mine * per, hi = on ? min(lo + per, nrec) : lo;
    const int c = lane & ((1 << lg) - 1), grp = lane >> lg, groups = 64 >> lg;
    float mx = -INFINITY, total = 0.0f;
    f32x4 x = {0, 0, 0, 0};
    for (int base = lo; base < hi; base += 64) {  // 64 records' maxima and sums at a time, one per lane
        float m = -INFINITY, l = 0.0f;
        if (base + lane < hi) {
            const f32x2 v = *reinterpret_cast<const f32x2*>(r + static_cast<long>(base + lane) * (D + 4));
            m = v.x;
            l = v.y;
        }
        const float top = fmaxf(mx, wave_max(m));
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        const float old = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - top);
        mx = top;
        total = total * old + group_sum(l * f, 6);
        x *= old;
        const int n = min(64, hi - base);
        constexpr int kAhead = 4;  // records in flight
        for (int k0 = 0; k0 < n; k0 += kAhead * groups) {
            float wt[kAhead];
            f32x4 y[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int k = k0 + j * groups + grp;
                wt[j] = __shfl(f, min(k, 63));  // every lane takes part
                if (k >= n || 4 * c >= D) wt[j] = 0.0f;
                y[j] = f32x4{0, 0, 0, 0};
                if (wt[j] != 0.0f)  // a record of weight 0 may hold nothing
                    y[j] = *reinterpret_cast<const f32x4*>(r + static_cast<long>(base + k) * (D + 4) + 4 + 4 * c);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) x += y[j] * wt[j];
        }
    }
    for (int m = 1 << lg; m < 64; m <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += __shfl_xor(x[i], m);
    if (W > 1) {
        float* p = part[w];
        if (grp == 0 && 4 * c < D) *reinterpret_cast<f32x4_a4*>(p + 4 * c) = f32x4_a4{x[0], x[1], x[2], x[3]};
        if (lane == 0) {
            p[256] = mx;
            p[257] = total;
        }
        __syncthreads();
        if (mine != 0 || !on) return;
        float top = mx;
#pragma unroll
        for (int o = 1; o < W; ++o) top = fmaxf(top, part[w + o][256]);
        const float own = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - top);
        total *= own;
        x *= own;
#pragma unroll
        for (int o = 1; o < W; ++o) {
            const float m = part[w + o][256], f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
            total += part[w + o][257] * f;
            if (grp == 0 && 4 * c < D)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] += part[w + o][4 * c + i] * f;
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (grp == 0 && 4 * c < D)
        *reinterpret_cast<f32x4_a4*>(out + t * ldo + static_cast<long>(h) * D + 4 * c) =
            f32x4_a4{x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
}

// the cut of a call, from what the host knows of it
struct Cut {
    bool even, staged;  // staged: the prefix goes to workgroups that share it through LDS
    int pre_tiles, pre_chunks, pre_per, pre_blocks, own_more, own_chunks, own_per, nrec;
    long own_first, own_blocks;
};

constexpr int kPreRecords = 64, kOwnRecords = 192;  // chunks at most
// Bytes of records at most, as long as one chunk of the prefix and one of the sequences' positions fit: a prompt's rows are
// many and their tables long, and 8192 rows of 32 heads of 128 under a table of 32768 positions had 17.7 GB.  So many rows
// leave few idle places with fewer chunks: 8192 rows on as many positions 4046 -> 2753 us, 1100 rows under a table of 131072
// 548 -> 180, 512 rows behind 130560 positions 5262 -> 5000.
constexpr long kMaxRecordBytes = 1L << 30;
constexpr int kSlots = 512;                         // workgroups on the GPU at a time: two per CU

int round_up(int x, int to) { return (x + to - 1) / to * to; }

Cut cut_of(const PagePool& P, int type, const PageBatch& B, int n_heads, int prefix_len) {
    Cut c{};
    const int D = P.head_dim, G = n_heads / P.n_kv_heads;
    c.even = (D == 64 || D == 128 || D == 256) && P.page_size % 16 == 0;
    const long rows = static_cast<long>(B.n_rows) * G;  // of a KV head
    const long most = kMaxRecordBytes / (rows * P.n_kv_heads * (D + 4) * 4);  // records of a row and head
    // Where sharing the prefix through LDS begins to pay: at 2^18 rows x positions both ways take the same (64 rows on 4096
    // positions 20.2 / 20.2 us, fp32 30.5 / 28.4), with twice as much it is ahead (128 on 4096 25.6 / 25.8, fp32 36.6 / 42.0) and
    // stays so.  Heads over 128 have one workgroup to a CU: fp16 from 2^20 on (512 on 2048 55.2 / 54.7, on 4096 65.3 / 73.7),
    // bf16 later (512 on 4096 79.6 / 79.5, 1920 on 32768 1048 / 1399), fp32 not at all (3334 either way).
    const int from = D <= 128 ? 18 : type == kKvF16 ? 20 : type == kKvBF16 ? 22 : 62;
    c.staged = rows > 32 && prefix_len >= 256 && rows * prefix_len >= 1L << from;
    const int own_tile = type == kKvF32 ? 16 : 32;
    const long cap = static_cast<long>(B.max_pages) * P.page_size;
    const long own = std::max(cap - prefix_len / own_tile * own_tile, 1L);
    if (prefix_len > 0) {
        const int tile_rows = c.staged ? kPrefixRows : 16;
        const int tile = c.staged ? kPrefixTile : own_tile, units = (prefix_len + tile - 1) / tile;
        c.pre_tiles = static_cast<int>((rows + tile_rows - 1) / tile_rows);
        const long streams = static_cast<long>(P.n_kv_heads) * c.pre_tiles;
        // Chunks: the fewest microseconds of a model of the GPU.  Staged: a workgroup takes 9 and 1.4 per tile (fp16, heads
        // of 128; bf16 and fp32 by their products; half as much again where two share a CU), fills one of 512 slots, the
        // sequences' workgroups the others (at half their tables' length: bytes at 4.7 TB/s), and 128 rows' record is
        // written and read at that rate.  Else an item is a wave of 16 rows; 5 tiles' time for its start and end.
        const double own_us = 0.5 * B.n_seqs * own * P.n_kv_heads * D * (type == kKvF32 ? 8 : 4) / 4.7e6;
        const double tile_us = (type == kKvF16 ? 1.4 : type == kKvBF16 ? 1.9 : 2.8) * D / 128;
        const int slots = D <= 128 ? kSlots : kSlots / 2;
        const double record_us = tile_rows * (D + 4) * 8 / 4.7e6;
        double best = 0.0;
        for (int n = 1; n <= kPreRecords && n <= units && (n == 1 || n < most); ++n) {
            const long items = streams * n, per = (units + n - 1) / n;
            double cost;
            if (c.staged) {
                const double alone = tile_us * per + 9.0, rounds = static_cast<double>((items + slots - 1) / slots);
                const double longest = rounds * (items <= slots / 2 || D > 128 ? alone : 1.5 * tile_us * per + 9.0);
                cost = std::max(longest, items * alone / slots + (D <= 128 ? own_us : 0.0)) + items * record_us;
            } else {
                const int waves = kPagedWaves * kSlots;
                const double rounds = items <= waves / 2 ? 0.65 : static_cast<double>((items + waves - 1) / waves);
                cost = 1.4 * (rounds * per + 5.0 * ((items + waves - 1) / waves)) + items * record_us;
            }
            if (best == 0.0 || cost < best) {
                best = cost;
                c.pre_per = static_cast<int>(per * tile);
            }
        }
        c.pre_chunks = (prefix_len + c.pre_per - 1) / c.pre_per;
        const long groups = c.staged ? streams * c.pre_chunks : (streams * c.pre_chunks + kPagedWaves - 1) / kPagedWaves;
        c.pre_blocks = static_cast<int>((groups + kPagedXcds - 1) / kPagedXcds * kPagedXcds);
    }
    // A sequence's own positions: chunks of one size, so that a long sequence has more of them and none is waited for; 256
    // positions, or less where the batch would leave waves idle.
    // sum of ceil(n G / 16) - 1 over the sequences that have rows: n G is a multiple of gcd(G, 16)
    c.own_more = static_cast<int>((rows - std::gcd(G, 16)) / 16);
    const long streams = static_cast<long>(P.n_kv_heads) * std::min<long>(1L * B.n_seqs + c.own_more, (rows + 15) / 16 + B.n_seqs);
    const long fill = own * streams / (kPagedWaves * kSlots);  // positions of a wave that fill the GPU once
    const long chunks = std::min<long>(kOwnRecords, std::max(most - c.pre_chunks, 1L)), least = (own + chunks - 1) / chunks;
    c.own_per = round_up(static_cast<int>(std::max({std::min(fill, 256L), least, 1L})), own_tile);
    c.own_chunks = static_cast<int>((own + c.own_per - 1) / c.own_per);
    c.own_first = static_cast<long>(c.own_chunks) * B.n_seqs * P.n_kv_heads;
    c.own_blocks = (c.own_first + static_cast<long>(c.own_chunks) * c.own_more * P.n_kv_heads + kPagedWaves - 1) / kPagedWaves;
    c.nrec = c.pre_chunks + c.own_chunks;
    return c;
}

bool fits(const Cut& c) { return c.pre_blocks + c.own_blocks < 1L << 24; }  // 256 threads each: a launch's limit

}  // namespace
}  // namespace dev

namespace detail {

long paged_attention_workspace_bytes(const PagePool& P, int type, const PageBatch& B, int n_heads, int prefix_len) {
    const dev::Cut c = dev::cut_of(P, type, B, n_heads, prefix_len);
    if (!dev::fits(c)) return kDeclined;
    return c.nrec == 1 ? 0 : static_cast<long>(B.n_rows) * n_heads * c.nrec * (P.head_dim + 4) * 4;
}

int launch_paged_attention(const PagePool& P, int type, const PageBatch& B, const int* prefix_pages, int prefix_len,
                           const float* q, long ldq, float* out, long ldo, int n_heads, float scale, float* ws,
                           hipStream_t stream) {
    const dev::Cut c = dev::cut_of(P, type, B, n_heads, prefix_len);
    dev::PagedAttnArgs a{};
    a.q = q, a.out = out, a.rec = ws, a.ldq = ldq, a.ldo = ldo;
    a.P = P, a.B = B;
    a.prefix_pages = prefix_pages, a.prefix_len = prefix_len;
    a.H = n_heads, a.G = n_heads / P.n_kv_heads, a.nrec = c.nrec;
    if (!dev::fits(c)) return kDeclined;
    a.pre_tiles = c.pre_tiles, a.pre_chunks = c.pre_chunks, a.pre_per = c.pre_per, a.pre_blocks = c.pre_blocks;
    a.own_more = c.own_more, a.own_chunks = c.own_chunks, a.own_per = c.own_per;
    a.own_first = static_cast<int>(c.own_first);
    a.by_G = dev::fast_div(a.G), a.by_Hkv = dev::fast_div(P.n_kv_heads);
    a.by_pre_tiles = dev::fast_div(std::max(c.pre_tiles, 1)), a.by_seqs = dev::fast_div(B.n_seqs);
    a.by_more = dev::fast_div(std::max(c.own_more, 1));
    a.qscale = scale * 1.44269504088896340736f;
    a.staged = c.staged;
    const auto run_rows = type == kKvF32   ? dev::run_paged_attn_f32
                          : type == kKvF16 ? dev::run_paged_attn_f16
                                           : dev::run_paged_attn_bf16;
    if (c.staged)
        (type == kKvF32   ? dev::run_paged_mixed_f32
         : type == kKvF16 ? dev::run_paged_mixed_f16
                          : dev::run_paged_mixed_bf16)(a, c.even, static_cast<int>(c.own_blocks), stream);
    else
        run_rows(a, c.even, static_cast<int>(c.pre_blocks + c.own_blocks), stream);
    if (c.nrec > 1) {
        const long pairs = static_cast<long>(B.n_rows) * n_heads;
        int lg = 0;
        while ((4 << lg) < P.head_dim) ++lg;
        // few pairs of many records: four waves to each, or a wave reads them one after the other
        const bool shared = pairs <= 2048 && c.nrec > 16;
        const auto join = shared ? dev::paged_join_kernel<4> : dev::paged_join_kernel<1>;
        const long groups = shared ? pairs : (pairs + 3) / 4;
        hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(groups)), dim3(256), 0, stream, ws, out, ldo, B.offsets, B.n_seqs,
                           B.n_rows, n_heads, dev::fast_div(n_heads), P.head_dim, lg, c.nrec);
    }
    return 0;
}

}  // namespace detail
}  // namespace cri
