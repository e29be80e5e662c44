// paged_attention.hip -- how a call of the paged attention is cut into workgroups, and the kernel that joins their
// records.
#include <numeric>

#include "paged_attention.hpp"

namespace cri {
namespace dev {
namespace {

// One wave per (row, head): the records' maxima and sums weigh the accumulators.  Bound by the records' bytes.
__global__ __launch_bounds__(256) void paged_join_kernel(const float* __restrict__ rec, float* __restrict__ out, long ldo,
                                                         const int* __restrict__ offsets, int n_seqs, int n_rows, int H,
                                                         int D, int lg, int nrec) {
    const int lane = threadIdx.x & 63;
    const int id = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int t = id / H, h = id % H;
    if (t >= n_rows || t < offsets[0] || t >= offsets[n_seqs]) return;  // rows of no sequence stay as they were
    const float* r = rec + static_cast<long>(id) * nrec * (D + 4);
    float m = -INFINITY, l = 0.0f;
    if (lane < nrec) {
        const f32x2 x = *reinterpret_cast<const f32x2*>(r + static_cast<long>(lane) * (D + 4));
        m = x.x;
        l = x.y;
    }
    const float mx = wave_max(m);
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
    const float total = group_sum(l * f, 6);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    // 2^lg lanes hold a record's accumulators, the wave's 64 >> lg groups of them take the records in turn
    const int c = lane & ((1 << lg) - 1), grp = lane >> lg, groups = 64 >> lg;
    f32x4 x = {0, 0, 0, 0};
    constexpr int kAhead = 4;  // records in flight
    for (int k0 = 0; k0 < nrec; k0 += kAhead * groups) {
        float wt[kAhead];
        f32x4 y[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int k = k0 + j * groups + grp;
            wt[j] = __shfl(f, min(k, nrec - 1));  // every lane takes part
            if (k >= nrec || 4 * c >= D) wt[j] = 0.0f;
            y[j] = f32x4{0, 0, 0, 0};
            if (wt[j] != 0.0f)  // a record of weight 0 may hold nothing
                y[j] = *reinterpret_cast<const f32x4*>(r + static_cast<long>(k) * (D + 4) + 4 + 4 * c);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) x += y[j] * wt[j];
    }
    for (int m = 1 << lg; m < 64; m <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += __shfl_xor(x[i], m);
    if (grp == 0 && 4 * c < D)
        *reinterpret_cast<f32x4_a4*>(out + t * ldo + static_cast<long>(h) * D + 4 * c) =
            f32x4_a4{x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
}

// the cut of a call, from what the host knows of it
struct Cut {
    bool even, staged;  // staged: the prefix goes to the kernel that shares it through LDS
    int pre_wq, pre_tiles, pre_chunks, pre_per, pre_blocks, own_wq, own_tiles, own_chunks, own_per, nrec;
    long own_blocks;
};

constexpr int kMaxRecords = 64;  // the joining wave keeps one record's maximum per lane
constexpr int kSlots = 512;      // workgroups on the GPU at a time: two per CU

int round_up(int x, int to) { return (x + to - 1) / to * to; }

Cut cut_of(const PagePool& P, int type, const PageBatch& B, int n_heads, int prefix_len) {
    Cut c{};
    const int D = P.head_dim, G = n_heads / P.n_kv_heads;
    c.even = (D == 64 || D == 128 || D == 256) && P.page_size % 16 == 0;
    const long rows = static_cast<long>(B.n_rows) * G;   // of a KV head
    const long mean = (rows + B.n_seqs - 1) / B.n_seqs;  // of a KV head and sequence
    c.staged = c.even && type != kKvF32 && D <= 128 && rows > 64 && prefix_len >= 256;
    const int tile = type == kKvF32 ? 16 : 32;
    constexpr int block = 16;  // rows of a wave
    auto waves_of = [&](long r) { return r <= block ? 1 : r <= 2 * block ? 2 : 4; };
    c.pre_wq = waves_of(rows);
    c.own_wq = waves_of(mean);
    if (prefix_len > 0) {
        const int tile_rows = c.staged ? kPrefixRows : block * c.pre_wq;
        const int unit = c.staged ? kPrefixTile : tile * (kPagedWaves / c.pre_wq);
        c.pre_tiles = static_cast<int>((rows + tile_rows - 1) / tile_rows);
        const long streams = static_cast<long>(P.n_kv_heads) * c.pre_tiles;
        const int units = (prefix_len + unit - 1) / unit;
        // chunks: rounds of workgroups times units of each (a workgroup that has its CU to itself takes two thirds of the
        // time), five units for a workgroup's start and end, a sixtieth for each one's records
        double best = 0.0;
        for (int n = 1; n <= kMaxRecords / 2 && n <= units; ++n) {
            const long groups = streams * n, per = (units + n - 1) / n;
            const double rounds = groups <= kSlots / 2 ? 0.65 : static_cast<double>((groups + kSlots - 1) / kSlots);
            const double cost = rounds * per + 5.0 * ((groups + kSlots - 1) / kSlots) + groups / 60.0;
            if (best == 0.0 || cost < best) {
                best = cost;
                c.pre_per = static_cast<int>(per * unit);
            }
        }
        c.pre_chunks = (prefix_len + c.pre_per - 1) / c.pre_per;
        c.pre_blocks = static_cast<int>((streams * c.pre_chunks + kPagedXcds - 1) / kPagedXcds * kPagedXcds);
    }
    // a sequence's own positions: chunks of one size, so that a long sequence has more of them and none is waited for;
    // 512 positions, or less where the batch would leave CUs idle
    const long cap = static_cast<long>(B.max_pages) * P.page_size;
    const long own = std::max(cap - prefix_len / tile * tile, 1L);
    const int rt = block * c.own_wq, unit = tile * (kPagedWaves / c.own_wq);
    // sum of ceil(n G / rt) over the sequences that have rows: n G is a multiple of gcd(G, rt)
    c.own_tiles = static_cast<int>((rows + std::min<long>(B.n_seqs, B.n_rows) * (rt - std::gcd(G, rt))) / rt);
    const long streams = static_cast<long>(P.n_kv_heads) * c.own_tiles;
    const long fill = own * streams / kSlots;  // positions per workgroup that fill the GPU once
    const long least = (own + kMaxRecords / 2 - 1) / (kMaxRecords / 2);
    c.own_per = round_up(static_cast<int>(std::max({std::min(fill, 512L), least, 1L})), 2 * unit);
    c.own_chunks = static_cast<int>((own + c.own_per - 1) / c.own_per);
    c.own_blocks = static_cast<long>(c.own_tiles) * c.own_chunks * P.n_kv_heads;
    c.nrec = c.pre_chunks + c.own_chunks;
    return c;
}

}  // namespace
}  // namespace dev

namespace detail {

long paged_attention_workspace_bytes(const PagePool& P, int type, const PageBatch& B, int n_heads, int prefix_len) {
    const dev::Cut c = dev::cut_of(P, type, B, n_heads, prefix_len);
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
    a.pre_wq = c.pre_wq, a.pre_tiles = c.pre_tiles, a.pre_chunks = c.pre_chunks, a.pre_per = c.pre_per;
    a.pre_blocks = c.pre_blocks;
    a.own_wq = c.own_wq, a.own_tiles = c.own_tiles, a.own_chunks = c.own_chunks, a.own_per = c.own_per;
    a.by_G = dev::fast_div(a.G), a.by_Hkv = dev::fast_div(P.n_kv_heads);
    a.by_pre_tiles = dev::fast_div(std::max(c.pre_tiles, 1)), a.by_own_tiles = dev::fast_div(std::max(c.own_tiles, 1));
    a.qscale = scale * 1.44269504088896340736f;
    a.staged = c.staged;
    if (c.staged) {
        (type == kKvF16 ? dev::run_paged_prefix_f16 : dev::run_paged_prefix_bf16)(a, stream);
        a.pre_blocks = 0;
    }
    const long blocks = a.pre_blocks + c.own_blocks;
    if (blocks > 0x7FFFFFFFL) return kDeclined;
    const auto run = type == kKvF32   ? dev::run_paged_attn_f32
                     : type == kKvF16 ? dev::run_paged_attn_f16
                                      : dev::run_paged_attn_bf16;
    run(a, c.even, static_cast<int>(blocks), stream);
    if (c.nrec > 1) {
        const long waves = static_cast<long>(B.n_rows) * n_heads;
        int lg = 0;
        while ((4 << lg) < P.head_dim) ++lg;
        hipLaunchKernelGGL(dev::paged_join_kernel, dim3(static_cast<unsigned>((waves + 3) / 4)), dim3(256), 0, stream, ws,
                           out, ldo, B.offsets, B.n_seqs, B.n_rows, n_heads, P.head_dim, lg, c.nrec);
    }
    return 0;
}

}  // namespace detail
}  // namespace cri
