// experts_route.hip -- each token's experts from the router's logits, and the pairs (token, choice) grouped by expert.
//
// A wave takes a token: lane l holds the logits of experts l C .. l C + C - 1 in registers, and k times the largest is found
// (the lane's own, a maximum over the wave, the first lane that has it: ties go to the lowest index) and struck out.  The
// order is the logits' own; only with a bias are scores computed first, in 64 bits, where different ones stay different.
// The weights of the k chosen, too, are computed in 64 bits, a lane each.
//
// Grouping is a counting sort, stable and without an order left to chance: counts per block of tokens (integer atomics in
// LDS, whose order does not matter), offsets from their sums, and the place of a pair from the pairs before it in its block,
// 64 at a time (the lanes of a wave with the same expert by one ballot per bit of its number).  Up to kSingle tokens one
// workgroup does it all; more take two launches, the counts of at most kBlocks blocks between them, which every block of
// the second adds up for itself.
// Bound by the chain of launches, loads and reductions: one token of 128 experts, 8 chosen, 4.9 us; 8192 of
// 256 with a bias 17.2 us and 10.5 for the second launch.
#include <algorithm>

#include "common.hpp"
#include "internal.hpp"

namespace cri {
namespace dev {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kMaxExperts = 1024;
constexpr int kSingle = 64;   // tokens that one workgroup takes alone
constexpr int kBlocks = 256;  // blocks of tokens otherwise

struct RouteArgs {
    const float* logits;  // null: ids are given
    long ldl;
    const float* bias;
    float scale;
    bool sigmoid, normalize;
    int* ids;
    float* weights;
    int* offsets;
    int* rows;
    int* slots;
    int* counts;  // [blocks][E]
    int M, E, k, per;  // per: tokens of a block
};

struct Shared {
    int run[kMaxExperts];                    // a block's next place of each expert
    int count[kMaxExperts];
    int parts[2][kThreads];
    uint16_t wave[kWaves][kMaxExperts];      // pairs of each expert in a wave's 64, then before them in the chunk
    int totals[kWaves];
};

// v of the lane that a DPP control names, 0 where there is none
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lower(uint32_t v) {
    return __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false);
}
// The largest of the wave; into lane 63 over 1, 2, 4 and 8 lanes of a row, then row after row.
__device__ __forceinline__ uint32_t wave_top(uint32_t v) {
    v = max(v, lower<0x111, 0xF>(v));
    v = max(v, lower<0x112, 0xF>(v));
    v = max(v, lower<0x114, 0xF>(v));
    v = max(v, lower<0x118, 0xF>(v));
    v = max(v, lower<0x142, 0xA>(v));
    v = max(v, lower<0x143, 0xC>(v));
    return __builtin_amdgcn_readlane(v, 63);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double lower64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, static_cast<uint64_t>(lower<CTRL, ROWS>(static_cast<uint32_t>(u))) |
                                          static_cast<uint64_t>(lower<CTRL, ROWS>(static_cast<uint32_t>(u >> 32))) << 32);
}
__device__ __forceinline__ double wave_sum64(double v) {
    v += lower64<0x111, 0xF>(v);
    v += lower64<0x112, 0xF>(v);
    v += lower64<0x114, 0xF>(v);
    v += lower64<0x118, 0xF>(v);
    v += lower64<0x142, 0xA>(v);
    v += lower64<0x143, 0xC>(v);
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u), 63))) |
                                          static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u >> 32), 63)))
                                              << 32);
}

// Numbers as unsigned integers of the same order, all above 0, which stands for what is never chosen.  (+0 and -0 are one.)
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    return u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
    return u ^ (u >> 63 ? ~0ull : 1ull << 63);
}

// e^y to about 2^-52: y = n ln 2 + r with ln 2 in two parts, the series of e^r up to r^13 / 13! (|r| <= ln 2 / 2: the rest is below
// 2^-57), times 2^n.  Fewer instructions than the library's exp, whose range reduction and special cases are not needed here.
__device__ __forceinline__ double exp64(double y) {
    y = fmin(fmax(y, -800.0), 800.0);  // beyond: 0 or infinity all the same
    const double n = rint(y * 1.4426950408889634);
    const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, y));
    constexpr double kOver[] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880,
                                1.0 / 3628800, 1.0 / 39916800, 1.0 / 479001600, 1.0 / 6227020800.0};
    double p = kOver[13];
#pragma unroll
    for (int i = 12; i >= 0; --i) p = fma(p, r, kOver[i]);
    return ldexp(p, static_cast<int>(n));
}
// 1 / d for d >= 1: the hardware's reciprocal and two steps of Newton's (past their range, and for infinity, a division)
__device__ __forceinline__ double reciprocal(double d) {
    if (d > 1e150) return 1.0 / d;
    double r = __builtin_amdgcn_rcp(d);
    r = fma(fma(-d, r, 1.0), r, r);
    return fma(fma(-d, r, 1.0), r, r);
}

// The choices of token t, by one wave; lane j returns choice j's expert, or -1.  WIDE: with a bias, by scores of 64 bits, whose
// upper halves are compared first and the lower ones only between equal upper ones.
template <int C, bool WIDE>
__device__ __forceinline__ int choose(const RouteArgs& a, int t) {
    const int lane = __lane_id();
    const float* z = a.logits + t * a.ldl;
    float x[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int e = lane * C + i;
        const float v = e < a.E ? z[e] : -INFINITY;
        x[i] = v == v ? v : -INFINITY;
    }
    float best = x[0];
#pragma unroll
    for (int i = 1; i < C; ++i) best = fmaxf(best, x[i]);
    const float most = wave_max(best);
    // of all experts: softmax's sum, where anything needs it
    auto part = [&](float v) { return v == most ? 1.0 : exp64(static_cast<double>(v) - most); };
    double all = 1.0;
    if (!a.sigmoid && (WIDE || !a.normalize) && most > -INFINITY) {
        all = 0.0;
#pragma unroll
        for (int i = 0; i < C; ++i) all += part(x[i]);
        all = wave_sum64(all);
    }
    const double over = 1.0 / all;
    auto score = [&](float v) { return a.sigmoid ? reciprocal(1.0 + exp64(-static_cast<double>(v))) : part(v) * over; };
    uint32_t high[C], low[WIDE ? C : 1] = {};
#pragma unroll
    for (int i = 0; i < C; ++i) {
        if constexpr (WIDE) {
            const int e = min(lane * C + i, a.E - 1);
            const double s = score(x[i]) + a.bias[e];
            const uint64_t u = x[i] > -INFINITY && s > -INFINITY ? ordered(s) : 0;  // (NaN is not above)
            high[i] = static_cast<uint32_t>(u >> 32);
            low[i] = static_cast<uint32_t>(u);
        } else {
            high[i] = x[i] > -INFINITY ? ordered(x[i]) : 0;
        }
    }
    // Up to four a lane are sorted once (neighbours exchanged where the later one is larger, so equal ones keep their order):
    // the lane's largest is then always the first, and a chosen one leaves by a shift.  More are searched each time.
    constexpr bool SORTED = C <= 4;
    int place[C];
#pragma unroll
    for (int i = 0; i < C; ++i) place[i] = i;
    if constexpr (SORTED) {
#pragma unroll
        for (int round = 0; round < C; ++round) {
#pragma unroll
            for (int i = round & 1; i + 1 < C; i += 2) {
                const bool more = high[i + 1] > high[i] || (WIDE && high[i + 1] == high[i] && low[WIDE ? i + 1 : 0] > low[WIDE ? i : 0]);
                const auto exchange = [&](auto& p, auto& q) {
                    const auto was = p;
                    p = more ? q : p;
                    q = more ? was : q;
                };
                exchange(high[i], high[i + 1]);
                exchange(place[i], place[i + 1]);
                if constexpr (WIDE) exchange(low[i], low[i + 1]);
            }
        }
    }
    int mine = -1;
    for (int j = 0; j < a.k; ++j) {
        uint32_t h = high[0], l = low[0];
        int at = place[0];
        if constexpr (!SORTED) {
#pragma unroll
            for (int i = 1; i < C; ++i) {
                const bool more = high[i] > h || (WIDE && high[i] == h && low[WIDE ? i : 0] > l);
                h = more ? high[i] : h;
                if (WIDE) l = more ? low[WIDE ? i : 0] : l;
                at = more ? i : at;
            }
        }
        const uint32_t top = wave_top(h);
        if (top == 0) break;
        unsigned long same = __ballot(h == top);
        if (WIDE && (same & (same - 1)) != 0) {
            const uint32_t rest = wave_top(h == top ? l : 0);
            same = __ballot(h == top && l == rest);
        }
        const int who = __builtin_ctzl(same);
        const int expert = who * C + __builtin_amdgcn_readlane(at, who);
        mine = lane == j ? expert : mine;
        const bool gone = lane == who;
        if constexpr (SORTED) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                high[i] = gone ? (i + 1 < C ? high[i + 1 < C ? i + 1 : i] : 0) : high[i];
                if (i + 1 < C) place[i] = gone ? place[i + 1 < C ? i + 1 : i] : place[i];
                if (WIDE && i + 1 < C) low[WIDE ? i : 0] = gone ? low[WIDE && i + 1 < C ? i + 1 : 0] : low[WIDE ? i : 0];
            }
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i) high[i] = gone && i == at ? 0 : high[i];
        }
    }
    const float value = mine >= 0 ? z[mine] : 0.0f;
    double w = mine >= 0 ? score(value) : 0.0;
    if (a.normalize) {
        const double sum = wave_sum64(w);
        w = sum > 0.0 ? w / sum : 0.0;
    }
    if (lane < a.k) {
        a.ids[static_cast<long>(t) * a.k + lane] = mine;
        a.weights[static_cast<long>(t) * a.k + lane] = static_cast<float>(w * a.scale);
    }
    return mine;
}

// exclusive sums of v over the workgroup's threads; the total in `all`
__device__ __forceinline__ int block_scan(int v, Shared& s, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int up = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(up, d);
        up += lane >= d ? o : 0;
    }
    if (lane == 63) s.totals[wave] = up;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const int n = s.totals[w];
        before += w < wave ? n : 0;
        all += n;
    }
    return before + up - v;
}

// an expert's number, or E for a pair without one
__device__ __forceinline__ int expert_of(const RouteArgs& a, long p) {
    const int e = a.ids[p];
    return e >= 0 && e < a.E ? e : a.E;
}

// The block's pairs to their places: run[e] is where its first pair of expert e goes.
__device__ __forceinline__ void place(const RouteArgs& a, Shared& s, long p0, long p1) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bits = 32 - __builtin_clz(a.E);
    for (long base = p0; base < p1; base += kThreads) {
        for (int w = 0; w < kWaves; ++w)
            if (tid < a.E) s.wave[w][tid] = 0;
        __syncthreads();
        const long p = base + tid;
        const int e = p < p1 ? expert_of(a, p) : a.E;
        unsigned long same = ~0ul;
        for (int i = 0; i < bits; ++i) {
            const unsigned long set = __ballot((e >> i) & 1);
            same &= (e >> i) & 1 ? set : ~set;
        }
        const int rank = __popcll(same & ((1ul << lane) - 1));
        if (e < a.E && rank == 0) s.wave[wave][e] = static_cast<uint16_t>(__popcll(same));
        __syncthreads();
        int more = 0;
        if (tid < a.E) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const int n = s.wave[w][tid];
                s.wave[w][tid] = static_cast<uint16_t>(more);
                more += n;
            }
        }
        __syncthreads();
        if (p < p1) {
            const int to = e < a.E ? s.run[e] + s.wave[wave][e] + rank : -1;
            a.slots[p] = to;
            if (to >= 0) a.rows[to] = static_cast<int>(p);
        }
        __syncthreads();
        if (tid < a.E) s.run[tid] += more;
    }
}

__device__ __forceinline__ void write_rest(const RouteArgs& a, int all, int block, int blocks) {
    const long R = static_cast<long>(a.M) * a.k;
    for (long r = all + block * static_cast<long>(kThreads) + threadIdx.x; r < R; r += static_cast<long>(blocks) * kThreads)
        a.rows[r] = -1;
}

// Chooses (with logits) and counts the block's pairs; a single block groups them, too.
template <int C, bool WIDE>
__global__ __launch_bounds__(kThreads) void route_kernel(const RouteArgs a) {
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < a.E) s.count[tid] = 0;
    __syncthreads();
    const int t0 = blockIdx.x * a.per, t1 = min(t0 + a.per, a.M);
    if (a.logits != nullptr) {
        for (int t = t0 + wave; t < t1; t += kWaves) {
            const int e = choose<C, WIDE>(a, t);
            if (lane < a.k && e >= 0) atomicAdd(&s.count[e], 1);
        }
    } else {
        for (long p = static_cast<long>(t0) * a.k + tid; p < static_cast<long>(t1) * a.k; p += kThreads) {
            const int e = expert_of(a, p);
            if (e < a.E) atomicAdd(&s.count[e], 1);
        }
    }
    __syncthreads();  // (the ids of this block are read again below: written by this workgroup)
    const int n = tid < a.E ? s.count[tid] : 0;
    if (gridDim.x > 1) {
        if (tid < a.E) a.counts[static_cast<long>(blockIdx.x) * a.E + tid] = n;
        return;
    }
    int all;
    const int before = block_scan(n, s, all);
    if (tid < a.E) {
        s.run[tid] = before;
        a.offsets[tid] = before;
    }
    if (tid == 0) a.offsets[a.E] = all;
    place(a, s, 0, static_cast<long>(a.M) * a.k);
    write_rest(a, all, 0, 1);
}

// The second launch: offsets from all blocks' counts, and the block's pairs to their places.
__global__ __launch_bounds__(kThreads) void group_kernel(const RouteArgs a, int blocks) {
    __shared__ Shared s;
    const int tid = threadIdx.x, block = blockIdx.x;
    // the counts of an expert by several threads, a run of blocks each
    int width = 64;
    while (width < a.E) width <<= 1;
    const int shares = kThreads / width, e = tid & (width - 1), share = tid / width;
    const int each = (blocks + shares - 1) / shares, b0 = share * each, b1 = min(b0 + each, blocks);
    int total = 0, before = 0;
    if (e < a.E) {
        for (int b = b0; b < b1; b += 16) {
            int n[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) n[i] = a.counts[static_cast<long>(min(b + i, b1 - 1)) * a.E + e];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                total += b + i < b1 ? n[i] : 0;
                before += b + i < min(b1, block) ? n[i] : 0;
            }
        }
    }
    s.parts[0][tid] = total;
    s.parts[1][tid] = before;
    __syncthreads();
    total = before = 0;
    if (tid < a.E) {
        for (int i = 0; i < shares; ++i) {
            total += s.parts[0][i * width + tid];
            before += s.parts[1][i * width + tid];
        }
    }
    int all;
    const int start = block_scan(total, s, all);
    if (tid < a.E) {
        s.run[tid] = start + before;
        if (block == 0) a.offsets[tid] = start;
    }
    if (block == 0 && tid == 0) a.offsets[a.E] = all;
    const int t0 = block * a.per, t1 = min(t0 + a.per, a.M);
    place(a, s, static_cast<long>(t0) * a.k, static_cast<long>(t1) * a.k);
    write_rest(a, all, block, blocks);
}

// tokens of a block: one block up to kSingle tokens, at most kBlocks of them else
int block_tokens(int M) { return M <= kSingle ? std::max(M, 1) : std::max((M + kBlocks - 1) / kBlocks, kWaves); }

void launch(RouteArgs a, hipStream_t stream) {
    a.per = block_tokens(a.M);
    const int blocks = std::max((a.M + a.per - 1) / a.per, 1);
    const bool biased = a.logits != nullptr && a.bias != nullptr;
    const int c = (a.E + 63) / 64;
    const auto run = a.logits == nullptr ? route_kernel<1, false>
                     : biased            ? (c == 1   ? route_kernel<1, true>
                                            : c == 2 ? route_kernel<2, true>
                                            : c <= 4 ? route_kernel<4, true>
                                            : c <= 8 ? route_kernel<8, true>
                                                     : route_kernel<16, true>)
                                         : (c == 1   ? route_kernel<1, false>
                                            : c == 2 ? route_kernel<2, false>
                                            : c <= 4 ? route_kernel<4, false>
                                            : c <= 8 ? route_kernel<8, false>
                                                     : route_kernel<16, false>);
    hipLaunchKernelGGL(run, dim3(blocks), dim3(kThreads), 0, stream, a);
    if (blocks > 1) hipLaunchKernelGGL(group_kernel, dim3(blocks), dim3(kThreads), 0, stream, a, blocks);
}

}  // namespace
}  // namespace dev

namespace detail {

long expert_group_workspace_bytes(int n_tokens, int, int n_experts) {
    if (n_tokens <= dev::kSingle) return 0;
    const int per = dev::block_tokens(n_tokens);
    return static_cast<long>((n_tokens + per - 1) / per) * n_experts * 4;
}

int launch_expert_route(const ExpertRouter& r, const float* logits, long ldl, int n_experts, int* ids, float* weights,
                        const ExpertRows& g, int* ws, hipStream_t stream) {
    dev::launch(dev::RouteArgs{logits, ldl, r.bias, r.scale, r.sigmoid, r.normalize, ids, weights, g.offsets, g.rows, g.slots, ws,
                               g.n_tokens, n_experts, g.top_k, 0},
                stream);
    return 0;
}

int launch_expert_group(const int* ids, int n_experts, const ExpertRows& g, int* ws, hipStream_t stream) {
    dev::launch(dev::RouteArgs{nullptr, 0, nullptr, 0.0f, false, false, const_cast<int*>(ids), nullptr, g.offsets, g.rows, g.slots,
                               ws, g.n_tokens, n_experts, g.top_k, 0},
                stream);
    return 0;
}

}  // namespace detail
}  // namespace cri
