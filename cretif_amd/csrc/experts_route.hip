// experts_route.hip -- each token's experts from the router's logits, and the pairs (token, choice) grouped by expert.
//
// A wave takes a token (two side by side where a block has more than 16): lane l holds the logits of experts
// l C .. l C + C - 1 in registers, and k times the largest is found (the lane's own, a maximum over the wave, the first lane that
// has it: ties go to the lowest index) and struck out.  The order is the logits' own; only with a bias are scores computed first,
// in 64 bits: sums of score and bias that differ by less than a few 2^-53 of themselves (saturated scores, or tiny ones under a bias
// that is not) may be the same number, whichever logit is larger.  The weights of the k chosen, too, are computed in 64 bits, a
// lane each.
//
// Grouping is a counting sort, stable and without an order left to chance: counts per block of tokens (integer atomics in
// LDS, whose order does not matter), offsets from their sums, and the place of a pair from the pairs before it in its block,
// 64 at a time (the lanes of a wave with the same expert by one ballot per bit of its number).  Up to kSingle tokens one
// workgroup does it all; more take two launches, the counts of at most kBlocks blocks between them, which every block of
// the second adds up for itself.
// One token of 128 experts, 8 chosen, is a chain of loads and reductions, 4.9 us.  8192 of 256 with a bias take 13.8 to 15 us, 69% of
// them in the vector units (17.2 a token at a time), and 7.2 to 7.7 for the second launch, whose blocks read all counts out of L2;
// 8192 tokens' given ids 2.5 and 8.5.
#include <algorithm>
#include <type_traits>

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
    int* counts;  // [blocks][padded(E)]
    int M, E, k, per;  // per: tokens of a block
};

__host__ __device__ inline int padded(int E) { return (E + 3) & ~3; }
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

struct Shared {
    int run[kMaxExperts];                    // a block's next place of each expert
    int count[kMaxExperts];
    union {
        uint16_t wave[kWaves][kMaxExperts];  // pairs of each expert in a wave's 64, then before them in the chunk
        i32x4 parts[2][kThreads];            // of four experts in a run of blocks, and of those before this one
    };
    int totals[kWaves];
};

// v of the lane that a DPP control names, 0 where there is none
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lower(uint32_t v) {
    return __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false);
}
// The largest of the wave, of T numbers side by side; into lane 63 over 1, 2, 4 and 8 lanes of a row, then row after row.
template <int T>
__device__ __forceinline__ void wave_tops(const uint32_t (&from)[T], uint32_t (&top)[T]) {
    uint32_t v[T];
    auto step = [&](auto&& moved) {
#pragma unroll
        for (int n = 0; n < T; ++n) v[n] = max(v[n], moved(v[n]));
    };
#pragma unroll
    for (int n = 0; n < T; ++n) v[n] = from[n];
    step([](uint32_t u) { return lower<0x111, 0xF>(u); });
    step([](uint32_t u) { return lower<0x112, 0xF>(u); });
    step([](uint32_t u) { return lower<0x114, 0xF>(u); });
    step([](uint32_t u) { return lower<0x118, 0xF>(u); });
    step([](uint32_t u) { return lower<0x142, 0xA>(u); });
    step([](uint32_t u) { return lower<0x143, 0xC>(u); });
#pragma unroll
    for (int n = 0; n < T; ++n) top[n] = __builtin_amdgcn_readlane(v[n], 63);
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

// The choices of T tokens t, t + step, ... by one wave, side by side (a chain of maxima each); lane j returns choice j's expert, or
// -1.  WIDE: with a bias, by scores of 64 bits, whose upper halves are compared first and the lower ones only between equal
// upper ones.
template <int C, bool WIDE, int T>
__device__ __forceinline__ void choose(const RouteArgs& a, int t, int step, int (&mine)[T]) {
    const int lane = __lane_id();
    const float* z[T];
    float x[T][C], most[T];
    uint32_t high[T][C], low[T][WIDE ? C : 1] = {};
    double all[T], over[T];
#pragma unroll
    for (int n = 0; n < T; ++n) {
        z[n] = a.logits + (t + n * step) * a.ldl;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int e = lane * C + i;
            const float v = e < a.E ? z[n][e] : -INFINITY;
            x[n][i] = v == v ? v : -INFINITY;
        }
    }
    // of all experts: softmax's sum, where anything needs it
    auto part = [&](int n, float v) { return v == most[n] ? 1.0 : exp64(static_cast<double>(v) - most[n]); };
    auto score = [&](int n, float v) { return a.sigmoid ? reciprocal(1.0 + exp64(-static_cast<double>(v))) : part(n, v) * over[n]; };
#pragma unroll
    for (int n = 0; n < T; ++n) {
        mine[n] = -1;
        all[n] = 1.0;
        if (a.sigmoid) continue;
        float best = x[n][0];
#pragma unroll
        for (int i = 1; i < C; ++i) best = fmaxf(best, x[n][i]);
        most[n] = wave_max(best);
        if ((WIDE || !a.normalize) && most[n] > -INFINITY) {
            all[n] = 0.0;
#pragma unroll
            for (int i = 0; i < C; ++i) all[n] += part(n, x[n][i]);
            all[n] = wave_sum64(all[n]);
        }
    }
#pragma unroll
    for (int n = 0; n < T; ++n) {
        over[n] = 1.0 / all[n];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            if constexpr (WIDE) {
                const int e = min(lane * C + i, a.E - 1);
                const double s = score(n, x[n][i]) + a.bias[e];
                const uint64_t u = x[n][i] > -INFINITY && s > -INFINITY ? ordered(s) : 0;  // (NaN is not above)
                high[n][i] = static_cast<uint32_t>(u >> 32);
                low[n][i] = static_cast<uint32_t>(u);
            } else {
                high[n][i] = x[n][i] > -INFINITY ? ordered(x[n][i]) : 0;
            }
        }
    }
    // Up to four a lane are sorted once (neighbours exchanged where the later one is larger, so equal ones keep their order):
    // the lane's largest is then always the first, and a chosen one leaves by a shift.  More are searched each time.
    constexpr bool SORTED = C <= 4;
    int place[T][C];
#pragma unroll
    for (int n = 0; n < T; ++n) {
#pragma unroll
        for (int i = 0; i < C; ++i) place[n][i] = i;
        if constexpr (SORTED) {
#pragma unroll
            for (int round = 0; round < C; ++round) {
#pragma unroll
                for (int i = round & 1; i + 1 < C; i += 2) {
                    const bool more = high[n][i + 1] > high[n][i] ||
                                      (WIDE && high[n][i + 1] == high[n][i] && low[n][WIDE ? i + 1 : 0] > low[n][WIDE ? i : 0]);
                    const auto exchange = [&](auto& p, auto& q) {
                        const auto was = p;
                        p = more ? q : p;
                        q = more ? was : q;
                    };
                    exchange(high[n][i], high[n][i + 1]);
                    exchange(place[n][i], place[n][i + 1]);
                    if constexpr (WIDE) exchange(low[n][i], low[n][i + 1]);
                }
            }
        }
    }
    for (int j = 0; j < a.k; ++j) {
        uint32_t h[T], l[T], top[T];
        int at[T];
#pragma unroll
        for (int n = 0; n < T; ++n) {
            h[n] = high[n][0];
            l[n] = low[n][0];
            at[n] = place[n][0];
            if constexpr (!SORTED) {
#pragma unroll
                for (int i = 1; i < C; ++i) {
                    const bool more = high[n][i] > h[n] || (WIDE && high[n][i] == h[n] && low[n][WIDE ? i : 0] > l[n]);
                    h[n] = more ? high[n][i] : h[n];
                    if (WIDE) l[n] = more ? low[n][WIDE ? i : 0] : l[n];
                    at[n] = more ? i : at[n];
                }
            }
        }
        wave_tops(h, top);
        uint32_t any = 0;
#pragma unroll
        for (int n = 0; n < T; ++n) any |= top[n];
        if (any == 0) break;
#pragma unroll
        for (int n = 0; n < T; ++n) {
            unsigned long same = __ballot(h[n] == top[n]);
            if (WIDE && (same & (same - 1)) != 0 && top[n] != 0) {
                uint32_t low_half[1] = {h[n] == top[n] ? l[n] : 0}, rest[1];
                wave_tops(low_half, rest);
                same = __ballot(h[n] == top[n] && l[n] == rest[0]);
            }
            const int who = __builtin_ctzl(same);
            const int expert = who * C + __builtin_amdgcn_readlane(at[n], who);
            mine[n] = lane == j && top[n] != 0 ? expert : mine[n];
            const bool gone = lane == who;  // (with nothing left everything is 0 already)
            if constexpr (SORTED) {
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    high[n][i] = gone ? (i + 1 < C ? high[n][i + 1 < C ? i + 1 : i] : 0) : high[n][i];
                    if (i + 1 < C) place[n][i] = gone ? place[n][i + 1 < C ? i + 1 : i] : place[n][i];
                    if (WIDE && i + 1 < C) low[n][WIDE ? i : 0] = gone ? low[n][WIDE && i + 1 < C ? i + 1 : 0] : low[n][WIDE ? i : 0];
                }
            } else {
#pragma unroll
                for (int i = 0; i < C; ++i) high[n][i] = gone && i == at[n] ? 0 : high[n][i];
            }
        }
    }
    double w[T];
#pragma unroll
    for (int n = 0; n < T; ++n) {
        const float value = mine[n] >= 0 ? z[n][mine[n]] : 0.0f;
        w[n] = mine[n] >= 0 ? score(n, value) : 0.0;
    }
#pragma unroll
    for (int n = 0; n < T; ++n) {
        if (a.normalize) {
            const double sum = wave_sum64(w[n]);
            w[n] = sum > 0.0 ? w[n] / sum : 0.0;
        }
        if (lane < a.k) {
            const long p = static_cast<long>(t + n * step) * a.k + lane;
            a.ids[p] = mine[n];
            a.weights[p] = static_cast<float>(w[n] * a.scale);
        }
    }
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

// The block's pairs to their places: run[e] is where its first pair of expert e goes.  `first`: the expert of the thread's first pair.
// run comes from counts that another call may have written over (a workspace shared by calls that are not ordered, ids that
// change meanwhile): a place that is no row is not followed.
__device__ __forceinline__ void place(const RouteArgs& a, Shared& s, long p0, long p1, int first) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bits = 32 - __builtin_clz(a.E);
    for (long base = p0; base < p1; base += kThreads) {
        for (int w = 0; w < kWaves; ++w)
            if (tid < a.E) s.wave[w][tid] = 0;
        __syncthreads();
        const long p = base + tid;
        const int e = base == p0 ? first : p < p1 ? expert_of(a, p) : a.E;
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
            if (to >= 0 && to < a.M * a.k) a.rows[to] = static_cast<int>(p);
        }
        __syncthreads();
        if (tid < a.E) s.run[tid] += more;
    }
}

__device__ __forceinline__ void write_rest(const RouteArgs& a, int all, int block, int blocks) {
    const long R = static_cast<long>(a.M) * a.k;
    for (long r = max(all, 0) + block * static_cast<long>(kThreads) + threadIdx.x; r < R; r += static_cast<long>(blocks) * kThreads)
        a.rows[r] = -1;
}

// Chooses (with logits) and counts the block's pairs; a single block groups them, too.
template <int C, bool WIDE, int T>
__global__ __launch_bounds__(kThreads) void route_kernel(const RouteArgs a) {
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < a.E) s.count[tid] = 0;
    __syncthreads();
    const int t0 = blockIdx.x * a.per, t1 = min(t0 + a.per, a.M);
    if (a.logits != nullptr) {
        const auto take = [&](auto tokens, int t) {
            int e[decltype(tokens)::value];
            choose<C, WIDE>(a, t, kWaves, e);
            for (int n : e)
                if (lane < a.k && n >= 0) atomicAdd(&s.count[n], 1);
        };
        int t = t0 + wave;
        if constexpr (T == 2)
            for (; t + kWaves < t1; t += 2 * kWaves) take(std::integral_constant<int, 2>{}, t);
        for (; t < t1; t += kWaves) take(std::integral_constant<int, 1>{}, t);
    } else {
        for (long p = static_cast<long>(t0) * a.k + tid; p < static_cast<long>(t1) * a.k; p += kThreads) {
            const int e = expert_of(a, p);
            if (e < a.E) atomicAdd(&s.count[e], 1);
        }
    }
    __syncthreads();  // (the ids of this block are read again below: written by this workgroup)
    const int n = tid < a.E ? s.count[tid] : 0;
    if (gridDim.x > 1) {
        if (tid < padded(a.E)) a.counts[static_cast<long>(blockIdx.x) * padded(a.E) + tid] = n;
        return;
    }
    int all;
    const int before = block_scan(n, s, all);
    if (tid < a.E) {
        s.run[tid] = before;
        a.offsets[tid] = before;
    }
    if (tid == 0) a.offsets[a.E] = all;
    const long pairs = static_cast<long>(a.M) * a.k;
    place(a, s, 0, pairs, tid < pairs ? expert_of(a, tid) : a.E);
    write_rest(a, all, 0, 1);
}

// The second launch: offsets from all blocks' counts, and the block's pairs to their places.
__global__ __launch_bounds__(kThreads) void group_kernel(const RouteArgs a, int blocks) {
    __shared__ Shared s;
    const int tid = threadIdx.x, block = blockIdx.x;
    const int t0 = block * a.per, t1 = min(t0 + a.per, a.M);
    const long p0 = static_cast<long>(t0) * a.k, p1 = static_cast<long>(t1) * a.k;
    const int first = p0 + tid < p1 ? expert_of(a, p0 + tid) : a.E;  // (asked for with the counts)
    // the counts of four experts by several threads, a run of blocks each
    const int row = padded(a.E), quads = row >> 2;
    int width = 16;
    while (width < quads) width <<= 1;
    const int shares = kThreads / width, q = tid & (width - 1), share = tid / width;
    const int each = (blocks + shares - 1) / shares, b0 = share * each, b1 = min(b0 + each, blocks);
    i32x4 sum = {0, 0, 0, 0}, earlier = sum;
    if (q < quads) {
        for (int b = b0; b < b1; b += 16) {
            i32x4_a4 n[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) n[i] = *reinterpret_cast<const i32x4_a4*>(a.counts + static_cast<long>(min(b + i, b1 - 1)) * row + 4 * q);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sum += b + i < b1 ? n[i] : i32x4{0, 0, 0, 0};
                earlier += b + i < min(b1, block) ? n[i] : i32x4{0, 0, 0, 0};
            }
        }
    }
    s.parts[0][tid] = sum;
    s.parts[1][tid] = earlier;
    __syncthreads();
    int total = 0, before = 0;
    if (tid < a.E) {
        for (int i = 0; i < shares; ++i) {
            total += s.parts[0][i * width + (tid >> 2)][tid & 3];
            before += s.parts[1][i * width + (tid >> 2)][tid & 3];
        }
    }
    int all;
    const int start = block_scan(total, s, all);
    if (tid < a.E) {
        s.run[tid] = start + before;
        if (block == 0) a.offsets[tid] = start;
    }
    if (block == 0 && tid == 0) a.offsets[a.E] = all;
    place(a, s, p0, p1, first);
    write_rest(a, all, block, blocks);
}

// tokens of a block: one block up to kSingle tokens, at most kBlocks of them else
int block_tokens(int M) { return M <= kSingle ? std::max(M, 1) : std::max((M + kBlocks - 1) / kBlocks, kWaves); }

void launch(RouteArgs a, hipStream_t stream) {
    a.per = block_tokens(a.M);
    const int blocks = std::max((a.M + a.per - 1) / a.per, 1);
    const bool biased = a.logits != nullptr && a.bias != nullptr, pairs = a.per > kWaves;
    const int c = a.logits == nullptr ? 1 : (a.E + 63) / 64;
#define CRI_ROUTE(C) \
    (biased ? (pairs && C < 16 ? route_kernel<C, true, C < 16 ? 2 : 1> : route_kernel<C, true, 1>) : (pairs ? route_kernel<C, false, 2> : route_kernel<C, false, 1>))
    const auto run = c == 1 ? CRI_ROUTE(1) : c == 2 ? CRI_ROUTE(2) : c <= 4 ? CRI_ROUTE(4) : c <= 8 ? CRI_ROUTE(8) : CRI_ROUTE(16);
#undef CRI_ROUTE
    hipLaunchKernelGGL(run, dim3(blocks), dim3(kThreads), 0, stream, a);
    if (blocks > 1) hipLaunchKernelGGL(group_kernel, dim3(blocks), dim3(kThreads), 0, stream, a, blocks);
}

}  // namespace
}  // namespace dev

namespace detail {

long expert_group_workspace_bytes(int n_tokens, int, int n_experts) {
    if (n_tokens <= dev::kSingle) return 0;
    const int per = dev::block_tokens(n_tokens);
    return static_cast<long>((n_tokens + per - 1) / per) * dev::padded(n_experts) * 4;
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
