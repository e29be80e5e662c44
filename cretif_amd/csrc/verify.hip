// verify.hip -- drafted tokens checked against the target's probabilities from given random numbers.
//
// Sequence s has the rows offsets[s] .. offsets[s + 1] - 1, n of them: n - 1 drafted tokens, then the row behind the
// last one.  Draft j (token x, target probabilities p, draft probabilities q, number u of its row) is accepted when
// u q(x) < p(x); at the first that is not, the token is drawn from max(p - q, 0) instead, and when all are accepted
// from the last row's p, both by inverting the running sum at the row's second number d: the smallest v whose sum of
// weights up to and with v exceeds d times the total.
//
//   * u q(x) < p(x) is decided in 64 bits, where the product of two 32-bit numbers is exact.
//   * Weights are differences in 64 bits and so are their sums, whose order is fixed: thread, wave, slice.
//   * Bound by memory: one row of p and of q per sequence (2 V floats), whatever the number of drafts.
//   * Up to 32768 tokens a sequence's row fits the registers of one workgroup of 1024 threads, and one kernel does it all
//     (verify_row_kernel).  Us in a graph, against the two kernels below at 33000: one sequence 7.0 / 9.0, 64 9.2 / 12.8, 200
//     12.0 / 19.3, 256 14.0 / 20.3; 200 with sure drafts, 25.6 MB, 9.7.  1000 tokens: 3.9 for one sequence, 4.5 for 256.
//   * Longer rows are cut into slices over workgroups, so that a single sequence, too, is read by many CUs
//     (verify_sums_kernel).  The second kernel finds the slice by the slices' sums and the token within it in one pass of
//     1024 threads, eight tokens each, over that slice alone, which the first kernel has left in the caches.  128256
//     tokens: 64 sequences 12.6 us (65.7 MB at 5.2 TB/s) and 6.3 us, one sequence 4.0 and 6.3, the second being the chain of
//     trips to memory behind the first's sums.
#include <algorithm>

#include "common.hpp"
#include "internal.hpp"

namespace cri {
namespace dev {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / 64;
constexpr int kPer = 8;                          // tokens of a picking thread
constexpr int kMaxSlice = kPer * kPickThreads;  // tokens of a slice

struct VerifyArgs {
    const float* target;
    const float* draft;
    long ldt, ldd;
    const int* ids;
    const float* u;      // decide about the drafts
    const float* draws;  // draw the token
    const int* offsets;
    int* out;
    int* accepted;
    double* sums;  // [n_seqs][slices]: sums of the weights, of p
    int* counts;   // [n_seqs]: drafts accepted, -1 for a sequence of no rows
    int n_seqs, n_rows, V, slices, per;
};

// the sequence's first row, its row count and the drafts accepted; count 0: none
__device__ __forceinline__ void accept(const VerifyArgs& a, int s, int& first, int& n, int& acc) {
    first = a.offsets[s];
    n = a.offsets[s + 1] - first;
    acc = 0;
    if (n <= 0 || first < 0 || first > a.n_rows - n) {
        n = 0;
        return;
    }
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < n - 1; base += 64) {
        const int j = base + lane;
        bool stop = false;
        if (j < n - 1) {
            const long r = first + j;
            const int x = a.ids[r];
            stop = true;
            if (x >= 0 && x < a.V) {
                const double q = a.draft ? static_cast<double>(a.draft[r * a.ldd + x]) : 1.0;
                stop = !(a.u[r] * q < static_cast<double>(a.target[r * a.ldt + x]));
            }
        }
        const unsigned long b = __ballot(stop);
        if (b != 0) {
            acc = base + __builtin_ctzl(b);
            return;
        }
    }
    acc = n - 1;
}

// the weights of tokens: what the draft leaves of p, or p itself
struct Weight {
    const float* p;
    const float* q;  // null: none
    int sure;        // the token a draft without probabilities is sure of, or -1
    // NaN and negative p count as zero, a NaN q leaves nothing (both maxima take the zero)
    static __device__ __forceinline__ double of(float pv, float qv) {
        return fmax(static_cast<double>(fmaxf(pv, 0.0f)) - static_cast<double>(qv), 0.0);
    }
    // tokens v .. v + 3, zeros from hi on
    __device__ __forceinline__ void load4(int v, int hi, f32x4& pv, f32x4& qv) const {
        pv = qv = f32x4{0, 0, 0, 0};
        if (v + 4 <= hi) {
            pv = ld_f32x4(p + v);
            if (q != nullptr) qv = ld_f32x4(q + v);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                if (v + i < hi) {
                    pv[i] = p[v + i];
                    if (q != nullptr) qv[i] = q[v + i];
                }
            }
        }
    }
    // what load4 read, without the sure token
    __device__ __forceinline__ void drop4(int v, f32x4& pv) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) pv[i] = v + i == sure ? 0.0f : pv[i];
    }
};
__device__ __forceinline__ Weight weight_of(const VerifyArgs& a, int first, int n, int acc) {
    const long r = first + acc;
    const bool rejected = acc < n - 1;
    Weight w;
    w.p = a.target + r * a.ldt;
    w.q = rejected && a.draft ? a.draft + r * a.ldd : nullptr;
    w.sure = rejected && !a.draft ? a.ids[r] : -1;
    return w;
}

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {  // zero where the source lane is outside
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {  // of a uniform lane
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// sums over the lanes up to and with each; prev: without the lane's own
__device__ __forceinline__ double scan_up(double v, int lane, double& prev) {
    v += dpp_f64<0x111>(v);  // row_shr 1, 2, 4, 8: within 16 lanes
    v += dpp_f64<0x112>(v);
    v += dpp_f64<0x114>(v);
    v += dpp_f64<0x118>(v);
    const double a = lane_f64(v, 15), b = a + lane_f64(v, 31), c = b + lane_f64(v, 47);
    const double base = lane < 16 ? 0.0 : lane < 32 ? a : lane < 48 ? b : c;
    prev = base + dpp_f64<0x111>(v);
    return base + v;
}
__device__ __forceinline__ double wave_sum(double v) {
    double prev;
    return lane_f64(scan_up(v, threadIdx.x & 63, prev), 63);
}

// grid (sequences x slices): the slice's sums
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(const VerifyArgs a) {
    __shared__ double part[2][kWaves];
    const int s = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    int first, n, acc;
    accept(a, s, first, n, acc);
    if (slice == 0 && threadIdx.x == 0) a.counts[s] = n == 0 ? -1 : acc;
    if (n == 0) return;
    const Weight W = weight_of(a, first, n, acc);
    const int lo = slice * a.per, hi = min(lo + a.per, a.V);
    double w = 0.0, t = 0.0;
    constexpr int kAhead = 4;  // loads of p and of q in flight
    for (int v0 = lo + 4 * threadIdx.x; v0 < hi; v0 += 4 * kThreads * kAhead) {
        f32x4 p[kAhead], q[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) W.load4(v0 + 4 * kThreads * j, hi, p[j], q[j]);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) t += Weight::of(p[j][i], 0.0f);
            W.drop4(v0 + 4 * kThreads * j, p[j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) w += Weight::of(p[j][i], q[j][i]);
        }
    }
    w = wave_sum(w);
    t = wave_sum(t);
    if ((threadIdx.x & 63) == 0) {
        part[0][threadIdx.x >> 6] = w;
        part[1][threadIdx.x >> 6] = t;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        w = t = 0.0;
        for (int i = 0; i < kWaves; ++i) {
            w += part[0][i];
            t += part[1][i];
        }
        a.sums[(static_cast<long>(s) * a.slices + slice) * 2] = w;
        a.sums[(static_cast<long>(s) * a.slices + slice) * 2 + 1] = t;
    }
}

// the sequence's output rows but the drawn one; id: the thread's drafted token
__device__ __forceinline__ void write_rest(const VerifyArgs& a, int first, int n, int acc, int id) {
    if (static_cast<int>(threadIdx.x) < acc) a.out[first + threadIdx.x] = id;
    for (int j = threadIdx.x + kPickThreads; j < acc; j += kPickThreads) a.out[first + j] = a.ids[first + j];
    for (int j = acc + 1 + threadIdx.x; j < n; j += kPickThreads) a.out[first + j] = -1;
}

// grid (sequences): the token, the sequence's output rows
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(const VerifyArgs a) {
    __shared__ double part[kPickWaves];
    __shared__ int found[kPickWaves], last[kPickWaves];
    const int s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int acc = a.counts[s], first = a.offsets[s], n = a.offsets[s + 1] - first;
    if (acc < 0) {
        if (threadIdx.x == 0) a.accepted[s] = 0;
        return;
    }
    Weight W = weight_of(a, first, n, acc);
    const float number = a.draws[first + acc];  // (on their way beside the sums)
    const int id = static_cast<int>(threadIdx.x) < acc ? a.ids[first + threadIdx.x] : -1;
    // every wave: the totals, then the first slice whose running sum exceeds the wanted one, else the last with weight
    const double* sums = a.sums + static_cast<long>(s) * a.slices * 2;
    double total = 0.0, plain = 0.0;
    for (int i = lane; i < a.slices; i += 64) {
        total += sums[2 * i];
        plain += sums[2 * i + 1];
    }
    total = wave_sum(total);
    plain = wave_sum(plain);
    const int which = total > 0.0 ? 0 : 1;  // the draft leaves nothing: from p itself
    if (which) {
        W.q = nullptr;
        W.sure = -1;
        total = plain;
    }
    const double want = number * total;
    double before = 0.0, run = 0.0;
    int slice = -1;
    for (int base = 0; base < a.slices; base += 64) {
        const int i = base + lane;
        const double x = i < a.slices ? sums[2 * i + which] : 0.0;
        double prev;
        const double c = scan_up(x, lane, prev), at = run + prev;
        const unsigned long hit = __ballot(x > 0.0 && run + c > want), any = __ballot(x > 0.0);
        if (any != 0) {
            const int pick = hit ? __builtin_ctzl(hit) : 63 - __builtin_clzl(any);
            slice = base + pick;
            before = lane_f64(at, pick);
        }
        if (hit != 0) break;
        run += lane_f64(c, 63);
    }
    int token = -1;  // no weight anywhere
    if (slice >= 0) {
        const int lo = slice * a.per, hi = min(lo + a.per, a.V), v0 = lo + kPer * threadIdx.x;
        double x[kPer], sum = 0.0;
#pragma unroll
        for (int j = 0; j < kPer; j += 4) {
            f32x4 p, q;
            W.load4(v0 + j, hi, p, q);
            W.drop4(v0 + j, p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[j + i] = Weight::of(p[i], q[i]);
                sum += x[j + i];
            }
        }
        double prev;
        const double c = scan_up(sum, lane, prev);
        if (lane == 63) part[wave] = c;
        __syncthreads();
        double base = before;
        for (int i = 0; i < wave; ++i) base += part[i];
        const unsigned long hit = __ballot(sum > 0.0 && base + c > want), any = __ballot(sum > 0.0);
        // the thread's token: the first whose running sum exceeds the wanted one, else its last with weight
        int mine = -1;
        double at = base + prev;
        bool done = false;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            at += x[j];
            if (x[j] > 0.0 && !done) {
                mine = v0 + j;
                done = at > want;
            }
        }
        const int hit_token = __builtin_amdgcn_readlane(mine, hit ? __builtin_ctzl(hit) : 0);
        const int any_token = __builtin_amdgcn_readlane(mine, any ? 63 - __builtin_clzl(any) : 0);
        if (lane == 0) {
            found[wave] = hit ? hit_token : -1;
            last[wave] = any ? any_token : -1;
        }
        __syncthreads();
        for (int i = 0; i < kPickWaves; ++i)
            if (last[i] >= 0) token = last[i];
        for (int i = kPickWaves - 1; i >= 0; --i)
            if (found[i] >= 0) token = found[i];
    }
    if (threadIdx.x == 0) {
        a.out[first + acc] = token;
        a.accepted[s] = acc;
    }
    write_rest(a, first, n, acc, id);
}

// grid (sequences), vocabularies up to kRowVocab: the whole of it in one kernel.  Wave w holds the w-th of the row's
// sixteenths in registers, 256 tokens at a time; the waves' sums name the wave whose tokens are drawn from, which sums its
// 256s one by one.
constexpr int kQuads = 8, kRowVocab = 4 * kQuads * kPickThreads;  // kQuads: of a thread

// QUADS: of a thread at most; Q: there are draft probabilities
template <int QUADS, bool Q>
__global__ __launch_bounds__(kPickThreads) void verify_row_kernel(const VerifyArgs a) {
    __shared__ double part[2][kPickWaves];
    const int s = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int first, n, acc;
    accept(a, s, first, n, acc);
    if (n == 0) {
        if (threadIdx.x == 0) a.accepted[s] = 0;
        return;
    }
    Weight W = weight_of(a, first, n, acc);
    const int slabs = (a.V + 256 * kPickWaves - 1) / (256 * kPickWaves), v0 = wave * slabs * 256 + 4 * lane;
    f32x4 p[QUADS], q[Q ? QUADS : 1];
    const float number = a.draws[first + acc];
    const int id = static_cast<int>(threadIdx.x) < acc ? a.ids[first + threadIdx.x] : -1;
    auto load = [&]() {
#pragma unroll
        for (int j = 0; j < QUADS; ++j) W.load4(v0 + 256 * j, j < slabs ? a.V : 0, p[j], q[Q ? j : 0]);
        if constexpr (!Q) {
#pragma unroll
            for (int j = 0; j < QUADS; ++j) W.drop4(v0 + 256 * j, p[j]);
        }
    };
    auto weight = [&](int j, int i) { return Weight::of(p[j][i], Q ? q[j][i] : 0.0f); };
    load();

    double c, want;
    int pick;
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {  // again from p itself where the draft leaves nothing
        double w = 0.0;
#pragma unroll
        for (int j = 0; j < QUADS; ++j)
            if (j < slabs) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w += weight(j, i);
            }
        w = wave_sum(w);
        if (lane == 0) part[turn][wave] = w;
        __syncthreads();
        const double x = lane < kPickWaves ? part[turn][lane] : 0.0;
        double prev;
        c = scan_up(x, lane, prev);
        const double total = lane_f64(c, 63);
        want = number * total;
        const unsigned long hit = __ballot(x > 0.0 && c > want), any = __ballot(x > 0.0);
        pick = hit ? __builtin_ctzl(hit) : any ? 63 - __builtin_clzl(any) : -1;
        c = prev;
        if (total > 0.0) break;
        W.q = nullptr;
        W.sure = -1;
        load();
    }
    if (wave == max(pick, 0)) {
        int token = -1;
        if (pick >= 0) {
            double run = lane_f64(c, pick), at = run, x[4] = {};
            int slab = 0;
            bool done = false;
#pragma unroll
            for (int j = 0; j < QUADS; ++j) {
                if (j >= slabs || done) continue;
                double y[4], sum = 0.0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[i] = weight(j, i);
                    sum += y[i];
                }
                sum = wave_sum(sum);
                if (sum > 0.0) {  // the first whose running sum exceeds the wanted one, else the last with weight
                    slab = j, at = run;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = y[i];
                    done = run + sum > want;
                }
                run += sum;
            }
            const double sum = ((x[0] + x[1]) + x[2]) + x[3];
            double prev;
            const double up = scan_up(sum, lane, prev);
            const unsigned long hit = __ballot(sum > 0.0 && at + up > want), any = __ballot(sum > 0.0);
            int mine = 0;
            double here = at + prev;
            done = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                here += x[i];
                if (x[i] > 0.0 && !done) {
                    mine = i;
                    done = here > want;
                }
            }
            const int who = hit ? __builtin_ctzl(hit) : 63 - __builtin_clzl(any);
            token = wave * slabs * 256 + slab * 256 + 4 * who + __builtin_amdgcn_readlane(mine, who);
        }
        if (lane == 0) {
            a.out[first + acc] = token;
            a.accepted[s] = acc;
        }
    }
    write_rest(a, first, n, acc, id);
}

// tokens of a slice: about 1024 workgroups over all sequences, 1024 to kMaxSlice tokens each
int slice_of(int n_seqs, int V) {
    const int slices = std::max((1024 + n_seqs - 1) / n_seqs, 1);
    return std::min(std::max((V / slices + 1023) / 1024 * 1024, 1024), kMaxSlice);
}

}  // namespace
}  // namespace dev

namespace detail {

long verify_workspace_bytes(int n_seqs, int vocab) {
    const int per = dev::slice_of(n_seqs, vocab), slices = (vocab - 1) / per + 1;
    return static_cast<long>(n_seqs) * (slices * 16L + 4);
}

int launch_verify_drafts(const float* target, long ldt, const float* draft, long ldd, const int* ids, const float* u,
                         const float* draws, const int* offsets, int n_seqs, int n_rows, int vocab, int* out, int* accepted,
                         double* ws, hipStream_t stream) {
    if (vocab <= dev::kRowVocab) {
        const dev::VerifyArgs a{target, draft, ldt, ldd, ids, u, draws, offsets, out, accepted, nullptr, nullptr,
                                n_seqs, n_rows, vocab, 1, vocab};
        const auto run = vocab <= dev::kRowVocab / 4 ? (draft ? dev::verify_row_kernel<dev::kQuads / 4, true>
                                                              : dev::verify_row_kernel<dev::kQuads / 4, false>)
                                                     : (draft ? dev::verify_row_kernel<dev::kQuads, true>
                                                              : dev::verify_row_kernel<dev::kQuads, false>);
        hipLaunchKernelGGL(run, dim3(n_seqs), dim3(dev::kPickThreads), 0, stream, a);
        return 0;
    }
    const int per = dev::slice_of(n_seqs, vocab), slices = (vocab - 1) / per + 1;
    if (static_cast<long>(n_seqs) * slices >= 1L << 24) return kDeclined;  // 256 threads each: a launch's limit
    const dev::VerifyArgs a{target, draft, ldt, ldd, ids, u, draws, offsets, out, accepted, ws,
                            reinterpret_cast<int*>(ws + 2L * n_seqs * slices), n_seqs, n_rows, vocab, slices, per};
    hipLaunchKernelGGL(dev::verify_sums_kernel, dim3(static_cast<unsigned>(n_seqs) * slices), dim3(dev::kThreads), 0, stream, a);
    hipLaunchKernelGGL(dev::verify_pick_kernel, dim3(n_seqs), dim3(dev::kPickThreads), 0, stream, a);
    return 0;
}

}  // namespace detail
}  // namespace cri
