// verify.hip -- drafted tokens checked against the target's probabilities from given random numbers.
//
// Sequence s has the rows offsets[s] .. offsets[s + 1] - 1, n of them: n - 1 drafted tokens, then the row behind the
// last one.  Draft j (token x, target probabilities p, draft probabilities q, number u of its row) is accepted when
// u q(x) < p(x); at the first that is not, the token is drawn from max(p - q, 0) instead, and when all are accepted
// from the last row's p, both by inverting the running sum at the row's second number d: the smallest v whose sum of
// weights up to and with v exceeds d times the total.
//
//   * u q(x) < p(x) is decided in 64 bits, where the product of two 32-bit numbers is exact.
//   * Weights are differences in 64 bits and so are their sums, whose order is fixed: per lane, wave, slice.
//   * Bound by memory: one row of p and of q per sequence (2 V floats), whatever the number of drafts.  A sequence's
//     rows are cut into slices over workgroups, so that a single sequence, too, is read by many CUs; the second
//     kernel finds the slice by the slices' sums and the token within it, re-reading that slice alone.
#include <algorithm>

#include "common.hpp"
#include "internal.hpp"

namespace cri {
namespace dev {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

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

// the weight of token v: what the draft leaves of p, or p itself
struct Weight {
    const float* p;
    const float* q;  // null: none
    int sure;        // the token a draft without probabilities is sure of, or -1
    __device__ __forceinline__ void at(int v, double& w, double& t) const {
        t = p[v] > 0.0f ? static_cast<double>(p[v]) : 0.0;  // NaN counts as zero
        w = t;
        if (q != nullptr) {
            w = t - static_cast<double>(q[v]);
            w = w > 0.0 ? w : 0.0;
        }
        if (v == sure) w = 0.0;
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

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// grid (sequences x slices): the slice's sums
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(const VerifyArgs a) {
    __shared__ double part[2][kWaves];
    const int s = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    int first, n, acc;
    accept(a, s, first, n, acc);
    if (n == 0) return;
    const Weight W = weight_of(a, first, n, acc);
    const int lo = slice * a.per, hi = min(lo + a.per, a.V);
    double w = 0.0, t = 0.0;
    for (int v = lo + threadIdx.x; v < hi; v += kThreads) {
        double x, y;
        W.at(v, x, y);
        w += x;
        t += y;
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

// grid (sequences): the token, the sequence's output rows
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(const VerifyArgs a) {
    __shared__ double part[kWaves];
    __shared__ int found[kWaves], last[kWaves];
    const int s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int first, n, acc;
    accept(a, s, first, n, acc);
    if (n == 0) {
        if (threadIdx.x == 0) a.accepted[s] = 0;
        return;
    }
    Weight W = weight_of(a, first, n, acc);
    const double* sums = a.sums + static_cast<long>(s) * a.slices * 2;
    double total = 0.0, plain = 0.0;
    for (int i = 0; i < a.slices; ++i) {
        total += sums[2 * i];
        plain += sums[2 * i + 1];
    }
    const int which = total > 0.0 ? 0 : 1;  // the draft leaves nothing: from p itself
    if (which) {
        W.q = nullptr;
        W.sure = -1;
        total = plain;
    }
    const double want = a.draws[first + acc] * total;
    // the slice: the first whose running sum exceeds the wanted one, else the last with any weight
    double before = 0.0, run = 0.0;
    int slice = -1, heavy = -1;
    double heavy_before = 0.0;
    for (int i = 0; i < a.slices; ++i) {
        const double x = sums[2 * i + which];
        if (x > 0.0) {
            heavy = i;
            heavy_before = run;
        }
        if (run + x > want) {
            slice = i;
            before = run;
            break;
        }
        run += x;
    }
    if (slice < 0) {
        slice = heavy;
        before = heavy_before;
    }
    int token = -1;  // no weight anywhere
    if (slice >= 0) {
        const int lo = slice * a.per, hi = min(lo + a.per, a.V);
        double at = before;
        int best = -1;
        for (int v0 = lo; v0 < hi; v0 += kThreads) {
            const int v = v0 + threadIdx.x;
            double x = 0.0, y;
            if (v < hi) W.at(v, x, y);
            double c = x;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const double o = __shfl_up(c, m);
                if (lane >= m) c += o;
            }
            if (lane == 63) part[wave] = c;
            __syncthreads();
            double base = at;
            for (int i = 0; i < wave; ++i) base += part[i];
            const unsigned long hit = __ballot(x > 0.0 && base + c > want), any = __ballot(x > 0.0);
            if (lane == 0) {
                found[wave] = hit ? v0 + wave * 64 + __builtin_ctzl(hit) : -1;
                last[wave] = any ? v0 + wave * 64 + 63 - __builtin_clzl(any) : -1;
            }
            __syncthreads();
            for (int i = 0; i < kWaves; ++i) {
                at += part[i];
                if (last[i] >= 0) best = last[i];
            }
            for (int i = kWaves - 1; i >= 0; --i)
                if (found[i] >= 0) token = found[i];
            __syncthreads();
            if (token >= 0) break;
        }
        if (token < 0) token = best;
    }
    for (int j = threadIdx.x; j < n; j += kThreads)
        a.out[first + j] = j < acc ? a.ids[first + j] : j == acc ? token : -1;
    if (threadIdx.x == 0) a.accepted[s] = acc;
}

// slices of a row: about 1024 workgroups over all sequences, of at least 1024 tokens
int slices_of(int n_seqs, int V) {
    const int most = (V + 1023) / 1024;
    return std::max(1, std::min(most, (1024 + n_seqs - 1) / n_seqs));
}

}  // namespace
}  // namespace dev

namespace detail {

long verify_workspace_bytes(int n_seqs, int vocab) {
    return static_cast<long>(n_seqs) * dev::slices_of(n_seqs, vocab) * 16;
}

int launch_verify_drafts(const float* target, long ldt, const float* draft, long ldd, const int* ids, const float* u,
                         const float* draws, const int* offsets, int n_seqs, int n_rows, int vocab, int* out, int* accepted, double* ws,
                         hipStream_t stream) {
    dev::VerifyArgs a{target, draft, ldt, ldd, ids, u, draws, offsets, out, accepted, ws, n_seqs, n_rows, vocab, 0, 0};
    a.slices = dev::slices_of(n_seqs, vocab);
    a.per = (vocab + a.slices - 1) / a.slices;
    hipLaunchKernelGGL(dev::verify_sums_kernel, dim3(static_cast<unsigned>(n_seqs) * a.slices), dim3(dev::kThreads), 0, stream, a);
    hipLaunchKernelGGL(dev::verify_pick_kernel, dim3(n_seqs), dim3(dev::kThreads), 0, stream, a);
    return 0;
}

}  // namespace detail
}  // namespace cri
