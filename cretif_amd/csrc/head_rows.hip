// head_rows.hip -- query and key heads normed and rotated, and keys and values appended to a paged cache.
//
// Per head row x of head_dim elements: y = x * rsqrt(mean(x^2) + eps) * w (w null: y = x), then the pairs (a, b) of
// the first rot_dim elements turn by the angle p * theta^(-2i / rot_dim) of position p and pair i:
// (a cos - b sin, b cos + a sin).  Values go to the cache as they are.
//
//   * Bound by memory: every row is read once and written once.  A row lies in the registers of head_dim / 8 lanes
//     (rounded up to a power of two), eight elements each: for adjacent pairs eight consecutive ones, for halves four
//     of each half, so both elements of a pair are in one lane, the norm is a sum over the row's lanes on DPP, and
//     nothing goes through LDS.
//   * A lane meets the same four pairs in every row of its token, so a workgroup takes one token and its lanes
//     compute their four angles once: the exponent and the product with the position in 64 bits (at position 10^6 a
//     32-bit angle is off by 0.06 radians), reduced to a half turn in 64 bits, sine and cosine in 32.
//   * The sequence of a row is found by the wave: 64 offsets compared at a time.
//
// 8192 rows, 32/8 heads of 128 out of a fused product: 65 us, 335 MB at 5.2 TB/s (a large copy moves 4.7); 6921 rows
// appended in bf16 with their queries 60 us, 312 MB at 5.2; one row 3.0 us, 64 rows 4.1, which are three trips to memory.
#include "paged.hpp"

namespace cri {
namespace dev {
namespace {

constexpr int kThreads = 256;

struct RowArgs {
    const float* q;
    const float* k;
    const float* v;
    float* q_out;
    float* k_out;
    long ldq, ldk, ldv, ldqo, ldko;
    const int* positions;
    HeadRotation R;
    PagePool P;
    PageBatch B;
    int H, Hkv, D, lg;  // lg: log2 of the lanes of a row
    int nrows;          // rows of a token: H + Hkv (+ Hkv values)
};

// the sequence that row t belongs to, the place of its first row and its row count; false for a row of none
__device__ __forceinline__ bool find_sequence(const PageBatch& B, int t, int& seq, int& first, int& count) {
    const int lane = threadIdx.x & 63;
    int s = 0;
    for (int base = 0; base < B.n_seqs; base += 64) {
        const int i = base + lane;
        const bool before = i < B.n_seqs && B.offsets[i + 1] <= t;
        const int n = __popcll(__ballot(before));
        s += n;
        if (n < 64) break;
    }
    if (s >= B.n_seqs) return false;
    first = B.offsets[s];
    const int end = B.offsets[s + 1];
    seq = s;
    count = end - first;
    return t >= first && t < end;
}

template <int TYPE>
__device__ __forceinline__ void store4(typename KvType<TYPE>::elem* p, const float* x) {
    if constexpr (TYPE == kKvF32)
        *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    else if constexpr (TYPE == kKvF16)
        *reinterpret_cast<h16x4*>(p) = __builtin_convertvector((f32x4{x[0], x[1], x[2], x[3]}), h16x4);
    else
        *reinterpret_cast<b16x4*>(p) = __builtin_convertvector((f32x4{x[0], x[1], x[2], x[3]}), b16x4);
}

// grid (tokens, parts of a token's rows); PAGED: k and v rows go to the cache, rounded to its type (to nearest)
template <int TYPE, bool PAGED>
__global__ __launch_bounds__(kThreads) void head_rows_kernel(const RowArgs a) {
    typedef typename KvType<TYPE>::elem elem;
    const int t = blockIdx.x, L = 1 << a.lg, c = threadIdx.x & (L - 1), per = kThreads >> a.lg;
    const bool on = c < a.D / 8;
    // the lane's eight elements: quads qa and qb, the four pairs 4 c .. 4 c + 3 where it rotates
    const int r8 = a.R.rot_dim / 8;
    const bool turn = c < r8;
    const bool split = a.R.halves && turn;
    const int qa = split ? 4 * c : 8 * c, qb = split ? 4 * (c + r8) : 8 * c + 4;

    int pos;
    long place = 0;
    if constexpr (PAGED) {
        int seq, first, count;
        if (!find_sequence(a.B, t, seq, first, count)) return;
        pos = a.B.lens[seq] - count + (t - first);
        if (pos < 0) return;
        const int pi = page_index(a.P, pos);
        if (pi >= a.B.max_pages) return;
        const int page = a.B.pages[static_cast<long>(seq) * a.B.max_pages + pi];
        if (page < 0 || page >= a.P.n_pages) return;
        place = page * a.P.stride + static_cast<long>(pos - pi * a.P.page_size) * a.P.n_kv_heads * a.D;
    } else {
        pos = a.positions[t];
    }
    float cs[4] = {1.0f, 1.0f, 1.0f, 1.0f}, sn[4] = {};
    if (turn) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // half turns: the angle over pi, less an even number
            const double x = pos * exp2((4 * c + i) * a.R.log2_step) * 0.31830988618379067154;
            sincospif(static_cast<float>(x - 2.0 * rint(0.5 * x)), &sn[i], &cs[i]);
        }
    }
    for (int r = blockIdx.y * per + (threadIdx.x >> a.lg); r < a.nrows; r += gridDim.y * per) {
        const bool is_q = r < a.H, is_k = !is_q && r < a.H + a.Hkv;
        const int h = is_q ? r : is_k ? r - a.H : r - a.H - a.Hkv;
        const float* src = is_q ? a.q + t * a.ldq : is_k ? a.k + t * a.ldk : a.v + t * a.ldv;
        src += static_cast<long>(h) * a.D;
        float x[8] = {};
        if (on) {
            const f32x4 u = ld_f32x4(src + qa), w = ld_f32x4(src + qb);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = u[i];
                x[4 + i] = w[i];
            }
        }
        const float* norm = is_q ? a.R.q_norm : is_k ? a.R.k_norm : nullptr;
        if (norm != nullptr) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
            s = group_sum(s, a.lg);
            const float f = 1.0f / sqrtf(s / a.D + a.R.eps);
            if (on) {
                const f32x4 u = ld_f32x4(norm + qa), w = ld_f32x4(norm + qb);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] *= f * u[i];
                    x[4 + i] *= f * w[i];
                }
            }
        }
        if (turn && (is_q || is_k)) {
            // pair i: (x[i], x[4 + i]) of two halves, (x[2 i], x[2 i + 1]) of neighbours
            float y[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = split ? x[i] : x[2 * i], w = split ? x[4 + i] : x[2 * i + 1];
                const float p = u * cs[i] - w * sn[i], q = w * cs[i] + u * sn[i];
                y[i] = p;
                y[4 + i] = q;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = split ? y[i] : (i & 1) ? y[4 + i / 2] : y[i / 2];
                x[4 + i] = split ? y[4 + i] : (i & 1) ? y[4 + 2 + i / 2] : y[2 + i / 2];
            }
        }
        if (!on) continue;
        if (!PAGED || is_q) {
            float* dst = (is_q ? a.q_out + t * a.ldqo : a.k_out + t * a.ldko) + static_cast<long>(h) * a.D;
            *reinterpret_cast<f32x4_a4*>(dst + qa) = f32x4_a4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4_a4*>(dst + qb) = f32x4_a4{x[4], x[5], x[6], x[7]};
        } else {
            elem* dst = static_cast<elem*>(is_k ? a.P.k : a.P.v) + place + static_cast<long>(h) * a.D;
            store4<TYPE>(dst + qa, x);
            store4<TYPE>(dst + qb, x + 4);
        }
    }
}

// lanes of a row and the grid
void set_rows(RowArgs& a, int rows) {
    a.nrows = rows;
    a.lg = 0;
    while ((8 << a.lg) < a.D) ++a.lg;
}

dim3 grid_of(const RowArgs& a, int tokens) {
    const int per = kThreads >> a.lg, parts = (a.nrows + per - 1) / per;
    // few tokens: a workgroup per part of a token's rows, so that none waits for two; from 1024 on, which fill the GPU, one
    // per token, whose angles serve all its rows
    return dim3(static_cast<unsigned>(tokens), static_cast<unsigned>(tokens >= 1024 ? 1 : parts));
}

}  // namespace
}  // namespace dev

namespace detail {

int launch_qk_norm_rope(const HeadRotation& R, const float* q, long ldq, const float* k, long ldk, float* q_out,
                        long ldqo, float* k_out, long ldko, const int* positions, int M, int n_heads, int n_kv_heads,
                        int head_dim, hipStream_t stream) {
    dev::RowArgs a{};
    a.q = q, a.k = k, a.q_out = q_out, a.k_out = k_out;
    a.ldq = ldq, a.ldk = ldk, a.ldqo = ldqo, a.ldko = ldko;
    a.positions = positions;
    a.R = R;
    a.H = n_heads, a.Hkv = n_kv_heads, a.D = head_dim;
    dev::set_rows(a, n_heads + n_kv_heads);
    hipLaunchKernelGGL((dev::head_rows_kernel<kKvF32, false>), dev::grid_of(a, M), dim3(dev::kThreads), 0, stream, a);
    return 0;
}

int launch_paged_append(const PagePool& P, int type, const PageBatch& B, const HeadRotation& R, const float* q,
                        long ldq, float* q_out, long ldqo, int n_heads, const float* k, long ldk, const float* v,
                        long ldv, hipStream_t stream) {
    dev::RowArgs a{};
    a.q = q, a.k = k, a.v = v, a.q_out = q_out;
    a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldqo = ldqo;
    a.R = R, a.P = P, a.B = B;
    a.H = q ? n_heads : 0, a.Hkv = P.n_kv_heads, a.D = P.head_dim;
    dev::set_rows(a, a.H + 2 * a.Hkv);
    const dim3 grid = dev::grid_of(a, B.n_rows), block(dev::kThreads);
    if (type == kKvF32)
        hipLaunchKernelGGL((dev::head_rows_kernel<kKvF32, true>), grid, block, 0, stream, a);
    else if (type == kKvF16)
        hipLaunchKernelGGL((dev::head_rows_kernel<kKvF16, true>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((dev::head_rows_kernel<kKvBF16, true>), grid, block, 0, stream, a);
    return 0;
}

}  // namespace detail
}  // namespace cri
