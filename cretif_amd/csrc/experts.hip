// experts.hip -- a layer of experts: the activations as planes for the grouped products, the products' choice of kernel,
// and the weighted sum of a token's experts.  The products are in experts_gemm.hpp, the routing in experts_route.hip.
#include <algorithm>
#include <cmath>

#include "act.hpp"
#include "experts.hpp"

namespace cri {
namespace dev {
namespace {

typedef _Float16 eh8 __attribute__((ext_vector_type(8)));

// Activations as the products take them: row r is 2^exps[r] (hi + lo), |hi| up to 2^15, hi and lo to the nearest half, per 64
// k 64 of hi and 64 of lo, zeros from K on; for Q4_K also the sums over 32 k times 2^-6 (32 terms below 2^15 then fit
// fp16) in the same two parts.  A workgroup per row, read twice (the second time from the caches): K floats in, as many
// bytes out; 4096 x 2048 takes 15 us, 32768 x 1024 45 (5.9 TB/s).
struct PlanesArgs {
    const float* x;
    long ldx;
    const int* end;  // rows from *end on are not needed, or null
    uint8_t* planes;
    uint8_t* sums;  // null: not needed
    int* exps;
    int K, depth;
};

__global__ __launch_bounds__(256) void planes_kernel(const PlanesArgs a) {
    __shared__ float most[4];
    const int r = blockIdx.x, tid = threadIdx.x;
    if (a.end != nullptr && r >= *a.end) return;
    const float* x = a.x + r * a.ldx;
    const int chunks = a.K >> 3, all = a.depth * 32;  // of 8
    float mx = 0.0f;
    for (int c = tid; c < chunks; c += 256) {
        const f32x4 u = ld_f32x4(x + 8 * c), v = ld_f32x4(x + 8 * c + 4);
        mx = fmaxf(mx, fmaxf(fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(u.z), fabsf(u.w))),
                             fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)))));
    }
    mx = wave_max(mx);
    if ((tid & 63) == 0) most[tid >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    int ex = 0;
    if (mx > 0.0f) {
        frexpf(mx, &ex);
        ex -= 15;
    }
    if (tid == 0) a.exps[r] = ex;
    uint8_t* plane = a.planes + r * static_cast<long>(a.depth) * 1024;
    for (int c = tid; c < all; c += 256) {  // (all is a multiple of 32, so lanes of a quad stay together)
        f32x4 u = f32x4{0, 0, 0, 0}, v = u;
        if (c < chunks) {
            u = ld_f32x4(x + 8 * c);
            v = ld_f32x4(x + 8 * c + 4);
        }
        eh8 hi, lo;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = ldexpf(i < 4 ? u[i] : v[i - 4], -ex);
            sum += y;
            hi[i] = static_cast<_Float16>(y);
            lo[i] = static_cast<_Float16>(y - static_cast<float>(hi[i]));
        }
        uint8_t* to = plane + (c >> 3) * 256 + (c & 7) * 16;
        *reinterpret_cast<eh8*>(to) = hi;
        *reinterpret_cast<eh8*>(to + 128) = lo;
        if (a.sums != nullptr) {
            sum += dpp<kQuadPerm1032>(sum);
            sum += dpp<kQuadPerm2301>(sum);
            if ((c & 3) == 0) {
                sum *= 0.015625f;
                _Float16* o = reinterpret_cast<_Float16*>(a.sums + (r * static_cast<long>(a.depth) + (c >> 5)) * 32) + ((c >> 2) & 7);
                o[0] = static_cast<_Float16>(sum);
                o[8] = static_cast<_Float16>(sum - static_cast<float>(o[0]));
            }
        }
    }
}

// out[t] = residual[t] + sum over the token's choices, in their order, of weight * p[slot]; choices without an expert are
// left out, whatever their weight.  Bound by memory: k + 2 rows per token.
struct CombineArgs {
    const float* p;  // [splits][R, ldp], 16-byte aligned rows, to be added up
    const float* weights;
    const int* slots;
    const float* residual;  // or null
    float* out;
    long ldp, ldr, ldo;
    int N, k, R, splits;
};

__global__ __launch_bounds__(256) void combine_kernel(const CombineArgs a) {
    const int t = blockIdx.x, col = (blockIdx.y * 256 + threadIdx.x) * 4;
    if (col >= a.N) return;
    const int left = a.N - col;
    const int* slots = a.slots + static_cast<long>(t) * a.k;
    const float* weights = a.weights + static_cast<long>(t) * a.k;
    const float* res = a.residual == nullptr ? nullptr : a.residual + t * a.ldr + col;
    f32x4 first = f32x4{0, 0, 0, 0}, sum = first;
    if (res != nullptr) {
        if (left >= 4) {
            first = ld_f32x4(res);
        } else {
            for (int i = 0; i < left; ++i) first[i] = res[i];
        }
    }
    for (int j0 = 0; j0 < a.k; j0 += 4) {
        f32x4 v[4];
        float w[4];
        bool there[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = min(j0 + i, a.k - 1), slot = slots[j];
            there[i] = j0 + i < a.k && slot >= 0 && slot < a.R;
            w[i] = weights[j];
            const float* p = a.p + (there[i] ? slot : 0) * a.ldp + col;
            v[i] = *reinterpret_cast<const f32x4*>(p);
            for (int s = 1; s < a.splits; ++s) v[i] += *reinterpret_cast<const f32x4*>(p + s * (a.R * a.ldp));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (there[i]) {
#pragma unroll
                for (int c = 0; c < 4; ++c) sum[c] = __builtin_fmaf(w[i], v[i][c], sum[c]);
            }
    }
    sum += first;
    float* out = a.out + t * a.ldo + col;
    if (left >= 4) {
        *reinterpret_cast<f32x4_a4*>(out) = f32x4_a4{sum.x, sum.y, sum.z, sum.w};
    } else {
        for (int i = 0; i < left; ++i) out[i] = sum[i];
    }
}

// The parts of k of a product (SwiGLU: of both) added up in order: out[r], for the rows that have an expert.
struct JoinArgs {
    const float* p;  // [splits][matrices][R, ldp], 16-byte aligned rows
    const int* end;
    float* out;
    long ldp, ldo;
    int N, R, splits;
};

template <bool SWIGLU>
__global__ __launch_bounds__(256) void join_kernel(const JoinArgs a) {
    constexpr int NT = SWIGLU ? 2 : 1;
    const int r = blockIdx.x, col = (blockIdx.y * 256 + threadIdx.x) * 4;
    if (col >= a.N || r >= *a.end) return;
    const long part = a.R * a.ldp;
    const float* p = a.p + r * a.ldp + col;
    f32x4 v[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) v[n] = *reinterpret_cast<const f32x4*>(p + n * part);
    for (int s = 1; s < a.splits; ++s)
#pragma unroll
        for (int n = 0; n < NT; ++n) v[n] += *reinterpret_cast<const f32x4*>(p + (s * NT + n) * part);
    if constexpr (SWIGLU) {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[0][c] = silu_f(v[0][c]) * v[1][c];
    }
    float* out = a.out + r * a.ldo + col;
    if (a.N - col >= 4) {
        *reinterpret_cast<f32x4_a4*>(out) = f32x4_a4{v[0].x, v[0].y, v[0].z, v[0].w};
    } else {
        for (int i = 0; i < a.N - col; ++i) out[i] = v[0][i];
    }
}

}  // namespace
}  // namespace dev

namespace detail {
namespace {

// Which kernel: few with tiles of 2^lg rows and so many waves, else rows with tiles of bm and k in so many parts.
struct Plan {
    bool few;
    int bm, lg, waves, splits;
};
// what is made of the products (cri_expert_op)
enum class Use { kMatmul, kSwiglu, kCombine };

// The one that a rough model of both gives the least time, in us; it knows only host numbers, so rows are taken to be spread
// over the experts.  All read the weights of the experts that have rows at 5.5 TB/s at best (as counted here: the calls that this
// was fitted to named some experts more than others, 48 tokens, 4 of 60, 38 and not 58).  few_kernel: 8 us, 0.6 ns for each
// unit that a tile meets (that often as a 256th of the GPU) and 0.1 ns for each row of it.  rows_kernel: 8.8 us with the planes'
// pass, then stages of 64 k at 0.42, 0.52 or 0.88 us (16, 32, 64 rows) while a CU has one workgroup or less, 0.47, 0.52 or 0.96 us
// for each beyond, some of a last round that is not full; an expert's further tiles read its weights again at 0.28 of the
// cost.  k in several parts costs their sums a way to memory and back at 3.8 TB/s and a launch (the combination adds them up
// itself).  `weight` is what decoding and scaling a format takes of either, beside Q4_0; Q6_K, whose decoding is the longest, gains
// most by 64 rows that share it (1000 tokens, 2 of 16, 2048 -> 2048: 80.5 us against 82.9 with 32).  Over 189 calls of all formats what it
// takes was 1.5% slower than the best on average, 29% at most.
// Measured, few (8 rows, 4 waves) / 16 / 32 / 64 rows, us: SwiGLU 2048 -> 1024 of 64 experts, 8 each, Q4_K: 4 tokens 18 / 24 / 27 /
// 38, 16: 26 / 30 / 34 / 50, 48: 49 / 40 / 44 / 67, 256: 169 / 82 / 81 / 98, 512: 314 / 140 / 118 / 128, 1024: 643 / 270 / 195 / 195.
// 8192 -> 2048 Q4_0, one of 8 experts each, 128 tokens: 61 / 66 / 74 / 106, k in two parts - / 42 / 47 / 64, in four - / 39 / 44 / 45.
Plan plan_products(const ExpertMatrix& w, const ExpertRows& g, Use use) {
    const bool swiglu = use == Use::kSwiglu;
    const double few_weight[] = {1.35, 1.2, 1.65, 1.1, 1.75, 1.55}, rows_weight[] = {1.7, 1.0, 1.2, 1.1, 1.2, 1.3};  // by format
    const int depth = (w.K + dev::kUnitK - 1) / dev::kUnitK, tiles = (w.N + dev::kUnitCols - 1) / dev::kUnitCols;
    const double R = static_cast<double>(g.n_tokens) * g.top_k, E = w.n_experts;
    const double used = E * (1.0 - std::pow(1.0 - 1.0 / E, R)), matrices = swiglu ? 2.0 : 1.0;
    const auto row_tiles = [&](int bm) { return std::min(std::max(used, R / bm + used / 2), R); };
    const double memory = used * tiles * depth * matrices * dev::unit_bytes(w.fmt) / 5.5e6;

    const bool single = R < 1.15 * used;  // an expert's rows: hardly ever more than one
    const int lg = single ? 0 : g.n_tokens <= 4 ? 2 : 3;
    const double units = tiles * depth * matrices * 1e-3;
    Plan best{true, 0, lg, std::min(depth, lg < 3 && (used * tiles <= 256 || depth >= 16) ? 8 : 4), 1};
    double least = 8.0 + std::max(memory, units * (0.6 * few_weight[w.fmt] * row_tiles(1 << lg) + 0.1 * R));
    const double blocks = dev::rows_blocks(tiles, swiglu);
    const double part = R * w.N * matrices * 4e-6;  // MB
    const struct {
        int bm;
        double one, each;
    } kinds[] = {{16, 0.42, 0.47}, {32, 0.52, 0.52}, {64, 0.88, 0.96}};
    for (const auto& k : kinds) {
        for (int splits = 1; splits <= std::min(depth, 8) && (splits == 1 || part * splits <= 256); splits *= 2) {
            double load = row_tiles(k.bm) * blocks * splits / 256;  // workgroups of a CU
            if (load > 1.0) load += 0.38 * (std::ceil(load) - load);
            const double shared = w.fmt == kFmtQ6_K && k.bm == 64 ? 0.87 : 1.0;
            const double stage = std::max(k.one, k.each * load) * rows_weight[w.fmt] * shared;
            const int stages = splits == 1 ? (w.K + 63) / 64 : 4 * ((depth + splits - 1) / splits);
            const double join = splits == 1 ? 0.0 : use == Use::kCombine ? part * 2 * (splits - 1) / 3.8 : 2.3 + part * 2 * splits / 3.8;
            const double us = 8.8 + join + std::max(memory * (0.72 + 0.28 * row_tiles(k.bm) / used), stages * stage);
            if (us < least) {
                least = us;
                best = Plan{false, k.bm, 0, 0, splits};
            }
        }
    }
    return best;
}

long up16(long bytes) { return (bytes + 15) & ~15L; }

// bytes of the planes, sums and exponents of `rows` rows
struct PlaneBytes {
    long planes, sums, exps;
    long all() const { return planes + sums + exps; }
};
PlaneBytes plane_bytes(const ExpertMatrix& w, long rows) {
    const long depth = (w.K + dev::kUnitK - 1) / dev::kUnitK;
    return {rows * depth * 1024, w.fmt == kFmtQ4_K ? rows * depth * 32 : 0, up16(rows * 4)};
}

dev::ProductArgs product_args(const ExpertMatrix& w, const ExpertRows& g, const float* x, long ldx, bool gather, float* out,
                              long ldo) {
    dev::ProductArgs a{};
    a.w[0] = a.w[1] = static_cast<const uint8_t*>(w.data);
    a.g = dev::Groups{g.offsets, g.rows, g.slots, w.n_experts, g.top_k, g.n_tokens * g.top_k};
    a.x = x;
    a.ldx = ldx;
    a.out = out;
    a.ldo = ldo;
    a.N = w.N;
    a.K = w.K;
    a.tiles = (w.N + dev::kUnitCols - 1) / dev::kUnitCols;
    a.depth = (w.K + dev::kUnitK - 1) / dev::kUnitK;
    a.gather = gather;
    a.over_k = ((1u << 31) + g.top_k - 1) / g.top_k;
    return a;
}

long product_columns(const ExpertMatrix& w) { return (w.N + 3L) & ~3L; }

// bytes of the parts of k that are to be added up
long part_bytes(const ExpertMatrix& w, long rows, const Plan& plan, bool swiglu) {
    return plan.few || plan.splits == 1 ? 0 : up16(plan.splits * (swiglu ? 2 : 1) * rows * product_columns(w) * 4);
}

// The product of w (and up: SiLU(x w^T) * (x up^T)) into out, rows in grouped order; for Use::kCombine out is
// [plan.splits][R][ldo].
int launch_products(const Plan& plan, Use use, const ExpertMatrix& w, const ExpertMatrix* up, const ExpertRows& g, const float* x,
                    long ldx, bool gather, float* out, long ldo, void* ws, hipStream_t stream) {
    const long R = static_cast<long>(g.n_tokens) * g.top_k;
    const int depth = (w.K + dev::kUnitK - 1) / dev::kUnitK, tiles = (w.N + dev::kUnitCols - 1) / dev::kUnitCols;
    const bool swiglu = up != nullptr;
    dev::ProductArgs a = product_args(w, g, x, ldx, gather, out, ldo);
    if (swiglu) a.w[1] = static_cast<const uint8_t*>(up->data);
    const int blocks = plan.few ? tiles : dev::rows_blocks(tiles, swiglu) * plan.splits;
    const long groups = (dev::most_tiles(R, w.n_experts, plan.few ? 1 << plan.lg : plan.bm) * blocks + 7) / 8 * 8;
    if (groups >= 1L << 23) return kDeclined;  // up to 512 threads each: a launch's limit
    if (plan.few) {
        switch (w.fmt) {
            case kFmtQ8_0: dev::expert_few<kFmtQ8_0>(a, swiglu, plan.lg, plan.waves, groups, stream); break;
            case kFmtQ4_0: dev::expert_few<kFmtQ4_0>(a, swiglu, plan.lg, plan.waves, groups, stream); break;
            case kFmtQ5_0: dev::expert_few<kFmtQ5_0>(a, swiglu, plan.lg, plan.waves, groups, stream); break;
            case kFmtQ4_K: dev::expert_few<kFmtQ4_K>(a, swiglu, plan.lg, plan.waves, groups, stream); break;
            case kFmtQ6_K: dev::expert_few<kFmtQ6_K>(a, swiglu, plan.lg, plan.waves, groups, stream); break;
            default: dev::expert_few<kFmtF16>(a, swiglu, plan.lg, plan.waves, groups, stream);
        }
        return 0;
    }
    const long rows = gather ? g.n_tokens : R;
    const PlaneBytes b = plane_bytes(w, rows);
    uint8_t* const room = static_cast<uint8_t*>(ws);
    const dev::PlanesArgs p{x, ldx, gather ? nullptr : g.offsets + w.n_experts, room, b.sums ? room + b.planes : nullptr,
                            reinterpret_cast<int*>(room + b.planes + b.sums), w.K, depth};
    hipLaunchKernelGGL(dev::planes_kernel, dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream, p);
    a.planes = p.planes;
    a.sums = p.sums;
    a.exps = p.exps;
    a.splits = plan.splits;
    const bool join = plan.splits > 1 && use != Use::kCombine;
    if (join) {
        a.out = reinterpret_cast<float*>(room + b.all());
        a.ldo = product_columns(w);
    }
    switch (w.fmt) {
        case kFmtQ8_0: dev::expert_rows<kFmtQ8_0>(a, swiglu, plan.bm, groups, stream); break;
        case kFmtQ4_0: dev::expert_rows<kFmtQ4_0>(a, swiglu, plan.bm, groups, stream); break;
        case kFmtQ5_0: dev::expert_rows<kFmtQ5_0>(a, swiglu, plan.bm, groups, stream); break;
        case kFmtQ4_K: dev::expert_rows<kFmtQ4_K>(a, swiglu, plan.bm, groups, stream); break;
        case kFmtQ6_K: dev::expert_rows<kFmtQ6_K>(a, swiglu, plan.bm, groups, stream); break;
        default: dev::expert_rows<kFmtF16>(a, swiglu, plan.bm, groups, stream);
    }
    if (join) {
        const dev::JoinArgs j{a.out, g.offsets + w.n_experts, out, a.ldo, ldo, w.N, static_cast<int>(R), plan.splits};
        hipLaunchKernelGGL(swiglu ? dev::join_kernel<true> : dev::join_kernel<false>,
                           dim3(static_cast<unsigned>(R), static_cast<unsigned>((w.N + 1023) / 1024)), dim3(256), 0, stream, j);
    }
    return 0;
}

// Whether a call's weighted sums are taken in one launch, two workgroups per token and column tile, which read an expert's
// weights for every token that has it: where those are two rounds of workgroups at most.  Us, two launches / one: 1024 -> 2048
// Q6_K, 8 of 64 experts each: 1 token 11.1 / 8.0, 4 16.2 / 15.0, 5 18.5 / 19.8, 8 21.5 / 26.1; 1536 -> 576 Q8_0, 4 of 32: 12 tokens
// 12.7 / 11.7.
bool token_takes(const ExpertMatrix& w, const ExpertRows& g) {
    return static_cast<long>(g.n_tokens) * ((w.N + dev::kUnitCols - 1) / dev::kUnitCols) <= 256;
}

}  // namespace

void expert_plan(const ExpertMatrix& w, const ExpertRows& g, int op, int (&plan)[3]) {
    const bool one = op == static_cast<int>(Use::kCombine) && token_takes(w, g);
    const Plan p = plan_products(w, g, static_cast<Use>(op));
    plan[0] = one ? 0 : p.few ? 1 << p.lg : p.bm;
    plan[1] = one ? 1 : p.splits;
    plan[2] = one ? 16 : p.few ? p.waves : 4;
}

long expert_product_workspace_bytes(const ExpertMatrix& w, const ExpertRows& g, bool swiglu, bool gather) {
    const Plan plan = plan_products(w, g, swiglu ? Use::kSwiglu : Use::kMatmul);
    const long R = static_cast<long>(g.n_tokens) * g.top_k;
    return plan.few ? 0 : plane_bytes(w, gather ? g.n_tokens : R).all() + part_bytes(w, R, plan, swiglu);
}

int launch_expert_products(const ExpertMatrix& w, const ExpertMatrix* up, const ExpertRows& g, const float* x, long ldx,
                           bool gather, float* out, long ldo, void* ws, hipStream_t stream) {
    const Use use = up != nullptr ? Use::kSwiglu : Use::kMatmul;
    return launch_products(plan_products(w, g, use), use, w, up, g, x, ldx, gather, out, ldo, ws, stream);
}

// combine: the products of all rows, then what the products need
long expert_combine_workspace_bytes(const ExpertMatrix& w, const ExpertRows& g) {
    if (token_takes(w, g)) return 0;
    const Plan plan = plan_products(w, g, Use::kCombine);
    const long R = static_cast<long>(g.n_tokens) * g.top_k;
    return up16(plan.splits * R * product_columns(w) * 4) + (plan.few ? 0 : plane_bytes(w, R).all());
}

int launch_expert_combine(const ExpertMatrix& w, const ExpertRows& g, const float* h, long ldh, const float* weights,
                          const float* residual, long ldr, float* out, long ldo, void* ws, hipStream_t stream) {
    if (token_takes(w, g)) {
        const dev::ProductArgs a = product_args(w, g, h, ldh, false, out, ldo);
        const dev::TokenArgs b{weights, residual, ldr};
        switch (w.fmt) {
            case kFmtQ8_0: dev::expert_token<kFmtQ8_0>(a, b, g.n_tokens, stream); break;
            case kFmtQ4_0: dev::expert_token<kFmtQ4_0>(a, b, g.n_tokens, stream); break;
            case kFmtQ5_0: dev::expert_token<kFmtQ5_0>(a, b, g.n_tokens, stream); break;
            case kFmtQ4_K: dev::expert_token<kFmtQ4_K>(a, b, g.n_tokens, stream); break;
            case kFmtQ6_K: dev::expert_token<kFmtQ6_K>(a, b, g.n_tokens, stream); break;
            default: dev::expert_token<kFmtF16>(a, b, g.n_tokens, stream);
        }
        return 0;
    }
    const long R = static_cast<long>(g.n_tokens) * g.top_k, ldp = product_columns(w);
    float* const p = static_cast<float*>(ws);
    const Plan plan = plan_products(w, g, Use::kCombine);
    const int rc = launch_products(plan, Use::kCombine, w, nullptr, g, h, ldh, false, p, ldp,
                                   reinterpret_cast<uint8_t*>(p) + up16(plan.splits * R * ldp * 4), stream);
    if (rc != 0) return rc;
    const dev::CombineArgs c{p, weights, g.slots, residual, out, ldp, ldr, ldo, w.N, g.top_k, static_cast<int>(R), plan.splits};
    hipLaunchKernelGGL(dev::combine_kernel, dim3(static_cast<unsigned>(g.n_tokens), static_cast<unsigned>((w.N + 1023) / 1024)),
                       dim3(256), 0, stream, c);
    return 0;
}

}  // namespace detail
}  // namespace cri
