// experts_pack.hip -- GGUF blocks [E, N, K] laid out once for the products of a layer of experts (experts.hpp says how),
// each weight's own bits moved to where the lane that multiplies it finds them; rows from N on and values from K on are
// weights of zero.  Runs once per matrix.
#include "decode.hpp"
#include "experts.hpp"

namespace cri {
namespace dev {
namespace {

struct PackArgs {
    const uint8_t* src;
    uint8_t* dst;
    long row_bytes, units;  // units of all experts
    int N, K, tiles, depth;  // column tiles and units along k of an expert
};

// the integer that element k of a row stands for, before the scale; `zero` where there is none
template <int FMT>
__device__ __forceinline__ uint32_t code(const uint8_t* row, int k) {
    if constexpr (FMT == kFmtQ8_0) {
        return static_cast<uint32_t>(static_cast<int8_t>(row[(k >> 5) * 34 + 2 + (k & 31)]) + 128);
    } else if constexpr (FMT == kFmtQ4_0) {
        const uint8_t* b = row + (k >> 5) * 18;
        return (b[2 + ((k & 31) >> 1)] >> (4 * (k & 1))) & 15u;
    } else if constexpr (FMT == kFmtQ5_0) {
        const uint8_t* b = row + (k >> 5) * 22;
        const int e = k & 31;
        return ((b[6 + (e & 15)] >> (4 * (e >> 4))) & 15u) | (((b[2 + (e >> 3)] >> (e & 7)) & 1u) << 4);
    } else if constexpr (FMT == kFmtQ4_K) {
        const uint8_t* b = row + (k >> 8) * 144 + 16;
        const int e = k & 255;
        return (b[(e >> 6) * 32 + (e & 31)] >> (4 * ((e >> 5) & 1))) & 15u;
    } else if constexpr (FMT == kFmtQ6_K) {
        const uint8_t* b = row + (k >> 8) * 210;
        const int e = k & 255, c = e >> 7, l = e & 31, quarter = (e >> 5) & 3;
        const uint32_t low = (b[64 * c + 32 * (quarter & 1) + l] >> (4 * (quarter >> 1))) & 15u;
        return low | (((b[128 + 32 * c + l] >> (2 * quarter)) & 3u) << 4);
    } else {
        return row[2 * k] | (static_cast<uint32_t>(row[2 * k + 1]) << 8);
    }
}

// nibble j of a step's dword (experts.hpp)
__device__ constexpr int kNibbleAt[8] = {0, 16, 4, 20, 8, 24, 12, 28};

constexpr int run_bytes(int fmt) { return kUnitK / (fmt == kFmtQ4_K || fmt == kFmtQ6_K ? 256 : fmt == kFmtF16 ? 1 : 32) * (fmt == kFmtQ8_0 ? 34 : fmt == kFmtQ4_0 ? 18 : fmt == kFmtQ5_0 ? 22 : fmt == kFmtQ4_K ? 144 : fmt == kFmtQ6_K ? 210 : 2); }

// A wave per unit: its 32 rows' bytes go to LDS, two at a time over consecutive lanes (a block begins at any even address), then
// lane (n, h) writes its own quants, lanes below 32 the scales of column n.
template <int FMT>
__global__ __launch_bounds__(256) void pack_kernel(const PackArgs a) {
    constexpr int kRun = run_bytes(FMT);  // bytes of a row in a unit
    __shared__ __attribute__((aligned(4))) uint8_t lds[4][FMT == kFmtF16 ? 4 : kUnitCols * kRun];  // (FP16: straight from memory)
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5, wave = threadIdx.x >> 6;
    const long u = static_cast<long>(blockIdx.x) * 4 + wave;
    const bool there = u < a.units;
    const long per = static_cast<long>(a.tiles) * a.depth, e = there ? u / per : 0, in = there ? u - e * per : 0;
    const int tile = static_cast<int>(in / a.depth), k0 = static_cast<int>(in - static_cast<long>(tile) * a.depth) * kUnitK;
    const long start = static_cast<long>(k0 / kUnitK) * kRun;
    const int rows = min(kUnitCols, a.N - tile * kUnitCols), bytes = static_cast<int>(min(static_cast<long>(kRun), a.row_bytes - start));
    const uint8_t* from = a.src + (e * a.N + static_cast<long>(tile) * kUnitCols) * a.row_bytes + start;
    if (there && FMT != kFmtF16) {
        if ((reinterpret_cast<uintptr_t>(a.src) & 1) == 0) {  // (row_bytes is even)
#pragma unroll 8
            for (int i = lane; i < rows * (kRun / 2); i += 64) {
                const int r = i / (kRun / 2), c = 2 * (i - r * (kRun / 2));
                if (c < bytes) *reinterpret_cast<uint16_t*>(&lds[wave][r * kRun + c]) = *reinterpret_cast<const uint16_t*>(from + r * a.row_bytes + c);
            }
        } else {
            for (int i = lane; i < rows * kRun; i += 64) {
                const int r = i / kRun, c = i - r * kRun;
                if (c < bytes) lds[wave][i] = from[r * a.row_bytes + c];
            }
        }
    }
    __syncthreads();
    if (!there) return;
    const bool real = n < rows;
    const uint8_t* row = FMT == kFmtF16 ? from + (real ? n : 0) * a.row_bytes : &lds[wave][(real ? n : 0) * kRun];
    uint8_t* unit = a.dst + u * unit_bytes(FMT);
    auto at = [&](int i, int j) -> uint32_t {  // weight j of the lane's step i
        const int k = 16 * i + 8 * h + j;
        return real && k0 + k < a.K ? code<FMT>(row, k) : 0u;
    };
    if constexpr (FMT == kFmtF16) {
        for (int i = 0; i < 16; ++i) {
            u32x4 v;
            for (int j = 0; j < 4; ++j) v[j] = at(i, 2 * j) | (at(i, 2 * j + 1) << 16);
            *reinterpret_cast<u32x4*>(unit + 1024 * i + 16 * lane) = v;
        }
        return;
    } else if constexpr (FMT == kFmtQ8_0) {
        for (int i = 0; i < 8; ++i) {
            u32x4 v;
            for (int j = 0; j < 4; ++j) {
                const int s = 2 * i + (j >> 1), w = 4 * (j & 1);
                v[j] = at(s, w) | (at(s, w + 1) << 16) | (at(s, w + 2) << 8) | (at(s, w + 3) << 24);
            }
            *reinterpret_cast<u32x4*>(unit + 1024 * i + 16 * lane) = v;
        }
    } else {
        uint32_t high[8] = {};
        for (int i = 0; i < 4; ++i) {
            u32x4 v = u32x4{0, 0, 0, 0};
            for (int s = 0; s < 4; ++s) {
                for (int j = 0; j < 8; ++j) {
                    const uint32_t q = at(4 * i + s, j);
                    v[s] |= (q & 15u) << kNibbleAt[j];
                    if (FMT == kFmtQ5_0) high[i] |= (q >> 4) << (4 * s + (j >> 1) + 16 * (j & 1));
                    if (FMT == kFmtQ6_K) high[2 * i + (s >> 1)] |= (q >> 4) << (2 * (4 * (s & 1) + (j >> 1)) + 16 * (j & 1));
                }
            }
            *reinterpret_cast<u32x4*>(unit + 1024 * i + 16 * lane) = v;
        }
        if constexpr (FMT == kFmtQ5_0) {
            *reinterpret_cast<u32x4*>(unit + 4096 + 16 * lane) = u32x4{high[0], high[1], high[2], high[3]};
        } else if constexpr (FMT == kFmtQ6_K) {
            *reinterpret_cast<u32x4*>(unit + 4096 + 16 * lane) = u32x4{high[0], high[1], high[2], high[3]};
            *reinterpret_cast<u32x4*>(unit + 5120 + 16 * lane) = u32x4{high[4], high[5], high[6], high[7]};
        }
    }
    if (h != 0) return;
    auto half = [&](const uint8_t* p) { return static_cast<uint32_t>(p[0] | (p[1] << 8)); };
    if constexpr (FMT == kFmtQ8_0 || FMT == kFmtQ4_0 || FMT == kFmtQ5_0) {
        constexpr int size = FMT == kFmtQ8_0 ? 34 : FMT == kFmtQ4_0 ? 18 : 22;
        u32x4 d = u32x4{0, 0, 0, 0};
        for (int i = 0; i < 8; ++i)
            if (real && k0 + 32 * i < a.K) d[i >> 1] |= half(row + i * size) << (16 * (i & 1));
        *reinterpret_cast<u32x4*>(unit + unit_bytes(FMT) - 512 + 16 * n) = d;
    } else if constexpr (FMT == kFmtQ4_K) {
        const uint8_t* b = row;
        u32x4 s = u32x4{0, 0, 0, 0};
        for (int i = 0; i < 8 && real; ++i) {
            const uint8_t* c = b + 4;
            const uint32_t sc = i < 4 ? c[i] & 63u : (c[i + 4] & 15u) | ((c[i - 4] >> 6) << 4);
            const uint32_t mn = i < 4 ? c[i + 4] & 63u : (c[i + 4] >> 4) | ((c[i] >> 6) << 4);
            s[i >> 2] |= sc << (8 * (i & 3));
            s[2 + (i >> 2)] |= mn << (8 * (i & 3));
        }
        *reinterpret_cast<u32x4*>(unit + 4096 + 16 * n) = s;
        *reinterpret_cast<uint32_t*>(unit + 4608 + 4 * n) = real ? half(b) | (half(b + 2) << 16) : 0u;
    } else {
        const uint8_t* b = row;
        u32x4 s = u32x4{0, 0, 0, 0};
        for (int i = 0; i < 16 && real; ++i) s[i >> 2] |= static_cast<uint32_t>(b[192 + i]) << (8 * (i & 3));
        *reinterpret_cast<u32x4*>(unit + 6144 + 16 * n) = s;
        *reinterpret_cast<uint16_t*>(unit + 6656 + 2 * n) = static_cast<uint16_t>(real ? half(b + 208) : 0u);
    }
}

}  // namespace
}  // namespace dev

namespace detail {

long expert_units(int n_experts, int N, int K) {
    return static_cast<long>(n_experts) * ((N + dev::kUnitCols - 1) / dev::kUnitCols) * ((K + dev::kUnitK - 1) / dev::kUnitK);
}

long expert_packed_bytes(int fmt, int n_experts, int N, int K) { return expert_units(n_experts, N, K) * dev::unit_bytes(fmt); }

int launch_expert_pack(int fmt, const void* src, int n_experts, int N, int K, void* dst, hipStream_t stream) {
    const dev::PackArgs a{static_cast<const uint8_t*>(src), static_cast<uint8_t*>(dst), row_bytes(fmt, K),
                          expert_units(n_experts, N, K), N, K, (N + dev::kUnitCols - 1) / dev::kUnitCols,
                          (K + dev::kUnitK - 1) / dev::kUnitK};
    const auto run = fmt == kFmtQ8_0   ? dev::pack_kernel<kFmtQ8_0>
                     : fmt == kFmtQ4_0 ? dev::pack_kernel<kFmtQ4_0>
                     : fmt == kFmtQ5_0 ? dev::pack_kernel<kFmtQ5_0>
                     : fmt == kFmtQ4_K ? dev::pack_kernel<kFmtQ4_K>
                     : fmt == kFmtQ6_K ? dev::pack_kernel<kFmtQ6_K>
                                       : dev::pack_kernel<kFmtF16>;
    hipLaunchKernelGGL(run, dim3(static_cast<unsigned>((a.units + 3) / 4)), dim3(256), 0, stream, a);
    return 0;
}

}  // namespace detail
}  // namespace cri
