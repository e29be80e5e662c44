// experts_check.cpp -- cuinfer/experts.h from a host program: `cpu` the refusals (nothing reaches the GPU), `gpu` two experts
// whose matrices are multiples of the identity, so that results are known without arithmetic.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <stdexcept>
#include <vector>

#include "cuinfer/experts.h"
#include "cuinfer/hip_utils.h"

using namespace cuinfer;

#define EXPECT(x)                                            \
    do {                                                     \
        if (!(x)) {                                          \
            std::printf("line %d: %s\n", __LINE__, #x);      \
            return 1;                                        \
        }                                                    \
    } while (0)

template <class F>
bool throws(F f, const char* word) {
    try {
        f();
    } catch (const std::runtime_error& e) {
        return std::strstr(e.what(), word) != nullptr;
    }
    return false;
}

char* fake(int i) { return reinterpret_cast<char*>(static_cast<uintptr_t>(i) << 24); }

int cpu() {
    const ExpertWeights w{fake(1), CRI_Q4_K, 4, 64, 512};
    ExpertGroups g{reinterpret_cast<int*>(fake(2)), reinterpret_cast<int*>(fake(3)), reinterpret_cast<int*>(fake(4)), 3, 2, 4};
    float *x = reinterpret_cast<float*>(fake(5)), *out = reinterpret_cast<float*>(fake(6)), *c = reinterpret_cast<float*>(fake(7));
    int* ids = reinterpret_cast<int*>(fake(8));
    EXPECT(expert_packed_bytes(CRI_Q4_K, 4, 64, 512) > 4 * 64 * 512 / 2);
    EXPECT(group_experts_workspace_bytes(g) == 0);
    EXPECT(expert_matmul_workspace_bytes(w, g) >= 0 && expert_swiglu_workspace_bytes(w, g) >= 0 && expert_combine_workspace_bytes(w, g) >= 0);
    EXPECT(throws([&] { expert_packed_bytes(CRI_Q4_K, 4, 64, 500); }, "multiple of 256"));
    EXPECT(throws([&] { pack_experts(CRI_Q4_K, fake(9), 4, 64, 512, fake(10) + 4); }, "aligned"));
    EXPECT(throws([&] { route_experts({nullptr, 1.0f, 7, 1}, x, 4, ids, c, g, nullptr, 0); }, "scoring"));
    EXPECT(throws([&] { group_experts(nullptr, g, nullptr, 0); }, "null ids"));
    EXPECT(throws([&] { expert_matmul(w, g, x, 511, false, out, 64, fake(11), 1 << 20); }, "x"));
    ExpertWeights up = w;
    up.N = 32;
    EXPECT(throws([&] { expert_swiglu(w, up, g, x, 512, out, 64, fake(11), 1 << 20); }, "same format"));
    EXPECT(throws([&] { expert_combine(w, g, x, 512, c, out + 1, 64, out, 64, fake(11), 1 << 20); }, "overlap"));
    g.top_k = 5;
    EXPECT(throws([&] { group_experts_workspace_bytes(g); }, "top_k=5"));
    return 0;
}

template <class T>
T* up(const std::vector<T>& h) {
    T* d = nullptr;
    CUINFER_CHECK_HIP(hipMalloc(&d, h.size() * sizeof(T)));
    CUINFER_CHECK_HIP(hipMemcpy(d, h.data(), h.size() * sizeof(T), hipMemcpyHostToDevice));
    return d;
}
template <class T>
std::vector<T> down(const T* d, size_t n) {
    std::vector<T> h(n);
    CUINFER_CHECK_HIP(hipDeviceSynchronize());
    CUINFER_CHECK_HIP(hipMemcpy(h.data(), d, n * sizeof(T), hipMemcpyDeviceToHost));
    return h;
}
void* room(long long bytes) {
    void* p = nullptr;
    CUINFER_CHECK_HIP(hipMalloc(&p, bytes + 16));
    return p;
}

int gpu() {
    const int E = 2, D = 32, M = 3;
    std::vector<uint16_t> blocks(E * D * D, 0);
    for (int i = 0; i < D; ++i) {
        blocks[i * D + i] = 0x3C00;          // expert 0: 1
        blocks[(D + i) * D + i] = 0x4000;    // expert 1: 2
    }
    const ExpertWeights w{room(expert_packed_bytes(CRI_FP16, E, D, D)), CRI_FP16, E, D, D};
    pack_experts(CRI_FP16, up(blocks), E, D, D, const_cast<void*>(w.data));
    const ExpertGroups g{up(std::vector<int>(E + 1, 9)), up(std::vector<int>(M, 9)), up(std::vector<int>(M, 9)), M, 1, E};
    int* ids = up(std::vector<int>(M, 9));
    float* weights = up(std::vector<float>(M, 9.0f));
    const long long rb = group_experts_workspace_bytes(g);
    // tokens 0 and 2 to expert 1, token 1 to none
    float* logits = up(std::vector<float>{0.0f, 1.0f, -INFINITY, -INFINITY, -3.0f, -2.0f});
    route_experts({nullptr, 0.5f, CRI_SCORE_SOFTMAX, 1}, logits, E, ids, weights, g, room(rb), rb);
    EXPECT((down(ids, M) == std::vector<int>{1, -1, 1}));
    EXPECT((down(weights, M) == std::vector<float>{0.5f, 0.0f, 0.5f}));
    EXPECT((down(g.offsets, E + 1) == std::vector<int>{0, 0, 2}));
    EXPECT((down(g.rows, M) == std::vector<int>{0, 2, -1}));
    EXPECT((down(g.slots, M) == std::vector<int>{0, -1, 1}));
    std::vector<float> x(M * D);
    for (int i = 0; i < M * D; ++i) x[i] = static_cast<float>(20 + i);
    float *dx = up(x), *out = up(std::vector<float>(M * D, 7.0f));
    long long bytes = expert_matmul_workspace_bytes(w, g);
    expert_matmul(w, g, dx, D, false, out, D, room(bytes), bytes);
    auto o = down(out, M * D);
    for (int i = 0; i < D; ++i) EXPECT(o[i] == 2 * x[i] && o[D + i] == 2 * x[2 * D + i] && o[2 * D + i] == 7.0f);
    bytes = expert_swiglu_workspace_bytes(w, g);
    expert_swiglu(w, w, g, dx, D, out, D, room(bytes), bytes);  // silu(v) = v from 20 on, to the last bit
    o = down(out, M * D);
    for (int i = 0; i < D; ++i) {
        const float a = 4 * x[i] * x[i], b = 4 * x[2 * D + i] * x[2 * D + i];
        EXPECT(std::fabs(o[i] - a) <= 1e-6f * a && std::fabs(o[D + i] - b) <= 1e-6f * b && o[2 * D + i] == 7.0f);
    }
    // grouped rows 0 and 1 are 20 .. and 20 + D ..; token 1 keeps its residual
    float* res = up(std::vector<float>(M * D, 1.0f));
    bytes = expert_combine_workspace_bytes(w, g);
    expert_combine(w, g, dx, D, weights, res, D, res, D, room(bytes), bytes);
    o = down(res, M * D);
    for (int i = 0; i < D; ++i) EXPECT(o[i] == 1.0f + x[i] && o[D + i] == 1.0f && o[2 * D + i] == 1.0f + x[D + i]);
    group_experts(up(std::vector<int>{1, 0, 5}), g, room(rb), rb);
    EXPECT((down(g.offsets, E + 1) == std::vector<int>{0, 1, 2}));
    EXPECT((down(g.slots, M) == std::vector<int>{1, 0, -1}));
    return 0;
}

int main(int argc, char** argv) {
    if (argc != 2) return 2;
    const int rc = std::strcmp(argv[1], "gpu") == 0 ? gpu() : cpu();
    if (rc == 0) std::printf("ok\n");
    return rc;
}
