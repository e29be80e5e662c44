// serving_check.cpp -- cuinfer/serving.h from a host program: `cpu` the refusals (nothing reaches the GPU), `gpu` one
// token appended, attended and verified, whose results are known without arithmetic.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstring>
#include <stdexcept>
#include <string>
#include <vector>

#include "cuinfer/hip_utils.h"
#include "cuinfer/serving.h"

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

float* fake() { return reinterpret_cast<float*>(1 << 20); }

int cpu() {
    PagedKV kv{fake(), fake(), 16 * 64, CRI_FP16, 4, 16, 1, 64};
    PagedBatch b{reinterpret_cast<int*>(fake()), reinterpret_cast<int*>(fake()), reinterpret_cast<int*>(fake()), 1, 1, 2};
    HeadRotation rot{nullptr, nullptr, 1e-6f, 1e4f, 64, CRI_ROPE_HALVES};
    EXPECT(paged_attention_workspace_bytes(kv, b, 32, 2) > 0);
    EXPECT(throws([&] { paged_attention_workspace_bytes(kv, b, -1, 2); }, "negative"));
    EXPECT(throws([&] { paged_attention(kv, b, nullptr, 32, fake(), 128, fake() + 4096, 128, 2, 1.0f, fake(), 1 << 30); },
                  "prefix_pages"));
    EXPECT(throws([&] { paged_append(kv, b, rot, nullptr, 0, nullptr, 0, 0, fake(), 63, fake(), 64); }, "below its width"));
    rot.rot_dim = 12;
    EXPECT(throws([&] { qk_norm_rope(rot, fake(), 64, nullptr, 0, fake(), 64, nullptr, 0, nullptr, 1, 1, 0, 64); }, "rot_dim"));
    EXPECT(throws([&] { verify_drafts_workspace_bytes(-1, 5); }, "negative"));
    EXPECT(throws([&] {
        verify_drafts(fake(), 4, nullptr, 0, nullptr, fake(), fake(), nullptr, 1, 1, 5, nullptr, nullptr, fake(), 0);
    }, "null"));
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

int gpu() {
    const int D = 64, H = 2, ps = 16;
    std::vector<float> zero(3 * ps * D, 0.0f), q(H * D, 1.0f), k(D, 2.0f), v(D);
    for (int i = 0; i < D; ++i) v[i] = 0.5f * i;
    PagedKV kv{up(zero), up(zero), ps * D, CRI_FP32, 3, ps, 1, D};
    PagedBatch b{up<int>({0, 1}), up<int>({1}), up<int>({2}), 1, 1, 1};
    HeadRotation rot{nullptr, nullptr, 0.0f, 1e4f, D, CRI_ROPE_HALVES};
    float *dq = up(q), *dk = up(k), *dv = up(v), *qo = up(std::vector<float>(H * D, 7.0f)), *out = up(std::vector<float>(H * D, 7.0f));
    paged_append(kv, b, rot, dq, H * D, qo, H * D, H, dk, D, dv, D);
    EXPECT(down(qo, H * D) == q);  // position 0: not turned
    const auto kp = down(static_cast<float*>(kv.k), 3 * ps * D), vp = down(static_cast<float*>(kv.v), 3 * ps * D);
    for (int i = 0; i < 3 * ps * D; ++i) {
        const int at = i - 2 * ps * D;
        EXPECT(kp[i] == (at >= 0 && at < D ? k[at] : 0.0f) && vp[i] == (at >= 0 && at < D ? v[at] : 0.0f));
    }
    const long long bytes = paged_attention_workspace_bytes(kv, b, 0, H);
    void* ws = nullptr;
    CUINFER_CHECK_HIP(hipMalloc(&ws, bytes + 16));
    paged_attention(kv, b, nullptr, 0, qo, H * D, out, H * D, H, 0.125f, ws, bytes);
    const auto o = down(out, H * D);
    for (int i = 0; i < H * D; ++i) EXPECT(o[i] == v[i % D]);  // one position: its value

    // two drafts: the first sure to be accepted, the second impossible; the third row is not reached
    std::vector<float> p(3 * 4, 0.0f);
    p[2] = 1.0f;      // row 0: token 2
    p[4 + 3] = 1.0f;  // row 1: token 3
    p[8 + 0] = 1.0f;
    int* ids = up<int>({2, 1, 0});
    int *tok = up<int>({9, 9, 9}), *acc = up<int>({9});
    float* u = up<float>({0.5f, 0.5f, 0.5f});
    const long long vb = verify_drafts_workspace_bytes(1, 4);
    void* vs = nullptr;
    CUINFER_CHECK_HIP(hipMalloc(&vs, vb));
    verify_drafts(up(p), 4, nullptr, 0, ids, u, u, up<int>({0, 3}), 1, 3, 4, tok, acc, vs, vb);
    EXPECT((down(tok, 3) == std::vector<int>{2, 3, -1}));
    EXPECT(down(acc, 1)[0] == 1);
    return 0;
}

int main(int argc, char** argv) {
    if (argc != 2) return 2;
    const int rc = std::strcmp(argv[1], "gpu") == 0 ? gpu() : cpu();
    if (rc == 0) std::printf("ok\n");
    return rc;
}
