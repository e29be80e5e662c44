// experts_file_check.cpp -- the matrices of a layer of experts from a GGUF file (its path the second argument): `cpu` finds the 3-D
// tensor that load_weight_quantized refuses, `gpu` uploads, lays out and multiplies it.  The file holds blk.0.ffn_gate_exps.weight, FP16
// {K 32, N 3, E 2}, expert e's row n being 4 e + n + 1 at k = n and 0 elsewhere.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstring>
#include <stdexcept>
#include <vector>

#include "cuinfer/experts.h"
#include "cuinfer/gguf_parser.h"
#include "cuinfer/hip_utils.h"
#include "cuinfer/weights.h"

using namespace cuinfer;

#define EXPECT(x)                                       \
    do {                                                \
        if (!(x)) {                                     \
            std::printf("line %d: %s\n", __LINE__, #x); \
            return 1;                                   \
        }                                               \
    } while (0)

template <class T>
T* room(size_t n, const T* from = nullptr) {
    T* d = nullptr;
    CUINFER_CHECK_HIP(hipMalloc(&d, n * sizeof(T) + 16));
    if (from) CUINFER_CHECK_HIP(hipMemcpy(d, from, n * sizeof(T), hipMemcpyHostToDevice));
    return d;
}

int run(const char* path, bool gpu) {
    const GGUFParser parser(path);
    const char* name = "blk.0.ffn_gate_exps.weight";
    const GGUFTensorInfo* info = parser.find_tensor(name);
    EXPECT(info && info->dimensions == (std::vector<uint64_t>{32, 3, 2}));
    EXPECT(ggml_type_to_weight_format(info->type) == WeightFormat::FP16 && info->byte_size() == 2 * 3 * 32 * 2);
    bool refused = false;
    try {
        WeightFormat f;
        load_weight_quantized(parser, name, f);
    } catch (const std::runtime_error& e) {
        refused = std::strstr(e.what(), "2-D") != nullptr;
    }
    EXPECT(refused);
    if (!gpu) return 0;
    const int K = 32, N = 3, E = 2, M = 2;
    void* raw = room<char>(info->byte_size(), static_cast<const char*>(parser.tensor_data(*info)));
    void* packed = room<char>(expert_packed_bytes(CRI_FP16, E, N, K));
    pack_experts(CRI_FP16, raw, E, N, K, packed);
    const ExpertWeights w{packed, CRI_FP16, E, N, K};
    const ExpertGroups g{room<int>(E + 1), room<int>(M), room<int>(M), M, 1, E};
    const int ids[] = {1, 0};
    group_experts(room<int>(M, ids), g, nullptr, 0);
    std::vector<float> x(M * K, 1.0f), out(M * N);
    float* d = room<float>(M * N);
    const long long bytes = expert_matmul_workspace_bytes(w, g);
    expert_matmul(w, g, room<float>(M * K, x.data()), K, false, d, N, room<char>(bytes), bytes);
    CUINFER_CHECK_HIP(hipDeviceSynchronize());
    CUINFER_CHECK_HIP(hipMemcpy(out.data(), d, M * N * sizeof(float), hipMemcpyDeviceToHost));
    EXPECT((out == std::vector<float>{1, 2, 3, 5, 6, 7}));  // expert 0's row, then expert 1's
    return 0;
}

int main(int argc, char** argv) {
    if (argc != 3) return 2;
    const int rc = run(argv[2], std::strcmp(argv[1], "gpu") == 0);
    if (rc == 0) std::printf("ok\n");
    return rc;
}
