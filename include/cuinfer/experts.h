// experts.h -- a layer of experts in the C++ layer: cri_expert_pack, cri_expert_route, cri_expert_group, cri_expert_matmul,
// cri_expert_swiglu and cri_expert_combine (cri.h says what each computes) with errors thrown as std::runtime_error.  No
// counterpart in the reference, whose models have one FFN.  Device pointers throughout; nothing is allocated and nothing
// synchronises.
#pragma once

#include <hip/hip_runtime_api.h>

#include "../cri.h"

namespace cuinfer {

using ExpertWeights = cri_expert_weights;
using ExpertGroups = cri_expert_groups;
using ExpertRouter = cri_expert_router;

// GGUF blocks [n_experts, N, K] laid out once: expert_packed_bytes of device memory.  (Q4_0: element i in byte i / 2, as in
// matmul_q4_0, not upstream GGML's order.)
long long expert_packed_bytes(int format, int n_experts, int N, int K);
void pack_experts(int format, const void* src, int n_experts, int N, int K, void* packed, hipStream_t stream = 0);

// The router's logits to each token's experts, their weights and the groups; or given ids to the groups.
long long group_experts_workspace_bytes(const ExpertGroups& groups);
void route_experts(const ExpertRouter& router, const float* logits, int ldl, int* ids, float* weights,
                   const ExpertGroups& groups, void* workspace, long long workspace_bytes, hipStream_t stream = 0);
void group_experts(const int* ids, const ExpertGroups& groups, void* workspace, long long workspace_bytes,
                   hipStream_t stream = 0);

// Products of the grouped rows; x has a row per token or, with grouped, per grouped row.
long long expert_matmul_workspace_bytes(const ExpertWeights& w, const ExpertGroups& groups, bool grouped = false);
void expert_matmul(const ExpertWeights& w, const ExpertGroups& groups, const float* x, int ldx, bool grouped, float* out,
                   int ldo, void* workspace, long long workspace_bytes, hipStream_t stream = 0);
long long expert_swiglu_workspace_bytes(const ExpertWeights& gate, const ExpertGroups& groups);
void expert_swiglu(const ExpertWeights& gate, const ExpertWeights& up, const ExpertGroups& groups, const float* x, int ldx,
                   float* out, int ldo, void* workspace, long long workspace_bytes, hipStream_t stream = 0);

// The weighted sum of a token's experts' products, onto residual (may be null, or out).
long long expert_combine_workspace_bytes(const ExpertWeights& w, const ExpertGroups& groups);
void expert_combine(const ExpertWeights& w, const ExpertGroups& groups, const float* x, int ldx, const float* weights,
                    const float* residual, int ldr, float* out, int ldo, void* workspace, long long workspace_bytes,
                    hipStream_t stream = 0);

}  // namespace cuinfer
