// serving.h -- a batch over a paged cache, in the C++ layer: cri_qk_norm_rope, cri_paged_append,
// cri_paged_attention and cri_verify_drafts (cri.h says what each computes) with errors thrown as
// std::runtime_error.  No counterpart in the reference, which decodes one sequence over a contiguous
// cache.  Device pointers throughout; nothing is allocated and nothing synchronises.
#pragma once

#include <hip/hip_runtime_api.h>

#include "../cri.h"

namespace cuinfer {

using PagedKV = cri_paged_kv;
using PagedBatch = cri_paged_batch;
using HeadRotation = cri_rotation;

// q_out and k_out = the heads of q and k, normed and rotated at positions[m]; in place is fine.
void qk_norm_rope(const HeadRotation& rot, const float* q, int ldq, const float* k, int ldk, float* q_out, int ldq_out,
                  float* k_out, int ldk_out, const int* positions, int M, int n_heads, int n_kv_heads, int head_dim,
                  hipStream_t stream = 0);

// The batch's k rows, normed and rotated, and v rows go to their pages; q (may be null) to q_out.
void paged_append(const PagedKV& kv, const PagedBatch& batch, const HeadRotation& rot, const float* q, int ldq, float* q_out,
                  int ldq_out, int n_heads, const float* k, int ldk, const float* v, int ldv, hipStream_t stream = 0);

// Attention of the batch's rows, positions below prefix_len through prefix_pages, which all share.
// workspace: paged_attention_workspace_bytes of it.
void paged_attention(const PagedKV& kv, const PagedBatch& batch, const int* prefix_pages, int prefix_len, const float* q,
                     int ldq, float* out, int ldo, int n_heads, float scale, void* workspace, long long workspace_bytes,
                     hipStream_t stream = 0);
long long paged_attention_workspace_bytes(const PagedKV& kv, const PagedBatch& batch, int prefix_len, int n_heads);

// Drafted tokens accepted or replaced; draft may be null (sure drafts).  workspace:
// verify_drafts_workspace_bytes of it.
void verify_drafts(const float* target, long long ldt, const float* draft, long long ldd, const int* draft_ids,
                   const float* uniforms, const float* draws, const int* offsets, int n_seqs, int n_rows, int vocab,
                   int* out_ids, int* n_accepted, void* workspace, long long workspace_bytes, hipStream_t stream = 0);
long long verify_drafts_workspace_bytes(int n_seqs, int vocab);

}  // namespace cuinfer
