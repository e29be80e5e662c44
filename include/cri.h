/*
 * cri.h -- C ABI of the MI355X (gfx950) fused dequant+matmul library.
 *
 * Every entry point takes device pointers owned by the caller, enqueues its
 * kernels on `stream` (0 = the null stream) and returns without
 * synchronising.  The library allocates no device memory and keeps no state
 * between calls, so calls are re-entrant on any stream.
 *
 * Return value: CRI_OK (0) on success, otherwise a negative cri_status; the
 * thread-local message from cri_last_error_string() says what was wrong.
 * Unlike the reference (which silently truncates K/32 and K/256), shapes are
 * validated before anything is launched.  Errors that happen while a kernel
 * executes surface at the caller's next synchronisation, as in the reference.
 *
 * Conventions (ref:include/cuinfer/kernels/matmul_quant.h:1-22):
 *   A : fp32 [M, K] row-major activations
 *   B : [N, K] weights in GGUF row order: row n is K/bs consecutive blocks
 *   C : fp32 [M, N] row-major output, fully overwritten (never accumulated)
 *   A, B and C must not overlap.
 */
#ifndef CRI_H
#define CRI_H

#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum cri_status {
    CRI_OK = 0,
    CRI_ERR_INVALID_ARGUMENT = -1, /* null pointer or negative dimension       */
    CRI_ERR_SHAPE = -2,            /* K not a multiple of the block size, etc. */
    CRI_ERR_ALIGNMENT = -3,        /* pointer misaligned for its element type  */
    CRI_ERR_LAUNCH = -4,           /* the HIP runtime rejected a launch        */
    CRI_ERR_UNSUPPORTED = -5,      /* format id unknown                        */
    CRI_ERR_FILE = -6              /* GGUF file missing, unreadable, malformed */
} cri_status;

/* Weight formats; the numbering is shared with cri_matmul()/cri_dequantize(). */
typedef enum cri_format {
    CRI_Q8_0 = 0,
    CRI_Q4_0 = 1,
    CRI_Q5_0 = 2,
    CRI_Q4_K = 3,
    CRI_Q6_K = 4,
    CRI_FP16 = 5,
    CRI_FP32 = 6, /* only for cri_embedding_rows, cri_gguf_tensor.format and cri_paged_kv.type */
    CRI_BF16 = 7  /* only for cri_paged_kv.type */
} cri_format;

/* ---- fused dequant + matmul: C[M,N] = A[M,K] * dequant(B[N,K])^T ---------- */

/* replaces cuinfer::matmul_q8_0, ref:include/cuinfer/kernels/matmul_quant.h:37 (K % 32 == 0) */
int cri_matmul_q8_0(const float* A, const void* B, float* C, int M, int N, int K, hipStream_t stream);
/* replaces cuinfer::matmul_q4_0, ref:include/cuinfer/kernels/matmul_quant.h:50 (K % 32 == 0) */
int cri_matmul_q4_0(const float* A, const void* B, float* C, int M, int N, int K, hipStream_t stream);
/* replaces cuinfer::matmul_q5_0, ref:include/cuinfer/kernels/matmul_quant.h:63 (K % 32 == 0) */
int cri_matmul_q5_0(const float* A, const void* B, float* C, int M, int N, int K, hipStream_t stream);
/* replaces cuinfer::matmul_q4_k, ref:include/cuinfer/kernels/matmul_quant.h:76 (K % 256 == 0) */
int cri_matmul_q4_k(const float* A, const void* B, float* C, int M, int N, int K, hipStream_t stream);
/* replaces cuinfer::matmul_q6_k, ref:include/cuinfer/kernels/matmul_quant.h:88 (K % 256 == 0) */
int cri_matmul_q6_k(const float* A, const void* B, float* C, int M, int N, int K, hipStream_t stream);
/* replaces cuinfer::matmul_fp16, ref:include/cuinfer/kernels/matmul_quant.h:104 (K % 32 == 0,
 * as the reference requires; B must be 2-byte aligned) */
int cri_matmul_fp16(const float* A, const void* B, float* C, int M, int N, int K, hipStream_t stream);
/* format-switched form of the six above; mirrors the switch of matmul_dispatch,
 * ref:src/model.cu:797-825 (FP32 weights are not part of this library) */
int cri_matmul(int format, const float* A, const void* B, float* C, int M, int N, int K, hipStream_t stream);
/* cri_matmul with a caller workspace (no counterpart in the reference, whose matmuls take none):
 * the products whose K cri_matmul splits over workgroups with fp32 atomics -- 9..16 rows, and
 * above 16 rows the prefill GEMM's shapes with few output tiles (K % 256 == 0, e.g.
 * 512 x 2048 x 8192) -- store the partial sums in the workspace instead and add them in split
 * order in a second launch, so C has the same bits on every call (and the prefill shapes skip
 * the atomics and the zero fill: 512 x 2048 x 8192 Q4_K 41.1 -> 37.3 us).  Some prefill shapes that
 * cri_matmul does not split (e.g. 2048 x 2048 x 8192 Q8_0) are faster split into a workspace on
 * larger tiles (132 -> 108 us), and then are.  Every other shape runs as cri_matmul: 1..8 rows and
 * unsplit products are deterministic there; above 16 rows with K % 256 != 0 the k range may still
 * be split with atomics.
 *
 * workspace: device memory, 16-byte aligned, cri_matmul_workspace_bytes(format, M, N, K) bytes; C
 * 16-byte aligned and N a multiple of 4.  For 2..16 rows and for the prefill shapes that cri_matmul
 * splits this is required (CRI_ERR_INVALID_ARGUMENT for no workspace or one too small,
 * CRI_ERR_ALIGNMENT).  For the prefill shapes that it does not split, a workspace that is missing,
 * smaller or not so aligned is no error: the call runs as cri_matmul, whose sums are in another
 * order.  So C's bits depend on the shape and on whether the advertised size and the alignment are
 * given, and on nothing else.  Calls sharing a workspace must be ordered on one stream. */
int cri_matmul_ws(int format, const float* A, const void* B, float* C, int M, int N, int K, void* workspace,
                  long long workspace_bytes, hipStream_t stream);
/* the most bytes of workspace cri_matmul_ws uses for this shape (0 when it uses none; a negative
 * cri_status for invalid arguments) */
long long cri_matmul_workspace_bytes(int format, int M, int N, int K);

/* ---- standalone dequant: dst[n_blocks * bs] = dequant(src) --------------- */

/* replaces cuinfer::dequantize_q8_0, ref:include/cuinfer/quantization.h:145 */
int cri_dequantize_q8_0(const void* src, float* dst, int n_blocks, hipStream_t stream);
/* replaces cuinfer::dequantize_q4_0, ref:include/cuinfer/quantization.h:152 */
int cri_dequantize_q4_0(const void* src, float* dst, int n_blocks, hipStream_t stream);
/* replaces cuinfer::dequantize_q5_0, ref:include/cuinfer/quantization.h:159 */
int cri_dequantize_q5_0(const void* src, float* dst, int n_blocks, hipStream_t stream);
/* replaces cuinfer::dequantize_q6_k, ref:include/cuinfer/quantization.h:166 */
int cri_dequantize_q6_k(const void* src, float* dst, int n_blocks, hipStream_t stream);
/* replaces cuinfer::dequantize_q4_k, ref:include/cuinfer/quantization.h:173 */
int cri_dequantize_q4_k(const void* src, float* dst, int n_blocks, hipStream_t stream);

/* ---- fp32 neighbours of the path ----------------------------------------- */

/* C[M,N] = A[M,K] * B[N,K]^T, all fp32; replaces cuinfer::matmul_transposed_b,
 * ref:include/cuinfer/embedding.h:136-137 (any K >= 1) */
int cri_matmul_transposed_b(const float* A, const float* B, float* C, int M, int N, int K,
                            hipStream_t stream);

/* C[h] = A[h] * B[h / (n_heads / n_kv_heads)] with A [n_heads, M, K],
 * B [n_kv_heads, K, N], C [n_heads, M, N], all fp32; replaces
 * cuinfer::batched_matmul_gqa, ref:include/cuinfer/attention.h:79-82
 * (n_heads % n_kv_heads == 0 is checked here; the reference checks it only in
 * AttentionBlock, ref:src/attention.cu:534-539) */
int cri_batched_matmul_gqa(const float* A, const float* B, float* C, int n_heads, int n_kv_heads,
                           int M, int N, int K, hipStream_t stream);

/* out[h, :] = softmax(scale * Q[h, :] . K[t, h / G, :] over t < kv_len) V[t, h / G, :]
 * for one query token, G = n_heads / n_kv_heads; Q [n_heads, head_dim],
 * K_cache / V_cache [>= kv_len, n_kv_heads, head_dim] (position stride
 * n_kv_heads * head_dim), out [n_heads, head_dim], all fp32; replaces
 * cuinfer::fused_decode_attention, ref:include/cuinfer/attention.h:161-167
 * (kernel ref:src/attention.cu:410-511).  Checked here: n_heads % n_kv_heads
 * == 0, kv_len >= 1 (the reference returns NaN for an empty cache) and
 * head_dim <= 256. */
int cri_fused_decode_attention(const float* Q, const float* K_cache, const float* V_cache, float* output,
                               int n_heads, int n_kv_heads, int head_dim, int kv_len, float scale,
                               hipStream_t stream);

/* Split form of cri_fused_decode_attention, with no counterpart in the
 * reference: for callers that can keep a device workspace (a decode loop or a
 * captured graph).  The cache positions are split over workgroups that each
 * read their K/V rows once for all the query heads of a KV head and write a
 * partial softmax state (max, sum, accumulator) per head to `workspace`; a
 * second kernel merges them.  The result equals cri_fused_decode_attention's
 * to fp32 rounding.  `workspace`: device memory, 16-byte aligned; the call
 * uses at most cri_fused_decode_attention_workspace_size() bytes of it (fewer
 * chunks when workspace_bytes is smaller; CRI_ERR_SHAPE below one record per
 * head).  Calls that share a workspace must be ordered on one stream.  Shapes
 * the split kernel does not take (head_dim > 128, head_dim % 4 != 0, Q/K/V not
 * 16-byte aligned) run cri_fused_decode_attention and leave the workspace
 * untouched. */
int cri_fused_decode_attention_ws(const float* Q, const float* K_cache, const float* V_cache, float* output,
                                  int n_heads, int n_kv_heads, int head_dim, int kv_len, float scale,
                                  void* workspace, long long workspace_bytes, hipStream_t stream);
/* No counterpart in the reference: cri_fused_decode_attention_ws without a
 * workspace argument and without any allocation, for callers that cannot call
 * hipMalloc (code under HIP graph capture, tight serving loops, harnesses that
 * forbid it).  The partial records live in a static device array of 1 MiB per
 * GPU (held until the process ends; every record is written before it is read,
 * so nothing needs clearing): fewer position chunks are used when a shape's
 * records would not fit, and CRI_ERR_SHAPE is returned when one record per head,
 * n_heads * (head_dim + 4) * 4 bytes, exceeds 1 MiB.  Needs 4 | head_dim <= 128
 * and 16-byte aligned Q, K_cache, V_cache (CRI_ERR_UNSUPPORTED otherwise).
 * Every call on one GPU shares that GPU's array: calls that overlap on one GPU
 * (different streams, or host threads) race and must be ordered by the caller.
 * The result equals cri_fused_decode_attention_ws's for the same shape. */
int cri_fused_decode_attention_noalloc(const float* Q, const float* K_cache, const float* V_cache, float* output,
                                       int n_heads, int n_kv_heads, int head_dim, int kv_len, float scale,
                                       hipStream_t stream);
/* Prompt attention over the [kv_len, n_kv_heads, head_dim] caches, the reference's prefill flow
 * (AttentionBlock::forward_from_qkv after the cache append, ref:src/attention.cu:809-871: Q K^T and
 * P V through batched_matmul_gqa around scale, causal mask and softmax), from 32 rows on at head_dim
 * 64 and 128 as one kernel without materialized scores: M query rows (already
 * rotated) at Q + m * ldq, [n_heads * head_dim] each, at positions pos .. pos + M - 1; row m
 * attends to cache positions [0, pos + m]; output row m at output + m * n_heads * head_dim.  The
 * caches must hold rows 0 .. pos + M - 1 (rows past them are never read into the products).
 * head_dim a multiple of 4 up to 128, ldq a multiple of 4; K_cache, V_cache, output and the
 * workspace 16-byte aligned; workspace_bytes at least
 * cri_prefill_attention_workspace_bytes(M, n_heads, n_kv_heads, head_dim, pos + M), which is the size
 * of the materialized flow's scores for every shape. */
int cri_prefill_attention(const float* Q, int ldq, const float* K_cache, const float* V_cache, float* output, int M,
                          int n_heads, int n_kv_heads, int head_dim, int pos, float scale, void* workspace,
                          long long workspace_bytes, hipStream_t stream);
long long cri_prefill_attention_workspace_bytes(int M, int n_heads, int n_kv_heads, int head_dim, int kv_len);
/* Workspace bytes cri_fused_decode_attention_ws uses for this shape (0 for an
 * empty problem; a negative cri_status for invalid arguments). */
long long cri_fused_decode_attention_workspace_size(int n_heads, int n_kv_heads, int head_dim, int kv_len);

/* ---- neighbour fusions: the activation computed while the matmul stages it -- */

/* C[M,N] = normed[M,K] * dequant(B[N,K])^T with v = hidden + residual and
 * normed = v * norm_weight * rsqrt(mean_k(v^2) + eps), the RMSNorm that feeds
 * q/k/v and gate/up (ref:src/kernels/elementwise.cu:463-513, called at
 * ref:src/model.cu:961-967 and :1012-1018 before matmul_dispatch).  v is also
 * written to hidden_out [M, K] when it is not null; hidden_out must not overlap
 * hidden or residual (checked).  residual may be null (plain RMSNorm).  No
 * counterpart in the reference: it replaces a rmsnorm_residual launch and the
 * normed buffer.  Decode batches only (1 <= M <= 16; CRI_ERR_UNSUPPORTED
 * above), every format; fp32 accuracy as cri_matmul at M <= 16. */
int cri_matmul_rmsnorm(int format, const float* hidden, const float* residual, const float* norm_weight,
                       float* hidden_out, const void* B, float* C, int M, int N, int K, float eps,
                       hipStream_t stream);
/* C[M,N] = (silu(gate) * up)[M,K] * dequant(B[N,K])^T, silu(x) = x / (1 + exp(-x)):
 * the FFN down projection of ref:src/model.cu:996-1002 with its silu and
 * multiply launches folded in.  gate and up rows are `ld` floats apart (ld >= K;
 * gate = buf, up = buf + inter, ld = 2 * inter reads a fused gate/up output).
 * No counterpart in the reference.  Decode batches only (1 <= M <= 16). */
int cri_matmul_swiglu(int format, const float* gate, const float* up, int ld, const void* B, float* C, int M,
                      int N, int K, hipStream_t stream);

/* Standalone forms, for batches the fused prologues do not take.
 * replaces cuinfer::rmsnorm_residual, ref:include/cuinfer/kernels/elementwise.h:107
 * (output may alias input; residual may be null) */
int cri_rmsnorm_residual(const float* input, const float* residual, const float* weight, float* output,
                         float* normed, int rows, int n, float eps, hipStream_t stream);
/* out = silu(gate) * up over n elements: cuinfer::silu then cuinfer::multiply,
 * ref:include/cuinfer/kernels/elementwise.h:23 and :75 (out may alias gate or up) */
int cri_silu_mul(const float* gate, const float* up, float* out, long long n, hipStream_t stream);

/* ---- GGUF files: the weights' on-disk format -------------------------------
 * A reader with the reference's parsing rules (ref:src/gguf_parser.cpp; the C++
 * class is cuinfer::GGUFParser in cuinfer/gguf_parser.h), for hosts that bind C.
 * The file is memory-mapped; names and strings returned stay valid until
 * cri_gguf_close.  A tensor's data lying past the end of the file is rejected at
 * open (CRI_ERR_FILE). */
typedef struct cri_gguf cri_gguf;
typedef struct cri_gguf_tensor {
    const char* name;
    int ggml_type;         /* GGML type tag (0 F32, 1 F16, 2 Q4_0, 6 Q5_0, 8 Q8_0, 12 Q4_K, 14 Q6_K, ...) */
    int format;            /* cri_format of the data, CRI_FP32, or -1 for types the matmuls do not take */
    int n_dims;
    long long dims[8];     /* dims[0] innermost: a [N, K] weight is {K, N} */
    long long n_elements;
    long long byte_size;   /* -1 for a GGML type this reader does not know */
    long long data_offset; /* bytes from the start of the file */
} cri_gguf_tensor;
typedef struct cri_gguf_model {
    char architecture[64]; /* general.architecture */
    unsigned context_length, embedding_length, block_count, head_count, head_count_kv, feed_forward_length,
        rope_dimension_count, vocab_size; /* bit i of `missing` set: field i (in this order) absent */
    float rope_freq_base;  /* default 10000 */
    float rms_norm_eps;    /* default 1e-5 */
    int tie_word_embeddings; /* 1 when there is no output.weight */
    unsigned missing;
} cri_gguf_model;
/* replaces cuinfer::GGUFParser::GGUFParser, ref:include/cuinfer/gguf_parser.h:165 */
int cri_gguf_open(const char* path, cri_gguf** out);
void cri_gguf_close(cri_gguf* file);
int cri_gguf_version(const cri_gguf* file);
long long cri_gguf_tensor_count(const cri_gguf* file);
long long cri_gguf_metadata_count(const cri_gguf* file);
/* index of the named tensor, or -1 (find_tensor, ref:include/cuinfer/gguf_parser.h:236) */
int cri_gguf_find_tensor(const cri_gguf* file, const char* name);
int cri_gguf_tensor_info(const cri_gguf* file, int index, cri_gguf_tensor* out);
/* host pointer into the mapping (tensor_data, ref:include/cuinfer/gguf_parser.h:240) */
const void* cri_gguf_tensor_data(const cri_gguf* file, int index);
/* GGUF value type tag of a metadata key, or -1 */
int cri_gguf_metadata_type(const cri_gguf* file, const char* key);
/* typed getters: CRI_ERR_SHAPE for a missing key or another type (get_*, ref:include/cuinfer/gguf_parser.h:197-201) */
int cri_gguf_get_u32(const cri_gguf* file, const char* key, unsigned* out);
int cri_gguf_get_i32(const cri_gguf* file, const char* key, int* out);
int cri_gguf_get_u64(const cri_gguf* file, const char* key, unsigned long long* out);
int cri_gguf_get_f32(const cri_gguf* file, const char* key, float* out);
int cri_gguf_get_string(const cri_gguf* file, const char* key, const char** out);
long long cri_gguf_get_array_length(const cri_gguf* file, const char* key);
/* the model helpers, ref:include/cuinfer/gguf_parser.h:208-230 */
int cri_gguf_model_params(const cri_gguf* file, cri_gguf_model* out);
/* the tensor's raw bytes to device memory; returns when the copy is done
 * (the upload of load_weight_quantized, ref:src/model.cu:406-411) */
int cri_gguf_upload(const cri_gguf* file, int index, void* device_dst, long long dst_bytes, hipStream_t stream);

/* out[i, :] = dequant(row ids[i] of table [vocab, dim]) in fp32, bit-identical to
 * dequantize + gather; ids outside [0, vocab) give zero rows.  format: a
 * cri_format or CRI_FP32.  Lets the token embedding stay in its file format
 * when the LM head reuses it (the reference dequantizes the tied table to
 * FP32, ref:src/model.cu:603); no counterpart in the reference. */
int cri_embedding_rows(int format, const void* table, const int* ids, float* out, int n_ids, int dim, int vocab,
                       hipStream_t stream);

/* ---- the decode step: TransformerModel::forward's layer loop ---------------
 * A decoder owns its weights (copied in), activation buffers, KV cache
 * [n_layers][max_seq_len, n_kv_heads, head_dim] and workspace, all allocated at
 * create; forward and replay allocate nothing.  The C++ class is
 * cuinfer::DecodeStep (cuinfer/decode_step.h).  It replaces the quantized path
 * of TransformerModel::forward, ref:src/model.cu:831-1039 (embedding, per layer
 * RMSNorm, q/k/v, RoPE, KV append, attention, o, residual + RMSNorm, gate/up,
 * SiLU * up, down, residual; final RMSNorm, LM head) and the greedy
 * argmax_sample, ref:src/embedding.cu:305-326.  Batch row m of a call at
 * position p attends to cache positions [0, p + m] (the reference's causal
 * mask; one token: its fused decode attention).  The position is kept in
 * device memory, so a captured step replays correctly token after token. */
typedef struct cri_decoder cri_decoder;
typedef struct cri_decoder_config {
    int n_layers, dim, n_heads, n_kv_heads, head_dim, ffn_dim, vocab_size, max_seq_len;
    int max_batch; /* tokens per call, 1..65535 (up to 16 use the fused norm prologues) */
    float rms_norm_eps, rope_theta;
} cri_decoder_config;
/* one layer's tensors; weights [N, K] in GGUF row order, in host or device memory
 * (copied at set time); norms fp32 [dim]; formats: cri_format, not CRI_FP32 */
typedef struct cri_decoder_layer {
    const float* attn_norm;
    const float* ffn_norm;
    int q_format, k_format, v_format, o_format, gate_format, up_format, down_format;
    const void *q, *k, *v, *o, *gate, *up, *down;
} cri_decoder_layer;
int cri_decoder_create(const cri_decoder_config* config, cri_decoder** out);
void cri_decoder_destroy(cri_decoder* dec);
int cri_decoder_set_layer(cri_decoder* dec, int layer, const cri_decoder_layer* weights);
/* token table [vocab, dim]: a cri_format or CRI_FP32 */
int cri_decoder_set_embedding(cri_decoder* dec, int format, const void* table);
/* final norm fp32 [dim] and LM head [vocab, dim]; format -1 ties the head to the token table */
int cri_decoder_set_output(cri_decoder* dec, const float* output_norm, int format, const void* lm_head);
/* M tokens (device int32 [M]) at positions position() .. +M-1 -> logits (device fp32 [M, vocab]);
 * next_ids (device int32 [M] or NULL) <- argmax of each logits row (ties: the smallest index).
 * CRI_ERR_SHAPE when position() + M would exceed max_seq_len. */
int cri_decoder_forward(cri_decoder* dec, const int* token_ids, int M, float* logits, int* next_ids,
                        hipStream_t stream);
/* A prompt as the reference's generate() consumes it (ref:src/model.cu:1063-1078, which runs
 * forward() and reads only the last row's logits): every layer runs on the M tokens (caches
 * appended, position advanced by M), the final RMSNorm, LM head and argmax for token M - 1 only:
 * logits (device fp32 [vocab]), next_id (device int32 [1] or NULL).  No counterpart in the
 * reference's API (its forward() always returns every row). */
int cri_decoder_prefill(cri_decoder* dec, const int* token_ids, int M, float* logits, int* next_id,
                        hipStream_t stream);
/* capture the same call as one HIP graph on a non-null stream (nothing runs), and replay it:
 * each replay is one more step of M tokens; next_ids == token_ids generates greedily */
/* cri_decoder_forward that also writes the residual stream entering each layer and the final
 * norm: hidden_taps (device fp32 [n_layers + 1, M, dim]) slice i = the hidden state layer i
 * reads (slice n_layers: the final RMSNorm's input).  Same kernels as cri_decoder_forward plus
 * one small kernel per slice; for checking a step layer by layer.  Has no counterpart in the
 * reference (its forward keeps no per-layer state). */
int cri_decoder_forward_taps(cri_decoder* dec, const int* token_ids, int M, float* logits, int* next_ids,
                             float* hidden_taps, hipStream_t stream);
/* any cri_decoder_set_* call discards a captured graph (replay then fails until the next capture) */
int cri_decoder_capture(cri_decoder* dec, const int* token_ids, int M, float* logits, int* next_ids,
                        hipStream_t stream);
int cri_decoder_replay(cri_decoder* dec, hipStream_t stream);
/* the sequence position (0 = empty cache); set with a kernel on `stream` */
int cri_decoder_set_position(cri_decoder* dec, int pos, hipStream_t stream);
int cri_decoder_position(const cri_decoder* dec);
/* the layer's K and V cache, [max_seq_len, n_kv_heads, head_dim] fp32 device memory */
int cri_decoder_kv_cache(cri_decoder* dec, int layer, float** k_cache, float** v_cache);
long long cri_decoder_weight_bytes(const cri_decoder* dec);
/* weight bytes one step of M tokens reads: every layer's matrices and norms, the final norm and
 * LM head, and M token-table rows (the whole table when the head is tied to it) */
long long cri_decoder_step_weight_bytes(const cri_decoder* dec, int M);

/* ---- serving a batch from a paged cache ------------------------------------
 * No counterpart in the reference, which decodes one sequence over a contiguous cache.  A layer of a
 * batched step is: the fused q/k/v product, cri_paged_append, cri_paged_attention, the o product; a
 * step that checks drafted tokens ends with cri_verify_drafts.  Activations are fp32, as everywhere
 * in this library; the cache is fp32, fp16 or bf16.
 *
 * All of these enqueue on `stream` without synchronising, allocate nothing and may be captured in a
 * HIP graph (what a descriptor points to is read when the kernels run, the descriptor itself and
 * every host number at the call).  Calls that share a workspace must be ordered on one stream.
 *
 * A pool of pages: page p holds the K rows of page_size positions at k + p * page_stride elements,
 * [page_size, n_kv_heads, head_dim], and the V rows likewise at v.  head_dim a multiple of 8, up to
 * 256; page_stride a multiple of 8 and at least page_size * n_kv_heads * head_dim; k and v 16-byte
 * aligned. */
typedef struct cri_paged_kv {
    void* k;
    void* v;
    long long page_stride; /* elements */
    int type;              /* CRI_FP32, CRI_FP16 or CRI_BF16 */
    int n_pages, page_size, n_kv_heads, head_dim;
} cri_paged_kv;
/* A ragged batch: sequence s has the rows offsets[s] .. offsets[s + 1] - 1 of q, k, v and the
 * outputs (n_s of them, 0 or more), and holds lens[s] positions, those rows' included: its i-th row
 * is at position lens[s] - n_s + i.  Position p lies in page pages[s * max_pages + p / page_size], at
 * p % page_size.  offsets must not decrease.  n_rows: rows that the buffers have; rows before
 * offsets[0] and from offsets[n_seqs] on (a padded batch) are neither read nor written.
 * max_pages * page_size at most 2^30. */
typedef struct cri_paged_batch {
    const int* offsets; /* device [n_seqs + 1] */
    const int* lens;    /* device [n_seqs] */
    const int* pages;   /* device [n_seqs, max_pages] */
    int n_seqs, n_rows, max_pages;
} cri_paged_batch;
/* Norms and rotation of query and key heads.  A head x becomes x * w / sqrt(mean(x^2) + eps) with w
 * the norm weights [head_dim] (null: x as it is), then each pair (a, b) of its first rot_dim elements
 * becomes (a cos - b sin, b cos + a sin) at the angle p * theta^(-2 i / rot_dim) for position p and
 * pair i; elements from rot_dim on are not turned.  rot_dim a multiple of 8, up to head_dim (0: no
 * rotation).  Angles are computed in 64 bits. */
typedef enum cri_rope_pairs {
    CRI_ROPE_ADJACENT = 0, /* pair i: elements 2 i and 2 i + 1, the decoder's layout */
    CRI_ROPE_HALVES = 1    /* pair i: elements i and i + rot_dim / 2 */
} cri_rope_pairs;
typedef struct cri_rotation {
    const float* q_norm; /* device, or null */
    const float* k_norm;
    float eps;
    float theta;
    int rot_dim;
    int pairs; /* cri_rope_pairs */
} cri_rotation;

/* q_out = the heads of q [M, n_heads, head_dim], k_out = the heads of k [M, n_kv_heads, head_dim],
 * normed and rotated, row m at position positions[m] (device int32).  Rows are ldq, ldk, ldq_out and
 * ldk_out floats apart (at least their heads' width).  q_out may be q with ldq_out == ldq, k_out k
 * with ldk_out == ldk; no other overlap of an output with another buffer (outputs of columns of one
 * row are fine; positions and norm weights count as buffers).  q or k may be left out with 0 heads.  Pointers 4-byte
 * aligned. */
int cri_qk_norm_rope(const cri_rotation* rot, const float* q, int ldq, const float* k, int ldk, float* q_out, int ldq_out,
                     float* k_out, int ldk_out, const int* positions, int M, int n_heads, int n_kv_heads, int head_dim,
                     hipStream_t stream);
/* The batch's k rows, normed and rotated at their positions, and v rows as they are, go to their
 * pages, rounded to the cache's type (to nearest even); with q not null, its n_heads heads go to
 * q_out, normed and rotated, as by cri_qk_norm_rope.  A row whose position has no page (below 0,
 * past the table's max_pages, a page number outside the pool) is left out: its page and q_out row
 * stay as they were.  Pages that are written must belong to one sequence.  q_out may be q with
 * ldq_out == ldq; no other overlap of q_out or the pool with another buffer, none of a page of k with one of v (pages of
 * the one between those of the other are fine). */
int cri_paged_append(const cri_paged_kv* kv, const cri_paged_batch* batch, const cri_rotation* rot, const float* q, int ldq,
                     float* q_out, int ldq_out, int n_heads, const float* k, int ldk, const float* v, int ldv,
                     hipStream_t stream);
/* out[row, h] = sum_j softmax_j(scale q[row, h] . k[j, h / G]) v[j, h / G] over the positions j in
 * [0, p] of the row's sequence, p the row's position, G = n_heads / n_kv_heads; one row per sequence
 * is a decode step, more are drafted tokens or a prompt's piece.  Positions j < prefix_len are read
 * through prefix_pages (device [ceil(prefix_len / page_size)]) instead of the sequence's own table:
 * a prefix that all sequences share, whose K and V are read once for the batch (its last page may
 * be partly filled; the sequences' own positions start at prefix_len of their own tables).
 * prefix_len 0: every position through its sequence's table.  A row at a position below 0 (a
 * negative lens counts as 0) sees nothing and gets zeros; positions past the table (max_pages *
 * page_size) are not seen.  Nothing behind a row's last position reaches it, whatever its pages hold
 * there; a NaN, or a value that is infinite, makes the rows that see it not finite; an infinite key does, or, where all
 * its products are -infinity, has no weight (a row that sees nothing else then gets zeros).  Table entries of
 * positions that rows see must be inside the pool (others give unspecified numbers in their
 * sequence's rows).
 *
 * q rows are ldq floats apart, out rows ldo; out must not overlap q or the pool.  n_heads a multiple
 * of n_kv_heads; n_rows * n_heads at most 2^24; scale finite.  q, out 4-byte aligned, workspace
 * 16-byte, cri_paged_attention_workspace_bytes of it (for the same kv, batch and prefix_len; only
 * their host numbers count, so one workspace serves every step with the same n_seqs, n_rows and
 * max_pages).  It holds head_dim + 4 floats per row, head and chunk of positions, up to 1 GiB; where two of those for every
 * row and head are more, as many (max_pages * page_size counts as the sequences' length: a table much wider than the
 * sequences costs records and time).  out and the workspace overlap no other buffer.  Sums, maxima and products are good to fp32 for every cache
 * type, in an order fixed by the host numbers and lens (fp16, whose probabilities are taken in two parts: within 2^-18 of a
 * head's largest element in its row, whatever the values; rows that would not be are multiplied in fp32, which takes longer). */
int cri_paged_attention(const cri_paged_kv* kv, const cri_paged_batch* batch, const int* prefix_pages, int prefix_len,
                        const float* q, int ldq, float* out, int ldo, int n_heads, float scale, void* workspace,
                        long long workspace_bytes, hipStream_t stream);
long long cri_paged_attention_workspace_bytes(const cri_paged_kv* kv, const cri_paged_batch* batch, int prefix_len,
                                              int n_heads);
/* Drafted tokens checked by rejection sampling.  Sequence s has the rows offsets[s] ..
 * offsets[s + 1] - 1 (n_s of them) of target (probabilities of the token that follows each row's
 * token, [n_rows, vocab], rows ldt floats apart), draft (the draft's probabilities, rows ldd apart;
 * null: the draft was sure of its tokens), draft_ids, uniforms and draws ([n_rows], random numbers in
 * [0, 1)).  Row j < n_s - 1 holds the drafted token that follows it; the last row's draft and
 * draft_ids are not read.  Draft j is accepted when uniforms[j] * draft[j][x] < target[j][x], x =
 * draft_ids[j] (a token outside [0, vocab) never is).  The first that is not is replaced by a token
 * drawn from max(target - draft, 0) of its row (of target where that leaves nothing; a sure draft:
 * target without x); with all accepted one more is drawn from the last row's target.  Drawing takes
 * the smallest token whose running sum of weights exceeds draws[that row] times their total (the last
 * token with any weight where rounding or the number leaves none; -1 where no token has weight).
 * The tokens follow the target's distribution when draws are independent of uniforms: a row's number
 * that has decided about its draft must not draw its replacement too.
 * out_ids [n_rows]: the accepted drafts, the drawn token, -1 in the sequence's remaining rows;
 * n_accepted [n_seqs].  Rows outside [offsets[0], offsets[n_seqs]) are neither read nor written, a
 * sequence of no rows gets n_accepted 0.  A target probability that is NaN or negative counts as
 * zero; where a draft's is NaN its token is not accepted and has no weight.  Comparisons and sums
 * are in 64 bits and in a fixed order.
 * out_ids, n_accepted and the workspace overlap neither each other nor an input.  workspace: 8-byte aligned, cri_verify_drafts_workspace_bytes. */
int cri_verify_drafts(const float* target, long long ldt, const float* draft, long long ldd, const int* draft_ids,
                      const float* uniforms, const float* draws, const int* offsets, int n_seqs, int n_rows,
                      int vocab, int* out_ids, int* n_accepted, void* workspace, long long workspace_bytes,
                      hipStream_t stream);
long long cri_verify_drafts_workspace_bytes(int n_seqs, int vocab);

/* ---- a layer of experts ------------------------------------------------------
 * No counterpart in the reference, whose models have one FFN.  The FFN of such a layer is: the router's product (cri_matmul or
 * cri_matmul_transposed_b: [E, dim] weights), cri_expert_route, cri_expert_swiglu, cri_expert_combine; cri_expert_matmul is for
 * other activations.  Which rows meet which expert stays on the device: nothing synchronises, host numbers alone decide launches
 * and workspaces, and a call may be captured in a HIP graph and replayed with other logits.  Results have the same bits at every
 * call with the same sizes and contents.  Calls that share a workspace must be ordered on one stream: if two run at once, both
 * results are unspecified, but nothing is read or written outside of their buffers.
 *
 * A matrix per expert, [n_experts, N, K] in GGUF blocks (ffn_gate_exps and the like), laid out once by cri_expert_pack: data
 * is 16-byte aligned, cri_expert_packed_bytes long.  K a multiple of 32 (Q4_K, Q6_K: 256), at least one block; up to 1024
 * experts. */
typedef struct cri_expert_weights {
    const void* data;
    int format; /* cri_format */
    int n_experts, N, K;
} cri_expert_weights;
long long cri_expert_packed_bytes(int format, int n_experts, int N, int K);
/* packed = the blocks at src (raw GGUF bytes, any alignment) in the products' order: the same bits, padded to 32 rows and 256
 * values (Q4_K 3% larger for its unpacked 6-bit scales).  src is not needed afterwards.  No overlap.  Q4_0 blocks have the element
 * order of cri_matmul_q4_0 (element i in byte i / 2); upstream GGML's files have another one (elements i and i + 16 in byte i), which
 * cannot be told apart here and has to be reordered first. */
int cri_expert_pack(int format, const void* src, int n_experts, int N, int K, void* packed, hipStream_t stream);
/* The pairs (token t, choice j), pair t * top_k + j, grouped by expert: the grouped rows of expert e are offsets[e] ..
 * offsets[e + 1] - 1, in the order of their pairs; rows[r] is the pair of grouped row r (-1 from offsets[n_experts] on),
 * slots[p] the grouped row of pair p (-1: it has no expert).  Written by cri_expert_route or cri_expert_group, read by the
 * products, which take entries that do not fit (no sorted offsets, a pair or row out of range) without reading or writing out
 * of bounds, the results being unspecified then.  top_k 1 .. 64 and at most n_experts, n_tokens * top_k at most 2^23. */
typedef struct cri_expert_groups {
    int* offsets; /* device [n_experts + 1] */
    int* rows;    /* device [n_tokens * top_k] */
    int* slots;   /* device [n_tokens * top_k] */
    int n_tokens, top_k, n_experts;
} cri_expert_groups;
typedef enum cri_expert_scoring { CRI_SCORE_SOFTMAX = 0, CRI_SCORE_SIGMOID = 1 } cri_expert_scoring;
typedef struct cri_expert_router {
    const float* bias; /* device [n_experts], added to the scores for the choice alone; or null */
    float scale;       /* of the weights */
    int scoring;       /* cri_expert_scoring */
    int normalize;     /* weights divided by their token's sum */
} cri_expert_router;
/* logits [n_tokens, n_experts], rows ldl floats apart -> ids and weights [n_tokens, top_k] and the groups.  A token's scores are
 * the softmax or the sigmoid of its logits; its top_k experts are those of the largest score plus bias (without a bias: of the
 * largest logit), in that order, the lowest number first where they are equal; their weights are the scores (without the
 * bias), divided by their sum with normalize (a sum of 0 leaves them 0), times scale.  An expert whose logit is -infinity or NaN (or whose bias makes its sum
 * so) is never chosen: a token left with fewer experts than top_k has id -1 and weight 0 in the choices behind, so a row of
 * -infinity (a padded batch's) causes no work.  Without a bias the order is exactly the logits'.  With one, score plus bias is
 * computed in 64 bits: sums that differ by less than about 2^-51 of themselves may count as equal or come in either order (the
 * sigmoids of 40 and 50 under one bias are equal, and so are scores of e^-50 and e^-49 beside a bias of 0.1).  workspace: 4-byte
 * aligned, cri_expert_group_workspace_bytes. */
int cri_expert_route(const cri_expert_router* router, const float* logits, int ldl, int* ids, float* weights,
                     const cri_expert_groups* groups, void* workspace, long long workspace_bytes, hipStream_t stream);
/* the groups of given ids [n_tokens, top_k]; ids outside [0, n_experts) are pairs without an expert (another GPU's, say), and a
 * token may name an expert twice */
int cri_expert_group(const int* ids, const cri_expert_groups* groups, void* workspace, long long workspace_bytes,
                     hipStream_t stream);
long long cri_expert_group_workspace_bytes(const cri_expert_groups* groups);
/* out[r, :] = x[row(r), :] W[e]^T for the grouped rows r of every expert e; row(r) is rows[r] / top_k (x: [n_tokens, K], a row
 * per token) or, with grouped, r (x: [n_tokens * top_k, K] in grouped order).  out [n_tokens * top_k, N]; its rows from
 * offsets[n_experts] on stay as they were.  Rows ldx and ldo floats apart, 4-byte aligned.  fp32 results: weights are exact,
 * activations have 22 bits of their row's (256 values' of their row's) largest magnitude, whatever that is (below 2^-126 results
 * have fp32's own step of 2^-149); a row that is not finite makes its own results not finite.  FP16 weights below 2^-14 (its subnormals) lose bits in the matrix units: a matrix of nothing else is
 * good to 1e-6 at weights of 2^-19, to 1e-5 at 2^-23.  out and the workspace (16-byte aligned) overlap no other buffer. */
int cri_expert_matmul(const cri_expert_weights* w, const cri_expert_groups* groups, const float* x, int ldx, int grouped,
                      float* out, int ldo, void* workspace, long long workspace_bytes, hipStream_t stream);
long long cri_expert_matmul_workspace_bytes(const cri_expert_weights* w, const cri_expert_groups* groups, int grouped);
/* out[r, :] = silu(x[row(r), :] gate[e]^T) * (x[row(r), :] up[e]^T), a row of x per token; gate and up have the same format and
 * sizes.  Else as cri_expert_matmul. */
int cri_expert_swiglu(const cri_expert_weights* gate, const cri_expert_weights* up, const cri_expert_groups* groups,
                      const float* x, int ldx, float* out, int ldo, void* workspace, long long workspace_bytes,
                      hipStream_t stream);
long long cri_expert_swiglu_workspace_bytes(const cri_expert_weights* gate, const cri_expert_groups* groups);
/* out[t, :] = residual[t, :] + sum_j weights[t, j] (x[slots[t top_k + j], :] W[e]^T), x [n_tokens * top_k, K] in grouped order (what
 * cri_expert_swiglu leaves), weights [n_tokens, top_k]; choices without an expert are left out.  residual (rows ldr apart) may be
 * null, or out itself with ldr == ldo; no other overlap of out or the workspace (16-byte aligned).  out [n_tokens, N] is written
 * whole. */
int cri_expert_combine(const cri_expert_weights* w, const cri_expert_groups* groups, const float* x, int ldx,
                       const float* weights, const float* residual, int ldr, float* out, int ldo, void* workspace,
                       long long workspace_bytes, hipStream_t stream);
long long cri_expert_combine_workspace_bytes(const cri_expert_weights* w, const cri_expert_groups* groups);
/* How a call of these sizes multiplies, which the numbers alone decide: plan[0] the rows of a tile (1, 4, 8: few rows, converted by
 * the workgroup that multiplies them; 16, 32, 64: many; 0: the combination in one launch), plan[1] the parts that K is shared in,
 * plan[2] the waves of a workgroup; 0, 0, 0 where there is nothing to do.  w: gate's for CRI_EXPERT_SWIGLU.  For tests and
 * measurements; touches no GPU. */
typedef enum cri_expert_op { CRI_EXPERT_MATMUL = 0, CRI_EXPERT_SWIGLU = 1, CRI_EXPERT_COMBINE = 2 } cri_expert_op;
int cri_expert_plan(const cri_expert_weights* w, const cri_expert_groups* groups, int op, int* plan);

/* ---- diagnostics ---------------------------------------------------------- */

/* Reads n_bytes (a multiple of 16) at src (16-byte aligned) once with 16-byte
 * loads and nothing else: the achievable streaming-read bandwidth that the
 * GEMV rooflines are read against.  sink (one device word) is written only if
 * the XOR of the words one thread reads (four 16-byte chunks, 4096 bytes apart)
 * equals 0x9E3779B9.  A measurement aid with no counterpart in the reference. */
int cri_stream_read(const void* src, long long n_bytes, unsigned* sink, hipStream_t stream);

/* cri_stream_read with the launch shape as parameters, for sweeping it:
 * loads_per_thread (1, 2, 4, 8 or 16) 16-byte loads in flight per thread;
 * grid_blocks 0 covers the buffer once with one pass per thread, otherwise
 * that many workgroups of 256 threads stride over it.  cri_stream_read is
 * (4, 0).  A measurement aid with no counterpart in the reference. */
int cri_stream_read_ex(const void* src, long long n_bytes, unsigned* sink, int loads_per_thread, int grid_blocks,
                       hipStream_t stream);

/* Writes the GPU's constant 100 MHz clock (wall_clock64) to *dst (device, 8-byte
 * aligned) from a one-wave kernel on `stream`: timestamps between the kernels of
 * a captured graph, where events cannot be recorded.  A measurement aid with no
 * counterpart in the reference. */
int cri_timestamp(unsigned long long* dst, hipStream_t stream);

/* Message for the last non-zero status returned on this thread ("" if none). */
const char* cri_last_error_string(void);
/* Bytes per block / elements per block of a format (0 if unknown). */
int cri_block_bytes(int format);
int cri_block_elems(int format);
/* Library ABI version (major * 10000 + minor * 100 + patch). */
int cri_version(void);

#ifdef __cplusplus
}
#endif
#endif /* CRI_H */
