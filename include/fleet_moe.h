/*
 * fleet_moe.h -- C ABI of the MI355X (gfx950) batch-1 MoE decode path for
 * DeepSeek-V2-Lite: router + greedy top-k, routed SwiGLU experts, the fused
 * shared expert, the weighted combine, and the multi-token grouped product.
 *
 * Conventions (match the reference launcher's, src/host/fleet_launch.hip:55-63,
 * 612-644, and its task-body ABI, src/kernels/fleet_kernel.hip:1057-1078):
 *   - every entry point returns 0 on success, a hipError_t value when a HIP
 *     call fails, or a FLEET_MOE_ERR_* code (>= 10000) for a rejected argument;
 *   - nothing here allocates: the caller owns every buffer (weights, inputs,
 *     outputs, workspace) as device memory, and passes plain device pointers;
 *   - work is enqueued on `stream` and is asynchronous; inputs are read-only;
 *   - a workspace must be zero-filled once before its first use and may then
 *     be reused by any number of calls that are ordered on one stream; two
 *     calls that overlap in time must not share a workspace;
 *   - weights use the reference's packed layout (src/host/pack_weights.py:
 *     41-54, 71-83, 125-146): bf16 bit patterns (uint16_t), experts as
 *     n_routed blocks of `expert_stride` elements [gate/up interleaved
 *     (2*I rows of H) | down (H rows of I)], the merged shared expert as
 *     [gate/up interleaved (2*SI rows of H) | down (H rows of SI)], SI =
 *     n_shared * I. Tensor bases must be 16-byte aligned (the packer aligns
 *     every tensor to 256 bytes).
 * The kernels are built for the DeepSeek-V2-Lite shape (hidden 2048,
 * moe_inter 1408, 64 routed experts, top-6, 2 shared experts); other shapes
 * are rejected with FLEET_MOE_ERR_DIMS.
 */
#ifndef FLEET_MOE_H
#define FLEET_MOE_H

#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FLEET_MOE_ERR_DIMS 10001      /* shape other than the supported one  */
#define FLEET_MOE_ERR_ARG 10002       /* null or misaligned pointer, bad count */
#define FLEET_MOE_ERR_WORKSPACE 10003 /* workspace smaller than required      */
#define FLEET_MOE_ERR_DEVICE 10004    /* device is not gfx950 / too few CUs   */
#define FLEET_MOE_ERR_CAPACITY 10005  /* more tokens than the static scratch holds */
#define FLEET_MOE_ERR_CAPTURE 10006   /* first call on a device made under graph capture */

/* Model scalars, the MoE subset of ModelDims (src/runtime/fleet_types.h:33-39)
 * and of the packed manifest's scalars (src/host/pack_weights.py:153-184). */
typedef struct fleet_moe_dims {
    int32_t hidden;        /* 2048 */
    int32_t moe_inter;     /* 1408 */
    int32_t n_routed;      /* 64   */
    int32_t n_shared;      /* 2: the shared expert has n_shared*moe_inter rows */
    int32_t top_k;         /* 6    */
    float routed_scaling;  /* 1.0  */
    float rms_eps;         /* 1e-6 */
} fleet_moe_dims;

/* One MoE layer's weights: the per-layer pointer tables of Weights
 * (src/runtime/fleet_types.h:44-59: layer_norm_post, layer_router,
 * layer_experts, layer_shared, expert_stride). */
typedef struct fleet_moe_layer {
    const uint16_t* norm;     /* post-attention RMSNorm weight bf16[hidden]; NULL = unit */
    const uint16_t* router;   /* bf16[n_routed][hidden] ("L{i}.router") */
    const uint16_t* experts;  /* n_routed blocks ("L{i}.experts") */
    int64_t expert_stride;    /* elements between experts: 3*hidden*moe_inter */
    const uint16_t* shared;   /* merged shared expert block ("L{i}.shared") */
} fleet_moe_layer;

/* Router logits and greedy top-k for n_tokens rows of x_norm.
 * Replaces the router GEMV of task_norm_router (src/kernels/fleet_kernel.hip:
 * 433-435) and select_experts_from (:469-494); semantics of
 * src/host/reference_decode.py:271-278 and HF MoEGate.forward
 * (reference/modeling_deepseek.py:420-467):
 *   logits = W_router . x_norm (fp32; evaluated exactly and rounded once),
 *   p = softmax(logits + logit_bias), ids = the top_k largest p in decreasing
 *   order, ties to the lowest index, weights = p[ids] * routed_scaling.
 * x_norm: fp32[n_tokens][hidden] (bf16-valued); logit_bias: fp32[n_routed]
 * or NULL; logits: fp32[n_tokens][n_routed] or NULL; ids: int32[n_tokens]
 * [top_k]; weights: fp32[n_tokens][top_k]. 1 <= n_tokens <= 65535. */
int fleet_moe_router_topk(const uint16_t* router, const float* x_norm, int32_t n_tokens,
                          const float* logit_bias, float* logits, int32_t* ids,
                          float* weights, const fleet_moe_dims* dims, hipStream_t stream);

/* The same, and x_bf16 (bf16[n_tokens][hidden], 16-byte aligned) = x_norm rounded
 * to bf16: the grouped step's input, from the launch that has x_norm at hand. */
int fleet_moe_router_topk_bf16(const uint16_t* router, const float* x_norm, int32_t n_tokens,
                               const float* logit_bias, float* logits, int32_t* ids,
                               float* weights, uint16_t* x_bf16, const fleet_moe_dims* dims,
                               hipStream_t stream);

/* The residual fold of the NORM_ROUTER prologue (stage_residual_f32,
 * src/kernels/fleet_kernel.hip:107-144, called at :405-425): the post-
 * attention residual x[1] = bf16(x[0] + bf16(p_0 + ... + p_{n-1})) from the
 * layer input and o_proj's n K-split fp32 partials (Activations.oproj_partial,
 * [n][hidden], n = 8 in the reference), the partials added in fp32 in index
 * order. fleet_moe_layer_decode takes that x[1] as its input; a graph whose
 * o_proj writes x[1] itself (OPROJ_ROW_SPLIT) needs no fold.
 * x, x_out: fp32[hidden] (may be equal); 1 <= n_partials <= 64. */
int fleet_moe_residual_fold(const float* x, const float* partials, int32_t n_partials,
                            float* x_out, const fleet_moe_dims* dims, hipStream_t stream);

/* Workspace bytes fleet_moe_layer_decode needs. */
size_t fleet_moe_layer_workspace_bytes(const fleet_moe_dims* dims);

/* One batch-1 MoE layer: x_out = bf16(x + moe(rms_norm(x))).
 * Replaces, for one token, the NORM_ROUTER (kind 4), EXPERT_GATE_UP (5) and
 * EXPERT_DOWN (6) task bodies and the expert-partial fold (src/kernels/
 * fleet_kernel.hip:398-456, 469-500, 826-889, 146-201; src/kernels/expert.h:
 * 45-116); semantics of src/host/reference_decode.py:294-302 (rms_norm, moe,
 * residual add) with the selection rule above.
 * x: fp32[hidden]; x_out: fp32[hidden] (may equal x); moe_out: bf16[hidden]
 * (the MoE output before the residual add) or NULL; ids: int32[top_k] or
 * NULL; weights: fp32[top_k] or NULL. One launch of 256 workgroups (one per
 * CU) that hand data to each other through the workspace, so all of them must
 * be resident at once: the entry point checks once per device that the device
 * has >= 256 CUs and that one workgroup of the kernel fits on a CU
 * (FLEET_MOE_ERR_DEVICE otherwise); a wait that still runs past its bound
 * (other work holding CUs) sets FLEET_MOE_ABORT_UNIT_WAIT or _ROUTER_WAIT. */
int fleet_moe_layer_decode(const fleet_moe_layer* layer, const float* x, float* x_out,
                           uint16_t* moe_out, int32_t* ids, float* weights,
                           void* workspace, size_t workspace_bytes,
                           const fleet_moe_dims* dims, hipStream_t stream);

/* Workspace bytes fleet_moe_dense_decode needs (dense_inter = 10944). */
size_t fleet_moe_dense_workspace_bytes(const fleet_moe_dims* dims, int32_t dense_inter);

/* Batch-1 dense SwiGLU layer (DeepSeek-V2-Lite layer 0, first_k_dense = 1):
 * x_out = bf16(x + mlp(rms_norm(x))), mlp(v) = down(bf16(bf16(silu(bf16(gate v)))
 * * bf16(up v))). Replaces the layer's NORM_ROUTER prologue and the
 * DENSE_GATE_UP (8) / DENSE_DOWN (9) task bodies (src/kernels/fleet_kernel.hip:
 * 891-903; src/host/taskgraph.py:444-474); semantics of src/host/
 * reference_decode.py:290-302 (dense_mlp, residual add).
 * norm: post-attention RMSNorm weight bf16[hidden] or NULL (unit); w: the
 * packed "L0.dense" block, [2*dense_inter][hidden] gate/up interleaved then
 * [hidden][dense_inter] down (src/host/pack_weights.py:143-146); x, x_out:
 * fp32[hidden] (may be equal); mlp_out: bf16[hidden] or NULL. One launch over
 * every CU. */
int fleet_moe_dense_decode(const uint16_t* norm, const uint16_t* w, int32_t dense_inter,
                           const float* x, float* x_out, uint16_t* mlp_out, void* workspace,
                           size_t workspace_bytes, const fleet_moe_dims* dims,
                           hipStream_t stream);

/* Workspace bytes fleet_moe_grouped needs for up to max_tokens tokens. */
size_t fleet_moe_grouped_workspace_bytes(const fleet_moe_dims* dims, int32_t max_tokens);

/* Multi-token grouped-expert product for one layer (no reference kernel; HF
 * DeepseekV2MoE.forward + moe_infer, reference/modeling_deepseek.py:568-664):
 * tokens are grouped by expert, every selected expert runs its SwiGLU over
 * its tokens (VALU GEMV for an expert holding <= 8 tokens, bf16 MFMA above
 * that), and out[t] = bf16(bf16(sum_k bf16(w[t][k] * E_{ids[t][k]}(x[t]))) +
 * shared(x[t])), the per-token combine of src/host/reference_decode.py:
 * 280-287, so grouped(T) equals T batch-1 MoE outputs up to fp32 summation
 * order. One launch over every CU (256 workgroups resident at once) for
 * n_tokens <= 8, two (gate/up, then down + combine) above that.
 * x_norm: bf16[n_tokens][hidden]; ids: int32[n_tokens][top_k] (each in
 * [0, n_routed), distinct per token; an id outside that range is clamped into
 * it and raises FLEET_MOE_ABORT_BAD_ID); weights: fp32[n_tokens][top_k];
 * out: bf16[n_tokens][hidden]. 1 <= n_tokens <= max_tokens of the workspace
 * (max_tokens <= 256). Workspace words carry a 32-bit call count; the call
 * numbered 2^32 - 1 clears them and restarts the count, so a workspace never
 * needs to be zero-filled again. */
int fleet_moe_grouped(const fleet_moe_layer* layer, int32_t n_tokens, const int32_t* ids,
                      const float* weights, const uint16_t* x_norm, uint16_t* out,
                      void* workspace, size_t workspace_bytes, const fleet_moe_dims* dims,
                      hipStream_t stream);

/* fleet_moe_grouped without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). No counterpart in the reference.
 * Same kernels, arguments and results as fleet_moe_grouped, but the workspace
 * is a static device array inside this library (FLEET_MOE_NOALLOC_SCRATCH_BYTES
 * per device, held until the process ends), laid out for at most
 * FLEET_MOE_NOALLOC_MAX_TOKENS tokens; n_tokens above that returns
 * FLEET_MOE_ERR_CAPACITY. Nothing is allocated by any call. The first call on
 * a device looks up that device's copy of the array and zero-fills it (a fill
 * kernel on `stream`, then a stream synchronize): it must not be made under
 * graph capture (FLEET_MOE_ERR_CAPTURE); later calls may be captured.
 * status: device uint32 that receives the step's FLEET_MOE_ABORT_* bits (0 =
 * healthy); the array's status word is cleared at the same time, so every
 * call reports its own. Every call on a device shares that device's array:
 * calls that overlap in time on one device (two streams, two host threads
 * without ordering) race and give unspecified results; order them on one
 * stream. */
#define FLEET_MOE_NOALLOC_MAX_TOKENS 64
#define FLEET_MOE_NOALLOC_SCRATCH_BYTES 7574528
int fleet_moe_grouped_noalloc(const fleet_moe_layer* layer, int32_t n_tokens,
                              const int32_t* ids, const float* weights, const uint16_t* x_norm,
                              uint16_t* out, uint32_t* status, const fleet_moe_dims* dims,
                              hipStream_t stream);

/* ------------------------------------------------------------------------
 * The rest of a decoder layer and of the decode step (absorbed MLA attention,
 * embedding, lm_head + argmax), so that the full 27-layer batch-1 decode runs
 * on this library: per token, embed, then per layer fleet_attn_decode and
 * fleet_moe_dense_decode / fleet_moe_layer_decode, then fleet_lm_head_argmax.
 * Fixed shape: 16 heads, kv_lora 512, qk_nope 128, qk_rope 64, v_head 128,
 * vocab 102400, max_pos <= 4096. */

/* One layer's attention weights: the per-layer pointer tables of Weights
 * (src/runtime/fleet_types.h:44-59: layer_norm_in, layer_qkv,
 * layer_kv_a_norm, layer_kv_b, layer_o_proj), i.e. the manifest tensors
 * "L{i}.norm_in", "L{i}.qkv" ([q_proj (3072) ; kv_a_proj_with_mqa (576)]
 * rows of hidden), "L{i}.kv_a_norm", "L{i}.kv_b" ([16 * 256][512]),
 * "L{i}.o_proj" ([hidden][2048]) (src/host/pack_weights.py:113-121). */
typedef struct fleet_attn_layer {
    const uint16_t* norm_in;    /* bf16[hidden] or NULL (unit) */
    const uint16_t* qkv;        /* bf16[3648][hidden] */
    const uint16_t* kv_a_norm;  /* bf16[512] or NULL (unit) */
    const uint16_t* kv_b;       /* bf16[4096][512] */
    const uint16_t* o_proj;     /* bf16[hidden][2048] */
} fleet_attn_layer;

/* Workspace bytes fleet_attn_decode, fleet_embed and fleet_lm_head_argmax
 * need (one workspace serves all three; about 2.4 MB). */
size_t fleet_attn_workspace_bytes(const fleet_moe_dims* dims);

/* The attention half of one decoder layer at one position:
 * x_out = bf16(x + o_proj(mla(rms_norm(x, norm_in)))). Replaces the
 * QKV_FUSED (kind 0), Q_ABSORB (14), ATTENTION (1), MERGE_UV (2) and O_PROJ
 * (3) task bodies (src/kernels/fleet_kernel.hip:647-660, 675-704, 706-803,
 * 805-830; src/kernels/attention.h:62-93, 171-222, 230-350, 358-420);
 * semantics of src/host/reference_decode.py:210-256 (attention_absorbed) and
 * :294-298 (the residual add). Writes this layer's cache row at the position
 * (c after kv_a_layernorm, then k_pe after RoPE, 576 bf16) and attends over
 * rows 0..position of `cache` ([max_pos][576] bf16: KVCache.data of one
 * layer, src/runtime/fleet_types.h:107-111). rope_cos / rope_sin:
 * fp32[max_pos][64] YaRN tables (the reference's act.cos / act.sin,
 * src/host/fleet_launch.hip:186-218). x, x_out: fp32[hidden] (may be equal).
 * The position is `pos` (0 <= pos < max_pos <= 4096, checked here) or, when
 * pos_dev is not NULL, the device int32 *pos_dev read by the kernels, so one
 * captured graph serves every step; a device position outside [0, max_pos)
 * sets FLEET_MOE_ABORT_POSITION in the workspace status and leaves x_out
 * unspecified. One launch of 256 workgroups on `stream`, all resident at once
 * (their stages hand data to each other through the workspace; a stage that
 * waits past its bound sets FLEET_MOE_ABORT_ATTN_WAIT). */
int fleet_attn_decode(const fleet_attn_layer* layer, const float* x, float* x_out,
                      uint16_t* cache, int32_t max_pos, int32_t pos, const int32_t* pos_dev,
                      const float* rope_cos, const float* rope_sin, void* workspace,
                      size_t workspace_bytes, const fleet_moe_dims* dims, hipStream_t stream);

/* ------------------------------------------------------------------------
 * The whole decode step in one launch (no separate counterpart in the
 * reference, whose persistent kernel runs a step's task graph in one launch:
 * src/kernels/fleet_kernel.hip:933-1040, driven by src/host/fleet_launch.hip).
 * Same arithmetic as embed, then per layer fleet_attn_decode and
 * fleet_moe_dense_decode / fleet_moe_layer_decode, then fleet_lm_head_argmax:
 * every result equals that sequence's bit for bit. */

/* One decoder layer: its attention weights, its FFN (the dense SwiGLU blob
 * "L{i}.dense" when dense is not NULL, with moe.norm as its post-attention
 * norm and the other moe fields unused; else the MoE layer moe) and its KV
 * cache (bf16 [max_pos][576]). */
typedef struct fleet_step_layer {
    fleet_attn_layer attn;
    fleet_moe_layer moe;
    const uint16_t* dense;
    uint16_t* cache;
} fleet_step_layer;

/* Most layers a fleet_decode_step / fleet_ffn_column layer table may hold. */
#define FLEET_STEP_MAX_LAYERS 64

/* The model: layers is a DEVICE array of n_layers (<= FLEET_STEP_MAX_LAYERS)
 * entries, which the kernel reads; embed, lm_head bf16 [102400][hidden];
 * final_norm bf16[hidden] or NULL; rope_cos / rope_sin fp32 [max_pos][64],
 * max_pos <= 4096. */
typedef struct fleet_step_model {
    const fleet_step_layer* layers;
    int32_t n_layers;
    int32_t max_pos;
    const uint16_t* embed;
    const uint16_t* final_norm;
    const uint16_t* lm_head;
    const float* rope_cos;
    const float* rope_sin;
} fleet_step_model;

/* Workspace bytes fleet_decode_step needs (one buffer; about 2.8 MB). */
size_t fleet_decode_step_workspace_bytes(const fleet_moe_dims* dims);

/* One greedy step at position *pos_dev for the token *token (device int32s):
 * x = embed[token], every layer (attention half, then FFN half), then
 * token = argmax(bf16(lm_head . rms_norm(x, final_norm))) (lowest index on
 * ties) into *token_out and *token_next (either may be NULL; token_next may
 * equal token, feeding the next step), and *pos_dev += 1. x_out: fp32[hidden]
 * receives the final residual, or NULL; logits: fp32[102400] or NULL. One
 * launch of 256 workgroups (one per CU), all resident at once (checked as for
 * fleet_moe_layer_decode). A position outside [0, max_pos) or a token outside
 * the vocabulary sets FLEET_MOE_ABORT_POSITION / _TOKEN and the step does
 * nothing else; a stage whose input never arrives sets
 * FLEET_MOE_ABORT_STEP_WAIT (or its stage's wait bit). Calls on one workspace
 * must be ordered on one stream. */
int fleet_decode_step(const fleet_step_model* model, const int32_t* token, int32_t* token_out,
                      int32_t* token_next, int32_t* pos_dev, float* x_out, float* logits,
                      void* workspace, size_t workspace_bytes, const fleet_moe_dims* dims,
                      hipStream_t stream);

/* Workspace bytes fleet_prefill needs (one buffer; about 130 MB). */
size_t fleet_prefill_workspace_bytes(const fleet_moe_dims* dims);

/* n_tokens prompt tokens (device int32) at positions pos0 .. through every
 * layer, all of a chunk's tokens at once: cache rows pos0 .. pos0 + n_tokens -
 * 1 of every layer and x_out (fp32[hidden], the last token's residual before
 * the final norm) are what n_tokens calls of fleet_decode_step leave; no logits
 * and no pick. layers: the HOST copy of model->layers (its pointers are kernel
 * arguments); model->lm_head and final_norm are not read. Every projection is
 * the exact dot product rounded once, as in the decode kernels; the attention's
 * fp64 sums run in another order than theirs before they are rounded to fp32, so
 * equality with the steps in every bit, which all tests show, is not guaranteed
 * for a value on an fp32 rounding boundary. status: a device uint32; a token outside the vocabulary sets
 * FLEET_MOE_ABORT_TOKEN there and counts as a zero row (as in fleet_embed).
 * pos0 + n_tokens <= max_pos is checked here. No two workgroups wait for each
 * other; the workspace needs no clearing. */
int fleet_prefill(const fleet_step_model* model, const fleet_step_layer* layers,
                  const int32_t* tokens, int32_t n_tokens, int32_t pos0, float* x_out,
                  uint32_t* status, void* workspace, size_t workspace_bytes,
                  const fleet_moe_dims* dims, hipStream_t stream);

/* The FLEET_MOE_ABORT_* bits recorded in a fleet_decode_step workspace (the
 * OR over its stages), read synchronously on `stream`. */
int fleet_decode_step_status(const void* workspace, uint32_t* status, hipStream_t stream);

/* The FFN half of every layer of the table chained on x in ONE launch (the
 * benchmark's config 3, reference_decode.py:294-302 without the attention
 * half): x_out = ffn_{n-1}(... ffn_0(x)), each x' = bf16(x + ffn(rms_norm(x)))
 * with the layer's dense or MoE FFN; equal bit for bit to chaining
 * fleet_moe_dense_decode / fleet_moe_layer_decode. layers: DEVICE array
 * (only the FFN fields are read); x, x_out: fp32[hidden] (may be equal);
 * workspace: as fleet_decode_step's (status: fleet_decode_step_status). */
int fleet_ffn_column(const fleet_step_layer* layers, int32_t n_layers, const float* x,
                     float* x_out, void* workspace, size_t workspace_bytes,
                     const fleet_moe_dims* dims, hipStream_t stream);

/* x = embed[*token] as fp32 (the EMBED task, src/kernels/fleet_kernel.hip:
 * 68-78). token: a device int32, so a decode loop can feed the previous
 * step's argmax without a host round trip; a token outside [0, 102400) sets
 * FLEET_MOE_ABORT_TOKEN in the (attention) workspace status and x = 0. */
int fleet_embed(const uint16_t* embed, const int32_t* token, float* x, void* workspace,
                size_t workspace_bytes, hipStream_t stream);

/* Greedy next token: logits = bf16(lm_head . rms_norm(x, final_norm)), token
 * = argmax with ties to the lowest index. Replaces the LM_HEAD (11) and
 * ARGMAX (12) task bodies (src/kernels/fleet_kernel.hip:905-920, 509-585);
 * semantics of HF's bf16 lm_head and torch.argmax as src/host/
 * reference_run.py:99-105 picks the greedy token. logits: fp32[102400]
 * (bf16-valued) or NULL; token_out, token_next: device int32 or NULL (both
 * receive the token; token_next is the input of the next fleet_embed, NULL
 * under teacher forcing); pos_advance: device int32 incremented by one after
 * the pick (the pos_dev of the next step) or NULL. Two launches. */
int fleet_lm_head_argmax(const float* x, const uint16_t* final_norm, const uint16_t* lm_head,
                         float* logits, int32_t* token_out, int32_t* token_next,
                         int32_t* pos_advance, void* workspace, size_t workspace_bytes,
                         const fleet_moe_dims* dims, hipStream_t stream);

/* ------------------------------------------------------------------------
 * Several sequences of one model: their latent cache in pages of 8-bit rows,
 * the attention over it, and the choice of beams (no counterpart in the
 * reference, which decodes one sequence greedily). A step of beam search is
 * fleet_beam_select, fleet_cache_remap by the chosen parents,
 * fleet_cache_grow by one position, and per layer fleet_cache_append and
 * fleet_cache_attend. Everything is enqueued on `stream`, nothing is
 * allocated or read back, and every call may be captured in a graph. */

#define FLEET_CACHE_ROW 576           /* values of one position: c (512), k_pe (64) */
#define FLEET_CACHE_PAGE_TOKENS 64    /* positions of a page */
#define FLEET_CACHE_BLOCK_TOKENS 16   /* positions that share a part's scale */
#define FLEET_CACHE_PAGE_BYTES 36992  /* one layer of a page */
#define FLEET_CACHE_MAX_SEQS 1024
#define FLEET_CACHE_MAX_HEADS 128

/* A cache. One layer of a page is FLEET_CACHE_PAGE_BYTES: four blocks of 16
 * positions, each [36 chunks][16 positions][16 bytes] of e4m3 codes (value
 * 16 * chunk + byte of a row), then fp32 scales [4 blocks][2], of c and of
 * k_pe, powers of two in [2^-110, 2^120], and 96 unused bytes. A row's value is
 * code * scale as a bf16 (beyond its range, with the scale 2^120 only: infinity). Sequence s holds positions 0 .. lens[s] - 1 in the pages
 * table[s][0 ..]; table[s][j] = -1 from page ceil(lens[s] / 64) on. refs[p] is
 * the number of table entries that name page p, 0 for a free page. All
 * sequences empty: table all -1, lens and refs zero (the pool may hold
 * anything). n_pages <= 2^24, n_seqs <= 1024, n_layers <= 64, max_pages <=
 * 2^20. */
typedef struct fleet_cache {
    uint8_t* pool;      /* [n_pages][n_layers][FLEET_CACHE_PAGE_BYTES], 16-byte aligned */
    int32_t* table;     /* [n_seqs][max_pages] */
    int32_t* lens;      /* [n_seqs] */
    int32_t* refs;      /* [n_pages] */
    int32_t n_pages;
    int32_t n_layers;
    int32_t n_seqs;
    int32_t max_pages;
} fleet_cache;

/* Workspace bytes of the fleet_cache_* calls (one workspace serves all calls on a
 * cache; about 34 MB). 0 for sizes outside the limits above. Its first 256 bytes are
 * zero before the first call. Its status word (fleet_moe_workspace_status; the uint32
 * at byte 8, cleared by writing 0) collects the FLEET_MOE_ABORT_* bits named below.
 * It also holds whether the last fleet_cache_grow was refused. */
size_t fleet_cache_workspace_bytes(int32_t n_pages, int32_t n_seqs);

/* Reorders, forks and frees sequences: row i of table and lens becomes what row
 * parents[i] (device int32[n_seqs]) was, or empty where parents[i] is -1; refs
 * follow, and a page that no row names any more is free. Pages are shared, not
 * copied. A parent outside [-1, n_seqs) counts as -1 and sets
 * FLEET_MOE_ABORT_BAD_ID. */
int fleet_cache_remap(const fleet_cache* cache, const int32_t* parents, void* workspace,
                      size_t workspace_bytes, hipStream_t stream);

/* Adds n_new[s] >= 0 (device int32[n_seqs]) positions to every sequence s, to be
 * written by fleet_cache_append: lens grows, and pages are taken from the free
 * ones, lowest first, for sequence 0, then 1, and so on. A last page that is
 * partly filled and shared is copied (the filled blocks, every layer) into the
 * first page its sequence takes, unless all its other holders left it in this
 * call before. All sequences grow or none: too few free pages or a table row
 * that is too short set FLEET_MOE_ABORT_NO_PAGE, a negative count or length
 * FLEET_MOE_ABORT_POSITION, a last page outside the pool
 * FLEET_MOE_ABORT_BAD_PAGE, and nothing changes: fleet_cache_append on this workspace
 * then writes nothing either, until a grow succeeds (one of zeros does). */
int fleet_cache_grow(const fleet_cache* cache, const int32_t* n_new, void* workspace,
                     size_t workspace_bytes, hipStream_t stream);

/* Moves the used pages to the front of the pool: with U of them in use, the k-th
 * used page at or behind U moves into the k-th free one before it; table and
 * refs follow. n_used: device int32 that receives U, or NULL. */
int fleet_cache_compact(const fleet_cache* cache, int32_t* n_used, void* workspace,
                        size_t workspace_bytes, hipStream_t stream);

/* Writes the newest positions of each sequence, of layers layer0 .. layer0 +
 * n_layers - 1. rows: bf16 [n_layers][n_rows][576], rows row_stride and layers
 * layer_stride elements apart (multiples of 8, so that a row is 16-byte
 * aligned; all rows of a layer before the next layer's, or all layers of a row before
 * the next row's). start: device int32[n_seqs + 1], not decreasing, start[n_seqs] <=
 * n_rows: rows start[s] .. start[s + 1] - 1 are the last of the lens[s]
 * positions of sequence s (rows before start[0] are nobody's); NULL: one row for each sequence (n_rows == n_seqs).
 * A block's scale is the least power of two that takes its new finite values
 * within the largest code, 448, and no less than the scale of older positions
 * in the block; where those have a smaller scale they are rounded again to the
 * new one. Rounding is to nearest even; an infinity becomes +-448 times the
 * scale, NaN stays NaN. After a grow that was refused, nothing is written, and its
 * status bits are set again. More rows than positions, or a length outside the
 * table, set FLEET_MOE_ABORT_POSITION, a page outside the pool or one that
 * another sequence holds too FLEET_MOE_ABORT_BAD_PAGE; such rows are not
 * written. */
int fleet_cache_append(const fleet_cache* cache, int32_t layer0, int32_t n_layers,
                       const uint16_t* rows, int64_t row_stride, int64_t layer_stride,
                       const int32_t* start, int32_t n_rows, void* workspace,
                       size_t workspace_bytes, hipStream_t stream);

/* The reverse: rows receives the newest positions of each sequence as bf16 (the
 * values the codes stand for). Rows that name no position or a page outside the
 * pool (status as above), and those before start[0] or behind start[n_seqs], are
 * left as they were. */
int fleet_cache_read(const fleet_cache* cache, int32_t layer0, int32_t n_layers, uint16_t* rows,
                     int64_t row_stride, int64_t layer_stride, const int32_t* start,
                     int32_t n_rows, void* workspace, size_t workspace_bytes,
                     hipStream_t stream);

/* Absorbed-MLA attention of one layer over the cache. q: bf16 [n_tokens][n_heads]
 * [576] (the absorbed query, then its rotated part), tokens q_stride elements
 * apart (a multiple of 8); start as above: token start[s] + j stands at position
 * lens[s] - (start[s+1] - start[s]) + j of sequence s. It sees the positions p up
 * to its own, with window > 0 only those above its own - window and those
 * below sinks. out[token][head][0..511] = sum_p softmax_p(scale * q . row_p)
 * c_p as bf16, lse[token][head] (fp32, may be NULL) = log sum_p exp(scale * q .
 * row_p); a token that sees nothing gets out = 0, lse = -infinity. NaN and
 * infinities reach only the tokens that see them. A score (scale * q . row) beyond the
 * range of fp32 is infinite: +infinity makes the outputs of its token and head NaN,
 * -infinity has the weight 0. Products are of bf16 values with fp32 sums;
 * before the second product the probabilities are rounded to 16 bits where a call has 32
 * (token, head) rows a sequence or fewer, to bf16's 8 where it has more. max_len: a bound
 * on lens that the host knows, for the division of the work (longer sequences
 * are still right), or 0. Outputs of tokens before start[0] or behind
 * start[n_seqs] are left as they were. A length outside the table sets FLEET_MOE_ABORT_POSITION, and the
 * sequence's tokens see nothing; positions in a page outside the pool are not
 * seen, and set FLEET_MOE_ABORT_BAD_PAGE. 1 <= n_heads <= 128, n_tokens * n_heads
 * <= 2^26, 0 < scale <= 2.3e38 (scale * log2(e) is an fp32 number). */
int fleet_cache_attend(const fleet_cache* cache, int32_t layer, const uint16_t* q,
                       int64_t q_stride, const int32_t* start, int32_t n_tokens,
                       int32_t n_heads, int32_t max_len, int32_t window, int32_t sinks,
                       float scale, uint16_t* out, float* lse, void* workspace,
                       size_t workspace_bytes, hipStream_t stream);

#define FLEET_BEAM_MAX_BEAMS 64
#define FLEET_BEAM_MAX_OUT 64

/* Workspace bytes of fleet_beam_select (0: outside its limits). */
size_t fleet_beam_workspace_bytes(int32_t n_groups, int32_t n_beams, int32_t n_out,
                                  int32_t vocab);

/* The n_out best continuations of each group of n_beams beams. logits: fp32 rows
 * of vocab, ld elements apart, row g * n_beams + b of beam b of group g; scores:
 * fp32 [n_groups][n_beams], the beams' log probabilities so far; finished:
 * uint8 [n_groups][n_beams] or NULL. Beam b offers every token t with the score
 * scores[b] + log softmax(logits[b])[t], a finished beam one continuation, eos
 * with its own score. Order: higher score (64 bits), then lower beam, higher
 * logit, lower token. (Log sums are taken to 2^-18, and in 64 bits where two beams'
 * candidates are closer than that leaves certain, which takes longer: 40 us for each
 * such beam of 102,400 logits.) A logit of NaN or -infinity is not offered, +infinity
 * counts as the largest finite number; a beam whose score is NaN or -infinity
 * offers nothing. out_scores fp32, parents int32 (row g * n_beams + b, as
 * fleet_cache_remap takes it), tokens int32 and out_finished uint8 (the parent
 * was finished, or the token is eos; may be NULL) are [n_groups][n_out], best first;
 * where a group offers fewer: -infinity, -1, -1, 0. eos < 0: no such token (a finished
 * beam then offers token -1). 1 <= n_beams, n_out <= 64, n_groups * n_beams <= 65535,
 * 1 <= vocab <= 2^24. Two launches; the workspace needs no clearing. */
int fleet_beam_select(const float* logits, int64_t ld, const float* scores,
                      const uint8_t* finished, int32_t n_groups, int32_t n_beams, int32_t n_out,
                      int32_t vocab, int32_t eos, float* out_scores, int32_t* parents,
                      int32_t* tokens, uint8_t* out_finished, void* workspace,
                      size_t workspace_bytes, hipStream_t stream);

/* Copies the workspace's sticky status word to *status (0 = healthy; a
 * nonzero value names a bounded wait that expired, see FLEET_MOE_ABORT_*),
 * synchronising `stream`. The reference's equivalent is the sticky rt.abort
 * word (src/runtime/fleet_runtime.h:194-198, 287-293). */
int fleet_moe_workspace_status(const void* workspace, uint32_t* status, hipStream_t stream);

#define FLEET_MOE_ABORT_ROUTER_WAIT 0x1u  /* router logits never published  */
#define FLEET_MOE_ABORT_UNIT_WAIT 0x2u    /* an expert unit never completed */
#define FLEET_MOE_ABORT_GROUP_WAIT 0x4u   /* grouped step phase never completed */
#define FLEET_MOE_ABORT_POSITION 0x8u     /* device position outside [0, max_pos) */
#define FLEET_MOE_ABORT_TOKEN 0x10u       /* device token outside the vocabulary */
#define FLEET_MOE_ABORT_ATTN_WAIT 0x20u   /* an attention stage never completed */
#define FLEET_MOE_ABORT_BAD_ID 0x40u      /* grouped: an expert id outside [0, n_routed)
                                             was clamped into range (output unspecified) */
#define FLEET_MOE_ABORT_STEP_WAIT 0x80u   /* fleet_decode_step: a stage's input residual
                                             (or an lm_head candidate) never arrived */
#define FLEET_MOE_ABORT_NO_PAGE 0x400u    /* fleet_cache_grow: too few free pages */
#define FLEET_MOE_ABORT_BAD_PAGE 0x800u   /* fleet_cache_*: a table entry outside the pool,
                                             or a shared page to be written */

/* Diagnostic: reads `bytes` of device memory with the weight-streaming load
 * pattern of the kernels above (16-byte non-temporal loads, 1 KB per wave
 * instruction) and nothing else. Gives the achievable HBM read rate, and is
 * the known-size kernel against which rocprofv3 FETCH_SIZE is calibrated.
 * The reference's equivalent is bench/microbench.hip section (c),
 * gemv_stream (:422-447). bytes must be a multiple of 4096; sink: a device
 * uint32 that is written only if the XOR of the data is 0x9e3779b9. */
int fleet_moe_stream_read(const void* buf, size_t bytes, uint32_t* sink, hipStream_t stream);

/* Human-readable text for a return code of this library. */
const char* fleet_moe_error_string(int code);

/* ABI version of this header (major * 100 + minor). */
int fleet_moe_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* FLEET_MOE_H */
