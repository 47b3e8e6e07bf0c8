/*
 * specfit_amd.h -- C ABI of the MI355X (gfx950) offloaded Qwen3-MoE
 * verification path.
 *
 * Every entry point is enqueue-only: it validates its arguments on the host,
 * launches HIP work on the caller's stream and returns.  Nothing here
 * allocates device memory, synchronises the host, or keeps mutable global
 * state; all buffers are owned by the caller.  Return value 0 means success;
 * a non-zero value is an SF_ERR_* code (argument errors) or a hipError_t
 * offset by SF_ERR_HIP_BASE.  sf_error_string() names either kind.
 *
 * Data types: "bf16" buffers hold IEEE bfloat16 bit patterns (uint16_t);
 * integer buffers are little-endian.  Streams are hipStream_t passed as an
 * opaque pointer (NULL = the legacy default stream).
 *
 * Reference interfaces replaced (paths relative to the SpecFit tree; "tf:" is
 * transformers/models/qwen3_moe/modeling_qwen3_moe.py of the pinned
 * transformers release):
 *   sf_router_topk       tf:258-267  Qwen3MoeTopKRouter.forward
 *   sf_dispatch          src/specfit/runtime/qwen3_offloaded_experts.py:173-178
 *                        (stable sort + unique_consecutive + route_tokens) and
 *                        :111-113,120-122 (unique / where of the legacy path)
 *   sf_grouped_swiglu    qwen3_offloaded_experts.py:38-62 (_expert_forward),
 *                        :132-138 and :198 (routing-weight scale), :186-190
 *                        (route gather)
 *   sf_expert_swiglu     qwen3_offloaded_experts.py:38-62 (_expert_forward
 *                        on already-gathered rows, no weight scale)
 *   sf_combine           qwen3_offloaded_experts.py:144-164 and :200-202
 *                        (index_add_ in canonical or arrival order)
 *   sf_copy_h2d          src/specfit/runtime/gpu_expert_cache.py:556-561
 *                        (slot.tensor.copy_(pinned_source, non_blocking=True))
 *   sf_expert_decode     the same copy when the transfer moves an
 *                        exponent-coded record (decoded into the slot)
 *   sf_tree_attention, sf_tree_attention_split
 *                        the attention of the verification forward:
 *                        eagle3_tree.py:1202-1240 runs the target with
 *                        Eagle3DraftTree.verification_attention_mask
 *                        (eagle3_types.py:450-473); each Qwen3 attention layer
 *                        then calls transformers sdpa_attention_forward
 *                        (integrations/sdpa_attention.py) with that mask
 *   sf_rms_norm          tf:294-299  Qwen3MoeRMSNorm.forward (the four norms
 *                        of every decoder layer of the verification forward)
 *   sf_qk_norm_rope      tf:162-167  the query/key norms and
 *                        apply_rotary_pos_emb (tf:58-81) of
 *                        Qwen3MoeAttention.forward
 *   sf_kv_append, sf_kv_compact, sf_kv_fold, sf_kv_read, sf_block_attention
 *                        the bf16 DynamicCache of the target and its
 *                        compaction (eagle3_tree.py:833-858), held in 8 bits,
 *                        and the attention over it
 *   sf_rotary            apply_rotary_pos_emb with angles from the positions
 *   sf_mx_quantize, sf_mx_values, sf_mx_linear, sf_mx_grouped_swiglu
 *                        the model's linear layers and experts
 *                        (qwen3_offloaded_experts.py:38-62) with weights held
 *                        in microscaled 4 bits
 *   sf_add_rms_norm      the residual's addition and the norm behind it, of a
 *                        decoder layer
 *   sf_logit_rules       the argmax of eagle3_tree.py:1241-1290 with rules on
 *                        the logits before it
 */
#ifndef SPECFIT_AMD_H
#define SPECFIT_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SF_ABI_VERSION 13

/* Argument error codes (hipError_t values are returned as SF_ERR_HIP_BASE + e). */
#define SF_OK 0
#define SF_ERR_INVALID_ARGUMENT 1
#define SF_ERR_UNSUPPORTED_SHAPE 2
#define SF_ERR_MISALIGNED 3
#define SF_ERR_TOO_MANY_EXPERTS 4
#define SF_ERR_SCRATCH_LIMIT 5
#define SF_ERR_HIP_BASE 1000

/* Largest expert count the router, dispatch and combine kernels accept. */
#define SF_MAX_EXPERTS 256
/* Largest top-k. */
#define SF_MAX_TOPK 32
/* Most rows that the products with 4-bit weights take in 16 bits and round where
 * they are read: one tile of the matrix instruction. */
#define SF_MX_RAW_ROWS 16
/* Values per chunk of an exponent-coded expert record (sf_expert_decode). */
#define SF_DECODE_CHUNK 4096

typedef void *sf_stream_t;

/* ABI version of the loaded library (SF_ABI_VERSION at build time). */
int sf_abi_version(void);

/* Static description of an error code; never NULL. */
const char *sf_error_string(int code);

/*
 * K1: router.  Replaces Qwen3MoeTopKRouter.forward (tf:258-267).
 *   logits[t,e] = bf16( sum_k hidden[t,k] * router_weight[e,k] )   (fp32 sum)
 *   p[t,:]      = softmax_fp32(logits[t,:])
 *   (v, idx)    = top_k(p[t,:]) in descending p; equal p -> lower expert id
 *   w[t,j]      = bf16( v_j / (v_0 + ... + v_{k-1}) )   if norm_topk_prob
 *               = bf16( v_j )                          otherwise
 * The fp32 summation order of the dot product and of the softmax sum is
 * fixed (see the kernel source), so logits, weights and indices are a pure
 * function of the inputs.
 *   hidden        bf16 [tokens, hidden_size]
 *   router_weight bf16 [num_experts, hidden_size]
 *   logits        bf16 [tokens, num_experts]          (output)
 *   topk_weights  bf16 [tokens, top_k]                (output)
 *   topk_index    int64 [tokens, top_k]               (output)
 * Limits: 1 <= num_experts <= SF_MAX_EXPERTS, 1 <= top_k <= min(num_experts,
 * SF_MAX_TOPK), hidden_size >= 1.  tokens == 0 launches nothing.
 */
int sf_router_topk(const void *hidden, const void *router_weight, int tokens,
                   int hidden_size, int num_experts, int top_k,
                   int norm_topk_prob, void *logits, void *topk_weights,
                   int64_t *topk_index, sf_stream_t stream);

/*
 * K2: token-to-expert dispatch.  Replaces the stable sort of the flattened
 * routes by expert id (qwen3_offloaded_experts.py:173-178).
 *   topk_index int64 [tokens, top_k]
 *   counts     int32 [num_experts + 1]  routes per expert; counts[num_experts]
 *              = number of entries outside [0, num_experts) (not dispatched)
 *   offsets    int32 [num_experts + 1]  exclusive prefix sum of counts
 *   perm_pos   int32 [tokens * top_k]   route position (t * top_k + j) of each
 *              permuted row; rows of one expert are contiguous and keep
 *              ascending position order (stable)
 *   inv_perm   int32 [tokens * top_k]   permuted row of each route position
 *              (-1 for an out-of-range entry)
 *   host_meta  NULL, or pinned host memory (hipHostMalloc) of int32
 *              [2, num_experts + 1]: the kernel also writes counts (row 0)
 *              and offsets (row 1) there, so the caller reads the routes per
 *              expert once the stream passes the kernel, with no separate
 *              device-to-host copy (the reference's one host read of the
 *              routed experts, qwen3_offloaded_experts.py:111-113).  Memory
 *              the device cannot map returns SF_ERR_INVALID_ARGUMENT.
 * One workgroup for up to 1024 routes, up to 256 above; any tokens >= 0.
 */
int sf_dispatch(const int64_t *topk_index, int tokens, int top_k,
                int num_experts, int32_t *counts, int32_t *offsets,
                int32_t *perm_pos, int32_t *inv_perm, int32_t *host_meta,
                sf_stream_t stream);

/*
 * K3: grouped SwiGLU expert MLP over dispatched rows.  Replaces the per-expert
 * loop of _expert_forward + weight scale (qwen3_offloaded_experts.py:38-62,
 * 132-138, 186-198).  For each listed expert e with rows
 * r in [offsets[e], offsets[e+1]) and token t = perm_pos[r] / top_k:
 *   gu   = bf16(hidden[t] . GU^T)          GU = packed[0 : 2*I*H] as [2I, H]
 *   act  = bf16(bf16(silu(gu[:I])) * gu[I:])
 *   y    = bf16(act . D^T)                 D  = packed[2*I*H :] as [H, I]
 *   rows[r] = bf16(y * route_weights[perm_pos[r]])   (y if route_weights NULL)
 * Packed expert layout: [gate (I x H) | up (I x H) | down (H x I)], row-major
 * bf16, as written by the reference's packed checkpoint.
 *   max_rows        an upper bound on the rows of any listed expert
 *                   (tokens * top_k always is).  It picks the kernel build
 *                   (registers sized for that many rows).  Any value >= 1
 *                   computes every row; with a value below some expert's
 *                   row count that expert's fp32 summation order is the one
 *                   of a smaller expert.
 * The MFMA kernels cover the Qwen3-30B-A3B (hidden 2048, intermediate 768)
 * and Qwen3-235B-A22B (hidden 4096, intermediate 1536) expert shapes with
 * 16-byte aligned buffers; other shapes run fp32 loop kernels with the same
 * rounding points.  The fp32 summation order of
 * an output depends on the shape and on its expert's row count only.
 *   expert_ids      host int32 [n_experts]: experts computed by this call
 *   expert_weights  host uint64 [n_experts]: device address of each expert's
 *                   packed weights (a cache slot)
 *   expert_row_begin, expert_row_count
 *                   host int32 [n_experts] each, or both NULL: each listed
 *                   expert's first permuted row and row count
 *                   (offsets[e] and offsets[e+1] - offsets[e]).  A caller
 *                   that has read the dispatch counts passes them, so the
 *                   kernels start streaming weights without first reading
 *                   offsets from device memory; with NULL they read them.
 *   act_workspace   bf16 [tokens * top_k, intermediate_size] scratch
 *   out_rows        bf16 [tokens * top_k, hidden_size] (rows of listed
 *                   experts are written, others untouched)
 * Experts of one call are independent; the result of an expert does not
 * depend on which other experts share the call.
 */
int sf_grouped_swiglu(const void *hidden, const int32_t *perm_pos,
                      const int32_t *offsets, const void *route_weights,
                      int tokens, int top_k, int hidden_size,
                      int intermediate_size, int n_experts, int max_rows,
                      const int32_t *expert_ids,
                      const uint64_t *expert_weights,
                      const int32_t *expert_row_begin,
                      const int32_t *expert_row_count, void *act_workspace,
                      void *out_rows, sf_stream_t stream);

/*
 * K3, device slot-table form: computes every expert e < num_experts whose
 * slot_of_expert[e] >= 0 and that has at least one row, reading its weights
 * at slot_base + slot_of_expert[e] * slot_stride_elems (bf16 elements).
 * slot_of_expert is a device int32 [num_experts] array whose entries are -1
 * or the index of a slot behind slot_base (the kernel trusts them, as it
 * trusts slot_base itself).  Needs no host-side knowledge of which experts
 * are active (no device-to-host read).
 * max_rows bounds the rows of any expert as for sf_grouped_swiglu (tokens
 * is one when every token's top_k experts are distinct, as a router's are).
 */
int sf_grouped_swiglu_table(const void *hidden, const int32_t *perm_pos,
                            const int32_t *offsets, const void *route_weights,
                            int tokens, int top_k, int hidden_size,
                            int intermediate_size, int num_experts, int max_rows,
                            const int32_t *slot_of_expert,
                            const void *slot_base, int64_t slot_stride_elems,
                            void *act_workspace, void *out_rows,
                            sf_stream_t stream);

/*
 * sf_grouped_swiglu_table with a bound on the number of slot_of_expert's
 * entries that are not -1 (0: not known), which picks between the kernels for
 * few and for many rows.  The results do not depend on it.
 */
int sf_grouped_swiglu_table_residents(const void *hidden, const int32_t *perm_pos,
                                      const int32_t *offsets,
                                      const void *route_weights, int tokens,
                                      int top_k, int hidden_size,
                                      int intermediate_size, int num_experts,
                                      int max_rows, int residents,
                                      const int32_t *slot_of_expert,
                                      const void *slot_base,
                                      int64_t slot_stride_elems,
                                      void *act_workspace, void *out_rows,
                                      sf_stream_t stream);

/*
 * K3, device slot-table form, allocating nothing.  No counterpart in the
 * reference: this entry point is for callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc).  Same arguments, results and limits as
 * sf_grouped_swiglu_table minus act_workspace: the [tokens * top_k,
 * intermediate_size] bf16 activation workspace is taken from a fixed device
 * array of SF_NOALLOC_SCRATCH_BYTES that each GPU the library runs on holds
 * until the process ends.
 * Limit: tokens * top_k * intermediate_size * 2 <= SF_NOALLOC_SCRATCH_BYTES
 * (4 MiB: 341 tokens at top_k 8 and intermediate 768), else
 * SF_ERR_SCRATCH_LIMIT and nothing is launched.
 * Every call on one GPU shares that GPU's array, which keeps the last
 * call's contents: calls that overlap on one GPU (kernels on concurrent
 * streams, or host threads) race.  Nothing in it needs to start at zero:
 * each activation row a launch reads is written first by the same launch.
 */
#define SF_NOALLOC_SCRATCH_BYTES (4u << 20)
int sf_grouped_swiglu_table_noalloc(const void *hidden, const int32_t *perm_pos,
                                    const int32_t *offsets,
                                    const void *route_weights, int tokens,
                                    int top_k, int hidden_size,
                                    int intermediate_size, int num_experts,
                                    int max_rows,
                                    const int32_t *slot_of_expert,
                                    const void *slot_base,
                                    int64_t slot_stride_elems, void *out_rows,
                                    sf_stream_t stream);

/*
 * K3 on already-gathered rows of one expert (the _expert_forward seam,
 * qwen3_offloaded_experts.py:38-62): out[m, H] = y without weight scale.
 *   rows bf16 [m, hidden_size] (row stride row_stride elements)
 */
int sf_expert_swiglu(const void *rows, int m, int64_t row_stride,
                     int hidden_size, int intermediate_size,
                     const void *packed_weights, void *act_workspace,
                     void *out, sf_stream_t stream);

/*
 * K4: weighted combine.  Replaces zeros_like + index_add_ of the expert
 * contributions (qwen3_offloaded_experts.py:144-164, 200-202).
 *   out[t] = sum over the routes j of token t, in ascending
 *            (expert_rank[topk_index[t,j]], j) order, of rows[inv_perm[t*K+j]]
 * With accumulate_fp32 == 0 every addition rounds to bf16, exactly as
 * sequential bf16 index_add_ calls; otherwise the sum is fp32 and rounded once.
 *   rows         bf16 [tokens * top_k, hidden_size] (K3 output)
 *   expert_rank  host int32 [num_experts] execution rank of each expert, or
 *                NULL for canonical ascending expert id
 *   out          bf16 [tokens, hidden_size]
 */
int sf_combine(const void *rows, const int64_t *topk_index,
               const int32_t *inv_perm, const int32_t *expert_rank,
               int tokens, int top_k, int num_experts, int hidden_size,
               int accumulate_fp32, void *out, sf_stream_t stream);

/*
 * Host-to-device copy of an expert from pinned (page-locked) host memory into
 * a cache slot, enqueued on `stream` (SDMA).  Replaces the non-blocking
 * slot.tensor.copy_(pinned) of gpu_expert_cache.py:556-561.
 */
int sf_copy_h2d(void *device_dst, const void *host_src, size_t bytes,
                sf_stream_t stream);

/*
 * Exponent-coded expert records: the host-to-device transfer of an expert
 * may move a lossless record of its bf16 weights instead of the raw bytes
 * (about 67% of them for N(0, 0.02) weights), decoded into the slot on the
 * device.  Together with sf_copy_h2d of the record into a staging buffer
 * this replaces the same slot.tensor.copy_(pinned_source)
 * (gpu_expert_cache.py:556-561); the slot ends with the same bytes.  The
 * exponent of a value is a cascade of codes into the 32-byte table:
 *   level 1, 2 bits (every value):       c < 3: table[c];       3: level 2
 *   level 2, 2 bits (n2 values):         c < 3: table[8 + c];   3: level 3
 *   level 3, 4 bits (n3 values):         c < 15: table[16 + c]; 15: raw byte
 * Record of n values (every section 256-byte aligned):
 *   S   [n] uint8                 sign << 7 | mantissa of value i
 *   P   2 planes of ceil(n/16) uint16 words: bit i%16 of word i/16 of
 *                                 plane p is bit p of value i's level-1 code
 *   L2  [ceil(n2/4)] uint8        level-2 codes in value order, entry j at
 *                                 bits 2(j%4) of byte j/4
 *   L3  [ceil(n3/2)] uint8        level-3 codes in value order, entry j at
 *                                 bits 4(j%2) of byte j/2
 *   R   [nr] uint8                raw exponent bytes in value order
 *   C2, C3, CR [c + 1] uint32     L2, L3 and R entries of the values before
 *                                 value k * SF_DECODE_CHUNK
 *                                 (c = ceil(n / SF_DECODE_CHUNK))
 * sf_expert_record_bytes returns the record size (-1 for invalid counts;
 * valid: 0 <= n_raw <= n_third <= n_second <= n_values).
 * sf_expert_decode writes out[i] = sign | exponent | mantissa of value i:
 *   record          device buffer of at least record_bytes >= the record size
 *   exponent_table  host array of 32 exponent bytes (entries 3..7, 11..15
 *                   and 31 unused)
 *   out             bf16 [n_values], 16-byte aligned like record
 */
int64_t sf_expert_record_bytes(int64_t n_values, int64_t n_second, int64_t n_third,
                               int64_t n_raw);
int sf_expert_decode(const void *record, size_t record_bytes, int64_t n_values,
                     const uint8_t *exponent_table, int n_second, int n_third, int n_raw,
                     void *out, sf_stream_t stream);

/*
 * K5: grouped-query attention of the verification forward over the cached
 * prefix plus the draft tree.  For query token qi and query head
 * qh = h * G + j (G = q_heads / kv_heads, h the key/value head):
 *   out[qi, qh, :] = sum_s p_s * v[h, s, :],
 *   p = softmax over admitted keys s of scale * (q[qi, qh, :] . k[h, s, :])
 * with scores and sums in fp32 and the result rounded to bf16 once.  The form
 * for 16-byte aligned rows, head_dim 64 or 128 and G >= 2 multiplies V by p
 * rounded to bf16 (relative to the row's running maximum), and by the rest of
 * that rounding for part of the keys.  Key s is admitted when
 * mask[qi * mask_stride_query + s] != 0; with mask == NULL, when
 * s <= keys - queries + qi (causal, aligned to the end of the keys).  A
 * query with no admitted key gets zeros.
 *   q     bf16, element (qi, qh, d) at qi*q_stride_token + qh*q_stride_head + d
 *   k, v  bf16, element (h, s, d) at h*stride_head + s*stride_token + d
 *         (k: 16-byte aligned rows)
 *   mask  uint8/bool [queries, >= keys] with row stride mask_stride_query
 *   out   bf16 [queries, q_heads, head_dim], contiguous
 * head_dim % 8 == 0, head_dim <= 256, G in {1, 2, 4, 8, 16}.
 */
int sf_tree_attention(const void *q, int64_t q_stride_token,
                      int64_t q_stride_head, const void *k,
                      int64_t k_stride_head, int64_t k_stride_token,
                      const void *v, int64_t v_stride_head,
                      int64_t v_stride_token, const uint8_t *mask,
                      int64_t mask_stride_query, int queries, int keys,
                      int q_heads, int kv_heads, int head_dim, float scale,
                      void *out, sf_stream_t stream);

/*
 * sf_tree_attention with scratch memory that lets a call of few query rows
 * split its keys over the chip: each split's (max, sum, accumulator) goes to
 * the workspace in fp32 and a second kernel merges them in split order.
 * sf_tree_attention_workspace returns the bytes a call of that shape (masked:
 * with a mask) with 16-byte aligned rows can use (0: it would not split).
 * workspace: device memory, 16-byte aligned, in use until the call's kernels
 * have run; with less than the needed bytes (or NULL) the call runs unsplit.
 * Results of the two forms differ by the order of the fp32 sums and by the
 * rounding of probabilities to bf16, each relative to its form's running
 * maximum.
 */
int64_t sf_tree_attention_workspace(int queries, int keys, int q_heads,
                                    int kv_heads, int head_dim, int masked);
int sf_tree_attention_split(const void *q, int64_t q_stride_token,
                            int64_t q_stride_head, const void *k,
                            int64_t k_stride_head, int64_t k_stride_token,
                            const void *v, int64_t v_stride_head,
                            int64_t v_stride_token, const uint8_t *mask,
                            int64_t mask_stride_query, int queries, int keys,
                            int q_heads, int kv_heads, int head_dim,
                            float scale, void *out, void *workspace,
                            int64_t workspace_bytes, sf_stream_t stream);

/*
 * K6: RMSNorm over the last dimension.  Replaces Qwen3MoeRMSNorm.forward
 * (tf:294-299):
 *   v = mean over d of float(x[r, d])^2 (fp32)
 *   out[r, d] = bf16(float(weight[d]) * bf16(float(x[r, d]) * rsqrt(v + eps)))
 *   x       bf16, row r at x + r * row_stride (elements), dim elements
 *   weight  bf16 [dim]
 *   out     bf16, row r at out + r * out_stride (may equal x: in place)
 * The fp32 sum of squares runs in a fixed order of its own, so results can
 * differ from the eager module by a last-place rounding of the variance.
 */
int sf_rms_norm(const void *x, int64_t row_stride, int rows, int dim,
                const void *weight, float eps, void *out, int64_t out_stride,
                sf_stream_t stream);

/*
 * K7: query/key RMSNorm and rotary embedding of one attention layer (batch
 * 1).  Replaces, in Qwen3MoeAttention.forward (tf:162-167),
 * q_norm(q.view(T, Hq, D)), k_norm(k.view(T, Hk, D)) and
 * apply_rotary_pos_emb (tf:58-81):
 *   n = sf_rms_norm's row result (same bits)
 *   out[h, t, d] = bf16(bf16(n[d] * cos[t, d]) + bf16(rot(n)[d] * sin[t, d]))
 *   rot(n)[d] = -n[d + D/2] for d < D/2, n[d - D/2] otherwise
 *   q, k        bf16 [tokens, q_heads | kv_heads, head_dim]: token t at
 *               q + t * q_stride_token (elements; >= q_heads * head_dim and a
 *               multiple of 8, e.g. one fused q/k/v projection row), heads
 *               contiguous within a token
 *   q_weight, k_weight  bf16 [head_dim]
 *   cos, sin    bf16 [tokens, head_dim], contiguous
 *   q_out, k_out  bf16 [q_heads | kv_heads, tokens, head_dim], contiguous
 * head_dim must be 128 (SF_ERR_UNSUPPORTED_SHAPE otherwise); all buffers
 * 16-byte aligned.
 */
int sf_qk_norm_rope(const void *q, int64_t q_stride_token, const void *k,
                    int64_t k_stride_token, int tokens, int q_heads,
                    int kv_heads, int head_dim, const void *q_weight,
                    const void *k_weight, float eps, const void *cos,
                    const void *sin, void *q_out, void *k_out,
                    sf_stream_t stream);

/*
 * K9: the block cache.  Keys and values of a sequence whose complete blocks
 * of SF_KV_BLOCK tokens are held in 8 bits, with one scale per block, head and
 * K or V, and whose last tokens are held in bf16 in a ring of blocks until
 * they are folded.  No counterpart in the reference, whose target keeps a bf16
 * DynamicCache; the calls take the places of its update and of
 * _compact_tree_cache (eagle3_tree.py:833-858).
 *   x^ = code * 2^e,  e the least integer >= SF_KV_MIN_EXPONENT with
 *                     max |x| over the block's finite values <= q 2^e,
 *   code = x / 2^e to the nearest (ties to even) int8 (q = 127) or e4m3
 *   (q = 448); a value that is not finite is held as NaN (int8: code -128).
 * Powers of two make x / 2^e and x^ exact, so the codes do not depend on how
 * they are computed and x^ is a bf16 number.
 *   k8, v8       [heads, capacity_blocks, 64 * head_dim] codes
 *   k_scale, v_scale  fp32 [heads, capacity_blocks]
 *   flags        int32 [heads, capacity_blocks]: bit 0 (1): the values (keys)
 *                hold a NaN code
 *   k_tail, v_tail  bf16 [heads, ring_blocks, 64 * head_dim]: block j of the
 *                sequence at j % ring_blocks
 *   tail_flags   int32 [heads, ring_blocks]: the values of the block may hold
 *                infinity or NaN
 * heads = batch * kv_heads (times the layers for sf_kv_compact and sf_kv_fold,
 * whose arrays then hold the layers one after another).  All buffers 16-byte
 * aligned; the ring starts zeroed.  Blocks below folded_blocks are read from
 * the 8-bit arrays, the others from the ring.  The order of values inside a
 * block is the library's own (csrc/kv_blocks.h).
 * head_dim 64 or 128.
 */
#define SF_KV_BLOCK 64
#define SF_KV_E4M3 0
#define SF_KV_INT8 1
#define SF_KV_MIN_EXPONENT (-60)
/* Positions that one sf_kv_compact call takes. */
#define SF_KV_MAX_MOVES 256
typedef struct sf_kv_cache {
  void *k8, *v8;
  float *k_scale, *v_scale;
  int32_t *flags;
  void *k_tail, *v_tail;
  int32_t *tail_flags;
  int32_t heads, head_dim, held;
  int32_t capacity_blocks, ring_blocks;
  int32_t folded_blocks;
} sf_kv_cache;

/*
 * Writes tokens [start, start + tokens) of every (sequence, head): element
 * (b, h, t, d) of k and v is read at b * stride_batch + h * stride_head +
 * t * stride_token + d.  Rows of the last block behind them become zeros.
 * The blocks touched must be at or above folded_blocks and fit the ring and
 * the capacity (SF_ERR_INVALID_ARGUMENT).
 */
int sf_kv_append(const sf_kv_cache *cache, int kv_heads, const void *k,
                 int64_t k_stride_batch, int64_t k_stride_head,
                 int64_t k_stride_token, const void *v, int64_t v_stride_batch,
                 int64_t v_stride_head, int64_t v_stride_token, int64_t start,
                 int tokens, sf_stream_t stream);

/*
 * Moves the rows of tokens base + positions[i] to base + first + i, i < count
 * (the accepted path of a draft tree): positions is a host array, strictly
 * ascending, with positions[i] >= first + i, and end is the number of tokens
 * the ring holds rows of.  count <= SF_KV_MAX_MOVES.
 */
int sf_kv_compact(const sf_kv_cache *cache, int64_t base, int first,
                  const int32_t *positions, int count, int64_t end,
                  sf_stream_t stream);

/*
 * Folds the ring's blocks [folded_blocks, folded_blocks + blocks), which are
 * complete, into the 8-bit arrays.  The ring keeps them.
 */
int sf_kv_fold(const sf_kv_cache *cache, int blocks, sf_stream_t stream);

/*
 * x^ of tokens [start, start + tokens) as bf16 [heads, tokens, head_dim],
 * contiguous, 16-byte aligned (the ring's rows as they are).
 */
int sf_kv_read(const sf_kv_cache *cache, int64_t start, int tokens, void *k,
               void *v, sf_stream_t stream);

/*
 * K10: grouped-query attention over a block cache of `keys` tokens:
 *   out[b, qi, qh, :] = sum_s p_s * v^[b, h, s, :],
 *   p = softmax over admitted keys s of scale * (q[b, qi, qh, :] . k^[b, h, s, :])
 * h = qh / (q_heads / kv_heads), scores and sums in fp32, the result rounded to bf16
 * once; for the product with v^, p is kept to 2^-16 of itself where a workgroup takes 16
 * rows (sf_block_attention_rows), and rounded to bf16 where it takes 256.  The mask
 * covers the last mask_keys keys; a key before them is admitted by every row.
 * With mask == NULL key s is admitted when s <= keys - queries + qi.  A row that
 * admits no key gets zeros, and only such a row: one with an admitted score of NaN or
 * +inf, or with nothing but scores of -inf, is NaN.  An infinite or NaN value of an
 * admitted key leaves its element infinite or NaN, whatever the key's weight.  What a
 * key that is not admitted holds has no effect.
 *   q     bf16, element (b, qi, qh, d) at b * q_stride_batch +
 *         qi * q_stride_token + qh * q_stride_head + d, 16-byte aligned rows
 *   mask  uint8/bool, element (b, qi, s) at b * mask_stride_batch +
 *         qi * mask_stride_query + (s - (keys - mask_keys))
 *   out   bf16 [batch, queries, q_heads, head_dim], contiguous
 *   workspace  16-byte aligned device memory of at least
 *         sf_block_attention_workspace bytes, in use until the call's kernels
 *         have run; with less (or NULL) the keys of a call are not split.
 */
int64_t sf_block_attention_workspace(int batch, int queries, int keys,
                                     int q_heads, int kv_heads, int head_dim);
/*
 * Query rows of a KV head that a workgroup takes in such a call: 16 (straight from the
 * cache) or 256 (tiles shared in LDS), 0 for shapes that the call refuses.
 */
int sf_block_attention_rows(int batch, int queries, int keys, int q_heads,
                            int kv_heads, int head_dim);
int sf_block_attention(const sf_kv_cache *cache, int batch, int kv_heads,
                       int keys, const void *q, int64_t q_stride_batch,
                       int64_t q_stride_head, int64_t q_stride_token,
                       int queries, int q_heads, const uint8_t *mask,
                       int64_t mask_stride_batch, int64_t mask_stride_query,
                       int mask_keys, float scale, void *out, void *workspace,
                       int64_t workspace_bytes, sf_stream_t stream);

/*
 * K11: rotary positions of queries and keys.  For pair i of a head's first
 * rotary_dim elements, (a, b) = elements (i, i + rotary_dim / 2), or
 * (2 i, 2 i + 1) if interleaved:
 *   angle = position * turns[i]  (in turns, fp64, reduced before its rounding)
 *   (a, b) -> factor * (a cos - b sin, b cos + a sin)
 * in fp32 with one rounding; the other elements are copied.
 *   x (q and k)  dtype [batch, tokens, heads, head_dim], element (b, t, h, d)
 *                at b * stride_batch + t * stride_token + h * stride_head + d
 *   positions    int64, (b, t) at b * position_stride + t (0: one row for all)
 *   turns        fp64 [rotary_dim / 2], |position * turns| < 2^51
 *   out          dtype [batch, heads, tokens, head_dim], contiguous
 * dtype: SF_BF16, SF_F16 or SF_F32; rotary_dim even, <= head_dim <= 1024;
 * batch * tokens < 2^27.
 */
#define SF_BF16 0
#define SF_F16 1
#define SF_F32 2
int sf_rotary(int dtype, const void *q, int64_t q_stride_batch,
              int64_t q_stride_token, int64_t q_stride_head, int q_heads,
              const void *k, int64_t k_stride_batch, int64_t k_stride_token,
              int64_t k_stride_head, int k_heads, const int64_t *positions,
              int64_t position_stride, const double *turns, float factor,
              int batch, int tokens, int head_dim, int rotary_dim,
              int interleaved, void *q_out, void *k_out, sf_stream_t stream);

/*
 * K12: rules on logits.  With n = counts[v] + occurrences of v in paths[r]
 * (entries outside [0, vocab) count for nothing), each step rounded to fp32:
 *   y = x                                        if n == 0
 *   y = (x < 0 ? x * repetition : x / repetition)
 *       - ((frequency * n) + presence)           otherwise
 *   y = y + bias[v]                              with a bias
 *   y = -inf                                     where allowed has a 0 bit
 *   x        dtype [rows, vocab], row stride logits_stride
 *   counts   int32 [vocab] or NULL
 *   paths    int32 [rows, path_length], contiguous, or NULL
 *   bias     fp32, element (r, v) at r * bias_stride + v, or NULL
 *   allowed  int32 words, bit v % 32 of word r * allowed_stride + v / 32, or NULL
 *   out      dtype [rows, vocab], row stride out_stride: y rounded to dtype
 *            (may equal logits), or NULL
 *   tokens   int64 [rows]: the lowest v of the largest y (fp32, a NaN above all;
 *            -1 where no y is above -inf), or NULL
 *   workspace  device memory of sf_logit_rules_workspace bytes (with tokens)
 */
int64_t sf_logit_rules_workspace(int rows, int vocab);
int sf_logit_rules(int dtype, const void *logits, int64_t logits_stride,
                   int rows, int vocab, const int32_t *counts,
                   const int32_t *paths, int path_length, float repetition,
                   float presence, float frequency, const float *bias,
                   int64_t bias_stride, const int32_t *allowed,
                   int64_t allowed_stride, void *out, int64_t out_stride,
                   int64_t *tokens, void *workspace, int64_t workspace_bytes,
                   sf_stream_t stream);

/*
 * K13: microscaled values.  32 neighbours of a row share the scale 2^e, held
 * as the byte e + 127, e the least integer from -127 up at which no value
 * rounds past the type's largest; values are rounded to nearest, ties to even.
 * A block with an infinity or a NaN has the byte 255 and reads as NaN.
 * With tiles = ceil(dim / 128), quads = ceil(dim / 512):
 *   held 0  rows in e4m3: codes [rows, tiles * 128] (zeros behind the row's
 *           end), scales [rows, quads * 16], the byte of block b (0..3) of tile
 *           t at t / 4 * 16 + b * 4 + t % 4
 *   held 1  a weight in e2m1: codes [R][tiles][4][16][16] with R = 2 * ceil(rows /
 *           32): 16 bytes of block b and row r of row tile and tile, the first of
 *           two values in the low half; scales [R][quads][4][16][4], the
 *           byte of tile t in t % 4; rows behind the last are zeros
 * Bytes of the last quad's missing tiles count for nothing.
 *   dtype       0 bf16, 1 fp16, 2 fp32
 *   x           [rows, dim], row stride row_stride; batch of them (held 1 only)
 *               at batch_stride elements, the outputs at codes_batch_stride and
 *               scales_batch_stride bytes
 * codes 16-byte and scales 4-byte aligned.  dim <= 2^30.
 */
int sf_mx_quantize(int dtype, const void *x, int64_t row_stride,
                   int64_t batch_stride, int rows, int dim, int batch,
                   int held, void *codes, int64_t codes_batch_stride,
                   void *scales, int64_t scales_batch_stride,
                   sf_stream_t stream);

/* The values held, to out [rows, dim] (contiguous, dtype as above). */
int sf_mx_values(int held, const void *codes, const void *scales, int rows,
                 int dim, int dtype, void *out, sf_stream_t stream);

/*
 * K14: the residual's addition and RMSNorm, with an 8-bit output.
 *   s = x + residual                   rounded to dtype (x without a residual)
 *   y = s * r * weight                 fp32; r = fp32(1 / sqrt(mean(s^2) + eps)),
 *                                      the mean in 64 bits
 *   sum = s, normed = y rounded to dtype, codes and scales = y in e4m3 (K13)
 * x and residual [rows, dim] with row strides; the outputs contiguous, each of
 * them NULL if not wanted (sum needs a residual; codes and scales go together).
 * Fewer than 2^24 rows, 2^26 of up to 512 columns.
 */
int sf_add_rms_norm(int dtype, const void *x, int64_t x_stride,
                    const void *residual, int64_t residual_stride, int rows,
                    int dim, const void *weight, double eps, void *sum,
                    void *normed, void *codes, void *scales,
                    sf_stream_t stream);

/*
 * K15: out[m, n] = T(sum_k x[m, k] w[n, k] + bias[n]), fp32 sums.
 *   x_dtype   3: rows in e4m3 (K13), x_scales theirs; 0 bf16 or 1 fp16: rows of
 *             row stride x_stride, rounded to e4m3 here
 *   workspace 16-byte aligned, rows * (tiles * 128 + quads * 16) bytes as K13 has
 *             them, for rows that are rounded beforehand.  NULL where
 *             sf_mx_linear_workspace is 0 (-1: an unsupported shape) and, for
 *             x_dtype 0 and 1, x is 16-byte aligned and x_stride a multiple of 8
 *   codes, scales   a weight in e2m1 [out_features, dim]
 *   bias      [out_features] of out_dtype, or NULL
 *   out_dtype 0 bf16, 1 fp16, whatever x_dtype; out has row stride out_stride
 * codes, scales and, for x_dtype 3, x and x_scales 16-byte aligned; rows <= 2^20,
 * dim <= 2^24, out_features <= 2^28, and fewer than 2^24 blocks of 128 rows by 256
 * outputs.
 */
int sf_mx_linear(int x_dtype, const void *x, const void *x_scales,
                 int64_t x_stride, int rows, int dim, const void *codes,
                 const void *scales, int out_features, const void *bias,
                 int out_dtype, void *out, int64_t out_stride,
                 void *workspace, sf_stream_t stream);
int64_t sf_mx_linear_workspace(int x_dtype, int rows, int dim,
                               int out_features);

/*
 * K16: K3 with the experts' weights in microscaled 4 bits, over every expert
 * e < num_experts that has rows and, with a table, slot_of_expert[e] >= 0.
 *   a       = e4m3(silu(x[t] . gate^T) * (x[t] . up^T))        fp32 up to a
 *   rows[r] = bf16((a . down^T) * route_weights[perm_pos[r]])
 *   x_dtype         3: rows in e4m3; 0: at most SF_MX_RAW_ROWS in bf16, hidden_size and
 *                   x_stride multiples of 8
 *   slots           records of sf_mx_expert_bytes at slot_stride bytes: the codes
 *                   of gate [I, H], up [I, H], down [H, I] and then their
 *                   scales (held 1), at the byte offsets that
 *                   sf_mx_expert_parts writes (6)
 *   slot_of_expert  device int32 [num_experts], or NULL: expert e in slot e
 *   act, act_scales scratch: rows in e4m3 [tokens * top_k, intermediate_size]
 *   out_rows        bf16 [tokens * top_k, hidden_size]
 * x, x_scales, slots, slot_stride, act and act_scales 16-byte, out_rows 8-byte
 * aligned.
 */
int64_t sf_mx_expert_bytes(int hidden_size, int intermediate_size);
int sf_mx_expert_parts(int hidden_size, int intermediate_size, int64_t *offsets);
int sf_mx_grouped_swiglu(int x_dtype, const void *x, const void *x_scales,
                         int64_t x_stride, const int32_t *perm_pos,
                         const int32_t *offsets, const void *route_weights,
                         int tokens, int top_k, int hidden_size,
                         int intermediate_size, int num_experts,
                         const int32_t *slot_of_expert, const void *slots,
                         int64_t slot_stride, void *act, void *act_scales,
                         void *out_rows, sf_stream_t stream);

/*
 * K16 for few tokens, without a dispatch: out[t] = bf16(sum over k of
 * route_weights[t, k] * expert(index[t, k])(x[t])), summed in fp32.
 *   index           int64 [tokens, top_k]; an expert outside 0 .. num_experts - 1
 *                   or in no slot counts for nothing
 *   route_weights   bf16 [tokens, top_k]
 *   out             bf16 [tokens, hidden_size]
 * The rest as above; out 2-byte aligned.
 */
int sf_mx_routed_swiglu(int x_dtype, const void *x, const void *x_scales,
                        int64_t x_stride, const int64_t *index,
                        const void *route_weights, int tokens, int top_k,
                        int hidden_size, int intermediate_size, int num_experts,
                        const int32_t *slot_of_expert, const void *slots,
                        int64_t slot_stride, void *act, void *act_scales,
                        void *out, sf_stream_t stream);

/*
 * A layer's routed experts in one call: sf_mx_routed_swiglu, or sf_dispatch
 * (with the rows' rounding in the same launch), sf_mx_grouped_swiglu's products
 * and the sum over a token's routes, in their order, in fp32.  The routes' rows
 * are kept in fp16 with a power of two for each 32 columns, and the output is
 * rounded once.  Expert e is in slot e.
 *   x_dtype     0 bf16 rows of row stride x_stride, any number and alignment of
 *               them; 3 rows in e4m3 as above
 *   workspace   sf_mx_experts_workspace bytes (-1: an unsupported shape, such as
 *               more than 2^28 routes), 16-byte aligned; calls that may overlap
 *               need one each
 * sf_mx_experts_form says which it is: 1 without a dispatch, 0 with one (-1: an
 * unsupported shape).
 */
int sf_mx_experts_form(int tokens, int top_k, int hidden_size,
                       int intermediate_size, int num_experts);
int64_t sf_mx_experts_workspace(int tokens, int top_k, int hidden_size,
                                int intermediate_size, int num_experts);
int sf_mx_experts(int x_dtype, const void *x, const void *x_scales,
                  int64_t x_stride, const int64_t *index,
                  const void *route_weights, int tokens, int top_k,
                  int hidden_size, int intermediate_size, int num_experts,
                  const void *slots, int64_t slot_stride, void *workspace,
                  void *out, sf_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* SPECFIT_AMD_H */
