/*
 * ane_decode.h -- single-token decode of a Llama-shaped model on MI355X with
 * every matrix product on the Q8_0 kernels of ane_hip.h (G mode).
 *
 * This is the driver around the GGML_OP_MUL_MAT hook: the steps on either
 * side of mul_mat in one decoder layer, as a ggml graph of a Llama model
 * runs them (the reference has SME kernels for these steps:
 * bytecode_interpreter.s:6508 rms_norm, 6617 silu, 6714 rope (adjacent
 * pairs, out[2i] = in[2i] cos - in[2i+1] sin), 11657 flash_attention; its
 * ggml backend routes MUL_MAT to the quantized path,
 * src/ggml-backend/ggml-ane.cpp:119-154):
 *
 *   qkv  = W_qkv . q8(rmsnorm(x) * attn_norm)       fused norm prologue
 *   attn = softmax(rope(q) rope(k)^T / sqrt(d)) v over positions 0..pos (GQA),
 *          k, v of pos appended to the fp16 cache      one fused kernel + combine,
 *                                                    which also emits q8(attn)
 *   x    = x + W_o . q8(attn)                        fused residual epilogue
 *   h    = q8(silu(gate) * up), gate|up = W_gate_up . q8(rmsnorm(x) * ffn_norm)
 *                                                    fused norm prologue and
 *                                                    SiLU/quantize epilogue
 *   x    = x + W_down . h                            fused residual epilogue
 *
 * q8(v) is the Q8 activation form of the G mode: per 32-block, amax/127 as
 * the fp32 scale and the values rounded to int8 (bytecode_interpreter.s
 * 0x19 arithmetic), stored as qx [K/32][32] int8 followed by dx [K/32] fp32.
 *
 * Layouts: weights are Q8_0 rows (ggml block layout) with the output
 * features as rows: W_qkv rows [q heads | k heads | v heads], W_gate_up rows
 * gate and up interleaved in groups of 32 (gate 0..31, up 0..31, gate
 * 32..63, up 32..63, ...), so that one workgroup owns both halves of every
 * 32-value block of SiLU(gate) * up.  KV cache: fp16 [n_kv_heads][ctx][head_dim].  RoPE table:
 * fp32 [ctx][head_dim/2][2] = (cos, sin) of pos * base^(-2i/head_dim),
 * applied to adjacent pairs (x[2i], x[2i+1]).  All pointers are device
 * memory; the layer array itself is host memory.
 */
#ifndef ANE_DECODE_H
#define ANE_DECODE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

struct ane_decode_config {
    uint32_t n_layers;
    uint32_t hidden;      /* model width (4096; a multiple of 256)         */
    uint32_t ffn;         /* feed-forward width (14336; a multiple of 256) */
    uint32_t n_heads;     /* query heads (32)                   */
    uint32_t n_kv_heads;  /* key/value heads (8)                */
    uint32_t head_dim;    /* 128 (the only supported value)     */
    uint32_t ctx;         /* KV cache capacity in positions (at most 2^20) */
    float eps;            /* RMSNorm epsilon                    */
};

struct ane_decode_layer {
    const void* w_qkv;      /* Q8_0 [(n_heads + 2 n_kv_heads) head_dim][hidden] */
    const void* w_o;        /* Q8_0 [hidden][n_heads head_dim]                  */
    const void* w_gate_up;  /* Q8_0 [2 ffn][hidden], gate/up in 32-row groups    */
    const void* w_down;     /* Q8_0 [hidden][ffn]                               */
    const float* attn_norm; /* [hidden]                                         */
    const float* ffn_norm;  /* [hidden]                                         */
    uint16_t* k_cache;      /* fp16 [n_kv_heads][ctx][head_dim]                 */
    uint16_t* v_cache;      /* fp16 [n_kv_heads][ctx][head_dim]                 */
};

/* Device workspace bytes for ane_decode_token (256-byte aligned sections). */
size_t ane_decode_workspace_size(const struct ane_decode_config* cfg);

/* One token at position pos (< ctx) through every layer: x (fp32 [hidden],
 * the residual stream) is updated in place, and k/v of pos are written into
 * each layer's cache; positions 0..pos of the caches are attended to.
 * Every step's preconditions are checked before the first launch (weights
 * 16-byte aligned, the products' LDS and rows-per-wave limits), so an error
 * return leaves x and the caches untouched.
 * Asynchronous on stream; returns an ane_status. */
int ane_decode_token(const struct ane_decode_config* cfg, const struct ane_decode_layer* layers,
                     const float* rope_table, uint32_t pos, float* x, void* workspace,
                     size_t workspace_bytes, void* stream);

/* The steps of ane_decode_token, for tests and for callers that schedule
 * them differently.  All asynchronous on stream. */

/* Q8_0 matvec (G mode, one token) with optional fusions: norm_w != NULL
 * applies x' = x * inv_rms(x) * norm_w before quantizing (inv_rms =
 * 1/sqrt(fl(fl(sum x^2 / K) + eps)), sum in fp64); residual != NULL adds
 * residual[n] to each output (residual may equal y). */
int ane_hip_q8_0_matvec_fused(uint32_t N, uint32_t K, const float* x, const float* norm_w, float eps,
                              const void* W, const float* residual, float* y, void* stream);

/* y = W . xq (+ residual) with xq already in the Q8 activation form (16-byte
 * aligned, K/32 * 36 bytes); bit-identical to ane_hip_q8_0_matvec_fused on
 * the fp32 vector xq was quantized from. */
int ane_hip_q8_0_matvec_q8(uint32_t N, uint32_t K, const void* xq, const void* W, const float* residual,
                           float* y, void* stream);

/* The gate|up product with SiLU*up fused into its epilogue: W has 2F rows,
 * gate and up interleaved in 32-row groups (rows 64k..64k+31 = gate rows
 * 32k.., rows 64k+32..64k+63 = up rows 32k..); with g|u = W . q8(rmsnorm(x)
 * * norm_w) (as ane_hip_q8_0_matvec_fused), xq = q8(silu(g) * u) in the Q8
 * activation form (F/32 * 36 bytes, 16-byte aligned, F % 32 == 0):
 * bit-identical to ane_hip_q8_0_matvec_fused + ane_hip_silu_mul_quant on
 * the de-interleaved output. */
int ane_hip_q8_0_gate_up_silu_quant(uint32_t F, uint32_t K, const float* x, const float* norm_w, float eps,
                                    const void* W, void* xq, void* stream);

/* y = W . q8(silu(gu[0..K)) * gu[K..2K)) (+ residual), silu(g) = g / (1 + e^-g):
 * the down projection with SiLU * up fused into its activation prologue;
 * bit-identical to ane_hip_silu_mul followed by ane_hip_q8_0_matvec_fused. */
int ane_hip_q8_0_matvec_silu(uint32_t N, uint32_t K, const float* gu, const void* W, const float* residual,
                             float* y, void* stream);

/* RoPE on the q and k heads of qkv (in place for q), then k and v of this
 * position converted to fp16 into the caches. */
int ane_hip_rope_kv_append(const struct ane_decode_config* cfg, float* qkv, const float* rope_table,
                           uint32_t pos, uint16_t* k_cache, uint16_t* v_cache, void* stream);

/* out[h] = softmax(q[h] . K[g]^T / sqrt(head_dim)) V[g] over positions
 * 0..len-1, g = h / (n_heads / n_kv_heads).  q: fp32 [n_heads][head_dim].
 * Two launches: per (kv head, chunk of the context) partial results, then a
 * merge per query head. */
size_t ane_hip_attention_workspace_size(const struct ane_decode_config* cfg);
int ane_hip_attention_decode(const struct ane_decode_config* cfg, const float* q, const uint16_t* k_cache,
                             const uint16_t* v_cache, uint32_t len, float* out, void* workspace,
                             size_t workspace_bytes, void* stream);

/* ane_hip_attention_decode at len = pos + 1 on unrotated q and k: RoPE of q
 * and k (as ane_hip_rope_kv_append) and the fp16 append of k and v at pos
 * happen inside the attention kernel; same results, one launch fewer.
 * out_q8 (optional, 16-byte aligned): out in the Q8 activation form too. */
int ane_hip_attention_decode_rope(const struct ane_decode_config* cfg, const float* qkv, const float* rope_table,
                                  uint32_t pos, uint16_t* k_cache, uint16_t* v_cache, float* out, void* out_q8,
                                  void* workspace, size_t workspace_bytes, void* stream);

/* h[i] = silu(gu[i]) * gu[n + i], i < n. */
int ane_hip_silu_mul(uint32_t n, const float* gu, float* h, void* stream);

/* xq = q8(h) for h as ane_hip_silu_mul computes it (n % 32 == 0, xq 16-byte
 * aligned, n/32 * 36 bytes). */
int ane_hip_silu_mul_quant(uint32_t n, const float* gu, void* xq, void* stream);

/* The build's RMSNorm on its own, one row: out = fl(fl(x * inv) * w),
 * inv = 1/sqrtf((float)(ss / K) + eps) with ss the fp64 sum of squares in
 * the fixed order the fused products use, so the output is bit-identical to
 * the normalised activation those kernels quantize.  K % 32 == 0,
 * K <= 2^19, x 16-byte aligned. */
int ane_hip_rms_norm(uint32_t K, const float* x, const float* w, float eps, float* out, void* stream);

/* out = fl(a + b), n elements (out may alias a or b). */
int ane_hip_add_fp32(uint32_t n, const float* a, const float* b, float* out, void* stream);

/* The reference's decode-step handlers in their exact fp32 operation
 * sequence (bytecode_interpreter.s; the estimates per the Arm ARM
 * pseudocode of FRSQRTE / FRECPE):
 *   0x51 rms_norm_fp32 (:6508-6565): rows x dim, out may alias in;
 *   0x54 silu_fp32     (:6617-6713): count elements;
 *   0x55 rope_fp32     (:6714-6912): rows x dim (each row rotated at pos,
 *        adjacent pairs, ratio theta^(2/dim));
 *   0x56 softmax_fp32  (:6913-7009): rows x dim, out may alias in.
 * The handlers loop in 16-lane vectors with no tail, so stream_exec refuses
 * dim % 16 != 0 for 0x51, 0x54 and 0x56; these kernel entries accept any
 * dim, a short last vector contributing nothing (identical for multiples
 * of 16). */
int ane_hip_rms_norm_fp32(uint32_t rows, uint32_t dim, float eps, const float* in, const float* w, float* out,
                          void* stream);
int ane_hip_silu_fp32(uint64_t count, const float* in, float* out, void* stream);
int ane_hip_rope_fp32(uint32_t rows, uint32_t dim, uint32_t pos, float theta, const float* in, float* out,
                      void* stream);
int ane_hip_softmax_fp32(uint32_t rows, uint32_t dim, const float* in, float* out, void* stream);

/* One token through the ggml backend (include/ggml-ane-hip.h): each layer's
 * four products are GGML_OP_MUL_MAT nodes computed by
 * ane_ggml_compute_forward on the backend's stream, with the steps around
 * them as separate kernels.
 *   ANE_DECODE_ARITH_BUILD: the products in G mode and the steps in the
 *     arithmetic of ane_decode_token (canonical fp64 RMSNorm, the RoPE table,
 *     the chunked attention, expf SiLU): x and the caches come out
 *     bit-identical to ane_decode_token's;
 *   ANE_DECODE_ARITH_REFERENCE: the products in R mode (opcode 0x57, what the
 *     reference hook runs) and the steps in the handlers' arithmetic:
 *     rms_norm_fp32, rope_fp32 at rope_theta on q and k (dim 128), an
 *     attention of 16-lane fma dot products scaled by fl(1/sqrt(128)),
 *     softmax_fp32 over positions 0..pos and 16-lane fma sums over the
 *     values, silu_fp32 times up, fp32 residual adds.
 * Sets the backend's Q8_0 mode accordingly.  x 16-byte aligned; workspace
 * from ane_decode_ggml_workspace_size (256-byte aligned).  Asynchronous. */
#define ANE_DECODE_ARITH_BUILD 0
#define ANE_DECODE_ARITH_REFERENCE 1
struct ane_ggml_backend;
size_t ane_decode_ggml_workspace_size(const struct ane_decode_config* cfg);
int ane_decode_token_ggml(const struct ane_decode_config* cfg, const struct ane_decode_layer* layers,
                          const float* rope_table, float rope_theta, uint32_t pos, float* x, void* workspace,
                          size_t workspace_bytes, struct ane_ggml_backend* backend, int arith);

/* ------------------------------------------------ paged cache, batches
 *
 * Several sequences on one K/V cache whose positions live in pages, so that
 * sequences grow without reserving ctx positions each and can share the pages
 * of a common prefix.  No counterpart in the reference.
 *
 * Sequence s holds positions 0 .. kv_len[s]-1; position p is row p % page_size
 * of page page_table[s][p / page_size].  Entries of the table past the
 * sequence's pages hold ANE_NO_PAGE.  page_refs[i] counts the table entries
 * that name page i; 0 means the page is free.  Every array is device memory
 * and is read when the kernels run, so a captured call follows the lengths and
 * tables of its replay.
 *
 * A page number outside the pool reads as zeros and is never written, and a
 * length past max_pages * page_size counts as that many positions: a broken
 * table gives wrong results, never an access outside the pool.  All calls are
 * asynchronous on stream; pointers must belong to the current device. */
#define ANE_NO_PAGE 0xffffffffu

/* Element types of activations (ggml's numbers). */
#define ANE_TYPE_F32 0
#define ANE_TYPE_F16 1

struct ane_paged_cache {
    uint32_t n_layers;
    uint32_t n_heads;     /* query heads: a multiple of n_kv_heads, at most 128 each */
    uint32_t n_kv_heads;
    uint32_t head_dim;    /* 64 or 128 */
    uint32_t page_size;   /* positions a page: a multiple of 16, at most 2^20 */
    uint32_t n_pages;     /* pages in the pool, below 2^31 */
    uint32_t n_seqs;      /* rows of page_table */
    uint32_t max_pages;   /* entries a row; max_pages * page_size at most 2^30 */
    uint16_t* k_pages;    /* fp16 [n_layers][n_pages][n_kv_heads][page_size][head_dim], 16-byte aligned */
    uint16_t* v_pages;    /* the same shape */
    uint32_t* page_table; /* [n_seqs][max_pages] */
    uint32_t* kv_len;     /* [n_seqs] */
    uint32_t* page_refs;  /* [n_pages]; NULL where only attention or append is called */
};

/* The batched calls below take n sequences: row i of the batch is sequence
 * seqs[i] of the cache (seqs NULL: sequence i; a number outside the cache is a
 * sequence without positions).  Packed rows: the new tokens of batch row i are
 * rows q_start[i] .. q_start[i+1]-1 of the activations (ascending, q_start[n]
 * <= n_tokens), its last positions: token t of m sits at kv_len - m + t.
 * q_start NULL: one new token a row.  Rows from q_start[n] on are left as they
 * were.  At most 2^23 tokens a call; attention also refuses a batch of more
 * workgroups than a launch takes (2^23: some 2^20 sequences on 8 kv heads).
 * Strides are in elements from one token to the next; a token's heads are
 * contiguous.  q, k, v, q_out and out are 16-byte aligned and their strides
 * multiples of 16 bytes. */

/* RoPE of q and k (adjacent pairs, the fp32 operations of
 * ane_hip_rope_kv_append) and the append of k and v, rounded to fp16, to the
 * pages of one layer.  in_type: of q, k and v; q_out: the rotated q in
 * q_out_type (may be q itself when the types and strides agree).  q and q_out
 * NULL: k and v only.  rope_table NULL: no rotation; else fp32 [rope_len]
 * [head_dim/2][2].  A token whose position is negative or not below rope_len is
 * not appended and its q_out row is zeros.
 * kv_len counts the new tokens already (ane_hip_pages_reserve).  A sequence may
 * be in the batch once; appending to a page that two sequences hold changes
 * both. */
int ane_hip_paged_rope_append(const struct ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                              const uint32_t* q_start, uint32_t n_tokens, int in_type, const void* q,
                              uint64_t q_stride, const void* k, const void* v, uint64_t kv_stride,
                              const float* rope_table, uint32_t rope_len, int q_out_type, void* q_out,
                              uint64_t q_out_stride, void* stream);

/* The same for models that normalise each q and k head, rotate halves or part of
 * a head, or scale the rotation for long contexts: with q_norm and k_norm (fp32
 * [head_dim], each may be NULL) a head becomes x / sqrt(mean(x^2) + eps) * w
 * first; then pair i of its leading rot_dim values (a, b) becomes (a c - b s,
 * a s + b c), c and s = factor * (cos, sin)(position * freqs[i]).  A head's mean
 * square is formed in fp64, so that heads of any fp32 values have their norm.  The
 * angle is formed in fp64, its cosine and sine exact to fp32, the rest in fp32; there
 * is no table and no bound on positions but the cache's.  rope NULL or rot_dim 0: no
 * rotation.  A token at a negative position is not appended and its q_out row is
 * zeros.  Everything else as above. */
struct ane_rope {
    uint32_t rot_dim;    /* a multiple of 16, at most head_dim */
    uint32_t halves;     /* 0: pairs (2i, 2i + 1); else (i, i + rot_dim / 2) */
    const double* freqs; /* device, [rot_dim / 2]: radians a position */
    double factor;       /* above 0, below 1e30; 1 for most models */
};
int ane_hip_paged_norm_rope_append(const struct ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                                   const uint32_t* q_start, uint32_t n_tokens, int in_type, const void* q,
                                   uint64_t q_stride, const void* k, const void* v, uint64_t kv_stride,
                                   const struct ane_rope* rope, const float* q_norm, const float* k_norm, float eps,
                                   int q_out_type, void* q_out, uint64_t q_out_stride, void* stream);

/* Causal attention of packed prompts with grouped heads: for each new token at
 * position p, out[h] = softmax(scale * q[h] . K[g][0..p]^T) V[g][0..p],
 * g = h / (n_heads / n_kv_heads); zeros for a token at a negative position.
 * Keys a token does not see never touch its result, whatever they hold; an
 * infinity or NaN it does see may make its result infinite or NaN.
 * type: of q and out.  F32: products of fp32 accuracy: q and the softmax
 * weights enter the matrix cores in fp16 parts that hold 22 bits of q and of
 * the weights that carry a row, and at least 18 of any that matters to it down to
 * 2^-56 of its largest (smaller ones count as multiples of 2^-73 of that).  F16:
 * q and the weights are rounded to fp16 once, the weights to multiples of 2^-30
 * of a row's largest below 2^-20 of it.  Scores, softmax and sums are fp32 in
 * both.  scale: positive,
 * below 1e30.  max_len: a bound on the lengths, which sizes the workspace and
 * the split of long rows (longer sequences are still computed whole); 0 stands
 * for max_pages * page_size.  out may be q when the strides agree.  The
 * workspace (256-byte aligned; NULL when its size is 0) belongs to the call
 * until it has run.  Its size is that of these very arguments: a smaller batch, whose
 * keys are split over more workgroups, may need more, so one kept for several
 * batches has the largest of their sizes. */
size_t ane_hip_attention_prompt_workspace_size(const struct ane_paged_cache* cache, uint32_t n, uint32_t n_tokens,
                                               uint32_t max_len);
int ane_hip_attention_prompt(const struct ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                             const uint32_t* q_start, uint32_t n_tokens, uint32_t max_len, int type, const void* q,
                             uint64_t q_stride, float scale, void* out, uint64_t out_stride, void* workspace,
                             size_t workspace_bytes, void* stream);

/* ane_hip_attention_prompt for models that are not plainly causal.  The new
 * token t of batch row i, at position p, sees the keys j of its sequence with
 *   j <= p, or j < prefix[i]       (prefix NULL: j <= p; a prefix seen from both sides)
 *   j >= first[t]                  (first NULL: all; the first position of t's document)
 *   p - j < window                 (window 0: all)
 * all three holding, and its score of one is
 *   s = scale * q[h] . K[g][j];  s = softcap * tanh(s / softcap) (softcap 0: as it
 *   is);  s - slopes[h] * |p - j| (slopes NULL: as it is).
 * A token that sees nothing gets zeros; a token at a negative position sees
 * nothing.  first is indexed by packed row, prefix by batch row; a prefix past
 * the length counts as the length, keys that no token of a tile sees are not read.
 * An entry from 2^31 on, a negative one of an int32 array, opens nothing: its first
 * lies behind every key (the token sees none), its prefix is none.
 * softcap: 0, or 2^-20 to 2^20.  Single tokens (q_start NULL) are the decode step.
 * Types, accuracy (of the score before the cap, in fp32) and everything else as
 * above; the cap adds 2^-22 of a capped score (F16: 2^-20).  The workspace is that
 * of the rule (with a window fewer keys are split). */
struct ane_attention_rule {
    float softcap;
    uint32_t window;
    const float* slopes;    /* device, [n_heads], or NULL */
    const uint32_t* first;  /* device, [n_tokens], or NULL */
    const uint32_t* prefix; /* device, [n], or NULL */
};
size_t ane_hip_attention_rule_workspace_size(const struct ane_paged_cache* cache, uint32_t n, uint32_t n_tokens,
                                             uint32_t max_len, const struct ane_attention_rule* rule);
int ane_hip_attention_rule(const struct ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                           const uint32_t* q_start, uint32_t n_tokens, uint32_t max_len,
                           const struct ane_attention_rule* rule, int type, const void* q, uint64_t q_stride, float scale,
                           void* out, uint64_t out_stride, void* workspace, size_t workspace_bytes, void* stream);

/* One new token of each of n sequences (row i of q and out), attending to
 * positions 0 .. kv_len-1 of its sequence; zeros where there are none.
 * With n_groups > 0, batch rows group_start[g] .. group_start[g+1]-1 (device,
 * [n_groups+1], ascending) share their first prefix_len[g] positions (device,
 * [n_groups]): those are read once for the whole group, out of the pages of
 * its first row; rows outside every group share nothing.  A prefix longer than
 * a row's or the first row's length counts as that length.  max_prefix and
 * max_len bound the prefix lengths and the lengths as max_len does above.  The
 * workspace as there. */
size_t ane_hip_attention_shared_workspace_size(const struct ane_paged_cache* cache, uint32_t n, uint32_t n_groups,
                                               uint32_t max_prefix, uint32_t max_len);
int ane_hip_attention_shared(const struct ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                             uint32_t n_groups, const uint32_t* group_start, const uint32_t* prefix_len,
                             uint32_t max_prefix, uint32_t max_len, int type, const void* q, uint64_t q_stride,
                             float scale, void* out, uint64_t out_stride, void* workspace, size_t workspace_bytes,
                             void* stream);

/* Pages.  Requests are device arrays of n entries, at most 65536 a call;
 * free pages are always taken lowest number first, so results do not depend
 * on timing.  served (optional, [n]): 1 for a request carried out, else 0.
 * Calls that change one cache must be ordered (one stream, or events).
 * The workspace (ane_hip_pages_workspace_size bytes, 256-byte aligned) belongs
 * to the call until it has run.
 *
 * reserve: sequence seqs[i] grows to new_len[i] positions (one that is that
 * long already stays as it is).  One for an unknown sequence, past max_pages *
 * page_size or for a sequence an earlier valid one names is refused; the others
 * are served in order, up to the first whose pages the pool does not have: it
 * and all later ones are refused.
 * fork: sequence dst[i], which must be empty, becomes a copy of src[i]: it
 * shares the whole pages and gets its own copy, in every layer, of the rows
 * used in a last, part-filled one, so that appending to either sequence
 * changes no other.  Served in order while the free pages last, as in
 * reserve; refused where dst is unknown, not empty, src itself or named by an
 * earlier valid request, or src is unknown.  A src that is another request's
 * dst counts as empty, as it was.
 * free: the sequences become empty and give their pages up (naming one twice
 * is naming it once).
 * copy: page dst[i] becomes a copy of page src[i] in every layer; a page
 * number outside the pool is skipped.  No dst may occur twice or be a src.
 * compact: the live pages move to the front of the pool (those at or past the
 * live count go, in order, into the free ones before it); page_table_out,
 * page_refs_out (NULL: the cache's own) get the table and counts that go with
 * it, n_live (optional) the number of live pages.  With arrays of their own
 * the cache's table and the moved pages stay readable as before until free
 * pages are written. */
size_t ane_hip_pages_workspace_size(const struct ane_paged_cache* cache);
int ane_hip_pages_reserve(const struct ane_paged_cache* cache, uint32_t n, const uint32_t* seqs,
                          const uint32_t* new_len, uint32_t* served, void* workspace, size_t workspace_bytes,
                          void* stream);
int ane_hip_pages_fork(const struct ane_paged_cache* cache, uint32_t n, const uint32_t* src, const uint32_t* dst,
                       uint32_t* served, void* workspace, size_t workspace_bytes, void* stream);
int ane_hip_pages_free(const struct ane_paged_cache* cache, uint32_t n, const uint32_t* seqs, void* stream);
int ane_hip_pages_copy(const struct ane_paged_cache* cache, uint32_t n, const uint32_t* src, const uint32_t* dst,
                       void* stream);
int ane_hip_pages_compact(const struct ane_paged_cache* cache, uint32_t* page_table_out, uint32_t* page_refs_out,
                          uint32_t* n_live, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------ int8 linear layers of a batch
 *
 * out = (q . w^T) with a scale for each token and each output channel, for T
 * tokens of K values and N output channels.  No counterpart in the reference,
 * whose int8 products have one scale a tensor.  Types are ANE_TYPE_F32 or
 * ANE_TYPE_F16; strides are in elements from one token (row of w) to the next,
 * the values of one are contiguous.  1 <= K < 2^17, T and N at most 65535 * 128,
 * T * N below 2^38, quantized tokens below 2^22 where K > 16384.  All calls are asynchronous on stream; pointers must belong
 * to the current device and be aligned to their elements, q and w (and their
 * strides, which are bytes) to 16 bytes.
 *
 * Weights: int8 rows [N][w_stride], w_stride >= K, each readable up to K rounded
 * up to 16; what stands there past K does not matter.
 * Quantized tokens: int8 rows [T][q_stride], q_stride >= K rounded up to 16,
 * zeros from K up to there.
 *
 * quantize_tokens: y = x, or with norm_w (fp32 [K]) y = fl(fl(x * inv) * norm_w),
 * inv as ane_hip_rms_norm has it; scales[t] = fl(max|y| / 127), q = y *
 * fl(fl(1 / max|y|) * 127) rounded to even, at most 127 in magnitude.  A token of zeros has scale
 * 1; one whose y holds an infinity or NaN a scale that is not finite, and its row
 * of any product is NaN.
 * dense_i8_scaled: out[t][n] = fl(fl((float)sum q w * q_scales[t]) * w_scales[n])
 * + bias[n] + residual[t][n], one rounding a step, the sum exact; bias (fp32 [N])
 * and residual (out's type; may be out itself with its stride) may be NULL.  It has
 * no workspace and so never splits K over workgroups, as linear_i8 does.
 * Weights (and quantized tokens) from 2 GiB on, N * w_stride >= 2^31, go through the
 * one kernel with 64-bit offsets, which takes 1.6 to 3.6 times as long.
 * linear_i8: both, q and scales in the workspace (256-byte aligned; it belongs to
 * the call until it has run).  The size for T tokens is enough for fewer of them as
 * well.  The same bits as the two calls.  out may lie in x, otherwise outputs share
 * no memory with what is read. */
int ane_hip_quantize_tokens(uint32_t T, uint32_t K, int type, const void* x, uint64_t x_stride, const float* norm_w,
                            float eps, int8_t* q, uint64_t q_stride, float* scales, void* stream);
int ane_hip_dense_i8_scaled(uint32_t T, uint32_t N, uint32_t K, const int8_t* q, uint64_t q_stride,
                            const float* q_scales, const int8_t* w, uint64_t w_stride, const float* w_scales,
                            const float* bias, const void* residual, uint64_t residual_stride, int out_type, void* out,
                            uint64_t out_stride, void* stream);
size_t ane_hip_linear_i8_workspace_size(uint32_t T, uint32_t N, uint32_t K);
int ane_hip_linear_i8(uint32_t T, uint32_t N, uint32_t K, int type, const void* x, uint64_t x_stride,
                      const float* norm_w, float eps, const int8_t* w, uint64_t w_stride, const float* w_scales,
                      const float* bias, const void* residual, uint64_t residual_stride, int out_type, void* out,
                      uint64_t out_stride, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ANE_DECODE_H */
