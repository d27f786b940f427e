/*
 * ssa_hip.h -- C ABI of libssa_hip.so, the MI355X (gfx950) implementation of
 * the SSA forward hot path (codebook routing, inverted index, candidate
 * selection, gathered exact attention).
 *
 * Conventions
 *   - Every pointer is device memory owned by the caller (the PyTorch caching
 *     allocator in ssa_amd).  The library allocates nothing and never
 *     synchronises: each call enqueues kernels on `stream` (a hipStream_t;
 *     NULL = the default stream) and returns.
 *   - Strides are in ELEMENTS; the last (feature) dimension is contiguous.
 *   - Every function returns SSA_OK (0) or an error status; argument checks run
 *     on the host before any launch.  ssa_last_error() gives the detail of the
 *     last failure on the calling thread.
 *   - Selections are bit-exact with the CPU oracle (oracle/ssa_oracle.c):
 *     fp32 scoring in one canonical fmaf order, ties to the lowest index.
 *
 * Reference interfaces replaced (chenxingqiang/SSA):
 *   CodebookRouter.forward        ssa/router.py:73-149
 *     _select_candidates          ssa/router.py:151-214
 *     _build_candidate_mask       ssa/router.py:216-259
 *     get_code_assignment         ssa/router.py:261-275
 *   sparse_exact_attention        ssa/attention.py:12-115
 */
#ifndef SSA_HIP_H
#define SSA_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* status codes */
#define SSA_OK 0
#define SSA_ERR_INVALID_ARGUMENT 1
#define SSA_ERR_UNSUPPORTED 2
#define SSA_ERR_WORKSPACE 3
#define SSA_ERR_HIP 4

/* element types of q / k / v / attention output */
#define SSA_DTYPE_F32 0
#define SSA_DTYPE_BF16 1
/* of pages of a K/V cache, beside the two above: 8-bit codes with a scale a row */
#define SSA_DTYPE_I8 2
#define SSA_DTYPE_E4M3 3

/* index element types */
#define SSA_INDEX_I32 0
#define SSA_INDEX_I64 1

/* candidate masks for ssa_select */
#define SSA_MASK_NONE 0   /* causal_mask=None: every key is eligible            */
#define SSA_MASK_CAUSAL 1 /* build_causal_mask(n): key j eligible iff j <= i     */
#define SSA_MASK_DENSE 2  /* any bool [n][n] mask: eligible iff mask[i][j] != 0  */

int ssa_version(void);
const char* ssa_status_str(int status);
const char* ssa_last_error(void);

/* rotary-embedding angle rows for ssa_rope */
#define SSA_ROPE_BY_POSITION 0 /* table row = token position (Hugging Face Qwen2)        */
#define SSA_ROPE_BY_HEAD 1     /* table row = head index (SSAAttention's apply_rope call) */

/* ---- layer prologue: rotary embedding ----------------------------------- */

/* Rotary embedding of q or k rows: features j < rot rotate in pairs
 * (j, j + rot/2), out = x * cos + rotate_half(x) * sin, and features j >= rot
 * pass through.  Replaces apply_rope (ssa/utils.py:7-41) as SSAAttention calls
 * it on [n, heads, d] per batch element (ssa/ssa_layer.py:115-120: rot = d/2,
 * angle row = head index, table freqs[:, :d/2]) and Hugging Face's
 * apply_rotary_pos_emb in the Qwen2 path (training/train_qwen.py:134-135:
 * rot = d, angle row = position, the model's cos/sin tables).
 *   x   [batch][n][h][d] strides (x_sb, x_sn, x_sh), type dtype
 *   cos_table, sin_table  [batch or 1][table_rows][>= rot], row stride t_sr,
 *       batch stride t_sb (0 = one table for every batch element), type table_dtype
 *   angle_axis  SSA_ROPE_BY_POSITION (row = token i) or SSA_ROPE_BY_HEAD (row = head)
 *   inverse != 0 applies the transpose of the rotation (the backward)
 *   out [batch][n][h][d] strides (o_sb, o_sn, o_sh), type out_dtype; out == x
 *       (same strides and type) rotates in place and leaves features >= rot alone.
 * Arithmetic matches torch's ops: bf16 x with bf16 tables rounds every product
 * and the sum to bf16; otherwise fp32 intermediates, the result rounded once. */
int ssa_rope(const void* x, int dtype, int64_t batch, int64_t n, int h, int d, int64_t x_sb,
             int64_t x_sn, int64_t x_sh, const void* cos_table, const void* sin_table,
             int table_dtype, int64_t t_sb, int64_t t_sr, int64_t table_rows, int rot,
             int angle_axis, int inverse, void* out, int out_dtype, int64_t o_sb, int64_t o_sn,
             int64_t o_sh, void* stream);

/* ---- stage (a): routing ------------------------------------------------- */

/* Routing vectors: out[b][h][i] = normalize(mean_{gg<group}(x[b][i][h*group+gg] . w^T)).
 * Replaces the W_qr / W_kr projection, the GQA mean and F.normalize of
 * ssa/router.py:102-117 (group = h_q/h_kv for queries, 1 for keys).
 *   x   [batch][n][h_in][d]  strides (x_sb, x_sn, x_sh)
 *   w   fp32 [d_s][d] contiguous (nn.Linear weight)
 *   out fp32 [batch][h_in/group][n][d_s] contiguous */
int ssa_route_vectors(const void* x, int dtype, int64_t batch, int64_t n, int h_in, int group,
                      int d, int64_t x_sb, int64_t x_sn, int64_t x_sh, const float* w, int d_s,
                      float* out, void* stream);

/* Row-wise F.normalize(x, dim=-1) of a fp32 [rows][d_s] matrix (the codebook,
 * ssa/router.py:118). */
int ssa_normalize_rows(const float* x, int64_t rows, int d_s, float* out, void* stream);

/* Codebook scoring and top-`top` codes per row (score desc, code asc).
 * Replaces einsum("shd,hcd->shc") / temperature and topk of ssa/router.py:121-130
 * (keys, top = b) and :141 (queries, top = a).
 *   xhat  fp32 [batch][h][rows][d_s]; chat fp32 [h][n_c][d_s]
 *   codes int32 [batch][h][rows][top]
 * With a workspace (ssa_code_topk_workspace_bytes) and top <= 32, d_s <= 32,
 * scores are screened on the matrix cores (bf16) with a proven error bound and
 * the survivors rescored exactly; workspace = NULL scores every code exactly.
 * Both give identical codes. */
size_t ssa_code_topk_workspace_bytes(int64_t batch, int h, int64_t rows, int n_c);
int ssa_code_topk(const float* xhat, int64_t batch, int h, int64_t rows, const float* chat,
                  int n_c, int d_s, float temperature, int top, int32_t* codes, void* workspace,
                  size_t workspace_bytes, void* stream);

/* Stage (a) end to end: q_codes = top-a query codes, k_codes = top-b key codes.
 * Replaces ssa/router.py:102-141.  The workspace holds the normalized routing
 * vectors and codebook (ssa_route_workspace_bytes).
 *   q [batch][n][h_q][d], k [batch][n][h_kv][d]; codebook fp32 [h_kv][n_c][d_s]
 *   q_codes int32 [batch][h_kv][n][a]; k_codes int32 [batch][h_kv][n][b] */
size_t ssa_route_workspace_bytes(int64_t batch, int64_t n, int h_kv, int n_c, int d_s);
int ssa_route_codes(const void* q, const void* k, int dtype, int64_t batch, int64_t n, int h_q,
                    int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb,
                    int64_t k_sn, int64_t k_sh, const float* w_qr, const float* w_kr,
                    const float* codebook, int d_s, int n_c, int a, int b, float temperature,
                    int32_t* q_codes, int32_t* k_codes, void* workspace, size_t workspace_bytes,
                    void* stream);

/* ---- stage (b): inverted index ------------------------------------------ */

/* Bucket c of head h lists every key j with c in k_codes[b][h][j][:], ascending.
 * No reference counterpart: it replaces the O(n^2) broadcast compare of
 * _build_candidate_mask (ssa/router.py:241-257) and reproduces its set.
 *   offsets  int32 [batch][h_kv][n_c+1]; postings int32 [batch][h_kv][n*b] */
size_t ssa_index_workspace_bytes(int64_t batch, int64_t n, int h_kv, int b, int n_c);
int ssa_build_index(const int32_t* k_codes, int64_t batch, int64_t n, int h_kv, int b, int n_c,
                    int32_t* offsets, int32_t* postings, void* workspace, size_t workspace_bytes,
                    void* stream);

/* Processing order for ssa_sparse_attention's row_order: the query positions of
 * each (batch, kv head) sorted by their smallest code min_t q_codes[b][h][i][t]
 * (stable, so ascending positions within a code).  Rows that share that code
 * share its bucket and much of their candidates, so processing them together
 * keeps the gathered K/V rows in cache.
 * No reference counterpart (the reference has no processing order; results do
 * not depend on it).  q_codes must lie in [0, n_c), as ssa_route_codes writes.
 *   q_codes int32 [batch][h_kv][n][a]; order int32 [batch][h_kv][n] */
size_t ssa_query_order_workspace_bytes(int64_t batch, int64_t n, int h_kv, int n_c);
int ssa_query_order(const int32_t* q_codes, int64_t batch, int64_t n, int h_kv, int a, int n_c,
                    int32_t* order, void* workspace, size_t workspace_bytes, void* stream);

/* ---- stage (c): candidate selection ------------------------------------- */

/* Top-k candidate keys per (query, kv head): union of the query's a buckets,
 * masked, deduplicated, rescored as mean_g(q.k / score_div) in fp32, ranked
 * (score desc, index asc); fewer than k candidates are followed by the lowest
 * non-candidate indices; k > n pads with 0.  Replaces
 * CodebookRouter._select_candidates (ssa/router.py:151-214).
 *   sorted != 0: selected keys by (score desc, index asc), as torch.topk orders
 *                them; sorted == 0: the same set, selected keys ascending (rows
 *                with at most k candidates then need no rescoring).  The filler
 *                and padding are the same in both orders.
 *   out    [batch][n][h_kv][top_k], index type out_index_dtype
 *   mask   (SSA_MASK_DENSE only) uint8 [batch][n][n], strides (mask_sb, mask_si); mask_sb may be 0
 *   stats  (nullable) int32 [batch][h_kv][n][2] = (candidates, postings read
 *          inside the mask window: j <= i when causal, all otherwise)
 *   row_prefix (nullable) int32 [batch][h_kv][n]: X per row such that the
 *          row's indices hold each key of [0, X) exactly once -- the last
 *          filler key + 1 for a row with filler, 0 otherwise (and 0 with k > n
 *          padding).  ssa_sparse_attention takes it to attend those keys in a
 *          dense pass.  No reference counterpart.
 *   workspace (nullable): with it, index order runs one wave per row; a row
 *          with more than k candidates leaves its candidate list in the
 *          workspace, which bf16 inputs with d = 64 or 128 then screen on the
 *          matrix cores (approximate scores with a proven error bound; only the
 *          keys near the k-th score are rescored exactly), and the remaining
 *          such rows (lists that do not fit, other types) take an exact
 *          one-block-per-row pass.  ssa_select_workspace_bytes(.., top_k) is
 *          the recommended size, (.., 0) the minimum (no lists).  Without a
 *          workspace, one block per row.  Results are identical in every case.
 *   row_order (nullable) int32 [batch][h_kv][n]: the order in which query rows
 *          are processed, as for ssa_sparse_attention (ssa_query_order groups
 *          rows that share buckets and candidate keys, which then hit in
 *          cache).  Results do not depend on it; a row never listed is not
 *          written and an entry outside [0, n) is skipped.
 * Limits: top_k <= 4096, g = h_q/h_kv <= 16, d <= 256 (d % 8 == 0), n < 2^31. */
size_t ssa_select_workspace_bytes(int64_t batch, int64_t n, int h_kv, int top_k);

/* Where ssa_select places its regions inside a workspace of workspace_bytes
 * (no reference counterpart; for tests and for callers that size or share
 * workspaces).  layout[11] receives byte offsets of the counter block, the
 * exact-pass row list, the screened-row entries, the per-row error bounds,
 * the candidate lists and their approximate scores, then the entries per
 * shard, the list entries per shard (0 = no screen), the shard count, the
 * counter block's size and the offset of the per-row candidate counts (one
 * int32 per row, between the error bounds and the lists).  Nothing is
 * launched or dereferenced. */
int ssa_select_workspace_layout(int64_t batch, int64_t n, int h_kv, size_t workspace_bytes,
                                int screen, int64_t* layout);

int ssa_select(const void* q, const void* k, int dtype, int64_t batch, int64_t n, int h_q,
               int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb,
               int64_t k_sn, int64_t k_sh, const int32_t* q_codes, int a, const int32_t* offsets,
               const int32_t* postings, int n_c, int b, int top_k, int mask_mode,
               const uint8_t* mask, int64_t mask_sb, int64_t mask_si, float score_div, int sorted,
               const int32_t* row_order, void* out, int out_index_dtype, int32_t* stats,
               int32_t* row_prefix, void* workspace, size_t workspace_bytes, void* stream);

/* ssa_select for a block of n_q query rows at key positions q_pos0 .. q_pos0 +
 * n_q - 1 against all n keys (0 <= q_pos0, q_pos0 + n_q <= n): q, q_codes,
 * out, stats and row_order hold n_q rows ([batch][n_q]..., [batch][h_kv][n_q]...);
 * the causal window and the dense mask use the key position.  n_q = n with
 * q_pos0 = 0 is ssa_select.  No reference counterpart: it serves incremental
 * decoding (new tokens against a key cache, ssa_design.md:225-234) and chunked
 * prefill.  Workspace: ssa_select_workspace_bytes(batch, n_q, h_kv, top_k). */
int ssa_select_block(const void* q, const void* k, int dtype, int64_t batch, int64_t n,
                     int64_t n_q, int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb,
                     int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh,
                     const int32_t* q_codes, int a, const int32_t* offsets,
                     const int32_t* postings, int n_c, int b, int top_k, int mask_mode,
                     const uint8_t* mask, int64_t mask_sb, int64_t mask_si, float score_div,
                     int sorted, const int32_t* row_order, void* out, int out_index_dtype,
                     int32_t* stats, int32_t* row_prefix, void* workspace, size_t workspace_bytes,
                     void* stream);

/* ssa_select_block without a workspace argument: no counterpart in the
 * reference; for callers that cannot allocate (code under HIP graph capture,
 * serving loops, harnesses that forbid hipMalloc).  The workspace is a static
 * device array of ssa_select_noalloc_scratch_bytes() bytes (64 MiB) that the
 * library holds on every device it runs on until the process ends; the call
 * allocates nothing and uses min(that, ssa_select_workspace_bytes(batch, n_q,
 * h_kv, top_k)) of it (rows whose candidate lists do not fit take the exact
 * pass, with identical results).  Shapes whose minimum workspace
 * (ssa_select_workspace_bytes(batch, n_q, h_kv, 0), about 20 bytes per
 * (batch, query row, kv head)) exceeds the array are rejected with
 * SSA_ERR_WORKSPACE.  Every call on one device shares the array: calls that
 * overlap on one device (other streams, other threads) race. */
size_t ssa_select_noalloc_scratch_bytes(void);
int ssa_select_block_noalloc(const void* q, const void* k, int dtype, int64_t batch, int64_t n,
                             int64_t n_q, int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb,
                             int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh,
                             const int32_t* q_codes, int a, const int32_t* offsets,
                             const int32_t* postings, int n_c, int b, int top_k, int mask_mode,
                             const uint8_t* mask, int64_t mask_sb, int64_t mask_si,
                             float score_div, int sorted, const int32_t* row_order, void* out,
                             int out_index_dtype, int32_t* stats, int32_t* row_prefix, void* stream);

/* ---- incremental decoding ----------------------------------------------- */

/* One decoding step for m new tokens against a key/value cache: no reference
 * counterpart (the reference runs whole sequences; ssa_design.md:225-234
 * describes decode-time routing against the cached keys' inverted index,
 * "maintained incrementally, avoiding re-scanning the full KV cache").
 * The caller owns the cache state:
 *   k_cache, v_cache [batch][max_len][h_kv][d] (strides kc_*, vc_*), holding
 *       n0 tokens; the step writes the new rows at n0 .. n0 + m - 1;
 *   k_codes int32 [batch][h_kv][max_len][b]: the keys' codes (written likewise);
 *   offsets/postings: an ssa_build_index index over keys 0 .. n_base - 1
 *       ([batch][h_kv][n_c + 1], [batch][h_kv][n_base * b]; n_base <= n0);
 *   tail_offsets int32 [batch][h_kv][n_c + 1], tail_postings int32
 *       [batch][h_kv][tail_cap]: rebuilt by the step over keys n_base ..
 *       n0 + m - 1 ((n0 + m - n_base) * b <= tail_cap, else SSA_ERR_WORKSPACE:
 *       rebuild the main index over every cached key and start a new tail);
 *   prep: the codebook prepared by ssa_decode_prepare (normalized rows, their
 *       bf16 copy and largest norm; prepare again when the codebook changes).
 * q [batch][m][h_q][d], k, v [batch][m][h_kv][d] (strided) are the new tokens.
 * The step routes them (top-a query and top-b key codes), selects each new
 * query's top_k keys among all cached keys from both indices (causal, index
 * order, the same selection as ssa_select_block over the whole cache) into
 * indices (nullable int32 [batch][m][h_kv][top_k]) and attends them
 * (ssa_sparse_attention_block; causal != 0 drops selected keys past the
 * query) into out [batch][m][h_q][d] (strides o_*, type out_dtype).  Limits
 * as the stages', plus a <= 32, d_s <= 32, n_c <= 16384, rows of 16 bytes. */
size_t ssa_decode_prepare_bytes(int h_kv, int n_c, int d_s);
int ssa_decode_prepare(const float* codebook, int h_kv, int n_c, int d_s, void* prep,
                       size_t prep_bytes, void* stream);
size_t ssa_decode_workspace_bytes(int64_t batch, int64_t m, int h_kv, int d_s, int n_c, int a,
                                  int b, int top_k);
int ssa_decode_step(const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t m,
                    int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb,
                    int64_t k_sn, int64_t k_sh, int64_t v_sb, int64_t v_sn, int64_t v_sh,
                    void* k_cache, void* v_cache, int64_t max_len, int64_t kc_sb, int64_t kc_sn,
                    int64_t kc_sh, int64_t vc_sb, int64_t vc_sn, int64_t vc_sh, int64_t n0,
                    const float* w_qr, const float* w_kr, const void* prep, int d_s, int n_c, int a,
                    int b, float temperature, int32_t* k_codes, const int32_t* offsets,
                    const int32_t* postings, int64_t n_base, int32_t* tail_offsets,
                    int32_t* tail_postings, int64_t tail_cap, int top_k, float score_div,
                    float scale_div, int causal, int32_t* indices, void* out, int out_dtype,
                    int64_t o_sb, int64_t o_sn, int64_t o_sh, void* workspace,
                    size_t workspace_bytes, void* stream);

/* ---- stage (d): gathered exact attention -------------------------------- */

/* out[b][i][hq] = softmax_m(q[b][i][hq] . k[b][idx[b][i][h][m]][h] / scale_div) . v[...]
 * with h = hq / (h_q/h_kv).  Replaces sparse_exact_attention (ssa/attention.py:12-115):
 * `scale_div` is the reference's `scale` (a divisor); duplicates count twice.
 * causal != 0 drops slots with idx > i (a row with no slot left outputs zeros).
 * Indices outside [0, n) are dropped and set *error_flag (nullable) to 1.
 * row_order (nullable) int32 [batch][h_kv][n]: a permutation of 0..n-1 per
 *   (batch, kv head) giving the order in which query rows are processed (e.g.
 *   grouped by routing code so that rows sharing candidates run together and
 *   hit in cache).  Results do not depend on it; a row never listed is not
 *   written, and an entry outside [0, n) is skipped and sets *error_flag.
 *   idx [batch][n][h_kv][top_k] strides (idx_sb, idx_sn, idx_sh)
 *   out [batch][n][h_q][d] strides (o_sb, o_sn, o_sh), type out_dtype
 * workspace (nullable) of ssa_sparse_attention_workspace_bytes(...) bytes: with
 *   it, the keys [0, X) that a row's indices hold exactly once (the lowest-key
 *   filler of a row with few candidates) are attended by a pass that streams
 *   them once per block of neighbouring rows, and the row pass skips them.
 *   The result is the same attention (a different summation order).
 * row_prefix (nullable) int32 [batch][h_kv][n]: X per row as ssa_select
 *   writes it (the caller vouches that the row's indices hold [0, X) once);
 *   without it the dense pass finds X from the indices (a bitmap per row).
 * row_stats (nullable) fp32 [batch][h_kv][n][g][2]: the bf16 matrix-core path
 *   (d 64 / 128, g <= 8) writes each (row, query head)'s softmax reference
 *   (the running maximum of q.k / scale_div in log2 units, 0 for a row with
 *   no slot) and 1 / sum there; other paths leave it as it was.  Given to the
 *   backward, it saves that kernel's first pass over the slots (fill it with
 *   NaN first: rows still NaN are recomputed).  No reference counterpart.
 * Limits: d a multiple of 8 in [8, 256], g <= 16. */
int ssa_sparse_attention(const void* q, const void* k, const void* v, int dtype, int64_t batch,
                         int64_t n, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn,
                         int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb,
                         int64_t v_sn, int64_t v_sh, const void* idx, int idx_dtype, int top_k,
                         int64_t idx_sb, int64_t idx_sn, int64_t idx_sh, float scale_div,
                         int causal, const int32_t* row_order, const int32_t* row_prefix,
                         void* out, int out_dtype, int64_t o_sb, int64_t o_sn,
                         int64_t o_sh, int32_t* error_flag, float* row_stats, void* workspace,
                         size_t workspace_bytes, void* stream);

/* Bytes of ssa_sparse_attention's optional workspace for n_q query rows; 0
 * where the dense-prefix pass does not run (fp32 inputs, d other than 64 or
 * 128, g > 8, top_k < 64).  No reference counterpart. */
size_t ssa_sparse_attention_workspace_bytes(int dtype, int64_t batch, int64_t n_q, int h_q, int h_kv,
                                            int d, int top_k);

/* ssa_sparse_attention for a block of n_q query rows at key positions q_pos0
 * .. q_pos0 + n_q - 1 (0 <= q_pos0, q_pos0 + n_q <= n): q, idx, out and
 * row_order hold n_q rows; `causal` compares indices with the key position.
 * n_q = n with q_pos0 = 0 is ssa_sparse_attention.  No reference counterpart:
 * it serves incremental decoding and chunked prefill. */
int ssa_sparse_attention_block(
    const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n, int64_t n_q,
    int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb,
    int64_t k_sn, int64_t k_sh, int64_t v_sb, int64_t v_sn, int64_t v_sh, const void* idx,
    int idx_dtype, int top_k, int64_t idx_sb, int64_t idx_sn, int64_t idx_sh, float scale_div,
    int causal, const int32_t* row_order, const int32_t* row_prefix, void* out, int out_dtype,
    int64_t o_sb, int64_t o_sn, int64_t o_sh, int32_t* error_flag, float* row_stats, void* workspace,
    size_t workspace_bytes, void* stream);

/* Key blocks per query block: replaces convert_indices_to_blocks
 * (ssa/triton_kernel.py:226-294).  idx [batch][n][h_kv][top_k] (strides
 * idx_sb, idx_sn, idx_sh; int32 or int64 by idx_dtype) -> out
 * [batch][nb][h_kv][n_k_blocks] (strides o_sb, o_sq, o_sh; SSA_INDEX_I32 or
 * _I64 by out_dtype), nb = ceil(n / block_size), n_k_blocks <= nb (the
 * reference takes min(top_k, nb)).  For each query block, the key blocks
 * (key j -> block j / block_size) its rows reference most often, by count
 * descending and then block id ascending (the reference leaves the order of
 * equal counts to torch.topk); rows of the last query block past n count as
 * top_k references to block 0 each, as in the reference.  block_size: a power
 * of 2 in [2, 256]; nb <= 8192.  Indices outside [0, n) are skipped and set
 * *error_flag (nullable) to 1. */
int ssa_block_indices(const void* idx, int idx_dtype, int64_t batch, int64_t n, int h_kv, int top_k,
                      int64_t idx_sb, int64_t idx_sn, int64_t idx_sh, int block_size, int n_k_blocks,
                      void* out, int out_dtype, int64_t o_sb, int64_t o_sq, int64_t o_sh,
                      int32_t* error_flag, void* stream);

/* Block-sparse exact attention: replaces ssa_triton_attention
 * (ssa/triton_kernel.py:141-223).  Query row i attends, causally (keys j <=
 * i), to every key of the n_k_blocks key blocks listed for its query block
 * i / block_size in blocks [batch][nb][h_kv][n_k_blocks] (strides b_sb, b_sq,
 * b_sh; int32 or int64 by idx_dtype).  Keys past n in the last block are
 * skipped; a block id outside [0, nb) sets *error_flag.  The softmax is exact
 * and normalised (the reference's kernel rescales and normalises its running
 * sums incorrectly, so its outputs are not a target); scores are q.k /
 * scale_div (the reference's default scale 1/sqrt(d) is scale_div =
 * sqrt(d)).  Other arguments as ssa_sparse_attention; it runs the same
 * kernels with the listed blocks expanded to keys on load. */
int ssa_block_sparse_attention(const void* q, const void* k, const void* v, int dtype, int64_t batch,
                               int64_t n, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn,
                               int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb,
                               int64_t v_sn, int64_t v_sh, const void* blocks, int idx_dtype,
                               int block_size, int n_k_blocks, int64_t b_sb, int64_t b_sq,
                               int64_t b_sh, float scale_div, void* out, int out_dtype,
                               int64_t o_sb, int64_t o_sn, int64_t o_sh, int32_t* error_flag,
                               void* stream);

/* Gradients of ssa_sparse_attention with respect to q, k and v, given the
 * forward output `out` and the output gradient `dout`.  Replaces the autograd
 * backward of sparse_exact_attention (gather -> einsum -> / scale -> softmax ->
 * einsum, ssa/attention.py:64-113), which the reference's training path runs
 * (tests/test_integration.py:32-49).  Same arguments as ssa_sparse_attention
 * for q, k, v, idx, scale_div, causal and row_order (duplicated slots count
 * once each, dropped slots not at all; an index outside [0, n) sets
 * *error_flag).  out and dout: [batch][n][h_q][d] with their own strides and
 * types (out_dtype, dout_dtype: f32 or bf16).
 *   dq fp32 [batch][n][h_q][d] contiguous: each processed row writes its own
 *      (a row never listed in row_order is not written);
 *   dk, dv fp32 [batch][n][h_kv][d] contiguous: zeroed, then accumulated.
 * Arithmetic is fp32 (softmax recomputed from q and k).  row_stats
 * (nullable): the forward's per-row softmax stats (ssa_sparse_attention's
 * row_stats); the matrix-core path then skips its first pass for every row
 * whose entry is not NaN.
 * Limits: d in [1, 256], g <= 16. */
int ssa_sparse_attention_backward(
    const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n, int h_q,
    int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn,
    int64_t k_sh, int64_t v_sb, int64_t v_sn, int64_t v_sh, const void* idx, int idx_dtype,
    int top_k, int64_t idx_sb, int64_t idx_sn, int64_t idx_sh, float scale_div, int causal,
    const int32_t* row_order, const void* out, int out_dtype, int64_t o_sb, int64_t o_sn,
    int64_t o_sh, const void* dout, int dout_dtype, int64_t do_sb, int64_t do_sn, int64_t do_sh,
    float* dq, float* dk, float* dv, int32_t* error_flag, const int32_t* row_prefix,
    const float* row_stats, void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of ssa_sparse_attention_backward's optional workspace (4 floats per
 * (row, query head)); 0 where the dense-prefix pass does not run (fp32 q/k/v
 * or dO, d other than 64 or 128, g > 8).  With row_prefix (X per row, as
 * ssa_select writes it) and this workspace, the keys [0, X) of each row are
 * differentiated by blocks of 8 neighbouring rows, whose dK/dV sums meet in
 * LDS before one fp32 atomic per (key, dim) and block.  No reference
 * counterpart. */
size_t ssa_sparse_attention_backward_workspace_bytes(int dtype, int dout_dtype, int64_t batch, int64_t n,
                                                     int h_q, int h_kv, int d);

/* ssa_sparse_attention_backward for indices that ssa_select produced (index
 * or score order, n >= top_k) from q_codes [batch][h_kv][n][a] and k_codes
 * [batch][h_kv][n][b] (ssa_route_codes), offsets / postings of
 * ssa_build_index, its row_prefix (required) and its causal routing flag
 * (router_causal: the mask was causal, else none).  Same results as
 * ssa_sparse_attention_backward (which pairs the indices hold is read from the
 * codes, row_prefix and the indices, never from scores).  dk and dv of the
 * candidate slots come from one pass per codebook
 * bucket: the rows holding a code and the keys holding it form a dense tile
 * (a pair sharing several codes counts in its smallest one), differentiated on
 * the matrix cores with one fp32 atomic per (key, dim) and 32-key chunk of a
 * bucket instead of one per selecting row.  Rows without filler (at least
 * top_k candidates) look their keys up in a bitmap of n bits each; the
 * workspace holds ssa_sparse_attention_backward_routed_workspace_bytes(...)
 * bytes, and rows past its bitmap capacity keep per-row atomics.  Shapes the
 * bucket pass does not take (fp32, d other than 64 / 128, g > 8, a > 32,
 * b > 8, N_c > 16384) run ssa_sparse_attention_backward's path.  No reference
 * counterpart (the reference's backward is autograd, ssa/attention.py:64-113). */
int ssa_sparse_attention_backward_routed(
    const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n, int h_q,
    int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn,
    int64_t k_sh, int64_t v_sb, int64_t v_sn, int64_t v_sh, const void* idx, int idx_dtype,
    int top_k, int64_t idx_sb, int64_t idx_sn, int64_t idx_sh, float scale_div, int causal,
    const int32_t* row_order, const void* out, int out_dtype, int64_t o_sb, int64_t o_sn,
    int64_t o_sh, const void* dout, int dout_dtype, int64_t do_sb, int64_t do_sn, int64_t do_sh,
    float* dq, float* dk, float* dv, int32_t* error_flag, const int32_t* row_prefix,
    const float* row_stats, const int32_t* q_codes, int a, const int32_t* k_codes, int b,
    const int32_t* offsets,
    const int32_t* postings, int n_c, int router_causal, void* workspace, size_t workspace_bytes,
    void* stream);

/* Bytes of ssa_sparse_attention_backward_routed's workspace with key bitmaps
 * for bitmap_rows rows without filler (negative: half of the batch x kv head
 * x n rows); ssa_sparse_attention_backward_workspace_bytes(...) where the
 * bucket pass does not run.  No reference counterpart. */
size_t ssa_sparse_attention_backward_routed_workspace_bytes(int dtype, int dout_dtype, int64_t batch,
                                                            int64_t n, int h_q, int h_kv, int d, int top_k,
                                                            int a, int b, int n_c, int64_t bitmap_rows);

/* ---- dense attention with a key interval per row ------------------------ */

/* Key intervals [lo, hi) of the usual masks, int32 [batch][n_q][2], for
 * ssa_masked_attention: query token i sits at key position q_pos0 + i of n keys.
 *   doc_starts (nullable) int32 [batch][docs + 1], ascending: document x of a
 *       sequence is the keys [doc_starts[x], doc_starts[x + 1]) and a token sees
 *       its own only; one before the first or from the last start on sees none.
 *       NULL: the sequence is one document (docs = 1).
 *   causal != 0: keys up to the token's own position; with prefix_lens (nullable
 *       int32 [batch][docs]) also the first prefix_lens[x] keys of its document,
 *       whatever its position.  causal == 0: the whole document.
 * No reference counterpart (the reference's dense attention takes an [n][n] bool
 * mask, ssa/attention.py:118-158). */
int ssa_mask_spans(const int32_t* doc_starts, int docs, const int32_t* prefix_lens, int64_t batch, int64_t n,
                   int64_t n_q, int64_t q_pos0, int causal, int32_t* spans, void* stream);

/* out[b][i][hq] = softmax_j(s) . v[b][j][h], h = hq / (h_q / h_kv), over the keys
 * lo <= j < hi of spans[b][i] (clamped to [0, n); NULL: j <= q_pos0 + i), with
 *   s = q[b][i][hq] . k[b][j][h] / scale_div,
 *   softcap c > 0:  s = c tanh(s / c)   (0: none),
 *   slopes (nullable) fp32 [h_q]:  s -= slopes[hq] |q_pos0 + i - j|.
 * A row that sees no key is zeros; a key that a row does not see has no influence
 * on it, whatever it holds.  Scores, weights' sums and products accumulate in
 * fp32; bf16 inputs round each weight to bf16 for the product with v.
 * Replaces dense_attention (ssa/attention.py:118-158) for masks of this form; the
 * cap and the distance bias have no reference counterpart.
 *   q [batch][n_q][h_q][d], k, v [batch][n][h_kv][d], out as q, all of type dtype,
 *   rows aligned to 16 bytes.
 *   out_low (nullable, out's strides and type) what rounding out to bf16 leaves
 *       of each value, rounded to bf16 (zeros for fp32), and
 *   lse (nullable) fp32 [batch][h_q][n_q] log2 of each row's sum of exp(s) (+inf
 *       for a row without a key): for the backward.
 *   workspace: ssa_masked_attention_workspace_bytes(...) bytes (0 for most shapes;
 *       few rows over many keys are split along the keys).
 * Limits: d a multiple of 8 up to 128, h_q / h_kv <= 16; scale_div, a softcap and their
 * product between 1e-30 and 1e30. */
size_t ssa_masked_attention_workspace_bytes(int dtype, int64_t batch, int64_t n, int64_t n_q, int h_q, int h_kv,
                                            int d);
int ssa_masked_attention(const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n,
                         int64_t n_q, int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn,
                         int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb, int64_t v_sn,
                         int64_t v_sh, const int32_t* spans, float scale_div, float softcap, const float* slopes,
                         void* out, int64_t o_sb, int64_t o_sn, int64_t o_sh, void* out_low, float* lse,
                         void* workspace, size_t workspace_bytes, void* stream);

/* Gradients of ssa_masked_attention with respect to q, k and v, given its output,
 * out_low (nullable: D = dout . out then takes the rounded output), its lse and the
 * output gradient.  Same arguments for the forward's; dout has
 * out's shape and type with its own strides.
 *   dq [batch][n_q][h_q][d], dk, dv [batch][n][h_kv][d], contiguous, of type dtype:
 *      written whole (a shared head's sums over its group included), each value
 *      rounded once.  No atomics: the same inputs give the same bits.
 *   q and dout: the heads of a group within 2 GiB of each other.
 *   workspace: ssa_masked_attention_backward_workspace_bytes(...) bytes.
 * Replaces the autograd backward of dense_attention (ssa/attention.py:118-158)
 * for masks of this form.  slopes get no gradient. */
size_t ssa_masked_attention_backward_workspace_bytes(int dtype, int64_t batch, int64_t n, int64_t n_q, int h_q,
                                                     int h_kv, int d);
int ssa_masked_attention_backward(
    const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n, int64_t n_q,
    int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb,
    int64_t k_sn, int64_t k_sh, int64_t v_sb, int64_t v_sn, int64_t v_sh, const int32_t* spans,
    float scale_div, float softcap, const float* slopes, const void* out, const void* out_low,
    int64_t o_sb, int64_t o_sn, int64_t o_sh, const void* dout, int64_t do_sb, int64_t do_sn, int64_t do_sh,
    const float* lse, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream);

/* ssa_mask_spans for causal rows with a sliding window: int32 spans [batch][n_q][4], two key
 * intervals a row.  A row at position p of a document that starts at a sees the keys
 * max(a, p - window + 1) .. p (the first interval) and a .. a + sinks - 1 up to its own, with
 * prefix_lens the first prefix_lens[x] too, whatever its position (the second, empty where
 * they meet the first, which then holds both).  spans aligned to 16 bytes. */
int ssa_mask_spans_window(const int32_t* doc_starts, int docs, const int32_t* prefix_lens, int64_t batch, int64_t n,
                          int64_t n_q, int64_t q_pos0, int64_t window, int64_t sinks, int32_t* spans, void* stream);

/* ssa_masked_attention whose rows see two key intervals: spans int32 [batch][n_q][4] (not
 * null, aligned to 16 bytes) holds lo, hi, lo2, hi2, each pair clamped to [0, n) and empty
 * where hi <= lo.  The two may lie in any order and overlap (a key in both counts once).  The
 * same other arguments and workspace. */
int ssa_masked_attention_two(const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n,
                             int64_t n_q, int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn,
                             int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh, int64_t v_sb, int64_t v_sn,
                             int64_t v_sh, const int32_t* spans, float scale_div, float softcap, const float* slopes,
                             void* out, int64_t o_sb, int64_t o_sn, int64_t o_sh, void* out_low, float* lse,
                             void* workspace, size_t workspace_bytes, void* stream);

/* Its gradients, as ssa_masked_attention_backward's, with a workspace of
 * ssa_masked_attention_two_backward_workspace_bytes(...) bytes. */
size_t ssa_masked_attention_two_backward_workspace_bytes(int dtype, int64_t batch, int64_t n, int64_t n_q, int h_q,
                                                         int h_kv, int d);
int ssa_masked_attention_two_backward(
    const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t n, int64_t n_q,
    int64_t q_pos0, int h_q, int h_kv, int d, int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb,
    int64_t k_sn, int64_t k_sh, int64_t v_sb, int64_t v_sn, int64_t v_sh, const int32_t* spans,
    float scale_div, float softcap, const float* slopes, const void* out, const void* out_low,
    int64_t o_sb, int64_t o_sn, int64_t o_sh, const void* dout, int64_t do_sb, int64_t do_sn, int64_t do_sh,
    const float* lse, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream);

/* ---- paged cache --------------------------------------------------------- */

/* Attention of new tokens over a paged K/V cache, a ragged batch in one call.
 * Sequence b's new tokens are rows starts[b] .. starts[b + 1] - 1 of q, k, v and
 * out ([tokens][heads][d], strides *_st, *_sh); its key j is row j % page_size of
 * page table[b][j / page_size] of the pools k_pages, v_pages
 * [num_pages][page_size][h_kv][d] (strides *_sp, *_st, *_sh), and cached[b] keys
 * are there already.  The call writes the new rows of k and v at keys cached[b]
 * ... (k = v = NULL: they are there) and attends new token t over keys
 * 0 .. cached[b] + t with ssa_masked_attention's score rule (positions count from
 * the sequence's first key).
 *   table int32 [batch][max_pages] (row stride table_stride), starts int32
 *       [batch + 1] ascending, cached int32 [batch]: device memory, read by the
 *       kernels, so that a captured call follows their values.
 *   max_new, max_len: the most new tokens and the most keys (new ones included) of
 *       a sequence; the launch is sized by them (they may say more than the tokens
 *       or the table hold; the workspace is asked for with the same).
 *   A sequence that breaks them, or the table's or the rows' range, is left out
 *       (its rows of out and its pages stay as they are), a page outside the pool
 *       is not touched (keys there read page 0): either sets *error_flag
 *       (nullable) to 1.  Rows of out of no sequence stay as they are.
 *   workspace: ssa_paged_step_workspace_bytes(...) bytes; calls that may run at
 *       once each need their own.
 * Limits: as ssa_masked_attention; page_size a power of 2 in [8, 4096].
 * No reference counterpart (ssa_design.md:225-234 describes decoding against a
 * cache; its code runs whole sequences). */
size_t ssa_paged_step_workspace_bytes(int dtype, int64_t tokens, int64_t batch, int h_q, int h_kv, int d,
                                      int64_t max_new, int64_t max_len);
int ssa_paged_step(const void* q, const void* k, const void* v, int dtype, int64_t tokens, int64_t batch, int h_q,
                   int h_kv, int d, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh, int64_t v_st,
                   int64_t v_sh, void* k_pages, void* v_pages, int64_t num_pages, int page_size, int64_t kp_sp,
                   int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st, int64_t vp_sh,
                   const int32_t* table, int64_t table_stride, int max_pages, const int32_t* starts,
                   const int32_t* cached, int64_t max_new, int64_t max_len, float scale_div, float softcap,
                   const float* slopes, void* out, int64_t o_st, int64_t o_sh, int32_t* error_flag,
                   void* workspace, size_t workspace_bytes, void* stream);

/* ssa_paged_step where out holds nothing yet: rows of no sequence, and of one that is
 * left out, are written as zeros.  batch must be positive where tokens is. */
int ssa_paged_step_zeroed(const void* q, const void* k, const void* v, int dtype, int64_t tokens, int64_t batch, int h_q,
                          int h_kv, int d, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh, int64_t v_st,
                          int64_t v_sh, void* k_pages, void* v_pages, int64_t num_pages, int page_size, int64_t kp_sp,
                          int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st, int64_t vp_sh, const int32_t* table,
                          int64_t table_stride, int max_pages, const int32_t* starts, const int32_t* cached,
                          int64_t max_new, int64_t max_len, float scale_div, float softcap, const float* slopes, void* out,
                          int64_t o_st, int64_t o_sh, int32_t* error_flag, void* workspace, size_t workspace_bytes,
                          void* stream);

/* ssa_paged_step with a sliding window, drafted trees and pages of 8 bits, each by itself
 * or together.
 *   window > 0: a token at position p sees the keys at positions p - window + 1 .. p and
 *       the first `sinks` positions (up to its own); the pages (table entries) between are
 *       not read.  0: none (sinks 0 too).
 *   parents (nullable) int32 [tokens]: new token i of a sequence is drafted behind its
 *       new token parents[starts[b] + i] < i, or behind the cached ones (-1).  It sees
 *       the cached keys, its ancestors and itself, and its position is cached[b] + its
 *       number of ancestors; its key is written at cached[b] + i as ever (ssa_paged_keep
 *       puts a path in order).  max_new (or tokens) at most 64.  Any other value of a
 *       parent counts as -1 and sets *error_flag.
 *   page_dtype: dtype, SSA_DTYPE_I8 or SSA_DTYPE_E4M3.  Of 8 bits a page row of a head is d
 *       codes, and k_scales, v_scales fp32 [num_pages][page_size][h_kv] (strides ks_*, vs_*
 *       in elements) say what one stands for: code * scale.  Rows written get scale =
 *       max |x| / 127 (or / 448) and the codes nearest to x / scale (ties to even); below
 *       2^-100 they are zeros, and one with an infinity or NaN has the scale NaN.  The
 *       call's own rows are attended as they are given.  Rows aligned to 8 bytes.
 *   zero_rows != 0: as ssa_paged_step_zeroed.
 * The other arguments and what is refused as ssa_paged_step; the workspace is
 * ssa_paged_step_general_workspace_bytes(...) bytes.  No reference counterpart. */
size_t ssa_paged_step_general_workspace_bytes(int dtype, int page_dtype, int64_t tokens, int64_t batch, int h_q,
                                              int h_kv, int d, int64_t max_new, int64_t max_len, int64_t window,
                                              int64_t sinks);
int ssa_paged_step_general(const void* q, const void* k, const void* v, int dtype, int64_t tokens, int64_t batch,
                           int h_q, int h_kv, int d, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
                           int64_t v_st, int64_t v_sh, void* k_pages, void* v_pages, int page_dtype,
                           float* k_scales, float* v_scales, int64_t num_pages, int page_size, int64_t kp_sp,
                           int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st, int64_t vp_sh,
                           int64_t ks_sp, int64_t ks_st, int64_t ks_sh, int64_t vs_sp, int64_t vs_st, int64_t vs_sh,
                           const int32_t* table, int64_t table_stride, int max_pages, const int32_t* starts,
                           const int32_t* cached, const int32_t* parents, int64_t max_new, int64_t max_len,
                           int64_t window, int64_t sinks, float scale_div, float softcap, const float* slopes,
                           void* out, int64_t o_st, int64_t o_sh, int zero_rows, int32_t* error_flag,
                           void* workspace, size_t workspace_bytes, void* stream);

/* Rows of a paged cache read back: row starts[b] + i of k_out and v_out
 * ([tokens][h_kv][d], contiguous, of type out_dtype) is key first[b] + i of sequence b,
 * for the rows up to starts[b + 1].  Pages of 8 bits are read as what they stand for,
 * rounded once; others as they are (out_dtype = page_dtype).  Rows of no sequence, and
 * keys past the table or in a page outside the pool, are zeros (the latter set
 * *error_flag, nullable). */
int ssa_paged_read(const void* k_pages, const void* v_pages, int page_dtype, const float* k_scales,
                   const float* v_scales, int64_t num_pages, int page_size, int h_kv, int d, int64_t kp_sp,
                   int64_t kp_st, int64_t kp_sh, int64_t vp_sp, int64_t vp_st, int64_t vp_sh, int64_t ks_sp,
                   int64_t ks_st, int64_t ks_sh, int64_t vs_sp, int64_t vs_st, int64_t vs_sh, int64_t batch,
                   const int32_t* table, int64_t table_stride, int max_pages, const int32_t* starts,
                   const int32_t* first, int64_t tokens, int out_dtype, void* k_out, void* v_out,
                   int32_t* error_flag, void* stream);

/* Keeps some of the tokens behind a sequence's cached ones, of a drafted tree the path that
 * was accepted: key cached[b] + kept[b][t] (codes and scale) goes to key cached[b] + t, for
 * t up to the first kept[b][t] below 0 or most_kept (at most 64).  kept int32
 * [batch][most_kept] (row stride kept_stride) ascends; from the first one that does not on,
 * nothing moves, and *error_flag (nullable) is set, as for pages outside the pool and keys
 * past the table, which are left out. */
int ssa_paged_keep(void* k_pages, void* v_pages, int page_dtype, float* k_scales, float* v_scales,
                   int64_t num_pages, int page_size, int h_kv, int d, int64_t kp_sp, int64_t kp_st, int64_t kp_sh,
                   int64_t vp_sp, int64_t vp_st, int64_t vp_sh, int64_t ks_sp, int64_t ks_st, int64_t ks_sh,
                   int64_t vs_sp, int64_t vs_st, int64_t vs_sh, int64_t batch, const int32_t* table,
                   int64_t table_stride, int max_pages, const int32_t* cached, const int32_t* kept,
                   int64_t kept_stride, int most_kept, int32_t* error_flag, void* stream);

/* ---- rotary positions with several axes ---------------------------------- */

/* Rotary embedding of q and k (k nullable with h_k = 0) whose tokens have a
 * position on each of `axes` axes (1 to 4): feature pair (m, m + rot / 2) turns by
 * positions[axis(m)][b][i] * freqs[m], the first sections[0] pairs by axis 0, the
 * next sections[1] by axis 1 and so on (sections: int32 [axes] in HOST memory, read
 * by the call, their sum rot / 2).  Features from rot on pass through.
 *   q [batch][n][h_q][d], k [batch][n][h_k][d], outputs likewise with their own
 *       strides; an output may be its input (same strides).
 *   positions int32 or int64 (SSA_INDEX_*) [axes][batch][n], strides p_sa, p_sb
 *       (0 to share), contiguous along n; freqs fp64 [rot / 2].
 *   inverse != 0 applies the transpose (the backward).
 * Angles are formed and reduced in 64 bits, the rotation is fp32, the result
 * rounded once.  No reference counterpart (ssa/utils.py:7-41 has one axis). */
int ssa_rope_axes(const void* q, const void* k, int dtype, int64_t batch, int64_t n, int h_q, int h_k, int d,
                  int64_t q_sb, int64_t q_sn, int64_t q_sh, int64_t k_sb, int64_t k_sn, int64_t k_sh,
                  const void* positions, int pos_dtype, int64_t p_sa, int64_t p_sb, int axes,
                  const int32_t* sections, const double* freqs, int rot, int inverse, void* q_out, int64_t qo_sb,
                  int64_t qo_sn, int64_t qo_sh, void* k_out, int64_t ko_sb, int64_t ko_sn, int64_t ko_sh,
                  void* stream);

/* ---- calls with packed arguments ----------------------------------------- */

/* Calls one of these entry points with its arguments from an array, in order, eight bytes
 * each: integers and pointers as int64_t, floats as double.  For callers to whom each argument
 * costs (a Python call of 50 arguments takes 5 microseconds, one of a packed array 2). */
#define SSA_CALL_MASK_SPANS 0
#define SSA_CALL_MASK_SPANS_WINDOW 1
#define SSA_CALL_MASKED_ATTENTION 2
#define SSA_CALL_MASKED_ATTENTION_TWO 3
#define SSA_CALL_MASKED_ATTENTION_BACKWARD 4
#define SSA_CALL_MASKED_ATTENTION_TWO_BACKWARD 5
#define SSA_CALL_PAGED_STEP 6
#define SSA_CALL_PAGED_STEP_ZEROED 7
#define SSA_CALL_PAGED_STEP_GENERAL 8
#define SSA_CALL_PAGED_READ 9
#define SSA_CALL_PAGED_KEEP 10
int ssa_call(int function, const int64_t* arguments);

#ifdef __cplusplus
}
#endif

#endif /* SSA_HIP_H */
