/* C ABI of libkv_attention.so -- hand-written gfx950 (MI355X) kernels for attention over keys that are not the
 * queries' own: an encoder's states (cross attention, forward and backward) and a cache in pages (the newest tokens of
 * every sequence, or trees of drafted ones), the writing of new tokens into the pages, and what comes before attention: norms of queries
 * and keys for each head and the rotation by position.
 *
 * Common rules
 *   - Every pointer is a device pointer owned by the caller.  Nothing is allocated, freed or synchronised here: each call
 *     enqueues kernels on `stream` (a hipStream_t, NULL = the default stream) and returns.  Work that is divided over the keys
 *     needs a workspace of the size that the *_workspace function gives for the same sizes; calls that overlap need
 *     one each.  Its contents before and after a call mean nothing.
 *   - q, o, d_o, dq: [B,Hq,Tq,D]; k, v, dk, dv: [B,Hkv,Tk,D]; Hq is a multiple of Hkv, and with G = Hq / Hkv query head
 *     h reads key head h / G.  Inputs have element strides int64[4] (batch, head, time, dim): the dim stride is 1, the others
 *     multiples of 16 bytes and not negative, base pointers 16-byte aligned; the time stride is not 0 where there is more than one
 *     row.  The rows of one head of k and v are addressed with 32-bit byte offsets: (Tk + 1024) * time_stride * element_size < 2^32,
 *     and those of q and d_o in the backward likewise where Hq == Hkv, else KV_ERR_TOO_LARGE.  Outputs are contiguous.
 *     KV_ERR_TOO_LARGE too where a launch of the call would have 2^32 threads or more (about 2^23 pairs of a batch entry and a key head times tiles
 *     of 128 rows, or keys in the backward, and up).
 *   - sm_scale is a number within 2^127 on either side of 0, else KV_ERR_ARG.
 *   - dtype: 0 = float32, 1 = float16, 2 = bfloat16.  D in {16,32,64,128,256}.
 *   - lens, q_lens, new_lens: int32 per batch entry with a stride in elements, or NULL = the whole length; values are clamped to
 *     [0, length].  Positions beyond a length are never used, whatever they hold.
 *   - Outputs are fully written.  Rows from q_lens[b] (new_lens[b]) on: O, LSE and dQ are 0, and dO is not read.  A row that sees no key, or
 *     none with a score above -inf: O is 0, LSE -inf, and it passes no gradient on.  Keys that no row sees: dK and dV are 0.
 *   - Softmax statistics and all sums are float32.  The probabilities, and dS, are rounded to the element type as operands of
 *     the second products (float32 stays float32); the scale is applied to the scores in float32.  No atomics: results do not
 *     change from call to call.
 *   - Return value: 0 on success, > 0 a hipError_t from a launch, < 0 one of KV_ERR_*; a call that returns KV_ERR_* has enqueued
 *     nothing.
 *   - Re-entrant.  The library's only mutable state is the kernels' LDS limits (hipFuncSetAttribute on the first call of each
 *     kernel shape on each device, guarded by a mutex): make that first call outside a HIP graph capture.
 */
#ifndef KV_ATTENTION_H
#define KV_ATTENTION_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KV_OK 0
#define KV_ERR_DTYPE (-1)
#define KV_ERR_HEAD_DIM (-2)
#define KV_ERR_ARG (-3)
#define KV_ERR_LAYOUT (-4)
#define KV_ERR_TOO_LARGE (-5)
#define KV_ERR_WORKSPACE (-6)

/* Bytes of workspace for kv_cross_forward with these sizes; 0 if it needs none, < 0 one of KV_ERR_*. */
int64_t kv_cross_forward_workspace(int B, int Hq, int Hkv, int Tq, int Tk, int D, int dtype);

/* O = softmax(sm_scale * Q K^T) V over the first lens[b] keys, LSE = log2 sum exp (scaled scores) [B,Hq,Tq] float32, or NULL. */
int kv_cross_forward(const void* q, const void* k, const void* v,
                     const int32_t* lens, int64_t lens_stride, const int32_t* q_lens, int64_t q_lens_stride,
                     void* o, float* lse, void* workspace, int64_t workspace_bytes,
                     const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                     int B, int Hq, int Hkv, int Tq, int Tk, int D, float sm_scale, int dtype, void* stream);

/* Bytes of workspace for kv_cross_backward with these sizes (not 0 if there is a query), < 0 one of KV_ERR_*. */
int64_t kv_cross_backward_workspace(int B, int Hq, int Hkv, int Tq, int Tk, int D, int dtype);

/* dQ, dK, dV from the forward's inputs, its O and LSE, and dO. */
int kv_cross_backward(const void* q, const void* k, const void* v,
                      const int32_t* lens, int64_t lens_stride, const int32_t* q_lens, int64_t q_lens_stride,
                      const void* o, const void* d_o, const float* lse, void* dq, void* dk, void* dv,
                      void* workspace, int64_t workspace_bytes,
                      const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                      const int64_t* o_strides, const int64_t* do_strides,
                      int B, int Hq, int Hkv, int Tq, int Tk, int D, float sm_scale, int dtype, void* stream);

/* Bytes of workspace for kv_paged_forward with these sizes; 0 if it needs none, < 0 one of KV_ERR_*. */
int64_t kv_paged_forward_workspace(int B, int Hq, int Hkv, int T, int D, int page_size, int width,
                                   int context_size, int back_contexts, int dtype);

/* The newest tokens of every sequence over its cache.  k_pages and v_pages: [num_pages,Hkv,page_size,D] with strides (page, head,
 * position, dim) as above, without a limit of 32-bit offsets.  page_table: int32 [B,width], rows table_stride elements apart, unit stride along a row; position
 * t of sequence b is position t % page_size of page page_table[b][t / page_size].  An entry outside [0, num_pages) is a page that is not
 * there: its positions are not seen.  lens[b] counts the new tokens; lengths beyond width * page_size count as that.
 * Token i of the n = new_lens[b] (or T) new ones is at position at = lens[b] - n + i and sees the positions j < lens[b] with
 * 0 <= at / context_size - j / context_size <= back_contexts: what row `at` of sa_forward sees.  context_size 1 is causal, and with back_contexts
 * = w a window of w + 1 positions; a token whose position is negative sees nothing.  width * page_size <= 2^30.
 * O and LSE as in kv_cross_forward.  The bits of a sequence's result depend on the sizes of the call (B, T, width * page_size), not on the
 * lengths or values of the other sequences.
 * A value that is not finite, at a position that one new token sees, reaches the other tokens of its sequence in the call. */
int kv_paged_forward(const void* q, const void* k_pages, const void* v_pages,
                     const int32_t* page_table, int64_t table_stride, const int32_t* lens, int64_t lens_stride,
                     const int32_t* new_lens, int64_t new_lens_stride,
                     void* o, float* lse, void* workspace, int64_t workspace_bytes,
                     const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                     int B, int Hq, int Hkv, int T, int D, int num_pages, int page_size, int width,
                     int context_size, int back_contexts, float sm_scale, int dtype, void* stream);

/* Writes the new tokens k, v [B,H,T,D] into the pages: token i of the n = new_lens[b] (or T) of sequence b to position lens[b] - n + i.
 * Positions below 0 or from width * page_size on, and pages that are not there, are left out.  Where two tokens of a call have the
 * same place (two sequences that share a page), it holds either of them afterwards, or sixteen bytes of one beside sixteen of
 * the other.  k and v do not overlap the pages.  The strides of the pages are not 0 where there is more than one page or head.
 * B * H * T * D * element_size < 2^35, else KV_ERR_TOO_LARGE. */
int kv_paged_append(const void* k, const void* v, void* k_pages, void* v_pages,
                    const int32_t* page_table, int64_t table_stride, const int32_t* lens, int64_t lens_stride,
                    const int32_t* new_lens, int64_t new_lens_stride,
                    const int64_t* k_strides, const int64_t* v_strides,
                    const int64_t* k_page_strides, const int64_t* v_page_strides,
                    int B, int H, int T, int D, int num_pages, int page_size, int width, int dtype, void* stream);

/* Trees of drafted tokens over the cache: as kv_paged_forward, but token i of the n new ones sees all positions before them, below lens[b] - n, and of
 * the new tokens those j with tree[b][i][j] != 0: bytes at the strides int64[3] (batch, token, token; a batch stride of 0 is one tree for all).
 * A token whose position lens[b] - n + i is negative sees nothing, and is not seen. */
int64_t kv_paged_tree_forward_workspace(int B, int Hq, int Hkv, int T, int D, int page_size, int width, int dtype);
int kv_paged_tree_forward(const void* q, const void* k_pages, const void* v_pages,
                          const int32_t* page_table, int64_t table_stride, const int32_t* lens, int64_t lens_stride,
                          const int32_t* new_lens, int64_t new_lens_stride, const void* tree, const int64_t* tree_strides,
                          void* o, float* lse, void* workspace, int64_t workspace_bytes,
                          const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                          int B, int Hq, int Hkv, int T, int D, int num_pages, int page_size, int width,
                          float sm_scale, int dtype, void* stream);

/* Keeps accepted tokens: K and V of position first[b] + kept[b][i] go to position first[b] + i, for i = 0, 1, ... up to the first entry that is
 * negative or not above the one before it, or M of them.  kept: int32 at the strides int64[2] (batch, entry).  Where the one or the other position is below
 * 0, past the table or on a page that is not there, the place stays as it is.  Pages that a call writes stand once in the table, and K and V are
 * one cache or do not overlap. */
int kv_paged_keep(void* k_pages, void* v_pages, const int32_t* page_table, int64_t table_stride,
                  const int32_t* first, int64_t first_stride, const int32_t* kept, const int64_t* kept_strides,
                  const int64_t* k_page_strides, const int64_t* v_page_strides,
                  int B, int H, int M, int D, int num_pages, int page_size, int width, int dtype, void* stream);

/* Norms of queries and keys for each head and the rotation by position.  A row x (D channels) of q [B,Hq,T,D] or k [B,Hkv,T,D] becomes
 *   y = x * w / sqrt(mean(x^2) + eps)      eps below 3.4e38; 0: y = x, and no weights
 * and of its first `rot` channels the pairs (a, b) become (a cos - b sin, b cos + a sin): channels i and i + rot / 2, or 2 i and 2 i + 1 if interleaved,
 * with cos[at][i] and sin[at][i].  at: positions[b][t] at the strides int64[2], or t where positions is NULL.
 * rot: a multiple of 16 up to D.  cos, sin: float32 [table_rows, rot / 2], rows a multiple of 4 elements apart, 16-byte aligned.  Weights: [D] of the element
 * type, or float32 where weights_f32 is set, 16-byte aligned, or NULL (ones).  Tokens from lens[b] on, and tokens whose position the table does not
 * have, are padding: their rows are 0, they are not read and pass no gradient on.  q_out and k_out are contiguous and written whole.
 * Sums are float32; results are rounded once.  Any Hq (up to 32767) and Hkv (16383), B * T < 2^31, else KV_ERR_TOO_LARGE. */
int kv_qk_norm_rope(const void* q, const void* k, const float* cos, const float* sin, int64_t cos_stride, int64_t sin_stride,
                    const void* q_weight, const void* k_weight, int weights_f32,
                    const int32_t* lens, int64_t lens_stride, const int32_t* positions, const int64_t* position_strides,
                    void* q_out, void* k_out, const int64_t* q_strides, const int64_t* k_strides,
                    int B, int Hq, int Hkv, int T, int D, int rot, int table_rows, int interleaved, float eps, int dtype, void* stream);

/* Bytes of workspace for kv_qk_norm_rope_backward where it is asked for gradients of weights. */
int64_t kv_qk_norm_rope_backward_workspace(int B, int Hq, int Hkv, int T, int D, int dtype);

/* dq, dk and, where the pointers are not NULL, the gradients of the weights (in the weights' type) from those of q_out and k_out. */
int kv_qk_norm_rope_backward(const void* q, const void* k, const void* d_q_out, const void* d_k_out,
                             const float* cos, const float* sin, int64_t cos_stride, int64_t sin_stride,
                             const void* q_weight, const void* k_weight, int weights_f32,
                             const int32_t* lens, int64_t lens_stride, const int32_t* positions, const int64_t* position_strides,
                             void* dq, void* dk, void* dq_weight, void* dk_weight, void* workspace, int64_t workspace_bytes,
                             const int64_t* q_strides, const int64_t* k_strides, const int64_t* dq_out_strides, const int64_t* dk_out_strides,
                             int B, int Hq, int Hkv, int T, int D, int rot, int table_rows, int interleaved, float eps, int dtype, void* stream);

/* kv_paged_append with norms and rotation on the way: q turned into q_out (contiguous, zeros from new_lens[b] on), k turned into the pages, v as it
 * is.  The position of a token's angles is positions[b][i], or where the token goes if positions is NULL; a token whose position the table of
 * angles does not have is left out of the pages, and its q_out is 0. */
int kv_paged_append_rope(const void* q, const void* k, const void* v, void* q_out, void* k_pages, void* v_pages,
                         const int32_t* page_table, int64_t table_stride, const int32_t* lens, int64_t lens_stride,
                         const int32_t* new_lens, int64_t new_lens_stride,
                         const float* cos, const float* sin, int64_t cos_stride, int64_t sin_stride,
                         const void* q_weight, const void* k_weight, int weights_f32,
                         const int32_t* positions, const int64_t* position_strides,
                         const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                         const int64_t* k_page_strides, const int64_t* v_page_strides,
                         int B, int Hq, int Hkv, int T, int D, int num_pages, int page_size, int width,
                         int rot, int table_rows, int interleaved, float eps, int dtype, void* stream);

/* Human-readable text for a return code of the functions above (static storage). */
const char* kv_error_string(int code);

#ifdef __cplusplus
}
#endif
#endif
