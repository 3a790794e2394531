/* C ABI of libkv_attention.so -- hand-written gfx950 (MI355X) kernels for attention over keys that are not the
 * queries' own: an encoder's states (cross attention, forward and backward) and a cache in pages (the newest tokens of
 * every sequence), and the writing of new tokens into the pages.
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

/* Human-readable text for a return code of the functions above (static storage). */
const char* kv_error_string(int code);

#ifdef __cplusplus
}
#endif
#endif
