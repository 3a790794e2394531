// extern "C" entries of norms and rotation: argument checks, parameter packing and dispatch on the element type.  See
// include/kv_attention.h for the contract.
#include "kv_check.h"
#include "kv_rope_launch.h"

using namespace kv;

namespace {

int check_rope(int B, int Hq, int Hkv, int T, int D, int rot, int table_rows, float eps, int dtype) {
  if (int rc = check_sizes(B, 1, 1, D, dtype)) return rc;
  if (Hq < 0 || Hkv < 0 || T < 0 || table_rows < 0 || rot < 16 || rot > D || rot % 16 != 0 || !(eps >= 0.0f) || eps > 3.4e38f) return KV_ERR_ARG;
  return (int64_t)B * T > kMostTokens || Hq > 65535 / 2 || Hkv > 65535 / 4 ? KV_ERR_TOO_LARGE : KV_OK;   // layers of a grid
}
int check_table(const float* cos, const float* sin, int64_t cos_stride, int64_t sin_stride, int rows) {
  if (rows == 0) return KV_OK;   // no position has angles: nothing is read
  if (!cos || !sin) return KV_ERR_ARG;
  for (const void* p : {(const void*)cos, (const void*)sin})
    if (reinterpret_cast<uintptr_t>(p) & 15u) return KV_ERR_LAYOUT;
  for (int64_t s : {cos_stride, sin_stride})
    if (s < 0 || s % 4 != 0) return KV_ERR_LAYOUT;
  return KV_OK;
}
int check_weights(const void* q_weight, const void* k_weight, float eps) {
  if ((q_weight || k_weight) && eps == 0.0f) return KV_ERR_ARG;   // weights are those of the norms
  return ((reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight)) & 15u) ? KV_ERR_LAYOUT : KV_OK;
}

}  // namespace

extern "C" {

int kv_qk_norm_rope(const void* q, const void* k, const float* cos, const float* sin, int64_t cos_stride, int64_t sin_stride,
                    const void* q_weight, const void* k_weight, int weights_f32, const int32_t* lens, int64_t lens_stride,
                    const int32_t* positions, const int64_t* position_strides, void* q_out, void* k_out, const int64_t* qs, const int64_t* ks,
                    int B, int Hq, int Hkv, int T, int D, int rot, int table_rows, int interleaved, float eps, int dtype, void* stream) {
  if (int rc = check_rope(B, Hq, Hkv, T, D, rot, table_rows, eps, dtype)) return rc;
  if (B == 0 || T == 0 || Hq + Hkv == 0) return KV_OK;
  RopeParams p{};
  const void* x[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t* st[2] = {qs, ks};
  const int heads[2] = {Hq, Hkv};
  for (int i = 0; i < 2; ++i) {
    if (heads[i] == 0) continue;
    if (int rc = check_layout(x[i], st[i], dtype, T, false)) return rc;
    if (int rc = check_out(out[i])) return rc;
    RopeSide& s = i ? p.k : p.q;
    s.x = x[i]; s.out = out[i]; s.weight = i ? k_weight : q_weight;
    s.sb = st[i][0]; s.sh = st[i][1]; s.st = st[i][2]; s.heads = heads[i];
  }
  if (int rc = check_table(cos, sin, cos_stride, sin_stride, table_rows)) return rc;
  if (int rc = check_weights(q_weight, k_weight, eps)) return rc;
  if (positions && !position_strides) return KV_ERR_ARG;
  p.table = RopeTable{cos, sin, cos_stride, sin_stride, table_rows, rot};
  p.lens = lens; p.lens_stride = lens_stride;
  p.positions = positions;
  if (positions) p.pos_sb = position_strides[0], p.pos_st = position_strides[1];
  p.B = B; p.T = T; p.eps = eps; p.weights_f32 = weights_f32 != 0;
  p.by_tokens = chunk_div(T);
  const RopeGrid g = forward_grid((int64_t)B * T, Hq, Hkv, D, elem_size(dtype));
  p.chunk = g.chunk; p.q_chunks = g.q_chunks;
  const bool streaming = past_caches((int64_t)B * (Hq + Hkv) * T, D, rot, interleaved != 0, elem_size(dtype));
  return by_dtype(dtype, [&](auto tag) { return launch_rope<decltype(tag)>(p, g, D, interleaved != 0, streaming, (hipStream_t)stream); });
}

int64_t kv_qk_norm_rope_backward_workspace(int B, int Hq, int Hkv, int T, int D, int dtype) {
  if (int rc = check_rope(B, Hq, Hkv, T, D, 16, 0, 0.0f, dtype)) return rc;
  if (B == 0 || T == 0 || Hq + Hkv == 0) return 0;
  const RopeGrid g = backward_grid((int64_t)B * T, Hq, Hkv, D, elem_size(dtype));
  return (int64_t)g.blocks * (g.q_chunks + g.k_chunks) * D * 4;
}

int kv_qk_norm_rope_backward(const void* q, const void* k, const void* d_q_out, const void* d_k_out, const float* cos, const float* sin,
                             int64_t cos_stride, int64_t sin_stride, const void* q_weight, const void* k_weight, int weights_f32,
                             const int32_t* lens, int64_t lens_stride, const int32_t* positions, const int64_t* position_strides, void* dq,
                             void* dk, void* dq_weight, void* dk_weight, void* workspace, int64_t workspace_bytes, const int64_t* qs,
                             const int64_t* ks, const int64_t* gqs, const int64_t* gks, int B, int Hq, int Hkv, int T, int D, int rot,
                             int table_rows, int interleaved, float eps, int dtype, void* stream) {
  if (int rc = check_rope(B, Hq, Hkv, T, D, rot, table_rows, eps, dtype)) return rc;
  const bool weights = dq_weight || dk_weight;
  if ((dq_weight && !q_weight) || (dk_weight && !k_weight)) return KV_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(dq_weight) | reinterpret_cast<uintptr_t>(dk_weight)) & 15u) != 0) return KV_ERR_LAYOUT;
  if (int rc = check_weights(q_weight, k_weight, eps)) return rc;
  const RopeGrid g = backward_grid((int64_t)B * T, Hq, Hkv, D, elem_size(dtype));
  RopeParams p{};
  const bool any = B > 0 && T > 0 && Hq + Hkv > 0;
  if (any) {
    const void* x[2] = {q, k};
    const void* grad[2] = {d_q_out, d_k_out};
    void* out[2] = {dq, dk};
    const int64_t *st[2] = {qs, ks}, *gst[2] = {gqs, gks};
    const int heads[2] = {Hq, Hkv};
    for (int i = 0; i < 2; ++i) {
      if (heads[i] == 0) continue;
      if (int rc = check_layout(x[i], st[i], dtype, T, false)) return rc;
      if (int rc = check_layout(grad[i], gst[i], dtype, T, false)) return rc;
      if (int rc = check_out(out[i])) return rc;
      RopeSide& s = i ? p.k : p.q;
      s.x = x[i]; s.g = grad[i]; s.out = out[i]; s.weight = i ? k_weight : q_weight;
      s.sb = st[i][0]; s.sh = st[i][1]; s.st = st[i][2]; s.heads = heads[i];
      s.g_sb = gst[i][0]; s.g_sh = gst[i][1]; s.g_st = gst[i][2];
    }
    if (int rc = check_table(cos, sin, cos_stride, sin_stride, table_rows)) return rc;
    if (positions && !position_strides) return KV_ERR_ARG;
    if (weights)
      if (int rc = check_workspace(workspace, workspace_bytes, (int64_t)g.blocks * (g.q_chunks + g.k_chunks) * D * 4)) return rc;
    p.table = RopeTable{cos, sin, cos_stride, sin_stride, table_rows, rot};
    p.lens = lens; p.lens_stride = lens_stride;
    p.positions = positions;
    if (positions) p.pos_sb = position_strides[0], p.pos_st = position_strides[1];
    p.B = B; p.T = T; p.eps = eps; p.weights_f32 = weights_f32 != 0;
    p.by_tokens = chunk_div(T);
    p.chunk = g.chunk; p.q_chunks = g.q_chunks;
    p.part = weights ? (float*)workspace : nullptr;
    const bool streaming = past_caches((int64_t)B * (Hq + Hkv) * T, D, rot, interleaved != 0, elem_size(dtype));
    if (int rc = by_dtype(dtype, [&](auto tag) { return launch_rope_backward<decltype(tag)>(p, g, D, interleaved != 0, streaming, (hipStream_t)stream); }))
      return rc;
  }
  if (!weights) return KV_OK;
  RopeSumParams s{};   // (with no row the weights' gradients are zeros)
  s.part = p.part; s.dq = dq_weight; s.dk = dk_weight; s.D = D; s.f32 = weights_f32 != 0;
  if (any) s.q_parts = g.q_chunks * g.blocks, s.k_parts = g.k_chunks * g.blocks;
  return by_dtype(dtype, [&](auto tag) { return launch_rope_sum<decltype(tag)>(s, (hipStream_t)stream); });
}

int kv_paged_append_rope(const void* q, const void* k, const void* v, void* q_out, void* k_pages, void* v_pages, const int32_t* page_table,
                         int64_t table_stride, const int32_t* lens, int64_t lens_stride, const int32_t* new_lens, int64_t new_lens_stride,
                         const float* cos, const float* sin, int64_t cos_stride, int64_t sin_stride, const void* q_weight,
                         const void* k_weight, int weights_f32, const int32_t* positions, const int64_t* position_strides, const int64_t* qs,
                         const int64_t* ks, const int64_t* vs, const int64_t* kps, const int64_t* vps, int B, int Hq, int Hkv, int T, int D,
                         int num_pages, int page_size, int width, int rot, int table_rows, int interleaved, float eps, int dtype,
                         void* stream) {
  if (int rc = check_rope(B, Hq, Hkv, T, D, rot, table_rows, eps, dtype)) return rc;
  if (num_pages < 0 || page_size < 1 || width < 0) return KV_ERR_ARG;
  if ((int64_t)width * page_size > (int64_t(1) << 30)) return KV_ERR_TOO_LARGE;
  if (B == 0 || T == 0 || Hq + Hkv == 0) return KV_OK;
  AppendRopeParams p{};
  if (Hq > 0) {
    if (int rc = check_layout(q, qs, dtype, T, false)) return rc;
    if (int rc = check_out(q_out)) return rc;
    p.q_sb = qs[0]; p.q_sh = qs[1]; p.q_st = qs[2];
  }
  const bool cache = Hkv > 0 && num_pages > 0 && width > 0;   // else there is no place for a key
  if (cache) {
    if (int rc = check_layout(k, ks, dtype, T, false)) return rc;
    if (int rc = check_layout(v, vs, dtype, T, false)) return rc;
    if (int rc = check_layout(k_pages, kps, dtype, page_size, false)) return rc;
    if (int rc = check_layout(v_pages, vps, dtype, page_size, false)) return rc;
    if (!page_table) return KV_ERR_ARG;
    for (const int64_t* s : {kps, vps})   // each place of the cache its own
      if ((s[0] == 0 && num_pages > 1) || (s[1] == 0 && Hkv > 1)) return KV_ERR_LAYOUT;
    p.k_sb = ks[0]; p.k_sh = ks[1]; p.k_st = ks[2];
    p.v_sb = vs[0]; p.v_sh = vs[1]; p.v_st = vs[2];
    p.kp_sp = kps[0]; p.kp_sh = kps[1]; p.kp_st = kps[2];
    p.vp_sp = vps[0]; p.vp_sh = vps[1]; p.vp_st = vps[2];
  } else if (Hq == 0) {
    return KV_OK;
  }
  if (!lens || (positions && !position_strides)) return KV_ERR_ARG;
  if (int rc = check_table(cos, sin, cos_stride, sin_stride, table_rows)) return rc;
  if (int rc = check_weights(q_weight, k_weight, eps)) return rc;
  p.q = q; p.k = k; p.v = v; p.q_out = q_out; p.k_pages = k_pages; p.v_pages = v_pages;
  p.q_weight = q_weight; p.k_weight = k_weight; p.weights_f32 = weights_f32 != 0;
  p.table = RopeTable{cos, sin, cos_stride, sin_stride, table_rows, rot};
  p.lens = lens; p.new_lens = new_lens; p.positions = positions; p.page_table = page_table;
  p.lens_stride = lens_stride; p.new_lens_stride = new_lens_stride; p.table_sb = table_stride;
  if (positions) p.pos_sb = position_strides[0], p.pos_st = position_strides[1];
  p.B = B; p.Hq = Hq; p.Hkv = cache ? Hkv : 0; p.T = T; p.width = width; p.num_pages = num_pages; p.page = page_size;
  p.eps = eps;
  p.by_tokens = chunk_div(T); p.by_page = chunk_div(page_size);
  const RopeGrid g = forward_grid((int64_t)B * T, Hq, p.Hkv, D, elem_size(dtype));
  p.chunk = g.chunk; p.q_chunks = g.q_chunks; p.k_chunks = g.k_chunks;
  const bool streaming = past_caches((int64_t)B * (Hq + 2 * p.Hkv) * T, D, rot, interleaved != 0, elem_size(dtype));
  return by_dtype(dtype, [&](auto tag) { return launch_append_rope<decltype(tag)>(p, g, D, interleaved != 0, streaming, (hipStream_t)stream); });
}

}  // extern "C"
