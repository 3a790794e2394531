// extern "C" surface of libkv_attention.so: argument checks, workspace layout, parameter packing and dispatch on the element
// type.  See include/kv_attention.h for the contract.
#include "kv_append.h"
#include "kv_check.h"
#include "kv_launch.h"

using namespace kv;

namespace {

#define KV_LAUNCH(fn, p)                                                     \
  by_dtype(dtype, [&](auto tag) {                                            \
    using E = decltype(tag);                                                 \
    return D == 256 ? fn<E, 1>(p, D, (hipStream_t)stream) : fn<E, 0>(p, D, (hipStream_t)stream); \
  })

#ifdef SA_NO_ASM_KERNELS
#define KV_LAUNCH_LONG(fn, p) KV_ERR_ARG   // (no call comes here)
#else
#define KV_LAUNCH_LONG(fn, p) (dtype == 1 ? fn<_Float16>(p, (hipStream_t)stream) : fn<__bf16>(p, (hipStream_t)stream))
#endif

RowMap row_map(int Hkv, int G, int T) { return RowMap{Hkv, G, T, chunk_div(G)}; }
Work work_map(int64_t nbh, int64_t n_tiles, const Shares& sh, int heads, bool tiles_first) {
  Work w{};
  TileMap& m = w.map;
  m.n_tiles = (int)n_tiles * sh.splits;
  m.nbh = (int)nbh;
  m.by_tiles = m.by_lead = chunk_div(m.n_tiles);
  m.by_heads = chunk_div(heads);
  w.splits = sh.splits;
  w.share = sh.share;
  w.by_splits = chunk_div(sh.splits);
  w.tiles_first = tiles_first;
  w.by_pairs = m.by_pairs = chunk_div(nbh % 8 == 0 ? (int)(nbh >> 3) : (int)nbh);
  return w;
}

// How a cross attention is divided: rows kernel, or tiles of rows (and, for dK and dV, of keys).
struct CrossPlan {
  int64_t nbh, rows;
  Shares fwd, dq, dkdv;
  int key_tile, dq_key_tile, row_tile;   // of the forward, dQ, dK and dV
  bool few, long_rows, long_keys;        // the rows kernel; the hand-scheduled forward and dQ; dK and dV
  int64_t fwd_bytes, stats_bytes, dq_bytes, bwd_bytes;
  int fwd_rc, bwd_rc;                    // KV_ERR_TOO_LARGE where a launch of the forward, or of the backward, would have too many threads
};
// KV_ERR_TOO_LARGE where a count of the kernels would pass 31 bits
int plan_cross(CrossPlan& c, int B, int Hq, int Hkv, int Tq, int Tk, int D, int dtype) {
  if (int rc = check_sizes(B, Hq, Hkv, D, dtype)) return rc;
  if (Tq < 0 || Tk < 0) return KV_ERR_ARG;
  c = CrossPlan{};
  if (B == 0 || Hq == 0) return KV_OK;
  c.nbh = (int64_t)B * Hkv;
  c.rows = (int64_t)(Hq / Hkv) * Tq;
  if (c.nbh > kMostCount || c.rows > kMostCount - 1024 || Tk > kMostCount - 1024) return KV_ERR_TOO_LARGE;
  c.fwd = c.dq = c.dkdv = Shares{1, 1};
  const int row_bytes = D * elem_size(dtype), key_threads = dtype != 0 && D == 256 ? 512 : 256;
  if (Tq == 0) {   // nothing but zeros for dK and dV
    c.bwd_rc = launchable(c.nbh * ceil_div(Tk, TILE_ROWS), key_threads) ? KV_OK : KV_ERR_TOO_LARGE;
    return KV_OK;
  }
  c.key_tile = c.row_tile = row_bytes <= 256 ? 64 : 32;
  c.dq_key_tile = elem_size(dtype) == 2 ? 64 : c.key_tile;
  const int64_t row_tiles = ceil_div(c.rows, TILE_ROWS), key_tiles = ceil_div(Tk, TILE_ROWS);
  c.few = few_rows(c.rows);
  const bool hand_scheduled = HAVE_ASM_KERNELS && D == 128 && dtype != 0;
  c.long_rows = hand_scheduled && long_rows((int64_t)B * Hq, Tq, Tk);
  c.long_keys = hand_scheduled && long_keys(c.nbh, c.rows, Tk);
  if (c.few) {
    const int64_t tiles = ceil_div(Tk, 32);
    c.fwd.share = rows_share(c.nbh, (int)c.rows, tiles, row_bytes, dtype == 0, by_length(B, 1, row_bytes));
    c.fwd.splits = (int)std::max<int64_t>(1, ceil_div(tiles, c.fwd.share));
  } else if (!c.long_rows) {
    c.fwd = tile_shares(c.nbh * row_tiles, ceil_div(Tk, c.key_tile), row_places(row_bytes), false, dtype == 0);
  }
  if (!c.long_rows) c.dq = tile_shares(c.nbh * row_tiles, ceil_div(Tk, c.dq_key_tile), row_places(row_bytes), false, dtype == 0);
  c.dkdv = tile_shares(c.nbh * key_tiles, ceil_div(c.rows, c.row_tile), key_places(row_bytes), true, dtype == 0);
  const int64_t fwd_blocks = c.nbh * (c.few ? 1 : row_tiles) * c.fwd.splits;   // (the hand-scheduled kernels have fewer)
  const int fwd_threads = c.few ? 64 * rows_waves(row_bytes, dtype == 0, fwd_blocks, c.fwd.share) : 256;
  if (!launchable(fwd_blocks, fwd_threads)) c.fwd_rc = KV_ERR_TOO_LARGE;
  if (!launchable(c.nbh * row_tiles * c.dq.splits, 256) || !launchable(c.nbh * key_tiles * c.dkdv.splits, key_threads)) c.bwd_rc = KV_ERR_TOO_LARGE;
  if (std::max(c.fwd.splits, c.dq.splits) > 1 && c.nbh * c.rows > kMostCount) return KV_ERR_TOO_LARGE;
  if (c.dkdv.splits > 1 && c.nbh * Tk > kMostCount) return KV_ERR_TOO_LARGE;
  if (c.fwd.splits > 1) c.fwd_bytes = c.fwd.splits * c.nbh * c.rows * (D + 2) * 4;
  c.stats_bytes = ceil_div(c.nbh * c.rows * 4, 256) * 256;
  const int64_t dq = c.dq.splits > 1 ? c.dq.splits * c.nbh * c.rows * D * 4 : 0;
  const int64_t dkdv = c.dkdv.splits > 1 ? (int64_t)c.dkdv.splits * 2 * c.nbh * Tk * D * 4 : 0;
  c.dq_bytes = dq;
  c.bwd_bytes = 2 * c.stats_bytes + dq + dkdv;
  return KV_OK;
}
// The rows of one head within 32-bit byte offsets: what the hand-scheduled kernels need of q and d_o.
bool rows_fit(const int64_t* s, int64_t n, int dtype) { return s[2] <= ((int64_t(1) << 32) - 1) / elem_size(dtype) / (n + 1024); }

// The hand-scheduled forward and dQ: a workgroup owns LONG_ROWS queries of one head; the heads of a key head follow each other.
template <typename P> void long_sides(P& p, int B, int Hq, int Hkv, int Tq, int Tk) {
  p.B = B; p.H = Hq; p.T = Tq; p.C = 1; p.R = 0;
  p.cdiv = chunk_div(1);
  p.other_T = Tk;
  p.group = Hq / Hkv;
  p.q_tiles = (int)ceil_div(Tq, LONG_ROWS);
  p.by_q_tiles = chunk_div(p.q_tiles);
  p.tiles = work_map((int64_t)B * Hkv, (int64_t)p.group * p.q_tiles, Shares{1, 1}, Hkv, false).map;
}

// How the rows kernel goes through the pages.
struct PagedPlan {
  int64_t nbh, rows, row_tiles, bytes;
  bool by_rows;              // trees: the rows kernel, or that of tiles
  int splits, share, tile;   // at most that many parts, of up to `share` tiles of `tile` keys
};
int plan_paged(PagedPlan& c, int B, int Hq, int Hkv, int T, int D, int page, int width, int C, int R, int dtype) {
  if (int rc = check_sizes(B, Hq, Hkv, D, dtype)) return rc;
  if (T < 0 || page < 1 || width < 0 || C < 1 || R < 0) return KV_ERR_ARG;
  c = PagedPlan{};
  const int64_t most = (int64_t)width * page;
  if (most > (int64_t(1) << 30)) return KV_ERR_TOO_LARGE;
  if (B == 0 || Hq == 0 || T == 0) return KV_OK;
  const int G = Hq / Hkv;
  c.nbh = (int64_t)B * Hkv;
  c.rows = (int64_t)G * T;
  c.tile = 32;
  if (c.nbh > kMostCount || c.rows > kMostCount - 1024) return KV_ERR_TOO_LARGE;
  c.row_tiles = ceil_div(c.rows, 32);
  // the most keys that the rows of a tile see together: those of R + 1 chunks for each chunk that its tokens lie in
  const int64_t tokens = std::min<int64_t>(T, 31 / G + 2), chunks = ceil_div(tokens - 1, C) + 1;
  const int64_t span = R > most || C > most ? most : std::min<int64_t>(most, (R + chunks) * C);
  const int64_t tiles = std::min(ceil_div(most, 32), ceil_div(span, 32) + 1);
  const int row_bytes = D * elem_size(dtype);
  c.share = rows_share(c.nbh * c.row_tiles, (int)std::min<int64_t>(c.rows, 32), tiles, row_bytes, dtype == 0, by_length(B, c.row_tiles, row_bytes));
  c.splits = (int)std::max<int64_t>(1, ceil_div(tiles, c.share));
  const int64_t blocks = c.nbh * c.row_tiles * c.splits;
  if (!launchable(blocks, 64 * rows_waves(row_bytes, dtype == 0, blocks, c.share))) return KV_ERR_TOO_LARGE;
  if (c.splits > 1 && c.nbh * c.rows > kMostCount) return KV_ERR_TOO_LARGE;
  if (c.splits > 1) c.bytes = c.splits * c.nbh * c.rows * (D + 2) * 4;
  return KV_OK;
}

// Trees: the rows kernel, or tiles of rows.
int plan_tree(PagedPlan& c, int B, int Hq, int Hkv, int T, int D, int page, int width, int dtype) {
  if (int rc = plan_paged(c, B, Hq, Hkv, T, D, page, width, 1, 0x7fffffff, dtype)) return rc;
  const int row_bytes = D * elem_size(dtype), waves = tree_waves(c.rows);
  c.by_rows = tree_by_rows(c.nbh, c.rows, ceil_div((int64_t)width * page, 32), row_bytes, dtype == 0);
  if (c.by_rows) return KV_OK;
  c.tile = row_bytes <= 256 ? 64 : 32;
  c.row_tiles = ceil_div(c.rows, waves * 32);
  const int64_t tiles = ceil_div((int64_t)width * page, c.tile);
  c.share = tree_share(c.nbh * c.row_tiles, tiles, row_bytes, waves, dtype == 0);
  // at most 256 MiB of parts
  const int64_t part = c.nbh * c.rows * (D + 2) * 4;
  c.share = (int)std::max<int64_t>(c.share, ceil_div(tiles, std::max<int64_t>(1, (256 << 20) / part)));
  c.splits = (int)std::max<int64_t>(1, ceil_div(tiles, c.share));
  if (!launchable(c.nbh * c.row_tiles * c.splits, waves * 128)) return KV_ERR_TOO_LARGE;
  if (c.splits > 1 && c.nbh * c.rows > kMostCount) return KV_ERR_TOO_LARGE;
  c.bytes = c.splits > 1 ? c.splits * c.nbh * c.rows * (D + 2) * 4 : 0;
  return KV_OK;
}

// P: the parameters of the kernel that leaves the parts, runs of up to `share` tiles of `tile` keys
template <typename P> JoinParams join_params(const P& p, int max_len, int splits, int share, int tile) {
  JoinParams j{};
  j.part_o = p.part_o, j.part_ml = p.part_ml, j.o = p.o, j.lse = p.lse;
  j.lens = p.lens, j.q_lens = p.q_lens, j.lens_stride = p.lens_stride, j.q_lens_stride = p.q_lens_stride;
  j.map = p.map, j.B = p.B, j.max_len = max_len, j.splits = splits, j.share = share, j.tile = tile;
  const RowMap& map = p.map;
  j.by_rows = chunk_div(map.rows());
  j.by_heads = chunk_div(map.Hkv);
  return j;
}

// The rows kernel's parameters, without windows; width 0: no page can be there.
RowsParams paged_rows(const PagedPlan& c, const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table, int64_t table_stride,
                      const int32_t* lens, int64_t lens_stride, const int32_t* new_lens, int64_t new_lens_stride, void* o, float* lse,
                      void* workspace, const int64_t* qs, const int64_t* ks, const int64_t* vs, int B, int Hq, int Hkv, int T, int D,
                      int num_pages, int page_size, int width, float sm_scale) {
  RowsParams p{};
  p.q = q; p.k = k_pages; p.v = v_pages; p.o = o; p.lse = lse;
  p.lens = lens; p.q_lens = new_lens; p.lens_stride = lens_stride; p.q_lens_stride = new_lens_stride;
  p.q_sb = qs[0]; p.q_sh = qs[1]; p.q_st = qs[2];
  p.map = row_map(Hkv, Hq / Hkv, T); p.B = B; p.scale_log2e = sm_scale * kLog2e;
  p.page = page_size; p.by_page = chunk_div(page_size);
  if (width > 0) {
    p.k_sp = ks[0]; p.k_sh = ks[1]; p.k_st = ks[2];
    p.v_sp = vs[0]; p.v_sh = vs[1]; p.v_st = vs[2];
    p.table = page_table; p.table_sb = table_stride; p.width = width; p.num_pages = num_pages;
    p.max_len = width * page_size;
  }
  p.splits = c.splits; p.share = c.share; p.row_tiles = (int)c.row_tiles;
  p.by_pairs = chunk_div((int)c.nbh); p.by_row_tiles = chunk_div(p.row_tiles); p.by_heads = chunk_div(Hkv);
  p.part_o = (float*)workspace;
  p.part_ml = p.part_o + c.splits * c.nbh * c.rows * D;
  return p;
}

}  // namespace

extern "C" {

int64_t kv_cross_forward_workspace(int B, int Hq, int Hkv, int Tq, int Tk, int D, int dtype) {
  CrossPlan c;
  if (int rc = plan_cross(c, B, Hq, Hkv, Tq, Tk, D, dtype)) return rc;
  return c.fwd_rc ? c.fwd_rc : c.fwd_bytes;
}

int kv_cross_forward(const void* q, const void* k, const void* v, const int32_t* lens, int64_t lens_stride, const int32_t* q_lens,
                     int64_t q_lens_stride, void* o, float* lse, void* workspace, int64_t workspace_bytes, const int64_t* qs,
                     const int64_t* ks, const int64_t* vs, int B, int Hq, int Hkv, int Tq, int Tk, int D, float sm_scale, int dtype,
                     void* stream) {
  CrossPlan c;
  if (int rc = plan_cross(c, B, Hq, Hkv, Tq, Tk, D, dtype)) return rc;
  if (c.fwd_rc) return c.fwd_rc;
  if (int rc = check_scale(sm_scale)) return rc;
  if (B == 0 || Hq == 0 || Tq == 0) return KV_OK;
  if (int rc = check_layout(q, qs, dtype, Tq, false)) return rc;
  if (Tk > 0) {
    if (int rc = check_layout(k, ks, dtype, Tk, true)) return rc;
    if (int rc = check_layout(v, vs, dtype, Tk, true)) return rc;
  }
  if (int rc = check_out(o)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, c.fwd_bytes)) return rc;
  const RowMap map = row_map(Hkv, Hq / Hkv, Tq);
  float* const part_o = (float*)workspace;
  float* const part_ml = part_o + c.fwd.splits * c.nbh * c.rows * D;
  if (c.few) {
    RowsParams p{};
    p.q = q; p.k = k; p.v = v; p.o = o; p.lse = lse;
    p.lens = lens; p.q_lens = q_lens; p.lens_stride = lens_stride; p.q_lens_stride = q_lens_stride;
    p.q_sb = qs[0]; p.q_sh = qs[1]; p.q_st = qs[2];
    if (Tk > 0) {
      p.k_sp = ks[0]; p.k_sh = ks[1]; p.k_st = ks[2];
      p.v_sp = vs[0]; p.v_sh = vs[1]; p.v_st = vs[2];
    }
    p.map = map; p.B = B; p.max_len = Tk; p.scale_log2e = sm_scale * kLog2e;
    p.splits = c.fwd.splits; p.share = c.fwd.share; p.row_tiles = 1;
    p.by_pairs = chunk_div((int)c.nbh); p.by_row_tiles = chunk_div(1); p.by_heads = chunk_div(Hkv);
    p.part_o = part_o; p.part_ml = part_ml;
    if (int rc = KV_LAUNCH(launch_rows, p)) return rc;
    if (c.fwd.splits == 1) return KV_OK;
    const JoinParams j = join_params(p, Tk, c.fwd.splits, c.fwd.share, 32);
    return KV_LAUNCH(launch_join, j);
  } else if (c.long_rows && Tk > 0 && rows_fit(qs, Tq, dtype)) {
    LongFwd p{};
    p.q = q; p.k = k; p.v = v; p.o = o; p.lse = lse;
    p.lens = q_lens; p.lens_stride = q_lens_stride; p.other_lens = lens; p.other_lens_stride = lens_stride;
    p.q_sb = qs[0]; p.q_sh = qs[1]; p.q_st = qs[2];
    p.k_sb = ks[0]; p.k_sh = ks[1]; p.k_st = ks[2];
    p.v_sb = vs[0]; p.v_sh = vs[1]; p.v_st = vs[2];
    p.scale_log2e = sm_scale * kLog2e;
    long_sides(p, B, Hq, Hkv, Tq, Tk);
    return KV_LAUNCH_LONG(launch_long_fwd, p);
  } else {
    FwdParams p{};
    p.q = q; p.k = k; p.v = v; p.o = o; p.lse = lse;
    p.lens = lens; p.q_lens = q_lens; p.lens_stride = lens_stride; p.q_lens_stride = q_lens_stride;
    p.q_sb = qs[0]; p.q_sh = qs[1]; p.q_st = qs[2];
    if (Tk > 0) {
      p.k_sb = ks[0]; p.k_sh = ks[1]; p.k_st = ks[2];
      p.v_sb = vs[0]; p.v_sh = vs[1]; p.v_st = vs[2];
    }
    p.map = map; p.B = B; p.Tk = Tk; p.scale_log2e = sm_scale * kLog2e;
    const int64_t tiles = ceil_div(c.rows, TILE_ROWS);
    p.work = work_map(c.nbh, tiles, c.fwd, Hkv, tiles_first(tiles));
    p.part_o = part_o; p.part_ml = part_ml;
    if (int rc = KV_LAUNCH(launch_cross_fwd, p)) return rc;
    if (c.fwd.splits == 1) return KV_OK;
    const JoinParams j = join_params(p, Tk, c.fwd.splits, c.fwd.share, c.key_tile);
    return KV_LAUNCH(launch_join, j);
  }
}

int64_t kv_cross_backward_workspace(int B, int Hq, int Hkv, int Tq, int Tk, int D, int dtype) {
  CrossPlan c;
  if (int rc = plan_cross(c, B, Hq, Hkv, Tq, Tk, D, dtype)) return rc;
  return c.bwd_rc ? c.bwd_rc : c.bwd_bytes;
}

int kv_cross_backward(const void* q, const void* k, const void* v, const int32_t* lens, int64_t lens_stride, const int32_t* q_lens,
                      int64_t q_lens_stride, const void* o, const void* d_o, const float* lse, void* dq, void* dk, void* dv,
                      void* workspace, int64_t workspace_bytes, const int64_t* qs, const int64_t* ks, const int64_t* vs,
                      const int64_t* os, const int64_t* gs, int B, int Hq, int Hkv, int Tq, int Tk, int D, float sm_scale, int dtype,
                      void* stream) {
  CrossPlan c;
  if (int rc = plan_cross(c, B, Hq, Hkv, Tq, Tk, D, dtype)) return rc;
  if (c.bwd_rc) return c.bwd_rc;
  if (int rc = check_scale(sm_scale)) return rc;
  if (B == 0 || Hq == 0) return KV_OK;
  if (Tq > 0) {
    const bool one_head = Hq == Hkv;
    if (int rc = check_layout(q, qs, dtype, Tq, one_head)) return rc;
    if (int rc = check_layout(d_o, gs, dtype, Tq, one_head)) return rc;
    if (int rc = check_layout(o, os, dtype, Tq, false)) return rc;
    if (!lse) return KV_ERR_ARG;
    if (int rc = check_out(dq)) return rc;
  }
  if (Tk > 0) {
    if (int rc = check_layout(k, ks, dtype, Tk, true)) return rc;
    if (int rc = check_layout(v, vs, dtype, Tk, true)) return rc;
    if (int rc = check_out(dk)) return rc;
    if (int rc = check_out(dv)) return rc;
  }
  if (int rc = check_workspace(workspace, workspace_bytes, c.bwd_bytes)) return rc;
  BwdParams p{};
  p.q = q; p.k = k; p.v = v; p.o = o; p.d_o = d_o; p.lse = lse; p.dq = dq; p.dk = dk; p.dv = dv;
  p.lens = lens; p.q_lens = q_lens; p.lens_stride = lens_stride; p.q_lens_stride = q_lens_stride;
  if (Tq > 0) {
    p.q_sb = qs[0]; p.q_sh = qs[1]; p.q_st = qs[2];
    p.o_sb = os[0]; p.o_sh = os[1]; p.o_st = os[2];
    p.g_sb = gs[0]; p.g_sh = gs[1]; p.g_st = gs[2];
  }
  if (Tk > 0) {
    p.k_sb = ks[0]; p.k_sh = ks[1]; p.k_st = ks[2];
    p.v_sb = vs[0]; p.v_sh = vs[1]; p.v_st = vs[2];
  }
  p.map = row_map(Hkv, Hq / Hkv, Tq); p.B = B; p.Tk = Tk;
  p.scale = sm_scale; p.scale_log2e = sm_scale * kLog2e;
  p.row_lse = (float*)workspace;
  p.row_delta = (float*)((char*)workspace + c.stats_bytes);
  p.part = (float*)((char*)workspace + 2 * c.stats_bytes);

  const int G = Hq / Hkv;
  // The hand-scheduled dK/dV kernel goes through the rows of all heads at one stride: one head, or heads that follow each other without
  // padding inside them.
  const bool one_run = Tq > 0 && rows_fit(qs, c.rows, dtype) && rows_fit(gs, c.rows, dtype) &&
                       (G == 1 || (!q_lens && qs[1] == Tq * qs[2] && gs[1] == Tq * gs[2]));
  const bool keys_by_hand = c.long_keys && one_run;
  LongBwd r{};
  if ((c.long_rows || c.long_keys) && Tq > 0 && Tk > 0) {
    r.q = q; r.k = k; r.v = v; r.d_o = d_o;
    r.scale = p.scale; r.scale_log2e = p.scale_log2e;
    r.q_sb = qs[0]; r.q_sh = qs[1]; r.q_st = qs[2];
    r.k_sb = ks[0]; r.k_sh = ks[1]; r.k_st = ks[2];
    r.v_sb = vs[0]; r.v_sh = vs[1]; r.v_st = vs[2];
    r.do_sb = gs[0]; r.do_sh = gs[1]; r.do_st = gs[2];
  }
  if (c.long_rows && Tk > 0 && rows_fit(qs, Tq, dtype) && rows_fit(gs, Tq, dtype)) {
    LongBwd d = r;
    d.lse = lse; d.dq = dq; d.o = o;
    d.o_sb = os[0]; d.o_sh = os[1]; d.o_st = os[2];
    d.lens = q_lens; d.lens_stride = q_lens_stride; d.other_lens = lens; d.other_lens_stride = lens_stride;
    d.delta_out = p.row_delta; d.lse_out = p.row_lse;
    d.token_major = !keys_by_hand;
    long_sides(d, B, Hq, Hkv, Tq, Tk);
    if (int rc = KV_LAUNCH_LONG(launch_long_dq, d)) return rc;
    c.dq.splits = 1;
  } else if (Tq > 0) {
    const int64_t tiles = ceil_div(c.rows, TILE_ROWS);
    p.head_major = keys_by_hand;
    p.work = work_map(c.nbh, tiles, c.dq, Hkv, tiles_first(tiles));
    if (int rc = KV_LAUNCH(launch_cross_dq, p)) return rc;
  }
  SumParams s{};
  s.lens = lens; s.q_lens = q_lens; s.lens_stride = lens_stride; s.q_lens_stride = q_lens_stride;
  s.B = B; s.Hkv = Hkv; s.Tk = Tk; s.Tq = Tq; s.group = G; s.by_heads = chunk_div(Hkv);
  if (c.dq.splits > 1) {
    SumSide& x = s.queries;
    x.part = p.part; x.map = p.map; x.out[0] = dq; x.step = c.nbh * c.rows * D;
    x.share = c.dq.share; x.tile = c.dq_key_tile; x.by_rows = chunk_div((int)c.rows);
    s.first_keys = 1;
  }
  if (Tk > 0 && keys_by_hand) {
    r.lse = p.row_lse; r.delta = p.row_delta; r.dk = dk; r.dv = dv;
    r.lens = lens; r.lens_stride = lens_stride; r.other_lens = q_lens; r.other_lens_stride = q_lens_stride;
    r.B = B; r.H = Hkv; r.T = Tk; r.C = 1; r.R = 0;
    r.cdiv = chunk_div(1);
    r.other_T = (int)c.rows;
    r.group = G;
    r.tiles = work_map(c.nbh, ceil_div(Tk, TILE_ROWS), Shares{1, 1}, Hkv, false).map;
    if (int rc = KV_LAUNCH_LONG(launch_long_dkdv, r)) return rc;
  } else if (Tk > 0) {
    p.part = (float*)((char*)p.part + c.dq_bytes);
    p.work = work_map(c.nbh, ceil_div(Tk, TILE_ROWS), c.dkdv, Hkv, false);
    if (int rc = KV_LAUNCH(launch_cross_dkdv, p)) return rc;
    if (c.dkdv.splits > 1) {
      SumSide& x = s.keys;
      x.part = p.part; x.map = row_map(Hkv, 1, Tk); x.out[0] = dk; x.out[1] = dv;
      x.second = c.nbh * Tk * D; x.step = 2 * x.second;
      x.share = c.dkdv.share; x.tile = c.row_tile; x.by_rows = chunk_div(Tk);
    }
  }
  return s.first_keys > 0 || s.keys.part ? KV_LAUNCH(launch_sum, s) : KV_OK;
}

int64_t kv_paged_forward_workspace(int B, int Hq, int Hkv, int T, int D, int page_size, int width, int context_size, int back_contexts,
                                   int dtype) {
  PagedPlan c;
  if (int rc = plan_paged(c, B, Hq, Hkv, T, D, page_size, width, context_size, back_contexts, dtype)) return rc;
  return c.bytes;
}

int kv_paged_forward(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table, int64_t table_stride,
                     const int32_t* lens, int64_t lens_stride, const int32_t* new_lens, int64_t new_lens_stride, void* o, float* lse,
                     void* workspace, int64_t workspace_bytes, const int64_t* qs, const int64_t* ks, const int64_t* vs, int B, int Hq,
                     int Hkv, int T, int D, int num_pages, int page_size, int width, int context_size, int back_contexts, float sm_scale,
                     int dtype, void* stream) {
  PagedPlan c;
  if (int rc = plan_paged(c, B, Hq, Hkv, T, D, page_size, width, context_size, back_contexts, dtype)) return rc;
  if (num_pages < 0) return KV_ERR_ARG;
  if (int rc = check_scale(sm_scale)) return rc;
  if (B == 0 || Hq == 0 || T == 0) return KV_OK;
  if (int rc = check_layout(q, qs, dtype, T, false)) return rc;
  if (!lens) return KV_ERR_ARG;
  const bool empty = num_pages == 0 || width == 0;   // no page can be there: no key is seen
  if (!empty) {
    if (!page_table) return KV_ERR_ARG;
    if (int rc = check_layout(k_pages, ks, dtype, page_size, false)) return rc;
    if (int rc = check_layout(v_pages, vs, dtype, page_size, false)) return rc;
  }
  if (int rc = check_out(o)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, c.bytes)) return rc;
  RowsParams p = paged_rows(c, q, k_pages, v_pages, page_table, table_stride, lens, lens_stride, new_lens, new_lens_stride, o, lse, workspace,
                            qs, ks, vs, B, Hq, Hkv, T, D, empty ? 0 : num_pages, page_size, empty ? 0 : width, sm_scale);
  // chunks matter below the longest length only
  const int most = width * page_size;
  p.win.C = std::max(1, std::min(context_size, most));
  p.win.R = std::min(back_contexts, most);
  p.win.cdiv = chunk_div(p.win.C);
  if (int rc = KV_LAUNCH(launch_rows_paged, p)) return rc;
  if (c.splits == 1) return KV_OK;
  JoinParams j = join_params(p, p.max_len, c.splits, c.share, 32);
  j.win = p.win;
  return KV_LAUNCH(launch_join, j);
}

int64_t kv_paged_tree_forward_workspace(int B, int Hq, int Hkv, int T, int D, int page_size, int width, int dtype) {
  PagedPlan c;
  if (int rc = plan_tree(c, B, Hq, Hkv, T, D, page_size, width, dtype)) return rc;
  return c.bytes;
}

int kv_paged_tree_forward(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table, int64_t table_stride,
                          const int32_t* lens, int64_t lens_stride, const int32_t* new_lens, int64_t new_lens_stride, const void* tree,
                          const int64_t* ts, void* o, float* lse, void* workspace, int64_t workspace_bytes, const int64_t* qs, const int64_t* ks,
                          const int64_t* vs, int B, int Hq, int Hkv, int T, int D, int num_pages, int page_size, int width, float sm_scale,
                          int dtype, void* stream) {
  PagedPlan c;
  if (int rc = plan_tree(c, B, Hq, Hkv, T, D, page_size, width, dtype)) return rc;
  if (num_pages < 0) return KV_ERR_ARG;
  if (int rc = check_scale(sm_scale)) return rc;
  if (B == 0 || Hq == 0 || T == 0) return KV_OK;
  if (int rc = check_layout(q, qs, dtype, T, false)) return rc;
  if (!lens || !tree || !ts) return KV_ERR_ARG;
  const bool empty = num_pages == 0 || width == 0;   // no page can be there: no key is seen
  if (!empty) {
    if (!page_table) return KV_ERR_ARG;
    if (int rc = check_layout(k_pages, ks, dtype, page_size, false)) return rc;
    if (int rc = check_layout(v_pages, vs, dtype, page_size, false)) return rc;
  }
  if (int rc = check_out(o)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, c.bytes)) return rc;
  TreeParams p{paged_rows(c, q, k_pages, v_pages, page_table, table_stride, lens, lens_stride, new_lens, new_lens_stride, o, lse, workspace,
                            qs, ks, vs, B, Hq, Hkv, T, D, empty ? 0 : num_pages, page_size, empty ? 0 : width, sm_scale)};
  p.tree = Tree{(const uint8_t*)tree, ts[0], ts[1], ts[2]};
  if (int rc = c.by_rows ? KV_LAUNCH(launch_rows_tree, p) : KV_LAUNCH(launch_tree, p)) return rc;
  if (c.splits == 1) return KV_OK;
  const JoinParams j = join_params(p, p.max_len, c.splits, c.share, c.tile);
  // many rows fill the GPU by themselves: 16384 of up to 16 parts, D = 128 22 -> 9 us; 512 of 64: 4.4 -> 8
  return c.nbh * c.rows >= 4096 ? KV_LAUNCH(launch_join_many, j) : KV_LAUNCH(launch_join, j);
}

int kv_paged_append(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* page_table, int64_t table_stride,
                    const int32_t* lens, int64_t lens_stride, const int32_t* new_lens, int64_t new_lens_stride, const int64_t* ks,
                    const int64_t* vs, const int64_t* kps, const int64_t* vps, int B, int H, int T, int D, int num_pages, int page_size,
                    int width, int dtype, void* stream) {
  if (int rc = check_sizes(B, H, H, D, dtype)) return rc;
  if (T < 0 || num_pages < 0 || page_size < 1 || width < 0) return KV_ERR_ARG;
  if ((int64_t)width * page_size > (int64_t(1) << 30)) return KV_ERR_TOO_LARGE;
  if (B == 0 || H == 0 || T == 0 || num_pages == 0 || width == 0) return KV_OK;
  if (int rc = check_layout(k, ks, dtype, T, false)) return rc;
  if (int rc = check_layout(v, vs, dtype, T, false)) return rc;
  if (int rc = check_layout(k_pages, kps, dtype, page_size, false)) return rc;
  if (int rc = check_layout(v_pages, vps, dtype, page_size, false)) return rc;
  if (!lens || !page_table) return KV_ERR_ARG;
  for (const int64_t* s : {kps, vps})   // each place of the cache its own
    if ((s[0] == 0 && num_pages > 1) || (s[1] == 0 && H > 1)) return KV_ERR_LAYOUT;
  const int64_t es = elem_size(dtype);
  AppendParams p{};
  p.k = (const char*)k; p.v = (const char*)v; p.k_pages = (char*)k_pages; p.v_pages = (char*)v_pages;
  p.lens = lens; p.new_lens = new_lens; p.table = page_table;
  p.lens_stride = lens_stride; p.new_lens_stride = new_lens_stride; p.table_sb = table_stride;
  p.k_sb = ks[0] * es; p.k_sh = ks[1] * es; p.k_st = ks[2] * es;
  p.v_sb = vs[0] * es; p.v_sh = vs[1] * es; p.v_st = vs[2] * es;
  p.kp_sp = kps[0] * es; p.kp_sh = kps[1] * es; p.kp_st = kps[2] * es;
  p.vp_sp = vps[0] * es; p.vp_sh = vps[1] * es; p.vp_st = vps[2] * es;
  p.B = B; p.H = H; p.T = T; p.width = width; p.num_pages = num_pages; p.page = page_size;
  p.chunks = (int)(D * es / 16);
  if ((int64_t)B * H > kMostCount || (int64_t)B * H * T > kMostCount / p.chunks) return KV_ERR_TOO_LARGE;
  p.total = (int64_t)B * H * T * p.chunks;
  p.by_chunks = chunk_div(p.chunks); p.by_tokens = chunk_div(T); p.by_heads = chunk_div(H); p.by_page = chunk_div(page_size);
  const bool streaming = p.total * 32 > (int64_t(32) << 20);   // more than the L2s of all XCDs hold
  (streaming ? append_kernel<true> : append_kernel<false>)<<<dim3((unsigned)ceil_div(p.total, 256)), dim3(256), 0, (hipStream_t)stream>>>(p);
  return (int)hipGetLastError();
}

int kv_paged_keep(void* k_pages, void* v_pages, const int32_t* page_table, int64_t table_stride, const int32_t* first, int64_t first_stride,
                  const int32_t* kept, const int64_t* kept_strides, const int64_t* kps, const int64_t* vps, int B, int H, int M, int D,
                  int num_pages, int page_size, int width, int dtype, void* stream) {
  if (int rc = check_sizes(B, H, H, D, dtype)) return rc;
  if (M < 0 || num_pages < 0 || page_size < 1 || width < 0) return KV_ERR_ARG;
  if ((int64_t)width * page_size > (int64_t(1) << 30)) return KV_ERR_TOO_LARGE;
  if (B == 0 || H == 0 || M == 0 || num_pages == 0 || width == 0) return KV_OK;
  if (int rc = check_layout(k_pages, kps, dtype, page_size, false)) return rc;
  if (int rc = check_layout(v_pages, vps, dtype, page_size, false)) return rc;
  if (!first || !kept || !kept_strides || !page_table) return KV_ERR_ARG;
  for (const int64_t* s : {kps, vps})   // each place of the cache its own
    if ((s[0] == 0 && num_pages > 1) || (s[1] == 0 && H > 1)) return KV_ERR_LAYOUT;
  const int64_t es = elem_size(dtype);
  KeepParams p{};
  p.k_pages = (char*)k_pages; p.v_pages = (char*)v_pages;
  p.first = first; p.kept = kept; p.table = page_table;
  p.first_stride = first_stride; p.kept_sb = kept_strides[0]; p.kept_si = kept_strides[1]; p.table_sb = table_stride;
  p.kp_sp = kps[0] * es; p.kp_sh = kps[1] * es; p.kp_st = kps[2] * es;
  p.vp_sp = vps[0] * es; p.vp_sh = vps[1] * es; p.vp_st = vps[2] * es;
  p.B = B; p.H = H; p.M = M; p.width = width; p.num_pages = num_pages; p.page = page_size;
  p.chunks = (int)(D * es / 16);
  if ((int64_t)B * H > kMostCount / p.chunks) return KV_ERR_TOO_LARGE;
  p.total = (int64_t)B * H * p.chunks;
  p.by_chunks = chunk_div(p.chunks); p.by_heads = chunk_div(H); p.by_page = chunk_div(page_size);
  // keys that are the values too move once: the second set of threads would read what the first has written
  const bool one = k_pages == v_pages && p.kp_sp == p.vp_sp && p.kp_sh == p.vp_sh && p.kp_st == p.vp_st;
  keep_kernel<<<dim3((unsigned)ceil_div(p.total, 256), one ? 1 : 2), dim3(256), 0, (hipStream_t)stream>>>(p);
  return (int)hipGetLastError();
}

const char* kv_error_string(int code) {
  switch (code) {
    case KV_OK: return "success";
    case KV_ERR_DTYPE: return "unsupported dtype id (0 = float32, 1 = float16, 2 = bfloat16)";
    case KV_ERR_HEAD_DIM: return "head dimension must be one of 16, 32, 64, 128, 256";
    case KV_ERR_ARG: return "invalid argument (null pointer, negative size, Hq not a multiple of Hkv, page_size or context_size < 1, "
                            "back_contexts < 0, a scale beyond 2^127, rot or eps out of range, weights without norms)";
    case KV_ERR_LAYOUT: return "unsupported layout (dim stride must be 1; pointers and strides 16-byte aligned, strides not negative)";
    case KV_ERR_TOO_LARGE: return "problem too large for one launch";
    case KV_ERR_WORKSPACE: return "workspace missing or smaller than the *_workspace function says";
  }
  return code > 0 ? hipGetErrorString((hipError_t)code) : "unknown error";
}

}  // extern "C"
