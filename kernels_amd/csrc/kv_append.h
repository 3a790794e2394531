// The keys and values of new tokens into a cache in pages, and accepted ones to the front of them.
#pragma once
#include "kv_common.h"

namespace kv {

// Token i of n = new_lens[b] of sequence b goes to position lens[b] - n + i.  Positions below 0 or past the table, and pages that are not there, are
// left out.  Bytes only: one thread moves sixteen of K and sixteen of V; consecutive threads go through the chunks of a row, then the tokens of
// a head.  Bound by memory: prompts of up to 2048 tokens for 8 sequences of 8 heads, D = 128, bfloat16 (67 MB read and written) 10.9-15.0 us,
// 4.5-6.2 TB/s over several GPUs, with stores past the caches; on one of them 12.9, and 16.1 with plain stores, which a call keeps whose rows stay in
// the L2 for the attention that follows; two or four pieces to a thread took 19 and 27 there.
struct AppendParams {
  const char *k, *v;
  char *k_pages, *v_pages;
  const int32_t *lens, *new_lens, *table;
  int64_t lens_stride, new_lens_stride, table_sb;
  int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;         // bytes
  int64_t kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;   // bytes
  int B, H, T, width, num_pages, page;
  int64_t total;          // B * H * T * chunks of a row
  ChunkDiv by_chunks, by_tokens, by_heads, by_page;
  int chunks;
};
template <bool STREAMING> __global__ __launch_bounds__(256) void append_kernel(const AppendParams p) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= p.total) return;
  const int x = div_by((int)id, p.by_chunks), chunk = (int)id - x * p.chunks;
  const int bh = div_by(x, p.by_tokens), t = x - bh * p.T;
  const int b = div_by(bh, p.by_heads), hd = bh - b * p.H;
  const int n = clamped_length(p.new_lens, p.new_lens_stride, b, p.T);
  const int64_t at = (int64_t)p.lens[b * p.lens_stride] - n + t;
  if (t >= n || at < 0 || at >= (int64_t)p.width * p.page) return;
  const int entry = div_by((int)at, p.by_page);
  const int32_t to = p.table[b * p.table_sb + entry];
  if ((uint32_t)to >= (uint32_t)p.num_pages) return;
  const int slot = (int)at - entry * p.page;
  const u32x4 kx = *reinterpret_cast<const u32x4*>(p.k + b * p.k_sb + hd * p.k_sh + t * p.k_st + chunk * 16);
  const u32x4 vx = *reinterpret_cast<const u32x4*>(p.v + b * p.v_sb + hd * p.v_sh + t * p.v_st + chunk * 16);
  char* const kp = p.k_pages + to * p.kp_sp + hd * p.kp_sh + slot * p.kp_st + chunk * 16;
  char* const vp = p.v_pages + to * p.vp_sp + hd * p.vp_sh + slot * p.vp_st + chunk * 16;
  if constexpr (STREAMING) {
    sa::store_streaming(kp, kx);
    sa::store_streaming(vp, vx);
  } else {
    *reinterpret_cast<u32x4*>(kp) = kx;
    *reinterpret_cast<u32x4*>(vp) = vx;
  }
}

// ---- accepted tokens --------------------------------------------------------------------------------------------------
// K and V of position first[b] + kept[b][i] to first[b] + i, for i = 0, 1, ... as long as the entries are not negative and ascend.  Bytes only.  An
// entry is never below its place, so what is read for one place is not written by a place before it: a thread goes through
// the places of one sixteen bytes of one head, a few loads ahead of its stores, and needs no other thread.
struct KeepParams {
  char *k_pages, *v_pages;
  const int32_t *first, *kept, *table;
  int64_t first_stride, kept_sb, kept_si, table_sb;
  int64_t kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;   // bytes
  int B, H, M, width, num_pages, page, chunks;
  int64_t total;          // B * H * chunks of a row
  ChunkDiv by_chunks, by_heads, by_page;
};
static __global__ __launch_bounds__(256) void keep_kernel(const KeepParams p) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= p.total) return;
  const bool values = blockIdx.y == 1;
  const int bh = div_by((int)id, p.by_chunks), chunk = (int)id - bh * p.chunks, b = div_by(bh, p.by_heads), hd = bh - b * p.H;
  char* const base = values ? p.v_pages + hd * p.vp_sh + chunk * 16 : p.k_pages + hd * p.kp_sh + chunk * 16;
  const int64_t sp = values ? p.vp_sp : p.kp_sp, st = values ? p.vp_st : p.kp_st;
  const int64_t first = p.first[b * p.first_stride], most = (int64_t)p.width * p.page;
  constexpr int U = 8;     // entries, then the pages of both places, then the bytes are on their way together; no branches around loads
  int before = -1;
  for (int i0 = 0; i0 < p.M; i0 += U) {
    int32_t entry[U], page[2 * U];
    int64_t at[2 * U];     // places that are read, and written; -1 past the table
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) entry[u] = p.kept[b * p.kept_sb + (i0 + u < p.M ? i0 + u : p.M - 1) * p.kept_si];
    bool on = true;        // still on the path
    uint32_t path = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      on = on && i0 + u < p.M && entry[u] > before;
      before = on ? entry[u] : before;
      path |= (on ? 1u : 0u) << u;
      at[u] = first + entry[u], at[U + u] = first + i0 + u;
    }
#pragma unroll
    for (int v = 0; v < 2 * U; ++v) {
      at[v] = at[v] >= 0 && at[v] < most ? at[v] : -1;
      page[v] = p.table[b * p.table_sb + div_by(at[v] < 0 ? 0 : (int)at[v], p.by_page)];
    }
#pragma unroll
    for (int v = 0; v < 2 * U; ++v) {   // to bytes from the base; what has no place, the first bytes (they are there, and not used)
      const bool there = at[v] >= 0 && (uint32_t)page[v] < (uint32_t)p.num_pages;
      if (!there) path &= ~(1u << v % U);
      const int k = there ? (int)at[v] : 0;
      at[v] = there ? page[v] * sp + (k - div_by(k, p.by_page) * p.page) * st : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const u32x4*>(base + at[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (path >> u & 1) *reinterpret_cast<u32x4*>(base + at[U + u]) = x[u];
    if (!on) return;
  }
}

}  // namespace kv
