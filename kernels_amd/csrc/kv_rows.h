// Attention of a few rows over a long run of keys: one decoding step over an encoder's states, or the newest tokens of every
// sequence over a cache in pages; and the joining of work that was split over the keys.
//
// The rows kernel is bound by reading K and V once.  A workgroup owns 32 rows (kv_common.h: up to 32 query heads of a key head, or a few
// tokens) and a run of keys.  Its waves go through tiles of 32 keys by themselves, every NW-th each, without a barrier: a wave keeps ST
// tiles of K and V on their way into LDS of its own, at addresses that each lane forms for its row, and joins the other waves at the end.
// The products are those of the tile kernels, on matrix instructions whatever the number of rows: at one row they run
// at a tenth of what the memory needs.  Batches of many lengths leave most of the parts that a sequence may have empty: with a workgroup for each
// (1 us even if empty, in a place of the few that the rings leave), shares had to be long, and the last ones ran alone; so the workgroups of
// rows_by_length_kernel find the parts that there are from the lengths.  One token, D = 128, us with a workgroup for each part -> by length: bfloat16,
// lengths log-uniform from 64 to 8192, 64 x 8 key heads 104 -> 95 (4.6 TB/s), 16 x 8 43 -> 31; float32, 32 x 8, log-uniform up to 3000 243 -> 100, from
// 1500 on 246 -> 228.  Sequences of one length pay for the gaps between the parts of a workgroup: bfloat16, all of 8192 16 x 8 99 -> 104, 64 x 8
// 363 -> 386; float32, all of 3000 248 -> 282.
#pragma once
#include "kv_fwd.h"

namespace kv {

// What the rows of a sequence see, of its first L keys: all of them (C = 0), or, in streaming, those of a row's chunk of C and the R chunks
// before it.
struct Windows {
  int C, R;
  ChunkDiv cdiv;
};
// Keys [lo, hi) of row r; the rows are those of the last `tokens` positions.
SA_BOTH void window_of(const Windows& w, const RowMap& map, int L, int tokens, int r, int& lo, int& hi) {
  int t, g;
  map.split(r, t, g);
  const int at = L - tokens + t, chunk = at < 0 ? 0 : div_by(at, w.cdiv);
  lo = (chunk > w.R ? chunk - w.R : 0) * w.C;
  hi = at < 0 ? 0 : (chunk + 1) * w.C < L ? (chunk + 1) * w.C : L;
}
// Tiles [first, last) of `tile` keys that some of the `used` rows from r0 on see.
SA_BOTH void tiles_seen(const Windows& w, const RowMap& map, int L, int tokens, int r0, int used, int tile, int& first, int& last) {
  int lo = 0, hi = L, ignored;
  if (w.C > 0) {
    window_of(w, map, L, tokens, r0, lo, ignored);
    window_of(w, map, L, tokens, r0 + used - 1, ignored, hi);
  }
  first = lo / tile, last = (hi + tile - 1) / tile;
  last = last > first ? last : first;
}

struct RowsParams {
  const void *q, *k, *v;
  void* o;               // contiguous [B, Hq, T, D]
  float* lse;            // contiguous [B, Hq, T] or null
  const int32_t *lens, *q_lens;
  int64_t lens_stride, q_lens_stride;
  int64_t q_sb, q_sh, q_st;
  int64_t k_sp, k_sh, k_st, v_sp, v_sh, v_st;   // sp: from page to page, or from batch entry to batch entry
  RowMap map;
  int B, max_len;
  float scale_log2e;
  // pages
  const int32_t* table;  // [B, width]
  int64_t table_sb;
  int width, num_pages, page;
  ChunkDiv by_page;
  Windows win;
  // division of the work
  int splits, share;     // the most parts that the tiles of 32 keys of a row tile are divided into, and the most tiles of a part
  int row_tiles;
  ChunkDiv by_pairs, by_row_tiles, by_heads;
  float* part_o;         // [splits, B * Hkv, rows, D]
  float* part_ml;        // [splits, B * Hkv, rows, 2]
};

// A wave's rings take 16 KiB at rows of 128 bytes; a workgroup has NW waves (rows_waves in kv_launch.h).
template <typename T, int D, int NW> struct RowsShape {
  static constexpr int ST = 2;                                         // tiles on their way; three leave room for one workgroup and are slower
  static constexpr int TILE = 32 * D;                                  // elements
  static constexpr int ENTRIES = 2 * ST * 64 * 4, OFFSETS = 64 * 8;    // bytes per wave, pages only
  static constexpr int OP = D + 4;                                     // floats per row of a wave's result
  static constexpr int RING = ST * 2 * TILE * (int)sizeof(T);          // bytes per wave
  static constexpr int bytes(bool paged) {
    const int ring = NW * (RING + (paged ? ENTRIES + OFFSETS : 0)), join = NW * (32 * OP + 64) * 4;
    return ring > join ? ring : join;
  }
};

constexpr int MAX_BY_LENGTH = 256;   // sequences
// The sum of x over this lane and those before it.
SA_DEV int wave_prefix_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // from one lane below, in rows of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);   // two
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);   // four
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);   // eight
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // the last lane of rows 0 and 2 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // lane 31 to rows 2 and 3
  return x;
}

// One part of the keys of 32 rows (r0 and following) of (b, hk).
template <typename T, int D, int NW, bool PAGED>
SA_DEV void rows_part(const RowsParams& p, char* smem_raw, int b, int hk, int split, int r0) {
  using G = Geom<T, D>;
  using S = RowsShape<T, D, NW>;
  using Frag = typename Elem<T>::Frag;
  constexpr int ST = S::ST, NF = G::NF, DB = G::DB, RPI = G::RPI, NI = 32 / RPI, NT = NW * 64;
  constexpr int IN_FLIGHT = (ST - 1) * 2 * NI < 63 ? (ST - 1) * 2 * NI : 63;
  static_assert(ST == 2, "the waits of the last tiles are written for two");

  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nbh = p.B * p.map.Hkv, bh = b * p.map.Hkv + hk, rows = p.map.rows();
  const int L = wave_length(p.lens, p.lens_stride, b, p.max_len);
  const int tokens = wave_length(p.q_lens, p.q_lens_stride, b, p.map.T), live = tokens * p.map.G;
  T* const out = reinterpret_cast<T*>(p.o);
  const int used = live - r0 < 32 ? live - r0 : 32;   // rows of this workgroup that are not padding
  if (p.splits == 1) {   // (with several splits the joining kernel writes the padding)
    const int first = used > 0 ? r0 + used : r0, last = r0 + 32 < rows ? r0 + 32 : rows;
    zero_rows<T, D, NT>(out, p.map, bh, first, last, tid);
    if (p.lse)
      for (int r = first + tid; r < last; r += NT) p.lse[p.map.flat(bh, r)] = 0.0f;
  }
  if (used <= 0) return;

  // windows: of this lane's row (padding has that of the last row), of all rows, of any row
  const int row = r0 + (c < used ? c : used - 1);
  int lo = 0, hi = L, lo_min = 0, lo_max = 0, hi_min = L, hi_max = L, first, last;
  if constexpr (PAGED) {
    window_of(p.win, p.map, L, tokens, row, lo, hi);
    window_of(p.win, p.map, L, tokens, r0, lo_min, hi_min);
    window_of(p.win, p.map, L, tokens, r0 + used - 1, lo_max, hi_max);
  }
  first = lo_min / 32, last = (hi_max + 31) / 32;
  if (p.splits > 1) {
    const int n = last > first ? last - first : 0, parts = parts_of(n, p.share);
    if (split >= parts) return;
    last = first + (int)((int64_t)n * (split + 1) / parts);
    first += (int)((int64_t)n * split / parts);
  }
  const int64_t part_row = ((int64_t)split * nbh + bh) * rows + r0;

  char* const own = smem_raw + wave * (S::RING + (PAGED ? S::ENTRIES + S::OFFSETS : 0));
  T* const ring = reinterpret_cast<T*>(own);
  int32_t* const entries = reinterpret_cast<int32_t*>(own + S::RING);                   // [2 * ST][64]
  int64_t* const offsets = reinterpret_cast<int64_t*>(own + S::RING + S::ENTRIES);      // [K | V][32]
  const T* const kbase = reinterpret_cast<const T*>(p.k) + (PAGED ? 0 : b * p.k_sp) + hk * p.k_sh;
  const T* const vbase = reinterpret_cast<const T*>(p.v) + (PAGED ? 0 : b * p.v_sp) + hk * p.v_sh;
  const int count = last - first - wave > 0 ? (last - first - wave + NW - 1) / NW : 0;   // of this wave's tiles
  auto tile_key = [&](int i) { return (first + wave + i * NW) * 32; };
  auto valid_key = [&](int k) { return k < L ? k : L - 1; };   // (a wave with a tile has L > 0)
  auto table_key = [&](int k) { return k < p.max_len ? k : p.max_len - 1; };
  auto fetch_entries = [&](int i) {   // of this wave's i-th tile
    if constexpr (PAGED) {
      const int k = table_key(tile_key(i) + c);
      copy_gather_word_asm(p.table + b * p.table_sb + div_by(k, p.by_page), lds_address(entries + i % (2 * ST) * 64));
    }
  };
  auto present = [&](int32_t page) { return (uint32_t)page < (uint32_t)p.num_pages; };
  auto issue = [&](int i) {
    T* const dst = ring + (i % ST) * 2 * S::TILE;
    const int k0 = tile_key(i);
    if constexpr (PAGED) {   // lanes of the lower half form the rows' places in K, the others in V
      const int k = table_key(k0 + c), in_page = k - div_by(k, p.by_page) * p.page;
      const int32_t e = entries[i % (2 * ST) * 64 + c];
      const int64_t page = present(e) ? e : 0;   // a page that is not there: any that is, its values are replaced below
      offsets[lane] = h == 0 ? page * p.k_sp + in_page * p.k_st : page * p.v_sp + in_page * p.v_st;
      sa::wave_exchange();
    }
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int r = j * RPI + lane / G::CPR, chunk = ((lane % G::CPR) ^ G::swz(r)) * G::VEC;
      int64_t ko, vo;
      if constexpr (PAGED) ko = offsets[r], vo = offsets[32 + r];
      else ko = valid_key(k0 + r) * p.k_st, vo = valid_key(k0 + r) * p.v_st;
      copy_gather_asm(kbase + ko + chunk, lds_address(dst + j * RPI * D));
      copy_gather_asm(vbase + vo + chunk, lds_address(dst + S::TILE + j * RPI * D));
    }
    if constexpr (PAGED) sa::wave_exchange();
  };

  const float sl2e = fmaxf(fabsf(p.scale_log2e), 1e-30f);
  Frag qf[NF];
  load_row<T, D>(qf, reinterpret_cast<const T*>(p.q) + b * p.q_sb + (int64_t)hk * p.map.G * p.q_sh + p.map.at(row, p.q_sh, p.q_st), true, lane);
  if constexpr (PAGED) {
#pragma unroll
    for (int i = 0; i < 2 * ST; ++i)
      if (i < count) fetch_entries(i);
    arrived_but<0>();
  }
#pragma unroll
  for (int i = 0; i < ST; ++i)
    if (i < count) issue(i);
  if (p.scale_log2e < 0.0f)
#pragma unroll
    for (int g = 0; g < NF; ++g) qf[g] = sa::negate<T>(qf[g]);

  RowState<DB> st;
  st.init();
  for (int i = 0; i < count; ++i) {
    if (i + 1 < count) arrived_but<IN_FLIGHT>();
    else arrived_but<0>();
    T* const keys = ring + (i % ST) * 2 * S::TILE;
    T* const values = keys + S::TILE;
    const int k0 = tile_key(i);
    bool here = k0 + c >= lo_min && k0 + c < hi_max;   // seen by some row
    if constexpr (PAGED) here = here && present(entries[i % (2 * ST) * 64 + c]);
    const uint32_t seen = (uint32_t)__builtin_amdgcn_ballot_w64(here);
    f32x16 s[1];
    clear(s);
    mul_rows<T, D>(s, keys, 0, qf, lane);
    if (seen != 0xFFFFFFFFu || k0 < lo_max || k0 + 32 > hi_min) {
      const uint32_t mask = sa::row_mask(lo - k0, hi - k0, h) & (seen >> (4 * h));
#pragma unroll
      for (int e = 0; e < 16; ++e) s[0][e] = sa::keep_or_neg_inf(s[0][e], sa::keep_bits(mask, e));
      // what stands in V where no row sees a key may be anything: 0 * NaN is not 0
#pragma unroll
      for (int j = 0; j < NI; ++j)
        if (!(seen >> (j * RPI + lane / G::CPR) & 1))
          *reinterpret_cast<u32x4*>(values + j * RPI * D + lane * G::VEC) = u32x4{0, 0, 0, 0};
      sa::wave_exchange();
    }
    softmax_step<T, D>(st, s, sl2e, values, lane);
    sa::reads_done();
    if (i + 2 * ST < count) fetch_entries(i + 2 * ST);
    if (i + ST < count) issue(i + ST);
  }

  // the waves' results, joined: O in [wave][row][OP], {m, l} behind
  const float l = sa::half_sum(st.l);
  __syncthreads();
  float* const wave_o = reinterpret_cast<float*>(smem_raw);
  float* const wave_ml = wave_o + NW * 32 * S::OP;
  if (c < used) {
    sa::store_acc_T<float, D, DB>(wave_o + (wave * 32 + c) * S::OP, st.o, 1.0f, h);
    if (h == 0) wave_ml[(wave * 32 + c) * 2] = st.m, wave_ml[(wave * 32 + c) * 2 + 1] = l;
  }
  __syncthreads();
  constexpr int Q4 = D / 4;
  for (int i = tid; i < used * Q4; i += NT) {
    const int r = i / Q4, d = i % Q4 * 4;
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, wave_ml[(w * 32 + r) * 2]);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = wave_ml[(w * 32 + r) * 2], lw = wave_ml[(w * 32 + r) * 2 + 1];
      const f32x4 ow = *reinterpret_cast<const f32x4*>(wave_o + (w * 32 + r) * S::OP + d);
      // a wave without a reference point has seen nothing, or only values that are not numbers
      const float f = mw == -INFINITY ? (lw == 0.0f ? 0.0f : 1.0f) : sa::fast_exp2(mw - m);
      sum += f * lw;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += f * ow[e];
    }
    if (p.splits > 1) {
      *reinterpret_cast<f32x4*>(p.part_o + (part_row + r) * D + d) = o;
      if (d == 0) p.part_ml[(part_row + r) * 2] = m, p.part_ml[(part_row + r) * 2 + 1] = sum;
    } else {
      const int64_t to = p.map.flat(bh, r0 + r);
      const bool some = !(sum == 0.0f);
      const float inv = some ? 1.0f / sum : 0.0f;
      sa::store4<T>(out + to * D + d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
      if (p.lse && d == 0) p.lse[to] = some ? m + __builtin_amdgcn_logf(sum) : -INFINITY;
    }
  }
}

// A workgroup for each part that there may be.
template <typename T, int D, int NW, bool PAGED>
__global__ __launch_bounds__(NW * 64) void rows_kernel(const RowsParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  // the splits and row tiles of a pair lie a multiple of the pairs apart: on one XCD where eight divides the pairs
  const int x = div_by(blockIdx.x, p.by_pairs), split = div_by(x, p.by_row_tiles);
  const int bh = blockIdx.x - x * (p.B * p.map.Hkv), b = div_by(bh, p.by_heads);
  rows_part<T, D, NW, PAGED>(p, smem_raw, b, bh - b * p.map.Hkv, split, (x - split * p.row_tiles) * 32);
}
// By length: as many workgroups as there are places; each takes the parts that lie the grid apart, of those that the lengths leave, whatever
// sequence they are of.  Lane l holds, of the sequences l, l + 64, ..., how many parts there are up to and with each.
template <typename T, int D, int NW, bool PAGED>
__global__ __launch_bounds__(NW * 64) void rows_by_length_kernel(const RowsParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  constexpr int GROUPS = MAX_BY_LENGTH / 64;
  const int lane = threadIdx.x & 63;
  int upto[GROUPS], total = 0;
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    const int b = j * 64 + lane, tokens = b < p.B ? clamped_length(p.q_lens, p.q_lens_stride, b, p.map.T) : 0;
    int first = 0, last = 0;
    if (tokens > 0)
      tiles_seen(p.win, p.map, clamped_length(p.lens, p.lens_stride, b, p.max_len), tokens, 0, tokens * p.map.G, 32, first, last);
    upto[j] = total + wave_prefix_sum(parts_of(last - first, p.share));
    total = __builtin_amdgcn_readlane(upto[j], 63);
  }
  for (int id = blockIdx.x; id < total * p.map.Hkv; id += gridDim.x) {
    const int part = div_by(id, p.by_heads);
    int b = 0, split = part;   // b: the sequences that end before the part
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      const int done = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto[j] <= part));
      b += done;
      if (done > 0) split = part - __builtin_amdgcn_readlane(upto[j], done - 1);
    }
    rows_part<T, D, NW, PAGED>(p, smem_raw, b, id - part * p.map.Hkv, split, 0);
    __syncthreads();   // the next part's rings lie over the waves' results
  }
}

// ---- joining --------------------------------------------------------------------------------------------------------
struct JoinParams {
  const float *part_o, *part_ml;   // [splits, B * Hkv, rows, D], [splits, B * Hkv, rows, 2]
  void* o;
  float* lse;
  const int32_t *lens, *q_lens;
  int64_t lens_stride, q_lens_stride;
  RowMap map;
  Windows win;
  int B, max_len;
  int splits, share, tile;         // as the parts were made: runs of tiles of `tile` keys
  ChunkDiv by_rows, by_heads;
};

// One row to SLOTS * D / 4 threads: slot j adds up the splits j, j + SLOTS, ..., the slots are added up in order.
template <typename T, int D, int SLOTS>
__global__ __launch_bounds__((SLOTS * D / 4 > 256 ? SLOTS * D / 4 : 256)) void join_kernel(const JoinParams p) {
  constexpr int Q4 = D / 4, PER_ROW = SLOTS * Q4, NT = PER_ROW > 256 ? PER_ROW : 256, RPB = NT / PER_ROW;
  __shared__ __attribute__((aligned(16))) float slot_o[SLOTS > 1 ? NT * 4 : 4];
  __shared__ float slot_ml[SLOTS > 1 ? RPB * SLOTS * 2 : 2];
  const int tid = threadIdx.x, in_block = tid / PER_ROW, slot = tid % PER_ROW / Q4, d = tid % Q4 * 4;
  const int rows = p.map.rows();
  const int64_t all = (int64_t)p.B * p.map.Hkv * rows, id = (int64_t)blockIdx.x * RPB + in_block;
  const bool inside = id < all;
  int bh = 0, row = 0, live = 0, parts = 0;
  if (inside) {
    bh = div_by((int)id, p.by_rows), row = (int)id - bh * rows;
    const int b = div_by(bh, p.by_heads), L = clamped_length(p.lens, p.lens_stride, b, p.max_len);
    const int tokens = clamped_length(p.q_lens, p.q_lens_stride, b, p.map.T), r0 = row & ~31;
    live = tokens * p.map.G;
    if (row < live) {
      int first, last;
      tiles_seen(p.win, p.map, L, tokens, r0, live - r0 < 32 ? live - r0 : 32, p.tile, first, last);
      parts = parts_of(last - first, p.share);
    }
  }
  float m = -INFINITY, l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (row < live) {
    // a few parts at a time, whose loads are on their way together; rows that have seen nothing in a part have a sum of 0
    constexpr int U = 4;
    const float* ml = p.part_ml + id * 2;
    for (int s0 = slot; s0 < parts; s0 += SLOTS * U) {
      float ms[U], ls[U], top = m;
      f32x4 os[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool there = s0 + u * SLOTS < parts;
        const int64_t s = there ? s0 + u * SLOTS : s0;   // (no branch around the loads)
        ms[u] = ml[s * all * 2];
        ls[u] = there ? ml[s * all * 2 + 1] : 0.0f;
        os[u] = *reinterpret_cast<const f32x4*>(p.part_o + (s * all + id) * D + d);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) top = ls[u] == 0.0f ? top : fmaxf(top, ms[u]);
      const float alpha = m == top ? 1.0f : sa::fast_exp2(m - top);
      m = top;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (ls[u] == 0.0f) continue;
        const float f = ms[u] == -INFINITY ? 1.0f : sa::fast_exp2(ms[u] - m);   // (-inf: values that are not numbers)
        l += f * ls[u];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += f * os[u][e];
      }
    }
  }
  if constexpr (SLOTS > 1) {
    *reinterpret_cast<f32x4*>(slot_o + tid * 4) = o;
    if (d == 0) slot_ml[(in_block * SLOTS + slot) * 2] = m, slot_ml[(in_block * SLOTS + slot) * 2 + 1] = l;
    __syncthreads();
    if (slot != 0) return;
#pragma unroll
    for (int j = 1; j < SLOTS; ++j) m = fmaxf(m, slot_ml[(in_block * SLOTS + j) * 2]);
    l = 0.0f, o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      const float mj = slot_ml[(in_block * SLOTS + j) * 2], lj = slot_ml[(in_block * SLOTS + j) * 2 + 1];
      const float f = mj == -INFINITY ? (lj == 0.0f ? 0.0f : 1.0f) : sa::fast_exp2(mj - m);
      const f32x4 oj = *reinterpret_cast<const f32x4*>(slot_o + (tid + j * Q4) * 4);
      l += f * lj;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += f * oj[e];
    }
  }
  if (!inside) return;
  const int64_t to = p.map.flat(bh, row);
  const bool some = row < live && !(l == 0.0f);
  const float inv = some ? 1.0f / l : 0.0f;
  if (!some) o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  sa::store4<T>(reinterpret_cast<T*>(p.o) + to * D + d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (p.lse && d == 0) p.lse[to] = row >= live ? 0.0f : some ? m + __builtin_amdgcn_logf(l) : -INFINITY;
}

// Gradients whose sums were split: parts [splits, B * Hkv, n, D] added up in order, rows from their limit on zero.
struct SumSide {
  const float* part;
  int64_t step, second;   // floats between the parts of consecutive splits, and from dK's to dV's
  void* out[2];           // dQ; or dK and dV
  RowMap map;             // of the rows of `out`
  int share, tile;        // as the parts were made (Work): runs of tiles of `tile` keys (dQ) or rows (dK, dV)
  ChunkDiv by_rows;
};
struct SumParams {
  SumSide queries, keys;
  int first_keys;         // layers of the grid: dQ below this one, dK and dV from it on
  const int32_t *lens, *q_lens;
  int64_t lens_stride, q_lens_stride;
  int B, Hkv, Tk, Tq;
  int group;              // query heads of a key head
  ChunkDiv by_heads;
};
template <typename T, int D> __global__ __launch_bounds__(256) void sum_kernel(const SumParams p) {
  constexpr int Q4 = D / 4, RPB = 256 / Q4;
  const bool keys = (int)blockIdx.y >= p.first_keys, second = (int)blockIdx.y > p.first_keys;
  const SumSide side = keys ? p.keys : p.queries;
  const int d = threadIdx.x % Q4 * 4, rows = side.map.rows();
  const int64_t id = (int64_t)blockIdx.x * RPB + threadIdx.x / Q4;
  if (id >= (int64_t)p.B * p.Hkv * rows) return;
  const int bh = div_by((int)id, side.by_rows), row = (int)id - bh * rows, b = div_by(bh, p.by_heads);
  const int rows_live = clamped_length(p.q_lens, p.q_lens_stride, b, p.Tq) * p.group, L = clamped_length(p.lens, p.lens_stride, b, p.Tk);
  const int limit = keys ? L : rows_live, run = keys ? rows_live : L;
  const int parts = parts_of((run + side.tile - 1) / side.tile, side.share);
  const float* const part = side.part + (second ? side.second : 0);
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if (row < limit)
#pragma unroll 4
    for (int s = 0; s < parts; ++s) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(part + s * side.step + id * D + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += x[e];
    }
  sa::store4<T>(reinterpret_cast<T*>(second ? side.out[1] : side.out[0]) + side.map.flat(bh, row) * D + d, sum[0], sum[1], sum[2], sum[3]);
}

}  // namespace kv
