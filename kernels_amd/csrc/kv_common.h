// Shared device code of attention over keys that are not the queries' own: cross attention (kv_fwd.h, kv_bwd.h) and
// attention of a few rows over a long run of keys, contiguous or in pages (kv_rows.h).
//
// Fragments, accumulators and products are those of sa_common.h.  Rows of a problem: the G query heads that share
// a key head are rows of one matrix product.  Row r of (batch entry b, key head hk) is token t = r / G of query head
// hk * G + r % G, so that the rows of the first n tokens are the first n * G rows, however many tokens a batch entry has, and 32
// consecutive rows are tokens that lie together.
#pragma once
#include "sa_common.h"

namespace kv {

using sa::ChunkDiv;
using sa::Elem;
using sa::TileMap;
using sa::chunk_div;
using sa::div_by;
using sa::f32x16;
using sa::f32x4;
using sa::u32x4;

// LDS tile of 32-row blocks without padding.  16-bit elements as in sa_common.h.  float32: 16-byte chunks are exchanged
// so that sixteen rows read at one chunk lie in different banks, and so do two rows four apart (the transposed product).
template <typename T, int D> struct Geom {
  static constexpr int VEC = Elem<T>::VEC;
  static constexpr int CPR = D / VEC;             // 16-byte chunks per row
  static constexpr int NF = D / (2 * VEC);        // row fragments per lane
  static constexpr int DB = D < 32 ? 1 : D / 32;  // 32-wide blocks along D
  static constexpr int RPI = 64 / CPR;            // rows that one copy instruction moves
  SA_DEV static int swz(int row) {
    if constexpr (Elem<T>::HALF) return sa::TileGeom<T, D>::swz(row);
    else if constexpr (CPR >= 16) return (row & 3) | ((row >> 3) & 1) << 2 | ((row >> 2) & 1) << 3;
    else if constexpr (CPR == 8) return ((row >> 1) & 3) | ((row >> 3) & 1) << 2;
    else return (row >> 2) & 3;
  }
  SA_DEV static int off(int row, int col) { return row * D + (((col / VEC) ^ swz(row)) * VEC | (col % VEC)); }
};

// acc[n][row][c] += sum_k tile[row0 + 32 * n + row][k] * b[k][c]
template <typename T, int D, int NB, int NF>
SA_DEV void mul_rows(f32x16 (&acc)[NB], const T* tile, int row0, const typename Elem<T>::Frag (&b)[NF], int lane) {
  using G = Geom<T, D>;
  static_assert(NF == G::NF, "one fragment per slice of the head dimension");
  if constexpr (Elem<T>::HALF) {
    sa::mma_rows_n<T, D>(reinterpret_cast<f32x16(&)[1][NB]>(acc), tile, row0,
                         reinterpret_cast<const typename Elem<T>::Frag(&)[1][NF]>(b), lane);
  } else {
    const int c = lane & 31, h = lane >> 5, sw = G::swz(c);
    const T* base = tile + (row0 + c) * D;
    constexpr int N = NB * NF;
    sa::pipeline<N, (N < 4 ? N : 4)>(
        [&](int it) { return *reinterpret_cast<const f32x4*>(base + it / NF * 32 * D + (((it % NF * 2 + h) ^ sw) * 4)); },
        [&](int it, const f32x4& a) { sa::mma(acc[it / NF], a, b[it % NF]); });
  }
}

// acc[m][x][c] += sum_r tile[row0 + r][m * 32 + x] * P[r][c] over the 32 rows from row0 on: float32 (16-bit elements: sa::mma_tr_n).
template <typename T, int D, int DB> SA_DEV void mul_tr(f32x16 (&acc)[DB], const T* tile, int row0, const f32x16& P, int lane) {
  using G = Geom<T, D>;
  static_assert(!Elem<T>::HALF && DB == G::DB, "float32, one accumulator per 32 columns");
  const int h = lane >> 5, c = D < 32 ? lane & 15 : lane & 31;   // D = 16: the product's rows from 16 on repeat the first
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = row0 + sa::crow(i, h);
#pragma unroll
    for (int m = 0; m < DB; ++m)
      acc[m] = __builtin_amdgcn_mfma_f32_32x32x2f32(tile[G::off(row, m * 32 + c)], P[i], acc[m], 0, 0, 0);
  }
}

SA_DEV void clear(f32x16& x) {
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.0f;
}
template <int N> SA_DEV void clear(f32x16 (&x)[N]) {
#pragma unroll
  for (int m = 0; m < N; ++m) clear(x[m]);
}

// ---- copies into LDS ----------------------------------------------------------------------------------------------
// One instruction moves 1 KiB, lane l's sixteen bytes to the l-th place.  A lane fetches the chunk that the layout wants there.

// 1 KiB of rows at addresses of the lanes' own, as assembly: the compiler waits for every copy that it knows of before it
// reads LDS, which would leave a wave with one tile in flight (see AsyncTile in sa_common.h).
SA_DEV void copy_gather_asm(const void* src, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(src) : "memory", "m0");
}
SA_DEV void copy_gather_word_asm(const void* src, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds_addr), "v"(src) : "memory", "m0");
}
// The low half of a generic address in LDS is the address there (a cast of the pointer would compare it with null first).
SA_DEV uint32_t lds_address(const void* p) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)p); }
// Until at most N of this wave's copies are on their way; no LDS access is moved ahead of it.
template <int N> SA_DEV void arrived_but() {
  static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// Rows [first, first + ROWS) of a [*, D] matrix with one row stride, by NW waves.  Rows past the last valid one come as zeros (the
// buffer's range check).  Offsets inside the matrix are 32-bit: the host checks that (rows + 1024) * stride fits.
template <typename T, int D, int ROWS, int NW> struct RowCopy {
  using G = Geom<T, D>;
  static constexpr int RPI = G::RPI, NI = ROWS / RPI, PER_WAVE = NI / NW;
  static_assert(ROWS % (RPI * NW) == 0, "the tile must split evenly over the waves");
  static constexpr int NVO = (RPI * NW) % 16 == 0 ? 1 : 16 / (RPI * NW);   // the exchange of chunks repeats every 16 rows
  __amdgpu_buffer_rsrc_t rsrc;
  uint32_t voff[NVO], istep, tstep;

  SA_DEV void init(const T* base, int64_t row_stride, int last_row, int wave, int lane) {
    constexpr uint32_t ES = (uint32_t)sizeof(T);
    const uint32_t rs = (uint32_t)row_stride;
    const int lrow = lane / G::CPR, ch = lane % G::CPR;
    const uint32_t bytes = ((uint32_t)last_row * rs + (uint32_t)D) * ES;
    rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, (int)bytes, 0x00020000);
#pragma unroll
    for (int j = 0; j < NVO; ++j)
      voff[j] = ((uint32_t)(wave * RPI + lrow) * rs + (uint32_t)((ch ^ G::swz((j * NW + wave) * RPI + lrow)) * G::VEC)) * ES;
    istep = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(NW * RPI) * rs * ES));
    tstep = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)ROWS * rs * ES));
  }
  SA_DEV void issue(T* tile, int t, int wave) const {   // rows [t * ROWS, (t + 1) * ROWS)
#pragma unroll
    for (int i = 0; i < PER_WAVE; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (SA_LDS void*)(tile + (i * NW + wave) * RPI * D), 16, (int)voff[i % NVO],
                                               (int)((uint32_t)t * tstep + (uint32_t)i * istep), 0, 0);
  }
};

// The tiles of two matrices that a step reads together, one behind the other in a stage.
template <typename T, int D, int ROWS, int NW> struct PairCopy {
  static constexpr bool SHARED = ROWS / Geom<T, D>::RPI % NW != 0;   // D = 16, 16-bit: half of the waves to a matrix
  static constexpr int EACH = SHARED ? NW / 2 : NW;
  using Copy = RowCopy<T, D, ROWS, EACH>;
  Copy a, b;   // SHARED: a is this wave's
  SA_DEV void init(const T* base_a, int64_t stride_a, const T* base_b, int64_t stride_b, int last_row, int wave, int lane) {
    const bool second = SHARED && wave >= EACH;
    a.init(second ? base_b : base_a, second ? stride_b : stride_a, last_row, wave % EACH, lane);
    if constexpr (!SHARED) b.init(base_b, stride_b, last_row, wave, lane);
  }
  SA_DEV void issue(T* stage, int t, int wave) const {
    a.issue(stage + (SHARED && wave >= EACH ? ROWS * D : 0), t, wave % EACH);
    if constexpr (!SHARED) b.issue(stage + ROWS * D, t, wave);
  }
};

// ---- rows ---------------------------------------------------------------------------------------------------------
// The rows of one (batch entry, key head): see the top of the file.
struct RowMap {
  int Hkv, G, T;        // T tokens
  ChunkDiv by_group;    // division by G
  SA_BOTH int rows() const { return G * T; }
  SA_BOTH void split(int r, int& t, int& g) const {
    t = div_by(r, by_group);
    g = r - t * G;
  }
  // element offset of row r in a tensor with these strides, from its (b, hk * G)
  SA_BOTH int64_t at(int r, int64_t sh, int64_t st) const {
    int t, g;
    split(r, t, g);
    return t * st + g * sh;
  }
  // row r of (b, hk) in a contiguous [B, Hkv * G, T] tensor
  SA_BOTH int64_t flat(int bh, int r) const {
    int t, g;
    split(r, t, g);
    return ((int64_t)bh * G + g) * T + t;
  }
};
SA_DEV int clamped_length(const int32_t* lens, int64_t stride, int b, int most) {
  if (!lens) return most;
  const int n = lens[(int64_t)b * stride];
  return n < 0 ? 0 : (n > most ? most : n);
}

// Tiles of ROWS consecutive rows at addresses of their own (several heads to a key head), by NW waves; the last valid row again in place
// of those past it.  As assembly, for rings of more than two stages.
template <typename T, int D, int ROWS, int NW> struct RowGather {
  using G = Geom<T, D>;
  static constexpr int PER_WAVE = ROWS / G::RPI / NW;
  static_assert(ROWS % (G::RPI * NW) == 0, "the tile must split evenly over the waves");
  SA_DEV static void issue(const T* base, int64_t sh, int64_t st, const RowMap& map, int row0, int live, T* tile, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < PER_WAVE; ++i) {
      const int first = (i * NW + wave) * G::RPI, in_tile = first + lane / G::CPR;
      const int r = row0 + in_tile < live ? row0 + in_tile : live - 1;
      copy_gather_asm(base + (map.at(r, sh, st) + ((lane % G::CPR) ^ G::swz(in_tile)) * G::VEC), lds_address(tile + first * D));
    }
  }
};
// Of a batch entry that the whole wave works on: in a scalar register, and so is what follows from it (loop counts, tile offsets).
SA_DEV int wave_length(const int32_t* lens, int64_t stride, int b, int most) {
  return __builtin_amdgcn_readfirstlane(clamped_length(lens, stride, b, most));
}

// Fragments of row `row` (a pointer to its first element), or zeros.
template <typename T, int D, int NF>
SA_DEV void load_row(typename Elem<T>::Frag (&f)[NF], const T* row, bool valid, int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int g = 0; g < NF; ++g) {
    f[g] = *reinterpret_cast<const typename Elem<T>::Frag*>(row + (g * 2 + h) * Elem<T>::VEC);
    if (!valid) f[g] = typename Elem<T>::Frag{};
  }
}

// The 32 rows from row0 on of an accumulator X^T[d][row], times mul, to a contiguous [B, Hkv * G, T, D] tensor; 16-bit elements go
// through a patch of LDS of the wave's own, so that memory sees whole rows.
template <typename T, int D, int DB>
SA_DEV void store_rows(T* out, const RowMap& map, int bh, int row0, T* patch, const f32x16 (&acc)[DB], float mul, int lane) {
  const int rows = map.rows();
  if constexpr (Elem<T>::HALF) {
    using P = sa::RowPatch<T, D>;
    const int c = lane & 31, h = lane >> 5;
    sa::wave_exchange();
#pragma unroll
    for (int m = 0; m < DB; ++m)
#pragma unroll
      for (int g = 0; g < (D < 32 ? D / 8 : 4); ++g)
        sa::store4<T>(patch + c * P::PITCH + m * 32 + 8 * g + 4 * h, acc[m][4 * g] * mul, acc[m][4 * g + 1] * mul,
                      acc[m][4 * g + 2] * mul, acc[m][4 * g + 3] * mul);
    sa::wave_exchange();
    const int rr = lane / P::CPR, ch = lane % P::CPR;
#pragma unroll
    for (int j = 0; j < 32 / P::RPI; ++j) {
      const int r = j * P::RPI + rr;
      const u32x4 x = *reinterpret_cast<const u32x4*>(patch + r * P::PITCH + ch * 8);
      if (row0 + r < rows) sa::store_streaming(out + map.flat(bh, row0 + r) * D + ch * 8, x);
    }
  } else {
    const int r = row0 + (lane & 31);
    if (r < rows) sa::store_acc_T<T, D, DB>(out + map.flat(bh, r) * D, acc, mul, lane >> 5);
  }
}
// Rows [row0, row1) become zeros.
template <typename T, int D, int NT> SA_DEV void zero_rows(T* out, const RowMap& map, int bh, int row0, int row1, int tid) {
  constexpr int CPR = Geom<T, D>::CPR;
  for (int ch = tid; ch < (row1 - row0) * CPR; ch += NT)
    sa::store_streaming(out + map.flat(bh, row0 + ch / CPR) * D + ch % CPR * Elem<T>::VEC, u32x4{0, 0, 0, 0});
}

// ---- split work -----------------------------------------------------------------------------------------------------
// Where the keys (or, for dK and dV, the rows) are divided over several workgroups, each leaves float32 sums and, in the forward, the
// reference point and the sum of its probabilities; a second kernel adds them up in the order of the splits.  A run of n tiles is divided
// into as many even parts as shares of `share` tiles would be, so that a long sequence takes more workgroups than a short one.
SA_BOTH int parts_of(int n, int share) { return (n + share - 1) / share; }

// A workgroup's (batch entry, key head), tile and split.  Pairs are dealt over the XCDs as in sa::tile_coords, with the tiles of a pair
// side by side; or, tiles_first, tile by tile over all pairs, the first tiles, which are never cut short by a length, at the beginning.
struct Work {
  TileMap map;           // tiles include the splits
  int splits;            // the most that a run of tiles is divided into
  int share, tiles_first;
  ChunkDiv by_splits, by_pairs;   // by_pairs: the pairs of an XCD, or all
};
SA_BOTH void work_of(const Work& w, int bid, int n_blocks, int& bh, int& tile, int& split) {
  if (w.tiles_first) {
    const bool dealt = (w.map.nbh & 7) == 0;
    const int idx = dealt ? bid >> 3 : bid, pairs = dealt ? w.map.nbh >> 3 : w.map.nbh;
    tile = div_by(idx, w.by_pairs);
    bh = idx - tile * pairs;
    if (dealt) bh = bh * 8 + (bid & 7);
  } else {
    sa::tile_coords(bid, n_blocks, w.map, bh, tile);
  }
  split = 0;
  if (w.splits > 1) {
    const int t = div_by(tile, w.by_splits);
    split = tile - t * w.splits, tile = t;
  }
}

// The part [first, last) of n tiles that split has to do; nothing for the splits that the run is too short for.
SA_BOTH void part_of(const Work& w, int n, int split, int& first, int& last) {
  first = 0, last = n;
  if (w.splits > 1) {
    const int parts = parts_of(n, w.share);
    first = split < parts ? (int)((int64_t)n * split / parts) : 0;
    last = split < parts ? (int)((int64_t)n * (split + 1) / parts) : 0;
  }
}

struct FwdParams {
  const void *q, *k, *v;
  void* o;             // contiguous [B, Hq, Tq, D]
  float* lse;          // contiguous [B, Hq, Tq] or null
  const int32_t *lens, *q_lens;
  int64_t lens_stride, q_lens_stride;
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  RowMap map;
  int B, Tk;
  float scale_log2e;
  Work work;
  float* part_o;       // [splits, B * Hkv, rows, D]
  float* part_ml;      // [splits, B * Hkv, rows, 2]
};

struct BwdParams {
  const void *q, *k, *v, *o, *d_o;
  const float* lse;    // contiguous [B, Hq, Tq]
  void *dq, *dk, *dv;  // contiguous
  const int32_t *lens, *q_lens;
  int64_t lens_stride, q_lens_stride;
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st, g_sb, g_sh, g_st;
  RowMap map;
  int B, Tk;
  float scale, scale_log2e;
  Work work;
  float *row_lse, *row_delta;   // [B * Hkv, rows]: written with dQ, read with dK and dV; 16-bit elements: lse / score_scale
  bool head_major;     // those in the order (head, token) instead of that of the rows
  float* part;         // dQ: [splits, B * Hkv, rows, D]; dK and dV: [splits, 2, B * Hkv, Tk, D]
};

}  // namespace kv
