// Trees of drafted tokens over a cache in pages, for more than 32 rows of a key head (few rows, and little work: kv_rows.h).
//
//   O = softmax(scale * Q K^T) V over the keys before the drafted tokens and those of the drafted ones that the tree names
//
// The tile kernel of kv_fwd.h with keys in pages: waves of 32 rows share tiles of TK keys, which go through LDS once for all of them, in two stages, so
// that K and V are read from memory once for 64 or 128 rows.  WR waves have rows of their own; up to 64 rows WK = 2 waves share each block of rows, one
// half of a tile's keys each, and add up their sums at the end: a tile's chain of products and exponentials, of which a wave can hide little, is half as
// long.  Each lane forms the place of one key of the next tile from its page.  WHOLE (pages of a multiple of sixteen positions): places are handed on in scalar
// registers, one for sixteen rows; other pages through LDS, one for each row.  Every row sees the keys before the drafted tokens, so masks are
// formed only where a tile reaches those, or where pages are missing; there the waves also tell each other which keys some row sees, and values
// that none does become zeros.
//
// Bound by memory up to 64 rows, by vector and matrix instructions, which hardly overlap, above: 64 rows, D = 128, bfloat16, 256 key heads of 8192 (1.07 GB)
// 217 us, 5.0 TB/s, log-uniform up to 8192 52-91 us for 32-58 us at a copy's rate (6.05 TB/s); 256 rows, 64 of 8192 92 us, 0.75 PFLOP/s, matrix units busy 43 %, vector units 43 %
// of the time.  64 rows in us: two waves of rows alone 64 (log-uniform) and 187 (from 4096 on), with places in scalar registers 59 and 179, two waves to each block
// of rows 52 and 172.
#pragma once
#include "kv_rows.h"

namespace kv {

// 1 KiB of rows that lie in one page, whose place is in scalar registers; lanes add their 32-bit offsets.  The five wait states of sa::copy_rows_asm.
SA_DEV void copy_group_asm(const void* base, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds_addr), "v"(voff), "s"(base) : "memory", "m0");
}

template <typename T, int D, int WR, int WK, bool WHOLE> struct TreeShape {
  static constexpr int NW = WR * WK, TK = fwd_tile<T, D>(), TQ = WR * 32, STAGE = 2 * TK * D;   // elements of a stage: [K | V][TK][D]
  static constexpr int OFFSETS = WHOLE ? 0 : 2 * TK * 8;                          // bytes per wave: [K | V][TK]
  static constexpr int RPI = Geom<T, D>::RPI, COPIES = (2 * TK / RPI + NW - 1) / NW;   // per wave and tile
  static constexpr int GROUP = RPI > 16 ? RPI : 16;                                    // WHOLE: rows that lie in one page
  static constexpr int STEP = COPIES < GROUP / RPI ? COPIES : GROUP / RPI;             // copies of a group
  static constexpr int OP = D + 4;                                                     // floats per row of a wave's sums
  static constexpr int bytes() {
    const int stages = 2 * STAGE * (int)sizeof(T), patches = sizeof(T) == 2 ? WR * 32 * (D + 8) * 2 : 0;   // patches and sums lie over the stages
    const int sums = WK > 1 ? WR * 32 * (OP + 2) * 4 : 0, over = patches > sums ? patches : sums;
    return (stages > over ? stages : over) + NW * OFFSETS + NW * 8;
  }
};

// The part `split` of the keys, for rows r0 and following of (b, hk).  WHOLE: sixteen rows (and those of a copy) lie in one page.
template <typename T, int D, int WR, int WK, bool WHOLE> SA_DEV void tree_part(const TreeParams& p, char* smem_raw, int b, int hk, int split, int r0) {
  using G = Geom<T, D>;
  using S = TreeShape<T, D, WR, WK, WHOLE>;
  using Frag = typename Elem<T>::Frag;
  constexpr int NW = S::NW, TK = S::TK, NB = TK / 32 / WK, NF = G::NF, DB = G::DB, RPI = G::RPI, NI = TK / RPI, NT = NW * 64;
  constexpr uint64_t ALL = TK == 64 ? ~0ull : 0xFFFFFFFFull;
  T* const smem = reinterpret_cast<T*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* const behind = smem_raw + S::bytes() - NW * (S::OFFSETS + 8);
  int64_t* const offsets = reinterpret_cast<int64_t*>(behind + wave * S::OFFSETS);
  uint32_t* const waves_see = reinterpret_cast<uint32_t*>(behind + NW * S::OFFSETS);   // [NW][NB]

  const int nbh = p.B * p.map.Hkv, bh = b * p.map.Hkv + hk, rows = p.map.rows();
  const int L = wave_length(p.lens, p.lens_stride, b, p.max_len);
  const int tokens = wave_length(p.q_lens, p.q_lens_stride, b, p.map.T), live = tokens * p.map.G, base = L - tokens;
  const int wr = wave % WR, wk = wave / WR, wr0 = r0 + wr * 32, row = wr0 + c;   // this wave's rows and blocks of keys
  T* const out = reinterpret_cast<T*>(p.o);
  if (r0 >= live) {   // padding: zeros (with several splits the joining kernel writes them)
    if (p.splits > 1) return;
    const int r1 = r0 + S::TQ < rows ? r0 + S::TQ : rows;
    zero_rows<T, D, NT>(out, p.map, bh, r0, r1, tid);
    if (p.lse)
      for (int r = r0 + tid; r < r1; r += NT) p.lse[p.map.flat(bh, r)] = 0.0f;
    return;
  }
  int t0 = 0, t1 = (L + TK - 1) / TK;
  if (p.splits > 1) {
    const int n = t1, parts = parts_of(n, p.share);
    if (split >= parts) return;   // (the joining kernel knows how many parts there are)
    // the last part's masks take as long as two tiles: 240 rows, 15 key heads of 6000 33.8 -> 32.3 us, 64 rows, 96 of 2000 26.0 -> 23.8, others 0-6 % less
    t0 = part_start(n + 2, parts, split), t1 = part_start(n + 2, parts, split + 1);
    t1 = t1 < n ? t1 : n;
  }
  const float sl2e = fmaxf(fabsf(p.scale_log2e), 1e-30f);   // never exactly 0, so that a masked score of -inf stays -inf after scaling
  const T* const kbase = reinterpret_cast<const T*>(p.k) + hk * p.k_sh;
  const T* const vbase = reinterpret_cast<const T*>(p.v) + hk * p.v_sh;
  auto present = [&](int32_t page) { return (uint32_t)page < (uint32_t)p.num_pages; };
  // The place of one key of a tile: its page's entry, and where it stands in the page.  Keys past the table: the last ones of it.
  struct Place {
    int32_t entry;
    uint32_t in_page;
  };
  auto place = [&](int t) {
    const int in_tile = TK == 64 ? lane : c, k = t * TK + in_tile;
    const int at = k < p.max_len ? k : WHOLE ? p.max_len - S::GROUP + in_tile % S::GROUP : p.max_len - 1;
    const int entry = div_by(at, p.by_page);
    return Place{p.table[b * p.table_sb + entry], (uint32_t)(at - entry * p.page)};
  };
  // WHOLE: a lane's row and chunk of a copy, beside the place of the copy's first row
  const uint32_t k_row = WHOLE ? (uint32_t)(lane / G::CPR) * (uint32_t)(p.k_st * (int64_t)sizeof(T)) : 0;
  const uint32_t v_row = WHOLE ? (uint32_t)(lane / G::CPR) * (uint32_t)(p.v_st * (int64_t)sizeof(T)) : 0;
  const bool alike = p.k_sp == p.v_sp && p.k_st == p.v_st;
  auto issue = [&](int t, const Place& at) {
    T* const stage = smem + ((t - t0) & 1) * S::STAGE;
    const int32_t page = present(at.entry) ? at.entry : 0;   // a page that is not there: any that is, its values are replaced
    if constexpr (WHOLE) {   // (byte strides below 2^32: the host's rule)
      auto offset = [&](int64_t sp, int64_t st) {
        return (uint64_t)(uint32_t)page * (uint32_t)(sp * (int64_t)sizeof(T)) + at.in_page * (uint32_t)(st * (int64_t)sizeof(T));
      };
      const uint64_t ko = offset(p.k_sp, p.k_st), vo = alike ? ko : offset(p.v_sp, p.v_st);
      // copy i of a tile: rows [i % NI * RPI, ...) of K, then of V; a wave's copies follow each other, those of GROUP rows in one page
#pragma unroll
      for (int x = 0; x < S::COPIES; x += S::STEP) {
        const int i = wave * S::COPIES + x;
        if (S::COPIES * NW > 2 * NI && i >= 2 * NI) break;
        const bool values = i >= NI;
        const int first = i % NI * RPI;
        const uint64_t from = values ? vo : ko;
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)from, first);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(from >> 32), first);
        const char* base = reinterpret_cast<const char*>(values ? vbase : kbase) + ((uint64_t)hi << 32 | lo);
        const uint32_t step = (uint32_t)(values ? p.v_st : p.k_st) * (uint32_t)(RPI * sizeof(T)), row = values ? v_row : k_row;
#pragma unroll
        for (int y = 0; y < S::STEP; ++y, base += step)
          copy_group_asm(base, row + (uint32_t)(((lane % G::CPR) ^ G::swz((i + y) % NI * RPI + lane / G::CPR)) * 16), lds_address(stage + (i + y) * RPI * D));
      }
    } else {
      const int in_tile = TK == 64 ? lane : c;
      if (TK == 64 || h == 0) offsets[in_tile] = page * p.k_sp + at.in_page * p.k_st;
      if (TK == 64 || h == 1) offsets[TK + in_tile] = page * p.v_sp + at.in_page * p.v_st;
      sa::wave_exchange();
#pragma unroll
      for (int x = 0; x < (2 * NI + NW - 1) / NW; ++x) {
        const int i = x * NW + wave;
        if (2 * NI % NW != 0 && i >= 2 * NI) break;
        const int r = i % NI * RPI + lane / G::CPR, chunk = ((lane % G::CPR) ^ G::swz(r)) * G::VEC;
        copy_gather_asm((i < NI ? kbase : vbase) + offsets[i / NI * TK + r] + chunk, lds_address(stage + i * RPI * D));
      }
      sa::wave_exchange();
    }
  };

  RowState<DB> st;
  st.init();
  if (t0 < t1) {
    Place at0 = place(t0), at1 = place(t0 + 1 < t1 ? t0 + 1 : t0);
    Frag qf[NF];
    int token = 0, ignored;
    {
      const int used = row < live ? row : live - 1;
      p.map.split(used, token, ignored);
      load_row<T, D>(qf, reinterpret_cast<const T*>(p.q) + b * p.q_sb + (int64_t)hk * p.map.G * p.q_sh + p.map.at(used, p.q_sh, p.q_st), true, lane);
      if (p.scale_log2e < 0.0f)
#pragma unroll
        for (int g = 0; g < NF; ++g) qf[g] = sa::negate<T>(qf[g]);
    }
    sa::wait_all_loads();   // the rows' fragments and the entries
    issue(t0, at0);
    for (int t = t0; t < t1; ++t) {
      arrived_but<0>();
      __syncthreads();   // every wave's share of tile t has arrived; the other stage, that of the tile before, is free
      const uint64_t there = __builtin_amdgcn_ballot_w64(present(at0.entry)) & ALL;
      if (t + 1 < t1) issue(t + 1, at1);
      at0 = at1;
      if (t + 2 < t1) at1 = place(t + 2);
      T* const keys = smem + ((t - t0) & 1) * S::STAGE;
      T* const values = keys + TK * D;
      const int k0 = t * TK + wk * NB * 32;
      const bool masked = (t + 1) * TK > base || there != ALL;   // of the whole workgroup
      if (wr0 >= live && !masked) continue;
      f32x16 s[NB];
      if (wr0 < live) {
        clear(s);
        mul_rows<T, D>(s, keys, wk * NB * 32, qf, lane);
      }
      if (masked) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          uint32_t mask = 0;
          if (wr0 < live) {
            mask = tree_mask(p.tree, p.map.T, b, token, tokens, base, k0 + n * 32, h) & ((uint32_t)(there >> ((wk * NB + n) * 32)) >> (4 * h));
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = sa::keep_or_neg_inf(s[n][i], sa::keep_bits(mask, i));
          }
          const uint32_t sees = any_row(mask);
          if (lane == 0) waves_see[wave * NB + n] = sees;
        }
        __syncthreads();
        uint32_t seen[TK / 32] = {};
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int n = 0; n < NB; ++n) seen[w / WR * NB + n] |= waves_see[w * NB + n];
        // what stands in V where no row sees a key may be anything: 0 * NaN is not 0
        for (int ch = tid; ch < TK * G::CPR; ch += NT) {
          const int r = ch / G::CPR;
          if (!(seen[TK == 64 ? r >> 5 : 0] >> (r & 31) & 1)) *reinterpret_cast<u32x4*>(values + ch * G::VEC) = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
      }
      if (wr0 < live) softmax_step<T, D>(st, s, sl2e, values + wk * NB * 32 * D, lane);
    }
  }
  float l = sa::half_sum(st.l);
  if constexpr (WK > 1) {   // the sums over the other blocks of keys, joined
    static_assert(WK == 2, "one wave adds another's");
    __syncthreads();
    float* const sums = reinterpret_cast<float*>(smem_raw) + (wr * 32 + c) * S::OP;
    float* const ml = reinterpret_cast<float*>(smem_raw) + WR * 32 * S::OP + (wr * 32 + c) * 2;
    if (wk == 1) {
      sa::store_acc_T<float, D, DB>(sums, st.o, 1.0f, h);
      if (h == 0) ml[0] = st.m, ml[1] = l;
    }
    __syncthreads();
    if (wk == 0) {
      const float m1 = ml[0], l1 = ml[1], m = fmaxf(st.m, m1);
      // without a reference point a wave has seen nothing, or only values that are not numbers
      const float f0 = st.m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : sa::fast_exp2(st.m - m);
      const float f1 = m1 == -INFINITY ? (l1 == 0.0f ? 0.0f : 1.0f) : sa::fast_exp2(m1 - m);
      st.m = m, l = f0 * l + f1 * l1;
#pragma unroll
      for (int n = 0; n < DB; ++n)
#pragma unroll
        for (int g = 0; g < (D < 32 ? D / 8 : 4); ++g) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(sums + n * 32 + 8 * g + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) st.o[n][4 * g + e] = f0 * st.o[n][4 * g + e] + f1 * x[e];
        }
    }
  }
  if (p.splits > 1) {
    if (row < live && wk == 0) {
      const int64_t part_row = ((int64_t)split * nbh + bh) * rows + row;
      sa::store_acc_T<float, D, DB>(p.part_o + part_row * D, st.o, 1.0f, h);
      if (h == 0) p.part_ml[part_row * 2] = st.m, p.part_ml[part_row * 2 + 1] = l;
    }
    return;
  }
  const bool valid = row < live, some = !(l == 0.0f);   // a row that sees no key (or none with a score above -inf) is zero
  if (!valid || !some) clear(st.o);
  __syncthreads();   // the patches lie over the tile stages
  if (wk > 0) return;
  store_rows<T, D, DB>(out, p.map, bh, wr0, smem + wr * sa::RowPatch<T, D>::ELEMS, st.o, valid && some ? 1.0f / l : 0.0f, lane);
  if (p.lse && h == 0 && row < rows)
    p.lse[p.map.flat(bh, row)] = !valid ? 0.0f : some ? st.m + __builtin_amdgcn_logf(l) : -INFINITY;
}

// A workgroup for each part that there may be.
template <typename T, int D, int WR, int WK, bool WHOLE> __global__ __launch_bounds__(WR * WK * 64) void tree_kernel(const TreeParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  const int x = div_by(blockIdx.x, p.by_pairs), split = div_by(x, p.by_row_tiles);
  const int bh = blockIdx.x - x * (p.B * p.map.Hkv), in_order = div_by(bh, p.by_heads);
  // the second parts of the sequences in reverse order: the places of a CU go to parts of different sequences (log-uniform up to 8192 69-101 -> 62-92 us)
  const int b = split & 1 ? p.B - 1 - in_order : in_order;
  tree_part<T, D, WR, WK, WHOLE>(p, smem_raw, b, bh - in_order * p.map.Hkv, split, (x - split * p.row_tiles) * WR * 32);
}

}  // namespace kv
