// Trees of drafted tokens over a cache in pages, from 33 rows of a key head on (up to 32: kv_rows.h).
//
// The tile kernel of kv_fwd.h with keys in pages: NW waves of 32 rows share tiles of TK keys, which go through LDS once for all of them, in two
// stages.  Each lane forms the place of one key of the next tile from its page, and hands it to the lanes that copy that row.  Every row sees the
// keys before the drafted tokens, so masks are formed only where a tile reaches those, or where pages are missing; there the waves also tell
// each other which keys some row sees, and values that none does become zeros.
#pragma once
#include "kv_rows.h"

namespace kv {

template <typename T, int D, int NW> struct TreeShape {
  static constexpr int TK = fwd_tile<T, D>(), TQ = NW * 32, STAGE = 2 * TK * D;   // elements of a stage: [K | V][TK][D]
  static constexpr int OFFSETS = 2 * TK * 8;                                      // bytes per wave: [K | V][TK]
  static constexpr int bytes() {
    const int stages = 2 * STAGE * (int)sizeof(T), patches = sizeof(T) == 2 ? NW * 32 * (D + 8) * 2 : 0;   // (patches lie over the stages)
    return (stages > patches ? stages : patches) + NW * OFFSETS + NW * 8;
  }
};

// The part `split` of the keys, for rows r0 and following of (b, hk).
template <typename T, int D, int NW> SA_DEV void tree_part(const RowsParams& p, char* smem_raw, int b, int hk, int split, int r0) {
  using G = Geom<T, D>;
  using S = TreeShape<T, D, NW>;
  using Frag = typename Elem<T>::Frag;
  constexpr int TK = S::TK, NB = TK / 32, NF = G::NF, DB = G::DB, RPI = G::RPI, NI = TK / RPI, NT = NW * 64;
  constexpr uint64_t ALL = TK == 64 ? ~0ull : 0xFFFFFFFFull;
  T* const smem = reinterpret_cast<T*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* const behind = smem_raw + S::bytes() - NW * (S::OFFSETS + 8);
  int64_t* const offsets = reinterpret_cast<int64_t*>(behind + wave * S::OFFSETS);
  uint32_t* const waves_see = reinterpret_cast<uint32_t*>(behind + NW * S::OFFSETS);   // [NW][2]

  const int nbh = p.B * p.map.Hkv, bh = b * p.map.Hkv + hk, rows = p.map.rows();
  const int L = wave_length(p.lens, p.lens_stride, b, p.max_len);
  const int tokens = wave_length(p.q_lens, p.q_lens_stride, b, p.map.T), live = tokens * p.map.G, base = L - tokens;
  const int wr0 = r0 + wave * 32, row = wr0 + c;
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
    t0 = (int)((int64_t)n * split / parts);
    t1 = (int)((int64_t)n * (split + 1) / parts);
  }
  const float sl2e = fmaxf(fabsf(p.scale_log2e), 1e-30f);   // never exactly 0, so that a masked score of -inf stays -inf after scaling
  const T* const kbase = reinterpret_cast<const T*>(p.k) + hk * p.k_sh;
  const T* const vbase = reinterpret_cast<const T*>(p.v) + hk * p.v_sh;
  auto key_of = [&](int t) {   // the key whose place this lane forms
    const int k = t * TK + (TK == 64 ? lane : c);
    return k < p.max_len ? k : p.max_len - 1;
  };
  auto entry = [&](int t) { return p.table[b * p.table_sb + div_by(key_of(t), p.by_page)]; };
  auto present = [&](int32_t page) { return (uint32_t)page < (uint32_t)p.num_pages; };
  auto issue = [&](int t, int32_t e) {
    T* const stage = smem + ((t - t0) & 1) * S::STAGE;
    const int k = key_of(t), in_page = k - div_by(k, p.by_page) * p.page;
    const int64_t page = present(e) ? e : 0;   // a page that is not there: any that is, its values are replaced
    if (TK == 64 || h == 0) offsets[TK == 64 ? lane : c] = page * p.k_sp + in_page * p.k_st;
    if (TK == 64 || h == 1) offsets[TK + (TK == 64 ? lane : c)] = page * p.v_sp + in_page * p.v_st;
    sa::wave_exchange();
#pragma unroll
    for (int x = 0; x < (2 * NI + NW - 1) / NW; ++x) {
      const int i = x * NW + wave;
      if (2 * NI % NW != 0 && i >= 2 * NI) break;
      const int r = i % NI * RPI + lane / G::CPR, chunk = ((lane % G::CPR) ^ G::swz(r)) * G::VEC;
      copy_gather_asm((i < NI ? kbase : vbase) + offsets[i / NI * TK + r] + chunk, lds_address(stage + i * RPI * D));
    }
    sa::wave_exchange();
  };

  RowState<DB> st;
  st.init();
  if (t0 < t1) {
    int32_t e0 = entry(t0), e1 = t0 + 1 < t1 ? entry(t0 + 1) : 0;
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
    issue(t0, e0);
    for (int t = t0; t < t1; ++t) {
      arrived_but<0>();
      __syncthreads();   // every wave's share of tile t has arrived; the other stage, that of the tile before, is free
      const uint64_t there = __builtin_amdgcn_ballot_w64(present(e0)) & ALL;
      if (t + 1 < t1) issue(t + 1, e1);
      e0 = e1;
      if (t + 2 < t1) e1 = entry(t + 2);
      T* const keys = smem + ((t - t0) & 1) * S::STAGE;
      T* const values = keys + TK * D;
      const int k0 = t * TK;
      const bool masked = k0 + TK > base || there != ALL;   // of the whole workgroup
      if (wr0 >= live && !masked) continue;
      f32x16 s[NB];
      if (wr0 < live) {
        clear(s);
        mul_rows<T, D>(s, keys, 0, qf, lane);
      }
      if (masked) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          uint32_t mask = 0;
          if (wr0 < live) {
            mask = tree_mask(p.tree, b, token, tokens, base, k0 + n * 32, h) & ((uint32_t)(there >> (n * 32)) >> (4 * h));
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = sa::keep_or_neg_inf(s[n][i], sa::keep_bits(mask, i));
          }
          const uint32_t sees = any_row(mask);
          if (lane == 0) waves_see[wave * 2 + n] = sees;
        }
        __syncthreads();
        uint32_t seen[2] = {0, 0};
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int n = 0; n < NB; ++n) seen[n] |= waves_see[w * 2 + n];
        // what stands in V where no row sees a key may be anything: 0 * NaN is not 0
        for (int ch = tid; ch < TK * G::CPR; ch += NT) {
          const int r = ch / G::CPR;
          if (!(seen[r >> 5] >> (r & 31) & 1)) *reinterpret_cast<u32x4*>(values + ch * G::VEC) = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
      }
      if (wr0 < live) softmax_step<T, D>(st, s, sl2e, values, lane);
    }
  }
  const float l = sa::half_sum(st.l);
  if (p.splits > 1) {
    if (row < live) {
      const int64_t part_row = ((int64_t)split * nbh + bh) * rows + row;
      sa::store_acc_T<float, D, DB>(p.part_o + part_row * D, st.o, 1.0f, h);
      if (h == 0) p.part_ml[part_row * 2] = st.m, p.part_ml[part_row * 2 + 1] = l;
    }
    return;
  }
  const bool valid = row < live, some = !(l == 0.0f);   // a row that sees no key (or none with a score above -inf) is zero
  if (!valid || !some) clear(st.o);
  __syncthreads();   // the patches lie over the tile stages
  store_rows<T, D, DB>(out, p.map, bh, wr0, smem + wave * sa::RowPatch<T, D>::ELEMS, st.o, valid && some ? 1.0f / l : 0.0f, lane);
  if (p.lse && h == 0 && row < rows)
    p.lse[p.map.flat(bh, row)] = !valid ? 0.0f : some ? st.m + __builtin_amdgcn_logf(l) : -INFINITY;
}

// A workgroup for each part that there may be.
template <typename T, int D, int NW> __global__ __launch_bounds__(NW * 64) void tree_kernel(const RowsParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  const int x = div_by(blockIdx.x, p.by_pairs), split = div_by(x, p.by_row_tiles);
  const int bh = blockIdx.x - x * (p.B * p.map.Hkv), b = div_by(bh, p.by_heads);
  tree_part<T, D, NW>(p, smem_raw, b, bh - b * p.map.Hkv, split, (x - split * p.row_tiles) * NW * 32);
}

}  // namespace kv
