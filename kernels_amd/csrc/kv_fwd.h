// Cross attention, forward: O = softmax(scale * Q K^T) V over the first lens[b] keys, and the base-2 log-sum-exp.
//
// One workgroup owns TQ = 32 * NW rows (kv_common.h) of one (batch entry, key head), each wave 32 of them and each lane one row: scores
// are formed transposed, so the running reference point and sum of a row are a lane's own and the probabilities are the second
// product's operand as they stand.  K and V go through LDS in tiles of TK keys, two stages, sent for one tile ahead.  All rows see
// the same keys: only the last tile needs a mask.
#pragma once
#include "kv_common.h"

namespace kv {

constexpr float kRescaleGap = 8.0f;    // the reference point moves when a score exceeds it by 2^8
constexpr float kSumLimit = 256.0f;    // sums up to this hold no probability above 2^8

// The running state of a lane's row: O^T = sum of p v, with p = exp2(score - m), l the sum of this lane's half of the p.
template <int DB> struct RowState {
  f32x16 o[DB];
  float m, l;
  SA_DEV void init() {
    clear(o);
    m = -INFINITY, l = 0.0f;
  }
};

// The maximum of a lane's scores, over both halves of its row.
template <int NB> SA_DEV float row_max(const f32x16 (&s)[NB]) {
  float mx = -INFINITY, mk[NB];   // one chain per block, so that consecutive instructions are independent
#pragma unroll
  for (int n = 0; n < NB; ++n) mk[n] = -INFINITY;
#pragma unroll
  for (int i = 0; i < 16; i += 2)
#pragma unroll
    for (int n = 0; n < NB; ++n) mk[n] = sa::fast_max3(mk[n], s[n][i], s[n][i + 1]);
#pragma unroll
  for (int n = 0; n < NB; ++n) mx = sa::fast_max(mx, mk[n]);
  return sa::half_max(mx);
}
// Moves the reference point to a maximum that exceeds it by more than kRescaleGap.
template <int DB> SA_DEV void move_reference(RowState<DB>& st, float mx) {
  const bool move = mx > st.m + kRescaleGap;   // false for -inf and NaN
  if (__builtin_amdgcn_ballot_w64(move) != 0) {
    const float alpha = move ? sa::fast_exp2(st.m - mx) : 1.0f;   // (0 where there was none)
    st.m = move ? mx : st.m;
    st.l *= alpha;
#pragma unroll
    for (int m = 0; m < DB; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[m][i] *= alpha;
  }
}

// One step on NB blocks of 32 keys: s holds their raw scores, masked ones -inf.  The maximum is looked for only where the probabilities
// relative to the present reference point show that it has been left behind; the result does not depend on which point it is, as
// long as the probabilities stay below 2^8 or so.  Where registers are short (the guessed probabilities stand beside the scores; head
// dimension 256), and in float32, whose matrix instructions leave the time, it is looked for every time.
template <typename T, int D, int NB, int DB>
SA_DEV void softmax_step(RowState<DB>& st, f32x16 (&s)[NB], float sl2e, const T* values, int lane) {
  using Frag = typename Elem<T>::Frag;
  constexpr bool GUESS = Elem<T>::HALF && DB < 8;
  Frag pb[NB][1][2];
  float sum[2];
  auto probabilities = [&](f32x16 (&p)[NB]) {
    const float m_use = st.m == -INFINITY ? 0.0f : st.m;
    sum[0] = sum[1] = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) p[n][i] = sa::fast_exp2(__builtin_fmaf(s[n][i], sl2e, -m_use));
      if constexpr (Elem<T>::HALF) sa::pack_c<T>(pb[n][0], p[n]);
#pragma unroll
      for (int i = 0; i < 16; i += 2) sum[0] += p[n][i], sum[1] += p[n][i + 1];
    }
  };
  if constexpr (GUESS) {
    f32x16 p[NB];
    bool search = __builtin_amdgcn_ballot_w64(st.m != -INFINITY) == 0;   // no lane has a reference point yet
    if (!search) {
      probabilities(p);
      const bool behind = !(sum[0] + sum[1] <= kSumLimit) || st.m == -INFINITY;   // true for NaN too
      search = __builtin_amdgcn_ballot_w64(behind) != 0;
    }
    if (search) {
      move_reference(st, row_max(s) * sl2e);
      probabilities(p);
    }
  } else {
    move_reference(st, row_max(s) * sl2e);
    probabilities(s);
  }
  st.l += sum[0] + sum[1];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if constexpr (Elem<T>::HALF) sa::mma_tr_n<T, D>(reinterpret_cast<f32x16(&)[1][DB]>(st.o), values, n, pb[n], lane);
    else mul_tr<T, D>(st.o, values, n * 32, s[n], lane);
  }
}

template <typename T, int D> constexpr int fwd_tile() { return D * (int)sizeof(T) <= 256 ? 64 : 32; }

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, (D * sizeof(T) == 512 ? (sizeof(T) == 2 ? 2 : 1) : 1)) void cross_fwd_kernel(const FwdParams p) {
  using G = Geom<T, D>;
  using Frag = typename Elem<T>::Frag;
  constexpr int TK = fwd_tile<T, D>(), TQ = NW * 32, NT = NW * 64, NB = TK / 32, NF = G::NF, DB = G::DB, STAGE = 2 * TK * D;
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  T* smem = reinterpret_cast<T*>(smem_raw);   // [stage][K | V][TK][D]

  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int bh, tile, split;
  work_of(p.work, blockIdx.x, gridDim.x, bh, tile, split);
  const int b = div_by(bh, p.work.map.by_heads), hk = bh - b * p.map.Hkv;
  const int L = wave_length(p.lens, p.lens_stride, b, p.Tk);
  const int rows = p.map.rows(), live = wave_length(p.q_lens, p.q_lens_stride, b, p.map.T) * p.map.G;
  const int r0 = tile * TQ, wr0 = r0 + wave * 32, row = wr0 + c;
  T* const out = reinterpret_cast<T*>(p.o);
  const int64_t part_row = (int64_t)split * p.B * p.map.Hkv * rows + (int64_t)bh * rows + row;
  if (r0 >= live) {   // padding: zeros (with several splits the joining kernel writes them)
    if (p.work.splits > 1) return;
    const int r1 = r0 + TQ < rows ? r0 + TQ : rows;
    zero_rows<T, D, NT>(out, p.map, bh, r0, r1, tid);
    if (p.lse)
      for (int r = r0 + tid; r < r1; r += NT) p.lse[p.map.flat(bh, r)] = 0.0f;
    return;
  }

  int t0, t1;
  part_of(p.work, (L + TK - 1) / TK, split, t0, t1);
  if (p.work.splits > 1 && t0 >= t1) return;   // (the joining kernel knows how many parts there are)
  // never exactly 0, so that a masked score of -inf stays -inf after scaling
  const float sl2e = fmaxf(fabsf(p.scale_log2e), 1e-30f);
  Frag qf[NF];
  {
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_sb + (int64_t)hk * p.map.G * p.q_sh;
    load_row<T, D>(qf, q + p.map.at(row < live ? row : live - 1, p.q_sh, p.q_st), true, lane);
    if (p.scale_log2e < 0.0f)
#pragma unroll
      for (int g = 0; g < NF; ++g) qf[g] = sa::negate<T>(qf[g]);
  }
  RowState<DB> st;
  st.init();
  if (t0 < t1) {
    PairCopy<T, D, TK, NW> tiles;
    tiles.init(reinterpret_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh, p.k_st,
               reinterpret_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh, p.v_st, L - 1, wave, lane);
    sa::wait_all_loads();   // the row's fragments
    tiles.issue(smem, t0, wave);
    for (int t = t0; t < t1; ++t) {
      sa::wait_loads<0>();
      __syncthreads();   // every wave's share of tile t has arrived; the other stage, that of the tile before, is free
      if (t + 1 < t1) tiles.issue(smem + ((t + 1 - t0) & 1) * STAGE, t + 1, wave);
      if (wr0 >= live) continue;
      const T* keys = smem + ((t - t0) & 1) * STAGE;
      f32x16 s[NB];
      clear(s);
      mul_rows<T, D>(s, keys, 0, qf, lane);
      if ((t + 1) * TK > L)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const uint32_t mask = sa::row_mask(0, L - t * TK - n * 32, h);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[n][i] = sa::keep_or_neg_inf(s[n][i], sa::keep_bits(mask, i));
        }
      softmax_step<T, D>(st, s, sl2e, keys + TK * D, lane);
    }
  }
  const float l = sa::half_sum(st.l);
  if (p.work.splits > 1) {
    if (row < live) {
      sa::store_acc_T<float, D, DB>(p.part_o + part_row * D, st.o, 1.0f, h);
      if (h == 0) p.part_ml[part_row * 2] = st.m, p.part_ml[part_row * 2 + 1] = l;
    }
    return;
  }
  // a row that sees no key (or none with a score above -inf) is zero
  const bool valid = row < live, some = !(l == 0.0f);
  if (!valid || !some) clear(st.o);
  __syncthreads();   // the patches lie over the tile stages
  store_rows<T, D, DB>(out, p.map, bh, wr0, smem + wave * sa::RowPatch<T, D>::ELEMS, st.o, valid && some ? 1.0f / l : 0.0f, lane);
  if (p.lse && h == 0 && row < rows)
    p.lse[p.map.flat(bh, row)] = !valid ? 0.0f : some ? st.m + __builtin_amdgcn_logf(l) : -INFINITY;
}

}  // namespace kv
