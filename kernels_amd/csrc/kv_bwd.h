// Cross attention, backward.  With P = exp2(scale * log2e * Q K^T - LSE), dP = dO V^T, delta = rowsum(O * dO), dS = P * (dP - delta):
//   cross_dq_kernel     dQ = scale * dS K               a lane owns a row, the keys go by
//   cross_dkdv_kernel   dV = P^T dO, dK = scale * dS^T Q  a lane owns a key, the rows of all query heads that share it go by, so
//                                                       that the sum over the heads is part of the product
// The first one forms delta (over few keys as rowsum(P * dP), in which O is not rounded: sa::few_keys_delta) and leaves it, beside the
// log-sum-exp, in the order of the rows for the second.  No atomics: a
// sum over workgroups (few rows and many keys, or the reverse) goes through float32 parts that are added up in order.
#pragma once
#include "sa_bwd.h"
#include "sa_bwd_split.h"
#include "kv_fwd.h"

namespace kv {

// dQ^T += K^T dS^T, negated, for the tile of TK keys whose first is k0: float32 (16-bit elements: sa::dq2_tile).  g holds -dO.
template <typename T, int D, int TK, int NF, int DB>
SA_DEV void dq_tile_f32(f32x16 (&acc)[DB], const T* keys, const T* values, int k0, int L, const typename Elem<T>::Frag (&q)[NF],
                        const typename Elem<T>::Frag (&g)[NF], float sl2e, float lse, float delta, int lane) {
#pragma unroll
  for (int n = 0; n < TK / 32; ++n) {
    if (k0 + n * 32 >= L) continue;
    f32x16 s[1], dp[1];
    clear(s);
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[0][i] = delta;
    mul_rows<T, D>(s, keys, n * 32, q, lane);
    mul_rows<T, D>(dp, values, n * 32, g, lane);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[0][i] = sa::fast_exp2(__builtin_fmaf(s[0][i], sl2e, -lse)) * dp[0][i];
    if (k0 + n * 32 + 32 > L) {
      const uint32_t mask = sa::row_mask(0, L - k0 - n * 32, lane >> 5);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][i] = sa::keep_or_zero(s[0][i], sa::keep_bits(mask, i));
    }
    mul_tr<T, D>(acc, keys, n * 32, s[0], lane);
  }
}

template <typename T> SA_DEV float dot(typename Elem<T>::Frag a, typename Elem<T>::Frag b, float acc) {
  if constexpr (Elem<T>::HALF) return sa::dot_frag(a, b, acc);
  else {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_fmaf(a[e], b[e], acc);
    return acc;
  }
}

template <typename T, int D> constexpr int dq_tile() { return Elem<T>::HALF ? 64 : fwd_tile<T, D>(); }

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) void cross_dq_kernel(const BwdParams p) {
  using G = Geom<T, D>;
  using Frag = typename Elem<T>::Frag;
  constexpr int TK = dq_tile<T, D>(), TQ = NW * 32, NT = NW * 64, NF = G::NF, DB = G::DB, STAGE = 2 * TK * D;
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
  T* const out = reinterpret_cast<T*>(p.dq);
  if (r0 >= live) {
    if (p.work.splits == 1) zero_rows<T, D, NT>(out, p.map, bh, r0, r0 + TQ < rows ? r0 + TQ : rows, tid);
    return;
  }
  int t0, t1;
  part_of(p.work, (L + TK - 1) / TK, split, t0, t1);
  if (t0 >= t1 && split > 0) return;   // (the first one leaves delta)
  PairCopy<T, D, TK, NW> tiles;
  tiles.init(reinterpret_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh, p.k_st,
             reinterpret_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh, p.v_st, L - 1, wave, lane);
  if (t0 < t1) tiles.issue(smem, t0, wave);

  const float sl2e = fabsf(p.scale_log2e);
  Frag qf[NF], gf[NF];
  float lse, delta = 0.0f;
  {
    const int r = row < live ? row : live - 1;
    int t, g;
    p.map.split(r, t, g);
    const int64_t head = (int64_t)hk * p.map.G + g;
    load_row<T, D>(qf, reinterpret_cast<const T*>(p.q) + b * p.q_sb + head * p.q_sh + t * p.q_st, true, lane);
    load_row<T, D>(gf, reinterpret_cast<const T*>(p.d_o) + b * p.g_sb + head * p.g_sh + t * p.g_st, true, lane);
    lse = p.lse[p.map.flat(bh, r)];
    if (lse == -INFINITY || row >= live) lse = INFINITY;   // P = exp2(-inf) = 0: no key is seen, or padding
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      if (p.scale_log2e < 0.0f) qf[i] = sa::negate<T>(qf[i]);
      gf[i] = sa::negate<T>(gf[i]);   // the dP accumulator starts at delta and ends at delta - dP
    }
    if (Elem<T>::HALF && L <= sa::FEW_KEYS) {
      delta = sa::few_keys_delta<T>(reinterpret_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh, p.k_st,
                                    reinterpret_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh, p.v_st, L, qf, gf, sl2e, lse, lane);
    } else {
      const T* o = reinterpret_cast<const T*>(p.o) + b * p.o_sb + head * p.o_sh + t * p.o_st;
#pragma unroll
      for (int i = 0; i < NF; ++i)
        delta = dot<T>(gf[i], *reinterpret_cast<const Frag*>(o + (i * 2 + h) * Elem<T>::VEC), delta);
      delta = -sa::half_sum(delta);
    }
    if (split == 0 && h == 0 && row < live) {
      const int64_t at = p.head_major ? p.map.flat(bh, row) : (int64_t)bh * rows + row;
      p.row_lse[at] = Elem<T>::HALF ? lse / sa::score_scale(p.scale_log2e) : lse;
      p.row_delta[at] = delta;
    }
  }
  f32x16 acc[DB], dinit;
  clear(acc);
#pragma unroll
  for (int i = 0; i < 16; ++i) dinit[i] = delta;
  const sa::WaveWindow win{0, L, 0, L, 0, L};
  auto next_tile = [&](int t) {   // waits for tile t, sends for the next one
    sa::wait_loads<0>();
    __syncthreads();
    if (t + 1 < t1) tiles.issue(smem + ((t + 1 - t0) & 1) * STAGE, t + 1, wave);
    return smem + ((t - t0) & 1) * STAGE;
  };
  int t = t0;
  if constexpr (Elem<T>::HALF && D == 256)   // a loop of their own: where two paths meet the compiler copies 128 accumulators
    for (; t < t1 && wr0 < live && (t + 1) * TK <= L; ++t) {
      const T* keys = next_tile(t);
      sa::dq2_tile_inside<T, D>(acc, keys, keys + TK * D, qf, gf, sl2e, lse, dinit, lane);
    }
  for (; t < t1; ++t) {
    const T* keys = next_tile(t);
    if (wr0 >= live) continue;
    if constexpr (!Elem<T>::HALF)
      dq_tile_f32<T, D, TK>(acc, keys, keys + TK * D, t * TK, L, qf, gf, sl2e, lse, delta, lane);
    else
      sa::dq2_tile<T, D, TK>(acc, keys, keys + TK * D, t * TK, win, qf, gf, sl2e, lse, dinit, lane);
  }
  if (p.work.splits > 1) {
    if (row < live)
      sa::store_acc_T<float, D, DB>(p.part + ((int64_t)split * p.B * p.map.Hkv * rows + (int64_t)bh * rows + row) * D, acc, -p.scale, h);
    return;
  }
  if (row >= live) clear(acc);
  __syncthreads();   // the patches lie over the tile stages
  store_rows<T, D, DB>(out, p.map, bh, wr0, smem + wave * sa::RowPatch<T, D>::ELEMS, acc, -p.scale, lane);
}

// dV^T += dO^T P and dK^T += Q^T dS, negated, for the TQ rows from r0 on, or one of them: float32 (16-bit elements: below).
// v holds -V.
template <typename T, int D, int TQ, bool WITH_DK, bool WITH_DV, int NF, int NV, int DK, int DV>
SA_DEV void dkdv_tile_f32(f32x16 (&dk)[DK], f32x16 (&dv)[DV], const T* qt, const T* gt, int r0, int live,
                          const typename Elem<T>::Frag (&k)[NF], const typename Elem<T>::Frag (&v)[NV], float scale_log2e,
                          const float* stats, int lane) {   // stats: {lse, delta} of RPW rows after one another
  constexpr int RPW = TQ / 4;
  auto place = [](int r) { return r / RPW * 2 * RPW + r % RPW; };
  const int h = lane >> 5;
#pragma unroll
  for (int n = 0; n < TQ / 32; ++n) {
    if (r0 + n * 32 >= live) continue;
    f32x16 s[1], dp[1];
    clear(s);
    mul_rows<T, D>(s, qt, n * 32, k, lane);
    if constexpr (WITH_DK) {
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[0][i] = stats[place(n * 32 + sa::crow(i, h)) + RPW];
      mul_rows<T, D>(dp, gt, n * 32, v, lane);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[0][i] = sa::fast_exp2(__builtin_fmaf(s[0][i], scale_log2e, -stats[place(n * 32 + sa::crow(i, h))]));
      if constexpr (WITH_DK) dp[0][i] *= s[0][i];
    }
    if (r0 + n * 32 + 32 > live) {
      const uint32_t mask = sa::row_mask(0, live - r0 - n * 32, h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[0][i] = sa::keep_or_zero(s[0][i], sa::keep_bits(mask, i));
        if constexpr (WITH_DK) dp[0][i] = sa::keep_or_zero(dp[0][i], sa::keep_bits(mask, i));
      }
    }
    if constexpr (WITH_DV) mul_tr<T, D>(dv, gt, n * 32, s[0], lane);
    if constexpr (WITH_DK) mul_tr<T, D>(dk, qt, n * 32, dp[0], lane);
  }
}

// The same, both gradients, 16-bit elements.  k holds -K (K for a negative scale), unrounded; the score accumulator starts at
// lse / score_scale, so that one multiplication by mul = -score_scale gives the exponent.  (K scaled and rounded, as streaming attention has it, saves that
// and takes dK and dV further from the exact result: relative errors 0.0030 instead of 0.0024 in bfloat16, whose own rounding is 0.0017.)
// rows(r) gives the four lse and the four delta values of the tile's rows r to r + 3; v holds -V.
template <typename T, int D, int TQ, int PG, int NF, int DB, typename Rows>
SA_DEV void dkdv_tile_16(f32x16 (&dk)[DB], f32x16 (&dv)[DB], const T* qt, const T* gt, int r0, int live,
                         const typename Elem<T>::Frag (&k)[NF], const typename Elem<T>::Frag (&v)[NF], float mul, Rows&& rows,
                         int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int n = 0; n < TQ / 32; ++n) {
    if (r0 + n * 32 >= live) continue;
    f32x16 s, dp;
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      f32x4 l4, d4;
      rows(n * 32 + 8 * g4 + 4 * h, l4, d4);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * g4 + e] = l4[e], dp[4 * g4 + e] = d4[e];
    }
    sa::mma_rows_pair<T, D, NF, PG>(s, dp, qt, gt, n * 32, k, v, lane);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = sa::fast_exp2(s[i] * mul);
      dp[i] *= s[i];   // = -dS
    }
    if (r0 + n * 32 + 32 > live) {
      const uint32_t mask = sa::row_mask(0, live - r0 - n * 32, h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t keep = sa::keep_bits(mask, i);
        s[i] = sa::keep_or_zero(s[i], keep);
        dp[i] = sa::keep_or_zero(dp[i], keep);
      }
    }
    sa::mma_tr_pair<T, D, DB, PG>(dv, dk, gt, qt, n, s, dp, lane);
  }
}

template <typename T, int D> constexpr int dkdv_tile() { return D * (int)sizeof(T) <= 256 ? 64 : 32; }
// Bytes of a stage: Q and dO tiles, and lse and delta of their rows.
template <typename T, int D> constexpr int dkdv_stage() { return 2 * dkdv_tile<T, D>() * (D * (int)sizeof(T) + (int)sizeof(float)); }

// PASS: 0 both gradients, 1 dV, 2 dK.  float32 at head dimension 256 takes a launch for each: two accumulators of 32 x 256 and the rows
// of K and V are all 512 registers of a lane.
template <typename T, int D, int NW, int PASS>
__global__ __launch_bounds__(NW * 64, (sizeof(T) == 2 && D == 64 ? 3 : 1)) void cross_dkdv_kernel(const BwdParams p) {
  using G = Geom<T, D>;
  using Frag = typename Elem<T>::Frag;
  constexpr bool WITH_DV = PASS != 2, WITH_DK = PASS != 1;
  constexpr int TQ = dkdv_tile<T, D>(), TKB = NW * 32, NT = NW * 64, NF = G::NF, DB = G::DB, TILE = TQ * D;
  constexpr int RPW = TQ / NW, STAGE = dkdv_stage<T, D>();
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];   // [stage]{[Q | dO][TQ][D], [wave]{lse, delta}[RPW]}

  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int bh, tile, split;
  work_of(p.work, blockIdx.x, gridDim.x, bh, tile, split);
  const int b = div_by(bh, p.work.map.by_heads), hk = bh - b * p.map.Hkv;
  const int L = wave_length(p.lens, p.lens_stride, b, p.Tk);
  const int rows = p.map.rows(), live = wave_length(p.q_lens, p.q_lens_stride, b, p.map.T) * p.map.G;
  const int k0 = tile * TKB, wk0 = k0 + wave * 32, key = wk0 + c;
  const RowMap keys{1, 1, p.Tk, chunk_div(1)};   // K's gradients are rows of one head each
  T* const dk_out = reinterpret_cast<T*>(p.dk);
  T* const dv_out = reinterpret_cast<T*>(p.dv);
  if (k0 >= L || live == 0) {
    if (p.work.splits == 1) {
      const int k1 = k0 + TKB < p.Tk ? k0 + TKB : p.Tk;
      if constexpr (WITH_DK) zero_rows<T, D, NT>(dk_out, keys, bh, k0, k1, tid);
      if constexpr (WITH_DV) zero_rows<T, D, NT>(dv_out, keys, bh, k0, k1, tid);
    }
    return;
  }
  int t0, t1;
  part_of(p.work, (live + TQ - 1) / TQ, split, t0, t1);
  if (t0 >= t1) return;

  const T* const q = reinterpret_cast<const T*>(p.q) + b * p.q_sb + (int64_t)hk * p.map.G * p.q_sh;
  const T* const g = reinterpret_cast<const T*>(p.d_o) + b * p.g_sb + (int64_t)hk * p.map.G * p.g_sh;
  const float* const lse_rows = p.row_lse + (int64_t)bh * rows;
  const float* const delta_rows = p.row_delta + (int64_t)bh * rows;
  // one head: whole tiles at a constant stride, rows past the last one as zeros.  Several: rows at addresses of their own, the last
  // one again in place of those past it
  PairCopy<T, D, TQ, NW> whole;
  const bool one_head = p.map.G == 1;
  if (one_head) whole.init(q, p.q_st, g, p.g_st, live - 1, wave, lane);
  auto issue_tile = [&](int t) {
    char* const stage = smem_raw + ((t - t0) & 1) * STAGE;
    T* const dst = reinterpret_cast<T*>(stage);
    if (lane < 2 * RPW) {   // lanes [0, RPW) fetch lse, [RPW, 2 * RPW) delta
      int r = t * TQ + wave * RPW + lane % RPW;
      r = r < live ? r : live - 1;
      sa::async_copy_f32((lane < RPW ? lse_rows : delta_rows) + r, reinterpret_cast<float*>(stage + 2 * TILE * sizeof(T)) + wave * 2 * RPW);
    }
    if (one_head) {
      whole.issue(dst, t, wave);
    } else {
#pragma unroll
      for (int i = 0; i < (TQ / G::RPI + NW - 1) / NW; ++i) {
        const int first = (i * NW + wave) * G::RPI;
        if (first < TQ) {
          const int in_tile = first + lane / G::CPR;
          int r = t * TQ + in_tile, tok, head;
          r = r < live ? r : live - 1;
          p.map.split(r, tok, head);
          const int chunk = ((lane % G::CPR) ^ G::swz(in_tile)) * G::VEC;
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(q + (tok * p.q_st + head * p.q_sh + chunk)),
                                           (SA_LDS void*)(dst + first * D), 16, 0, 0);
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(g + (tok * p.g_st + head * p.g_sh + chunk)),
                                           (SA_LDS void*)(dst + TILE + first * D), 16, 0, 0);
        }
      }
    }
  };
  if (t0 < t1) issue_tile(t0);

  Frag kf[NF], vf[WITH_DK ? NF : 1];
  {
    const bool valid = key < L;
    const int k = valid ? key : L - 1;
    load_row<T, D>(kf, reinterpret_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh + k * p.k_st, valid, lane);
    if constexpr (WITH_DK) {
      load_row<T, D>(vf, reinterpret_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh + k * p.v_st, valid, lane);
#pragma unroll
      for (int i = 0; i < NF; ++i) vf[i] = sa::negate<T>(vf[i]);
    }
    if constexpr (Elem<T>::HALF)
#pragma unroll
      for (int i = 0; i < NF; ++i)
        if (p.scale_log2e >= 0.0f) kf[i] = sa::negate<T>(kf[i]);
  }
  f32x16 dk[WITH_DK ? DB : 1], dv[WITH_DV ? DB : 1];
  clear(dk);
  clear(dv);
  sa::wait_all_loads();
  for (int t = t0; t < t1; ++t) {
    sa::wait_loads<0>();
    __syncthreads();
    if (t + 1 < t1) issue_tile(t + 1);
    const char* const stage = smem_raw + ((t - t0) & 1) * STAGE;
    const T* const qt = reinterpret_cast<const T*>(stage);
    const float* const stats = reinterpret_cast<const float*>(stage + 2 * TILE * sizeof(T));
    if (wk0 >= L) continue;
    if constexpr (Elem<T>::HALF) {
      dkdv_tile_16<T, D, TQ, (D == 64 ? 2 : 4)>(dk, dv, qt, qt + TILE, t * TQ, live, kf, vf, -sa::score_scale(p.scale_log2e),
                                                 [&](int r, f32x4& l4, f32x4& d4) {
        const float* chunk = stats + (r / RPW) * 2 * RPW + r % RPW;
        l4 = *reinterpret_cast<const f32x4*>(chunk);
        d4 = *reinterpret_cast<const f32x4*>(chunk + RPW);
      }, lane);
    } else {
      dkdv_tile_f32<T, D, TQ, WITH_DK, WITH_DV>(dk, dv, qt, qt + TILE, t * TQ, live, kf, vf, p.scale_log2e, stats, lane);
    }
  }
  if (p.work.splits > 1) {
    const int64_t each = (int64_t)p.B * p.map.Hkv * p.Tk;
    if (key < L) {
      float* part = p.part + ((int64_t)split * 2 * each + (int64_t)bh * p.Tk + key) * D;
      if constexpr (WITH_DK) sa::store_acc_T<float, D, DB>(part, dk, -p.scale, h);
      if constexpr (WITH_DV) sa::store_acc_T<float, D, DB>(part + each * D, dv, 1.0f, h);
    }
    return;
  }
  if (key >= L) clear(dk), clear(dv);
  __syncthreads();   // the patches lie over the tile stages
  T* patch = reinterpret_cast<T*>(smem_raw) + wave * sa::RowPatch<T, D>::ELEMS;
  if constexpr (WITH_DK) store_rows<T, D, DB>(dk_out, keys, bh, wk0, patch, dk, -p.scale, lane);
  if constexpr (WITH_DV) store_rows<T, D, DB>(dv_out, keys, bh, wk0, patch, dv, 1.0f, lane);
}

// dK and dV at head dimension 256, 16-bit elements: the four products of 32 keys divided between two waves of one SIMD, as in
// sa::dkdv_split_wide_kernel.  The score role holds K and dV and forms S, P and dV; the grad role holds V and dK and
// forms dP, and a step later, with the P that the other has left in LDS in float32, dS and dK.  Steps of 32 rows; a Q tile is read in two
// steps, a dO tile in one: rings of four and of three, two tiles ahead of the compute.
template <typename T, int D>
__global__ __launch_bounds__(512) void cross_dkdv_wide_kernel(const BwdParams p) {
  using E = Elem<T>;
  using G = Geom<T, D>;
  using Frag = typename E::Frag;
  using S = sa::DkdvSplitWide<T, D>;
  static_assert(E::HALF && D == 256, "16-bit elements, head dimension 256");
  constexpr int NP = S::NP, NW = 2 * NP, TQ = S::TQ, TKB = S::TKB, NT = NW * 64;
  constexpr int NF = G::NF, DB = G::DB, TILE = TQ * D, NQ = S::NQ, NG = S::NG;
  constexpr int RPW = TQ / NW;   // rows of lse / delta each wave stages
  static_assert(RPW % 4 == 0 && NQ == 4 && NG == 3, "two tiles ahead: see issue_tile");
  using Loader = sa::AsyncTile<T, D, TQ, NW, true>;
  using Gather = RowGather<T, D, TQ, NW>;
  static_assert(Gather::PER_WAVE == Loader::PER_WAVE, "the same number of copies either way");
  constexpr int LPT = 2 * Loader::PER_WAVE + 1;   // copies of a wave per tile

  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  T* const q_ring = reinterpret_cast<T*>(smem_raw);
  T* const g_ring = q_ring + NQ * TILE;
  float* const row_ring = reinterpret_cast<float*>(g_ring + NG * TILE);   // [NQ][NW chunks of {lse[RPW], delta[RPW]}]

  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pair = wave & (NP - 1);   // waves w and w + 4 run on the same SIMD
  const bool grad_role = wave >= NP;
  float* const xbuf = row_ring + NQ * 2 * TQ + pair * 2 * S::XSLOT + lane * 4;   // two slots of 16 values per lane

  int bh, tile, split;
  work_of(p.work, blockIdx.x, gridDim.x, bh, tile, split);
  const int b = div_by(bh, p.work.map.by_heads), hk = bh - b * p.map.Hkv;
  const int L = wave_length(p.lens, p.lens_stride, b, p.Tk);
  const int rows = p.map.rows(), live = wave_length(p.q_lens, p.q_lens_stride, b, p.map.T) * p.map.G;
  const int k0 = tile * TKB, wk0 = k0 + pair * 32, key = wk0 + c;
  const RowMap keys{1, 1, p.Tk, chunk_div(1)};
  T* const out = reinterpret_cast<T*>(grad_role ? p.dk : p.dv);
  if (k0 >= L || live == 0) {
    if (p.work.splits == 1) {
      const int k1 = k0 + TKB < p.Tk ? k0 + TKB : p.Tk;
      zero_rows<T, D, NT / 2>(out, keys, bh, k0, k1, tid % (NT / 2));
    }
    return;
  }
  int t0, t1;
  part_of(p.work, (live + TQ - 1) / TQ, split, t0, t1);
  if (t0 >= t1) return;
  const int n = t1 - t0;
  const bool seen = wk0 < L;   // of the pair's keys

  const T* const q = reinterpret_cast<const T*>(p.q) + b * p.q_sb + (int64_t)hk * p.map.G * p.q_sh;
  const T* const g = reinterpret_cast<const T*>(p.d_o) + b * p.g_sb + (int64_t)hk * p.map.G * p.g_sh;
  const float* const row_src = (lane < RPW ? p.row_lse : p.row_delta) + (int64_t)bh * rows;
  const bool one_head = p.map.G == 1;
  Loader ldq, ldg;   // of one head
  ldq.init(q, p.q_st, t0 * TQ, live - 1, wave, lane);
  ldg.init(g, p.g_st, t0 * TQ, live - 1, wave, lane);
  // The tile of step `it` goes where those of steps it - 4 (Q, lse, delta) and it - 3 (dO) were: sent for at the beginning of
  // step it - 2, when every wave has finished step it - 3, the last that reads either.
  auto issue_tile = [&](int it, int gs) {
    const int qs = it & (NQ - 1), row0 = (t0 + it) * TQ;
    if (lane < 2 * RPW) {
      const int r = row0 + wave * RPW + lane % RPW;
      sa::async_copy_f32<true>(row_src + (r < live ? r : live - 1), row_ring + (qs * NW + wave) * 2 * RPW);
    }
    if (one_head) {
      ldq.at(it).issue(q_ring + qs * TILE, wave);
      ldg.at(it).issue(g_ring + gs * TILE, wave);
    } else {
      Gather::issue(q, p.q_sh, p.q_st, p.map, row0, live, q_ring + qs * TILE, wave, lane);
      Gather::issue(g, p.g_sh, p.g_st, p.map, row0, live, g_ring + gs * TILE, wave, lane);
    }
  };
  // this wave's rows first, over the rings
  using Rows = sa::OwnRows<T, D>;
  static_assert(NW * Rows::ELEMS * sizeof(T) <= S::lds, "rows of all waves");
  T* const area = q_ring + wave * Rows::ELEMS;
  if (grad_role) Rows::send(reinterpret_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh, p.v_st, wk0, L - 1, area, lane);
  else Rows::send(reinterpret_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh, p.k_st, wk0, L - 1, area, lane);
  sa::landed();
  // resident fragments: -K (K for a negative scale) for the score role, -V for the grad role; the scores as in dkdv_tile_16
  Frag rf[1][NF];
  {
    uint32_t flip = grad_role || !(p.scale_log2e < 0.0f) ? E::SIGN : 0u;
    asm("" : "+v"(flip));
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      const Frag f = Rows::read(area, i, lane);
      rf[0][i] = __builtin_bit_cast(Frag, __builtin_bit_cast(u32x4, f) ^ flip);
    }
  }
  const float score_mul = -sa::score_scale(p.scale_log2e);
  __syncthreads();
  if (n > 0) issue_tile(0, 0);
  if (n > 1) issue_tile(1, 1);
  f32x16 acc[1][DB];   // dV^T[d][key] (score role) or -dK^T[d][key] (grad role)
  clear(acc[0]);

  // lse (which = 0) or delta (which = 1) of the 16 rows of step it's tile that this lane holds in a C fragment
  auto rows16 = [&](int it, int which, f32x16& x) {
    const float* src = row_ring + (it & (NQ - 1)) * 2 * TQ + which * RPW;
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const int r = 8 * g4 + 4 * h;
      const f32x4 v4 = *reinterpret_cast<const f32x4*>(src + (r / RPW) * 2 * RPW + r % RPW);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * g4 + e] = v4[e];
    }
  };
  auto masked = [&](int it, f32x16& x) {   // the rows of the last tile that are not there
    const int row0 = (t0 + it) * TQ;
    if (row0 + TQ <= live) return;
    asm volatile("");   // a real branch, not selects
    const uint32_t mask = sa::row_mask(0, live - row0, h);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = sa::keep_or_zero(x[i], sa::keep_bits(mask, i));
  };
  int gs = 0;   // stage of the current dO tile
  auto begin_step = [&](int it) {
    if (it + 1 < n) sa::wait_loads<LPT>();
    else sa::wait_loads<0>();
    __syncthreads();
    if (it + 2 < n) issue_tile(it + 2, gs == 0 ? 2 : gs - 1);
  };
  if (!grad_role) {
    for (int it = 0; it < n; ++it, gs = gs == NG - 1 ? 0 : gs + 1) {
      begin_step(it);
      if (!seen) continue;
      f32x16 s[1][1];
      rows16(it, 0, s[0][0]);
      sa::mma_rows_n<T, D>(s, q_ring + (it & (NQ - 1)) * TILE, 0, rf, lane);          // lse / score_scale - S[row][key]
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][0][i] = sa::fast_exp2(s[0][0][i] * score_mul);
      masked(it, s[0][0]);
      float* slot = xbuf + (it & 1) * S::XSLOT;
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<f32x4*>(slot + g4 * 256) = f32x4{s[0][0][4 * g4], s[0][0][4 * g4 + 1], s[0][0][4 * g4 + 2], s[0][0][4 * g4 + 3]};
      Frag pf[1][2];
      sa::pack_c<T>(pf[0], s[0][0]);
      sa::mma_tr_n<T, D>(acc, g_ring + gs * TILE, 0, pf, lane);                        // dV^T[d][key] += dO^T P
    }
    __syncthreads();   // the grad role's last step
  } else {
    f32x16 dp[1][1];   // delta - dP of the step before
    clear(dp[0]);
    for (int it = 0;; ++it, gs = gs == NG - 1 ? 0 : gs + 1) {
      if (it < n) begin_step(it);
      else __syncthreads();
      const bool prev = it > 0 && seen;
      Frag df[1][2];
      if (prev) {
        const float* slot = xbuf + ((it - 1) & 1) * S::XSLOT;
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const f32x4 p4 = *reinterpret_cast<const f32x4*>(slot + g4 * 256);
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[0][0][4 * g4 + e] *= p4[e];   // = -dS
        }
        masked(it - 1, dp[0][0]);
        sa::pack_c<T>(df[0], dp[0][0]);
      }
      if (it < n && seen) {
        rows16(it, 1, dp[0][0]);
        sa::mma_rows_n<T, D>(dp, g_ring + gs * TILE, 0, rf, lane);                      // delta - dP[row][key]
      }
      if (prev) sa::mma_tr_n<T, D>(acc, q_ring + ((it - 1) & (NQ - 1)) * TILE, 0, df, lane);   // -dK^T += Q^T (-dS)
      if (it == n) break;
    }
  }
  const float mul = grad_role ? -p.scale : 1.0f;
  if (p.work.splits > 1) {
    const int64_t each = (int64_t)p.B * p.map.Hkv * p.Tk;
    if (key < L)
      sa::store_acc_T<float, D, DB>(p.part + ((int64_t)(split * 2 + (grad_role ? 0 : 1)) * each + (int64_t)bh * p.Tk + key) * D, acc[0], mul, h);
    return;
  }
  if (key >= L) clear(acc[0]);
  __syncthreads();   // the row patches lie over the rings
  store_rows<T, D, DB>(out, keys, bh, wk0, q_ring + wave * sa::RowPatch<T, D>::ELEMS, acc[0], mul, lane);
}

}  // namespace kv
