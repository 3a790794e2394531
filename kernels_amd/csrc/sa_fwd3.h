// Software-pipelined forward kernel for 16-bit elements with swizzled tiles, head dimension 128.
//
// Same mathematics as fwd2_kernel, different ownership and order of work.  A workgroup of 4 waves
// owns 256 queries, a wave 64 of them (two blocks of 32) with their Q fragments and both O
// accumulators in registers, one wave per SIMD.  Key tiles of 64 rows (two blocks of 32) stream
// through a ring of four LDS stages; every K or V fragment read from LDS feeds two MFMAs, one per
// query block.  The loop is a sequence of MFMA slots: iteration j issues the 16 MFMAs of
// S(j+1) = K Q^T and the 16 of O += V^T P(j-1), and between them the softmax arithmetic of block j
// (exp2 against the reference maximum as it stands, row sums, rounding), which depends on neither.
// Scores and rounded probabilities are double-buffered.  The block maximum is only looked for when a
// block's row sums show that the reference has been left behind by more than 8 (log2 units); that
// search, the new probabilities and the rescaling of O are detours off the loop.  Blocks that are not
// inside the window of every query of the wave take a masking detour first.  A wave walks the tiles of
// its own queries' window; for the other tiles of the workgroup's window it only takes part in the tile
// hand-over (its share of the loads, the barrier).
//
// The loop is assembly with every register chosen by hand, generated by gen_fwd3_asm.py into
// sa_fwd3_asm.inc (register map there); this file keeps the set-up, the first tile loads and the
// epilogue in C++ and hands the state to the assembly in fixed registers.
#pragma once
#include <type_traits>
#include "sa_common.h"
#include "sa_fwd3_asm.inc"

namespace sa {

typedef float f32x32_f3 __attribute__((ext_vector_type(32)));
typedef uint32_t u32x32_f3 __attribute__((ext_vector_type(32)));
typedef uint32_t u32x16_f3 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x8_f3 __attribute__((ext_vector_type(8)));

// State handed to the assembly, each value in the registers the generated text names.
#define SA_FWD3_OPERANDS                                                                                \
  : "+{a[0:31]}"(r_o0), "+{a[32:63]}"(r_o1), "+{a[64:95]}"(r_o2), "+{a[96:127]}"(r_o3),                 \
    "+{a[128:159]}"(r_q0), "+{a[160:191]}"(r_q1), "={v[0:31]}"(r_s0), "={v[32:63]}"(r_s1),              \
    "={v[64:95]}"(r_pb), "={v[128:143]}"(r_akrt), "+{v[144:159]}"(r_base),      \
    "={v[160:167]}"(r_av), "={v168}"(r_m0), "={v169}"(r_m1), "={v170}"(r_l0), "={v171}"(r_l1),          \
    "+{v176}"(r_lo0), "+{v177}"(r_hi0), "+{v178}"(r_lo1), "+{v179}"(r_hi1), "+{v180}"(r_h4),            \
    "+{v[208:239]}"(r_scal), "+{v240}"(r_voffk), "+{v241}"(r_voffv)                                     \
  :                                                                                                     \
  : "v172", "v173", "v174", "v175", "v181", "v182", "v183", "v184", "v185", "v186", "v187", "v188",     \
    "v189", "v190", "v191", "v192", "v193", "v194", "v195", "v196", "v197", "v198", "v199", "v200",     \
    "v201", "v202", "v203", "v204", "v205", "v206", "v207",                                             \
    "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203",     \
    "a204", "a205", "a206", "a207", "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215",     \
    "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223",                                     \
    "s40", "s41", "s42", "s43", "s44", "s45", "s46", "s47", "s48", "s49", "s50", "s51", "s52", "s53",   \
    "s54", "s55", "s56", "s57", "s58", "s59", "s60", "s61", "s62", "s63", "s64", "s65", "s66", "s67",   \
    "s68", "s69", "s70", "s71", "s72", "s73", "s74", "s75", "s76", "s77", "s78", "vcc", "scc", "m0", "memory"

template <typename T, int D, int NST, typename P = FwdParams>
__global__ __launch_bounds__(256) void fwd3_kernel(const P p) {
  constexpr bool CROSS = IsCross<P>::value;
  using E = Elem<T>;
  using G = TileGeom<T, D>;
  using Frag = typename E::Frag;
  static_assert(G::SWZ && D == 128, "swizzled 16-bit tiles, head dimension 128");
  static_assert(NST == 4, "three stages in use, one being filled");
  constexpr bool BF16 = std::is_same<T, __bf16>::value;
  constexpr int NW = 4, TK = 64, WQ = 64, TQ = NW * WQ, NT = NW * 64;
  constexpr int NF = G::NF, DB = G::DB;
  constexpr int ROWB = D * (int)sizeof(T);       // bytes per tile row
  constexpr int TILE_B = TK * ROWB;              // bytes per K or V tile
  constexpr int TILE = TK * D;                   // elements
  constexpr int STAGE_B = 2 * TILE_B;            // [K tile][V tile]
  using Loader = AsyncTile<T, D, TK, NW, true>;   // copies as assembly, like those inside the loop
  static_assert((size_t)NW * RowPatch<T, D>::ELEMS * sizeof(T) <= 2 * (size_t)STAGE_B, "row patches fit the last two stages");

  extern __shared__ __attribute__((aligned(16))) char smem_raw[];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int T_ = p.T, C = p.C, R = p.R;
  auto cdiv = [&](int x) { return div_by(x, p.cdiv); };   // x / C
  // Per-lane values are derived from a thread id the compiler cannot see through, once before the assembly and
  // once after it: derived once, they would be kept alive across the assembly, where every register is spoken
  // for, and spilled.
  auto lane_id = [&]() {
    int t = tid;
    asm volatile("" : "+v"(t));
    return t & 63;
  };

  // never exactly 0, so that a masked score of -inf stays -inf after scaling
  const float sl2e = fmaxf(fabsf(p.scale_log2e), 1e-30f);
  const bool neg = p.scale_log2e < 0.0f;
  // all offsets are relative to the start of the workgroup's LDS allocation
  const uint32_t lds0 = (uint32_t)(uintptr_t)(SA_LDS char*)smem_raw;

  // ---- state handed to the assembly ------------------------------------------------------
  // Only the accumulators start at zero; scores, probabilities and the addresses of the tile being
  // read are outputs of the assembly, the rest is written in full by prepare().
  f32x32_f3 r_o0, r_o1, r_o2, r_o3, r_s0, r_s1;
  u32x32_f3 r_q0, r_q1, r_pb, r_scal;
  u32x16_f3 r_akrt, r_base;
  u32x8_f3 r_av;
  float r_m0, r_m1, r_l0, r_l1;   // reference maximum and row sum per query block: set and returned by the assembly
  uint32_t r_lo0, r_hi0, r_lo1, r_hi1, r_h4, r_voffk, r_voffv;

  // what the epilogue needs to know of the tile
  struct Out {
    T* o_base;
    float* lse_base;
    int q0, L;
  } cu;
  cu.o_base = nullptr;
  cu.lse_base = nullptr;
  cu.q0 = cu.L = 0;

  using Rows = OwnRows<T, D>;
  static_assert(NW * Rows::ELEMS * (int)sizeof(T) == STAGE_B && NST == 4, "32 rows per wave fill a stage");
  auto q_area = [&](int qb) { return reinterpret_cast<T*>(smem_raw + (2 + qb) * STAGE_B) + wave * Rows::ELEMS; };
  // Sets the tile up: first two key tiles on their way into stages 0 and 1, the Q rows into stages 2 and 3 (read into
  // registers once they have landed), every other input of the assembly written.  A tile that lies beyond its sequence is zero-filled
  // here and reported as false.
  auto prepare = [&](int bid) -> bool {
    const int lane = lane_id(), c = lane & 31, h = lane >> 5;
    int bh, qt;
    tile_coords(bid, gridDim.x, p.tiles, bh, qt);
    int b, hd, hk;   // hk: head of k and v
    if constexpr (CROSS) {
      const int g = div_by(qt, p.by_q_tiles);
      qt -= g * p.q_tiles;
      b = div_by(bh, p.tiles.by_heads), hk = bh - b * (p.H / p.group);
      hd = hk * p.group + g, bh = b * p.H + hd;
    } else {
      b = div_by(bh, p.tiles.by_heads), hd = bh - b * p.H, hk = hd;
    }
    int L = T_;
    if (p.lens) {
      // a scalar load: the lengths are read-only for the whole launch
      typedef const __attribute__((address_space(4))) int32_t* ConstLens;
      L = *((ConstLens)(uintptr_t)p.lens + (int64_t)b * p.lens_stride);
      L = L < 0 ? 0 : (L > T_ ? T_ : L);
    }
    const int q0 = qt * TQ;
    T* o_base = reinterpret_cast<T*>(p.o) + (int64_t)bh * T_ * D;
    float* lse_base = p.lse ? p.lse + (int64_t)bh * T_ : nullptr;
    if (q0 >= L) {
      const int q_end = q0 + TQ < T_ ? q0 + TQ : T_;
      zero_rows<T, D, NT>(o_base, q0, q_end, tid);
      if (lse_base)
        for (int r = q0 + tid; r < q_end; r += NT) lse_base[r] = 0.0f;
      return false;
    }
    int LK = L;   // keys
    if constexpr (CROSS) {
      LK = other_length(p, b);
      if (LK == 0) {
        const int q_end = q0 + TQ < T_ ? q0 + TQ : T_;
        zero_rows<T, D, NT>(o_base, q0, q_end, tid);
        if (lse_base)
          for (int r = q0 + tid; r < q_end; r += NT) lse_base[r] = r < L ? -INFINITY : 0.0f;
        return false;
      }
    }
    cu.o_base = o_base;
    cu.lse_base = lse_base;
    cu.q0 = q0;
    cu.L = L;

    // windows: this lane's two queries, the wave's 64, the workgroup's 256
    auto win_lo = [&](int q) { return CROSS ? 0 : (cdiv(q) > R ? cdiv(q) - R : 0) * C; };
    auto win_hi = [&](int q) { return CROSS ? LK : (cdiv(q) + 1) * C < L ? (cdiv(q) + 1) * C : L; };
    int qe[2];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      const int qrow = q0 + wave * WQ + qb * 32 + c;
      qe[qb] = qrow < L ? qrow : L - 1;   // queries past L mimic the last valid query
    }
    const int wq_first = q0 + wave * WQ < L ? q0 + wave * WQ : L - 1;
    const int wq_last = q0 + wave * WQ + WQ - 1 < L ? q0 + wave * WQ + WQ - 1 : L - 1;
    // a 32-key block inside [lo_max, hi_min) is inside the window of every query of this wave
    const int lo_max = win_lo(wq_last), hi_min = win_hi(wq_first);
    const int gq_last = q0 + TQ - 1 < L ? q0 + TQ - 1 : L - 1;
    const int kt0 = win_lo(q0) / TK, kt1 = (win_hi(gq_last) + TK - 1) / TK;
    // the tiles that hold a key some query of this wave sees: outside them the wave only takes part in the hand-over
    int wt0 = win_lo(wq_first) / TK, wt1 = (win_hi(wq_last) + TK - 1) / TK;
    wt0 = wt0 > kt0 ? wt0 : kt0;
    wt1 = wt1 < kt1 ? wt1 : kt1;

    // asynchronous tile loads
    const T* kbase = reinterpret_cast<const T*>(p.k) + (int64_t)b * p.k_sb + (int64_t)hk * p.k_sh;
    const T* vbase = reinterpret_cast<const T*>(p.v) + (int64_t)b * p.v_sb + (int64_t)hk * p.v_sh;
    auto stage_off = [&](int t) { return (uint32_t)(((t - kt0 + NST) % NST) * STAGE_B); };   // t >= kt0 - 1
    Loader ldk, ldv;
    ldk.init(kbase, p.k_st, kt0 * TK, LK - 1, wave, lane);
    ldv.init(vbase, p.v_st, kt0 * TK, LK - 1, wave, lane);
    auto issue_tile = [&](int t) {   // tiles are issued in ascending order
      T* st = reinterpret_cast<T*>(smem_raw + stage_off(t));
      ldk.issue(st, wave);
      ldv.issue(st + TILE, wave);
      ldk.advance();
      ldv.advance();
    };
    // the first NST - 2 tiles; the assembly issues tile t + NST - 2 while it works on tile t
#pragma unroll
    for (int i = 0; i < NST - 2; ++i)
      if (kt0 + i < kt1) issue_tile(kt0 + i);

    // this wave's Q rows go where the third and fourth tiles will be
    const T* qbase = reinterpret_cast<const T*>(p.q) + (int64_t)b * p.q_sb + (int64_t)hd * p.q_sh;
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) Rows::send(qbase, p.q_st, q0 + wave * WQ + qb * 32, L - 1, q_area(qb), lane);
    // LDS byte offsets inside a stage (block 0 of the K tile): row-major fragment g of this lane's row;
    // transposing reads of column block m, rows r_lo and r_lo + 8
    {
#pragma unroll
      for (int g = 0; g < NF; ++g) r_base[g] = (uint32_t)G::off(c, (g * 2 + h) * E::VEC) * (uint32_t)sizeof(T);
      const int g16 = lane >> 4, j = lane & 15;
      const int r_lo = 4 * (g16 >> 1) + (j >> 2);
      const int col = (g16 & 1) * 16 + 4 * (j & 3);
#pragma unroll
      for (int m = 0; m < DB; ++m) {
        r_base[8 + m] = (uint32_t)G::off(r_lo, m * 32 + col) * (uint32_t)sizeof(T);
        r_base[12 + m] = (uint32_t)G::off(r_lo + 8, m * 32 + col) * (uint32_t)sizeof(T);
      }
    }
    r_lo0 = (uint32_t)win_lo(qe[0]), r_hi0 = (uint32_t)win_hi(qe[0]);
    r_lo1 = (uint32_t)win_lo(qe[1]), r_hi1 = (uint32_t)win_hi(qe[1]);
    r_h4 = 4 * h;
    r_voffk = ldk.voff[0], r_voffv = ldv.voff[0];

    // wave-uniform inputs of the assembly, one per register of r_scal (names in sa_fwd3_asm.inc)
    // (the entries that carry nothing hold a run-time value rather than a constant: a constant there is
    // kept alive across the assembly for later use and, with every register bound, spilled for it)
#pragma unroll
    for (int i = 0; i < 32; ++i) r_scal[i] = __float_as_uint(sl2e);
    r_scal[SA_FWD3_SC_KT1] = (uint32_t)kt1;
    r_scal[SA_FWD3_SC_T] = (uint32_t)kt0;
    r_scal[SA_FWD3_SC_KB] = (uint32_t)(kt0 * TK);
    r_scal[SA_FWD3_SC_ST0] = lds0 + stage_off(kt0 - 1);
    r_scal[SA_FWD3_SC_ST1] = lds0 + stage_off(kt0);
    r_scal[SA_FWD3_SC_ST2] = lds0 + stage_off(kt0 + 1);
    r_scal[SA_FWD3_SC_ST3] = lds0 + stage_off(kt0 + NST - 2);
    r_scal[SA_FWD3_SC_WFIRST] = (uint32_t)wt0;
    r_scal[SA_FWD3_SC_WEND] = (uint32_t)wt1;
    r_scal[SA_FWD3_SC_WAVE_TILE] = (uint32_t)(wave * Loader::RPI * ROWB);
    r_scal[SA_FWD3_SC_NINF] = 0xff800000u;
    r_scal[SA_FWD3_SC_LO_MAX] = (uint32_t)lo_max;
    r_scal[SA_FWD3_SC_HI_MIN] = (uint32_t)hi_min;
    // buffer resources as Loader::init builds them: base, no stride, extent up to the last valid
    // row, raw 32-bit data format
    const uint64_t ka = (uint64_t)(uintptr_t)kbase, va = (uint64_t)(uintptr_t)vbase;
    const uint32_t es = (uint32_t)sizeof(T);
    r_scal[SA_FWD3_SC_RK0] = (uint32_t)ka;
    r_scal[SA_FWD3_SC_RK1] = (uint32_t)(ka >> 32) & 0xffffu;
    r_scal[SA_FWD3_SC_RK2] = ((uint32_t)(LK - 1) * (uint32_t)p.k_st + (uint32_t)D) * es;
    r_scal[SA_FWD3_SC_RK3] = 0x00020000u;
    r_scal[SA_FWD3_SC_RV0] = (uint32_t)va;
    r_scal[SA_FWD3_SC_RV1] = (uint32_t)(va >> 32) & 0xffffu;
    r_scal[SA_FWD3_SC_RV2] = ((uint32_t)(LK - 1) * (uint32_t)p.v_st + (uint32_t)D) * es;
    r_scal[SA_FWD3_SC_RV3] = 0x00020000u;
    r_scal[SA_FWD3_SC_SOFF_K] = ldk.soff;
    r_scal[SA_FWD3_SC_SOFF_V] = ldv.soff;
    r_scal[SA_FWD3_SC_ISTEP_K] = ldk.istep;
    r_scal[SA_FWD3_SC_ISTEP_V] = ldv.istep;
    r_scal[SA_FWD3_SC_TSTEP_K] = ldk.tstep;
    r_scal[SA_FWD3_SC_TSTEP_V] = ldv.tstep;
    return true;
  };

  // Normalises and stores one query block of the tile from the accumulators, through row patches in the last two stages.
  auto epilogue = [&](int qb) {
    const int lane = lane_id(), c = lane & 31, h = lane >> 5;
    {
      f32x16 oacc[DB];
#pragma unroll
      for (int m = 0; m < DB; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f32x32_f3& src = qb == 0 ? (m < 2 ? r_o0 : r_o1) : (m < 2 ? r_o2 : r_o3);
          oacc[m][i] = src[16 * (m & 1) + i];
        }
      const float m_run = qb == 0 ? r_m0 : r_m1;
      const float l_tot = half_sum(qb == 0 ? r_l0 : r_l1);
      const int qrow = cu.q0 + wave * WQ + qb * 32 + c;
      const bool valid = qrow < cu.L, some = !CROSS || !(l_tot == 0.0f);   // (some: a score above -inf)
      const float inv = valid && some ? 1.0f / l_tot : 0.0f;
      if (!valid || !some) {
#pragma unroll
        for (int m = 0; m < DB; ++m)
#pragma unroll
          for (int i = 0; i < 16; ++i) oacc[m][i] = 0.0f;
      }
      T* patch = reinterpret_cast<T*>(smem_raw + (NST - 2) * STAGE_B) + wave * RowPatch<T, D>::ELEMS;
      const int row0 = cu.q0 + wave * WQ + qb * 32;
      if (row0 < T_)
        store_rows_coalesced<T, D, DB>(patch, cu.o_base + (int64_t)row0 * D, T_ - row0, oacc, inv, lane);
      if (cu.lse_base && h == 0 && qrow < T_)
        cu.lse_base[qrow] = valid ? (some ? m_run + __builtin_amdgcn_logf(l_tot) : -INFINITY) : 0.0f;
    }
  };

  // ---- one tile per workgroup ---------------------------------------------------------------------
  if (!prepare((int)blockIdx.x)) return;
#pragma unroll
  for (int i = 0; i < 32; ++i) r_o0[i] = r_o1[i] = r_o2[i] = r_o3[i] = 0.0f;
  // first tiles and the Q rows here
  landed();
  {
    const int lane = lane_id();
#pragma unroll
    for (int g = 0; g < NF; ++g) {
      const u32x4 f0 = __builtin_bit_cast(u32x4, Rows::read(q_area(0), g, lane));
      const u32x4 f1 = __builtin_bit_cast(u32x4, Rows::read(q_area(1), g, lane));
#pragma unroll
      for (int e = 0; e < 4; ++e) r_q0[4 * g + e] = f0[e], r_q1[4 * g + e] = f1[e];
    }
  }
  reads_done();
  __builtin_amdgcn_s_barrier();
  if (neg) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      r_q0[i] ^= E::SIGN;
      r_q1[i] ^= E::SIGN;
    }
  }
  if constexpr (BF16) asm volatile(SA_FWD3_128_BF16 SA_FWD3_OPERANDS);
  else asm volatile(SA_FWD3_128_F16 SA_FWD3_OPERANDS);
  __syncthreads();   // every wave is done with the tile stages: the row patches may go there
  epilogue(0);
  epilogue(1);
}

}  // namespace sa
