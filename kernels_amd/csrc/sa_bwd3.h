// Software-pipelined dK/dV kernel for 16-bit elements with swizzled tiles, head dimension 128.
//
// Same mathematics and the same ownership as dkdv2_kernel (a workgroup of 4 waves owns 128
// keys, a wave 32 of them with K, V fragments and the dK, dV accumulators in registers; query
// tiles of 64 rows stream through LDS).  What differs is the order of work inside a wave.  One
// wave per SIMD means that nothing but the wave's own instruction stream can fill the matrix
// pipe, and a v_mfma_32x32x16 keeps that pipe busy for 8 passes during which the same wave can
// issue about five ordinary vector instructions or LDS reads for free.  The loop is therefore a
// sequence of MFMA "slots": every slot issues one MFMA, the LDS read that a slot fifteen places
// later will consume, and a share of the vector work of the PREVIOUS 32-query block (scores ->
// probabilities -> dS).  Per block n the slots are
//     A(n+1):  S = Q K^T and dP = dO V^T of the next block     | exp2, rounding of P(n)
//     dV(n):   dV^T += dO^T P                                   | dS = P o (dP - delta), rounding
//     dK(n):   dK^T += Q^T dS                                   | window mask, lse / delta of the next blocks
// so the matrix pipe never waits for the softmax arithmetic.  Block n+1 may belong to the next
// query tile while block n still reads the current one: three LDS stages (two in use, one being
// filled).
//
// There is one loop body and no per-block branch: every wave walks all 32-query blocks of the
// workgroup's window.  The K fragments carry the factor -scale*log2(e) and the score accumulator
// of a block starts at the lse of its rows (read from LDS straight into the accumulator, as delta
// is for dP), so the MFMAs leave lse - score*scale*log2(e) and the probability is one v_exp away.
// A (query, key) pair outside the key's own window is masked by starting its accumulator at +inf
// instead, which makes its probability exp2(-inf) = 0 with no extra work in the busy phase.  The first step pairs the first block's scores with an all-masked
// phantom block, the last one forms scores that nobody reads.
//
// The loop needs about 400 registers per lane, which the compiler's register allocator does not
// place well (it keeps copying whole accumulators between the two register files).  The
// whole loop (block steps, loop control, barrier, tile loads) is therefore assembly with every
// register chosen by hand, generated by gen_dkdv3_asm.py into sa_dkdv3_asm.inc (register map
// there); this file keeps the set-up, the first tile loads and the epilogue in C++ and hands the
// state to the assembly in fixed registers.
#pragma once
#include <type_traits>
#include "sa_common.h"
#include "sa_dkdv3_asm.inc"

namespace sa {

typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef uint32_t u32x32 __attribute__((ext_vector_type(32)));
typedef uint32_t u32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));

// Accumulation registers that the second half of a 16-entry fragment ring occupies (none with 8 entries).
#if SA_DKDV3_RING == 16
#define SA_DKDV3_RING_CLOBBERS                                                                         \
  "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203",      \
  "a204", "a205", "a206", "a207", "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215",      \
  "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223",
#else
#define SA_DKDV3_RING_CLOBBERS
#endif

// State handed to the assembly, each value in the registers the generated text names.
#define SA_DKDV3_OPERANDS                                                                              \
  : "+{a[0:31]}"(r_dv0), "+{a[32:63]}"(r_dv1), "+{a[64:95]}"(r_dk0), "+{a[96:127]}"(r_dk1),            \
    "+{a[128:159]}"(r_kf), "+{a[160:191]}"(r_vf), "+{v[0:31]}"(r_s), "+{v[32:63]}"(r_dp),              \
    "+{v[64:95]}"(r_prlr), "+{v[96:111]}"(r_pbds), "+{v[112:143]}"(r_ring), "+{v[144:159]}"(r_arow),   \
    "+{v[160:175]}"(r_atr), "+{v[176:191]}"(r_base), "+{v192}"(r_aldb), "+{v193}"(r_qlo),              \
    "+{v194}"(r_qhi), "+{v195}"(r_h4), "+{v[208:239]}"(r_scal), "+{v[240:247]}"(r_ptrs)                \
  :                                                                                                    \
  : "v196", "v197", "v198", "v199", "v200", "v201", "v202", "v203", "v204", "v205", "v206", "v207",    \
    SA_DKDV3_RING_CLOBBERS                                                                             \
    "s40", "s41", "s42", "s43", "s44", "s45", "s46", "s47", "s48", "s49", "s50", "s51", "s52", "s53",  \
    "s54", "s55", "s56", "s57", "s58", "s59", "s60", "s61", "s62", "s63", "s64", "s65", "s66", "s67",  \
    "s68", "s69", "vcc", "scc", "m0", "memory"

template <typename T, int D, int NST, typename P = BwdParams>
__global__ __launch_bounds__(256) void dkdv3_kernel(const P p) {
  constexpr bool CROSS = IsCross<P>::value;
  using E = Elem<T>;
  using G = TileGeom<T, D>;
  using Frag = typename E::Frag;
  static_assert(G::SWZ && D == 128, "swizzled 16-bit tiles, head dimension 128");
  static_assert(NST == 3, "two stages in use, one being filled");
  constexpr bool BF16 = std::is_same<T, __bf16>::value;
  constexpr int NW = 4, TQ = 64, TKB = NW * 32, NT = NW * 64;
  constexpr int NF = G::NF, DB = G::DB;
  constexpr int ROWB = D * (int)sizeof(T);       // bytes per tile row
  constexpr int TILE_B = TQ * ROWB;              // bytes per Q or dO tile
  constexpr int TILE = TQ * D;                   // elements
  constexpr int RPW = TQ / NW;                   // rows of lse / delta each wave stages
  // stage layout: [Q tile][dO tile][NW chunks of {lse[RPW], delta[RPW]}]
  constexpr int STAGE_B = 2 * TILE_B + 2 * TQ * (int)sizeof(float);
  using Loader = AsyncTile<T, D, TQ, NW>;

  extern __shared__ __attribute__((aligned(16))) char smem_raw[];

  const int tid = threadIdx.x;
  const int lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  int bh, kt, L;
  key_tile_coords(blockIdx.x, gridDim.x, p.tiles, TKB, p.T, p.lens, p.lens_stride, bh, kt, L);
  const int b = div_by(bh, p.tiles.by_heads), hd = bh - b * p.H;
  int LQ = L, hq = hd, rows = p.T;   // queries, their first head, and how many a head of lse and delta has
  if constexpr (CROSS) {
    LQ = other_length(p, b), hq = hd * p.group, rows = p.other_T;
    L = __builtin_amdgcn_readfirstlane(L);
  }
  const int T_ = p.T, C = p.C, R = p.R;
  auto cdiv = [&](int x) { return div_by(x, p.cdiv); };   // x / C
  const int k0 = kt * TKB;
  T* dk_base = reinterpret_cast<T*>(p.dk) + (int64_t)bh * T_ * D;
  T* dv_base = reinterpret_cast<T*>(p.dv) + (int64_t)bh * T_ * D;
  const int k_end = k0 + TKB < T_ ? k0 + TKB : T_;
  if (k0 >= L || (CROSS && LQ == 0)) {
    zero_rows<T, D, NT>(dk_base, k0, k_end, tid);
    zero_rows<T, D, NT>(dv_base, k0, k_end, tid);
    return;
  }

  // ---- windows ---------------------------------------------------------------------------
  auto win_lo = [&](int key) { return CROSS ? 0 : (cdiv(key)) * C; };
  auto win_hi = [&](int key) {
    if (CROSS) return LQ;
    const int64_t e = ((int64_t)(cdiv(key)) + R + 1) * (int64_t)C;
    return e < (int64_t)L ? (int)e : L;
  };
  const int krow = k0 + wave * 32 + c;
  const int ke = krow < L ? krow : L - 1;   // keys past L mimic the last valid key
  const int wk_first = k0 + wave * 32 < L ? k0 + wave * 32 : L - 1;
  const int wk_last = k0 + wave * 32 + 31 < L ? k0 + wave * 32 + 31 : L - 1;
  // a 32-query block inside [qlo_max, qhi_min) is inside the window of every key of this wave
  const int qhi_min = win_hi(wk_first), qlo_max = win_lo(wk_last);
  const int gk_last = k0 + TKB - 1 < L ? k0 + TKB - 1 : L - 1;
  const int qt0 = win_lo(k0) / TQ, qt1 = (win_hi(gk_last) + TQ - 1) / TQ;

  // ---- asynchronous tile loads ---------------------------------------------------------
  const T* qbase = reinterpret_cast<const T*>(p.q) + (int64_t)b * p.q_sb + (int64_t)hq * p.q_sh;
  const T* gbase = reinterpret_cast<const T*>(p.d_o) + (int64_t)b * p.do_sb + (int64_t)hq * p.do_sh;
  const float* lse_base = p.lse + (int64_t)bh * rows;
  const float* delta_base = p.delta + (int64_t)bh * rows;
  auto stage_off = [&](int t) { return (uint32_t)(((t - qt0 + NST) % NST) * STAGE_B); };   // t >= qt0 - 1
  Loader ldq, ldg;
  ldq.init(qbase, p.q_st, qt0 * TQ, LQ - 1, wave, lane);
  ldg.init(gbase, p.do_st, qt0 * TQ, LQ - 1, wave, lane);
  auto issue_tile = [&](int t) {   // tiles are issued in ascending order
    char* sp = smem_raw + stage_off(t);
    T* st = reinterpret_cast<T*>(sp);
    // lanes [0, RPW) fetch lse, lanes [RPW, 2*RPW) fetch delta of this wave's RPW rows
    if (lane < 2 * RPW) {
      int r = t * TQ + wave * RPW + (lane % RPW);
      r = r < LQ ? r : LQ - 1;
      const float* src = (lane < RPW ? lse_base : delta_base) + r;
      float* dst = reinterpret_cast<float*>(sp + 2 * TILE_B) + wave * 2 * RPW;
      async_copy_f32(src, dst);
    }
    ldq.issue(st, wave);
    ldg.issue(st + TILE, wave);
    ldq.advance();
    ldg.advance();
  };
  // this wave's K rows go where the third tile will be, its V rows beside the stages
  using Rows = OwnRows<T, D>;
  T* const k_area = reinterpret_cast<T*>(smem_raw + (NST - 1) * STAGE_B) + wave * Rows::ELEMS;
  T* const v_area = reinterpret_cast<T*>(smem_raw + NST * STAGE_B) + wave * Rows::ELEMS;
  const int wrow0 = k0 + wave * 32;
  Rows::send(reinterpret_cast<const T*>(p.k) + (int64_t)b * p.k_sb + (int64_t)hd * p.k_sh, p.k_st, wrow0, L - 1, k_area, lane);
  Rows::send(reinterpret_cast<const T*>(p.v) + (int64_t)b * p.v_sb + (int64_t)hd * p.v_sh, p.v_st, wrow0, L - 1, v_area, lane);
#pragma unroll
  for (int i = 0; i < NST - 1; ++i)
    if (qt0 + i < qt1) issue_tile(qt0 + i);

  // ---- state handed to the assembly ------------------------------------------------------
  f32x32 r_dv0, r_dv1, r_dk0, r_dk1, r_s, r_dp, r_prlr;
  u32x32 r_kf, r_vf, r_ring;
  u32x16 r_pbds, r_arow, r_atr, r_base;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    r_dv0[i] = r_dv1[i] = r_dk0[i] = r_dk1[i] = r_s[i] = r_dp[i] = r_prlr[i] = 0.0f;
    r_kf[i] = r_vf[i] = r_ring[i] = 0u;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) r_pbds[i] = r_arow[i] = r_atr[i] = r_base[i] = 0u;
  {
    // K and V fragments of this lane's key.  V enters negated: the dP accumulator starts at delta
    // and ends at delta - dP.  K enters multiplied by -scale*log2(e) and rounded to the element
    // type: the score accumulator starts at lse and ends at lse - score*scale*log2(e), whose
    // negated exp2 is the probability, with no vector instruction between MFMA and v_exp.
    // CROSS: K enters with its sign turned (twice where the scale is negative), nothing rounded, and the accumulator of
    // lse / (scale*log2(e)) - score is multiplied once more.  Rounded to bfloat16 the scaled K took dK and dV of long runs 1.7 times
    // as far from the exact result as a rounding of them does, unscaled 1.4 times.
    const float kmul = CROSS ? (p.scale_log2e < 0.0f ? 1.0f : -1.0f) : -p.scale_log2e;
    landed();
#pragma unroll
    for (int g = 0; g < NF; ++g) {
      Frag kf = Rows::read(k_area, g, lane);
#pragma unroll
      for (int e = 0; e < E::VEC; ++e) kf[e] = (T)((float)kf[e] * kmul);
      const Frag vf = negate<T>(Rows::read(v_area, g, lane));
      const u32x4 ku = __builtin_bit_cast(u32x4, kf), vu = __builtin_bit_cast(u32x4, vf);
#pragma unroll
      for (int e = 0; e < 4; ++e) r_kf[4 * g + e] = ku[e], r_vf[4 * g + e] = vu[e];
    }
    // per-lane LDS byte offsets inside a stage (block 0 of the tile): row-major fragment g of this
    // lane's row; transposing reads of column block m, rows r_lo and r_lo + 8
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
  uint32_t r_aldb = 2 * TILE_B + h * 16;   // lse / delta of this half's rows
  uint32_t r_qlo = (uint32_t)win_lo(ke), r_qhi = (uint32_t)win_hi(ke), r_h4 = 4 * h;
  // all offsets are relative to the start of the workgroup's LDS allocation
  const uint32_t lds0 = (uint32_t)(uintptr_t)(SA_LDS char*)smem_raw;

  // ---- first tiles visible, the rows read: the third tile may come ----------------------------
  reads_done();
  __builtin_amdgcn_s_barrier();

  // wave-uniform inputs of the assembly, one per register of r_scal (names in sa_dkdv3_asm.inc)
  u32x32 r_scal;
  u32x8 r_ptrs;
#pragma unroll
  for (int i = 0; i < 32; ++i) r_scal[i] = 0u;
  {
    const int t0 = qt0 - 1;   // tile of the first step's B side: the phantom block's
    if constexpr (CROSS) r_scal[SA_DKDV3_SC_MUL] = __float_as_uint(-score_scale(p.scale_log2e));
    r_scal[SA_DKDV3_SC_QT1] = (uint32_t)qt1;
    r_scal[SA_DKDV3_SC_T] = (uint32_t)t0;
    r_scal[SA_DKDV3_SC_Q64] = (uint32_t)(64 * t0);
    r_scal[SA_DKDV3_SC_ST0] = lds0 + stage_off(t0);
    r_scal[SA_DKDV3_SC_ST1] = lds0 + stage_off(t0 + 1);
    r_scal[SA_DKDV3_SC_ST2] = lds0 + stage_off(t0 + 2);
    r_scal[SA_DKDV3_SC_WAVE_TILE] = (uint32_t)(wave * Loader::RPI * ROWB);
    r_scal[SA_DKDV3_SC_WAVE_ROWS] = (uint32_t)(2 * TILE_B + wave * 2 * RPW * (int)sizeof(float));
    r_scal[SA_DKDV3_SC_LAST_ROW] = (uint32_t)(LQ - 1);
    r_scal[SA_DKDV3_SC_QLO_MAX] = (uint32_t)qlo_max;
    r_scal[SA_DKDV3_SC_QHI_MIN] = (uint32_t)qhi_min;
    // buffer resources as Loader::init builds them: base, no stride, extent up to the last valid
    // row, raw 32-bit data format
    const uint64_t qa = (uint64_t)(uintptr_t)qbase, ga = (uint64_t)(uintptr_t)gbase;
    const uint32_t es = (uint32_t)sizeof(T);
    r_scal[SA_DKDV3_SC_RQ0] = (uint32_t)qa;
    r_scal[SA_DKDV3_SC_RQ1] = (uint32_t)(qa >> 32) & 0xffffu;
    r_scal[SA_DKDV3_SC_RQ2] = ((uint32_t)(LQ - 1) * (uint32_t)p.q_st + (uint32_t)D) * es;
    r_scal[SA_DKDV3_SC_RQ3] = 0x00020000u;
    r_scal[SA_DKDV3_SC_RG0] = (uint32_t)ga;
    r_scal[SA_DKDV3_SC_RG1] = (uint32_t)(ga >> 32) & 0xffffu;
    r_scal[SA_DKDV3_SC_RG2] = ((uint32_t)(LQ - 1) * (uint32_t)p.do_st + (uint32_t)D) * es;
    r_scal[SA_DKDV3_SC_RG3] = 0x00020000u;
    r_scal[SA_DKDV3_SC_SOFF_Q] = ldq.soff;
    r_scal[SA_DKDV3_SC_SOFF_G] = ldg.soff;
    r_scal[SA_DKDV3_SC_ISTEP_Q] = ldq.istep;
    r_scal[SA_DKDV3_SC_ISTEP_G] = ldg.istep;
    r_scal[SA_DKDV3_SC_TSTEP_Q] = ldq.tstep;
    r_scal[SA_DKDV3_SC_TSTEP_G] = ldg.tstep;
    // per-lane state of the tile loads: buffer offsets, the lse (lanes 0-15) or delta (lanes 16-31)
    // row pointer, and the row this lane fetches for the next tile the assembly issues (qt0 + 2)
    const uint64_t rp = (uint64_t)(uintptr_t)((lane & 31) < RPW ? lse_base : delta_base);
    r_ptrs[0] = ldq.voff[0];
    r_ptrs[1] = ldg.voff[0];
    r_ptrs[2] = (uint32_t)rp;
    r_ptrs[3] = (uint32_t)(rp >> 32);
    r_ptrs[4] = (uint32_t)((qt0 + 2) * TQ + wave * RPW + (lane % RPW));
    r_ptrs[5] = r_ptrs[6] = r_ptrs[7] = 0u;
  }
  if constexpr (CROSS && BF16) asm volatile(SA_DKDV3_MUL_128_BF16 SA_DKDV3_OPERANDS);
  else if constexpr (CROSS) asm volatile(SA_DKDV3_MUL_128_F16 SA_DKDV3_OPERANDS);
  else if constexpr (BF16) asm volatile(SA_DKDV3_128_BF16 SA_DKDV3_OPERANDS);
  else asm volatile(SA_DKDV3_128_F16 SA_DKDV3_OPERANDS);

  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int m = 0; m < DB; ++m)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dv[m][i] = m < 2 ? r_dv0[16 * m + i] : r_dv1[16 * (m - 2) + i];
      dk[m][i] = m < 2 ? r_dk0[16 * m + i] : r_dk1[16 * (m - 2) + i];
    }
  if (krow >= L) {
#pragma unroll
    for (int m = 0; m < DB; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[m][i] = 0.0f, dv[m][i] = 0.0f;
  }
  // the row patches lie over the tile stages: wait until no wave reads the last tile any more
  __syncthreads();
  {
    T* patch = reinterpret_cast<T*>(smem_raw) + wave * RowPatch<T, D>::ELEMS;
    const int row0 = k0 + wave * 32;
    store_rows_coalesced<T, D, DB>(patch, dk_base + (int64_t)row0 * D, T_ - row0, dk, -p.scale, lane);
    store_rows_coalesced<T, D, DB>(patch, dv_base + (int64_t)row0 * D, T_ - row0, dv, 1.0f, lane);
  }
}

}  // namespace sa
