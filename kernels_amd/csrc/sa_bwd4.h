// Software-pipelined dQ kernel for 16-bit elements with swizzled tiles, head dimension 128.
//
// Same mathematics as dq2_kernel, different ownership and order of work.  A workgroup of 4 waves
// owns 256 queries, a wave 64 of them (two blocks of 32) with their Q and dO fragments and both dQ
// accumulators in registers, one wave per SIMD with the whole register file.  Key tiles of 64 rows
// (K and V, two blocks of 32) stream through a ring of four LDS stages; every fragment read from LDS
// feeds two MFMAs, one per query block.  The loop is a sequence of MFMA slots: iteration j issues the
// 32 MFMAs of S(j+1) = K Q^T and delta - dP(j+1) and the 16 of dQ^T -= K^T (-dS(j-1)), and between them
// the vector arithmetic of block j (P = exp2(S c - lse), -dS = P (delta - dP), rounding), which
// depends on neither; scores, dP and the rounded dS are double-buffered.  Blocks that are not inside
// the window of every query of the wave take a masking detour.  A wave walks the tiles of its own queries'
// window; for the other tiles of the workgroup's window it only takes part in the tile hand-over.
//
// The loop is assembly with every register chosen by hand, generated by gen_dq3_asm.py into
// sa_dq3_asm.inc (register map there); this file keeps the set-up, the first tile loads and the
// epilogue in C++ and hands the state to the assembly in fixed registers.
//
// The set-up fetches 192 KiB of rows (Q, dO, O) for a workgroup; as sixteen-byte loads of 32 rows each they took 19400 of the
// 172600 cycles of a workgroup on chunks of 256, 8 back.  As copies of whole rows (OwnRows), with the same change to
// dkdv3_kernel: forward and backward at B=4, H=16, T=4096, chunks of 128, 4 back 470 -> 436 us, of 64, 3 back 318 -> 295.
#pragma once
#include <type_traits>
#include "sa_common.h"
#include "sa_dq3_asm.inc"

namespace sa {

typedef float f32x32_d3 __attribute__((ext_vector_type(32)));
typedef uint32_t u32x32_d3 __attribute__((ext_vector_type(32)));
typedef uint32_t u32x16_d3 __attribute__((ext_vector_type(16)));

// State handed to the assembly, each value in the registers the generated text names.
#define SA_DQ3_OPERANDS                                                                                 \
  : "+{a[0:31]}"(r_a0), "+{a[32:63]}"(r_a1), "+{a[64:95]}"(r_a2), "+{a[96:127]}"(r_a3),                 \
    "+{a[128:159]}"(r_q0), "+{a[160:191]}"(r_q1), "+{a[192:223]}"(r_g0), "+{a[224:255]}"(r_g1),         \
    "={v[0:31]}"(r_s0), "={v[32:63]}"(r_s1), "={v[64:95]}"(r_p0), "={v[96:127]}"(r_p1),                 \
    "={v[128:159]}"(r_ds), "+{v[160:191]}"(r_scal), "+{v[192:207]}"(r_addr), "+{v[208:239]}"(r_dinit),  \
    "+{v240}"(r_nl0), "+{v241}"(r_nl1), "+{v242}"(r_lo0), "+{v243}"(r_hi0), "+{v244}"(r_lo1),           \
    "+{v245}"(r_hi1), "+{v246}"(r_h4), "+{v247}"(r_voffk), "+{v248}"(r_voffv)                           \
  :                                                                                                     \
  : "v250", "v251", "v252", "v253", "v254", "v255",                                                     \
    "s40", "s41", "s42", "s43", "s44", "s45", "s46", "s47", "s48", "s49", "s50", "s51", "s52", "s53",   \
    "s54", "s55", "s56", "s57", "s58", "s59", "s60", "s61", "s62", "s63", "s64", "s65", "s66", "s67",   \
    "s68", "s69", "s70", "s71", "vcc", "scc", "m0", "memory"

template <typename T, int D, int NST, typename P = BwdParams>
__global__ __launch_bounds__(256) void dq3_kernel(const P p) {
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
  using Loader = AsyncTile<T, D, TK, NW>;

  extern __shared__ __attribute__((aligned(16))) char smem_raw[];

  const int tid = threadIdx.x;
  const int lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  int bh, qt;
  tile_coords(blockIdx.x, gridDim.x, p.tiles, bh, qt);
  int b, hd, hk;   // hk: head of k and v
  if constexpr (CROSS) {
    const int g = div_by(qt, p.by_q_tiles);
    qt -= g * p.q_tiles;
    b = div_by(bh, p.tiles.by_heads), hk = bh - b * (p.H / p.group);
    hd = hk * p.group + g, bh = b * p.H + hd;
  } else {
    b = div_by(bh, p.tiles.by_heads), hd = bh - b * p.H, hk = hd;
  }
  const int T_ = p.T, C = p.C, R = p.R;
  auto cdiv = [&](int x) { return div_by(x, p.cdiv); };   // x / C

  int L = T_;
  if (p.lens) {
    L = p.lens[(int64_t)b * p.lens_stride];
    L = L < 0 ? 0 : (L > T_ ? T_ : L);
  }
  const int q0 = qt * TQ;
  T* dq_base = reinterpret_cast<T*>(p.dq) + (int64_t)bh * T_ * D;
  const int q_end = q0 + TQ < T_ ? q0 + TQ : T_;
  int LK = L;   // keys
  if constexpr (CROSS) LK = other_length(p, b);
  if (q0 >= L || (CROSS && LK == 0)) {   // (without a key nobody reads delta)
    zero_rows<T, D, NT>(dq_base, q0, q_end, tid);
    if (!CROSS && p.delta_out)
      for (int r = q0 + tid; r < q_end; r += NT) p.delta_out[(int64_t)bh * T_ + r] = 0.0f;
    return;
  }

  // ---- windows: this lane's two queries, the wave's 64, the workgroup's 256 ----------------
  auto win_lo = [&](int q) { return CROSS ? 0 : (cdiv(q) > R ? cdiv(q) - R : 0) * C; };
  auto win_hi = [&](int q) { return CROSS ? LK : (cdiv(q) + 1) * C < L ? (cdiv(q) + 1) * C : L; };
  int qrow[2], qe[2];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    qrow[qb] = q0 + wave * WQ + qb * 32 + c;
    qe[qb] = qrow[qb] < L ? qrow[qb] : L - 1;   // queries past L mimic the last valid query
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

  // ---- asynchronous tile loads ---------------------------------------------------------
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
  // This wave's rows: Q where the third and fourth tiles will be, dO where the second will be and beside the stages.
  using Rows = OwnRows<T, D>;
  static_assert(NW * Rows::ELEMS * (int)sizeof(T) == STAGE_B, "32 rows per wave fill a stage");
  const T* qbase = reinterpret_cast<const T*>(p.q) + (int64_t)b * p.q_sb + (int64_t)hd * p.q_sh;
  const T* gbase = reinterpret_cast<const T*>(p.d_o) + (int64_t)b * p.do_sb + (int64_t)hd * p.do_sh;
  auto q_area = [&](int qb) { return reinterpret_cast<T*>(smem_raw + (2 + qb) * STAGE_B) + wave * Rows::ELEMS; };
  auto g_area = [&](int qb) { return reinterpret_cast<T*>(smem_raw + (qb == 0 ? 1 : NST) * STAGE_B) + wave * Rows::ELEMS; };
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    Rows::send(qbase, p.q_st, q0 + wave * WQ + qb * 32, L - 1, q_area(qb), lane);
    Rows::send(gbase, p.do_st, q0 + wave * WQ + qb * 32, L - 1, g_area(qb), lane);
  }
  issue_tile(kt0);

  // ---- state handed to the assembly ------------------------------------------------------
  f32x32_d3 r_a0, r_a1, r_a2, r_a3, r_s0, r_s1, r_p0, r_p1, r_dinit;
  u32x32_d3 r_q0, r_q1, r_g0, r_g1, r_ds;
  u32x16_d3 r_addr;
  // Only the accumulators start at zero.  The score and dS registers are outputs of the assembly and
  // the fragments and addresses are written in full below.  The entries of r_scal that carry nothing
  // hold a run-time value rather than a constant: a constant there is kept alive across the assembly
  // for later use and, with every register bound, the whole vector is spilled for it.
  u32x32_d3 r_scal;
#pragma unroll
  for (int i = 0; i < 32; ++i) r_a0[i] = r_a1[i] = r_a2[i] = r_a3[i] = 0.0f;
  // all offsets are relative to the start of the workgroup's LDS allocation
  const uint32_t lds0 = (uint32_t)(uintptr_t)(SA_LDS char*)smem_raw;
  float r_nl0, r_nl1;
  {
    // Q fragments (negated for a negative softmax scale) and negated dO fragments of this lane's two
    // queries; lse and delta of those queries
    const bool neg = p.scale_log2e < 0.0f;
    // delta = rowsum(O * dO) is formed here when the caller has not run the delta kernel
    // (no branch around the loads: a value defined on one side only is copied where the sides join, and the copy
    // waits for the load; without a row of O to read, the dO row is read)
    RowDots<T, D> dots[2];
    float lse_q2[2];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      dots[qb].load(p.delta_out ? reinterpret_cast<const T*>(p.o) + (int64_t)b * p.o_sb + (int64_t)hd * p.o_sh : gbase,
                    p.delta_out ? p.o_st : p.do_st, q0 + wave * WQ + qb * 32, L - 1, lane);
      // rows past L: P = exp2(S c - inf) = 0
      lse_q2[qb] = qrow[qb] < L ? p.lse[(int64_t)bh * T_ + qe[qb]] : INFINITY;
      if constexpr (CROSS) lse_q2[qb] = lse_q2[qb] == -INFINITY ? INFINITY : lse_q2[qb];   // a row that sees nothing
    }
    landed();
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
      for (int g = 0; g < NF; ++g) {
        Frag qf = Rows::read(q_area(qb), g, lane);
        if (neg) qf = negate<T>(qf);
        const Frag gf = negate<T>(Rows::read(g_area(qb), g, lane));
        const u32x4 qu = __builtin_bit_cast(u32x4, qf), gu = __builtin_bit_cast(u32x4, gf);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (qb == 0) r_q0[4 * g + e] = qu[e], r_g0[4 * g + e] = gu[e];
          else r_q1[4 * g + e] = qu[e], r_g1[4 * g + e] = gu[e];
        }
      }
    }
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) dots[qb].partial(g_area(qb), reinterpret_cast<float*>(q_area(qb)), lane);
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      const float lse_q = lse_q2[qb];
      float delta_q;
      if constexpr (CROSS) {
        delta_q = RowDots<T, D>::total(reinterpret_cast<const float*>(q_area(qb)), lane);
        if (LK <= FEW_KEYS) {
          Frag qf[NF], gf[NF];
#pragma unroll
          for (int g = 0; g < NF; ++g) {
            u32x4 qu, gu;
#pragma unroll
            for (int e = 0; e < 4; ++e) qu[e] = (qb == 0 ? r_q0 : r_q1)[4 * g + e], gu[e] = (qb == 0 ? r_g0 : r_g1)[4 * g + e];
            qf[g] = __builtin_bit_cast(Frag, qu), gf[g] = __builtin_bit_cast(Frag, gu);
          }
          delta_q = few_keys_delta<T>(kbase, p.k_st, vbase, p.v_st, LK, qf, gf, fabsf(p.scale_log2e), lse_q, lane);
        }
        if (h == 0 && qrow[qb] < L) {
          const int64_t at = p.token_major ? ((int64_t)(bh - (hd - hk * p.group)) * T_ + (int64_t)qrow[qb] * p.group + (hd - hk * p.group))
                                           : (int64_t)bh * T_ + qrow[qb];
          p.delta_out[at] = delta_q;
          p.lse_out[at] = lse_q / score_scale(p.scale_log2e);
        }
      } else if (p.delta_out) {
        delta_q = RowDots<T, D>::total(reinterpret_cast<const float*>(q_area(qb)), lane);
        if (h == 0 && qrow[qb] < T_) p.delta_out[(int64_t)bh * T_ + qrow[qb]] = qrow[qb] < L ? delta_q : 0.0f;
      } else {
        delta_q = p.delta[(int64_t)bh * T_ + qe[qb]];
      }
      if (qb == 0) r_nl0 = -lse_q;
      else r_nl1 = -lse_q;
#pragma unroll
      for (int i = 0; i < 16; ++i) r_dinit[16 * qb + i] = delta_q;
    }
    // LDS addresses of this lane's fragments in the wave's first tiles: row-major fragment g of this lane's
    // row in the K tile of tile wt0; transposing reads of column block m, rows r_lo and r_lo + 8, in
    // the K tile of the stage before it (that of tile wt0 - 1, which the first iteration reads and
    // does not use)
#pragma unroll
    for (int g = 0; g < NF; ++g)
      r_addr[g] = lds0 + stage_off(wt0) + (uint32_t)G::off(c, (g * 2 + h) * E::VEC) * (uint32_t)sizeof(T);
    const int g16 = lane >> 4, j = lane & 15;
    const int r_lo = 4 * (g16 >> 1) + (j >> 2);
    const int col = (g16 & 1) * 16 + 4 * (j & 3);
#pragma unroll
    for (int m = 0; m < DB; ++m) {
      r_addr[8 + m] = lds0 + stage_off(wt0 - 1) + (uint32_t)G::off(r_lo, m * 32 + col) * (uint32_t)sizeof(T);
      r_addr[12 + m] = lds0 + stage_off(wt0 - 1) + (uint32_t)G::off(r_lo + 8, m * 32 + col) * (uint32_t)sizeof(T);
    }
  }
  uint32_t r_lo0 = (uint32_t)win_lo(qe[0]), r_hi0 = (uint32_t)win_hi(qe[0]);
  uint32_t r_lo1 = (uint32_t)win_lo(qe[1]), r_hi1 = (uint32_t)win_hi(qe[1]);
  uint32_t r_h4 = 4 * h;
  uint32_t r_voffk = ldk.voff[0], r_voffv = ldv.voff[0];
  // never exactly 0, so that a masked score of -inf stays -inf after scaling
  const float sl2e = fmaxf(fabsf(p.scale_log2e), 1e-30f);

  // wave-uniform inputs of the assembly, one per register of r_scal (names in sa_dq3_asm.inc)
  {
#pragma unroll
    for (int i = 0; i < 32; ++i) r_scal[i] = __float_as_uint(sl2e);
    r_scal[SA_DQ3_SC_KT1] = (uint32_t)kt1;
    r_scal[SA_DQ3_SC_T] = (uint32_t)kt0;
    r_scal[SA_DQ3_SC_KB] = (uint32_t)(kt0 * TK);
    r_scal[SA_DQ3_SC_ST0] = lds0 + stage_off(kt0 - 1);
    r_scal[SA_DQ3_SC_ST1] = lds0 + stage_off(kt0);
    r_scal[SA_DQ3_SC_ST2] = lds0 + stage_off(kt0 + 1);
    r_scal[SA_DQ3_SC_ST3] = lds0 + stage_off(kt0 + 2);
    r_scal[SA_DQ3_SC_WAVE_TILE] = (uint32_t)(wave * Loader::RPI * ROWB);
    r_scal[SA_DQ3_SC_NINF] = 0xff800000u;
    r_scal[SA_DQ3_SC_LO_MAX] = (uint32_t)lo_max;
    r_scal[SA_DQ3_SC_HI_MIN] = (uint32_t)hi_min;
    // buffer resources as Loader::init builds them: base, no stride, extent up to the last valid
    // row, raw 32-bit data format
    const uint64_t ka = (uint64_t)(uintptr_t)kbase, va = (uint64_t)(uintptr_t)vbase;
    const uint32_t es = (uint32_t)sizeof(T);
    r_scal[SA_DQ3_SC_RK0] = (uint32_t)ka;
    r_scal[SA_DQ3_SC_RK1] = (uint32_t)(ka >> 32) & 0xffffu;
    r_scal[SA_DQ3_SC_RK2] = ((uint32_t)(LK - 1) * (uint32_t)p.k_st + (uint32_t)D) * es;
    r_scal[SA_DQ3_SC_RK3] = 0x00020000u;
    r_scal[SA_DQ3_SC_RV0] = (uint32_t)va;
    r_scal[SA_DQ3_SC_RV1] = (uint32_t)(va >> 32) & 0xffffu;
    r_scal[SA_DQ3_SC_RV2] = ((uint32_t)(LK - 1) * (uint32_t)p.v_st + (uint32_t)D) * es;
    r_scal[SA_DQ3_SC_RV3] = 0x00020000u;
    r_scal[SA_DQ3_SC_SOFF_K] = ldk.soff + ldk.tstep;   // of tile kt0 + 2
    r_scal[SA_DQ3_SC_SOFF_V] = ldv.soff + ldv.tstep;
    r_scal[SA_DQ3_SC_ISTEP_K] = ldk.istep;
    r_scal[SA_DQ3_SC_ISTEP_V] = ldv.istep;
    r_scal[SA_DQ3_SC_TSTEP_K] = ldk.tstep;
    r_scal[SA_DQ3_SC_TSTEP_V] = ldv.tstep;
    r_scal[SA_DQ3_SC_WFIRST] = (uint32_t)wt0;
    r_scal[SA_DQ3_SC_WEND] = (uint32_t)wt1;
  }

  // ---- first tile visible, the rows read: the second tile may come --------------------------
  reads_done();
  __builtin_amdgcn_s_barrier();
  // Its copies are formed from the state handed to the assembly, read back: the loaders' own scalars, kept this far, do not fit.
  asm volatile("" : "+v"(r_scal), "+v"(r_voffk), "+v"(r_voffv));
  {
    auto scal = [&](int i) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)r_scal[i]); };
    if (scal(SA_DQ3_SC_KT1) - scal(SA_DQ3_SC_T) > 1) {
      const uint32_t tile = scal(SA_DQ3_SC_ST2) + scal(SA_DQ3_SC_WAVE_TILE);
      auto copies = [&](int r, int soff, int istep, int back, uint32_t voff, uint32_t dst) {
        const u32x4 rsrc = {scal(r), scal(r + 1), scal(r + 2), scal(r + 3)};
        const uint32_t so = scal(soff) - scal(back);   // the state holds the offset of the tile after it
#pragma unroll
        for (int i = 0; i < Loader::PER_WAVE; ++i)
          copy_rows_asm(rsrc, voff, so + i * scal(istep), dst + i * NW * Loader::RPI * ROWB);
      };
      copies(SA_DQ3_SC_RK0, SA_DQ3_SC_SOFF_K, SA_DQ3_SC_ISTEP_K, SA_DQ3_SC_TSTEP_K, r_voffk, tile);
      copies(SA_DQ3_SC_RV0, SA_DQ3_SC_SOFF_V, SA_DQ3_SC_ISTEP_V, SA_DQ3_SC_TSTEP_V, r_voffv, tile + TILE_B);
    }
  }

  if constexpr (BF16) asm volatile(SA_DQ3_128_BF16 SA_DQ3_OPERANDS);
  else asm volatile(SA_DQ3_128_F16 SA_DQ3_OPERANDS);

  // ---- epilogue --------------------------------------------------------------------
  __syncthreads();   // the row patches lie over the tile stages
  // (lane and wave indices are derived again from the thread index, which passes through an empty
  // statement so that no value computed from it before the assembly is carried across: the one free
  // vector register holds the index itself)
  int tid2 = threadIdx.x;
  asm volatile("" : "+v"(tid2));
  const int lane2 = tid2 & 63, wave2 = __builtin_amdgcn_readfirstlane(tid2 >> 6);
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    f32x16 acc[DB];
#pragma unroll
    for (int m = 0; m < DB; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const f32x32_d3& src = qb == 0 ? (m < 2 ? r_a0 : r_a1) : (m < 2 ? r_a2 : r_a3);
        acc[m][i] = src[16 * (m & 1) + i];
      }
    const int row0 = q0 + wave2 * WQ + qb * 32;
    if (row0 + (lane2 & 31) >= L) {
#pragma unroll
      for (int m = 0; m < DB; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[m][i] = 0.0f;
    }
    T* patch = reinterpret_cast<T*>(smem_raw) + wave2 * RowPatch<T, D>::ELEMS;
    store_rows_coalesced<T, D, DB>(patch, dq_base + (int64_t)row0 * D, T_ - row0, acc, -p.scale, lane2);
  }
}

}  // namespace sa
