// Launches of the kernels for keys that are not the queries' own, one explicit instantiation per element type and group of head
// dimensions (1: 256), and the rules by which work is divided.  Each returns 0, a hipError_t or a KV_ERR_* code.
#pragma once
#include <algorithm>
#include "../../include/kv_attention.h"
#include "kv_bwd.h"
#include "kv_rows.h"
#include "kv_tree.h"
#ifndef SA_NO_ASM_KERNELS
#include "sa_bwd3.h"
#include "sa_bwd4.h"
#include "sa_fwd3.h"
#endif

namespace kv {

template <typename T, int DGROUP> int launch_cross_fwd(const FwdParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_cross_dq(const BwdParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_cross_dkdv(const BwdParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_rows(const RowsParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_rows_paged(const RowsParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_rows_tree(const TreeParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_tree(const TreeParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_join(const JoinParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_join_many(const JoinParams& p, int D, hipStream_t st);   // one set of threads to a row, however many parts
template <typename T, int DGROUP> int launch_sum(const SumParams& p, int D, hipStream_t st);

// The hand-scheduled kernels of streaming attention on another sequence's keys: 16-bit elements, head dimension 128.  -DSA_NO_ASM_KERNELS
// leaves them out, as in sa_launch.h.
#ifdef SA_NO_ASM_KERNELS
constexpr bool HAVE_ASM_KERNELS = false;
#else
constexpr bool HAVE_ASM_KERNELS = true;
#endif
using LongFwd = sa::CrossOf<sa::FwdParams>;
using LongBwd = sa::CrossOf<sa::BwdParams>;
template <typename T> int launch_long_fwd(const LongFwd& p, hipStream_t st);
template <typename T> int launch_long_dq(const LongBwd& p, hipStream_t st);
template <typename T> int launch_long_dkdv(const LongBwd& p, hipStream_t st);

constexpr int64_t kMostCount = 0x7fffffff;   // pairs, rows, keys: what the kernels count in 31 bits
// The runtime takes fewer than 2^32 threads along a dimension of a grid.
inline bool launchable(int64_t blocks, int threads) { return blocks <= 0xffffffffLL / threads; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int TILE_ROWS = 128;   // rows (or keys) of a workgroup of the tile kernels: four waves of 32
constexpr int CUS = 256;

// How the run of tiles that each workgroup of the tile kernels goes through is divided.
//   Up to half as many workgroups as CUs: shares of at least two tiles, as long as there is a CU for each; of one in float32, whose tile takes
//   3-10 us (kernels of a pass in us, two -> one: 2 x 4 x 50 rows over up to 512, D = 64 55 -> 44; 4 x 8 x 100 over 130 63 -> 52; 4 x 300 over
//   150, D = 256 214 -> 168; bfloat16, 4 x 8 x 100 over 130, D = 64 23 -> 33).
//   Up to as many: shares of at least eight, up to 64 of them (adding up more costs what they save), as long as there is a place
//   for each (`places` workgroups fit a CU).  Forward and backward in us,
//   without -> with: 4 x 1 x 6105 rows over up to 14047 keys, D = 64 539 -> 388; 2 x 12 x 900 over 8000 303 -> 239; 2 x 4 x 3000 over 3000 162 -> 136;
//   12 x 8 x 5335 over 4 171 -> 117; D = 128, 2 x 16 x 300 over 4000 167 -> 156.  With more workgroups than CUs, 8 x 12 x 448 over up to
//   1500, D = 64 101 -> 112; at D = 256 2 x 3 x 4039 over up to 1246 184 -> 195.
//   Forward and dQ, where the workgroups do not fill the CUs several times over: shares of at most 100 tiles.  3 x 16 x 1424 over 14631,
//   4 key heads, D = 64 1350 -> 1244, with lengths from 64 on 1332 -> 1222; D = 256, 4 x 8 x 900 over up to 6000 714 -> 650.  Shares of 64: 4 x 12 x
//   1574 over 5451, lengths from 64 on 319 -> 351.  dK and dV, whose parts are twice as large: 4 x 12 x 5451 over 1574 407 -> 468 with 64.
struct Shares {
  int splits, share;
};
inline Shares tile_shares(int64_t workgroups, int64_t tiles, int places, bool keys, bool f32) {
  const int least = f32 ? 1 : 2;
  if (workgroups == 0 || tiles < 2 * least) return {1, 1};
  int64_t share = tiles;
  if (workgroups <= CUS / 2) share = std::max<int64_t>(least, ceil_div(tiles, CUS / workgroups));
  if (workgroups <= CUS) share = std::min(share, std::max<int64_t>(8, ceil_div(tiles, std::min<int64_t>(64, places * CUS / workgroups))));
  if (!keys && workgroups <= 4 * CUS) share = std::min(share, std::max<int64_t>(100, ceil_div(tiles, 8 * CUS / workgroups)));
  return {(int)ceil_div(tiles, share), (int)share};
}
// Workgroups of the forward and dQ, and of dK and dV, that fit a CU (their registers; head dimension 256 gains nothing from a second one).
inline int row_places(int row_bytes) { return row_bytes <= 128 ? 3 : row_bytes == 256 ? 2 : 1; }
inline int key_places(int row_bytes) { return row_bytes <= 128 ? 3 : 1; }

// Few tiles to a pair: tile by tile.
inline bool tiles_first(int64_t tiles) { return tiles <= 4; }

// Where the hand-scheduled kernels are taken.  Forward and dQ: a workgroup owns 256 queries of one head and a CU; from 512 keys on, where there is
// one for every CU and its rows are filled.  Forward, dQ in us, tile kernels -> these, bfloat16 and float16: 2 x 32 x 4096 queries over
// 8192 keys, 8 key heads 1000, 1354 -> 957, 1248; 32 x 16 x 200 over up to 1000 61.9, 74.6 -> 62.3, 78.6, and with
// a pass among others 273 -> 257 for all; 16 x 16 x 256 over 1500 57.6, 77.9 -> 55.0, 76.0;
// on the other side 8 x 16 x 1000 over 300 27.3, 38.5 -> 33.5, 43.6; 300 rows over 3000, ragged 71, 88 -> 76, 91; 4000 over 128 38.6, 62.8 -> 53.7,
// 77.3.  dK and dV: from 384 rows of a key head on, where there is a workgroup of 128 keys for every CU: the first 2308 -> 1760; 8 heads
// of 8000 over 8000 562 -> 430; 400 rows over up to 1000 123 -> 111; 1024 over 1500 133 -> 108; 300 over 3000, ragged 106 -> 107.
constexpr int LONG_ROWS = 256;
inline bool long_rows(int64_t heads, int64_t Tq, int64_t Tk) {
  const int64_t tiles = ceil_div(Tq, LONG_ROWS);
  return Tk >= 512 && 4 * Tq >= 3 * tiles * LONG_ROWS && heads * tiles >= CUS;
}
inline bool long_keys(int64_t key_heads, int64_t rows, int64_t Tk) { return rows >= 384 && key_heads * ceil_div(Tk, TILE_ROWS) >= CUS; }

// The rows kernel serves up to 32 rows of a key head.
inline bool few_rows(int64_t rows) { return rows <= 32; }
// How its keys are divided, from the sizes of the call: at most n tiles of 32 keys for each of `units` workgroups of `rows` rows.  A share is
// what leaves one workgroup for each CU if every sequence has all n tiles (a table that is much wider than its sequences leaves few workgroups:
// 8 units of 4096 positions, D = 128, 16-bit 10.7 us in a table of 4096, 17.9 in one of 32768, 47 in one of 131072), from four tiles on; short
// runs are not divided (the joining kernel takes about 4 us), and shares of
// many workgroups stay short, so that long sequences of a batch spread over the CUs that short ones have left: 16 tiles where workgroups go
// through the parts that there are (by_length), else 32, as parts that the lengths leave empty have workgroups then.  By length this begins at 48
// units: fewer keep their shares of up to 128 (us, -> 16 tiles, D = 128, 16-bit: all of 131072 4 x 8 368 -> 398, 5 x 8 470 -> 496, 3 x 8 303 -> 305;
// from half of 131072 on 4 x 8 314 -> 325, 3 x 8 290 -> 255; log-uniform up to 32768 5 x 8 67 -> 59, 12 x 2 40 -> 24, up to 131072 5 x 8 182 -> 186, 12 x 2
// 117 -> 71); from 48 on 6 x 8 log-uniform up to 131072 211 -> 184, all of 32768 156 -> 155, of 131072 546 -> 588; 8 x 8 log-uniform
// up to 32768 115 -> 62.  float32 is bound by its matrix instructions and gains by every division, down to one tile to a wave (128 units of 63 tiles, D = 64: 55 us in one share, 37 in two; 2 units of
// 13, D = 128 38 in one, 11.7 in seven; 32 of 10, D = 64 12.1 and 8.8).
// One token per sequence, in us for shares of 4, 8, 16, 32, 64, 128 tiles (* chosen), 16-bit elements, D = 128, four waves: 8 units of 63
// tiles 9.5*, 9.7, 12.0, 15.9, 22.3; of 1000 60.9, 45.9, 34.9, 28.0*, 32.2, 49.7; 32 units of 63 16.2, 12.6*, 14.2, 18.1, 25.1; of 250 49.7, 36.7, 29.6,
// 26.7*, 32.2, 50.2; 128 units of 16 16.3, 13.1, 11.0*; of 63 45.2, 35.7, 29.8, 26.9*, 28.9; two waves: 512 units of 16 33.4, 29.9, 23.8*; of
// 63 121, 111, 105, 99.7, 94.5*.  By length, shares of 12, 16*, 24, 32, 64: 64 sequences x 8 key heads of lengths log-uniform from 64 to 8192 98.7, 95.2, 95.6, 99.6,
// 117 (a workgroup for each part: 117, 112, 107, 107, 115); 16 x 8 31.5, 31.0, 31.1, 35.8, 60.4; 8 x 8 23.2, 21.6, 24.8, 30.7, 28.8; all of 8192 62.5, 58.3, 62.7, 54.8, 55.0; 2 x 8
// of 131072 208, 208, 206, 196, 192 and 187 with 128* (D = 32, 28 x 12 of up to 15484 80, 80, 76, 75, 71, a workgroup
// for each part of 32 69*).  D = 64, four waves: 8 units of 63 8.3*, 8.3, 9.9, 12.7, 16.5; 32 of 63
// 9.9, 9.0*, 10.7, 13.6, 17.4; 512 units of 63 78.3, 63.3, 57.5, 54.4, 49.2*; eight waves: 128 units of 63 35.3, 24.4, 20.6, 16.9, 15.3* (four: 19.7).
inline bool by_length(int64_t B, int64_t row_tiles, int row_bytes) { return B <= MAX_BY_LENGTH && row_tiles == 1 && row_bytes >= 128; }
inline int rows_share(int64_t units, int rows, int64_t n, int row_bytes, bool f32, bool by_length) {
  const int64_t least = !f32 || row_bytes <= 256 ? 4 : row_bytes == 512 ? 2 : 1;
  if (n <= (f32 ? 2 * least : row_bytes <= 128 ? 32 : 16)) return (int)std::max<int64_t>(n, 1);
  int64_t share = std::max(least, ceil_div(units * n, CUS));
  if (2 * share >= n && n <= 64 && !f32) return (int)n;
  const int64_t most_of_many = by_length ? 16 : 32;
  if ((units >= 48 || !by_length) && share > most_of_many && units * ceil_div(n, most_of_many) >= 4 * CUS) share = most_of_many;
  share = std::min<int64_t>(share, 128);
  // at most 256 parts to add up, and 256 MiB of them (the chunks of many long sequences)
  const int64_t part = units * rows * (row_bytes / (f32 ? 4 : 2) + 2) * 4;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(256, (256 << 20) / part));
  return (int)std::max(share, ceil_div(n, most));
}
// Waves of its workgroups, whose rings take most of the LDS.  Rows of 128 bytes: eight, one workgroup to a CU, where there are few workgroups with long
// shares or a CU for each (float16, us, four -> eight: 8 units of 10 tiles 6.1 -> 5.8; 16 of 22 8.2 -> 7.5), else four.  256 bytes: two where there is more than one workgroup for each place, so that one begins while the other one is in its
// run (512 units of 16 tiles 27.1 -> 23.8 us), else four; float32, whose matrix instructions take their time, always four: two waves of two
// workgroups may share a SIMD (128 units of 63 tiles 38 -> 54).
constexpr int rows_waves(int row_bytes, bool f32, int64_t workgroups, int share) {
  const bool many = workgroups >= 2 * CUS;
  if (row_bytes == 128) return (!many && share >= 24) || (workgroups <= CUS && share > 8) ? 8 : 4;
  if (row_bytes == 256) return many && !f32 ? 2 : 4;
  return row_bytes < 128 ? 4 : row_bytes == 512 ? 2 : 1;
}

// Trees: the rows kernel up to 32 rows of a key head and for little work altogether (blocks of 32 rows times tiles of 32 keys: few for each wave
// of the GPU), else the tile kernel.  Rows -> tiles, in us, D = 128, bfloat16: 64 rows, 8 key heads of 1000 11.7 -> 13.5, of 4096 14.1 -> 15.4, 32 of 4096 (8192
// blocks) 23.1 -> 20.8; 256 rows, 8 of 4096 (8192) 21.5 -> 23.9; 64 rows, 96 of 2000 (12096) 27.9 -> 23.5; 128 rows, 16 of 8192 31.5 -> 26.3; 256 rows, 64 of 8192 201 -> 92.  D = 256: 40
// rows, 16 of 500 18.7-25 -> 17.6, 64 of 2000 45-72 -> 32.  float32: 40 rows, 32 of 1000, D = 64 (2048) 14.9 -> 20.9; 256 rows, 16 of 2000, D = 128 95 -> 56.
inline bool tree_by_rows(int64_t units, int64_t rows, int64_t tiles, int row_bytes, bool f32) {
  const int64_t blocks = units * ceil_div(rows, 32) * tiles;
  return rows <= 32 || (f32 ? row_bytes <= 512 && blocks <= 4096 : row_bytes <= 256 && blocks <= 8192);
}
// Its waves: two of 32 rows, each twice where a tile has two blocks of keys, or four.  In us, two twice -> four: 64 rows, D = 128, 256 key heads of
// lengths log-uniform from 64 to 8192 50 -> 65, from 4096 on 168 -> 172; 256 rows, 64 of 8192 110 -> 92, from 4096 on and with fewer rows 88 -> 72; 800
// rows, 32 of 8000, D = 64 105 -> 93.
constexpr int tree_waves(int64_t rows) { return rows <= 64 ? 2 : 4; }
// Tiles (of 64 keys, or of 32 where rows take more than 256 bytes) of a part: what leaves a workgroup for each place, at least eight, or four where
// those leave half of the CUs without one, at most 2048 keys (1024 for four waves at D <= 64): a part writes and reads again 520 bytes for each of its rows at
// D = 128, an eighth of the keys and values of 2048 for 128 rows.  In us for shares of 4, 8, 16, 32 tiles (* chosen), means over three sets of
// lengths, bfloat16: 64 rows, D = 128, 256 key heads of 8192 307, 273, 236, 217*; from 4096 on 240, 212, 190, 178*; from 1 on 174, 154, 135, 136*; log-uniform
// 87, 76, 69, 65*; 96 of 2000 37, 28*, 28, 38; 256 rows, 64 of 8192 172, 134, 108, 95*, log-uniform 71, 62, 56, 72*; 128 rows, 128 of 4096 120, 92, 79*, 67,
// from 1 on 68, 55, 50*, 58, log-uniform 46, 40, 45*, 57; 240 rows, 15 of 6000 43, 36*, 36, 55; D = 64: 60 rows, 192 of 4000 55, 46, 41*, 41, log-uniform 28, 24, 26*, 36;
// 100 rows, 128 of 4000 55, 46, 42*, 50; D = 256: 80 rows, 64 of up to 2000 66, 50, 42*, 62.
// Where the workgroups of whole runs of up to 4096 keys fill every place, none is divided: nothing to write and join (runs in two or four parts -> whole, lengths
// full, from half on, from 1 on, log-uniform: 64 rows, 512 key heads of 4096, D = 128 218 -> 185, 181 -> 154, 129 -> 118, 65 -> 76; 128 rows 248 -> 193, 211 -> 167, 158 -> 132, 96 -> 101; 256 rows
// 501 -> 387, 416 -> 322, 273 -> 225, 163 -> 144; D = 64, 200 rows, 384 of 4000 206 -> 164, 159 -> 133, 111 -> 103, 78 -> 84).  Of 8192 keys the few longest run alone: 256 rows, 256 key heads 407 -> 363, 323 -> 290,
// 223 -> 255, 128 -> 213; so do D = 256's of 4096, 60 rows 445 -> 416, 367 -> 346, 262 -> 268, 155 -> 218, D = 32's, 100 rows, 768 of 4000 154 -> 144, 122 -> 115, 80 -> 89, 57 -> 74,
// and float32's, D = 64, 40 rows, 768 of 4000 487 -> 482, 387 -> 429, 289 -> 279, 183 -> 221.
inline int tree_share(int64_t workgroups, int64_t tiles, int row_bytes, int waves, bool f32) {
  const int64_t places = waves == 2 ? (row_bytes <= 128 ? 3 : 2) : (row_bytes <= 128 ? 3 : row_bytes == 256 ? 2 : 1);
  if (!f32 && (row_bytes == 128 || row_bytes == 256) && tiles <= 64 && workgroups >= places * CUS) return (int)std::max<int64_t>(tiles, 1);
  const int64_t least = workgroups * ceil_div(tiles, 8) > CUS / 2 ? 8 : 4;
  const int64_t most = row_bytes > 256 ? 64 : waves == 4 && row_bytes <= 128 ? 16 : 32;
  const int64_t share = std::min(most, std::max(least, ceil_div(workgroups * tiles, places * CUS)));
  return (int)std::min(std::max<int64_t>(tiles, 1), share);
}

}  // namespace kv
