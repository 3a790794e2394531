// Launches of the kernels for keys that are not the queries' own, one explicit instantiation per element type and group of head
// dimensions (1: 256), and the rules by which work is divided.  Each returns 0, a hipError_t or a KV_ERR_* code.
#pragma once
#include <algorithm>
#include "../../include/kv_attention.h"
#include "kv_bwd.h"
#include "kv_rows.h"

namespace kv {

template <typename T, int DGROUP> int launch_cross_fwd(const FwdParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_cross_dq(const BwdParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_cross_dkdv(const BwdParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_rows(const RowsParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_rows_paged(const RowsParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_join(const JoinParams& p, int D, hipStream_t st);
template <typename T, int DGROUP> int launch_sum(const SumParams& p, int D, hipStream_t st);

constexpr int64_t kMostBlocks = 0x7fffffff;
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int TILE_ROWS = 128;   // rows (or keys) of a workgroup of the tile kernels: four waves of 32
constexpr int CUS = 256;

// The tile kernels: with fewer workgroups than CUs the run of tiles that each goes through is divided, into shares of at least two
// tiles, as long as there is a CU for each share.  Two for every CU, forward and backward in us: 4 x 8 x 500 rows over up to 2048 keys
// at D = 256 264 -> 274 (173 -> 190 since), 2 x 16 x 300 over 4000, 4 key heads, D = 128 126 -> 134.
struct Shares {
  int splits, share;
};
inline Shares tile_shares(int64_t workgroups, int64_t tiles) {
  if (workgroups > CUS / 2 || workgroups == 0 || tiles < 4) return {1, 1};
  const int share = (int)std::max<int64_t>(2, ceil_div(tiles, CUS / workgroups));
  return {(int)ceil_div(tiles, share), share};
}

// Few tiles to a pair: tile by tile.
inline bool tiles_first(int64_t tiles) { return tiles <= 4; }

// The rows kernel serves up to 32 rows of a key head.  Its keys are divided into shares whose length follows from the longest that the call may hold,
// not from the number of workgroups: a sequence has the same bits alone and in any batch.  In us, shares of 16 tiles of 32 keys -> of 32:
// 8 sequences of up to 4096, 8 key heads, D = 128 24.9 -> 32.4; 64 of 2048 106 -> 101; 64 of up to 8192 112 -> 109.  At most 64 shares.
inline bool few_rows(int64_t rows) { return rows <= 32; }
inline int rows_share(int64_t tiles) { return (int)std::max<int64_t>(tiles <= 128 ? 16 : 32, ceil_div(tiles, 64)); }

}  // namespace kv
