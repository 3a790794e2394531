// Instantiations of the kernels in kv_*.h and their launches: one translation unit per element type (KV_DTYPE_ID 0 = float32, 1 = float16,
// 2 = bfloat16), kind (KV_KIND) and group of head dimensions (KV_DGROUP 0 = 16 to 128, 1 = 256).
#include <mutex>
#include "kv_launch.h"

namespace kv {

#if KV_DTYPE_ID == 0
using ElemT = float;
#elif KV_DTYPE_ID == 1
using ElemT = _Float16;
#elif KV_DTYPE_ID == 2
using ElemT = __bf16;
#else
#error "KV_DTYPE_ID must be 0, 1 or 2"
#endif

// A kernel with more than 64 KiB of LDS needs the limit raised once per kernel and device.
struct LdsLimit {
  static constexpr int kMaxDevices = 64;
  std::mutex mu;
  bool done[kMaxDevices] = {};
};
template <typename K> static int raise_lds(K kernel, size_t bytes, LdsLimit& state) {
  if (bytes <= 65536) return KV_OK;
  auto set = [&] { return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes); };
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return (int)e;
  if (dev < 0 || dev >= LdsLimit::kMaxDevices) return set();
  std::lock_guard<std::mutex> lock(state.mu);
  if (state.done[dev]) return KV_OK;
  const int rc = set();
  state.done[dev] = rc == 0;
  return rc;
}
template <typename K, typename P>
static int launch(K kernel, int64_t blocks, int threads, size_t lds, LdsLimit& state, const P& p, hipStream_t st, int layers = 1) {
  if (!launchable(blocks, threads)) return KV_ERR_TOO_LARGE;   // (the host has refused it before the first launch of a call)
  if (blocks == 0) return KV_OK;
  if (int rc = raise_lds(kernel, lds, state)) return rc;
  kernel<<<dim3((unsigned)blocks, layers), dim3(threads), lds, st>>>(p);
  return (int)hipGetLastError();
}
template <typename F> static int by_head_dim(int D, F&& f) {
#if KV_DGROUP == 0
  switch (D) {
    case 16: return f(std::integral_constant<int, 16>{});
    case 32: return f(std::integral_constant<int, 32>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
  }
#else
  if (D == 256) return f(std::integral_constant<int, 256>{});
#endif
  return KV_ERR_HEAD_DIM;
}
// LDS of a kernel with two stages, over which the waves' row patches lie at the end
template <typename T, int D> constexpr size_t with_patches(size_t stages, int waves) {
  const size_t patches = sizeof(T) == 2 ? (size_t)waves * 32 * (D + 8) * 2 : 0;
  return stages > patches ? stages : patches;
}

#if KV_KIND == 0
template <> int launch_cross_fwd<ElemT, KV_DGROUP>(const FwdParams& p, int D, hipStream_t st) {
  return by_head_dim(D, [&](auto d) {
    constexpr int DD = decltype(d)::value;
    static LdsLimit state;
    const size_t lds = with_patches<ElemT, DD>(2 * 2 * fwd_tile<ElemT, DD>() * DD * sizeof(ElemT), 4);
    return launch(cross_fwd_kernel<ElemT, DD, 4>, (int64_t)p.work.map.nbh * p.work.map.n_tiles, 256, lds, state, p, st);
  });
}
#elif KV_KIND == 1
template <> int launch_cross_dq<ElemT, KV_DGROUP>(const BwdParams& p, int D, hipStream_t st) {
  return by_head_dim(D, [&](auto d) {
    constexpr int DD = decltype(d)::value;
    static LdsLimit state;
    const size_t lds = with_patches<ElemT, DD>(2 * 2 * dq_tile<ElemT, DD>() * DD * sizeof(ElemT), 4);
    return launch(cross_dq_kernel<ElemT, DD, 4>, (int64_t)p.work.map.nbh * p.work.map.n_tiles, 256, lds, state, p, st);
  });
}
#elif KV_KIND == 2
template <int D, int PASS> static int launch_dkdv_pass(const BwdParams& p, hipStream_t st) {
  static LdsLimit state;
  const size_t lds = with_patches<ElemT, D>(2 * dkdv_stage<ElemT, D>(), 4);
  return launch(cross_dkdv_kernel<ElemT, D, 4, PASS>, (int64_t)p.work.map.nbh * p.work.map.n_tiles, 256, lds, state, p, st);
}
template <> int launch_cross_dkdv<ElemT, KV_DGROUP>(const BwdParams& p, int D, hipStream_t st) {
  return by_head_dim(D, [&](auto d) {
    constexpr int DD = decltype(d)::value;
    if constexpr (sizeof(ElemT) == 2 && DD == 256) {
      static LdsLimit state;
      return launch(cross_dkdv_wide_kernel<ElemT, DD>, (int64_t)p.work.map.nbh * p.work.map.n_tiles, 512, sa::DkdvSplitWide<ElemT, DD>::lds, state, p, st);
    } else if constexpr (DD == 256) {
      if (int rc = launch_dkdv_pass<DD, 1>(p, st)) return rc;
      return launch_dkdv_pass<DD, 2>(p, st);
    } else {
      return launch_dkdv_pass<DD, 0>(p, st);
    }
  });
}
#elif KV_KIND == 3
template <int D, int NW, bool PAGED> static int launch_rows_shape(const RowsParams& p, int64_t blocks, hipStream_t st) {
  constexpr int row_bytes = D * (int)sizeof(ElemT), lds = RowsShape<ElemT, D, NW>::bytes(PAGED), places = CUS * (163840 / lds);
  // by length where there are many workgroups: only the waves that many workgroups have
  if constexpr (row_bytes >= 128 && NW == rows_waves(row_bytes, sizeof(ElemT) == 4, 2 * CUS, 1)) {
    static_assert(2 * places >= 2 * CUS, "many in the sense of rows_waves");
    static LdsLimit state;
    if (p.splits > 1 && by_length(p.B, p.row_tiles, row_bytes) && blocks >= 2 * places)
      return launch(rows_by_length_kernel<ElemT, D, NW, PAGED>, places, NW * 64, lds, state, p, st);
  }
  static LdsLimit state;
  return launch(rows_kernel<ElemT, D, NW, PAGED>, blocks, NW * 64, lds, state, p, st);
}
template <bool PAGED> static int launch_rows_any(const RowsParams& p, int D, hipStream_t st) {
  return by_head_dim(D, [&](auto d) {
    constexpr int DD = decltype(d)::value, ROW = DD * (int)sizeof(ElemT);
    const int64_t blocks = (int64_t)p.B * p.map.Hkv * p.row_tiles * p.splits;
    const int waves = rows_waves(ROW, sizeof(ElemT) == 4, blocks, p.share);
    if constexpr (ROW == 128)
      if (waves == 8) return launch_rows_shape<DD, 8, PAGED>(p, blocks, st);
    if constexpr (ROW == 256 && sizeof(ElemT) == 2)
      if (waves == 2) return launch_rows_shape<DD, 2, PAGED>(p, blocks, st);
    return launch_rows_shape<DD, ROW <= 256 ? 4 : ROW == 512 ? 2 : 1, PAGED>(p, blocks, st);
  });
}
template <> int launch_rows<ElemT, KV_DGROUP>(const RowsParams& p, int D, hipStream_t st) { return launch_rows_any<false>(p, D, st); }
template <> int launch_rows_paged<ElemT, KV_DGROUP>(const RowsParams& p, int D, hipStream_t st) { return launch_rows_any<true>(p, D, st); }
template <> int launch_join<ElemT, KV_DGROUP>(const JoinParams& p, int D, hipStream_t st) {
  return by_head_dim(D, [&](auto d) {
    constexpr int DD = decltype(d)::value;
    static LdsLimit none;
    const int64_t rows = (int64_t)p.B * p.map.Hkv * p.map.rows();
    if (p.splits <= 8) return launch(join_kernel<ElemT, DD, 1>, ceil_div(rows, 256 / (DD / 4)), 256, 0, none, p, st);
    constexpr int NT = 8 * DD / 4 > 256 ? 8 * DD / 4 : 256;
    return launch(join_kernel<ElemT, DD, 8>, ceil_div(rows, NT / (8 * DD / 4)), NT, 0, none, p, st);
  });
}
template <> int launch_sum<ElemT, KV_DGROUP>(const SumParams& p, int D, hipStream_t st) {
  return by_head_dim(D, [&](auto d) {
    constexpr int DD = decltype(d)::value;
    static LdsLimit none;
    const bool queries = p.first_keys > 0, keys = p.keys.part != nullptr;
    const int64_t rows = std::max<int64_t>(queries ? p.queries.map.rows() : 0, keys ? p.keys.map.rows() : 0);
    return launch(sum_kernel<ElemT, DD>, ceil_div((int64_t)p.B * p.Hkv * rows, 256 / (DD / 4)), 256, 0, none, p, st, queries + 2 * keys);
  });
}
#elif KV_KIND == 4 && !defined(SA_NO_ASM_KERNELS)
constexpr size_t long_stages(int n, size_t tile_rows) { return n * 2 * tile_rows * 128 * sizeof(ElemT); }
static int64_t long_blocks(const sa::TileMap& m) { return (int64_t)m.nbh * m.n_tiles; }
template <> int launch_long_fwd<ElemT>(const LongFwd& p, hipStream_t st) {
  static LdsLimit state;
  return launch(sa::fwd3_kernel<ElemT, 128, 4, LongFwd>, long_blocks(p.tiles), 256, long_stages(4, 64), state, p, st);
}
template <> int launch_long_dq<ElemT>(const LongBwd& p, hipStream_t st) {
  static LdsLimit state;   // (a fifth stage for half of the dO rows)
  return launch(sa::dq3_kernel<ElemT, 128, 4, LongBwd>, long_blocks(p.tiles), 256, long_stages(5, 64), state, p, st);
}
template <> int launch_long_dkdv<ElemT>(const LongBwd& p, hipStream_t st) {
  static LdsLimit state;   // three stages with lse and delta, and the workgroup's V rows
  const size_t lds = long_stages(3, 64) + 3 * 2 * 64 * sizeof(float) + 128 * 128 * sizeof(ElemT);
  return launch(sa::dkdv3_kernel<ElemT, 128, 3, LongBwd>, long_blocks(p.tiles), 256, lds, state, p, st);
}
#endif

}  // namespace kv
