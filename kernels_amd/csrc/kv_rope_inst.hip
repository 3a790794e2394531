// Instantiations of the kernels in kv_rope.h and their launches: one translation unit per element type (KV_DTYPE_ID 0 = float32,
// 1 = float16, 2 = bfloat16).
#include "kv_rope_launch.h"

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

template <typename F> static int by_shape(int D, bool inter, bool streaming, F&& f) {
  auto stores = [&](auto d, auto i) {
    if constexpr (may_go_past_caches(decltype(d)::value * (int)sizeof(ElemT)))
      if (streaming) return f(d, i, std::true_type{});
    return f(d, i, std::false_type{});
  };
  auto pairs = [&](auto d) { return inter ? stores(d, std::true_type{}) : stores(d, std::false_type{}); };
  switch (D) {
    case 16: return pairs(std::integral_constant<int, 16>{});
    case 32: return pairs(std::integral_constant<int, 32>{});
    case 64: return pairs(std::integral_constant<int, 64>{});
    case 128: return pairs(std::integral_constant<int, 128>{});
    case 256: return pairs(std::integral_constant<int, 256>{});
  }
  return KV_ERR_HEAD_DIM;
}

template <> int launch_rope<ElemT>(const RopeParams& p, const RopeGrid& g, int D, bool inter, bool streaming, hipStream_t st) {
  return by_shape(D, inter, streaming, [&](auto d, auto i, auto s) {
    rope_kernel<ElemT, decltype(d)::value, decltype(i)::value, decltype(s)::value>
        <<<dim3(g.blocks, g.q_chunks + g.k_chunks), dim3(256), 0, st>>>(p);
    return (int)hipGetLastError();
  });
}
template <> int launch_rope_backward<ElemT>(const RopeParams& p, const RopeGrid& g, int D, bool inter, bool streaming, hipStream_t st) {
  return by_shape(D, inter, streaming, [&](auto d, auto i, auto s) {
    rope_backward_kernel<ElemT, decltype(d)::value, decltype(i)::value, decltype(s)::value>
        <<<dim3(g.blocks, g.q_chunks + g.k_chunks), dim3(256), 0, st>>>(p);
    return (int)hipGetLastError();
  });
}
template <> int launch_rope_sum<ElemT>(const RopeSumParams& p, hipStream_t st) {
  rope_sum_kernel<ElemT><<<dim3(p.D / 16, 2), dim3(256), 0, st>>>(p);
  return (int)hipGetLastError();
}
template <> int launch_append_rope<ElemT>(const AppendRopeParams& p, const RopeGrid& g, int D, bool inter, bool streaming, hipStream_t st) {
  return by_shape(D, inter, streaming, [&](auto d, auto i, auto s) {
    append_rope_kernel<ElemT, decltype(d)::value, decltype(i)::value, decltype(s)::value>
        <<<dim3(g.blocks, g.q_chunks + 2 * g.k_chunks), dim3(256), 0, st>>>(p);
    return (int)hipGetLastError();
  });
}

}  // namespace kv
