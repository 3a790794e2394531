// Argument checks of the entry points of libkv_attention.so.
#pragma once
#include <math.h>
#include "../../include/kv_attention.h"
#include "kv_common.h"

namespace kv {

constexpr float kLog2e = 1.4426950408889634f;

inline int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

inline int check_sizes(int B, int Hq, int Hkv, int D, int dtype) {
  if (dtype < 0 || dtype > 2) return KV_ERR_DTYPE;
  if (D != 16 && D != 32 && D != 64 && D != 128 && D != 256) return KV_ERR_HEAD_DIM;
  if (B < 0 || Hq < 0 || Hkv < 0 || (Hkv == 0) != (Hq == 0) || (Hkv > 0 && Hq % Hkv != 0)) return KV_ERR_ARG;
  return KV_OK;
}
// n rows; offsets32: addressed with 32-bit byte offsets from the first one
inline int check_layout(const void* p, const int64_t* s, int dtype, int64_t n, bool offsets32) {
  if (!p || !s) return KV_ERR_ARG;
  const int64_t es = elem_size(dtype), vec = 16 / es;
  if (s[3] != 1 || (reinterpret_cast<uintptr_t>(p) & 15u)) return KV_ERR_LAYOUT;
  for (int i = 0; i < 3; ++i)
    if (s[i] % vec != 0 || s[i] < 0) return KV_ERR_LAYOUT;
  if (s[2] == 0 && n > 1) return KV_ERR_LAYOUT;
  if (offsets32 && s[2] > ((int64_t(1) << 32) - 1) / es / (n + 1024)) return KV_ERR_TOO_LARGE;
  return KV_OK;
}
// Times log2(e) it has to be a number of float32.
inline int check_scale(float sm_scale) { return fabsf(sm_scale) <= 0x1p127f ? KV_OK : KV_ERR_ARG; }
inline int check_out(const void* p) { return !p ? KV_ERR_ARG : (reinterpret_cast<uintptr_t>(p) & 15u) ? KV_ERR_LAYOUT : KV_OK; }

inline int check_workspace(void* workspace, int64_t have, int64_t need) {
  if (need == 0) return KV_OK;
  if (!workspace || have < need) return KV_ERR_WORKSPACE;
  return (reinterpret_cast<uintptr_t>(workspace) & 15u) ? KV_ERR_LAYOUT : KV_OK;
}
template <typename F> inline int by_dtype(int dtype, F&& f) {
  switch (dtype) {
    case 0: return f(float{});
    case 1: return f(_Float16{});
    case 2: return f(__bf16{});
  }
  return KV_ERR_DTYPE;
}

}  // namespace kv
