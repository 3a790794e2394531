// Launches of the kernels of norms and rotation, one explicit instantiation per element type.  Each returns 0, a hipError_t or a KV_ERR_* code.
#pragma once
#include <algorithm>
#include "../../include/kv_attention.h"
#include "kv_rope.h"

namespace kv {

// How the heads and tokens of a call are dealt out: `chunk` heads to a layer of the grid, `blocks` workgroups to a layer.
struct RopeGrid {
  int chunk, q_chunks, k_chunks, blocks;
};
template <typename T> int launch_rope(const RopeParams& p, const RopeGrid& g, int D, bool inter, hipStream_t st);
template <typename T> int launch_rope_backward(const RopeParams& p, const RopeGrid& g, int D, bool inter, hipStream_t st);
template <typename T> int launch_rope_sum(const RopeSumParams& p, hipStream_t st);
template <typename T> int launch_append_rope(const AppendRopeParams& p, const RopeGrid& g, int D, bool inter, hipStream_t st);

constexpr int64_t kMostTokens = 0x7fffffff;   // of all sequences: what the kernels count in 31 bits
inline int64_t rope_tokens_per_block(int D, int elem_size) { return 256 * 32 / (D * elem_size); }   // two chunks of 16 bytes to a lane
inline RopeGrid rope_grid(int64_t tokens, int Hq, int Hkv, int D, int elem_size, int64_t most_blocks) {
  const int64_t groups = (tokens + rope_tokens_per_block(D, elem_size) - 1) / rope_tokens_per_block(D, elem_size);
  RopeGrid g{};
  g.chunk = 8;
  while (g.chunk > 1 && groups * ((Hq + Hkv + g.chunk - 1) / g.chunk) < 2048) g.chunk /= 2;
  g.q_chunks = (Hq + g.chunk - 1) / g.chunk;
  g.k_chunks = (Hkv + g.chunk - 1) / g.chunk;
  g.blocks = (int)std::max<int64_t>(1, std::min(groups, most_blocks / (g.q_chunks + g.k_chunks)));
  return g;
}

}  // namespace kv
