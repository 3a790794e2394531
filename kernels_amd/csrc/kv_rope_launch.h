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
template <typename T> int launch_rope(const RopeParams& p, const RopeGrid& g, int D, bool inter, bool streaming, hipStream_t st);
template <typename T> int launch_rope_backward(const RopeParams& p, const RopeGrid& g, int D, bool inter, bool streaming, hipStream_t st);
template <typename T> int launch_rope_sum(const RopeSumParams& p, hipStream_t st);
template <typename T> int launch_append_rope(const AppendRopeParams& p, const RopeGrid& g, int D, bool inter, bool streaming, hipStream_t st);

constexpr int64_t kMostTokens = 0x7fffffff;   // of all sequences: what the kernels count in 31 bits
inline int64_t rope_tokens_per_block(int D, int elem_size) { return 256 * 32 / (D * elem_size); }   // two chunks of 16 bytes to a lane
// A workgroup goes through up to eight heads, fewer where that leaves fewer than `split` workgroups, and a layer has at most most_blocks / layers of them, which go
// through the tokens.  The backward splits down to 512 and keeps to 1024, whose sums it adds up (forward and backward captured, us, split to 2048 ->
// 512: 2 x 20 heads x 1024, D = 128 21.5 -> 19.1; 32 x 24 x 200, D = 64 30.0 -> 26.4; at most 2048 -> 1024: 2 x 40 x 8192, D = 128 167 -> 163).
inline RopeGrid rope_grid(int64_t tokens, int Hq, int Hkv, int D, int elem_size, int64_t split, int64_t most_blocks) {
  const int64_t groups = (tokens + rope_tokens_per_block(D, elem_size) - 1) / rope_tokens_per_block(D, elem_size);
  RopeGrid g{};
  g.chunk = 8;
  while (g.chunk > 1 && groups * ((Hq + Hkv + g.chunk - 1) / g.chunk) < split) g.chunk /= 2;
  g.q_chunks = (Hq + g.chunk - 1) / g.chunk;
  g.k_chunks = (Hkv + g.chunk - 1) / g.chunk;
  g.blocks = (int)std::max<int64_t>(1, std::min(groups, most_blocks / std::max(1, g.q_chunks + g.k_chunks)));
  return g;
}
inline RopeGrid forward_grid(int64_t tokens, int Hq, int Hkv, int D, int elem_size) { return rope_grid(tokens, Hq, Hkv, D, elem_size, 2048, 1 << 22); }
inline RopeGrid backward_grid(int64_t tokens, int Hq, int Hkv, int D, int elem_size) { return rope_grid(tokens, Hq, Hkv, D, elem_size, 512, 1024); }

// Stores past the caches, where a call reads and writes more than the L2s of all XCDs hold and each store covers whole lines of 128 bytes: rows of 128 (RowStore), halves of longer
// rows; halves as pairs, some of the channels turned: half of those and half of the others, or a row of 256 bytes half of which is turned (RowStore).  In us, plain -> past the caches,
// bfloat16: 2 x 40 heads x 8192, D = 128, forward 76 -> 71, with gradients 189 -> 163; 2 x 2048 of them 20.9 -> 16.5; prompts of up to 2048 tokens of 8 sequences into pages
// 72 -> 65; half of the channels turned, 2 x 40 x 4096, D = 256 forward 78 -> 74, with gradients 187 -> 167, into pages 77 -> 74, float32, D = 128 182 -> 160; with stores of parts
// of lines, D = 128, a quarter turned 152 -> 174, three quarters forward 82 -> 105.
inline bool past_caches(int64_t rows, int D, int rot, bool inter, int elem_size) {
  const bool lines = inter ? D * elem_size % 256 == 0 : rot * elem_size % 256 == 0 && (D - rot) * elem_size % 256 == 0;
  return (lines || D * elem_size == 128 || (D * elem_size == 256 && 2 * rot == D)) && 2 * rows * D * elem_size > (int64_t(32) << 20);
}
constexpr bool may_go_past_caches(int row_bytes) { return row_bytes >= 128; }   // the kernels that there are: never so for shorter rows

}  // namespace kv
