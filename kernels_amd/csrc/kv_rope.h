// What comes before attention: norms of queries and keys for each head, the rotation of their channels by position, and both on the way
// into a cache in pages.
//
// A row is one token of one head, x of D channels.  y = x r w with r = 1 / sqrt(mean(x^2) + eps) and the weights w (r = w = 1 without norms);
// the first `rot` channels of y go in pairs (a, b), which are turned by the angle of the token's position: (a c - b s, b c + a s).  Backward,
// with g turned back by the angle (h = g w): dx = r (h - x r mean(h x r)) and dw = the sum over rows of g x r.
//
// Bound by memory: every row is read once and written once (twice read, the gradient and x, in the backward).  Two chunks of sixteen
// bytes to a lane, so that both sides of a pair are a lane's own, whether pairs are neighbours or halves; what lies past `rot`
// goes in two halves likewise.  The lanes of a row add up its squares among themselves.  A group of lanes keeps its token and goes
// through heads, so that cosines, sines (64 bytes of float32 to 32 of x) and weights are fetched once for several rows; one row at a time: two or four
// on their way together cost registers, and with them waves (2 x 40 heads x 8192, D = 128, forward and backward 163 us; with two and one rows 185, four and two 190,
// eight and four 209, before stores past the caches).  2 x 40 x 8192, D = 128, bfloat16: forward 336 MB read and written in 65-71 us, 4.7-5.2 TB/s.
#pragma once
#include "kv_common.h"

namespace kv {

// How D channels lie over lanes; 256 threads work on GROUPS tokens.
template <typename T, int D> struct RopeLanes {
  static constexpr int V = Elem<T>::VEC, LANES = D / (2 * V), GROUPS = 256 / LANES;
};

struct RopeSide {          // q or k
  const void *x, *g;       // g: the gradient of the turned rows (backward)
  void* out;               // contiguous [B, heads, T, D]: the turned rows, or the gradient of x
  const void* weight;      // [D] or null
  int64_t sb, sh, st, g_sb, g_sh, g_st;
  int heads;
};
struct RopeTable {
  const float *cos, *sin;  // [rows, rot / 2]
  int64_t cos_st, sin_st;
  int rows, rot;
};
struct RopeParams {
  RopeSide q, k;
  RopeTable table;
  const int32_t *lens, *positions;   // or null: all of T, and 0, 1, ...
  int64_t lens_stride, pos_sb, pos_st;
  int B, T;
  float eps;               // 0: no norms
  bool weights_f32;
  int chunk, q_chunks;     // heads that a workgroup goes through; layers of the grid that are q's
  ChunkDiv by_tokens;
  float* part;             // backward: [layers, gridDim.x, D] sums of dw, or null
};

// A lane's two chunks of V elements.  Both sides of a pair are a lane's own; and the first chunks of a row's lanes follow each other, as do the second
// ones, so that a store covers half of a row (halves, some of the channels turned: the halves of those and the halves of the others.  With chunks of the others side by side
// in a lane prompts of up to 2048 tokens of 8 sequences into pages, whose values are not turned, took 66.8 us instead of 63.8).
template <typename T, int D, bool INTER> struct RopeLane {
  static constexpr int V = RopeLanes<T, D>::V;
  int a, b;
  bool a_turned, b_turned;
  SA_DEV RopeLane(int lane, int rot) {
    if constexpr (INTER) {
      a = V * lane, b = D / 2 + V * lane;
      a_turned = a < rot, b_turned = b < rot;
    } else {
      a_turned = b_turned = 2 * V * lane < rot;
      a = a_turned ? V * lane : rot / 2 + V * lane;
      b = a_turned ? rot / 2 + V * lane : D / 2 + V * lane;
    }
  }
};
template <typename T> SA_DEV void unpack(float* x, const T* from) {
  const auto f = *reinterpret_cast<const typename Elem<T>::Frag*>(from);
#pragma unroll
  for (int e = 0; e < Elem<T>::VEC; ++e) x[e] = (float)f[e];
}
template <typename T> SA_DEV u32x4 packed(const float* x) {
  typename Elem<T>::Frag f;
#pragma unroll
  for (int e = 0; e < Elem<T>::VEC; ++e) f[e] = (T)x[e];
  return __builtin_bit_cast(u32x4, f);
}
template <int N> SA_DEV void load_floats(float* x, const float* from) {
  typedef float Part __attribute__((ext_vector_type(N < 4 ? N : 4)));
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const Part f = *reinterpret_cast<const Part*>(from + e);
#pragma unroll
    for (int i = 0; i < (N < 4 ? N : 4); ++i) x[e + i] = f[i];
  }
}
// The weights of a lane's channels, in their type or in float32.
template <typename T, int V> SA_DEV void load_weights(float (&w)[2 * V], const void* weight, bool f32, int a, int b) {
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) w[e] = 1.0f;
  if (!weight) return;
  if (f32) {
    const float* p = reinterpret_cast<const float*>(weight);
    load_floats<V>(w, p + a);
    load_floats<V>(w + V, p + b);
  } else {
    unpack<T>(w, reinterpret_cast<const T*>(weight) + a);
    unpack<T>(w + V, reinterpret_cast<const T*>(weight) + b);
  }
}
// The sum over the LANES lanes of a row, in all of them.
template <int LANES> SA_DEV float row_sum(float x) {
  auto add = [&](auto ctrl) { x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, false)); };
  if constexpr (LANES >= 2) add(std::integral_constant<int, 0xB1>{});    // the neighbour
  if constexpr (LANES >= 4) add(std::integral_constant<int, 0x4E>{});    // the other pair of four
  if constexpr (LANES >= 8) add(std::integral_constant<int, 0x141>{});   // eight, mirrored
  if constexpr (LANES >= 16) add(std::integral_constant<int, 0x140>{});  // sixteen, mirrored
  if constexpr (LANES >= 32) x += __shfl_xor(x, 16);
  return x;
}
// The pairs of a lane: elements 2 e and 2 e + 1 of its two chunks (INTER), or e of each.
template <bool INTER, int V> SA_DEV void turn(float (&x)[2 * V], const float (&c)[V], const float (&s)[V], bool a_turned, bool b_turned) {
  auto pairs = [&](int first, int last) {
#pragma unroll
    for (int e = first; e < last; ++e) {
      const int i = INTER ? 2 * e : e, j = INTER ? 2 * e + 1 : V + e;
      const float a = x[i], b = x[j];
      x[i] = a * c[e] - b * s[e];
      x[j] = b * c[e] + a * s[e];
    }
  };
  if constexpr (INTER) {
    if (a_turned) pairs(0, V / 2);
    if (b_turned) pairs(V / 2, V);
  } else if (a_turned) {
    pairs(0, V);
  }
}
// x -> the turned row
template <int D, int LANES, bool INTER, int V, typename Lane>
SA_DEV void norm_and_turn(float (&x)[2 * V], const float (&w)[2 * V], const float (&c)[V], const float (&s)[V], const Lane& lane, float eps) {
  if (eps > 0.0f) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) sum += x[e] * x[e];
    const float r = rsqrtf(row_sum<LANES>(sum) * (1.0f / D) + eps);
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) x[e] *= r * w[e];
  }
  turn<INTER>(x, c, s, lane.a_turned, lane.b_turned);
}

// The token of a group of lanes: where it is, and the row of the table.
struct RopeToken {
  int b, t, at;
  bool live;               // not padding, and at a position that the table has
};
// (tokens behind the last one: not live, in place of the last)
SA_DEV RopeToken rope_token(const RopeParams& p, int64_t id, int64_t tokens) {
  RopeToken x;
  const int token = (int)(id < tokens ? id : tokens - 1);
  x.b = div_by(token, p.by_tokens), x.t = token - x.b * p.T;
  x.at = p.positions ? p.positions[x.b * p.pos_sb + x.t * p.pos_st] : x.t;
  x.live = id < tokens && x.t < clamped_length(p.lens, p.lens_stride, x.b, p.T) && (uint32_t)x.at < (uint32_t)p.table.rows;
  return x;
}
template <bool INTER, int V, typename Lane> SA_DEV void load_angles(float (&c)[V], float (&s)[V], const RopeTable& table, int at, const Lane& lane) {
  const float *cos = table.cos + at * table.cos_st, *sin = table.sin + at * table.sin_st;
  if constexpr (INTER) {
    if (lane.a_turned) load_floats<V / 2>(c, cos + lane.a / 2), load_floats<V / 2>(s, sin + lane.a / 2);
    if (lane.b_turned) load_floats<V / 2>(c + V / 2, cos + lane.b / 2), load_floats<V / 2>(s + V / 2, sin + lane.b / 2);
  } else if (lane.a_turned) {
    load_floats<V>(c, cos + lane.a);
    load_floats<V>(s, sin + lane.a);
  }
}

// Where a lane's two chunks of a row go.  Rows of 128 bytes: the groups of lanes of two tokens that follow each other exchange a chunk (in the order of
// lanes that the half mirror gives), so that each store covers whole rows.  In us, with a half of a row to a store -> whole rows -> past the caches, D = 64, 16 bits: 4 x
// 32 heads x 8192 forward 66 -> 60 -> 58, 8 x 24 x 1500-3000 38 -> 34.5 -> 25.5; with gradients 8 x 32 x 4096 150 -> 126, prompts of up to 2048 tokens of 8 sequences into pages 46 -> 27.
// Likewise the halves of a row of 256 bytes of which half is turned, in calls that store past the caches: D = 128, 2 x 40 x 8192 forward 81 -> 71, with gradients 191 -> 163, prompts into
// pages 77 -> 64 (64 bytes to a store and plain -> whole lines past the caches).
template <typename T, int D, bool INTER, bool STREAMING> struct RowStore {
  using L = RopeLanes<T, D>;
  static constexpr bool PAIRS = L::LANES == 4, HALVES = L::LANES == 8 && !INTER && STREAMING;
  // The tokens from here on that the loop of a group has to take part in: both of a pair, or its own.
  SA_DEV static int64_t leader(int64_t id) { return PAIRS ? id & ~int64_t(1) : id; }
  T *first, *second;
  bool has_first, has_second, exchanged = PAIRS, odd = false;
  SA_DEV static int other(int x) { return __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, false); }
  // to: this group's row; there: it is to be written
  SA_DEV RowStore(T* to, bool there, int64_t id, int rot, const RopeLane<T, D, INTER>& lane) {
    if constexpr (PAIRS) {
      const RopeLane<T, D, INTER> mirrored(L::LANES - 1 - threadIdx.x % L::LANES, rot);
      const uint64_t own = reinterpret_cast<uint64_t>(to);
      T* const others = reinterpret_cast<T*>((uint64_t)(uint32_t)other((int)(own >> 32)) << 32 | (uint32_t)other((int)own));
      const bool others_there = other(there ? 1 : 0) != 0;
      odd = id & 1;
      first = odd ? others + mirrored.b : to + lane.a;
      second = odd ? to + lane.b : others + mirrored.a;
      has_first = odd ? others_there : there;
      has_second = odd ? there : others_there;
    } else {
      first = to + lane.a, second = to + lane.b;
      has_first = has_second = there;
      if constexpr (HALVES) {
        exchanged = 2 * rot == D, odd = threadIdx.x & 4;
        const RopeLane<T, D, INTER> mirrored(L::LANES - 1 - threadIdx.x % L::LANES, rot);
        if (exchanged) first = to + (odd ? mirrored.b : lane.a), second = to + (odd ? lane.b : mirrored.a);
      }
    }
  }
  SA_DEV static void store(T* to, const u32x4& v) {
    if constexpr (STREAMING) sa::store_streaming(to, v);
    else *reinterpret_cast<u32x4*>(to) = v;
  }
  SA_DEV void put(const float* x) const {
    if constexpr (PAIRS || HALVES) {
      put(packed<T>(x), packed<T>(x + L::V));
    } else if (has_first) {
      store(first, packed<T>(x));
      store(second, packed<T>(x + L::V));
    }
  }
  // The two chunks as bytes.
  SA_DEV void put(u32x4 one, u32x4 two) const {
    if constexpr (PAIRS || HALVES) {
      if (exchanged)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t got = (uint32_t)other((int)(odd ? one[e] : two[e]));
          one[e] = odd ? got : one[e], two[e] = odd ? two[e] : got;
        }
      if (has_first) store(first, one);
      if (has_second) store(second, two);
    } else if (has_first) {
      store(first, one);
      store(second, two);
    }
  }
  SA_DEV void next(int64_t step) { first += step, second += step; }
};

// (five waves to a SIMD: up to 96 registers, which come in eights, and none spills)
template <typename T, int D, bool INTER, bool STREAMING> __global__ __launch_bounds__(256, 5) void rope_kernel(const RopeParams p) {
  using L = RopeLanes<T, D>;
  constexpr int V = L::V;
  const RopeLane<T, D, INTER> lane(threadIdx.x % L::LANES, p.table.rot);
  const bool keys = (int)blockIdx.y >= p.q_chunks;
  const RopeSide& side = keys ? p.k : p.q;
  const int h0 = ((int)blockIdx.y - (keys ? p.q_chunks : 0)) * p.chunk, h1 = h0 + p.chunk < side.heads ? h0 + p.chunk : side.heads;
  const int64_t step = (int64_t)gridDim.x * L::GROUPS, tokens = (int64_t)p.B * p.T;
  float w[2 * V];
  load_weights<T, V>(w, side.weight, p.weights_f32, lane.a, lane.b);
  for (int64_t id = (int64_t)blockIdx.x * L::GROUPS + threadIdx.x / L::LANES; RowStore<T, D, INTER, STREAMING>::leader(id) < tokens; id += step) {
    const RopeToken token = rope_token(p, id, tokens);
    const T* x = reinterpret_cast<const T*>(side.x) + token.b * side.sb + token.t * side.st + h0 * side.sh;
    RowStore<T, D, INTER, STREAMING> to(reinterpret_cast<T*>(side.out) + (((int64_t)token.b * side.heads + h0) * p.T + token.t) * D, id < tokens, id, p.table.rot, lane);
    float c[V], s[V], row[2 * V];
    if (token.live) load_angles<INTER>(c, s, p.table, token.at, lane);
    for (int h = h0; h < h1; ++h, x += side.sh, to.next((int64_t)p.T * D)) {
      if (token.live) {
        unpack<T>(row, x + lane.a);
        unpack<T>(row + V, x + lane.b);
        norm_and_turn<D, L::LANES, INTER, V>(row, w, c, s, lane, p.eps);
      } else {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) row[e] = 0.0f;
      }
      to.put(row);
    }
  }
}

// Gradients of x, and in p.part each workgroup's sums of those of the weights, in the order of its tokens and then of its groups of lanes.
template <typename T, int D, bool INTER, bool STREAMING> __global__ __launch_bounds__(256) void rope_backward_kernel(const RopeParams p) {
  using L = RopeLanes<T, D>;
  constexpr int V = L::V;
  __shared__ __attribute__((aligned(16))) float sums[L::GROUPS * D];
  const RopeLane<T, D, INTER> lane(threadIdx.x % L::LANES, p.table.rot);
  const bool keys = (int)blockIdx.y >= p.q_chunks, norm = p.eps > 0.0f;
  const RopeSide& side = keys ? p.k : p.q;
  const int h0 = ((int)blockIdx.y - (keys ? p.q_chunks : 0)) * p.chunk, h1 = h0 + p.chunk < side.heads ? h0 + p.chunk : side.heads;
  const int64_t step = (int64_t)gridDim.x * L::GROUPS, tokens = (int64_t)p.B * p.T;
  float w[2 * V], dw[2 * V];
  load_weights<T, V>(w, side.weight, p.weights_f32, lane.a, lane.b);
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) dw[e] = 0.0f;
  for (int64_t id = (int64_t)blockIdx.x * L::GROUPS + threadIdx.x / L::LANES; RowStore<T, D, INTER, STREAMING>::leader(id) < tokens; id += step) {
    const RopeToken token = rope_token(p, id, tokens);
    const T* x = reinterpret_cast<const T*>(side.x) + token.b * side.sb + token.t * side.st + h0 * side.sh;
    const T* g = reinterpret_cast<const T*>(side.g) + token.b * side.g_sb + token.t * side.g_st + h0 * side.g_sh;
    RowStore<T, D, INTER, STREAMING> to(reinterpret_cast<T*>(side.out) + (((int64_t)token.b * side.heads + h0) * p.T + token.t) * D, id < tokens, id, p.table.rot, lane);
    float c[V], s[V], xs[2 * V], gs[2 * V];
    if (token.live) {
      load_angles<INTER>(c, s, p.table, token.at, lane);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] = -s[e];
    }
    for (int h = h0; h < h1; ++h, x += side.sh, g += side.g_sh, to.next((int64_t)p.T * D)) {
      if (token.live) {
        unpack<T>(gs, g + lane.a);
        unpack<T>(gs + V, g + lane.b);
        if (norm) {
          unpack<T>(xs, x + lane.a);
          unpack<T>(xs + V, x + lane.b);
        }
        turn<INTER>(gs, c, s, lane.a_turned, lane.b_turned);
        if (norm) {
          float squares = 0.0f, dot = 0.0f;
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) squares += xs[e] * xs[e];
          const float r = rsqrtf(row_sum<L::LANES>(squares) * (1.0f / D) + p.eps);
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) {
            xs[e] *= r;
            dw[e] += gs[e] * xs[e];
            gs[e] *= w[e];
            dot += gs[e] * xs[e];
          }
          const float mean = row_sum<L::LANES>(dot) * (1.0f / D);
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) gs[e] = r * (gs[e] - xs[e] * mean);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) gs[e] = 0.0f;
      }
      to.put(gs);
    }
  }
  if (!p.part) return;
  float* const own = sums + threadIdx.x / L::LANES * D;
#pragma unroll
  for (int e = 0; e < V; ++e) own[lane.a + e] = dw[e], own[lane.b + e] = dw[V + e];
  __syncthreads();
  if (threadIdx.x < D) {
    float sum = 0.0f;
    for (int i = 0; i < L::GROUPS; ++i) sum += sums[i * D + threadIdx.x];
    p.part[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * D + threadIdx.x] = sum;
  }
}

// The workgroups' sums, added up: sixteen channels of q's weights or k's to a workgroup.
struct RopeSumParams {
  const float* part;
  void *dq, *dk;           // [D] or null
  int q_parts, k_parts, D;
  bool f32;
};
template <typename T> __global__ __launch_bounds__(256) void rope_sum_kernel(const RopeSumParams p) {
  __shared__ __attribute__((aligned(16))) f32x4 sums[256];
  const bool keys = blockIdx.y == 1;
  void* const out = keys ? p.dk : p.dq;
  if (!out) return;
  const int n = keys ? p.k_parts : p.q_parts, d = (int)blockIdx.x * 16 + threadIdx.x % 4 * 4;
  const float* part = p.part + (keys ? (int64_t)p.q_parts * p.D : 0) + d;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int i = threadIdx.x / 4; i < n; i += 64) sum += *reinterpret_cast<const f32x4*>(part + (int64_t)i * p.D);
  sums[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x >= 4) return;
  for (int i = 1; i < 64; ++i) sum += sums[i * 4 + threadIdx.x];
  if (p.f32) *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(out) + d) = sum;
  else sa::store4<T>(reinterpret_cast<T*>(out) + d, sum[0], sum[1], sum[2], sum[3]);
}

// ---- into the pages ---------------------------------------------------------------------------------------------------
// Token i of n = new_lens[b] of sequence b goes to position lens[b] - n + i, its angle is that of its entry in `positions`, or of that position.  k is
// turned and v goes as bytes: by way of float32 numbers, signalling NaN of 16 bits would come back quiet; q is turned into a tensor of its own.
struct AppendRopeParams {
  const void *q, *k, *v;
  void *q_out, *k_pages, *v_pages;    // q_out contiguous [B, Hq, T, D]
  const void *q_weight, *k_weight;
  RopeTable table;
  const int32_t *lens, *new_lens, *positions, *page_table;
  int64_t lens_stride, new_lens_stride, pos_sb, pos_st, table_sb;
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  int64_t kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;
  int B, Hq, Hkv, T, width, num_pages, page;
  float eps;
  bool weights_f32;
  int chunk, q_chunks, k_chunks;      // layers of the grid: q's, k's, then v's
  ChunkDiv by_tokens, by_page;
};
// Four waves to a SIMD in 16 bits: told so, the compiler keeps all but 2 to 14 scalar registers (bfloat16, D = 16: 47 to 80) where five waves spill 51 to 81
// (bfloat16, 32 / 8 heads, D = 128, five -> four, us: prompts of up to 2048 tokens of 8 sequences 63-68 -> 62-66, up to 1024 of 2 13.3 -> 11.6).
template <typename T, int D, bool INTER, bool STREAMING>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4, sizeof(T) == 2 ? 4 : 8))) void append_rope_kernel(const AppendRopeParams p) {
  using L = RopeLanes<T, D>;
  constexpr int V = L::V;
  const int layer = blockIdx.y, kind = layer < p.q_chunks ? 0 : layer < p.q_chunks + p.k_chunks ? 1 : 2;
  const RopeLane<T, D, INTER> lane(threadIdx.x % L::LANES, kind == 2 ? 0 : p.table.rot);
  const int heads = kind == 0 ? p.Hq : p.Hkv, h0 = (layer - (kind == 0 ? 0 : kind == 1 ? p.q_chunks : p.q_chunks + p.k_chunks)) * p.chunk;
  const int h1 = h0 + p.chunk < heads ? h0 + p.chunk : heads;
  const T* const from = reinterpret_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v);
  const int64_t sb = kind == 0 ? p.q_sb : kind == 1 ? p.k_sb : p.v_sb, sh = kind == 0 ? p.q_sh : kind == 1 ? p.k_sh : p.v_sh;
  const int64_t st = kind == 0 ? p.q_st : kind == 1 ? p.k_st : p.v_st;
  const int64_t step = (int64_t)gridDim.x * L::GROUPS, tokens = (int64_t)p.B * p.T;
  float w[2 * V];
  load_weights<T, V>(w, kind == 0 ? p.q_weight : kind == 1 ? p.k_weight : nullptr, p.weights_f32, lane.a, lane.b);
  for (int64_t id = (int64_t)blockIdx.x * L::GROUPS + threadIdx.x / L::LANES; RowStore<T, D, INTER, STREAMING>::leader(id) < tokens; id += step) {
    const int token = (int)(id < tokens ? id : tokens - 1), b = div_by(token, p.by_tokens), t = token - b * p.T;
    const int n = clamped_length(p.new_lens, p.new_lens_stride, b, p.T);
    const int64_t place = (int64_t)p.lens[b * p.lens_stride] - n + t;
    const int64_t at = p.positions ? p.positions[b * p.pos_sb + t * p.pos_st] : place;
    const bool live = id < tokens && t < n && at >= 0 && at < p.table.rows;
    T* own = nullptr;
    int64_t own_sh = (int64_t)p.T * D;
    bool there = id < tokens;
    if (kind == 0) {
      own = reinterpret_cast<T*>(p.q_out) + (((int64_t)b * heads + h0) * p.T + t) * D;
    } else {
      own_sh = kind == 1 ? p.kp_sh : p.vp_sh;
      there = live && place >= 0 && place < (int64_t)p.width * p.page;
      if (there) {
        const int entry = div_by((int)place, p.by_page), slot = (int)place - entry * p.page;
        const int32_t page = p.page_table[b * p.table_sb + entry];
        there = (uint32_t)page < (uint32_t)p.num_pages;
        own = (kind == 1 ? reinterpret_cast<T*>(p.k_pages) + page * p.kp_sp + slot * p.kp_st : reinterpret_cast<T*>(p.v_pages) + page * p.vp_sp + slot * p.vp_st) + h0 * own_sh;
      }
      if (!RowStore<T, D, INTER, STREAMING>::PAIRS && !there) continue;
    }
    RowStore<T, D, INTER, STREAMING> to(own, there, id, kind == 2 ? 0 : p.table.rot, lane);
    const T* x = from + b * sb + t * st + h0 * sh;
    float c[V], s[V], row[2 * V];
    if (live && kind != 2) load_angles<INTER>(c, s, p.table, (int)at, lane);
    for (int h = h0; h < h1; ++h, x += sh, to.next(own_sh)) {
      u32x4 one = {0, 0, 0, 0}, two = one;
      if (live && kind == 2) {
        one = *reinterpret_cast<const u32x4*>(x + lane.a), two = *reinterpret_cast<const u32x4*>(x + lane.b);
      } else if (live) {
        unpack<T>(row, x + lane.a);
        unpack<T>(row + V, x + lane.b);
        norm_and_turn<D, L::LANES, INTER, V>(row, w, c, s, lane, p.eps);
        one = packed<T>(row), two = packed<T>(row + V);
      }
      to.put(one, two);   // (one call for both: of stores that it joins the compiler has dropped that they go past the caches)
    }
  }
}

}  // namespace kv
