// Tree attention: arguments, the cut of the work into pieces, and the paths of the nodes,
// shared by the mma.sync kernel (few rows) and the tcgen05 kernel (many).
#pragma once

#include "paged.cuh"

namespace iron {

constexpr int kTMaxBatch = 1024;
constexpr int kTMaxNodes = 128;

struct TreeArgs {
  const uint16_t *q, *k_new, *v_new, *k, *v;
  const int *table, *lens, *parents;
  uint16_t *out;
  float *ws;         // partials: what a piece of the work leaves of a unit that it holds in part
  unsigned *counts;  // pieces of a unit that are done (0 between calls)
  int64_t qs[3], ks[3], os[3];  // element strides {batch, node, head}
  int B, N, Hq, Hkv, groups /* row groups per (sequence, kv head) */, page_shift, M, P;
  float scale_log2;
  unsigned wait_us;  // how long the loads of the tcgen05 form wait for room
};

__device__ __forceinline__ int cached_len(const TreeArgs &a, int b) {
  return min(max(ld_act_i32(a.lens + b), 0), a.M << a.page_shift);
}

// Tiles of a sequence: its cached tokens, then its nodes.
template <class T>
__device__ __forceinline__ int tile_count(const TreeArgs &a, int b) {
  return (cached_len(a, b) + T::kTile - 1) / T::kTile + (a.N + T::kTile - 1) / T::kTile;
}

// A unit = (sequence, kv head, row group) costs its tiles and T::kUnitCost more, for what is
// done once per unit (Q, paths, output); the work is cut into pieces of equal cost.
// Exclusive prefix sum over the sequences of one unit's cost into pref[0 .. B].
template <class T, int kThreads>
__device__ __forceinline__ void cost_prefix(const TreeArgs &a, int *pref, int *warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int v = b < a.B ? tile_count<T>(a, b) + T::kUnitCost : 0;
    const int mine = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += warp_sums[w];
      total += warp_sums[w];
    }
    if (b < a.B) pref[b] = base + before + v - mine;
    base += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) pref[a.B] = base;
  __syncthreads();
}

// `total` cost cut into `pieces` equal parts (none empty): where part c starts, and the
// part that holds position w.
__device__ __forceinline__ int64_t piece_start(int64_t total, int c, int pieces) { return total * c / pieces; }
__device__ __forceinline__ int piece_of(int64_t total, int64_t w, int pieces) {
  return static_cast<int>(((w + 1) * pieces - 1) / total);
}

// The tiles [first, first + count) of one unit that lie in [w, w_end), and where the unit's
// share of that range ends. count 0: no more tiles before w_end.
struct Segment {
  int b, h, group, tiles /* of the unit */, first, count;
  int64_t next;
};
template <class T>
__device__ __forceinline__ Segment next_segment(const TreeArgs &a, const int *pref, int64_t w, int64_t w_end) {
  Segment s = {};
  const int per = a.Hkv * a.groups;
  while (w < w_end) {
    const int x = static_cast<int>(w / per);
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {  // the last sequence that starts at or before it
      const int mid = (lo + hi + 1) >> 1;
      if (pref[mid] <= x) lo = mid; else hi = mid - 1;
    }
    const int cost = pref[lo + 1] - pref[lo];
    const int64_t rem = w - static_cast<int64_t>(pref[lo]) * per;
    const int unit = static_cast<int>(rem / cost), from = static_cast<int>(rem - static_cast<int64_t>(unit) * cost);
    const int to = static_cast<int>(min(static_cast<int64_t>(cost), from + (w_end - w)));
    w += to - from;
    s.first = max(0, from - T::kUnitCost);
    s.count = to - T::kUnitCost - s.first;
    if (s.count > 0) {
      s.b = lo;
      s.tiles = cost - T::kUnitCost;
      s.h = unit / a.groups;
      s.group = unit % a.groups;
      s.next = w;
      return s;
    }
  }
  s.count = 0;
  s.next = w_end;
  return s;
}

// The pieces that hold tiles of a unit: [c0, c1], found by one CTA of kThreads threads.
struct UnitSpan {
  int c0, c1;
};
template <class T, int kThreads>
__device__ __forceinline__ UnitSpan find_span(const TreeArgs &a, int b, int unit, int ctas) {
  __shared__ int sums[2][kThreads / 32];
  int before = 0, all = 0;
  for (int i = threadIdx.x; i < a.B; i += kThreads) {
    const int t = tile_count<T>(a, i) + T::kUnitCost;
    all += t;
    if (i < b) before += t;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sums[0][threadIdx.x >> 5] = all;
    sums[1][threadIdx.x >> 5] = before;
  }
  __syncthreads();
  all = before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    all += sums[0][w];
    before += sums[1][w];
  }
  const int per = a.Hkv * a.groups, cost = tile_count<T>(a, b) + T::kUnitCost;
  const int64_t total = static_cast<int64_t>(all) * per;
  const int64_t w = static_cast<int64_t>(before) * per + static_cast<int64_t>(unit) * cost;
  const int pieces = static_cast<int>(min(static_cast<int64_t>(ctas), total));
  return {piece_of(total, w + T::kUnitCost, pieces), piece_of(total, w + cost - 1, pieces)};
}

// The paths of a sequence's nodes, found by one warp: up[i] is -1 for a used node and -2 for
// an unused one, bits[i] the nodes on its path (none if unused). Pointer doubling: a round
// joins every node's path with that of the node it points to and points further, so a
// chain of n nodes takes log2 n rounds (walking it up took 12 us for 64 nodes on B200).
struct TreePaths {
  int up[kTMaxNodes];
  uint4 bits[kTMaxNodes];
};
__device__ __forceinline__ void tree_paths(TreePaths &t, const int *parents, int n) {
  constexpr int kPer = kTMaxNodes / 32;
  const int lane = threadIdx.x & 31;
  int up[kPer];
  uint4 m[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = k * 32 + lane;
    up[k] = i < n ? ld_act_i32(parents + i) : -2;
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = k * 32 + lane;
    if (up[k] < -1 || up[k] >= i) up[k] = -2;
    const uint32_t own = 1u << lane;
    m[k] = make_uint4(k == 0 ? own : 0u, k == 1 ? own : 0u, k == 2 ? own : 0u, k == 3 ? own : 0u);
    t.up[i] = up[k];
    t.bits[i] = m[k];
  }
  while (__any_sync(0xffffffffu, up[0] >= 0 || up[1] >= 0 || up[2] >= 0 || up[3] >= 0)) {
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (up[k] >= 0) {
        const uint4 o = t.bits[up[k]];
        m[k] = make_uint4(m[k].x | o.x, m[k].y | o.y, m[k].z | o.z, m[k].w | o.w);
        up[k] = t.up[up[k]];
      }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      t.up[k * 32 + lane] = up[k];
      t.bits[k * 32 + lane] = m[k];
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k)
    if (up[k] == -2) t.bits[k * 32 + lane] = make_uint4(0u, 0u, 0u, 0u);
  __syncwarp();
}
static_assert(kTMaxNodes == 128, "four words of 32 nodes");

// The tcgen05 form (tree_attention_tc.cu).
size_t tree_tc_workspace(int head_dim);
int tree_tc_launch(TreeArgs a, int head_dim, cudaStream_t s);
unsigned tree_wait_us();  // the limit that iron_tree_attn_set_wait_us set

}  // namespace iron
