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
  float *ws;  // partials: what a piece of the work leaves of a unit that it holds in part
  int64_t qs[3], ks[3], os[3];  // element strides {batch, node, head}
  int B, N, Hq, Hkv, groups /* row groups per (sequence, kv head) */, page_shift, M, P;
  float scale_log2;
};

__device__ __forceinline__ int cached_len(const TreeArgs &a, int b) {
  return min(max(ld_act_i32(a.lens + b), 0), a.M << a.page_shift);
}

// Tiles of a sequence: its cached tokens, then its nodes.
template <int kTile>
__device__ __forceinline__ int tile_count(const TreeArgs &a, int b) {
  return (cached_len(a, b) + kTile - 1) / kTile + (a.N + kTile - 1) / kTile;
}

// Exclusive prefix sum of the sequences' tile counts into pref[0 .. B].
template <int kThreads, int kTile>
__device__ __forceinline__ void tile_prefix(const TreeArgs &a, int *pref, int *warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int v = b < a.B ? tile_count<kTile>(a, b) : 0;
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

// `total` tiles cut into `pieces` equal parts (none empty): where part c starts, and the
// part that holds tile w.
__device__ __forceinline__ int64_t piece_start(int64_t total, int c, int pieces) { return total * c / pieces; }
__device__ __forceinline__ int piece_of(int64_t total, int64_t w, int pieces) {
  return static_cast<int>(((w + 1) * pieces - 1) / total);
}

// The part of a unit = (sequence, kv head, row group) that starts at tile w of all and ends
// with the unit or at w_end.
struct Segment {
  int b, h, group, tiles /* of the unit */, first, count;
};
__device__ __forceinline__ Segment find_segment(const TreeArgs &a, const int *pref, int64_t w, int64_t w_end) {
  const int per = a.Hkv * a.groups, x = static_cast<int>(w / per);
  int lo = 0, hi = a.B - 1;
  while (lo < hi) {  // the last sequence that starts at or before it
    const int mid = (lo + hi + 1) >> 1;
    if (pref[mid] <= x) lo = mid; else hi = mid - 1;
  }
  Segment s;
  s.b = lo;
  s.tiles = pref[lo + 1] - pref[lo];
  const int64_t rem = w - static_cast<int64_t>(pref[lo]) * per;
  const int unit = static_cast<int>(rem / s.tiles);
  s.first = static_cast<int>(rem % s.tiles);
  s.count = static_cast<int>(min(static_cast<int64_t>(s.tiles - s.first), w_end - w));
  s.h = unit / a.groups;
  s.group = unit % a.groups;
  return s;
}

// The pieces that hold a unit: [c0, c1], found by one CTA of kThreads threads.
struct UnitSpan {
  int c0, c1;
};
template <int kThreads, int kTile>
__device__ __forceinline__ UnitSpan find_span(const TreeArgs &a, int b, int unit, int ctas) {
  __shared__ int sums[2][kThreads / 32];
  int before = 0, all = 0;
  for (int i = threadIdx.x; i < a.B; i += kThreads) {
    const int t = tile_count<kTile>(a, i);
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
  const int per = a.Hkv * a.groups, tiles = tile_count<kTile>(a, b);
  const int64_t total = static_cast<int64_t>(all) * per;
  const int64_t w = static_cast<int64_t>(before) * per + static_cast<int64_t>(unit) * tiles;
  const int pieces = static_cast<int>(min(static_cast<int64_t>(ctas), total));
  return {piece_of(total, w, pieces), piece_of(total, w + tiles - 1, pieces)};
}

// Node i's path as bits, or none and false if it is unused. parents [kTMaxNodes].
__device__ __forceinline__ bool tree_path(const int *parents, int i, uint32_t (&bits)[kTMaxNodes / 32]) {
#pragma unroll
  for (int w = 0; w < kTMaxNodes / 32; ++w) bits[w] = 0;
  int j = i;
  while (true) {
#pragma unroll
    for (int w = 0; w < kTMaxNodes / 32; ++w)
      if (j >> 5 == w) bits[w] |= 1u << (j & 31);
    const int p = parents[j];
    if (p == -1) return true;
    if (p < 0 || p >= j) break;
    j = p;
  }
#pragma unroll
  for (int w = 0; w < kTMaxNodes / 32; ++w) bits[w] = 0;
  return false;
}

// The tcgen05 form (tree_attention_tc.cu).
size_t tree_tc_workspace(int head_dim);
int tree_tc_launch(TreeArgs a, int head_dim, bool pdl, cudaStream_t s);

}  // namespace iron
