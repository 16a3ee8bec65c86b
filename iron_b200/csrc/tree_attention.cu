// Attention of a tree of drafted tokens over a paged KV cache.
//
// Rows: the Hq / Hkv query heads of all nodes share a kv head, so a (sequence, kv head)
// has num_nodes * group rows that read the same cached K and V. They are cut into groups of
// 16 or 32 rows (mma.sync m16n8k16 has 16). Work: every unit = (sequence, kv head, row
// group) is a list of 64-token tiles -- the cached ones, then the tree's own nodes -- and
// the concatenation of all units' tiles is cut into as many equal pieces as CTAs fit on
// the GPU. Lengths are read on the device, so ragged batches and tables wider than the
// sequences balance all the same. A piece that holds a part of a unit leaves its (max, sum,
// output) as a partial, and the last of the unit's pieces to finish joins them, in the
// order of the tiles (B200, one sequence of 301 tokens, 8 nodes: 20 us per call from Python
// against 25 with a second kernel for the join; 11.8 against 10.5 inside a CUDA graph).
#include "tree.cuh"

namespace iron {

constexpr int kTTile = 64;     // tokens per tile: 16 per warp
constexpr int kTWarps = 4;
struct TreeCut {
  static constexpr int kTile = kTTile, kUnitCost = 1;
};

// kM: groups of 16 rows that a warp holds, and a unit has.
template <int D, int kM>
struct TreeCfg {
  static constexpr int kStages = 3, kCtasPerSm = D == 64 && kM == 1 ? 3 : 2, kRows = 16 * kM;
  static constexpr int kPart = kRows * (2 + D);  // floats of a partial: O, then (m, l)
  static constexpr int kRing = kTWarps * kStages * Stage<D>::kBytes;  // the stages; after them the merge
  static constexpr int kMerge = kTWarps * kRows * D * 4;
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

// Joins partials of one unit, those of pieces first, first + step, ... <= last, in the order
// of its tiles, by one CTA; a thread owns 4 values of a row. kJoin of them are loaded at a
// time, so the join takes a memory round trip per kJoin. A unit of more than 2 kJoin pieces
// is joined in two steps (B200, one sequence of 4608 tokens, 4 nodes: 24.5 -> 14.5 us; with
// 10 to 14 pieces per unit two steps take 1 us more than one): each kJoin pieces by the
// last of them to finish, which leaves the result in the place of the first's, then those
// by the last of all (`to`: that place; null: the output).
constexpr int kJoin = 8;

template <int D, int kM>
__device__ __forceinline__ void join(const TreeArgs &a, int b, int h, int row0, int c0, int first, int last, int step, float *to) {
  using C = TreeCfg<D, kM>;
  const int g = a.Hq / a.Hkv;
  for (int idx0 = 0; idx0 < C::kRows * D / 4; idx0 += 32 * kTWarps) {
    const int idx = idx0 + threadIdx.x, r = idx / (D / 4), d = idx % (D / 4) * 4, row = row0 + r;
    const bool in_rows = row < a.N * g;
    float M = -INFINITY, L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
    bool dead = false;
    for (int c = first; c <= last && in_rows; c += kJoin * step) {
      float2 ml[kJoin];
      float4 o[kJoin];
#pragma unroll
      for (int i = 0; i < kJoin; ++i) {
        const int p = c + i * step;
        ml[i] = make_float2(-INFINITY, 0.f);
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p > last) continue;
        const float *part = a.ws + (static_cast<int64_t>(p) * 2 + (p == c0)) * C::kPart;
        ml[i] = __ldcg(reinterpret_cast<const float2 *>(part + C::kRows * D + 2 * r));
        o[i] = __ldcg(reinterpret_cast<const float4 *>(part + r * D + d));
      }
      float top = M;
#pragma unroll
      for (int i = 0; i < kJoin; ++i) top = fmaxf(top, ml[i].x);
      const float f0 = rescale(M, top);
      M = top;
      L *= f0;
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] *= f0;
#pragma unroll
      for (int i = 0; i < kJoin; ++i) {
        const float f = rescale(ml[i].x, M);
        dead |= ml[i].y < 0.f;
        L += ml[i].y * f;
        O[0] += o[i].x * f;
        O[1] += o[i].y * f;
        O[2] += o[i].z * f;
        O[3] += o[i].w * f;
      }
    }
    if (to) {
      __syncthreads();  // a row's (m, l) is read by several threads
      if (!in_rows) continue;
      if (d == 0) *reinterpret_cast<float2 *>(to + C::kRows * D + 2 * r) = make_float2(M, dead ? -1.f : L);
      *reinterpret_cast<float4 *>(to + r * D + d) = make_float4(O[0], O[1], O[2], O[3]);
    } else if (in_rows) {
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = dead ? 0.f : normalised(O[e], L);
      *reinterpret_cast<uint2 *>(a.out + b * a.os[0] + row / g * a.os[1] + (h * g + row % g) * a.os[2] + d) =
          make_uint2(pack_bf16x2(O[0], O[1]), pack_bf16x2(O[2], O[3]));
    }
  }
}

// Counts this CTA in at `count` (its stores before are in memory first). True for the last
// of `n`, which sees the stores of all of them and leaves the counter at 0.
__device__ __forceinline__ bool last_of(unsigned *count, int n, bool *flag) {
  __syncthreads();
  if (threadIdx.x == 0) {
    // release: the block's stores (ordered before by the barrier); acquire: the others'
    unsigned before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
    *flag = before == static_cast<unsigned>(n - 1);
    if (*flag) *count = 0;  // ready for the next call
  }
  __syncthreads();
  return *flag;
}

template <int D, int kM>
__global__ void __launch_bounds__(32 * kTWarps, TreeCfg<D, kM>::kCtasPerSm) tree_attn_kernel(TreeArgs a) {
  using C = TreeCfg<D, kM>;
  constexpr int kStages = C::kStages, kRows = C::kRows;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red_m[kTWarps][kRows], red_l[kTWarps][kRows];
  __shared__ int pref[kTMaxBatch + 1], warp_sums[kTWarps];
  __shared__ TreePaths tree;
  __shared__ __align__(16) uint32_t paths[kRows][kTMaxNodes / 32];
  __shared__ uint32_t usable[kTMaxNodes / 32];
  __shared__ bool last_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tid = lane & 3;
  Stage<D> *ring = reinterpret_cast<Stage<D> *>(smem) + warp * kStages;
  float (*red_o)[kRows][D] = reinterpret_cast<float (*)[kRows][D]>(smem);
  pdl_launch_dependents();
  pdl_wait();
  cost_prefix<TreeCut, 32 * kTWarps>(a, pref, warp_sums);
  const int g = a.Hq / a.Hkv;
  const int64_t total = static_cast<int64_t>(pref[a.B]) * a.Hkv * a.groups;
  const int pieces = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total));  // none is empty
  if (static_cast<int>(blockIdx.x) >= pieces) return;
  const int64_t w = piece_start(total, blockIdx.x, pieces);
  const int64_t w_end = piece_start(total, blockIdx.x + 1, pieces);
  const int page = 1 << a.page_shift;

  for (Segment sg = next_segment<TreeCut>(a, pref, w, w_end); sg.count > 0;
       sg = next_segment<TreeCut>(a, pref, sg.next, w_end)) {
    const int b = sg.b, h = sg.h, row0 = sg.group * kRows, first = sg.first, count = sg.count;
    const int len = cached_len(a, b), ctiles = (len + kTTile - 1) / kTTile;
    const int *table = a.table + static_cast<int64_t>(b) * a.M;
    // the warp's blocks: cached tiles first .. ctiles - 1 (block 4 i + warp of tokens), then nodes
    const int ncached = max(0, min(first + count, ctiles) - first);
    // page of the cached block of tile first + i: 32 of them per load, one per lane
    auto entry = [&](int i) {
      const int t = (first + i + lane) * kTTile + warp * 16;
      return i + lane < ncached && t < len ? ld_act_i32(table + (t >> a.page_shift)) : -1;
    };
    int pages = entry(0);
    auto request = [&](int i, int stage) {  // block of tile first + i
      if (i < ncached) {
        if ((i & 31) == 0 && i > 0) pages = entry(i);
        const int p = __shfl_sync(0xffffffffu, pages, i & 31), t = (first + i) * kTTile + warp * 16;
        const int n = p >= 0 && p < a.P ? min(16, len - t) : 0;
        const int64_t at0 = n > 0 ? (((static_cast<int64_t>(p) * a.Hkv + h) << a.page_shift) + (t & (page - 1))) * D : 0;
        ring[stage].load(a.k + at0, a.v + at0, D, D, n);
        cp_async_commit();
        return n;
      }
      cp_async_commit();
      return 0;
    };
    int valid[kStages];  // tokens of the blocks in flight
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) valid[s] = request(s, s);

    WarpAttn<D> at[kM];
    const int rows = a.N * g;
    auto q_row = [&](int r) {
      return r < rows ? a.q + b * a.qs[0] + r / g * a.qs[1] + (h * g + r % g) * a.qs[2] : nullptr;
    };
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      at[m].clear();
      at[m].load_q(q_row(row0 + 16 * m + gid), q_row(row0 + 16 * m + gid + 8));
    }
    if (first + count > ctiles) {  // the tree's nodes are part of this piece: their paths
      if (warp == 0) {
        tree_paths(tree, a.parents + static_cast<int64_t>(b) * a.N, a.N);
#pragma unroll
        for (int k = 0; k < kTMaxNodes / 32; ++k) {
          const unsigned all = __ballot_sync(0xffffffffu, tree.up[k * 32 + lane] == -1);
          if (lane == 0) usable[k] = all;
        }
        if (lane < kRows) {
          const int i = (row0 + lane) / g;
          *reinterpret_cast<uint4 *>(paths[lane]) = i < a.N ? tree.bits[i] : make_uint4(0u, 0u, 0u, 0u);
        }
      }
      __syncthreads();
    }
    for (int i0 = 0; i0 < ncached; i0 += kStages) {
#pragma unroll
      for (int s = 0; s < kStages; ++s) {
        const int i = i0 + s;
        if (i >= ncached) break;
        cp_async_wait<kStages - 2>();
        __syncwarp();  // the block is here, and every lane is done with the stage refilled next
        constexpr int kLast = kStages - 1;
        valid[(s + kLast) % kStages] = request(i + kLast, (s + kLast) % kStages);
        if (valid[s] > 0) {
          const uint32_t see[2] = {0xffffu >> (16 - valid[s]), 0xffffu >> (16 - valid[s])};
#pragma unroll
          for (int m = 0; m < kM; ++m) at[m].step(ring[s], a.scale_log2, see);
        }
      }
    }
    cp_async_wait<0>();
    __syncwarp();
    for (int i = max(first, ctiles); i < first + count; ++i) {
      const int j0 = (i - ctiles) * kTTile + warp * 16;
      if (j0 >= a.N) continue;
      const uint32_t can = usable[j0 >> 5] >> (j0 & 31) & 0xffffu;
      const int64_t at0 = b * a.ks[0] + j0 * a.ks[1] + h * a.ks[2];
      Stage<D> &st = ring[0];
      st.load(a.k_new + at0, a.v_new + at0, a.ks[1], a.ks[1], can ? 32 - __clz(can) : 0);
      cp_async_commit();
      cp_async_wait<0>();
      __syncwarp();
      uint32_t see[kM][2];
#pragma unroll
      for (int m = 0; m < 2 * kM; ++m) see[m >> 1][m & 1] = paths[8 * m + gid][j0 >> 5] >> (j0 & 31) & 0xffffu;
      // a masked token's probability is 0, but 0 * inf is not: values that are not finite
      // leave the tile and are added to the rows that see them
      bool odd = false;
#pragma unroll
      for (int v = 0; v < D / 16; ++v) {
        const int idx = v * 32 + lane;
        uint4 *p = reinterpret_cast<uint4 *>(st.x + (16 + idx / (D / 8)) * Stage<D>::kRow + idx % (D / 8) * 8);
        uint4 y = *p;
        uint32_t *e = reinterpret_cast<uint32_t *>(&y);
        bool change = false;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if ((e[c] & 0x7f80u) == 0x7f80u) e[c] &= 0xffff0000u, change = true;
          if ((e[c] & 0x7f800000u) == 0x7f800000u) e[c] &= 0xffffu, change = true;
        }
        if (change) *p = y;
        odd |= change;
      }
      odd = __any_sync(0xffffffffu, odd);
      __syncwarp();
#pragma unroll
      for (int m = 0; m < kM; ++m) at[m].step(st, a.scale_log2, see[m]);
      if (odd) {  // after the step, which rescales O
        for (int t = 0; t < 16; ++t) {
          if (!(can >> t & 1u)) continue;
          const uint16_t *vt = a.v_new + at0 + t * a.ks[1];
#pragma unroll
          for (int j = 0; j < D / 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float f = bf16_bits_to_float(ld_act_u16(vt + 8 * j + 2 * tid + e));
              if (isfinite(f)) continue;
#pragma unroll
              for (int m = 0; m < 2 * kM; ++m)
                if (see[m >> 1][m & 1] >> t & 1u) at[m >> 1].o[j][2 * (m & 1) + e] += f;
            }
        }
      }
      __syncwarp();  // done with the stage
    }
#pragma unroll
    for (int m = 0; m < kM; ++m) at[m].finish();
    __syncthreads();  // every warp is done with the V tiles
#pragma unroll
    for (int m = 0; m < 2 * kM; ++m) {
      const WarpAttn<D> &x = at[m >> 1];
      const int r = 8 * m + gid, e = m & 1;
      if (tid == 0) {
        red_m[warp][r] = x.m[e];
        red_l[warp][r] = x.l[e];
      }
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2 *>(&red_o[warp][r][8 * j + 2 * tid]) = make_float2(x.o[j][2 * e], x.o[j][2 * e + 1]);
    }
    __syncthreads();
    const bool whole = count == sg.tiles;
    const bool has_tree = first + count > ctiles;
    float *part = a.ws + (static_cast<int64_t>(blockIdx.x) * 2 + (first == 0 ? 1 : 0)) * C::kPart;
#pragma unroll 2
    for (int idx = threadIdx.x; idx < kRows * D / 4; idx += 32 * kTWarps) {
      const int r = idx / (D / 4), d = idx % (D / 4) * 4, rr = row0 + r;
      if (rr >= rows) break;
      float M = -INFINITY, L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < kTWarps; ++q) M = fmaxf(M, red_m[q][r]);
#pragma unroll
      for (int q = 0; q < kTWarps; ++q) {
        const float f = rescale(red_m[q][r], M);
        const float4 o = *reinterpret_cast<const float4 *>(&red_o[q][r][d]);
        L += red_l[q][r] * f;
        O[0] += o.x * f;
        O[1] += o.y * f;
        O[2] += o.z * f;
        O[3] += o.w * f;
      }
      // an unused node: its path is empty (a used one holds the node itself)
      bool dead = false;
      if (has_tree) dead = (paths[r][0] | paths[r][1] | paths[r][2] | paths[r][3]) == 0;
      if (whole) {
#pragma unroll
        for (int e = 0; e < 4; ++e) O[e] = dead ? 0.f : normalised(O[e], L);
        *reinterpret_cast<uint2 *>(a.out + b * a.os[0] + rr / g * a.os[1] + (h * g + rr % g) * a.os[2] + d) =
            make_uint2(pack_bf16x2(O[0], O[1]), pack_bf16x2(O[2], O[3]));
      } else {
        // a sum of -1: the join writes zeros
        if (d == 0) *reinterpret_cast<float2 *>(part + kRows * D + 2 * r) = make_float2(M, dead ? -1.f : L);
        *reinterpret_cast<float4 *>(part + r * D + d) = make_float4(O[0], O[1], O[2], O[3]);
      }
    }
    if (whole) {
      __syncthreads();  // shared memory is used again
    } else {
      const int unit = h * a.groups + sg.group, cost = sg.tiles + TreeCut::kUnitCost;
      const int64_t start = static_cast<int64_t>(pref[b]) * a.Hkv * a.groups + static_cast<int64_t>(unit) * cost;
      const int c0 = piece_of(total, start + TreeCut::kUnitCost, pieces), c1 = piece_of(total, start + cost - 1, pieces);
      unsigned *count = a.counts + 2 * gridDim.x + static_cast<int64_t>(b) * a.Hkv * a.groups + unit;
      if (c1 - c0 < 2 * kJoin) {
        if (last_of(count, c1 - c0 + 1, &last_s)) join<D, kM>(a, b, h, row0, c0, c0, c1, 1, nullptr);
      } else {
        const int p0 = c0 + (static_cast<int>(blockIdx.x) - c0) / kJoin * kJoin, p1 = min(p0 + kJoin - 1, c1);
        const int place = 2 * p0 + (p0 == c0);  // as the partial's: one unit per place
        if (last_of(a.counts + place, p1 - p0 + 1, &last_s)) {
          join<D, kM>(a, b, h, row0, c0, p0, p1, 1, a.ws + static_cast<int64_t>(place) * C::kPart);
          if (last_of(count, (c1 - c0) / kJoin + 1, &last_s)) join<D, kM>(a, b, h, row0, c0, c0, c1, kJoin, nullptr);
        }
      }
      __syncthreads();
    }
  }
}

}  // namespace iron

using namespace iron;

static int tree_pieces(int head_dim, int unit) {
  return sm_count() * (head_dim == 64 && unit == 16 ? TreeCfg<64, 1>::kCtasPerSm : TreeCfg<64, 2>::kCtasPerSm);
}
static_assert(TreeCfg<64, 2>::kCtasPerSm == TreeCfg<128, 1>::kCtasPerSm);
static_assert(TreeCfg<64, 2>::kCtasPerSm == TreeCfg<128, 2>::kCtasPerSm);

// Rows of a unit. 32 read K and V half as often as 16; 16 are cut finer and have less to
// join. 32 are taken where a CTA's share of full tables is at least 32 tiles of 16 rows.
// B200, 32 rows, us with 16 / 32: head dim 64, 1 x 4608 tokens (3 tiles) 18 / 20, 4 x 4608 (10)
// 24 / 32, 16 x 4608 (41) 52 / 49, 64 x 2304 (83) 113 / 89; head dim 128, 1 x 16384 (14) 37 / 42,
// 8 x 32768 (221) 371 / 225.
static int unit_rows(int rows, int64_t tiles, int head_dim) {
  return rows > 16 && tiles >= 32LL * tree_pieces(head_dim, 16) ? 32 : 16;
}
// 64-token tiles of 16 rows that full tables hold.
static int64_t full_tiles(const iron_page_pool *c, int rows) {
  const int64_t longest = static_cast<int64_t>(c->max_pages) * c->page_size;
  return static_cast<int64_t>(c->slots) * c->kv_heads * ((rows + 15) / 16) * ((longest + kTTile - 1) / kTTile);
}

// Bytes of the mma.sync form's counters, two per piece and one per unit, rounded up to 16.
static size_t tree_counters(int B, int N, int Hq, int Hkv, int head_dim) {
  const size_t units = static_cast<size_t>(B) * Hkv * ((static_cast<size_t>(N) * (Hq / Hkv) + 15) / 16);
  return ((2 * static_cast<size_t>(tree_pieces(head_dim, 16)) + units) * sizeof(unsigned) + 15) / 16 * 16;
}

static bool no_tree(int batch, int num_nodes, int num_heads, int kv_heads, int head_dim) {
  return batch <= 0 || num_nodes <= 0 || num_heads <= 0 || kv_heads <= 0 || (head_dim != 64 && head_dim != 128);
}

extern "C" size_t iron_tree_attn_counter_bytes(int batch, int num_nodes, int num_heads, int kv_heads, int head_dim) {
  return no_tree(batch, num_nodes, num_heads, kv_heads, head_dim) ? 0 : tree_counters(batch, num_nodes, num_heads, kv_heads, head_dim);
}

extern "C" size_t iron_tree_attn_workspace_bytes(int batch, int num_nodes, int num_heads, int kv_heads, int head_dim) {
  if (no_tree(batch, num_nodes, num_heads, kv_heads, head_dim)) return 0;
  // the counters, then the partials of any form
  const size_t f16 = static_cast<size_t>(tree_pieces(head_dim, 16)) * 2 * 16 * (2 + head_dim) * sizeof(float);
  const size_t f32 = static_cast<size_t>(tree_pieces(head_dim, 32)) * 2 * 32 * (2 + head_dim) * sizeof(float);
  const size_t few = f16 > f32 ? f16 : f32, many = tree_tc_workspace(head_dim);
  return tree_counters(batch, num_nodes, num_heads, kv_heads, head_dim) + (few > many ? few : many);
}

// The tensor cores' 128-row tiles are used from kTensorRows rows of a (sequence, kv head) on,
// where the form above would need a second unit of 32; but up to kFewRows rows only if full
// tables hold more than kFewTiles tiles of 16 rows: that form's pipeline takes about 13 us
// (head dim 64) or 18 (128) to fill and drain. B200, us, here / there: 32 rows, 16 x 4608 tokens
// at head dim 64 49 / 62, 64 x 2304 87 / 130, 8 x 32768 at 128 230 / 310; 36 rows 74 / 62, 154 / 132
// and 437 / 309; 64 rows, 1 x 300 (160 tiles) 11 / 14, 1 x 4608 (2304) 22 / 23 and at 128 32 / 41,
// 4 x 4608 (9216) 35 / 27 and 57 / 44; 104 rows, 1 x 2304 (2016) 19 / 20 and 28 / 36; 256 rows,
// 1 x 300 at 128 (640) 26 / 21.
constexpr int kTensorRows = 33, kFewRows = 128, kFewTiles = 2560;

// The tcgen05 form takes positive scales that do not vanish in log2 units, and new rows
// whose strides TMA takes (not 0: broadcast views go to the other form).
static bool use_tensor_form(const TreeArgs &a, int64_t tiles) {
  for (int i = 0; i < 3; ++i) {
    const int n = i == 0 ? a.B : i == 1 ? a.N : a.Hkv;
    if (n > 1 && (a.ks[i] <= 0 || a.ks[i] >= (1LL << 38))) return false;
  }
  const int rows = a.N * (a.Hq / a.Hkv);
  return rows >= kTensorRows && (rows > kFewRows || tiles > kFewTiles) && a.scale_log2 >= 1e-30f;
}

template <int D, int kM>
static int launch_few(const TreeArgs &a, cudaStream_t s) {
  using C = TreeCfg<D, kM>;
  static PerDeviceOnce once;
  const int st = once.run([] {
    return call_status(cudaFuncSetAttribute(tree_attn_kernel<D, kM>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  });
  if (st != IRON_OK) return st;
  return launch(tree_attn_kernel<D, kM>, dim3(tree_pieces(D, C::kRows)), dim3(32 * kTWarps), C::kSmem, s, true, a);
}

extern "C" int iron_tree_attn(const iron_page_pool *c, const uint16_t *q, const uint16_t *k_new, const uint16_t *v_new,
                              const int32_t *parents, uint16_t *out, int num_nodes, int num_heads,
                              const int64_t *q_strides, const int64_t *kv_strides, const int64_t *out_strides,
                              float scale, void *workspace, size_t workspace_bytes, unsigned flags, void *stream) {
  (void)flags;
  const int chk = pool_geometry_check(c);
  if (chk != IRON_OK) return chk;
  if (!c->lens || !q || !k_new || !v_new || !parents || !out || !q_strides || !kv_strides || !out_strides || !workspace)
    return IRON_ERR_NULL;
  if (c->layers != 1 || num_nodes <= 0 || num_heads <= 0 || num_heads % c->kv_heads) return IRON_ERR_SHAPE;
  const int g = num_heads / c->kv_heads;
  if (num_nodes > kTMaxNodes || g > 16 || c->slots > kTMaxBatch) return IRON_ERR_UNSUPPORTED;
  if (!aligned16(q) || !aligned16(k_new) || !aligned16(v_new) || !aligned16(out) || !aligned16(workspace))
    return IRON_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 || kv_strides[i] % 8 || out_strides[i] % 8) return IRON_ERR_ALIGN;
  if (workspace_bytes < iron_tree_attn_workspace_bytes(c->slots, num_nodes, num_heads, c->kv_heads, c->head_dim))
    return IRON_ERR_WORKSPACE;
  TreeArgs a = {};
  a.q = q;
  a.k_new = k_new;
  a.v_new = v_new;
  a.k = c->k;
  a.v = c->v;
  a.table = c->page_table;
  a.lens = c->lens;
  a.parents = parents;
  a.out = out;
  a.counts = static_cast<unsigned *>(workspace);
  a.ws = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) +
                                   tree_counters(c->slots, num_nodes, num_heads, c->kv_heads, c->head_dim));
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i];
    a.ks[i] = kv_strides[i];
    a.os[i] = out_strides[i];
  }
  a.B = c->slots;
  a.N = num_nodes;
  a.Hq = num_heads;
  a.Hkv = c->kv_heads;
  // the tiles (and unit costs) of all sequences are counted in ints
  const int64_t longest = static_cast<int64_t>(c->max_pages) * c->page_size;
  if (c->slots * ((longest + kTTile - 1) / kTTile + kTMaxNodes / kTTile + 3) > 0x7fffffff) return IRON_ERR_SHAPE;
  const int64_t tiles = full_tiles(c, num_nodes * g);
  const int unit = unit_rows(num_nodes * g, tiles, c->head_dim);
  a.groups = (num_nodes * g + unit - 1) / unit;
  a.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  a.M = c->max_pages;
  a.P = c->num_pages;
  a.scale_log2 = scale * kLog2e;
  a.wait_us = tree_wait_us();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (use_tensor_form(a, tiles)) return tree_tc_launch(a, c->head_dim, s);
  const bool two = unit == 32;
  if (c->head_dim == 128) return two ? launch_few<128, 2>(a, s) : launch_few<128, 1>(a, s);
  return two ? launch_few<64, 2>(a, s) : launch_few<64, 1>(a, s);
}
