// Attention of a tree of drafted tokens over a paged KV cache.
//
// Rows: the Hq / Hkv query heads of all nodes share a kv head, so a (sequence, kv head)
// has num_nodes * group rows that read the same cached K and V. They are cut into groups
// of 16 rows (the M of mma.sync m16n8k16). Work: every unit = (sequence, kv head, row
// group) is a list of 64-token tiles -- the cached ones, then the tree's own nodes -- and
// the concatenation of all units' tiles is cut into as many equal pieces as CTAs fit on
// the GPU. Lengths are read on the device, so ragged batches and tables wider than the
// sequences balance all the same. A piece that holds a part of a unit leaves its (max, sum,
// output) as a partial, and the last of the unit's pieces to finish joins them, in the
// order of the tiles (B200, one sequence of 301 tokens, 8 nodes: 20 us per call from Python
// against 25 with a second kernel for the join; 11.8 against 10.5 inside a CUDA graph).
#include "tree.cuh"

namespace iron {

constexpr int kTRows = 16;     // rows per unit
constexpr int kTTile = 64;     // tokens per tile: 16 per warp
constexpr int kTWarps = 4;
struct TreeCut {
  static constexpr int kTile = kTTile, kUnitCost = 1;
};

template <int D>
struct TreeCfg {
  static constexpr int kStages = 3, kCtasPerSm = D == 64 ? 3 : 2;
  static constexpr int kRing = kTWarps * kStages * Stage<D>::kBytes;  // the stages; after them the merge
  static constexpr int kMerge = kTWarps * kTRows * D * 4;
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

// Joins the partials of one unit (pieces c0 .. c1), in the order of its tiles, by one CTA; a
// thread owns 4 values of a row. kJoin pieces are loaded at a time, so a unit of many
// pieces costs a memory round trip per kJoin of them.
constexpr int kJoin = 8;

template <int D>
__device__ __forceinline__ void join_unit(const TreeArgs &a, int b, int h, int row0, int c0, int c1) {
  const int g = a.Hq / a.Hkv;
#pragma unroll 2
  for (int idx = threadIdx.x; idx < kTRows * D / 4; idx += 32 * kTWarps) {
    const int r = idx / (D / 4), d = idx % (D / 4) * 4, row = row0 + r;
    if (row >= a.N * g) break;
    float M = -INFINITY, L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
    bool dead = false;
    for (int c = c0; c <= c1; c += kJoin) {
      float2 ml[kJoin];
      float4 o[kJoin];
#pragma unroll
      for (int i = 0; i < kJoin; ++i) {
        const bool in = c + i <= c1;
        const float *part = a.ws + (static_cast<int64_t>(in ? c + i : c0) * 2 + (c + i == c0 || !in ? 1 : 0)) * kTRows * (2 + D);
        ml[i] = __ldcg(reinterpret_cast<const float2 *>(part + kTRows * D + 2 * r));
        o[i] = __ldcg(reinterpret_cast<const float4 *>(part + r * D + d));
        if (!in) ml[i] = make_float2(-INFINITY, 0.f), o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
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
#pragma unroll
    for (int e = 0; e < 4; ++e) O[e] = dead ? 0.f : normalised(O[e], L);
    *reinterpret_cast<uint2 *>(a.out + b * a.os[0] + row / g * a.os[1] + (h * g + row % g) * a.os[2] + d) =
        make_uint2(pack_bf16x2(O[0], O[1]), pack_bf16x2(O[2], O[3]));
  }
}

template <int D>
__global__ void __launch_bounds__(32 * kTWarps, TreeCfg<D>::kCtasPerSm) tree_attn_kernel(TreeArgs a) {
  using C = TreeCfg<D>;
  constexpr int kStages = C::kStages;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red_m[kTWarps][kTRows], red_l[kTWarps][kTRows];
  __shared__ int pref[kTMaxBatch + 1], warp_sums[kTWarps];
  __shared__ TreePaths tree;
  __shared__ __align__(16) uint32_t paths[kTRows][kTMaxNodes / 32];
  __shared__ uint32_t usable[kTMaxNodes / 32];
  __shared__ bool last_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tid = lane & 3;
  Stage<D> *ring = reinterpret_cast<Stage<D> *>(smem) + warp * kStages;
  float (*red_o)[kTRows][D] = reinterpret_cast<float (*)[kTRows][D]>(smem);
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
    const int b = sg.b, h = sg.h, row0 = sg.group * kTRows, first = sg.first, count = sg.count;
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

    WarpAttn<D> at;
    at.clear();
    const int r_lo = row0 + gid, r_hi = row0 + gid + 8, rows = a.N * g;
    const uint16_t *qb = a.q + b * a.qs[0];
    at.load_q(r_lo < rows ? qb + r_lo / g * a.qs[1] + (h * g + r_lo % g) * a.qs[2] : nullptr,
              r_hi < rows ? qb + r_hi / g * a.qs[1] + (h * g + r_hi % g) * a.qs[2] : nullptr);
    if (first + count > ctiles) {  // the tree's nodes are part of this piece: their paths
      if (warp == 0) {
        tree_paths(tree, a.parents + static_cast<int64_t>(b) * a.N, a.N);
#pragma unroll
        for (int k = 0; k < kTMaxNodes / 32; ++k) {
          const unsigned all = __ballot_sync(0xffffffffu, tree.up[k * 32 + lane] == -1);
          if (lane == 0) usable[k] = all;
        }
        if (lane < kTRows) {
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
          at.step(ring[s], a.scale_log2, see);
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
      const uint32_t see[2] = {paths[gid][j0 >> 5] >> (j0 & 31) & 0xffffu, paths[gid + 8][j0 >> 5] >> (j0 & 31) & 0xffffu};
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
      if (__any_sync(0xffffffffu, odd)) {
        __syncwarp();
        for (int t = 0; t < 16; ++t) {
          if (!(can >> t & 1u)) continue;
          const uint16_t *vt = a.v_new + at0 + t * a.ks[1];
#pragma unroll
          for (int j = 0; j < D / 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float f = bf16_bits_to_float(ld_act_u16(vt + 8 * j + 2 * tid + e));
              if (isfinite(f)) continue;
              if (see[0] >> t & 1u) at.o[j][e] += f;
              if (see[1] >> t & 1u) at.o[j][2 + e] += f;
            }
        }
      }
      at.step(st, a.scale_log2, see);
      __syncwarp();  // done with the stage
    }
    at.finish();
    __syncthreads();  // every warp is done with the V tiles
    if (tid == 0) {
      red_m[warp][gid] = at.m[0];
      red_m[warp][gid + 8] = at.m[1];
      red_l[warp][gid] = at.l[0];
      red_l[warp][gid + 8] = at.l[1];
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      *reinterpret_cast<float2 *>(&red_o[warp][gid][8 * j + 2 * tid]) = make_float2(at.o[j][0], at.o[j][1]);
      *reinterpret_cast<float2 *>(&red_o[warp][gid + 8][8 * j + 2 * tid]) = make_float2(at.o[j][2], at.o[j][3]);
    }
    __syncthreads();
    const bool whole = count == sg.tiles;
    const bool has_tree = first + count > ctiles;
    float *part = a.ws + (static_cast<int64_t>(blockIdx.x) * 2 + (first == 0 ? 1 : 0)) * kTRows * (2 + D);  // O, then (m, l)
    for (int idx = threadIdx.x; idx < kTRows * D; idx += 32 * kTWarps) {
      const int r = idx / D, d = idx % D;
      float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
      for (int q = 0; q < kTWarps; ++q) M = fmaxf(M, red_m[q][r]);
#pragma unroll
      for (int q = 0; q < kTWarps; ++q) {
        const float f = rescale(red_m[q][r], M);
        L += red_l[q][r] * f;
        O += red_o[q][r][d] * f;
      }
      // an unused node: its path is empty (a used one holds the node itself)
      bool dead = false;
      if (has_tree) dead = (paths[r][0] | paths[r][1] | paths[r][2] | paths[r][3]) == 0;
      if (whole) {
        const int rr = row0 + r;
        if (rr < rows)
          a.out[b * a.os[0] + rr / g * a.os[1] + (h * g + rr % g) * a.os[2] + d] =
              float_to_bf16_bits(dead ? 0.f : normalised(O, L));
      } else {
        if (d == 0) {
          part[kTRows * D + 2 * r] = M;
          part[kTRows * D + 2 * r + 1] = dead ? -1.f : L;  // -1: the join writes zeros
        }
        part[r * D + d] = O;
      }
    }
    __syncthreads();  // shared memory is used again
    if (!whole) {
      // this piece's part is in memory before it is counted; the one that completes the
      // count has seen all of them
      const int unit = h * a.groups + sg.group, cost = sg.tiles + TreeCut::kUnitCost;
      const int64_t start = static_cast<int64_t>(pref[b]) * a.Hkv * a.groups + static_cast<int64_t>(unit) * cost;
      const int c0 = piece_of(total, start + TreeCut::kUnitCost, pieces), c1 = piece_of(total, start + cost - 1, pieces);
      unsigned *count = a.counts + static_cast<int64_t>(b) * a.Hkv * a.groups + unit;
      if (threadIdx.x == 0) {
        // release: the block's stores (ordered before by the barrier); acquire: the others'
        unsigned before;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
        last_s = before == static_cast<unsigned>(c1 - c0);
        if (last_s) *count = 0;  // ready for the next call
      }
      __syncthreads();
      if (last_s) join_unit<D>(a, b, h, row0, c0, c1);
      __syncthreads();
    }
  }
}

}  // namespace iron

using namespace iron;

static int tree_pieces(int head_dim) {
  return sm_count() * (head_dim == 128 ? TreeCfg<128>::kCtasPerSm : TreeCfg<64>::kCtasPerSm);
}

// Bytes of a counter per unit of the mma.sync form, rounded up to 16.
static size_t tree_counters(int B, int N, int Hq, int Hkv) {
  const size_t groups = (static_cast<size_t>(N) * (Hq / Hkv) + kTRows - 1) / kTRows;
  return (B * Hkv * groups * sizeof(unsigned) + 15) / 16 * 16;
}

extern "C" size_t iron_tree_attn_workspace_bytes(int batch, int num_nodes, int num_heads, int kv_heads, int head_dim) {
  if (batch <= 0 || num_nodes <= 0 || num_heads <= 0 || kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  // the counters of the units that are cut, then the partials
  const size_t few = tree_counters(batch, num_nodes, num_heads, kv_heads) +
                     static_cast<size_t>(tree_pieces(head_dim)) * 2 * kTRows * (2 + head_dim) * sizeof(float);
  const size_t many = tree_counters(batch, num_nodes, num_heads, kv_heads) + tree_tc_workspace(head_dim);
  return few > many ? few : many;
}

// Rows of a (sequence, kv head) from which the tensor cores' 128-row tiles are used.
constexpr int kTensorRows = 33;

// The tcgen05 form takes positive scales that do not vanish in log2 units, and new rows
// whose strides TMA takes (not 0: broadcast views go to the other form).
static bool use_tensor_form(const TreeArgs &a) {
  for (int i = 0; i < 3; ++i) {
    const int n = i == 0 ? a.B : i == 1 ? a.N : a.Hkv;
    if (n > 1 && (a.ks[i] <= 0 || a.ks[i] >= (1LL << 38))) return false;
  }
  return a.N * (a.Hq / a.Hkv) >= kTensorRows && a.scale_log2 >= 1e-30f;
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
  a.ws = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + tree_counters(c->slots, num_nodes, num_heads, c->kv_heads));
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i];
    a.ks[i] = kv_strides[i];
    a.os[i] = out_strides[i];
  }
  a.B = c->slots;
  a.N = num_nodes;
  a.Hq = num_heads;
  a.Hkv = c->kv_heads;
  a.groups = (num_nodes * g + kTRows - 1) / kTRows;
  a.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  a.M = c->max_pages;
  a.P = c->num_pages;
  a.scale_log2 = scale * kLog2e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = c->head_dim == 128;
  if (use_tensor_form(a)) return tree_tc_launch(a, c->head_dim, s);
  const int pieces = tree_pieces(c->head_dim);
  static PerDeviceOnce once;
  int st = once.run([] {
    cudaError_t e = cudaFuncSetAttribute(tree_attn_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, TreeCfg<64>::kSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(tree_attn_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, TreeCfg<128>::kSmem);
    return call_status(e);
  });
  if (st != IRON_OK) return st;
  return launch(wide ? tree_attn_kernel<128> : tree_attn_kernel<64>, dim3(pieces), dim3(32 * kTWarps),
                wide ? TreeCfg<128>::kSmem : TreeCfg<64>::kSmem, s, true, a);
}
