// Decode attention over the pages that a cheap score selects.
//
// One kernel; a cluster of CTAs per (sequence, kv head):
//   1. each CTA scores its share of the pages from their summaries;
//   2. after a cluster barrier every CTA has all keys (its own and, through distributed
//      shared memory, the others') and picks the same pages;
//   3. the kept pages' 16-token blocks are dealt out to the cluster's warps;
//   4. each CTA merges its warps, and the cluster merges its CTAs, each rank a share of the
//      output (fixed order throughout).
// The score is a sum of products of whole numbers: over the heads, q8 meets hi8 where it is
// positive and lo8 where it is negative, = hi8 . (sum of the positive q8) + lo8 . (sum of
// the negative q8), so one 16-bit weight vector of 2 D values serves the whole query group,
// and dp2a (two 16 x 8 bit products per instruction) sums it exactly.
//
// Bound: HBM (summaries of all pages, K and V of the kept ones) for batches, the latency of
// the four steps for single sequences. As four kernels (score, pick, attend, join) the
// steps of all sequences waited for one another, and 64 sequences of 32768 tokens, 64 pages
// kept, took 240 us on B200.
#include <cfloat>

#include <cooperative_groups.h>

#include "paged.cuh"

namespace iron {

namespace cg = cooperative_groups;

constexpr int kSWarps = 4;
constexpr int kSThreads = 32 * kSWarps;
constexpr int kMaxTop = 4096;  // the kept pages are listed in shared memory

struct SelectArgs {
  const uint16_t *q, *k, *v;
  const int8_t *codes;
  const float *scales;
  const int *table, *lens;
  uint16_t *out;
  int *selected;
  uint32_t *keys;  // workspace [B, Hkv, M] where a sequence's keys do not fit in shared memory, else null
  int64_t qs[2], os[2];
  int Hq, Hkv, page_shift, M, P, top;
  float scale_log2;
};

__device__ __forceinline__ int cached_len(const SelectArgs &a, int b) {
  return min(max(ld_act_i32(a.lens + b), 0), a.M << a.page_shift);
}

// The query group's weights: wgt[0 .. D) the sums of its negative q8 (they meet lo8),
// wgt[D .. 2 D) of its positive ones (they meet hi8). q8 = rint(q / a * 127) with IEEE
// division, |sum| <= 16 * 127. Thread d < D holds x[i] = q of head i, dimension d.
template <int D>
__device__ __forceinline__ void query_weights(const float (&x)[16], int g, int16_t *wgt, float *red) {
  float top = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    nan |= x[i] != x[i];
    top = fmaxf(top, fabsf(x[i]));
  }
  top = warp_max(nan ? INFINITY : top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSWarps; ++w) top = fmaxf(top, red[w]);
  const bool fine = top > 0.f && top < INFINITY;
  if (threadIdx.x < D) {
    int neg = 0, pos = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i >= g) break;
      const int q8 = fine ? static_cast<int>(rintf(__fmul_rn(__fdiv_rn(x[i], top), 127.f))) : 0;
      neg += min(q8, 0);
      pos += max(q8, 0);
    }
    wgt[threadIdx.x] = static_cast<int16_t>(neg);
    wgt[D + threadIdx.x] = static_cast<int16_t>(pos);
  }
  __syncthreads();
}

// An fp32 score as an unsigned key of the same order.
__device__ __forceinline__ uint32_t score_key(float s) {
  const uint32_t u = __float_as_uint(s);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int D>
struct SelectCfg {
  static constexpr int kStages = 3, kCtasPerSm = D == 64 ? 3 : 2;
  static constexpr int kRing = kSWarps * kStages * Stage<D>::kBytes;  // the stages; before them the keys, after them the merge
  static constexpr int kMerge = kSWarps * 16 * D * 4;
  static_assert(kMerge + 16 * (2 + D) * 4 <= kRing, "the merge of the warps and its result fit in the ring");
};

template <int D>
__global__ void __launch_bounds__(kSThreads, SelectCfg<D>::kCtasPerSm) select_kernel(SelectArgs a) {
  using C = SelectCfg<D>;
  constexpr int kStages = C::kStages;
  extern __shared__ __align__(16) uint8_t dyn[];
  uint32_t *key_s = reinterpret_cast<uint32_t *>(dyn);
  Stage<D> *ring = reinterpret_cast<Stage<D> *>(dyn) + (threadIdx.x >> 5) * kStages;
  float (*red_o)[16][D] = reinterpret_cast<float (*)[16][D]>(dyn);
  int2 *kept = reinterpret_cast<int2 *>(dyn + C::kRing);  // {place in the sequence, page of the pool}
  __shared__ __align__(16) int16_t wgt[2 * D];
  __shared__ float red[kSWarps], red_m[kSWarps][16], red_l[kSWarps][16];
  float (*part)[2 + D] = reinterpret_cast<float (*)[2 + D]>(dyn + C::kMerge);  // this CTA's (max, sum, output) per head
  __shared__ __align__(16) int hist[512];  // 256 bins; at the end every CTA's (max, sum) per head
  __shared__ int warp_sums[kSWarps], pick[3];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  const int unit = blockIdx.x / ranks, h = unit % a.Hkv, b = unit / a.Hkv, g = a.Hq / a.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tid = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const uint16_t *q = a.q + b * a.qs[0] + static_cast<int64_t>(h) * g * a.qs[1];
  float x[16];  // for the weights: requested together with the length
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = i < g && threadIdx.x < D ? bf16_bits_to_float(ld_act_u16(q + i * a.qs[1] + threadIdx.x)) : 0.f;
  const int len = cached_len(a, b), n = (len + (1 << a.page_shift) - 1) >> a.page_shift;
  const int *table = a.table + static_cast<int64_t>(b) * a.M;
  int *sel = a.selected + (static_cast<int64_t>(b) * a.Hkv + h) * a.top;
  auto meet = [&] {  // all CTAs of the cluster
    if (ranks > 1) cluster.sync(); else __syncthreads();
  };
  const int count = min(n, a.top);  // pages kept

  if (n > a.top) {
    // ---- 1. scores: 2 D / 16 lanes per page, 16 codes per lane, 8 pages in flight per
    // lane; a page's number is read into its key's place first ----
    const int chunk = (n + ranks - 1) / ranks, lo = min(n, rank * chunk), hi = min(n, lo + chunk);
    uint32_t *keys = a.keys ? a.keys + (static_cast<int64_t>(b) * a.Hkv + h) * a.M : key_s;
    for (int i = lo + threadIdx.x; i < hi; i += kSThreads) keys[i] = static_cast<uint32_t>(ld_act_i32(table + i));
    query_weights<D>(x, g, wgt, red);
    constexpr int kLanes = 2 * D / 16, kPages = 32 / kLanes, kU = 8;
    const int lanepart = lane % kLanes, sub = lane / kLanes;
    int wv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) wv[i] = reinterpret_cast<const int *>(wgt)[lanepart * 8 + i];
    for (int i0 = lo + warp * kPages; i0 < hi; i0 += kU * kSWarps * kPages) {
      uint4 c[kU];
      float scale[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int i = i0 + u * kSWarps * kPages + sub, p = i < hi ? static_cast<int>(keys[i]) : -1;
        const bool ok = p >= 0 && p < a.P;
        const int64_t at = static_cast<int64_t>(ok ? p : 0) * a.Hkv + h;
        c[u] = ok ? ld_act_v4(a.codes + at * 2 * D + lanepart * 16) : make_uint4(0, 0, 0, 0);
        scale[u] = ok ? ld_act_f32(a.scales + at) : 0.f;
      }
      __syncwarp();  // the numbers have been read
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int i = i0 + u * kSWarps * kPages + sub;
        const int cw[4] = {static_cast<int>(c[u].x), static_cast<int>(c[u].y), static_cast<int>(c[u].z), static_cast<int>(c[u].w)};
        int sum = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum = __dp2a_lo(wv[2 * e], cw[e], sum);
          sum = __dp2a_hi(wv[2 * e + 1], cw[e], sum);
        }
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lanepart == 0 && i < hi)
          keys[i] = score_key(fminf(fmaxf(__fmul_rn(__int2float_rn(sum), scale[u]), -FLT_MAX), FLT_MAX));
      }
    }
    // ---- 2. all keys here, then the pages to keep: the last page, the first one (top > 1)
    // and the best `want` of the others ----
    if (a.keys) __threadfence();
    meet();
    if (!a.keys && ranks > 1) {
      for (int i0 = threadIdx.x; i0 < n; i0 += 4 * kSThreads) {
        uint32_t k[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * kSThreads, r = i / chunk;
          if (i < n && r != rank) k[u] = cluster.map_shared_rank(key_s, r)[i];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * kSThreads;
          if (i < n && i / chunk != rank) key_s[i] = k[u];
        }
      }
      __syncthreads();
    }
    auto key = [&](int i) { return a.keys ? __ldcg(keys + i) : keys[i]; };
    const int lead = a.top > 1 ? 1 : 0, want = a.top - 1 - lead;  // pages lead .. n - 2 compete
    uint32_t prefix = 0, mask = 0;
    int left = want;  // still to be found among the keys that match the prefix
    if (want > 0) {
      // a radix search for the want-th largest key, 8 bits per pass from the first bit in
      // which the keys differ (scores of one sequence share sign and exponent)
      uint32_t all = 0xffffffffu, any = 0;
      for (int i = lead + threadIdx.x; i < n - 1; i += kSThreads) {
        const uint32_t k = key(i);
        all &= k;
        any |= k;
      }
      all = __reduce_and_sync(0xffffffffu, all);
      any = __reduce_or_sync(0xffffffffu, any);
      if (lane == 0) {
        hist[warp] = static_cast<int>(all);
        hist[kSWarps + warp] = static_cast<int>(any);
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kSWarps; ++w) {
        all &= static_cast<uint32_t>(hist[w]);
        any |= static_cast<uint32_t>(hist[kSWarps + w]);
      }
      __syncthreads();
      int bits = 32 - __clz(all ^ any);  // keys agree above this many low bits
      mask = bits == 32 ? 0u : ~((1u << bits) - 1u);
      prefix = all & mask;
      while (bits > 0) {
        const int shift = max(0, bits - 8);
        const uint32_t low = (1u << (bits - shift)) - 1u;
        hist[threadIdx.x] = 0;
        hist[threadIdx.x + 128] = 0;
        __syncthreads();
        for (int i = lead + threadIdx.x; i < n - 1; i += kSThreads) {
          const uint32_t k = key(i);
          if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & low], 1);
        }
        __syncthreads();
        // suffix sums: thread t holds bins 255 - 2 t and 254 - 2 t
        const int bin = 255 - 2 * threadIdx.x, c0 = hist[bin], c1 = hist[bin - 1];
        int v = c0 + c1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += u;
        }
        if (lane == 31) warp_sums[warp] = v;
        __syncthreads();
        for (int w = 0; w < warp; ++w) v += warp_sums[w];
        const int above1 = v - c1, above0 = above1 - c0;  // keys above bin - 1, above bin
        if (above1 >= left && above0 < left) {
          pick[0] = bin;
          pick[1] = left - above0;
          pick[2] = c0;
        } else if (v >= left && above1 < left) {
          pick[0] = bin - 1;
          pick[1] = left - above1;
          pick[2] = c1;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(pick[0]) << shift;
        mask |= low << shift;
        left = pick[1];
        const bool whole = pick[1] == pick[2];  // the bin's keys are all kept
        bits = shift;
        __syncthreads();
        if (whole) break;
      }
    }
    // the list, ascending: keys above the prefix, and the first `left` that match it (the
    // lowest pages of equal keys). A thread takes consecutive pages; one prefix sum gives it
    // how many pages of each kind come before.
    const int per = (n + kSThreads - 1) / kSThreads, i0 = threadIdx.x * per, i1 = min(n, i0 + per);
    auto kind = [&](int i) {  // 2: kept, 1: kept if among the first `left`, 0: not
      if (i == n - 1 || (i == 0 && lead)) return 2;
      if (want <= 0) return 0;
      const uint32_t k = key(i) & mask;
      return k > prefix ? 2 : k == prefix ? 1 : 0;
    };
    int above = 0, equal = 0;
    for (int i = i0; i < i1; ++i) {
      const int k = kind(i);
      above += k == 2;
      equal += k == 1;
    }
    int2 v = make_int2(above, equal);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int ux = __shfl_up_sync(0xffffffffu, v.x, o), uy = __shfl_up_sync(0xffffffffu, v.y, o);
      if (lane >= o) v.x += ux, v.y += uy;
    }
    if (lane == 31) {
      hist[warp] = v.x;
      hist[kSWarps + warp] = v.y;
    }
    __syncthreads();
    for (int w = 0; w < warp; ++w) v.x += hist[w], v.y += hist[kSWarps + w];
    v.x -= above;
    v.y -= equal;
    for (int i = i0; i < i1; ++i) {
      const int k = kind(i);
      if (k == 2 || (k == 1 && v.y < left)) {
        const int to = v.x + min(v.y, left);
        kept[to] = make_int2(i, ld_act_i32(table + i));
        if (rank == 0) sel[to] = i;
      }
      v.x += k == 2;
      v.y += k == 1;
    }
    // no CTA may reuse its keys (the ring) while another one copies them
    meet();
  } else {
    for (int i = threadIdx.x; i < a.top; i += kSThreads) {
      if (i < n) kept[i] = make_int2(i, ld_act_i32(table + i));
      if (rank == 0) sel[i] = i < n ? i : -1;
    }
    __syncthreads();
  }

  // ---- 3. attention over the kept pages' blocks: block i to warp i % (ranks * kSWarps) ----
  WarpAttn<D> at;
  at.clear();
  at.load_q(gid < g ? q + gid * a.qs[1] : nullptr, gid + 8 < g ? q + (gid + 8) * a.qs[1] : nullptr);
  const int bshift = a.page_shift - 4, blocks = count << bshift, step = ranks * kSWarps;
  auto rows = [&](int i, int2 &e) {  // valid tokens of block i
    e = kept[i >> bshift];
    const int in = min(16, len - (e.x << a.page_shift) - ((i & ((1 << bshift) - 1)) << 4));
    return e.y >= 0 && e.y < a.P ? in : 0;
  };
  auto request = [&](int i, int stage) {
    if (i < blocks) {
      int2 e;
      const int valid = rows(i, e);
      const int64_t at0 = valid > 0 ? (((static_cast<int64_t>(e.y) * a.Hkv + h) << a.page_shift) +
                                       ((i & ((1 << bshift) - 1)) << 4)) * D : 0;
      ring[stage].load(a.k + at0, a.v + at0, D, D, valid);
    }
    cp_async_commit();
  };
  const int first = rank * kSWarps + warp;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) request(first + s * step, s);
  int stage = 0;
  for (int i = first; i < blocks; i += step) {
    cp_async_wait<kStages - 2>();
    __syncwarp();  // the block is here, and every lane is done with the stage refilled next
    request(i + (kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1);
    int2 e;
    const int valid = rows(i, e);
    if (valid > 0) {
      const uint32_t see[2] = {0xffffu >> (16 - valid), 0xffffu >> (16 - valid)};
      at.step(ring[stage], a.scale_log2, see);
    }
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  at.finish();
  __syncthreads();  // every warp is done with the ring

  // ---- 4. the warps of this CTA, then the CTAs of the cluster ----
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
  for (int idx = threadIdx.x; idx < g * D; idx += kSThreads) {
    const int r = idx / D, d = idx % D;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < kSWarps; ++w) M = fmaxf(M, red_m[w][r]);
#pragma unroll
    for (int w = 0; w < kSWarps; ++w) {
      const float f = rescale(red_m[w][r], M);
      L += red_l[w][r] * f;
      O += red_o[w][r][d] * f;
    }
    if (d == 0) {
      part[r][0] = M;
      part[r][1] = L;
    }
    part[r][2 + d] = O;
  }
  meet();
  // rank r joins every ranks-th group of 128 values; all reads of other CTAs' memory are
  // issued before any is used
  float2 (*ml)[16] = reinterpret_cast<float2 (*)[16]>(hist);  
  static_assert(sizeof(hist) >= 16 * 16 * sizeof(float2), "room for every CTA's (max, sum)");
  for (int i = threadIdx.x; i < ranks * g; i += kSThreads) {
    const float *o = cluster.map_shared_rank(&part[i % g][0], i / g);
    ml[i / g][i % g] = make_float2(o[0], o[1]);
  }
  __syncthreads();
  for (int idx = rank * kSThreads + threadIdx.x; idx < g * D; idx += ranks * kSThreads) {
    const int r = idx / D, d = idx % D;
    float o[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) o[c] = c < ranks ? cluster.map_shared_rank(&part[r][0], c)[2 + d] : 0.f;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int c = 0; c < ranks; ++c) M = fmaxf(M, ml[c][r].x);
#pragma unroll
    for (int c = 0; c < 16; ++c)
      if (c < ranks) {
        const float f = rescale(ml[c][r].x, M);
        L += ml[c][r].y * f;
        O += o[c] * f;
      }
    a.out[b * a.os[0] + (static_cast<int64_t>(h) * g + r) * a.os[1] + d] = float_to_bf16_bits(normalised(O, L));
  }
  meet();  // no CTA leaves while another one reads its part
}

}  // namespace iron

using namespace iron;

// Sequences whose keys do not fit in the ring's shared memory keep them in the workspace.
static bool keys_in_workspace(int head_dim, int max_pages) {
  return static_cast<int64_t>(max_pages) * 4 > (head_dim == 128 ? SelectCfg<128>::kRing : SelectCfg<64>::kRing);
}

// CTAs of a (sequence, kv head): clusters as large as leave every warp a block of the kept
// pages, while all CTAs run at once (what is done once per CTA takes as long as some 100 KB
// of pages: at 16 sequences, head dim 128, clusters of 2 took 60 us, of 8 89 us on B200).
static int select_ranks(int units, int top, int page, int ctas_per_sm) {
  const int64_t blocks = static_cast<int64_t>(top) * page / 16;
  int r = 16;
  while (r > 1 && (static_cast<int64_t>(units) * r > static_cast<int64_t>(ctas_per_sm) * sm_count() || blocks < r * kSWarps)) r /= 2;
  return r;
}

template <int D>
static int launch_select(const SelectArgs &a, int B, int page, cudaStream_t s) {
  const int ranks = select_ranks(B * a.Hkv, a.top, page, SelectCfg<D>::kCtasPerSm);
  const int list = (a.top < a.M ? a.top : a.M) * static_cast<int>(sizeof(int2));
  static PerDeviceOnce once;
  const int st = once.run([] {
    cudaError_t e = cudaFuncSetAttribute(select_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         SelectCfg<D>::kRing + kMaxTop * static_cast<int>(sizeof(int2)));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(select_kernel<D>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return call_status(e);
  });
  if (st != IRON_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(B * a.Hkv * ranks);
  cfg.blockDim = dim3(kSThreads);
  cfg.dynamicSmemBytes = SelectCfg<D>::kRing + list;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return call_status(cudaLaunchKernelEx(&cfg, select_kernel<D>, a));
}

extern "C" size_t iron_page_select_attn_workspace_bytes(int batch, int num_heads, int kv_heads, int head_dim,
                                                        int max_pages, int top_pages, int page_size) {
  if (batch <= 0 || num_heads <= 0 || kv_heads <= 0 || max_pages <= 0 || top_pages <= 0 || page_size <= 0) return 0;
  return keys_in_workspace(head_dim, max_pages) ? static_cast<size_t>(batch) * kv_heads * max_pages * 4 : 16;
}

extern "C" int iron_page_select_attn(const iron_page_pool *c, const uint16_t *q, uint16_t *out, int32_t *selected,
                                     int num_heads, int top_pages, const int64_t *q_strides,
                                     const int64_t *out_strides, float scale, void *workspace, size_t workspace_bytes,
                                     unsigned flags, void *stream) {
  (void)flags;
  const int chk = pool_geometry_check(c);
  if (chk != IRON_OK) return chk;
  if (!c->lens || !c->codes || !q || !out || !selected || !q_strides || !out_strides || !workspace) return IRON_ERR_NULL;
  if (c->layers != 1 || num_heads <= 0 || num_heads % c->kv_heads || top_pages <= 0) return IRON_ERR_SHAPE;
  if (c->slots > 65535) return IRON_ERR_SHAPE;
  if (num_heads / c->kv_heads > 16 || top_pages > kMaxTop) return IRON_ERR_UNSUPPORTED;
  if (!aligned16(q)) return IRON_ERR_ALIGN;
  for (int i = 0; i < 2; ++i)
    if (q_strides[i] % 8 || out_strides[i] % 8) return IRON_ERR_ALIGN;
  if (workspace_bytes < iron_page_select_attn_workspace_bytes(c->slots, num_heads, c->kv_heads, c->head_dim,
                                                              c->max_pages, top_pages, c->page_size))
    return IRON_ERR_WORKSPACE;
  SelectArgs a = {};
  a.q = q;
  a.k = c->k;
  a.v = c->v;
  a.codes = c->codes;
  a.scales = c->scales;
  a.table = c->page_table;
  a.lens = c->lens;
  a.out = out;
  a.selected = selected;
  a.keys = keys_in_workspace(c->head_dim, c->max_pages) ? static_cast<uint32_t *>(workspace) : nullptr;
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = q_strides[i];
    a.os[i] = out_strides[i];
  }
  a.Hq = num_heads;
  a.Hkv = c->kv_heads;
  a.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  a.M = c->max_pages;
  a.P = c->num_pages;
  a.top = top_pages;
  a.scale_log2 = scale * kLog2e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c->head_dim == 128 ? launch_select<128>(a, c->slots, c->page_size, s)
                            : launch_select<64>(a, c->slots, c->page_size, s);
}
