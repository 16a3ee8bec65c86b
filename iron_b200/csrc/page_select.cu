// Decode attention over the pages that a cheap score selects.
//
// For few (sequence, kv head) units one kernel, a cluster of CTAs per unit:
//   1. each CTA scores its share of the pages from their summaries;
//   2. after a cluster barrier every CTA has all keys (its own and, through distributed
//      shared memory, the others') and picks the same pages;
//   3. the kept pages' 16-token blocks are dealt out to the cluster's warps;
//   4. each CTA merges its warps, and the cluster merges its CTAs, each rank a share of the
//      output (fixed order throughout).
// With more units clusters run in waves of which the last is partly empty. Where that costs
// more than two further launches, steps 1 and 2 are a kernel of their own (one CTA per unit, little
// shared memory), the kept blocks of all units are cut into as many equal pieces as CTAs
// run at once, and a third kernel joins the units that were cut.
// The score is a sum of products of whole numbers: over the heads, q8 meets hi8 where it is
// positive and lo8 where it is negative, = hi8 . (sum of the positive q8) + lo8 . (sum of
// the negative q8), so one 16-bit weight vector of 2 D values serves the whole query group,
// and dp2a (two 16 x 8 bit products per instruction) sums it exactly.
//
// Bound: HBM (summaries of all pages, K and V of the kept ones) for batches, the latency of
// the four steps for single sequences. B200, 64 sequences of 32768 tokens, 64 pages kept:
// 240 us with a kernel per step and one block per warp in flight, 141 as clusters, 122 in
// pieces (with 3 stages in 3 CTAs per SM 8 us more, with 10 in 1 15 more; without any
// arithmetic on the blocks 10 less).
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
  float *ws;       // workspace: partials of cut units, two per CTA: O [16][D], then (max, sum) [16]
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

// An fp32 score as an unsigned key of the same order (-0 would come before 0: the caller adds 0,
// which makes 0 of it).
__device__ __forceinline__ uint32_t score_key(float s) {
  const uint32_t u = __float_as_uint(s);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int D>
struct SelectCfg {
  static constexpr int kStages = D == 64 ? 5 : 3, kCtasPerSm = 2;
  static constexpr int kRing = kSWarps * kStages * Stage<D>::kBytes;  // the stages; before them the keys, after them the merge
  static constexpr int kMerge = kSWarps * 16 * D * 4;
  static_assert(kMerge + 16 * (2 + D) * 4 <= kRing, "the merge of the warps and its result fit in the ring");
};

// Attention of one CTA over blocks first, first + step, ... < blocks (a warp each) of the
// pages in `kept`: block i lies in page kept[i >> bshift].
template <int D>
__device__ __forceinline__ void attend_blocks(const SelectArgs &a, WarpAttn<D> &at, Stage<D> *ring, const int2 *kept,
                                              int len, int h, int first, int step, int blocks) {
  constexpr int kStages = SelectCfg<D>::kStages;
  const int bshift = a.page_shift - 4;
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
}

// The warps' results into shared memory; merged<D>(r, d) is then the CTA's.
template <int D>
struct WarpMerge {
  float (*o)[16][D];
  float (*m)[16], (*l)[16];
  __device__ __forceinline__ void put(const WarpAttn<D> &at) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tid = lane & 3;
    if (tid == 0) {
      m[warp][gid] = at.m[0];
      m[warp][gid + 8] = at.m[1];
      l[warp][gid] = at.l[0];
      l[warp][gid + 8] = at.l[1];
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      *reinterpret_cast<float2 *>(&o[warp][gid][8 * j + 2 * tid]) = make_float2(at.o[j][0], at.o[j][1]);
      *reinterpret_cast<float2 *>(&o[warp][gid + 8][8 * j + 2 * tid]) = make_float2(at.o[j][2], at.o[j][3]);
    }
  }
  __device__ __forceinline__ void get(int r, int d, float &M, float &L, float &O) const {
    M = -INFINITY;
    L = O = 0.f;
#pragma unroll
    for (int w = 0; w < kSWarps; ++w) M = fmaxf(M, m[w][r]);
#pragma unroll
    for (int w = 0; w < kSWarps; ++w) {
      const float f = rescale(m[w][r], M);
      L += l[w][r] * f;
      O += o[w][r][d] * f;
    }
  }
};

// kAttend: all four steps; else the choice alone (its list goes to `selected`).
template <int D, bool kAttend>
__global__ void __launch_bounds__(kSThreads, kAttend ? SelectCfg<D>::kCtasPerSm : 4) select_kernel(SelectArgs a) {
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

  // The same for all threads, whatever length each has read: nothing may write it meanwhile, but
  // if someone does, the barriers that follow must still match (B200, one sequence of 8192
  // tokens: 12.4 us, 12.1 without).
  const bool choose = __syncthreads_or(n > a.top);
  if (choose) {
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
          keys[i] = score_key(fminf(fmaxf(__fmul_rn(__int2float_rn(sum), scale[u]) + 0.f, -FLT_MAX), FLT_MAX));
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
        const int to = min(v.x + min(v.y, left), count - 1);
        if constexpr (kAttend) kept[to] = make_int2(i, ld_act_i32(table + i));
        if (rank == 0) sel[to] = i;
      }
      v.x += k == 2;
      v.y += k == 1;
    }
    // no CTA may reuse its keys (the ring), or leave, while another one copies them
    meet();
  } else {
    for (int i = threadIdx.x; i < a.top; i += kSThreads) {
      if constexpr (kAttend)
        if (i < n) kept[i] = make_int2(i, ld_act_i32(table + i));
      if (rank == 0) sel[i] = i < n ? i : -1;
    }
    __syncthreads();
  }

  if constexpr (!kAttend) return;

  // ---- 3. attention over the kept pages' blocks: block i to warp i % (ranks * kSWarps) ----
  WarpAttn<D> at;
  at.clear();
  at.load_q(gid < g ? q + gid * a.qs[1] : nullptr, gid + 8 < g ? q + (gid + 8) * a.qs[1] : nullptr);
  attend_blocks<D>(a, at, ring, kept, len, h, rank * kSWarps + warp, ranks * kSWarps, count << (a.page_shift - 4));
  __syncthreads();  // every warp is done with the ring

  // ---- 4. the warps of this CTA, then the CTAs of the cluster ----
  WarpMerge<D> merge{red_o, red_m, red_l};
  merge.put(at);
  __syncthreads();
  for (int idx = threadIdx.x; idx < g * D; idx += kSThreads) {
    const int r = idx / D, d = idx % D;
    float M, L, O;
    merge.get(r, d, M, L, O);
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
  // Every CTA meets the others as often as one that chose: CTAs that read different lengths
  // (someone writes them meanwhile, against the rules) get wrong results, but none leaves while
  // another one still reads its shared memory. (A table of `top` pages leaves no CTA a choice;
  // 300 tokens in a table of 1000 pages: 6.5 us, 5.8 without.)
  if (ranks > 1 && !choose && a.M > a.top) {
    meet();
    meet();
  }
}

// Pieces: `per` blocks per unit (those past a unit's own do nothing), cut into gridDim.x
// equal parts.
template <int D>
__global__ void __launch_bounds__(kSThreads, SelectCfg<D>::kCtasPerSm) select_attend_kernel(SelectArgs a, int units, int per) {
  using C = SelectCfg<D>;
  extern __shared__ __align__(16) uint8_t dyn[];
  Stage<D> *ring = reinterpret_cast<Stage<D> *>(dyn) + (threadIdx.x >> 5) * C::kStages;
  int2 *kept = reinterpret_cast<int2 *>(dyn + C::kRing);
  __shared__ float red_m[kSWarps][16], red_l[kSWarps][16];
  WarpMerge<D> merge{reinterpret_cast<float (*)[16][D]>(dyn), red_m, red_l};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, g = a.Hq / a.Hkv, bshift = a.page_shift - 4;
  const int64_t total = static_cast<int64_t>(units) * per;
  int64_t w = total * blockIdx.x / gridDim.x;
  const int64_t w_end = total * (blockIdx.x + 1) / gridDim.x;
  pdl_launch_dependents();
  pdl_wait();
  while (w < w_end) {
    const int unit = static_cast<int>(w / per), b0 = static_cast<int>(w % per);
    const int b1 = static_cast<int>(min(static_cast<int64_t>(per), b0 + (w_end - w)));
    w += b1 - b0;
    const int h = unit % a.Hkv, b = unit / a.Hkv;
    const int len = cached_len(a, b), n = (len + (1 << a.page_shift) - 1) >> a.page_shift;
    const int blocks = min(b1, min(n, a.top) << bshift);
    const int *sel = a.selected + static_cast<int64_t>(unit) * a.top, *table = a.table + static_cast<int64_t>(b) * a.M;
    for (int i = (b0 >> bshift) + threadIdx.x; i < (blocks + (1 << bshift) - 1) >> bshift; i += kSThreads) {
      // (a place outside the sequence: the length has changed since the choice)
      const int at = ld_act_i32(sel + i);
      kept[i] = at >= 0 && at < n ? make_int2(at, ld_act_i32(table + at)) : make_int2(0, -1);
    }
    const uint16_t *q = a.q + b * a.qs[0] + static_cast<int64_t>(h) * g * a.qs[1];
    WarpAttn<D> at;
    at.clear();
    at.load_q(gid < g ? q + gid * a.qs[1] : nullptr, gid + 8 < g ? q + (gid + 8) * a.qs[1] : nullptr);
    __syncthreads();  // the list is there, and the merge before is done with the ring
    attend_blocks<D>(a, at, ring, kept, len, h, b0 + warp, kSWarps, blocks);
    __syncthreads();
    merge.put(at);
    __syncthreads();
    const bool whole = b0 == 0 && b1 == per;
    float *part = a.ws + (static_cast<int64_t>(blockIdx.x) * 2 + (b0 == 0 ? 1 : 0)) * 16 * (D + 2);
    for (int idx = threadIdx.x; idx < g * D; idx += kSThreads) {
      const int r = idx / D, d = idx % D;
      float M, L, O;
      merge.get(r, d, M, L, O);
      if (whole) {
        a.out[b * a.os[0] + (static_cast<int64_t>(h) * g + r) * a.os[1] + d] = float_to_bf16_bits(normalised(O, L));
      } else {
        if (d == 0) {
          part[16 * D + 2 * r] = M;
          part[16 * D + 2 * r + 1] = L;
        }
        part[r * D + d] = O;
      }
    }
    __syncthreads();  // kept and the merge may be used again
  }
}

// Joins the pieces of one unit, in order; a unit that one piece held whole has none.
template <int D>
__global__ void __launch_bounds__(256) select_join_kernel(SelectArgs a, int units, int per, int pieces) {
  pdl_launch_dependents();
  pdl_wait();
  const int unit = blockIdx.x, h = unit % a.Hkv, b = unit / a.Hkv, g = a.Hq / a.Hkv;
  const int64_t total = static_cast<int64_t>(units) * per, w = static_cast<int64_t>(unit) * per;
  const int c0 = static_cast<int>(((w + 1) * pieces - 1) / total), c1 = static_cast<int>(((w + per) * pieces - 1) / total);
  if (c0 == c1) return;
  for (int idx = threadIdx.x; idx < g * D; idx += 256) {
    const int r = idx / D, d = idx % D;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int c = c0; c <= c1; c += 4) {
      float2 ml[4];
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = c + i <= c1;
        const float *part = a.ws + (static_cast<int64_t>(in ? c + i : c0) * 2 + (c + i == c0 || !in ? 1 : 0)) * 16 * (D + 2);
        ml[i] = __ldcg(reinterpret_cast<const float2 *>(part + 16 * D + 2 * r));
        o[i] = __ldcg(part + r * D + d);
        if (!in) ml[i] = make_float2(-INFINITY, 0.f), o[i] = 0.f;
      }
      float top = M;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i].x);
      const float f0 = rescale(M, top);
      M = top;
      L *= f0;
      O *= f0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = rescale(ml[i].x, M);
        L += ml[i].y * f;
        O += o[i] * f;
      }
    }
    a.out[b * a.os[0] + (static_cast<int64_t>(h) * g + r) * a.os[1] + d] = float_to_bf16_bits(normalised(O, L));
  }
}

}  // namespace iron

using namespace iron;

// Sequences whose keys do not fit in the ring's shared memory keep them in the workspace.
static bool keys_in_workspace(int head_dim, int max_pages) {
  return static_cast<int64_t>(max_pages) * 4 > (head_dim == 128 ? SelectCfg<128>::kRing : SelectCfg<64>::kRing);
}

// The form with the least time, in bytes that a CTA could move meanwhile at its share of the
// memory's bandwidth (48 us per MB; summaries go at half of it). Clusters go in waves of
// CTAs that run at once; each CTA takes 190 KB for what is done once per CTA, 5 KB more per
// rank that it meets, and its part of the unit's bytes. Clusters of 16 leave about a quarter
// of the SMs idle. Pieces take 450 KB for three kernels and the joins, a unit's summaries
// in one CTA, twice as slowly (nothing else runs), and an even share of all pages. B200, us,
// pieces / clusters: 32768 tokens, 64 pages of 64, head dim 64: 128 units 48 / 42, 152
// 53 / 62, 256 73 / 68, 384 97 / 116, 512 121 / 128; head dim 128, 32 pages: 64 units 44 / 27,
// 152 75 / 65, 256 94 / 79, 384 118 / 128, 512 139 / 142; 8192 tokens, 16 pages: 256 units
// 27 / 22, 384 35 / 43. Cluster sizes: 128 units of 32768 tokens, 32 pages, head dim 128: 1 CTA
// 61, 2 41, 4 53; 8 units of 8192 tokens, 16 pages: 1 CTA 17, 8 11.9, 16 12.6; 16 units, 1024
// pages: 8 CTAs 105, 16 121.
struct SelectPlan {
  bool pieces;
  int ranks;  // CTAs of a unit's cluster
};
static SelectPlan select_plan(int64_t units, int top, int page, int head_dim, int max_pages, int ctas) {
  const int64_t blocks = static_cast<int64_t>(top < max_pages ? top : max_pages) * page / 16;
  const int64_t pages = blocks * 16 * head_dim * 4, summaries = static_cast<int64_t>(max_pages) * (2 * head_dim + 4);
  SelectPlan best = {true, 1};
  int64_t least = 450 * 1024 + (units > ctas ? summaries * units / ctas : summaries) + 3 * summaries + pages * units / ctas;
  for (int r = 1; r <= 16 && (r == 1 || blocks >= r * kSWarps); r *= 2) {
    const int fit = r == 16 ? ctas * 3 / 4 : ctas;
    const int64_t cost = ((units * r + fit - 1) / fit) * (190 * 1024 + 5 * 1024 * r + (pages + 2 * summaries) / r);
    if (cost < least) {
      best = {false, r};
      least = cost;
    }
  }
  return best;
}

template <int D>
static int launch_select(const SelectArgs &a, int B, int page, cudaStream_t s) {
  using C = SelectCfg<D>;
  const int ctas = C::kCtasPerSm * sm_count(), units = B * a.Hkv, longest = a.top < a.M ? a.top : a.M;
  const auto [pieces, ranks] = select_plan(units, a.top, page, D, a.M, ctas);
  const int list = longest * static_cast<int>(sizeof(int2));
  static PerDeviceOnce once;
  const int st = once.run([] {
    const int most = C::kRing + kMaxTop * static_cast<int>(sizeof(int2));
    cudaError_t e = cudaFuncSetAttribute(select_kernel<D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(select_kernel<D, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(select_kernel<D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kRing);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(select_attend_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    return call_status(e);
  });
  if (st != IRON_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * ranks);
  cfg.blockDim = dim3(kSThreads);
  cfg.dynamicSmemBytes = pieces ? (a.keys ? 0 : a.M * sizeof(uint32_t)) : static_cast<size_t>(C::kRing + list);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (!pieces) return call_status(cudaLaunchKernelEx(&cfg, select_kernel<D, true>, a));
  int e = call_status(cudaLaunchKernelEx(&cfg, select_kernel<D, false>, a));
  if (e != IRON_OK) return e;
  const int per = longest * (page / 16);
  const int64_t total = static_cast<int64_t>(units) * per;
  const int grid = static_cast<int>(total < ctas ? total : ctas);
  e = launch(select_attend_kernel<D>, dim3(grid), dim3(kSThreads), C::kRing + list, s, true, a, units, per);
  if (e != IRON_OK) return e;
  return launch(select_join_kernel<D>, dim3(units), dim3(256), 0, s, true, a, units, per, grid);
}

// The workspace: partials of cut units, then the keys that do not fit in shared memory.
static size_t select_partials(int64_t units, int top, int page, int head_dim, int max_pages) {
  const int ctas = (head_dim == 128 ? SelectCfg<128>::kCtasPerSm : SelectCfg<64>::kCtasPerSm) * sm_count();
  return select_plan(units, top, page, head_dim, max_pages, ctas).pieces
             ? static_cast<size_t>(ctas) * 2 * 16 * (head_dim + 2) * sizeof(float)
             : 0;
}

extern "C" size_t iron_page_select_attn_workspace_bytes(int batch, int num_heads, int kv_heads, int head_dim,
                                                        int max_pages, int top_pages, int page_size) {
  if (batch <= 0 || num_heads <= 0 || kv_heads <= 0 || max_pages <= 0 || top_pages <= 0 || page_size <= 0) return 0;
  return 16 + select_partials(static_cast<int64_t>(batch) * kv_heads, top_pages, page_size, head_dim, max_pages) +
         (keys_in_workspace(head_dim, max_pages) ? static_cast<size_t>(batch) * kv_heads * max_pages * 4 : 0);
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
  if (!aligned16(q) || !aligned16(workspace)) return IRON_ERR_ALIGN;
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
  a.ws = static_cast<float *>(workspace);
  a.keys = keys_in_workspace(c->head_dim, c->max_pages)
               ? reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(workspace) +
                                              select_partials(static_cast<int64_t>(c->slots) * c->kv_heads, top_pages,
                                                              c->page_size, c->head_dim, c->max_pages))
               : nullptr;
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
