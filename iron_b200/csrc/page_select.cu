// Decode attention over the pages that a cheap score selects.
//
// Four steps per (sequence, kv head): score every page from its summary, pick the pages,
// attend to them (split over CTAs), join the splits. The score is a sum of products of
// whole numbers: over the heads, q8 meets hi8 where it is positive and lo8 where it is
// negative, = hi8 . (sum of the positive q8) + lo8 . (sum of the negative q8), so one 16-bit weight vector of 2 D values serves the
// whole query group, and dp2a (two 16 x 8 bit products per instruction) sums it exactly.
#include <cfloat>

#include "paged.cuh"

namespace iron {

constexpr int kSWarps = 4;
constexpr int kPickThreads = 256;

struct SelectArgs {
  const uint16_t *q, *k, *v;
  const int8_t *codes;
  const float *scales;
  const int *table, *lens;
  uint16_t *out;
  int *selected;
  float *scores;  // workspace [B, Hkv, M]
  float *ws;      // workspace [B, Hq, splits, 2 + D]
  int64_t qs[2], os[2];
  int Hq, Hkv, page_shift, M, P, top, splits;
  float scale_log2;
};

__device__ __forceinline__ int cached_len(const SelectArgs &a, int b) {
  return min(max(ld_act_i32(a.lens + b), 0), a.M << a.page_shift);
}
__device__ __forceinline__ int cached_pages(const SelectArgs &a, int b) {
  return (cached_len(a, b) + (1 << a.page_shift) - 1) >> a.page_shift;
}

// The query group's weights: wgt[0 .. D) the sums of its negative q8 (they meet lo8),
// wgt[D .. 2 D) of its positive ones (they meet hi8). q8 = rint(q / a * 127) with IEEE
// division, |sum| <= 16 * 127.
template <int D, int kThreads>
__device__ __forceinline__ void query_weights(const SelectArgs &a, int b, int h, int16_t *wgt, float *red) {
  const int g = a.Hq / a.Hkv;
  const uint16_t *q = a.q + b * a.qs[0] + static_cast<int64_t>(h) * g * a.qs[1];
  float top = 0.f;
  bool nan = false;
  for (int i = threadIdx.x; i < g * D; i += kThreads) {
    const float x = fabsf(bf16_bits_to_float(ld_act_u16(q + i / D * a.qs[1] + i % D)));
    nan |= x != x;
    top = fmaxf(top, x);
  }
  top = warp_max(nan ? INFINITY : top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, red[w]);
  const bool fine = top > 0.f && top < INFINITY;
  for (int d = threadIdx.x; d < D; d += kThreads) {
    int neg = 0, pos = 0;
    for (int i = 0; i < g; ++i) {
      const float x = bf16_bits_to_float(ld_act_u16(q + i * a.qs[1] + d));
      const int q8 = fine ? static_cast<int>(rintf(__fmul_rn(__fdiv_rn(x, top), 127.f))) : 0;
      neg += min(q8, 0);
      pos += max(q8, 0);
    }
    wgt[d] = static_cast<int16_t>(neg);
    wgt[D + d] = static_cast<int16_t>(pos);
  }
  __syncthreads();
}

// Scores of the pages first, first + step, ... of one (sequence, kv head): 2 D / 16 lanes
// per page, 16 codes per lane.
template <int D>
__global__ void __launch_bounds__(32 * kSWarps) select_score_kernel(SelectArgs a) {
  __shared__ __align__(16) int16_t wgt[2 * D];
  __shared__ float red[kSWarps];
  const int h = blockIdx.y, b = blockIdx.z;
  pdl_launch_dependents();
  pdl_wait();
  const int n = cached_pages(a, b);
  if (n <= a.top || static_cast<int>(blockIdx.x) * kSWarps >= n) return;  // all pages are kept
  query_weights<D, 32 * kSWarps>(a, b, h, wgt, red);
  constexpr int kLanes = 2 * D / 16, kPages = 32 / kLanes;
  const int lane = threadIdx.x & 31, part = lane % kLanes, sub = lane / kLanes;
  int wv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) wv[i] = reinterpret_cast<const int *>(wgt)[part * 8 + i];
  const int *table = a.table + static_cast<int64_t>(b) * a.M;
  float *scores = a.scores + (static_cast<int64_t>(b) * a.Hkv + h) * a.M;
  const int warp = blockIdx.x * kSWarps + (threadIdx.x >> 5), warps = gridDim.x * kSWarps;
  for (int i0 = warp * kPages; i0 < n; i0 += warps * kPages) {
    const int i = i0 + sub;
    int p = i < n ? ld_act_i32(table + i) : -1;
    const bool ok = p >= 0 && p < a.P;
    const int64_t at = static_cast<int64_t>(ok ? p : 0) * a.Hkv + h;
    const uint4 c = ok ? ld_act_v4(a.codes + at * 2 * D + part * 16) : make_uint4(0, 0, 0, 0);
    const float scale = ok ? ld_act_f32(a.scales + at) : 0.f;
    const int cw[4] = {static_cast<int>(c.x), static_cast<int>(c.y), static_cast<int>(c.z), static_cast<int>(c.w)};
    int sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sum = __dp2a_lo(wv[2 * e], cw[e], sum);
      sum = __dp2a_hi(wv[2 * e + 1], cw[e], sum);
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (part == 0 && i < n)
      scores[i] = fminf(fmaxf(__fmul_rn(__int2float_rn(sum), scale), -FLT_MAX), FLT_MAX);
  }
}

// An fp32 score as an unsigned key of the same order.
__device__ __forceinline__ uint32_t score_key(float s) {
  const uint32_t u = __float_as_uint(s);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA per (sequence, kv head): the pages to keep, ascending. The last page and (top >
// 1) the first are kept; of the others the `want` best, found by a radix search for the
// want-th largest key, 8 bits per pass; of equal keys the lowest pages.
__global__ void __launch_bounds__(kPickThreads) select_pick_kernel(SelectArgs a) {
  __shared__ int hist[256], warp_sums[kPickThreads / 32], pick[2];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int n = cached_pages(a, b);
  int *sel = a.selected + (static_cast<int64_t>(b) * a.Hkv + h) * a.top;
  if (n <= a.top) {
    for (int i = threadIdx.x; i < a.top; i += kPickThreads) sel[i] = i < n ? i : -1;
    return;
  }
  const int lead = a.top > 1 ? 1 : 0, want = a.top - 1 - lead;  // pages lead .. n - 2 compete
  const float *scores = a.scores + (static_cast<int64_t>(b) * a.Hkv + h) * a.M;
  uint32_t prefix = 0, mask = 0;
  int left = want;  // still to be found among the keys that match the prefix
  if (want > 0)
    for (int shift = 24; shift >= 0; shift -= 8) {
      hist[threadIdx.x] = 0;
      __syncthreads();
      for (int i = lead + threadIdx.x; i < n - 1; i += kPickThreads) {
        const uint32_t k = score_key(ld_act_f32(scores + i));
        if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & 255u], 1);
      }
      __syncthreads();
      // suffix sums: thread t holds bin 255 - t
      const int bin = 255 - threadIdx.x, c = hist[bin];
      int v = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (lane == 31) warp_sums[warp] = v;
      __syncthreads();
      for (int w = 0; w < warp; ++w) v += warp_sums[w];
      if (v >= left && v - c < left) {
        pick[0] = bin;
        pick[1] = left - (v - c);
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(pick[0]) << shift;
      mask |= 255u << shift;
      left = pick[1];
      __syncthreads();
    }
  // keys above `prefix`, and the first `left` equal to it, in page order
  int out = 0, ties = 0;
  for (int i0 = 0; i0 < n; i0 += kPickThreads) {
    const int i = i0 + threadIdx.x;
    const bool forced = i == n - 1 || (i == 0 && lead);
    const bool in = want > 0 && i < n && !forced && i >= lead;
    const uint32_t k = in ? score_key(ld_act_f32(scores + i)) : 0;
    const unsigned eq = __ballot_sync(0xffffffffu, in && k == prefix);
    if (lane == 0) warp_sums[warp] = __popc(eq);
    __syncthreads();
    int rank = ties + __popc(eq & ((1u << lane) - 1u));
    for (int w = 0; w < kPickThreads / 32; ++w) {
      if (w < warp) rank += warp_sums[w];
      ties += warp_sums[w];
    }
    __syncthreads();
    const bool keep = (forced && i < n) || (in && (k > prefix || (k == prefix && rank < left)));
    const unsigned m = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) warp_sums[warp] = __popc(m);
    __syncthreads();
    int at = out + __popc(m & ((1u << lane) - 1u));
    for (int w = 0; w < kPickThreads / 32; ++w) {
      if (w < warp) at += warp_sums[w];
      out += warp_sums[w];
    }
    __syncthreads();
    if (keep) sel[at] = i;
  }
}

// Split x of the kept pages' 16-token blocks of one (sequence, kv head); a warp takes every
// fourth block of the split.
template <int D>
__global__ void __launch_bounds__(32 * kSWarps) select_attend_kernel(SelectArgs a) {
  using Attn = WarpAttn<D>;
  constexpr int kVBytes = kSWarps * 16 * Attn::kVStride * 2, kOBytes = kSWarps * 16 * D * 4;
  __shared__ __align__(16) uint8_t smem[kVBytes > kOBytes ? kVBytes : kOBytes];
  __shared__ float red_m[kSWarps][16], red_l[kSWarps][16];
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z, g = a.Hq / a.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tid = lane & 3;
  uint16_t *vs = reinterpret_cast<uint16_t *>(smem) + warp * 16 * Attn::kVStride;
  float (*red_o)[16][D] = reinterpret_cast<float (*)[16][D]>(smem);
  pdl_launch_dependents();
  pdl_wait();
  const int len = cached_len(a, b), kept = min(cached_pages(a, b), a.top), bpp = (1 << a.page_shift) / 16;
  const int *sel = a.selected + (static_cast<int64_t>(b) * a.Hkv + h) * a.top;
  const int *table = a.table + static_cast<int64_t>(b) * a.M;
  const uint16_t *q = a.q + b * a.qs[0] + static_cast<int64_t>(h) * g * a.qs[1];
  Attn at;
  at.clear();
  at.load_q(gid < g ? q + gid * a.qs[1] : nullptr, gid + 8 < g ? q + (gid + 8) * a.qs[1] : nullptr);
  const int blocks = kept * bpp;
  const int lo = static_cast<int>(static_cast<int64_t>(blocks) * split / a.splits);
  const int hi = static_cast<int>(static_cast<int64_t>(blocks) * (split + 1) / a.splits);
  WarpBlock<D> blk;
  for (int i = lo + warp; i < hi; i += kSWarps) {
    const int page = ld_act_i32(sel + i / bpp), r = i % bpp * 16;
    const int n = min(16, len - (page << a.page_shift) - r);
    const int p = ld_act_i32(table + page);
    if (n <= 0 || p < 0 || p >= a.P) continue;
    const int64_t at0 = ((static_cast<int64_t>(p) * a.Hkv + h) << a.page_shift) + r;
    blk.load(a.k + at0 * D, a.v + at0 * D, D, D, n);
    const uint32_t see[2] = {0xffffu >> (16 - n), 0xffffu >> (16 - n)};
    at.stage_v(blk, vs);
    at.step(blk.k, vs, a.scale_log2, see);
  }
  at.finish();
  __syncthreads();
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
  for (int idx = threadIdx.x; idx < g * D; idx += 32 * kSWarps) {
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
    float *part = a.ws + ((static_cast<int64_t>(b) * a.Hq + h * g + r) * a.splits + split) * (2 + D);
    if (d == 0) {
      part[0] = M;
      part[1] = L;
    }
    part[2 + d] = O;
  }
}

// Joins the splits of one query head, in order.
template <int D>
__global__ void __launch_bounds__(D) select_join_kernel(SelectArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int hq = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const float *part = a.ws + (static_cast<int64_t>(b) * a.Hq + hq) * a.splits * (2 + D);
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, ld_act_f32(part + s * (2 + D)));
  for (int s = 0; s < a.splits; ++s) {
    const float f = rescale(ld_act_f32(part + s * (2 + D)), M);
    L += ld_act_f32(part + s * (2 + D) + 1) * f;
    O += ld_act_f32(part + s * (2 + D) + 2 + d) * f;
  }
  a.out[b * a.os[0] + hq * a.os[1] + d] = float_to_bf16_bits(normalised(O, L));
}

}  // namespace iron

using namespace iron;

// Splits of a (sequence, kv head): enough CTAs for two per SM, at least 64 tokens each.
static int select_splits(int B, int Hkv, int top, int page) {
  const int64_t tokens = static_cast<int64_t>(top) * page;
  int s = 1;
  while (static_cast<int64_t>(B) * Hkv * s < 2LL * sm_count() && tokens / (2 * s) >= 64 && s < 64) s *= 2;
  return s;
}

extern "C" size_t iron_page_select_attn_workspace_bytes(int batch, int num_heads, int kv_heads, int head_dim,
                                                        int max_pages, int top_pages, int page_size) {
  if (batch <= 0 || num_heads <= 0 || kv_heads <= 0 || max_pages <= 0 || top_pages <= 0 || page_size <= 0) return 0;
  const size_t splits = select_splits(batch, kv_heads, top_pages, page_size);
  return (static_cast<size_t>(batch) * kv_heads * max_pages +
          static_cast<size_t>(batch) * num_heads * splits * (2 + head_dim)) * sizeof(float);
}

extern "C" int iron_page_select_attn(const iron_page_pool *c, const uint16_t *q, uint16_t *out, int32_t *selected,
                                     int num_heads, int top_pages, const int64_t *q_strides,
                                     const int64_t *out_strides, float scale, void *workspace, size_t workspace_bytes,
                                     unsigned flags, void *stream) {
  const int chk = pool_geometry_check(c);
  if (chk != IRON_OK) return chk;
  if (!c->lens || !c->codes || !q || !out || !selected || !q_strides || !out_strides || !workspace) return IRON_ERR_NULL;
  if (c->layers != 1 || num_heads <= 0 || num_heads % c->kv_heads || top_pages <= 0) return IRON_ERR_SHAPE;
  if (c->slots > 65535 || num_heads > 65535) return IRON_ERR_SHAPE;
  if (num_heads / c->kv_heads > 16) return IRON_ERR_UNSUPPORTED;
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
  a.scores = static_cast<float *>(workspace);
  a.ws = a.scores + static_cast<size_t>(c->slots) * c->kv_heads * c->max_pages;
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
  a.splits = select_splits(c->slots, c->kv_heads, top_pages, c->page_size);
  a.scale_log2 = scale * kLog2e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = c->head_dim == 128;
  const int B = c->slots;
  int st = launch(wide ? select_score_kernel<128> : select_score_kernel<64>,
                  dim3(max(1, min(64, (a.M + 63) / 64)), a.Hkv, B), dim3(32 * kSWarps), 0, s,
                  (flags & IRON_FLAG_PDL) != 0, a);
  if (st == IRON_OK) st = launch(select_pick_kernel, dim3(a.Hkv, B), dim3(kPickThreads), 0, s, true, a);
  if (st == IRON_OK)
    st = launch(wide ? select_attend_kernel<128> : select_attend_kernel<64>, dim3(a.splits, a.Hkv, B),
                dim3(32 * kSWarps), 0, s, true, a);
  if (st == IRON_OK)
    st = launch(wide ? select_join_kernel<128> : select_join_kernel<64>, dim3(a.Hq, B), dim3(wide ? 128 : 64), 0, s,
                true, a);
  return st;
}
