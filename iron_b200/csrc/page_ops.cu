// Page operators of the paged KV cache: append, fork (share, copy, reorder, free) and
// compact.
//
// A pool is bf16 [layers, P, Hkv, page, D]; a page table int32 [S, M] (-1: no page);
// refs int32 [P] counts the table rows that hold a page. Every operator is two launches:
// a plan by one CTA (who gets which page, from block-wide prefix sums over slots and over
// the pool's reference counts, so the lowest free pages go out in slot order and the
// result does not depend on any order of execution; fork has more CTAs beside it, which
// copy the reference counts) and a grid that moves the rows. The only atomics add to integer
// reference counts, whose sum has no order.
//
// Bounds: the data grids by HBM (each moved row is read once and written once, 16 bytes
// per thread and access, 4 or 8 accesses in flight per thread); the plans by the latency
// of a few dependent reads.
#include <cfloat>

#include "paged.cuh"

namespace iron {

constexpr int kPlanThreads = 1024;
constexpr int kMaxSlots = 2048;  // plan state per slot in shared memory

// ---- block-wide helpers of the plans (kPlanThreads threads) -----------------------------

// Inclusive prefix sum over the block's threads; *total gets the block's sum.
__device__ __forceinline__ int block_scan(int v, int *warp_sums, int *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  if (warp > 0) v += warp_sums[warp - 1];
  *total = warp_sums[31];
  __syncthreads();  // warp_sums may be used again
  return v;
}

// The lowest `want` pages p of [lo, hi) whose (refs[p] > 0) == used, ascending, into
// list. Returns how many there were (at most want). 8192 reference counts per pass, the
// next pass's loads issued before this one's prefix sum.
__device__ int collect_pages(const int *refs, int lo, int hi, bool used, int want, int *list, int *counts /* 256 */) {
  constexpr int kPer = 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int found = 0;
  int next[kPer];
  auto fetch = [&](int base) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = base + i * kPlanThreads + static_cast<int>(threadIdx.x);
      next[i] = p < hi ? ld_act_i32(refs + p) : (used ? 0 : 1);
    }
  };
  if (want > 0) fetch(lo);
  for (int base = lo; base < hi && found < want; base += kPer * kPlanThreads) {
    int cur[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) cur[i] = next[i];
    if (base + kPer * kPlanThreads < hi) fetch(base + kPer * kPlanThreads);
    unsigned hit[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      hit[i] = __ballot_sync(0xffffffffu, (cur[i] > 0) == used);
      if (lane == 0) counts[i * 32 + warp] = __popc(hit[i]);
    }
    __syncthreads();
    if (warp == 0) {  // exclusive prefix sum of the 256 counts, 8 per lane
      int c[kPer], sum = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        c[i] = counts[lane * kPer + i];
        sum += c[i];
      }
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      int at = incl - sum;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        counts[lane * kPer + i] = at;
        at += c[i];
      }
      if (lane == 31) counts[256] = at;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = found + counts[i * 32 + warp] + __popc(hit[i] & ((1u << lane) - 1u));
      if ((hit[i] >> lane & 1u) && r < want) list[r] = base + i * kPlanThreads + static_cast<int>(threadIdx.x);
    }
    found += counts[256];
    __syncthreads();  // counts may be used again
  }
  return min(found, want);
}

// ---- append ---------------------------------------------------------------------------

struct AppendArgs {
  const uint16_t *k_new, *v_new;  // [layers, S, N, Hkv, D]
  const int *index;               // [S, N]
  uint16_t *k, *v;                // pools
  int *table, *refs;
  const int *lens;
  int *lens_out, *status;
  int8_t *codes;                  // [layers, P, Hkv, 2, D] or null
  float *scales;                  // [layers, P, Hkv]
  int *take;                      // workspace [S]: rows appended per slot
  int *list;                      // workspace [P]: free pages
  int64_t layer_stride;           // elements of one layer of a pool
  int layers, S, N, Hkv, D, page, P, M;
};

__global__ void __launch_bounds__(kPlanThreads) append_plan_kernel(AppendArgs a) {
  __shared__ int take[kMaxSlots], need[kMaxSlots];
  __shared__ int warp_sums[32], counts[257], refused;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  for (int s = threadIdx.x; s < a.S; s += kPlanThreads) take[s] = a.N;
  if (threadIdx.x == 0) refused = 0;
  __syncthreads();
  // rows to append: up to the first index outside [0, N); 512 entries per warp and step
  const int per = (a.N + 511) / 512;
  for (int c = warp; c < a.S * per; c += kPlanThreads / 32) {
    const int s = c / per, j0 = (c % per) * 512;
    int first = a.N;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = j0 + i * 32 + lane;
      if (j < a.N) {
        const int x = ld_act_i32(a.index + static_cast<int64_t>(s) * a.N + j);
        if ((x < 0 || x >= a.N) && j < first) first = j;
      }
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0 && first < a.N) atomicMin(&take[s], first);
  }
  __syncthreads();
  // pages each slot needs: its touched table entries that are still -1
  for (int s = warp; s < a.S; s += kPlanThreads / 32) {
    const int n = take[s], len = ld_act_i32(a.lens + s);
    int miss = 0;
    bool off = len < 0 || static_cast<int64_t>(len) + n > static_cast<int64_t>(a.M) * a.page;
    if (n > 0 && !off) {
      const int last = (len + n - 1) / a.page;
      for (int at = len / a.page; at <= last; at += 32) {
        const int t = at + lane <= last ? ld_act_i32(a.table + static_cast<int64_t>(s) * a.M + at + lane) : 0;
        const bool in = at + lane <= last;
        miss += __popc(__ballot_sync(0xffffffffu, in && t < 0));
        // a page that another row holds too (or no page of this pool) is never written
        const bool bad = in && t >= 0 && (t >= a.P || ld_act_i32(a.refs + t) > 1);
        if (__any_sync(0xffffffffu, bad)) off = true;
      }
    }
    __syncwarp();
    if (lane == 0) {
      if (off) {
        take[s] = 0;
        miss = 0;
        atomicAdd(&refused, 1);
      }
      need[s] = miss;
    }
  }
  __syncthreads();
  // need[] becomes its inclusive prefix sum
  int total = 0;
  for (int s0 = 0; s0 < a.S; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int sum;
    const int v = block_scan(s < a.S ? need[s] : 0, warp_sums, &sum);
    if (s < a.S) need[s] = total + v;
    total += sum;
  }
  __syncthreads();
  const int got = collect_pages(a.refs, 0, a.P, false, total, a.list, counts);
  __syncthreads();
  for (int s = warp; s < a.S; s += kPlanThreads / 32) {
    const int end = need[s], begin = s > 0 ? need[s - 1] : 0;
    const bool off = end > begin && end > got;
    const int n = off ? 0 : take[s], len = ld_act_i32(a.lens + s);
    if (end > begin && !off) {
      int r = begin;
      const int last = (len + n - 1) / a.page;
      for (int at = len / a.page; at <= last; at += 32) {
        int *e = a.table + static_cast<int64_t>(s) * a.M + at + lane;
        const bool miss = at + lane <= last && ld_act_i32(e) < 0;
        const unsigned m = __ballot_sync(0xffffffffu, miss);
        if (miss) {
          const int p = a.list[r + __popc(m & ((1u << lane) - 1u))];
          *e = p;
          a.refs[p] = 1;
        }
        r += __popc(m);
      }
    }
    __syncwarp();
    if (lane == 0) {
      if (off) atomicAdd(&refused, 1);
      a.take[s] = n;
      a.lens_out[s] = len + n;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) a.status[0] = refused;
}

// One CTA: one touched page of one slot, one layer, K or V. Threads are rows x 16-byte
// columns of a token's Hkv * D values, so a thread's column (8 dims of one head) is fixed
// and the bounds of a page that becomes full are folded into the same pass (minimum and
// maximum of bf16 pairs are exact in bf16).
// The page's row numbers go through shared memory first, so that all of a thread's row
// loads are independent; 3 CTAs per SM x 256 threads x 8 loads of 16 bytes are in flight.
// B200, 16 layers, 4 prompts of up to 2048 tokens (402 MB moved): 64 us; 107 with the numbers
// loaded per row and 2 CTAs per SM.
constexpr int kAppendThreads = 256;

template <bool kSummaries>
__global__ void __launch_bounds__(kAppendThreads, 3) append_write_kernel(AppendArgs a) {
  extern __shared__ __align__(16) uint16_t bounds[];  // [row groups][2][Hkv * D] (pages that become full)
  __shared__ int rows_s[128];
  const int s = blockIdx.y, layer = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  pdl_launch_dependents();
  pdl_wait();
  const int n = ld_act_i32(a.take + s), end = ld_act_i32(a.lens_out + s), len = end - n;
  const int pi = len / a.page + blockIdx.x;           // the page's place in the slot
  const int t0 = max(len, pi * a.page), t1 = min(end, (pi + 1) * a.page);
  if (n <= 0 || t0 >= t1) return;
  const int p = ld_act_i32(a.table + static_cast<int64_t>(s) * a.M + pi);
  if (static_cast<int>(threadIdx.x) < t1 - t0)
    rows_s[threadIdx.x] = ld_act_i32(a.index + static_cast<int64_t>(s) * a.N + t0 - len + threadIdx.x);
  __syncthreads();
  const int vpr = a.Hkv * a.D / 8;                    // 16-byte columns per token
  const int width = min(vpr, kAppendThreads), groups = min(kAppendThreads / width, 64);
  const int g = threadIdx.x / width, c0 = threadIdx.x % width;
  const int row = a.Hkv * a.D;
  const uint16_t *src = (is_v ? a.v_new : a.k_new) + (static_cast<int64_t>(layer) * a.S + s) * a.N * row;
  uint16_t *dst = (is_v ? a.v : a.k) + layer * a.layer_stride + static_cast<int64_t>(p) * row * a.page;
  const bool full = kSummaries && !is_v && t1 == (pi + 1) * a.page;
  const __nv_bfloat162 inf = __float2bfloat162_rn(INFINITY);
  for (int c = c0; c < vpr && g < groups; c += width) {
    const int h = c * 8 / a.D, d = c * 8 % a.D;
    uint16_t *to = dst + (static_cast<int64_t>(h) * a.page - pi * a.page) * a.D + d;
    __nv_bfloat162 lo[4] = {inf, inf, inf, inf}, hi[4] = {__hneg2(inf), __hneg2(inf), __hneg2(inf), __hneg2(inf)};
    auto fold = [&](const uint4 &x) {
      const __nv_bfloat162 *w = reinterpret_cast<const __nv_bfloat162 *>(&x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = __hmin2_nan(lo[i], w[i]);
        hi[i] = __hmax2_nan(hi[i], w[i]);
      }
    };
    constexpr int kU = 8;
    for (int t = t0 + g; t < t1; t += kU * groups) {
      uint4 x[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (t + u * groups < t1)
          x[u] = ld_act_v4(src + static_cast<int64_t>(rows_s[t + u * groups - t0]) * row + c * 8);
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (t + u * groups < t1) {
          *reinterpret_cast<uint4 *>(to + static_cast<int64_t>(t + u * groups) * a.D) = x[u];
          if (full) fold(x[u]);
        }
    }
    if (full) {
      for (int t = pi * a.page + g; t < t0; t += groups)  // rows that were there before
        fold(ld_act_v4(to + static_cast<int64_t>(t) * a.D));
      *reinterpret_cast<uint4 *>(bounds + (g * 2 + 0) * row + c * 8) = *reinterpret_cast<const uint4 *>(lo);
      *reinterpret_cast<uint4 *>(bounds + (g * 2 + 1) * row + c * 8) = *reinterpret_cast<const uint4 *>(hi);
    }
  }
  if (!full) return;
  __syncthreads();
  // bounds of the page per head: a warp per head; the scale is the largest |key| / 127,
  // the codes are rounded outwards (down for the lower bound, up for the upper one). The
  // division is IEEE's, so the codes are the same wherever they are computed.
  const int lane = threadIdx.x & 31;
  for (int h = threadIdx.x >> 5; h < a.Hkv; h += kAppendThreads / 32) {
    float lo[4], hi[4], top = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = i * 32 + lane;
      lo[i] = INFINITY;
      hi[i] = -INFINITY;
      if (d < a.D) {
        for (int q = 0; q < groups; ++q) {
          const float l = bf16_bits_to_float(bounds[(q * 2 + 0) * row + h * a.D + d]);
          const float u = bf16_bits_to_float(bounds[(q * 2 + 1) * row + h * a.D + d]);
          nan |= l != l;
          lo[i] = fminf(lo[i], l);
          hi[i] = fmaxf(hi[i], u);
        }
        top = fmaxf(top, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
      }
    }
    top = warp_max(nan ? INFINITY : top);
    const float scale = __fdiv_rn(top, 127.f);
    const bool fine = top < INFINITY;
    const int64_t at = (static_cast<int64_t>(layer) * a.P + p) * a.Hkv + h;
    int8_t *out = a.codes + at * 2 * a.D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = i * 32 + lane;
      if (d < a.D) {
        const float by = scale > 0.f ? scale : 1.f;
        const float l = fine ? floorf(__fdiv_rn(lo[i], by)) : -127.f;
        const float u = fine ? ceilf(__fdiv_rn(hi[i], by)) : 127.f;
        out[d] = static_cast<int8_t>(fmaxf(fminf(l, 127.f), -127.f));
        out[a.D + d] = static_cast<int8_t>(fmaxf(fminf(u, 127.f), -127.f));
      }
    }
    if (lane == 0) a.scales[at] = fine ? scale : FLT_MAX;
  }
}

// ---- fork -----------------------------------------------------------------------------

struct ForkArgs {
  const int *source, *table, *lens, *refs;
  uint16_t *k, *v;
  int *table_out, *lens_out, *refs_out, *status;
  int *fresh;          // workspace [S]: the page a slot's partial page is copied to, or -1
  int *from;           // workspace [S]: the old slot, or -1
  int4 *copies;        // workspace [S]: {old page, new page, rows} of the partial pages to copy
  int *count;          // workspace [1]
  int64_t layer_stride;
  int layers, S, Hkv, D, page, P, M;
};

// Block 0 plans; the others copy the reference counts to refs_out.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(ForkArgs a) {
  __shared__ int src[kMaxSlots], keeper[kMaxSlots], length[kMaxSlots], list[kMaxSlots];
  __shared__ int warp_sums[32], counts[257], refused;
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x > 0) {
    for (int p = (blockIdx.x - 1) * kPlanThreads + threadIdx.x; p < a.P; p += (gridDim.x - 1) * kPlanThreads)
      a.refs_out[p] = ld_act_i32(a.refs + p);
    return;
  }
  for (int s = threadIdx.x; s < a.S; s += kPlanThreads) {
    const int r = ld_act_i32(a.source + s);
    src[s] = r >= 0 && r < a.S ? r : -1;
    keeper[s] = a.S;
    length[s] = max(0, min(ld_act_i32(a.lens + s), a.M * a.page));
  }
  if (threadIdx.x == 0) refused = 0;
  __syncthreads();
  // who keeps the partial page of old slot r: r itself (-1 here) or its lowest child
  for (int s = threadIdx.x; s < a.S; s += kPlanThreads)
    if (src[s] >= 0) atomicMin(&keeper[src[s]], src[s] == s ? -1 : s);
  __syncthreads();
  // a slot's rank among those that copy, and the page that it copies from: requested before
  // the free pages are looked for
  constexpr int kPer = kMaxSlots / kPlanThreads;
  int rank[kPer], from[kPer], before = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = i * kPlanThreads + threadIdx.x, r = s < a.S ? src[s] : -1;
    const bool copy = r >= 0 && length[r] % a.page > 0 && r != s && keeper[r] != s;
    from[i] = copy ? ld_act_i32(a.table + static_cast<int64_t>(r) * a.M + length[r] / a.page) : -1;
    int sum = 0;
    if (i * kPlanThreads < a.S) rank[i] = before + block_scan(copy ? 1 : 0, warp_sums, &sum) - 1;
    if (!copy) rank[i] = -1;
    before += sum;
  }
  const int got = collect_pages(a.refs, 0, a.P, false, before, list, counts);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = i * kPlanThreads + threadIdx.x;
    if (s >= a.S) break;
    const bool off = rank[i] >= got;  // no page left: the slot stays empty
    const int to = rank[i] >= 0 && !off ? list[rank[i]] : -1, len = src[s] >= 0 && !off ? length[src[s]] : 0;
    a.fresh[s] = to;
    a.from[s] = off ? -1 : src[s];
    a.lens_out[s] = len;
    if (off) atomicAdd(&refused, 1);
    // a table entry that is no page of the pool: nothing to copy
    if (to >= 0) a.copies[rank[i]] = make_int4(from[i], to, from[i] >= 0 && from[i] < a.P ? len % a.page : 0, 0);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.status[0] = refused;
    a.count[0] = got;
  }
}

constexpr int kCopyThreads = 256;
constexpr int kCopyPer = 4;  // 16-byte accesses in flight per thread
constexpr int kCopyBytes = kCopyThreads * kCopyPer * 16;

// Copies `bytes` (a multiple of 16, both ends 16-byte aligned) by one CTA.
__device__ __forceinline__ void copy_block(const uint8_t *src, uint8_t *dst, int bytes) {
  for (int at = threadIdx.x * 16; at < bytes; at += kCopyBytes) {
    uint4 x[kCopyPer];
#pragma unroll
    for (int i = 0; i < kCopyPer; ++i)
      if (at + i * kCopyThreads * 16 < bytes) x[i] = ld_act_v4(src + at + i * kCopyThreads * 16);
#pragma unroll
    for (int i = 0; i < kCopyPer; ++i)
      if (at + i * kCopyThreads * 16 < bytes) *reinterpret_cast<uint4 *>(dst + at + i * kCopyThreads * 16) = x[i];
  }
}

// Writes the new table and the reference counts, then copies the valid rows of the partial
// pages: a warp per (copy, layer, K or V, head), rows * D contiguous values, 8 accesses of
// 16 bytes in flight per lane. (A CTA per such item measured 85 us against 29 for 60 copies
// in 16 layers and 8 heads, 122 MB moved: most CTAs had little or nothing to do.)
__global__ void __launch_bounds__(kCopyThreads) fork_copy_kernel(ForkArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int warp = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5), warps = gridDim.x * (kCopyThreads / 32);
  const int per = (a.M + 31) / 32;  // a warp takes 32 entries of one row
  for (int64_t it = warp; it < static_cast<int64_t>(a.S) * per; it += warps) {
    const int s = static_cast<int>(it / per), at = static_cast<int>(it % per) * 32 + lane;
    const int r = ld_act_i32(a.from + s), fresh = ld_act_i32(a.fresh + s), len = ld_act_i32(a.lens_out + s);
    if (at >= a.M) continue;
    const int pages = (len + a.page - 1) / a.page;
    const int old = ld_act_i32(a.table + static_cast<int64_t>(s) * a.M + at);
    int now = -1;
    if (at < pages)
      now = at == len / a.page && fresh >= 0 ? fresh : ld_act_i32(a.table + static_cast<int64_t>(r) * a.M + at);
    a.table_out[static_cast<int64_t>(s) * a.M + at] = now;
    if (old != now) {
      if (old >= 0 && old < a.P) atomicSub(a.refs_out + old, 1);
      if (now >= 0 && now < a.P) atomicAdd(a.refs_out + now, 1);
    }
  }
  const int planes = 2 * a.layers * a.Hkv;
  const int64_t items = static_cast<int64_t>(ld_act_i32(a.count)) * planes;
  for (int64_t it = warp; it < items; it += warps) {
    const int4 c = *reinterpret_cast<const int4 *>(a.copies + it / planes);
    const int plane = static_cast<int>(it % planes), h = plane % a.Hkv, lv = plane / a.Hkv;
    uint16_t *pool = ((lv & 1) ? a.v : a.k) + (lv >> 1) * a.layer_stride;
    const uint4 *from = reinterpret_cast<const uint4 *>(pool + (static_cast<int64_t>(c.x) * a.Hkv + h) * a.page * a.D);
    uint4 *to = reinterpret_cast<uint4 *>(pool + (static_cast<int64_t>(c.y) * a.Hkv + h) * a.page * a.D);
    const int n = c.z * a.D / 8;
    for (int i = lane; i < n; i += 8 * 32) {
      uint4 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (i + u * 32 < n) x[u] = ld_act_v4(from + i + u * 32);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (i + u * 32 < n) to[i + u * 32] = x[u];
    }
  }
}

// ---- compact --------------------------------------------------------------------------

struct CompactArgs {
  const int *table, *refs;
  uint16_t *k, *v;
  int8_t *codes;
  float *scales;
  int *table_out, *refs_out, *used;
  int *moves;      // workspace: [1] count, padded to 4 ints
  int *dst, *src;  // workspace [P / 2 + 1] each
  int *where;      // workspace [P]: a moved page's new place
  int64_t layer_stride;
  int layers, S, Hkv, D, page, P, M;
};

// Used pages stay where they are if they are below U, the number of used pages; the i-th
// used page from U on moves to the i-th free page below U. Sources and destinations are
// disjoint, so the moves run in any order, and as few pages move as can.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(CompactArgs a) {
  __shared__ int warp_sums[32], counts[257];
  pdl_launch_dependents();
  pdl_wait();
  int mine = 0;
  for (int p = threadIdx.x; p < a.P; p += kPlanThreads) mine += ld_act_i32(a.refs + p) > 0;
  int used;
  block_scan(mine, warp_sums, &used);
  const int most = min(used, a.P - used);
  const int m = collect_pages(a.refs, used, a.P, true, most, a.src, counts);
  collect_pages(a.refs, 0, used, false, m, a.dst, counts);
  __syncthreads();
  for (int i = threadIdx.x; i < m; i += kPlanThreads) a.where[a.src[i]] = a.dst[i];
  if (threadIdx.x == 0) {
    a.moves[0] = m;
    a.used[0] = used;
  }
}

// Grid-stride over the table, the reference counts and the moved pages' bytes in pieces
// of kCopyBytes: every (move, layer, K or V) is page_bytes / kCopyBytes pieces.
__global__ void __launch_bounds__(kCopyThreads) compact_copy_kernel(CompactArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int m = ld_act_i32(a.moves), used = ld_act_i32(a.used);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kCopyThreads;
  for (int64_t i = first; i < static_cast<int64_t>(a.S) * a.M; i += stride) {
    const int t = ld_act_i32(a.table + i);
    a.table_out[i] = t >= used && t < a.P ? ld_act_i32(a.where + t) : t;
  }
  if (a.refs_out != a.refs)
    for (int64_t p = first; p < a.P; p += stride) {
      const int r = ld_act_i32(a.refs + p);
      // places that a move fills or empties are written by the move, below
      if ((p < used) == (r > 0)) a.refs_out[p] = r;
    }
  for (int64_t i = first; i < m; i += stride) {
    const int src = ld_act_i32(a.src + i), dst = ld_act_i32(a.dst + i), r = ld_act_i32(a.refs + src);
    a.refs_out[dst] = r;
    a.refs_out[src] = 0;
  }
  const int page_bytes = a.Hkv * a.page * a.D * 2;
  const int pieces = (page_bytes + kCopyBytes - 1) / kCopyBytes;
  const int64_t items = static_cast<int64_t>(m) * a.layers * 2 * pieces;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int piece = static_cast<int>(it % pieces);
    const int64_t q = it / pieces;
    const int plane = static_cast<int>(q % (2 * a.layers)), i = static_cast<int>(q / (2 * a.layers));
    uint8_t *pool = reinterpret_cast<uint8_t *>(((plane & 1) ? a.v : a.k) + (plane >> 1) * a.layer_stride) +
                    piece * kCopyBytes;
    copy_block(pool + static_cast<int64_t>(ld_act_i32(a.src + i)) * page_bytes,
               pool + static_cast<int64_t>(ld_act_i32(a.dst + i)) * page_bytes,
               min(kCopyBytes, page_bytes - piece * kCopyBytes));
  }
  if (!a.codes) return;
  // summaries: a thread per (move, layer, 16 bytes of codes), and one scale per head
  const int per = a.Hkv * 2 * a.D / 16;
  for (int64_t it = first; it < static_cast<int64_t>(m) * a.layers * per; it += stride) {
    const int c = static_cast<int>(it % per), layer = static_cast<int>(it / per % a.layers);
    const int i = static_cast<int>(it / per / a.layers);
    const int64_t src = static_cast<int64_t>(layer) * a.P + ld_act_i32(a.src + i);
    const int64_t dst = static_cast<int64_t>(layer) * a.P + ld_act_i32(a.dst + i);
    *reinterpret_cast<uint4 *>(a.codes + dst * per * 16 + c * 16) = ld_act_v4(a.codes + src * per * 16 + c * 16);
    if (c < a.Hkv) a.scales[dst * a.Hkv + c] = ld_act_f32(a.scales + src * a.Hkv + c);
  }
}

}  // namespace iron

using namespace iron;

// Checks shared by the three operators.
static int pool_check(const iron_page_pool *c) {
  const int chk = pool_geometry_check(c);
  if (chk != IRON_OK) return chk;
  if (!c->refs) return IRON_ERR_NULL;
  return c->slots > kMaxSlots ? IRON_ERR_UNSUPPORTED : IRON_OK;
}

static bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}

extern "C" size_t iron_page_append_workspace_bytes(int slots, int num_pages) {
  return slots > 0 && num_pages > 0 ? (static_cast<size_t>(slots) + num_pages) * sizeof(int) : 0;
}

extern "C" int iron_page_append(const iron_page_pool *c, const uint16_t *k_new, const uint16_t *v_new,
                                const int32_t *index, int num_new, int32_t *lens_out, int32_t *status,
                                void *workspace, size_t workspace_bytes, unsigned flags, void *stream) {
  (void)flags;
  const int chk = pool_check(c);
  if (chk != IRON_OK) return chk;
  if (!k_new || !v_new || !index || !c->lens || !lens_out || !status || !workspace) return IRON_ERR_NULL;
  if (num_new <= 0 || num_new > (1 << 24)) return IRON_ERR_SHAPE;
  if (!aligned16(k_new) || !aligned16(v_new)) return IRON_ERR_ALIGN;
  if (workspace_bytes < iron_page_append_workspace_bytes(c->slots, c->num_pages)) return IRON_ERR_WORKSPACE;
  AppendArgs a = {};
  a.k_new = k_new;
  a.v_new = v_new;
  a.index = index;
  a.k = c->k;
  a.v = c->v;
  a.table = c->page_table;
  a.refs = c->refs;
  a.lens = c->lens;
  a.lens_out = lens_out;
  a.status = status;
  a.codes = c->codes;
  a.scales = c->scales;
  a.take = static_cast<int *>(workspace);
  a.list = a.take + c->slots;
  a.layers = c->layers;
  a.S = c->slots;
  a.N = num_new;
  a.Hkv = c->kv_heads;
  a.D = c->head_dim;
  a.page = c->page_size;
  a.P = c->num_pages;
  a.M = c->max_pages;
  a.layer_stride = static_cast<int64_t>(a.P) * a.Hkv * a.page * a.D;
  const int touched = min((num_new + a.page - 2) / a.page + 1, a.M);
  const int vpr = a.Hkv * a.D / 8, width = vpr < kAppendThreads ? vpr : kAppendThreads;
  const int groups = kAppendThreads / width < 64 ? kAppendThreads / width : 64;
  const size_t smem = a.codes ? static_cast<size_t>(groups) * 2 * a.Hkv * a.D * sizeof(uint16_t) : 0;
  // nothing may be refused once the plan runs: it takes pages and moves the lengths
  if (smem > 200 * 1024) return IRON_ERR_UNSUPPORTED;
  auto kern = a.codes ? append_write_kernel<true> : append_write_kernel<false>;
  if (smem > 48 * 1024) {
    const int e = call_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    if (e != IRON_OK) return e;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int st = launch(append_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, true, a);
  if (st != IRON_OK) return st;
  return launch(kern, dim3(touched, a.S, 2 * a.layers), dim3(kAppendThreads), smem, s, true, a);
}

extern "C" size_t iron_page_fork_workspace_bytes(int slots) {
  return slots > 0 ? static_cast<size_t>(slots) * 6 * sizeof(int) + 16 : 0;
}

extern "C" int iron_page_fork(const iron_page_pool *c, const int32_t *source, int32_t *page_table_out,
                              int32_t *lens_out, int32_t *refs_out, int32_t *status, void *workspace,
                              size_t workspace_bytes, unsigned flags, void *stream) {
  (void)flags;
  const int chk = pool_check(c);
  if (chk != IRON_OK) return chk;
  if (!source || !c->lens || !page_table_out || !lens_out || !refs_out || !status || !workspace) return IRON_ERR_NULL;
  if (workspace_bytes < iron_page_fork_workspace_bytes(c->slots)) return IRON_ERR_WORKSPACE;
  if (!aligned16(workspace)) return IRON_ERR_ALIGN;
  const size_t tb = static_cast<size_t>(c->slots) * c->max_pages * sizeof(int), rb = c->num_pages * sizeof(int);
  // rows are gathered from the old table while the new one is written
  if (overlap(c->page_table, tb, page_table_out, tb) || overlap(c->refs, rb, refs_out, rb)) return IRON_ERR_ARG;
  ForkArgs a = {};
  a.source = source;
  a.table = c->page_table;
  a.lens = c->lens;
  a.refs = c->refs;
  a.k = c->k;
  a.v = c->v;
  a.table_out = page_table_out;
  a.lens_out = lens_out;
  a.refs_out = refs_out;
  a.status = status;
  a.copies = static_cast<int4 *>(workspace);
  a.fresh = reinterpret_cast<int *>(a.copies + c->slots);
  a.from = a.fresh + c->slots;
  a.count = a.from + c->slots;
  a.layers = c->layers;
  a.S = c->slots;
  a.Hkv = c->kv_heads;
  a.D = c->head_dim;
  a.page = c->page_size;
  a.P = c->num_pages;
  a.M = c->max_pages;
  a.layer_stride = static_cast<int64_t>(a.P) * a.Hkv * a.page * a.D;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int copiers = min(64, (a.P + kPlanThreads - 1) / kPlanThreads);
  int st = launch(fork_plan_kernel, dim3(1 + copiers), dim3(kPlanThreads), 0, s, true, a);
  if (st != IRON_OK) return st;
  return launch(fork_copy_kernel, dim3(sm_count() * 8), dim3(kCopyThreads), 0, s, true, a);
}

extern "C" size_t iron_page_compact_workspace_bytes(int num_pages) {
  return num_pages > 0 ? (static_cast<size_t>(num_pages) + 2 * (num_pages / 2 + 1) + 4) * sizeof(int) : 0;
}

extern "C" int iron_page_compact(const iron_page_pool *c, int32_t *page_table_out, int32_t *refs_out, int32_t *used,
                                 void *workspace, size_t workspace_bytes, unsigned flags, void *stream) {
  (void)flags;
  const int chk = pool_check(c);
  if (chk != IRON_OK) return chk;
  if (!page_table_out || !refs_out || !used || !workspace) return IRON_ERR_NULL;
  if (workspace_bytes < iron_page_compact_workspace_bytes(c->num_pages)) return IRON_ERR_WORKSPACE;
  const size_t tb = static_cast<size_t>(c->slots) * c->max_pages * sizeof(int), rb = c->num_pages * sizeof(int);
  if ((page_table_out != c->page_table && overlap(c->page_table, tb, page_table_out, tb)) ||
      (refs_out != c->refs && overlap(c->refs, rb, refs_out, rb)))
    return IRON_ERR_ARG;
  CompactArgs a = {};
  a.table = c->page_table;
  a.refs = c->refs;
  a.k = c->k;
  a.v = c->v;
  a.codes = c->codes;
  a.scales = c->scales;
  a.table_out = page_table_out;
  a.refs_out = refs_out;
  a.used = used;
  a.moves = static_cast<int *>(workspace);
  a.dst = a.moves + 4;
  a.src = a.dst + c->num_pages / 2 + 1;
  a.where = a.src + c->num_pages / 2 + 1;
  a.layers = c->layers;
  a.S = c->slots;
  a.Hkv = c->kv_heads;
  a.D = c->head_dim;
  a.page = c->page_size;
  a.P = c->num_pages;
  a.M = c->max_pages;
  a.layer_stride = static_cast<int64_t>(a.P) * a.Hkv * a.page * a.D;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int st = launch(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, true, a);
  if (st != IRON_OK) return st;
  return launch(compact_copy_kernel, dim3(sm_count() * 8), dim3(kCopyThreads), 0, s, true, a);
}
