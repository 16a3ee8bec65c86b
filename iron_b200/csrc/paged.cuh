// Shared by the operators on a paged KV cache: argument checks and the warp-level
// attention step on 16 tokens (mma.sync m16n8k16, online softmax in fp32).
#pragma once

#include "common.cuh"

namespace iron {

constexpr float kLog2e = 1.4426950408889634f;

// The pool's geometry, common to all entry points.
inline int pool_geometry_check(const iron_page_pool *c) {
  if (!c || !c->k || !c->v || !c->page_table) return IRON_ERR_NULL;
  if (c->layers <= 0 || c->slots <= 0 || c->num_pages <= 0 || c->max_pages <= 0 || c->kv_heads <= 0)
    return IRON_ERR_SHAPE;
  if (c->layers > 16384 || c->kv_heads > 1024 || c->num_pages > (1 << 24)) return IRON_ERR_SHAPE;
  if (c->head_dim != 64 && c->head_dim != 128) return IRON_ERR_UNSUPPORTED;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return IRON_ERR_UNSUPPORTED;
  // a length rounded up to a whole tile (of 128 tokens at most) stays an int
  if (static_cast<int64_t>(c->max_pages) * c->page_size > 0x7fffffff - 127) return IRON_ERR_SHAPE;
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->codes)) return IRON_ERR_ALIGN;
  if ((c->codes != nullptr) != (c->scales != nullptr)) return IRON_ERR_ARG;
  return IRON_OK;
}

// ---- a warp's attention over blocks of 16 tokens ------------------------------------------
// Rows are up to 16 query rows (gid = lane / 4 and gid + 8); tokens come 16 at a time
// through a ring of shared-memory stages of the warp's own, filled by asynchronous copies
// kStages - 1 blocks ahead (one block in registers, the form before, kept 4 KB per warp in
// flight: 2.8 TB/s on B200 at 64 sequences). Rows are padded to an odd number of 16-byte
// pieces, so that ldmatrix meets no bank conflicts. S = Q K^T and O += P V are mma.sync
// m16n8k16, the softmax runs online in fp32.

// Asynchronous 16-byte global -> shared copy; zeros instead where !full (nothing is read).
__device__ __forceinline__ void cp_async16_zfill(void *dst, const void *src, bool full) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(full ? 16 : 0)
               : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], const void *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p)))
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], const void *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p)))
               : "memory");
}

// Two p >= 0 as two bf16 parts each: hi is p cut off after 8 bits, lo = kSplit p - hi, rounded
// (minus0 and minus1 are the -hi). Both parts are positive where p is, so that a value of +-inf
// times them stays one: 0 * inf, or infinities of both signs, would be NaN.
constexpr float kSplit = 1.f + 1.f / 1048576.f;
__device__ __forceinline__ uint32_t split_hi(float p0, float p1, float &minus0, float &minus1) {
  uint32_t hi;
  asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(p1), "f"(p0));
  minus0 = __uint_as_float(hi << 16 | 0x80000000u);
  minus1 = __uint_as_float((hi & 0xffff0000u) | 0x80000000u);
  return hi;
}

// A stage: 16 rows of K, then 16 rows of V.
template <int D>
struct Stage {
  static constexpr int kRow = D + 8;            // elements
  static constexpr int kElems = 2 * 16 * kRow;  // K and V
  static constexpr int kBytes = kElems * 2;
  uint16_t x[kElems];

  // rows >= n become zero and are not read (n <= 0: none is)
  __device__ __forceinline__ void load(const uint16_t *k, const uint16_t *v, int64_t krow, int64_t vrow, int n) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int idx = i * 32 + lane, row = idx / (D / 8), c = idx % (D / 8);
      cp_async16_zfill(x + row * kRow + c * 8, row < n ? k + row * krow + c * 8 : k, row < n);
      cp_async16_zfill(x + (16 + row) * kRow + c * 8, row < n ? v + row * vrow + c * 8 : v, row < n);
    }
  }
};

template <int D>
struct WarpAttn {
  uint32_t q[D / 16][4];
  float o[D / 8][4];
  float m[2], l[2];  // running maximum (log2 units) and this lane's share of the sum, rows gid and gid + 8

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }

  // q rows at lo and hi (null: a zero row)
  __device__ __forceinline__ void load_q(const uint16_t *lo, const uint16_t *hi) {
    const int tid = threadIdx.x & 3;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int d = 16 * ks + 2 * tid;
      q[ks][0] = lo ? ld_act_u32(lo + d) : 0u;
      q[ks][1] = hi ? ld_act_u32(hi + d) : 0u;
      q[ks][2] = lo ? ld_act_u32(lo + d + 8) : 0u;
      q[ks][3] = hi ? ld_act_u32(hi + d + 8) : 0u;
    }
  }

  // One block; bit t of see[0] / see[1]: row gid / gid + 8 sees token t.
  __device__ __forceinline__ void step(const Stage<D> &st, float scale_log2, const uint32_t (&see)[2]) {
    const int lane = threadIdx.x & 31, tid = lane & 3;
    float s[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        uint32_t b[4];
        ldsm_x4(b, st.x + (nt * 8 + (lane & 7)) * Stage<D>::kRow + (4 * j + (lane >> 3)) * 8);
        mma_bf16_16816(s[nt], q[2 * j], b[0], b[1]);
        mma_bf16_16816(s[nt], q[2 * j + 1], b[2], b[3]);
      }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = nt * 8 + 2 * tid + (e & 1);
        s[nt][e] = (see[e >> 1] >> t & 1u) ? s[nt][e] * scale_log2 : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[nt][e]);
      }
    float ref[2], al[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      const float mn = fmaxf(m[r], mx[r]);
      ref[r] = mn == -INFINITY ? 0.f : mn;  // a row that has seen nothing yet
      al[r] = ex2_approx(m[r] - ref[r]);
      m[r] = mn;
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[nt][e] = ex2_approx(s[nt][e] - ref[e >> 1]);
        sum[e >> 1] += s[nt][e];
      }
    l[0] = l[0] * al[0] + sum[0];
    l[1] = l[1] * al[1] + sum[1];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      o[j][0] *= al[0];
      o[j][1] *= al[0];
      o[j][2] *= al[1];
      o[j][3] *= al[1];
    }
    // P enters the product with V as two bf16 parts, hi + lo, which hold it to 2^-16: one
    // bf16 would be off by up to 2^-8 of each term, as much as the output's own rounding.
    // The second pair of MMAs costs nothing where K and V bound the kernel.
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p0 = s[i >> 1][2 * (i & 1)], p1 = s[i >> 1][2 * (i & 1) + 1];
      float m0, m1;
      hi[i] = split_hi(p0, p1, m0, m1);
      lo[i] = pack_bf16x2(fmaf(p0, kSplit, m0), fmaf(p1, kSplit, m1));
    }
#pragma unroll
    for (int jp = 0; jp < D / 16; ++jp) {
      uint32_t b[4];
      ldsm_x4_t(b, st.x + (16 + (lane & 7) + ((lane >> 3) & 1) * 8) * Stage<D>::kRow + jp * 16 + (lane >> 4) * 8);
      mma_bf16_16816(o[2 * jp], hi, b[0], b[1]);
      mma_bf16_16816(o[2 * jp + 1], hi, b[2], b[3]);
      mma_bf16_16816(o[2 * jp], lo, b[0], b[1]);
      mma_bf16_16816(o[2 * jp + 1], lo, b[2], b[3]);
    }
  }

  // the row sums over the four lanes of each row
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
  }
};

// The factor that brings a partial of maximum m (log2 units) to the common maximum M.
// Partials that saw nothing (m = -inf) get 0, which keeps a NaN in them a NaN.
__device__ __forceinline__ float rescale(float m, float M) { return exp2f(m - (M == -INFINITY ? 0.f : M)); }
// O / L; a row that saw nothing is zero.
__device__ __forceinline__ float normalised(float o, float l) { return l == 0.f ? 0.f : o / l; }

}  // namespace iron
