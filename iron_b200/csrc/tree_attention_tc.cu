// Tree attention on the 5th-generation tensor cores, for many rows per kv head.
//
// Rows: num_nodes * group rows of a (sequence, kv head) read the same K and V; a unit is up
// to 256 of them, a tile is 128 tokens. One CTA per SM takes an equal share of all units'
// tiles (tree.cuh). Two streams of 128 rows run staggered, so that one's softmax overlaps
// the other's MMAs: with more than 128 rows stream s is the unit's rows 128 s ... and both
// see every tile; with fewer, both hold the same rows and stream s sees every second tile
// (its issuing warp goes through all of them); stream 0 then joins both results, whose rows
// lie in the same TMEM lanes.
//
// Warps: 0-3 and 4-7 the softmax of stream 0 and 1 (a thread owns one row: no shuffles), 8
// and 9 issue the MMAs of stream 0 and 1, 10 loads (TMA, one box per page and 64 columns),
// 11 finds the nodes' paths and zeroes the rows of V that hold nothing.
//   S = Q K^T     128 x 128 x D (D = 128: x 64), both operands in shared memory (K-major)
//   P -> TMEM     64 tokens at a time, in columns of its own: bf16 hi and lo parts (P = hi +
//                 lo to 2^-16: one bf16 would double the error of the rounded output)
//   O += P V      128 x D x 64, hi then lo; A from TMEM, V as it lies in the page (MN-major)
// S is read into registers whole, so the MMAs of the next S run under this one's softmax.
// TMEM (512 columns): S0, S1, O0, O1, P0, P1. O is rescaled only when a row's maximum has
// grown by more than 2^8 (P stays below 2^8, exact in the sums' fp32 range).
//
// Bounds (B200): per 128 tokens and stream 1024 cycles of ex2 (16 per cycle and SM for 128
// rows), and on the tensor cores 250 of S and 530 of P V at D = 64, 770 and 960 at D = 128
// (measured alone: S of 64 columns 48 cycles per MMA, of 128 columns 62; P V 33 and 60).
// 16 sequences of 4608 tokens, 64 nodes of 4 heads: D = 64 114 us, D = 128 133 (when D = 64 took
// 107: without the MMAs 100, without ex2 88, without all arithmetic of the softmax 71): no unit is
// full (issue 40 %, ex2 36 %, tensor 27 %); the 550 instructions of a warp per 64 tokens, with
// two such warps per scheduler, set the pace. 8 sequences of
// 32768 tokens, D = 128: 296 us, tensor cores 68 % busy (347 in long runs, at the power
// limit). What a tile must not hold (past the length, unused nodes) is masked in S and
// zeroed in V.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "tc.cuh"
#include "tree.cuh"

namespace iron {
namespace gemm {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();  // gemm_tc.cu
}

__device__ unsigned g_tree_status;  // 0 = ok, else the first failing role's code

namespace treetc {

constexpr int kTile = 128;
constexpr int kThreads = 384;  // three warpgroups
// registers: 384 x 168 at launch = 2 x 128 x 216 (a row of S is 128 of them) + 128 x 72
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
static_assert(kThreads * 168 == 256 * kSoftmaxRegs + 128 * kOtherRegs, "the split must not exceed the launch's registers");
// a unit's start and end take as long as about 3 tiles (B200: 5 us against 1.1 to 2.6)
struct Cut {
  static constexpr int kTile = treetc::kTile, kUnitCost = 3;
};
constexpr int kMasks = 8;  // tiles' masks in flight: stages + 2 at least

// Bounded wait for a barrier phase: false after limit_us, or once *stop is set (some role
// gave up, so what it owes the others will not come). Both are looked at every 256 polls only,
// which waits of the usual length never reach.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, const volatile int *stop, uint32_t limit_us = 2000000) {
  uint64_t start = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 255u) == 0u) {
      if (stop && *stop) return false;
      const uint64_t now = tc::globaltimer_ns();
      if (start == 0) start = now;
      else if (now - start > limit_us * 1000ull) return false;
    }
  }
}
// The loads' wait for room, whose limit the caller sets; a limit of 0 looks once.
__device__ __forceinline__ bool wait_room(uint32_t bar, uint32_t parity, const volatile int *stop, uint32_t limit_us) {
  if (limit_us > 0) return wait_phase(bar, parity, stop, limit_us);
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done;
}

template <int D>
struct Cfg {
  static constexpr int kStages = D == 64 ? 4 : 2;
  // tables of paths in flight: preparing tile i means that tile i - kStages is done with
  static constexpr int kTrees = kStages + 3;
  static constexpr int kPanels = D / 64;
  static constexpr int kScores = D == 64 ? 128 : 64;       // tokens of one S
  // TMEM columns: S of both streams, O of both, P (64 tokens, hi then lo) of both
  static constexpr int kTmemS = 0, kTmemO = 2 * kScores, kTmemP = kTmemO + 2 * D;
  static_assert(kTmemP + 128 == 512, "TMEM is full");
  static constexpr uint32_t kPanel = kTile * 128;          // 128 rows x 64 bf16
  static constexpr uint32_t kOperand = kPanels * kPanel;   // Q tile, K tile or V tile
  static constexpr uint32_t kSmem = 1024 + 2 * kOperand + 2 * kStages * kOperand;
  static constexpr int kPart = kTile * D + 2 * kTile;      // floats of one stream's partial: O [D][128], then (m, l)
};

// two fp32 operations per instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A value that is the same in all lanes, in a form the compiler knows to be so: loops and
// addresses derived from it stay in uniform registers.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

struct Bars {  // mbarrier addresses
  uint32_t base;
  template <int S> __device__ uint32_t kfull(int i) const { return base + 8 * i; }
  template <int S> __device__ uint32_t kempty(int i) const { return base + 8 * (S + i); }
  template <int S> __device__ uint32_t vfull(int i) const { return base + 8 * (2 * S + i); }
  template <int S> __device__ uint32_t vempty(int i) const { return base + 8 * (3 * S + i); }
  template <int S> __device__ uint32_t sfull(int s) const { return base + 8 * (4 * S + s); }
  template <int S> __device__ uint32_t sfree(int s) const { return base + 8 * (4 * S + 2 + s); }
  template <int S> __device__ uint32_t pfull(int s) const { return base + 8 * (4 * S + 4 + s); }
  template <int S> __device__ uint32_t pvdone(int s) const { return base + 8 * (4 * S + 6 + s); }
  template <int S> __device__ uint32_t qfull(int i) const { return base + 8 * (4 * S + 8 + i); }
  template <int S> __device__ uint32_t vready(int i) const { return base + 8 * (4 * S + 14 + kMasks + i); }
  template <int S> __device__ uint32_t paths(int i) const { return base + 8 * (5 * S + 14 + kMasks + i); }
  template <int S> __device__ uint32_t drain(int s) const { return base + 8 * (4 * S + 10 + s); }
  template <int S> __device__ uint32_t other() const { return base + 8 * (4 * S + 12); }
  template <int S> __device__ uint32_t joined() const { return base + 8 * (4 * S + 13); }
  template <int S> __device__ uint32_t mask(int i) const { return base + 8 * (4 * S + 14 + i); }
};

struct Maps {
  CUtensorMap k, v, k_new, v_new;
};

// Tiles of a segment that stream s handles, and the segment's form.
struct Streams {
  bool both;  // both streams see every tile (more than 128 rows)
  int n[2];
};
__device__ __forceinline__ Streams streams_of(const TreeArgs &a, const Segment &sg) {
  const int rows = a.N * (a.Hq / a.Hkv) - sg.group * 256;
  Streams st;
  st.both = rows > 128;
  st.n[0] = st.both ? sg.count : (sg.count + 1) / 2;
  st.n[1] = st.both ? sg.count : sg.count / 2;
  return st;
}

// Halves of a tile that hold something: a short last tile has one.
__device__ __forceinline__ int halves_of(const TreeArgs &a, int i, int ctiles, int len) {
  return (i >= ctiles ? a.N - (i - ctiles) * kTile : len - i * kTile) > kTile / 2 ? 2 : 1;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
tree_tc_kernel(const __grid_constant__ Maps maps, const TreeArgs a) {
  using C = Cfg<D>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_store[5 * S + 14 + kMasks + C::kTrees];
  __shared__ uint32_t tmem_slot;
  __shared__ int pref[kTMaxBatch + 1], warp_sums[kThreads / 32];
  __shared__ __align__(16) uint32_t masks[kMasks][4];
  __shared__ TreePaths trees[C::kTrees];
  __shared__ float2 other_ml[kTile];        // (m, l) of stream 1, for the join of both streams
  __shared__ int odd_flag;                  // V of the tree held values that are not finite
  __shared__ int stop;                      // a wait ran out
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (base - raw);
  const uint32_t q0 = base, k0 = base + 2 * C::kOperand, v0 = k0 + S * C::kOperand;
  const Bars bars{smem_addr(bar_store)};
  auto wait_phase = [&](uint32_t bar, uint32_t parity) { return treetc::wait_phase(bar, parity, &stop); };
  auto drain = [&](uint32_t bar, uint32_t parity) { treetc::wait_phase(bar, parity, nullptr); };  // what is in flight
  auto give_up = [&](unsigned role) {
    *const_cast<volatile int *>(&stop) = 1;
    atomicCAS(&g_tree_status, 0u, role);
  };

  pdl_launch_dependents();
  pdl_wait();
  cost_prefix<Cut, kThreads>(a, pref, warp_sums);
  const int64_t total = static_cast<int64_t>(pref[a.B]) * a.Hkv * a.groups;
  const int pieces = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total));  // none is empty
  if (static_cast<int>(blockIdx.x) >= pieces) return;
  const int64_t w_begin = piece_start(total, blockIdx.x, pieces), w_end = piece_start(total, blockIdx.x + 1, pieces);

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      tc::mbar_init_u32(bars.kfull<S>(i), 1);
      tc::mbar_init_u32(bars.kempty<S>(i), 2);
      tc::mbar_init_u32(bars.vfull<S>(i), 1);
      tc::mbar_init_u32(bars.vempty<S>(i), 2);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init_u32(bars.sfull<S>(i), 1);
      tc::mbar_init_u32(bars.sfree<S>(i), 4);
      tc::mbar_init_u32(bars.pfull<S>(i), 4);
      tc::mbar_init_u32(bars.pvdone<S>(i), 1);
      tc::mbar_init_u32(bars.qfull<S>(i), 4);
    }
    for (int i = 0; i < S; ++i) tc::mbar_init_u32(bars.vready<S>(i), 1);
    for (int i = 0; i < C::kTrees; ++i) tc::mbar_init_u32(bars.paths<S>(i), 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init_u32(bars.drain<S>(i), 1);
    for (int i = 0; i < kMasks; ++i) tc::mbar_init_u32(bars.mask<S>(i), 1);
    tc::mbar_init_u32(bars.other<S>(), 4);
    tc::mbar_init_u32(bars.joined<S>(), 4);
    odd_flag = 0;
    stop = 0;
    mbar_init_fence();
  }
  if (warp == 8) tc::tmem_alloc(smem_addr(&tmem_slot), 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const int g = a.Hq / a.Hkv, rows_all = a.N * g;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 10) {
      // ---- loads ----
      if (lane == 0) {
        tc::prefetch_tmap(&maps.k);
        tc::prefetch_tmap(&maps.v);
      }
      const int page = 1 << a.page_shift, ppt = kTile >> a.page_shift;  // pages per tile
      bool ok = true;
      int it = 0, sent_v = 0;  // tiles whose K and V are on their way or there
      for (Segment sg = next_segment<Cut>(a, pref, w_begin, w_end); sg.count > 0 && ok;
           sg = next_segment<Cut>(a, pref, sg.next, w_end)) {
        const int len = cached_len(a, sg.b), ctiles = (len + kTile - 1) / kTile;
        const int *table = a.table + static_cast<int64_t>(sg.b) * a.M;
        // 32 table entries at a time, the next ones requested while these are used
        const int per = 32 >> (7 - a.page_shift);  // tiles per 32 entries
        auto entries = [&](int tile) {
          const int e = tile * ppt + lane;
          return e < a.M ? ld_act_i32(table + e) : -1;
        };
        int cur = entries(sg.first), next = entries(sg.first + per), used = 0;
        for (int i = sg.first; i < sg.first + sg.count; ++i) {
          const int s = it % S;
          const bool tree = i >= ctiles;
          // this tile's pages: lane l < ppt holds page l and its valid rows
          if (used == per) {
            cur = next;
            next = entries(i + per);
            used = 0;
          }
          const int pid = __shfl_sync(0xffffffffu, cur, (used * ppt + lane) & 31);
          ++used;
          int n = 0;
          if (!tree && lane < ppt && pid >= 0 && pid < a.P) n = max(0, min(page, len - i * kTile - lane * page));
          uint32_t bits = 0;  // lane w < 4: the valid tokens of word w
          for (int p = 0; p < ppt; ++p) {
            const int np = __shfl_sync(0xffffffffu, n, p);
            const int lo = max(p * page, 32 * lane), hi = min(p * page + np, 32 * lane + 32);
            if (hi > lo) bits |= (hi - lo == 32 ? 0xffffffffu : (1u << (hi - lo)) - 1u) << (lo & 31);
          }
          const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, n > 0));
          const uint32_t bytes = tree ? C::kOperand : boxes * page * D * 2;
          const uint32_t parity = ((it / S) & 1) ^ 1;
          ok = __all_sync(0xffffffffu, wait_room(bars.kempty<S>(s), parity, &stop, a.wait_us));
          if (!ok) break;
          if (lane < 4) masks[it % kMasks][lane] = bits;
          __syncwarp();
          if (lane == 0) {
            tc::arrive(bars.mask<S>(it % kMasks));
            tc::expect_tx(bars.kfull<S>(s), bytes);
          }
          __syncwarp();
          auto load = [&](const CUtensorMap *pages, const CUtensorMap *fresh, uint32_t dst, uint32_t bar) {
            if (tree) {
              if (lane < C::kPanels) tc::tma_load_4d(dst + lane * C::kPanel, fresh, lane * 64, 0, sg.h, sg.b, bar);
            } else if (n > 0) {
#pragma unroll
              for (int c = 0; c < C::kPanels; ++c)
                tc::tma_load_4d(dst + c * C::kPanel + lane * page * 128, pages, c * 64, 0, sg.h, pid, bar);
            }
          };
          load(&maps.k, &maps.k_new, k0 + s * C::kOperand, bars.kfull<S>(s));
          ++it;
          ok = __all_sync(0xffffffffu, wait_room(bars.vempty<S>(s), parity, &stop, a.wait_us));
          if (!ok) break;
          if (lane == 0) tc::expect_tx(bars.vfull<S>(s), bytes);
          __syncwarp();
          load(&maps.v, &maps.v_new, v0 + s * C::kOperand, bars.vfull<S>(s));
          sent_v = it;
        }
      }
      if (!ok) {
        if (lane == 0) give_up(1);
        // copies in flight land before the CTA's shared memory goes away
        for (int j = max(0, it - S); j < it; ++j) drain(bars.kfull<S>(j % S), (j / S) & 1);
        for (int j = max(0, sent_v - S); j < sent_v; ++j) drain(bars.vfull<S>(j % S), (j / S) & 1);
      }
    } else if (warp < 10) {
      // ---- MMAs of stream `s`: the warp stays converged, an elected lane issues. (One warp for
      // both streams was what bound the kernel: its instructions share their scheduler with
      // two softmax warps, and each stream waited for the other one's turn.) A wait names a
      // phase by its parity alone, so neither stream may get two phases away from a slot: each
      // goes through all tiles in order, and waits for and releases those of the other too. ----
      const int s = warp - 8;
      constexpr uint32_t idesc_s = tc::idesc_bf16_f32(kTile, C::kScores);
      constexpr uint32_t idesc_o = tc::idesc_bf16_f32(kTile, D) | (1u << 16);  // B (V) is MN-major
      bool ok = true;
      int it0 = 0;
      bool owed = false;  // V of the last segment's last tile is still to be released
      uint32_t pc = 0, qc = 0, sn = 0;
      auto pass_k = [&](int it) {
        ok &= wait_phase(bars.kfull<S>(it % S), (it / S) & 1);
        tc::arrive_if(lane == 0, bars.kempty<S>(it % S));
      };
      auto pass_v = [&](int it) {
        ok &= wait_phase(bars.vready<S>(it % S), (it / S) & 1);
        tc::arrive_if(lane == 0, bars.vempty<S>(it % S));
      };
      for (Segment sg = next_segment<Cut>(a, pref, w_begin, w_end); uniform(sg.count) > 0;
           sg = next_segment<Cut>(a, pref, sg.next, w_end)) {
        const Streams st = streams_of(a, sg);
        const int len = uniform(cached_len(a, sg.b)), ctiles = (len + kTile - 1) / kTile;
        const int first = uniform(sg.first), n = uniform(st.n[s]);
        const bool both = uniform(st.both);
        const int it0s = it0 + (both ? 0 : s), step = both ? 1 : 2;
        auto halves = [&](int j) { return halves_of(a, first + (both ? j : 2 * j + s), ctiles, len); };
        // S of tile j: all of it (h = 0), or its half h
        auto scores = [&](int j, int h, bool last) {
          const int it = it0s + j * step, slot = it % S;
          if (!both && h == 0 && it > it0) pass_k(it - 1);
          ok &= wait_phase(bars.kfull<S>(slot), (it / S) & 1);
          if (sn > 0) ok &= wait_phase(bars.sfree<S>(s), (sn - 1) & 1);
          ++sn;
          tc::fence_after_sync();
          // a step of the start address is a step of the descriptor's low bits (16-byte units)
          const uint64_t q = tc::sdesc_kmajor_sw128(q0 + s * C::kOperand);
          const uint64_t k = tc::sdesc_kmajor_sw128(k0 + slot * C::kOperand + h * (C::kPanel / 2));
          if (tc::elect_one()) {
#pragma unroll
            for (int c = 0; c < C::kPanels; ++c)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                tc::mma_bf16(tmem + C::kTmemS + s * C::kScores, q + c * (C::kPanel >> 4) + kk * 2,
                             k + c * (C::kPanel >> 4) + kk * 2, idesc_s, c > 0 || kk > 0);
            tc::mma_commit(bars.sfull<S>(s));
            if (last) tc::mma_commit(bars.kempty<S>(slot));
          }
          __syncwarp();
        };
        auto values = [&](int j, int h, bool last) {
          const int it = it0s + j * step, slot = it % S;
          if (!both && h == 0 && it > it0) pass_v(it - 1);
          ok &= wait_phase(bars.vready<S>(slot), (it / S) & 1);
          ok &= wait_phase(bars.pfull<S>(s), pc++ & 1);
          tc::fence_after_sync();
          const uint32_t p = tmem + C::kTmemP + s * 64, o = tmem + C::kTmemO + s * D;
          const uint64_t v = tc::sdesc_mnmajor_sw128(v0 + slot * C::kOperand + h * (C::kPanel / 2), C::kPanel);
          if (tc::elect_one()) {
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                tc::mma_bf16_ts(o, p + part * 32 + kk * 8, v + kk * (2048 >> 4), idesc_o, j > 0 || h > 0 || part > 0 || kk > 0);
            tc::mma_commit(bars.pvdone<S>(s));
            if (last) tc::mma_commit(bars.vempty<S>(slot));
          }
          __syncwarp();
        };
        if (n > 0) {
          ok &= wait_phase(bars.qfull<S>(s), qc++ & 1);
          int k = halves(0);
          scores(0, 0, C::kScores == kTile || k == 1);
          if (owed) pass_v(it0 - 1);
          owed = false;
          // the S that follows goes out before the P V of the last half that the present S
          // holds: it runs while that half's softmax does, and the softmax never waits for it
          for (int j = 0; j < n; ++j) {
            const int next = j + 1 < n ? halves(j + 1) : 0;
            for (int h = 0; h < k; ++h) {
              if (C::kScores < kTile && h + 1 < k) scores(j, h + 1, h + 2 == k);
              else if (h + 1 == k && next > 0) scores(j + 1, 0, C::kScores == kTile || next == 1);
              values(j, h, h + 1 == k);
            }
            k = next;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
        }
        it0 += uniform(sg.count);
        if (!both && ((sg.count - 1) & 1) != s) {  // the last tile is the other stream's
          pass_k(it0 - 1);
          // its V once the next segment's first K is on its way
          if (owed) pass_v(it0 - 2);
          owed = true;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      if (!ok && lane == 0) give_up(2);
      // every MMA issued is done before TMEM is freed
      if (tc::elect_one()) tc::mma_commit(bars.drain<S>(s));
      __syncwarp();
      drain(bars.drain<S>(s), 0);
      __syncwarp();
    } else {
      // ---- preparation: warp 11 ----
      bool ok = true;
      int it = 0, trees_done = 0;
      for (Segment sg = next_segment<Cut>(a, pref, w_begin, w_end); sg.count > 0 && ok;
           sg = next_segment<Cut>(a, pref, sg.next, w_end)) {
        const int ctiles = (cached_len(a, sg.b) + kTile - 1) / kTile;
        TreePaths &tree = trees[trees_done % C::kTrees];
        if (sg.first + sg.count > ctiles) {
          tree_paths(tree, a.parents + static_cast<int64_t>(sg.b) * a.N, a.N);
          tc::arrive_if(lane == 0, bars.paths<S>(trees_done % C::kTrees));
          ++trees_done;
        }
        for (int i = sg.first; i < sg.first + sg.count; ++i, ++it) {
          const int slot = it % S;
          ok = __all_sync(0xffffffffu, wait_phase(bars.vfull<S>(slot), (it / S) & 1));
          if (!ok) break;
          const bool nodes = i >= ctiles;
          const uint4 valid = *reinterpret_cast<const uint4 *>(masks[it % kMasks]);
          if (nodes || (valid.x & valid.y & valid.z & valid.w) != 0xffffffffu) {
            // rows of V that hold nothing are zeroed, and so are a node's values that are not
            // finite (0 * inf is not 0; rows that see them get them added at the end)
            bool odd = false;
#pragma unroll 1
            for (int r = lane; r < kTile; r += 32) {
              const bool keep = nodes ? tree.up[r] == -1 : masks[it % kMasks][r >> 5] >> (r & 31) & 1u;
              if (keep && !nodes) continue;
              uint8_t *vrow = smem + 2 * C::kOperand + (S + slot) * C::kOperand + r * 128;
#pragma unroll
              for (int c = 0; c < D / 8; ++c) {
                // lanes start at different pieces of their rows: no bank conflicts
                uint4 *e = reinterpret_cast<uint4 *>(vrow + (c >> 3) * C::kPanel + (((c & 7) ^ (r & 7)) << 4));
                uint4 y = keep ? *e : make_uint4(0, 0, 0, 0);
                bool change = !keep;
                if (keep) {
                  uint32_t *u = reinterpret_cast<uint32_t *>(&y);
#pragma unroll
                  for (int q = 0; q < 4; ++q) {
                    if ((u[q] & 0x7f80u) == 0x7f80u) u[q] &= 0xffff0000u, change = odd = true;
                    if ((u[q] & 0x7f800000u) == 0x7f800000u) u[q] &= 0xffffu, change = odd = true;
                  }
                }
                if (change) *e = y;
              }
            }
            if (odd) atomicExch(&odd_flag, 1);
            tc::fence_proxy_async_smem();
          }
          __syncwarp();
          tc::arrive_if(lane == 0, bars.vready<S>(slot));
        }
      }
      if (!ok && lane == 0) give_up(5);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---- softmax of one stream: thread = row ----
    const int s = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t to = tmem + lanes + C::kTmemO + s * D, tp = tmem + lanes + C::kTmemP + s * 64;
    uint8_t *qs = smem + s * C::kOperand;
    bool ok = true;
    int it0 = 0;
    uint32_t sc = 0 /* S of this stream */, vc = 0 /* P V */, jc = 0;
    int trees_seen = 0;
    // The stream's rows of Q into shared memory, swizzled as TMA would write them (16-byte
    // piece c of row r at c ^ (r % 8)): 8 lanes per row and panel of 64. The first S of the
    // segment may run as soon as they are there, while the segment before is still written out.
    auto load_q = [&](const Segment &g_, const Streams &st) {
      if (st.n[s] == 0) return;
      const int own = g_.group * 256 + (st.both ? s * 128 : 0) + r;
      const int64_t off = own < rows_all ? g_.b * a.qs[0] + own / g * a.qs[1] + (g_.h * g + own % g) * a.qs[2] : -1;
      uint4 x[8 * C::kPanels];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, off, i * 4 + (lane >> 3));
#pragma unroll
        for (int c = 0; c < C::kPanels; ++c)
          x[i * C::kPanels + c] = at >= 0 ? ld_act_v4(a.q + at + c * 64 + (lane & 7) * 8) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = (warp & 3) * 32 + i * 4 + (lane >> 3);
#pragma unroll
        for (int c = 0; c < C::kPanels; ++c)
          *reinterpret_cast<uint4 *>(qs + c * C::kPanel + row * 128 + (((lane & 7) ^ (row & 7)) << 4)) =
              x[i * C::kPanels + c];
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      tc::arrive_if(lane == 0, bars.qfull<S>(s));
    };
    Segment sg = next_segment<Cut>(a, pref, w_begin, w_end);
    Streams st = streams_of(a, sg);
    if (sg.count > 0) load_q(sg, st);
    while (sg.count > 0) {
      const int b = sg.b, h = sg.h, n = st.n[s];
      const int len = cached_len(a, b), ctiles = (len + kTile - 1) / kTile;
      const bool has_tree = sg.first + sg.count > ctiles;
      const int row = sg.group * 256 + (st.both ? s * 128 : 0) + r;
      const bool live = row < rows_all;
      const int node = live ? row / g : 0, hq = h * g + (live ? row % g : 0);
      float m = -INFINITY, l = 0.f;
      uint4 path = make_uint4(0u, 0u, 0u, 0u);
      bool huge = false;
      for (int j = 0; j < n && ok; ++j) {
        const int i = sg.first + (st.both ? j : 2 * j + s), it = it0 + i - sg.first;
        const bool nodes = i >= ctiles;
        uint4 see;
#pragma unroll 1
        for (int half = 0, halves = halves_of(a, i, ctiles, len); half < halves; ++half) {
          const uint32_t ts = tmem + lanes + C::kTmemS + s * C::kScores + (C::kScores == kTile ? half * 64 : 0);
          if (half == 0 || C::kScores < kTile) ok = __all_sync(0xffffffffu, wait_phase(bars.sfull<S>(s), sc++ & 1));
          if (ok && half == 0) {
            // (the masks have barriers of their own: K's may be a phase further by now)
            ok = __all_sync(0xffffffffu, wait_phase(bars.mask<S>(it % kMasks), (it / kMasks) & 1));
            if (ok && has_tree && j == n - 1) {  // the row's path, while its table is there
              const int t = trees_seen % C::kTrees;
              ok = __all_sync(0xffffffffu, wait_phase(bars.paths<S>(t), (trees_seen / C::kTrees) & 1));
              if (ok && live) path = trees[t].bits[node];
            }
            see = nodes ? path : *reinterpret_cast<const uint4 *>(masks[it % kMasks]);
          }
          if (!ok) break;
          tc::fence_after_sync();
          uint32_t x[64];
          tc::tmem_ld64(ts, x);
          if (C::kScores < kTile || half == halves - 1) {  // S is in registers: the next one may be written
            tc::fence_before_sync();
            __syncwarp();
            tc::arrive_if(lane == 0, bars.sfree<S>(s));
          }
          const uint32_t see0 = half ? see.z : see.x, see1 = half ? see.w : see.y;
          if (nodes || (see0 & see1) != 0xffffffffu) {  // the same for all threads
#pragma unroll
            for (int t = 0; t < 64; ++t)
              if (!((t < 32 ? see0 : see1) >> (t & 31) & 1u)) x[t] = 0xff800000u;  // -inf
          }
          // the row's maximum, its factor and the probabilities
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int t = 0; t < 64; t += 2)
            mx[(t >> 1) & 3] = max3(mx[(t >> 1) & 3], __uint_as_float(x[t]), __uint_as_float(x[t + 1]));
          const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * a.scale_log2;
          const bool first = j == 0 && half == 0;
          const bool grow = first || top > m + 8.f || (m == -INFINITY && top != -INFINITY);
          if (__any_sync(0xffffffffu, grow)) {
            const float to_m = grow ? top : m;
            if (!first) {
              const float f = grow ? ex2_approx(m - to_m) : 1.f;  // ex2(-inf) = 0: nothing seen before
              l *= f;
              // O is rescaled where it lies, once this stream's P V so far are complete
              ok = __all_sync(0xffffffffu, wait_phase(bars.pvdone<S>(s), (vc - 1) & 1));
              if (!ok) break;
              tc::fence_after_sync();
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                tc::tmem_ld16(to + c, o);
#pragma unroll
                for (int q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
                tc::tmem_st16(to + c, o);
              }
            }
            m = to_m;
            // past 2^20 the fused product below would keep digits that m has lost
            huge = __any_sync(0xffffffffu, fabsf(m == -INFINITY ? 0.f : m) > 1048576.f);
          }
          float ref = m == -INFINITY ? 0.f : m, by = a.scale_log2;
          if (huge) {  // the product is rounded first
#pragma unroll
            for (int t = 0; t < 64; ++t) x[t] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(x[t]), by), ref));
            ref = 0.f;
            by = 1.f;
          }
          const uint64_t by2 = pack2(by, by), ref2 = pack2(-ref, -ref), split = pack2(kSplit, kSplit);
          uint64_t sum[4] = {0, 0, 0, 0};
          uint32_t hi[32], lo[32];
#pragma unroll
          for (int q = 0; q < 32; ++q) {
            float p0, p1;
            unpack2(fma2(pack2(__uint_as_float(x[2 * q]), __uint_as_float(x[2 * q + 1])), by2, ref2), p0, p1);
            p0 = ex2_approx(p0);
            p1 = ex2_approx(p1);
            const uint64_t p = pack2(p0, p1);
            sum[q & 3] = add2(sum[q & 3], p);
            float m0, m1;
            hi[q] = split_hi(p0, p1, m0, m1);
            unpack2(fma2(p, split, pack2(m0, m1)), p0, p1);
            lo[q] = pack_bf16x2(p0, p1);
          }
          // the P V before has read P (only one may be under way)
          if (vc > 0) {
            ok = __all_sync(0xffffffffu, wait_phase(bars.pvdone<S>(s), (vc - 1) & 1));
            if (!ok) break;
            tc::fence_after_sync();
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            tc::tmem_st16(tp + 16 * c, hi + 16 * c);
            tc::tmem_st16(tp + 32 + 16 * c, lo + 16 * c);
          }
          tc::tmem_st_wait();
          tc::fence_before_sync();
          __syncwarp();
          tc::arrive_if(lane == 0, bars.pfull<S>(s));
          ++vc;
          float s0, s1;
          unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
          l += s0 + s1;
        }
      }
      if (!ok) break;
      trees_seen += has_tree;
      const Segment next = next_segment<Cut>(a, pref, sg.next, w_end);
      const Streams nst = streams_of(a, next);
      if (next.count > 0) load_q(next, nst);  // every S of this stream is complete: Q may be replaced
      // ---- the segment's result ----
      const bool direct = sg.count == sg.tiles, join = !st.both && st.n[1] > 0;
      if (n > 0) ok = __all_sync(0xffffffffu, wait_phase(bars.pvdone<S>(s), (vc - 1) & 1));
      if (!ok) break;
      if (join && s == 1) {
        other_ml[r] = make_float2(m, l);
        tc::fence_before_sync();
        __syncwarp();
        tc::arrive_if(lane == 0, bars.other<S>());
        // stream 0 reads this stream's O from TMEM before the next segment overwrites it
        ok = __all_sync(0xffffffffu, wait_phase(bars.joined<S>(), jc++ & 1));
        if (!ok) break;
        tc::fence_after_sync();
      } else if (n > 0) {
        float f0 = 1.f, f1 = 0.f;
        if (join) {
          ok = __all_sync(0xffffffffu, wait_phase(bars.other<S>(), jc++ & 1));
          if (!ok) break;
          const float2 o = other_ml[r];
          const float M = fmaxf(m, o.x);
          f0 = rescale(m, M);
          f1 = rescale(o.x, M);
          l = l * f0 + o.y * f1;
          m = M;
        }
        tc::fence_after_sync();
        const bool dead = has_tree && (path.x | path.y | path.z | path.w) == 0;
        const bool odd = has_tree && *reinterpret_cast<volatile int *>(&odd_flag) != 0;
        const float inv = l == 0.f || dead ? 0.f : 1.f / l;
        uint16_t *dst = a.out + b * a.os[0] + node * a.os[1] + hq * a.os[2];
        float *part = a.ws + ((static_cast<int64_t>(blockIdx.x) * 2 + (sg.first == 0 ? 1 : 0)) * 2 + s) * C::kPart;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tc::tmem_ld32(to + c, o);
          if (join) {
            uint32_t o1[32];
            tc::tmem_ld32(to + D + c, o1);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = __float_as_uint(__uint_as_float(o[e]) * f0 + __uint_as_float(o1[e]) * f1);
          }
          if (odd && live)
            for (int j = 0; j < a.N; ++j) {
              const uint32_t word = j < 32 ? path.x : j < 64 ? path.y : j < 96 ? path.z : path.w;
              if (!(word >> (j & 31) & 1u)) continue;
              const uint16_t *v = a.v_new + b * a.ks[0] + j * a.ks[1] + h * a.ks[2] + c;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float f = bf16_bits_to_float(ld_act_u16(v + e));
                if (!isfinite(f)) o[e] = __float_as_uint(__uint_as_float(o[e]) + f);
              }
            }
          if (direct) {
            if (live)
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint32_t y[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  // a row that saw nothing (l = 0) or an unused node is zero
                  const float f0 = inv == 0.f ? 0.f : __uint_as_float(o[e + 2 * q]) * inv;
                  const float f1 = inv == 0.f ? 0.f : __uint_as_float(o[e + 2 * q + 1]) * inv;
                  y[q] = pack_bf16x2(f0, f1);
                }
                *reinterpret_cast<uint4 *>(dst + c + e) = make_uint4(y[0], y[1], y[2], y[3]);
              }
          } else {
            // column by column: the lanes of a warp write 128 contiguous bytes
#pragma unroll
            for (int e = 0; e < 32; ++e) part[(c + e) * kTile + r] = __uint_as_float(o[e]);
          }
        }
        if (!direct) {
          part[kTile * D + 2 * r] = m;
          part[kTile * D + 2 * r + 1] = dead ? -1.f : l;  // -1: the join kernel writes zeros
        }
        if (join) {
          tc::fence_before_sync();
          __syncwarp();
          tc::arrive_if(lane == 0, bars.joined<S>());
        }
      }
      it0 += sg.count;
      sg = next;
      st = nst;
    }
    if (!ok && lane == 0) give_up(3u + s);
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 8) tc::tmem_free(tmem, 512);
}

// Joins the partials of 32 rows of one unit, in the order of its tiles: lane = row, a warp
// per D / 8 dimensions, kJoin pieces loaded at a time.
template <int D>
__global__ void __launch_bounds__(256) tree_tc_join_kernel(TreeArgs a, int ctas) {
  using C = Cfg<D>;
  constexpr int kDims = D / 8, kJoin = 32 / kDims;
  pdl_launch_dependents();
  pdl_wait();
  const int per = a.Hkv * a.groups, g = a.Hq / a.Hkv;
  const int b = blockIdx.x / per, unit = blockIdx.x % per, h = unit / a.groups, group = unit % a.groups;
  const int rows = min(256, a.N * g - group * 256), first = blockIdx.y * 32;
  if (first >= rows) return;
  const UnitSpan sp = find_span<Cut, 256>(a, b, unit, ctas);
  if (sp.c0 == sp.c1) return;  // written by the piece that held it
  const int ru = first + (threadIdx.x & 31), d0 = (threadIdx.x >> 5) * kDims;
  const int r = ru % 128, s = ru / 128;
  float M = -INFINITY, L = 0.f, O[kDims];
#pragma unroll
  for (int e = 0; e < kDims; ++e) O[e] = 0.f;
  bool dead = false;
  for (int c = sp.c0; c <= sp.c1; c += kJoin) {
    float2 ml[kJoin];
    float o[kJoin][kDims];
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      const bool in = c + i <= sp.c1;
      const float *part = a.ws + ((static_cast<int64_t>(in ? c + i : sp.c0) * 2 + (c + i == sp.c0 || !in ? 1 : 0)) * 2 + s) * C::kPart;
      ml[i] = __ldcg(reinterpret_cast<const float2 *>(part + kTile * D + 2 * r));
#pragma unroll
      for (int e = 0; e < kDims; ++e) o[i][e] = __ldcg(part + (d0 + e) * kTile + r);
      if (!in) {
        ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int e = 0; e < kDims; ++e) o[i][e] = 0.f;
      }
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) top = fmaxf(top, ml[i].x);
    const float f0 = rescale(M, top);
    M = top;
    L *= f0;
#pragma unroll
    for (int e = 0; e < kDims; ++e) O[e] *= f0;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      const float f = rescale(ml[i].x, M);
      dead |= ml[i].y < 0.f;
      L += ml[i].y * f;
#pragma unroll
      for (int e = 0; e < kDims; ++e) O[e] += o[i][e] * f;
    }
  }
  if (ru >= rows) return;
  const int row = group * 256 + ru;
  uint16_t *dst = a.out + b * a.os[0] + row / g * a.os[1] + (h * g + row % g) * a.os[2] + d0;
#pragma unroll
  for (int e = 0; e < kDims; ++e) O[e] = dead ? 0.f : normalised(O[e], L);
#pragma unroll
  for (int e = 0; e < kDims; e += 8)
    *reinterpret_cast<uint4 *>(dst + e) = make_uint4(pack_bf16x2(O[e], O[e + 1]), pack_bf16x2(O[e + 2], O[e + 3]),
                                                     pack_bf16x2(O[e + 4], O[e + 5]), pack_bf16x2(O[e + 6], O[e + 7]));
}

static int make_map(CUtensorMap *m, const void *ptr, const uint64_t (&dims)[4], const uint64_t (&strides)[3], int rows) {
  auto fn = gemm::encode_fn();
  if (!fn) return IRON_ERR_UNSUPPORTED;
  cuuint64_t d[4] = {dims[0], dims[1], dims[2], dims[3]}, st[3] = {strides[0], strides[1], strides[2]};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1}, es[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(ptr), d, st, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? IRON_OK
             : IRON_ERR_ARG;
}

template <int D>
static int launch_tc(TreeArgs a, cudaStream_t s) {
  using C = Cfg<D>;
  static PerDeviceOnce once;
  const int st0 = once.run([] {
    return call_status(cudaFuncSetAttribute(tree_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  });
  if (st0 != IRON_OK) return st0;
  a.groups = (a.N * (a.Hq / a.Hkv) + 255) / 256;
  Maps maps;
  const uint64_t page = 1ull << a.page_shift, B = a.B, N = a.N, H = a.Hkv;
  const uint64_t pd[4] = {D, page, H, static_cast<uint64_t>(a.P)}, ps[3] = {D * 2, page * D * 2, H * page * D * 2};
  // a dimension of one element may have any stride: give TMA one that it takes
  auto step = [](int64_t stride, uint64_t n) { return n > 1 ? static_cast<uint64_t>(stride) * 2 : 16ull; };
  const uint64_t nd[4] = {D, N, H, B}, ns[3] = {step(a.ks[1], N), step(a.ks[2], H), step(a.ks[0], B)};
  int st = make_map(&maps.k, a.k, pd, ps, static_cast<int>(page));
  if (st == IRON_OK) st = make_map(&maps.v, a.v, pd, ps, static_cast<int>(page));
  if (st == IRON_OK) st = make_map(&maps.k_new, a.k_new, nd, ns, kTile);
  if (st == IRON_OK) st = make_map(&maps.v_new, a.v_new, nd, ns, kTile);
  if (st != IRON_OK) return st;
  const int ctas = sm_count();
  st = launch(tree_tc_kernel<D>, dim3(ctas), dim3(kThreads), C::kSmem, s, true, maps, a);
  if (st != IRON_OK) return st;
  const int rows = a.N * (a.Hq / a.Hkv);
  return launch(tree_tc_join_kernel<D>, dim3(a.B * a.Hkv * a.groups, ((rows < 256 ? rows : 256) + 31) / 32), dim3(256), 0, s,
                true, a, ctas);
}

}  // namespace treetc

size_t tree_tc_workspace(int head_dim) {
  const size_t part = head_dim == 128 ? treetc::Cfg<128>::kPart : treetc::Cfg<64>::kPart;
  return static_cast<size_t>(sm_count()) * 4 * part * sizeof(float);
}

int tree_tc_launch(TreeArgs a, int head_dim, cudaStream_t s) {
  return head_dim == 128 ? treetc::launch_tc<128>(a, s) : treetc::launch_tc<64>(a, s);
}

}  // namespace iron

static std::atomic<unsigned> g_tree_wait_us{2000000};

unsigned iron::tree_wait_us() { return g_tree_wait_us.load(std::memory_order_relaxed); }

extern "C" int iron_tree_attn_set_wait_us(unsigned limit_us) {
  g_tree_wait_us.store(limit_us, std::memory_order_relaxed);
  return IRON_OK;
}

extern "C" int iron_tree_attn_status(int reset) {
  // the copies below run on the default stream, which other streams need not wait for
  if (cudaDeviceSynchronize() != cudaSuccess) return iron::launch_status();
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, iron::g_tree_status, sizeof(v)) != cudaSuccess) return iron::launch_status();
  if (reset) {
    const unsigned z = 0;
    if (cudaMemcpyToSymbol(iron::g_tree_status, &z, sizeof(z)) != cudaSuccess) return iron::launch_status();
  }
  return v ? IRON_ERR_TIMEOUT : IRON_OK;
}
