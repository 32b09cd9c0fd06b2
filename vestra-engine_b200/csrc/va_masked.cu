// Masked attention over packed documents, head_dim 64, on tcgen05 tensor cores.
//
//   out_i = sum_j p_ij V_j / sum_j p_ij,  p_ij = exp(score_ij - max), j < limit_i
//   score_ij = cap tanh(scale q_i.k_j / cap) - slope_h |f(P_i) - f(j)|
// Every mask the operator offers (documents, frame-causal, prefix) leaves a row the first
// limit_i keys of its document, and limit_i does not fall with i, so a query tile needs the
// keys [0, limit of its last row), and a 128-key tile is compared element by element only
// where some row's limit lies inside or before it.
//
// CTA = one tile of 128 query rows of one key head: tile_tokens tokens x the `group` query
// heads that share the key head (one 3-D TMA box), so shared key heads read K and V once
// and a single token still fills as many rows as it has heads.  8 warps, two CTAs per SM
// (TMEM 256 columns and at most 100 KB of shared memory each), so that one CTA's
// exponentials cover the other's waits:
//   warp 0    TMA producer: Q, then K_j (3 stages) and V_j (2 stages)
//   warp 1    TMEM owner and UMMA issuer; in a document's last tile it first zeroes the V rows
//             past the document (a masked probability is 0, but 0 x NaN is not)
//   warps 4-7 softmax, one query row per thread
// TMEM: S [0, 128) F32, P [128, 192) packed 16-bit pairs, O [192, 256) F32.  The chain per
// key tile is QK(j+2) | softmax(j) | PV(j) as in the layer path's one-tile kernel.
//
// Few query tiles leave SMs idle, so a tile's keys can be cut over a cluster of CTAs; the
// partial rows meet through distributed shared memory in rank order: no workspace, no
// second launch, the same bits on every run.
#include <algorithm>
#include <queue>
#include <vector>

#include "va_internal.h"
#include "va_ptx.cuh"

namespace va {

namespace {

constexpr int kTile = 128;
constexpr int kHeadDim = 64;
constexpr int kThreads = 256;
constexpr int kKStages = 3;
constexpr int kVStages = 2;
constexpr uint32_t kTileBytes = kTile * kHeadDim * 2;
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 192;
constexpr int kMaxSplits = 16;

struct Smem {
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kK = kTileBytes;
  static constexpr uint32_t kV = kK + kKStages * kTileBytes;
  static constexpr uint32_t kBar = kV + kVStages * kTileBytes;
  // q_full, k_full[3], k_empty[3], v_full[2], v_empty[2], s_full, s_free, p_full, pv_done, o_final
  static constexpr uint32_t kNumBars = 1 + 2 * kKStages + 2 * kVStages + 5;
  static constexpr uint32_t kMisc = kBar + 8 * kNumBars;
  static constexpr uint32_t kMl = kMisc + 64;  // split tiles: (maximum, sum) per row
  static constexpr uint32_t kBytes = kMl + 2 * kTile * 4;
  static constexpr uint32_t kLaunchBytes = kBytes + 1024;
  // A split tile's unnormalised rows [128][64] F32 lie over Q and K stage 0, which nothing
  // reads once the last product is done; 16-byte chunk c of row r at chunk c ^ (r & 15).
  static constexpr uint32_t kPart = 0;
};
static_assert(2 * (Smem::kLaunchBytes + 1024) <= 228 * 1024, "two CTAs per SM");
static_assert(kTile * kHeadDim * 4 <= (1 + kKStages) * kTileBytes, "partial rows fit");

struct Ctl {
  uint32_t base;
  uint8_t* smem;
  __device__ uint32_t bar(int i) const { return base + Smem::kBar + 8u * i; }
  __device__ uint32_t q_full() const { return bar(0); }
  __device__ uint32_t k_full(int s) const { return bar(1 + s); }
  __device__ uint32_t k_empty(int s) const { return bar(1 + kKStages + s); }
  __device__ uint32_t v_full(int s) const { return bar(1 + 2 * kKStages + s); }
  __device__ uint32_t v_empty(int s) const { return bar(1 + 2 * kKStages + kVStages + s); }
  __device__ uint32_t s_full() const { return bar(Smem::kNumBars - 5); }
  __device__ uint32_t s_free() const { return bar(Smem::kNumBars - 4); }
  __device__ uint32_t p_full() const { return bar(Smem::kNumBars - 3); }
  __device__ uint32_t pv_done() const { return bar(Smem::kNumBars - 2); }
  __device__ uint32_t o_final() const { return bar(Smem::kNumBars - 1); }
  __device__ int* misc(int i) const { return reinterpret_cast<int*>(smem + Smem::kMisc) + i; }
  __device__ uint32_t* tmem_slot() const { return reinterpret_cast<uint32_t*>(misc(0)); }
  __device__ volatile int* abort_flag() const { return misc(1); }
  __device__ volatile int* k_issued() const { return misc(2); }
  __device__ volatile int* k_consumed() const { return misc(3); }
  __device__ volatile int* v_issued() const { return misc(4); }
  __device__ volatile int* v_consumed() const { return misc(5); }
  __device__ volatile int* mma_done() const { return misc(6); }
  __device__ float* ml() const { return reinterpret_cast<float*>(smem + Smem::kMl); }
  __device__ uint32_t sQ() const { return base + Smem::kQ; }
  __device__ uint32_t sK(int s) const { return base + Smem::kK + s * kTileBytes; }
  __device__ uint32_t sV(int s) const { return base + Smem::kV + s * kTileBytes; }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > kWaitLimitNs) break;
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// This CTA's tile and its key tiles [t0, t0 + n).
struct Geom {
  MaskedItem it;
  int kvh, rank, t0, n, rows;
};
__device__ __forceinline__ Geom make_geom(const MaskedArgs& a) {
  Geom g;
  int u = static_cast<int>(blockIdx.x);
  g.rank = u % a.splits;
  u /= a.splits;
  g.kvh = u % a.t.kv_heads;
  g.it = a.item[u / a.t.kv_heads];
  const int total = (g.it.keys + kTile - 1) / kTile;
  g.t0 = static_cast<int>(static_cast<int64_t>(g.rank) * total / a.splits);
  g.n = static_cast<int>(static_cast<int64_t>(g.rank + 1) * total / a.splits) - g.t0;
  g.rows = g.it.tokens * a.group;
  return g;
}

__device__ __forceinline__ void run_producer(const Ctl& c, const Geom& g, const MaskedArgs& a,
                                             const CUtensorMap* mq, const CUtensorMap* mk,
                                             const CUtensorMap* mv, int* err) {
  if (g.n == 0) return;
  volatile int* abort_flag = c.abort_flag();
  // The box always brings tile_tokens x group rows; past the tensor's end they are zeros.
  mbar_arrive_expect_tx(c.q_full(), a.tile_tokens * a.group * kHeadDim * 2);
  tma_load_3d(c.sQ(), mq, c.q_full(), 0, g.kvh * a.group, g.it.q_row);
  auto load_k = [&](int j) {
    const int s = j % kKStages;
    if (!mbar_wait(c.k_empty(s), ((j / kKStages) & 1) ^ 1, abort_flag, err, kDevTimeoutProducer)) return false;
    mbar_arrive_expect_tx(c.k_full(s), kTileBytes);
    tma_load_3d(c.sK(s), mk, c.k_full(s), 0, g.kvh, g.it.k_row + (g.t0 + j) * kTile);
    *c.k_issued() = j + 1;
    return true;
  };
  auto load_v = [&](int j) {
    const int s = j % kVStages;
    if (!mbar_wait(c.v_empty(s), ((j / kVStages) & 1) ^ 1, abort_flag, err, kDevTimeoutProducer)) return false;
    mbar_arrive_expect_tx(c.v_full(s), kTileBytes);
    tma_load_3d(c.sV(s), mv, c.v_full(s), 0, g.kvh, g.it.k_row + (g.t0 + j) * kTile);
    *c.v_issued() = j + 1;
    return true;
  };
  bool ok = load_k(0);
  if (ok && g.n > 1) ok = load_k(1);
  for (int j = 0; ok && j < g.n; ++j) {
    ok = load_v(j);
    if (ok && j + 2 < g.n) ok = load_k(j + 2);
  }
}

// UMMA issuer (the whole warp waits, lane 0 issues): QK(0), QK(1), then per key tile PV(j), QK(j+2).
template <bool kF16>
__device__ __forceinline__ void run_mma(const Ctl& c, const Geom& g, uint32_t tmem, int* err) {
  constexpr uint32_t idesc_qk = kF16 ? idesc_f16_f32(kTile, kTile, false, false)
                                     : idesc_bf16_f32(kTile, kTile, false, false);
  constexpr uint32_t idesc_pv = kF16 ? idesc_f16_f32(kTile, kHeadDim, false, true)
                                     : idesc_bf16_f32(kTile, kHeadDim, false, true);
  constexpr uint64_t kStageStep = kTileBytes >> 4;  // descriptor start-field step per stage
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = c.abort_flag();
  const uint64_t dq = sdesc_sw128(c.sQ(), 16, 1024);
  const uint64_t dk0 = sdesc_sw128(c.sK(0), 16, 1024);
  const uint64_t dv0 = sdesc_sw128(c.sV(0), 8192, 1024);  // V tile, MN-major
  const uint32_t tS = tmem + kColS, tP = tmem + kColP, tO = tmem + kColO;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    const bool r = mbar_wait(bar, parity, abort_flag, err, kDevTimeoutMma);
    return __all_sync(0xffffffffu, r) != 0;
  };
  auto qk = [&](int jj) {
    const int s = jj % kKStages;
    bool r = wait(c.k_full(s), (jj / kKStages) & 1);
    if (r && lane == 0) *c.k_consumed() = jj + 1;
    if (r && jj > 0) r = wait(c.s_free(), (jj - 1) & 1);
    if (r && lane == 0) {
      tc_fence_after();
      umma_ss_k64(tS, dq, dk0 + s * kStageStep, idesc_qk, 0u);
      tc_commit(c.s_full());
      tc_commit(c.k_empty(s));
    }
    __syncwarp();
    return r;
  };
  bool ok = g.n > 0 && wait(c.q_full(), 0);
  if (ok) ok = qk(0);
  if (ok && g.n > 1) ok = qk(1);
  for (int j = 0; ok && j < g.n; ++j) {
    const int s = j % kVStages;
    ok = wait(c.v_full(s), (j / kVStages) & 1);
    if (ok && lane == 0) *c.v_consumed() = j + 1;
    if (!ok) break;
    const int valid = g.it.doc_keys - (g.t0 + j) * kTile;  // rows of this V tile inside the document
    if (valid < kTile) {
      for (int i = valid * 8 + lane; i < kTile * 8; i += 32) st_shared_v4(c.sV(s) + i * 16, make_uint4(0, 0, 0, 0));
      fence_proxy_async_smem();
      __syncwarp();
    }
    ok = wait(c.p_full(), j & 1);
    if (!ok) break;
    if (lane == 0) {
      tc_fence_after();
      umma_ts_k128_mn(tO, tP, dv0 + s * kStageStep, idesc_pv, j > 0 ? 1u : 0u);
      tc_commit(c.pv_done());
      tc_commit(c.v_empty(s));
    }
    __syncwarp();
    if (j + 2 < g.n) ok = qk(j + 2);
  }
  // Always committed, also after an abort (the teardown waits for it before TMEM is freed).
  if (lane == 0) {
    tc_commit(c.o_final());
    *c.mma_done() = 1;
  }
  __syncwarp();
}

__device__ __forceinline__ void store_row16(uint8_t* dst, const float* o, float inv, bool f16) {
  uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = o[8 * c + 2 * i] * inv, hi = o[8 * c + 2 * i + 1] * inv;
      w[i] = f16 ? f16x2_from_f32(lo, hi) : pack_bf16x2(lo, hi);
    }
    d[c] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <bool kF16, bool kCap, bool kBias>
__global__ void __launch_bounds__(kThreads, 2)
    masked_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ MaskedArgs a, int* err) {
  // A row's probabilities are 2^(x - m + kOffset), m at most 2^kGrow behind the row's maximum:
  // at most 2^8 in bf16.  f16 ends at 2^16 and loses what is below 2^-24, so there the offset
  // lifts the row to at most 2^15 and the smallest kept probability is 2^-35 of the largest.
  constexpr float kGrow = kF16 ? 4.0f : 8.0f;
  constexpr float kOffset = kF16 ? 11.0f : 0.0f;
  extern __shared__ uint8_t smem_raw[];
  Ctl c;
  {
    const uint32_t raw = smem_u32(smem_raw);
    c.base = (raw + 1023u) & ~1023u;
    c.smem = smem_raw + (c.base - raw);
  }
  const Geom g = make_geom(a);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(c.q_full(), 1);
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(c.k_full(s), 1);
      mbar_init(c.k_empty(s), 1);
    }
    for (int s = 0; s < kVStages; ++s) {
      mbar_init(c.v_full(s), 1);
      mbar_init(c.v_empty(s), 1);
    }
    mbar_init(c.s_full(), 1);
    mbar_init(c.s_free(), 128);
    mbar_init(c.p_full(), 128);
    mbar_init(c.pv_done(), 1);
    mbar_init(c.o_final(), 1);
    for (int i = 1; i < 7; ++i) *c.misc(i) = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(c.tmem_slot()), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *c.tmem_slot();
  volatile int* abort_flag = c.abort_flag();

  if (warp < 4) {
    if (warp == 0) {
      if (lane == 0) run_producer(c, g, a, &map_q, &map_k, &map_v, err);
      __syncwarp();
    } else if (warp == 1) {
      run_mma<kF16>(c, g, tmem, err);
    }
    if (a.splits > 1) {
      cluster_sync();  // partial rows written
      cluster_sync();  // and read
    }
  } else {
    const int quad = warp & 3;
    const int r = quad * 32 + lane;  // row of the tile
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t tS = tmem + lane_off + kColS, tP = tmem + lane_off + kColP, tO = tmem + lane_off + kColO;
    const int tok = r / a.group;
    const int head = g.kvh * a.group + (r - tok * a.group);
    const bool live = r < g.rows;
    const bool warp_live = quad * 32 < g.rows;
    const int pos = g.it.first + tok;  // key position of the row
    // floor(pos / frame), also below zero
    const int frame = pos >= 0 ? pos / a.t.frame : -1 - (-1 - pos) / a.t.frame;
    int limit = g.it.doc_keys;
    if (a.t.causal) {
      const int64_t e = (static_cast<int64_t>(frame) + 1) * a.t.frame;
      limit = static_cast<int>(max(static_cast<int64_t>(0),
                                   min(static_cast<int64_t>(limit), max(e, static_cast<int64_t>(g.it.prefix)))));
    }
    if (!live) limit = 0;
    const float slope = kBias ? a.slopes[live ? head : 0] : 0.0f;
    const float fpos = static_cast<float>(frame);
    const float sl2 = a.t.scale_log2;
    float m = -INFINITY;  // running maximum, log2 domain, may lag by kGrow
    float l = 0.0f;
    bool ok = true;
    for (int j = 0; j < g.n; ++j) {
      ok = mbar_wait(c.s_full(), j & 1, abort_flag, err, kDevTimeoutConsumer);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (!warp_live) {
        // Rows nobody reads: hand the tile on, P only once PV(j-1) is done, as the live warps
        // do, so that this arrival counts for tile j.
        mbar_arrive(c.s_free());
        if (j > 0) {
          ok = mbar_wait(c.pv_done(), (j - 1) & 1, abort_flag, err, kDevTimeoutConsumer);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        mbar_arrive(c.p_full());
        continue;
      }
      tc_fence_after();
      float s[128];
#pragma unroll
      for (int q = 0; q < 128; q += 32) tmem_ld32(tS + q, s + q);
      tc_fence_before();
      mbar_arrive(c.s_free());  // QK of the next tile may overwrite S
      const int k0 = (g.t0 + j) * kTile;
      const int lim = limit - k0;
      if constexpr (kCap) {
        // cap log2(e) tanh(z) = cap log2(e) (1 - 2 / (1 + e^(2z)))
#pragma unroll
        for (int q = 0; q < 128; ++q)
          s[q] = a.t.cap_out * (1.0f - __fdividef(2.0f, 1.0f + ex2(s[q] * a.t.cap_in)));
      }
      if constexpr (kBias) {
        const float4* ft = reinterpret_cast<const float4*>(a.frame_of + k0);
#pragma unroll
        for (int q = 0; q < 32; ++q) {
          const float4 f = __ldg(ft + q);
          const float w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[4 * q + e] = fmaf(-slope, fabsf(fpos - w[e]), kCap ? s[4 * q + e] : s[4 * q + e] * sl2);
        }
      }
      constexpr bool kScaled = kCap || kBias;  // s already in the log2 domain
      if (__any_sync(0xffffffffu, lim < kTile)) {
#pragma unroll
        for (int q = 0; q < 128; ++q)
          if (q >= lim) s[q] = -INFINITY;
      }
      // Row maximum as a tree of 3-input maxima.
      float mx8[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mx8[i] = max3f(s[i], s[8 + i], s[16 + i]);
#pragma unroll
      for (int q = 24; q < 120; q += 16)
#pragma unroll
        for (int i = 0; i < 8; ++i) mx8[i] = max3f(mx8[i], s[q + i], s[q + 8 + i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) mx8[i] = fmaxf(mx8[i], s[120 + i]);
      float mx = max3f(max3f(mx8[0], mx8[1], mx8[2]), max3f(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
      if (!kScaled) mx *= sl2;
      const bool grow = mx > m + kGrow;  // m = -inf: as soon as a key is seen
      const float m_new = grow ? mx : m;
      const float alpha = grow ? ex2(m - m_new) : 1.0f;
      const float neg = m_new == -INFINITY ? 0.0f : kOffset - m_new;  // no key yet: every x is -inf
      const uint64_t sc2 = f32x2_pack(sl2, sl2), neg2 = f32x2_pack(neg, neg);
      uint32_t pk[64];
      uint64_t acc[4];
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const uint64_t v = f32x2_pack(s[2 * i], s[2 * i + 1]);
        float x0, x1;
        f32x2_unpack(kScaled ? f32x2_add(v, neg2) : f32x2_fma(v, sc2, neg2), x0, x1);
        const float p0 = ex2(x0), p1 = ex2(x1);
        const uint64_t pp = f32x2_pack(p0, p1);
        acc[i & 3] = i < 4 ? pp : f32x2_add(acc[i & 3], pp);
        pk[i] = kF16 ? f16x2_from_f32(p0, p1) : pack_bf16x2(p0, p1);
      }
      float s0, s1;
      f32x2_unpack(f32x2_add(f32x2_add(acc[0], acc[1]), f32x2_add(acc[2], acc[3])), s0, s1);
      if (j > 0) {
        // PV(j-1) has finished reading P and adding into O.
        ok = mbar_wait(c.pv_done(), (j - 1) & 1, abort_flag, err, kDevTimeoutConsumer);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
      }
      tmem_st64(tP, pk);
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
        float o[64];
        tmem_ld32(tO, o);
        tmem_ld32(tO + 32, o + 32);
        uint32_t u[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) u[i] = __float_as_uint(o[i] * alpha);
        tmem_st64(tO, u);
      }
      tmem_wait_st();
      l = l * alpha + (s0 + s1);
      m = m_new;
      tc_fence_before();
      mbar_arrive(c.p_full());
    }
    if (ok && g.n > 0) {
      ok = mbar_wait(c.o_final(), 0, abort_flag, err, kDevTimeoutConsumer);
      ok = __all_sync(0xffffffffu, ok);
    }
    const bool f16 = kF16;
    uint8_t* out = static_cast<uint8_t*>(a.out.data);
    if (a.splits == 1) {
      if (ok && warp_live) {
        float o[64];
        if (g.n > 0) {
          tc_fence_after();
          tmem_ld32(tO, o);
          tmem_ld32(tO + 32, o + 32);
        }
        if (l == 0.0f) {  // no key seen
#pragma unroll
          for (int i = 0; i < 64; ++i) o[i] = 0.0f;
        }
        if (live)
          store_row16(out + 2 * ((g.it.q_row + static_cast<int64_t>(tok)) * a.out.token_stride + head * a.out.head_stride),
                      o, l == 0.0f ? 0.0f : 1.0f / l, f16);
      }
    } else {
      if (warp_live) {
        float o[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) o[i] = 0.0f;
        if (ok && g.n > 0) {
          tc_fence_after();
          tmem_ld32(tO, o);
          tmem_ld32(tO + 32, o + 32);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
          st_shared_v4(c.base + Smem::kPart + r * 256 + ((i ^ (r & 15)) << 4),
                       make_uint4(__float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]),
                                  __float_as_uint(o[4 * i + 2]), __float_as_uint(o[4 * i + 3])));
        c.ml()[2 * r] = m;
        c.ml()[2 * r + 1] = l;
      }
      __syncwarp();
      cluster_sync();
      // Rank q joins rows [q rows / splits, (q + 1) rows / splits): 16 threads a row.
      const int r0 = g.rank * g.rows / a.splits, r1 = (g.rank + 1) * g.rows / a.splits;
      const uint32_t part = c.base + Smem::kPart, ml = c.base + Smem::kMl;
      for (int i = static_cast<int>(threadIdx.x) - 128; i < (r1 - r0) * 16; i += 128) {
        const int row = r0 + (i >> 4), ch = i & 15;
        float mt = -INFINITY;
        for (int p = 0; p < a.splits; ++p) mt = fmaxf(mt, ld_cluster_v2(cluster_addr(ml + row * 8, p)).x);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float lt = 0.0f;
        for (int p = 0; p < a.splits; ++p) {
          const float2 q = ld_cluster_v2(cluster_addr(ml + row * 8, p));
          const float f = q.x == -INFINITY ? 0.0f : ex2(q.x - mt);
          const float4 v = ld_cluster_v4(cluster_addr(part + row * 256 + ((ch ^ (row & 15)) << 4), p));
          o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
          lt += f * q.y;
        }
        const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
        if (lt == 0.0f) o = make_float4(0.f, 0.f, 0.f, 0.f);
        const int t = row / a.group, h = g.kvh * a.group + (row - t * a.group);
        uint2 w;
        if (f16) {
          w = make_uint2(f16x2_from_f32(o.x * inv, o.y * inv), f16x2_from_f32(o.z * inv, o.w * inv));
        } else {
          w = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
        }
        if (ok)
          *reinterpret_cast<uint2*>(
              out + 2 * ((g.it.q_row + static_cast<int64_t>(t)) * a.out.token_stride + h * a.out.head_stride + 4 * ch)) = w;
      }
      __syncwarp();
      cluster_sync();
    }
  }
  // Drain what an abort left in flight, then free TMEM.
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *c.abort_flag()) {
    if (*c.k_issued() > 0 && *c.k_consumed() == 0) drain(c.q_full(), 0);
    for (int j = *c.k_consumed(); j < *c.k_issued(); ++j) drain(c.k_full(j % kKStages), (j / kKStages) & 1);
    for (int j = *c.v_consumed(); j < *c.v_issued(); ++j) drain(c.v_full(j % kVStages), (j / kVStages) & 1);
    if (*c.mma_done()) drain(c.o_final(), 0);
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <bool kF16, bool kCap, bool kBias>
cudaError_t launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const MaskedArgs& a,
                   int64_t blocks, int* err, cudaStream_t st) {
  auto kern = masked_attn_kernel<kF16, kCap, kBias>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem::kLaunchBytes);
  if (e == cudaSuccess && a.splits > 8)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Smem::kLaunchBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, a, err);
}

}  // namespace

// Time model of a launch in key-tile units: a CTA costs its key tiles plus kFixed (setup, first
// loads, output), a split one kJoin more; CTAs go to 2 x sms slots in grid order.
int masked_splits(const int* key_tiles, int64_t items, int kv_heads, int sms) {
  constexpr double kFixed = 4.0, kJoin = 2.0;
  const int slots = 2 * sms;
  int most = 0;
  double total = 0.0;
  for (int64_t i = 0; i < items; ++i) {
    most = std::max(most, key_tiles[i]);
    total += key_tiles[i];
  }
  // Work for many rounds: cutting it finer gains nothing that the order does not give.
  if (items * kv_heads >= 16 * static_cast<int64_t>(slots)) return 1;
  int best = 1;
  double best_time = 0.0;
  for (int s = 1; s <= kMaxSplits; s *= 2) {
    if (s > 1 && 2 * s > most) break;  // at least two tiles a CTA in the longest item
    std::priority_queue<double, std::vector<double>, std::greater<double>> free_at;
    for (int i = 0; i < slots; ++i) free_at.push(0.0);
    double end = 0.0;
    for (int64_t i = 0; i < items; ++i) {
      const double cost = static_cast<double>((key_tiles[i] + s - 1) / s) + kFixed + (s > 1 ? kJoin : 0.0);
      for (int h = 0; h < kv_heads * s; ++h) {
        const double t = free_at.top() + cost;
        free_at.pop();
        free_at.push(t);
        end = std::max(end, t);
      }
    }
    if (s == 1 || end < 0.97 * best_time) {
      best = s;
      best_time = end;
    }
  }
  return best;
}

cudaError_t launch_masked(const HeadsRef& q, const HeadsRef& k, const HeadsRef& v, int64_t q_rows, int64_t k_rows,
                          const MaskedArgs& a, int dtype, int* err, cudaStream_t st) {
  if (a.items == 0) return cudaSuccess;
  const int64_t blocks = static_cast<int64_t>(a.items) * a.t.kv_heads * a.splits;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  CUtensorMap mq, mk, mv;
  // A single head's stride is never stepped over: any legal value will do.
  auto head_bytes = [](const HeadsRef& h) { return static_cast<uint64_t>(h.heads > 1 ? h.head_stride * 2 : 128); };
  // k_rows 0 (no document has keys): the maps are never used, but must encode.
  if (!encode_tma_heads(&mq, q.data, q.heads, q_rows, head_bytes(q), q.token_stride * 2, a.group, a.tile_tokens) ||
      !encode_tma_heads(&mk, k.data, k.heads, std::max<int64_t>(k_rows, 1), head_bytes(k), k.token_stride * 2, 1, kTile) ||
      !encode_tma_heads(&mv, v.data, v.heads, std::max<int64_t>(k_rows, 1), head_bytes(v), v.token_stride * 2, 1, kTile))
    return cudaErrorInvalidValue;
  const bool f16 = dtype == kF16, cap = a.t.cap_out > 0.0f, bias = a.slopes != nullptr;
  using Fn = cudaError_t (*)(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const MaskedArgs&, int64_t,
                             int*, cudaStream_t);
  static const Fn fn[2][2][2] = {
      {{launch<false, false, false>, launch<false, false, true>}, {launch<false, true, false>, launch<false, true, true>}},
      {{launch<true, false, false>, launch<true, false, true>}, {launch<true, true, false>, launch<true, true, true>}}};
  return fn[f16][cap][bias](mq, mk, mv, a, blocks, err, st);
}

}  // namespace va
