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
// and a single token still fills as many rows as it has heads.  10 warps, two CTAs per SM
// (TMEM 256 columns and at most 100 KB of shared memory each), so that one CTA's
// exponentials cover the other's waits:
//   warp 0    TMA producer: Q, then K_j (3 stages) and V_j (2 stages)
//   warp 1    TMEM owner and UMMA issuer; in a document's last tile it first zeroes the V rows
//             past the document (a masked probability is 0, but 0 x NaN is not)
//   warps 2-9 softmax: two warps share a TMEM lane quadrant (16-lane loads), four threads a
//             row, 32 columns of two rows per thread, so that 16 warps per SM overlap their
//             loads, maxima and MUFU work (one row per thread on four warps spilled and ran at
//             half the rate)
// TMEM: S [0, 128) F32, P [128, 192) packed 16-bit pairs, O [192, 256) F32.  The chain per
// key tile is QK(j+2) | softmax(j) | PV(j) as in the layer path's one-tile kernel.
//
// Few query tiles leave SMs idle, so a tile's keys can be cut over a cluster of CTAs; the
// partial rows meet through distributed shared memory in rank order: no workspace, no
// second launch, the same bits on every run.
//
// What bounds it: this form runs all exponentials on MUFU (one per 256 FLOP, 18.3 a clock and SM: 0.46 us of a
// 128 x 128 tile at 1.965 GHz); in full waves a tile takes 0.81 us of an SM, the rest being what two CTAs do not hide
// of its chain.  MUFU is no floor of the operator: the layer path's key-split kernel gives part of the exponentials to
// FMA warps and runs the plain 10,392-token window at 811 TFLOP/s with a row maximum, this one at 724.
// Measured on B200: full waves 763 TFLOP/s; four packed f16 documents of 731 to 4,330 tokens x 12 heads 129 us
// (637 TFLOP/s); a 10,392-token window x 12 heads without a cap 458 us, with cap 30 490 to 525 (632 to 677 TFLOP/s),
// with cap 60 633, in f16 with cap 30 656, and 1084 where scores pass 0.6 of the cap (an exponential and a reciprocal
// more each); 866 new rows over 10,392 keys, cap 50, three CTAs a tile, 58 us (476), without a cap 56; causal documents
// with a distance bias, 16 / 4 heads, 87 us (490).
#include <algorithm>
#include <atomic>
#include <queue>
#include <vector>

#include "va_internal.h"
#include "va_ptx.cuh"
#include "va_stream.cuh"
#include "va_tmem16.cuh"

namespace va {

namespace {

constexpr int kTile = 128;
constexpr int kHeadDim = 64;
constexpr int kThreads = 320;
constexpr int kFirstSoftmaxWarp = 2;
constexpr int kSoftmaxThreads = 256;
constexpr int kKStages = 3;
constexpr int kVStages = 2;
constexpr uint32_t kTileBytes = kTile * kHeadDim * 2;
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 192;
constexpr int kMaxSplits = 16;
// See masked_attn_kernel: caps up to 50 (72.13 in the log2 domain), for values up to 2^kFixedValues.
constexpr float kFixedCap = 72.2f;
constexpr int kFixedKeys = 1024;
constexpr int kFixedValues = 79;

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

__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > kWaitLimitNs) break;
  }
}

// One arrival for the warp, after every lane's work before it.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
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

__device__ __forceinline__ void load_k(const Ctl& c, const Geom& g, const CUtensorMap* mk, int j) {
  const int s = j % kKStages;
  mbar_arrive_expect_tx(c.k_full(s), kTileBytes);
  tma_load_3d(c.sK(s), mk, c.k_full(s), 0, g.kvh, g.it.k_row + (g.t0 + j) * kTile);
  *c.k_issued() = j + 1;
}
__device__ __forceinline__ void load_v(const Ctl& c, const Geom& g, const CUtensorMap* mv, int j) {
  const int s = j % kVStages;
  mbar_arrive_expect_tx(c.v_full(s), kTileBytes);
  tma_load_3d(c.sV(s), mv, c.v_full(s), 0, g.kvh, g.it.k_row + (g.t0 + j) * kTile);
  *c.v_issued() = j + 1;
}

// Q, K(0), K(1) and V(0): their stages start out free.
__device__ __forceinline__ void first_loads(const Ctl& c, const Geom& g, const MaskedArgs& a, const CUtensorMap* mq,
                                            const CUtensorMap* mk, const CUtensorMap* mv) {
  // The box always brings tile_tokens x group rows; past the tensor's end they are zeros.
  mbar_arrive_expect_tx(c.q_full(), a.tile_tokens * a.group * kHeadDim * 2);
  tma_load_3d(c.sQ(), mq, c.q_full(), 0, g.kvh * a.group, g.it.q_row);
  load_k(c, g, mk, 0);
  if (g.n > 1) load_k(c, g, mk, 1);
  load_v(c, g, mv, 0);
}

// The rest of the loads (one thread), in the order the UMMA chain reads them.
__device__ __forceinline__ void run_producer(const Ctl& c, const Geom& g, const CUtensorMap* mk,
                                             const CUtensorMap* mv, int* err) {
  volatile int* abort_flag = c.abort_flag();
  for (int j = 2; j < g.n + 1; ++j) {
    if (j < g.n) {
      if (!mbar_wait(c.k_empty(j % kKStages), ((j / kKStages) & 1) ^ 1, abort_flag, err, kDevTimeoutProducer)) return;
      load_k(c, g, mk, j);
    }
    const int v = j - 1;
    if (!mbar_wait(c.v_empty(v % kVStages), ((v / kVStages) & 1) ^ 1, abort_flag, err, kDevTimeoutProducer)) return;
    load_v(c, g, mv, v);
  }
}

// UMMA issuer (the whole warp waits, lane 0 issues): QK(0), QK(1), then per key tile PV(j), QK(j+2).
template <bool kF16, bool kCap>
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
  // A warp of softmax chooses the form of the cap by the range of its scores, and rows past the tile's last may not
  // take part: they hold another document's queries (which another CTA may be overwriting, out may be q), or, where
  // the heads that share a key head do not divide 128, what an earlier CTA left.  Zeros score 0.
  if (kCap && ok && g.rows < kTile) {
    for (int i = g.rows * 8 + lane; i < kTile * 8; i += 32) st_shared_v4(c.sQ() + i * 16, make_uint4(0, 0, 0, 0));
    fence_proxy_async_smem();
    __syncwarp();
  }
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

// Maxima of the thread's two rows over its 32 columns each (3-input maxima, two chains a row).
__device__ __forceinline__ void row_maxima(const float* s, float* mx) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* v = s + 2 * i;  // pairs v[4k], v[4k + 1]
    float a = max3f(v[0], v[1], v[4]), b = max3f(v[5], v[8], v[9]);
#pragma unroll
    for (int k = 3; k < 15; k += 2) {
      a = max3f(a, v[4 * k], v[4 * k + 1]);
      b = max3f(b, v[4 * k + 4], v[4 * k + 5]);
    }
    mx[i] = max3f(a, b, fmaxf(v[60], v[61]));
  }
}

// Scores of the thread's columns (relative to its first) from lim[i] on become v.
__device__ __forceinline__ void hide(float* s, const int* lim, float v) {
#pragma unroll
  for (int k = 0; k < 16; ++k)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (8 * k + e >= lim[0]) s[4 * k + e] = v;
      if (8 * k + e >= lim[1]) s[4 * k + 2 + e] = v;
    }
}

// s <- cap log2(e) tanh(scale s / cap) + offset.  While every |s| of the warp's part of the tile is at
// most a range, by an odd polynomial on the FMA pipe: tanh(z) = z P(z^2), fitted here (reweighted
// least squares on Chebyshev nodes of z^2): P quadratic for |z| <= 0.3 (relative error 1.2e-6),
// cubic for |z| <= 0.6 (2.2e-6, and scores of at most 77, so within 1.7e-4).  Else
// cap log2(e) (1 - 2 / (1 + e^(2z))): two MUFU operations a score.
__device__ __forceinline__ float largest(const float* s) {
  float mx[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int q = 0; q < 64; q += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) mx[i] = max3f(mx[i], fabsf(s[q + 2 * i]), fabsf(s[q + 2 * i + 1]));
  // a NaN passes: the polynomials hand it on as well
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
// The polynomials of one pair of scores: kCubic for the wider range.
template <bool kCubic>
struct CapPoly {
  uint64_t k0, k1, k2, k3, off;
  __device__ __forceinline__ CapPoly(const AttnTerms& t, float offset) {
    const float* p = t.cap_poly + (kCubic ? 3 : 0);
    k0 = f32x2_pack(p[0], p[0]), k1 = f32x2_pack(p[1], p[1]), k2 = f32x2_pack(p[2], p[2]);
    if (kCubic) k3 = f32x2_pack(p[3], p[3]);
    off = f32x2_pack(offset, offset);
  }
  __device__ __forceinline__ uint64_t operator()(uint64_t v) const {
    const uint64_t u = f32x2_mul(v, v);
    const uint64_t p = f32x2_fma(kCubic ? f32x2_fma(k3, u, k2) : k2, u, k1);
    return f32x2_fma(f32x2_fma(p, u, k0), v, off);
  }
};
template <bool kCubic>
__device__ __forceinline__ void cap_poly(float* s, const AttnTerms& t, float offset) {
  const CapPoly<kCubic> poly(t, offset);
#pragma unroll
  for (int q = 0; q < 32; ++q) f32x2_unpack(poly(f32x2_pack(s[2 * q], s[2 * q + 1])), s[2 * q], s[2 * q + 1]);
}
__device__ __forceinline__ void cap_scores(float* s, const AttnTerms& t, float offset) {
  const float top = largest(s);
  if (__all_sync(0xffffffffu, top <= t.cap_range[0])) {
    cap_poly<false>(s, t, offset);
  } else if (__all_sync(0xffffffffu, top <= t.cap_range[1])) {
    cap_poly<true>(s, t, offset);
  } else {
    const float high = t.cap_out + offset, twice = -2.0f * t.cap_out;
#pragma unroll
    for (int q = 0; q < 64; ++q) s[q] = fmaf(twice, rcp(1.0f + ex2(s[q] * t.cap_in)), high);
  }
}

// s <- s (times scale log2(e) unless capped before) - slope |f(row) - f(key)|, f(x) = floor(x / frame),
// for the thread's columns k0 + c0 + 8k + {0, 1}, the rows' frame indices and slopes (times
// log2(e)) given.  Frame indices stay below 2^24, so their differences are exact.
//   frame 1: the distances step by 8 from block to block;
//   no frame starts inside the tile: one distance per row;
//   else: floor((x + 1/2) / frame) by an addition of 3 * 2^22 rounded down, x = the key's offset
//   from a frame start inside or just before the tile, so below 256 and never near a step.
// side: -1 when no visible key of the tile lies in a later frame than a row, +1 when none lies in an
// earlier one (the distance is then the difference or its negative), else 0.
template <bool kCap>
__device__ __forceinline__ void bias_scores(float* s, const AttnTerms& t, int k0, int c0, const int* frame,
                                            const float* slope, int side) {
  const uint64_t sc2 = f32x2_pack(t.scale_log2, t.scale_log2);
  uint64_t ns[2], d[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float v = side < 0 ? slope[i] : -slope[i];
    ns[i] = f32x2_pack(v, v);
  }
  auto add_bias = [&](int k, int i) {
    uint64_t v = f32x2_pack(s[4 * k + 2 * i], s[4 * k + 2 * i + 1]);
    if (!kCap) v = f32x2_mul(v, sc2);
    f32x2_unpack(f32x2_fma(d[i] & 0x7fffffff7fffffffull, ns[i], v), s[4 * k + 2 * i], s[4 * k + 2 * i + 1]);
  };
  if (t.frame == 1) {
    const uint64_t step = f32x2_pack(8.0f, 8.0f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float at = static_cast<float>(k0 + c0 - frame[i]);
      d[i] = f32x2_pack(at, at + 1.0f);
    }
    if (side != 0) {
#pragma unroll
      for (int k = 0; k < 16; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint64_t v = f32x2_pack(s[4 * k + 2 * i], s[4 * k + 2 * i + 1]);
          if (!kCap) v = f32x2_mul(v, sc2);
          f32x2_unpack(f32x2_fma(d[i], ns[i], v), s[4 * k + 2 * i], s[4 * k + 2 * i + 1]);
          d[i] = f32x2_add(d[i], step);
        }
      return;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        add_bias(k, i);
        d[i] = f32x2_add(d[i], step);
      }
    return;
  }
  if (side < 0) ns[0] ^= 0x8000000080000000ull, ns[1] ^= 0x8000000080000000ull;  // below: distances
  int base = k0 / t.frame;              // frame of the tile's first key
  int start = base * t.frame - k0;      // its start, at most 0
  if (start + t.frame >= kTile) {       // the next frame starts past the tile
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float v = static_cast<float>(base - frame[i]);
      d[i] = f32x2_pack(v, v);
    }
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) add_bias(k, i);
    return;
  }
  if (start < -kTile) base += 1, start += t.frame;  // (frame > 128)
  const float magic = 12582912.0f, inv = 1.0f / static_cast<float>(t.frame);
  const uint64_t step = f32x2_pack(8.0f, 8.0f), m2 = f32x2_pack(magic, magic), inv2 = f32x2_pack(inv, inv);
  const float x0 = static_cast<float>(c0 - start) + 0.5f;
  uint64_t x = f32x2_pack(x0, x0 + 1.0f), rel[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float v = static_cast<float>(base - frame[i]);
    rel[i] = f32x2_pack(v, v);
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    uint64_t f;
    asm("fma.rm.f32x2 %0, %1, %2, %3;" : "=l"(f) : "l"(x), "l"(inv2), "l"(m2));
    f = f32x2_sub(f, m2);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      d[i] = f32x2_add(f, rel[i]);
      add_bias(k, i);
    }
    x = f32x2_add(x, step);
  }
}

// kFixed (capped scores without a bias, bf16, cap log2(e) <= kFixedCap): every score lies in
// [-cap, cap], so the exponent's reference is the constant cap log2(e) - top instead
// of the row's maximum: probabilities lie in [2^(top - 2 kFixedCap), 2^top].  top is as high as values up to 2^79
// allow, 127 - 79 - log2(keys of the longest document): 24 for the 2^24 keys a document may have (probabilities
// from 2^-120 up, inside bf16's and F32's normal range), 34 for a 10,392-token window, so that rows whose keys all
// score near -cap keep small values (down to about 2^(4 - top); below they meet F32's smallest numbers).
// No maximum, exchange or rescaling is needed (a 10,392-token
// window 611 us against 684).  Where the row's maximum is the reference, the largest probability
// is exactly 1; here it is rounded like the others, which shows in rows that see few keys (error
// up to 1.6 times that of an F32 softmax rounded to bf16, against 1.1), so every row of the
// launch has to see kFixedKeys keys.
template <bool kF16, bool kCap, bool kBias, bool kFixed>
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
  // Warp 0 sets up the barriers and sends the first loads off while warp 1 waits for TMEM; the
  // other warps meet them at the CTA-wide barrier.
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
    mbar_init(c.s_free(), kSoftmaxThreads / 32);  // one arrival per warp
    mbar_init(c.p_full(), kSoftmaxThreads / 32);
    mbar_init(c.pv_done(), 1);
    mbar_init(c.o_final(), 1);
    for (int i = 1; i < 7; ++i) *c.misc(i) = 0;
    fence_mbar_init();
    if (g.n > 0) first_loads(c, g, a, &map_q, &map_k, &map_v);
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

  if (warp < kFirstSoftmaxWarp) {
    if (warp == 0) {
      if (lane == 0) run_producer(c, g, &map_k, &map_v, err);
      __syncwarp();
    } else {
      run_mma<kF16, kCap>(c, g, tmem, err);
    }
    if (a.splits > 1) {
      cluster_sync();  // partial rows written
      cluster_sync();  // and read
    }
  } else {
    const int quad = warp & 3;
    const int lane_base = quad * 32 + ((warp - kFirstSoftmaxWarp) >> 2) * 16;
    const uint32_t lane_off = static_cast<uint32_t>(lane_base) << 16;
    const uint32_t tS = tmem + lane_off + kColS, tP = tmem + lane_off + kColP, tO = tmem + lane_off + kColO;
    const int c0 = 2 * (lane & 3);  // first of the thread's column pair in every 8 columns
    const bool warp_live = lane_base < g.rows;
    // The thread's two rows of the tile.
    int limit[2], row[2];
    int frame[2];
    float slope[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      row[i] = lane_base + (lane >> 2) + 8 * i;
      // Rows past the tile's last take its place: nobody reads them, and no warp masks for them.
      const int at = min(row[i], g.rows - 1);
      const int tok = at / a.group;
      const int head = g.kvh * a.group + (at - tok * a.group);
      const int pos = g.it.first + tok;  // key position of the row
      // floor(pos / frame), also below zero
      frame[i] = pos >= 0 ? pos / a.t.frame : -1 - (-1 - pos) / a.t.frame;
      limit[i] = g.it.doc_keys;
      if (a.t.causal) {
        const int64_t e = (static_cast<int64_t>(frame[i]) + 1) * a.t.frame;
        limit[i] = static_cast<int>(max(static_cast<int64_t>(0),
                                        min(static_cast<int64_t>(limit[i]), max(e, static_cast<int64_t>(g.it.prefix)))));
      }
      slope[i] = kBias ? a.slopes[head] : 0.0f;
    }
    const float sl2 = a.t.scale_log2;
    // Running maxima, log2 domain, may lag by kGrow (kFixed: the constant reference).
    float m[2] = {kFixed ? 0.0f : -INFINITY, kFixed ? 0.0f : -INFINITY};
    float l[2] = {0.0f, 0.0f};            // partial sums over the thread's columns
    bool ok = true;
    for (int j = 0; j < g.n; ++j) {
      ok = mbar_wait(c.s_full(), j & 1, abort_flag, err, kDevTimeoutConsumer);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (!warp_live) {
        // Rows nobody reads: hand the tile on, P only once PV(j-1) is done, as the live warps
        // do, so that this arrival counts for tile j.
        warp_arrive(c.s_free());
        if (j > 0) {
          ok = mbar_wait(c.pv_done(), (j - 1) & 1, abort_flag, err, kDevTimeoutConsumer);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        warp_arrive(c.p_full());
        continue;
      }
      tc_fence_after();
      float s[64];  // block k: s[4k], s[4k+1] row 0, columns 8k + c0, +1; s[4k+2], s[4k+3] row 1
      tmem_ld_16x256b_x16(tS, s);
      tc_fence_before();
      warp_arrive(c.s_free());  // QK of the next tile may overwrite S
      const int k0 = (g.t0 + j) * kTile;
      const bool partial = __any_sync(0xffffffffu, min(limit[0], limit[1]) < k0 + kTile);
      const int lim[2] = {limit[0] - k0 - c0, limit[1] - k0 - c0};
      uint32_t pk[32];  // 16x128b order: block k: (row 0 pair k), (row 1 pair k)
      uint64_t acc[2] = {0, 0};
      // The exponentials of a pair.  They enter the second product in the operands' type (a tensor-core product has
      // operands of one type), the sum in F32: against 64 bits the result is 1 to 9 % further off than an F32
      // softmax rounded once (the 9 where a bias leaves few keys).
      auto emit = [&](int k, int i, uint64_t x) {
        float x0, x1;
        f32x2_unpack(x, x0, x1);
        const float p0 = ex2(x0), p1 = ex2(x1);
        const uint64_t pp = f32x2_pack(p0, p1);
        acc[i] = k == 0 ? pp : f32x2_add(acc[i], pp);
        pk[2 * k + i] = kF16 ? f16x2_from_f32(p0, p1) : pack_bf16x2(p0, p1);
      };
      bool grow[2] = {false, false};
      float alpha[2] = {1.0f, 1.0f};
      // kFixed, nothing hidden: polynomial and exponential pair by pair, so that the FMA pipe and
      // MUFU work at once.
      bool fused = false;
      if constexpr (kFixed) {
        auto both = [&](auto poly) {
#pragma unroll
          for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) emit(k, i, poly(f32x2_pack(s[4 * k + 2 * i], s[4 * k + 2 * i + 1])));
          fused = true;
        };
        if (!partial) {
          const float top = largest(s);
          if (__all_sync(0xffffffffu, top <= a.t.cap_range[0]))
            both(CapPoly<false>(a.t, a.fixed));
          else if (__all_sync(0xffffffffu, top <= a.t.cap_range[1]))
            both(CapPoly<true>(a.t, a.fixed));
        }
      }
      if (!fused) {
        if constexpr (kCap) {
          if (partial) hide(s, lim, 0.0f);  // hidden keys may hold anything: out of the range check
          cap_scores(s, a.t, kFixed ? a.fixed : 0.0f);  // kFixed: the exponent itself
        }
        if constexpr (kBias) {
          const bool past = k0 + kTile - 1 <= g.it.first || (a.t.causal && g.it.prefix == 0);
          const bool ahead = k0 >= g.it.first + g.it.tokens - 1;
          bias_scores<kCap>(s, a.t, k0, c0, frame, slope, past ? -1 : ahead ? 1 : 0);
        }
        constexpr bool kScaled = kCap || kBias;  // s already in the log2 domain
        if (partial) hide(s, lim, -INFINITY);
        uint64_t neg2[2] = {0, 0};
        float mx[2];
        if (!kFixed) row_maxima(s, mx);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (kFixed) break;
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
          if (!kScaled) mx[i] *= sl2;
          grow[i] = mx[i] > m[i] + kGrow;  // m = -inf: as soon as a key is seen
          if (grow[i]) {
            alpha[i] = ex2(m[i] - mx[i]);
            m[i] = mx[i];
          }
          const float neg = m[i] == -INFINITY ? 0.0f : kOffset - m[i];  // no key yet: every x is -inf
          neg2[i] = f32x2_pack(neg, neg);
        }
        const uint64_t sc2 = f32x2_pack(sl2, sl2);
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint64_t v = f32x2_pack(s[4 * k + 2 * i], s[4 * k + 2 * i + 1]);
            emit(k, i, kFixed ? v : kScaled ? f32x2_add(v, neg2[i]) : f32x2_fma(v, sc2, neg2[i]));
          }
      }
      if (j > 0) {
        // PV(j-1) has finished reading P and adding into O.
        ok = mbar_wait(c.pv_done(), (j - 1) & 1, abort_flag, err, kDevTimeoutConsumer);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
      }
      tmem_st_16x128b_x16(tP, pk);
      if (!kFixed && j > 0 && __any_sync(0xffffffffu, grow[0] || grow[1])) {
        float o[32];  // block k: o[4k], o[4k+1] row 0; o[4k+2], o[4k+3] row 1
        tmem_ld_16x256b_x8(tO, o);
        uint32_t w[32];
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) w[4 * k + e] = __float_as_uint(o[4 * k + e] * alpha[e >> 1]);
        tmem_st_16x256b_x8(tO, w);
      }
      tmem_wait_st();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float u0, u1;
        f32x2_unpack(acc[i], u0, u1);
        l[i] = kFixed ? l[i] + (u0 + u1) : l[i] * alpha[i] + (u0 + u1);
      }
      tc_fence_before();
      warp_arrive(c.p_full());
    }
    if (ok && g.n > 0) {
      ok = mbar_wait(c.o_final(), 0, abort_flag, err, kDevTimeoutConsumer);
      ok = __all_sync(0xffffffffu, ok);
    }
    float o[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] = 0.0f;
    if (ok && warp_live && g.n > 0) {
      tc_fence_after();
      tmem_ld_16x256b_x8(tO, o);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    uint8_t* out = static_cast<uint8_t*>(a.out.data);
    if (a.splits == 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!ok || row[i] >= g.rows) continue;
        const int tok = row[i] / a.group, head = g.kvh * a.group + (row[i] - tok * a.group);
        uint8_t* dst = out + 2 * ((g.it.q_row + static_cast<int64_t>(tok)) * a.out.token_stride + head * a.out.head_stride + c0);
        const float inv = 1.0f / l[i];
        const bool none = l[i] == 0.0f;  // no key seen
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float x0 = none ? 0.0f : o[4 * k + 2 * i] * inv, x1 = none ? 0.0f : o[4 * k + 2 * i + 1] * inv;
          *reinterpret_cast<uint32_t*>(dst + 16 * k) = kF16 ? f16x2_from_f32(x0, x1) : pack_bf16x2(x0, x1);
        }
      }
    } else {
      if (warp_live) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = row[i];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            // channels 8k + c0, +1: half of 16-byte chunk 2k + c0 / 4
            const uint32_t at = Smem::kPart + r * 256 + (((2 * k + (c0 >> 2)) ^ (r & 15)) << 4) + 4 * (c0 & 2);
            *reinterpret_cast<float2*>(c.smem + at) = make_float2(o[4 * k + 2 * i], o[4 * k + 2 * i + 1]);
          }
          if ((lane & 3) == 0) {
            c.ml()[2 * r] = m[i];
            c.ml()[2 * r + 1] = l[i];
          }
        }
      }
      __syncwarp();
      cluster_sync();
      // Rank q joins rows [q rows / splits, (q + 1) rows / splits): 16 threads a row.
      const int r0 = g.rank * g.rows / a.splits, r1 = (g.rank + 1) * g.rows / a.splits;
      const uint32_t part = c.base + Smem::kPart, ml = c.base + Smem::kMl;
      for (int i = static_cast<int>(threadIdx.x) - 32 * kFirstSoftmaxWarp; i < (r1 - r0) * 16; i += kSoftmaxThreads) {
        const int r = r0 + (i >> 4), ch = i & 15;
        // Every CTA's (maximum, sum) of the row and its chunk, four CTAs at a time: the eight remote
        // loads are issued before the first is used, and the batch is folded in like a key tile.
        float mt = -INFINITY, lt = 0.0f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p0 = 0; p0 < a.splits; p0 += 4) {
          float2 q[4];
          float4 v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (p0 + e < a.splits) {
              q[e] = ld_cluster_v2(cluster_addr(ml + r * 8, p0 + e));
              v[e] = ld_cluster_v4(cluster_addr(part + r * 256 + ((ch ^ (r & 15)) << 4), p0 + e));
            } else {
              q[e] = make_float2(-INFINITY, 0.0f);
            }
          const float m_new = fmaxf(fmaxf(mt, fmaxf(q[0].x, q[1].x)), fmaxf(q[2].x, q[3].x));
          const float old = mt == -INFINITY ? 0.0f : ex2(mt - m_new);
          sum.x *= old, sum.y *= old, sum.z *= old, sum.w *= old;
          lt *= old;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (q[e].y != 0.0f) {  // keys seen (a row of NaN scores has a NaN sum and no maximum)
              const float f = ex2(q[e].x - m_new);
              sum.x += f * v[e].x, sum.y += f * v[e].y, sum.z += f * v[e].z, sum.w += f * v[e].w;
              lt += f * q[e].y;
            }
          mt = m_new;
        }
        const float inv = 1.0f / lt;
        if (lt == 0.0f) sum = make_float4(0.f, 0.f, 0.f, 0.f);
        else sum.x *= inv, sum.y *= inv, sum.z *= inv, sum.w *= inv;
        const int t = r / a.group, h = g.kvh * a.group + (r - t * a.group);
        const uint2 w = kF16 ? make_uint2(f16x2_from_f32(sum.x, sum.y), f16x2_from_f32(sum.z, sum.w))
                             : make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
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

template <bool kF16, bool kCap, bool kBias, bool kFixed = false>
cudaError_t launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const MaskedArgs& a,
                   int64_t blocks, int* err, cudaStream_t st) {
  auto kern = masked_attn_kernel<kF16, kCap, kBias, kFixed>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = prepare_kernel(reinterpret_cast<const void*>(kern), Smem::kLaunchBytes, ready);
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

// Time model of a launch, in key tiles of a CTA that has its SM alone (1.13 us plain, 1.5 us with a
// cap or a bias): two CTAs on one SM run at kShared of that each (measured 1.56 and 2.0 us),
// a CTA pays kFixed (barriers, TMEM, first loads, output) and a split one kJoin more.  CTAs go to
// the first free slot in grid order.
constexpr double kShared = 0.725, kFixed = 2.7, kJoin = 2.0;
double masked_time(const int* key_tiles, int64_t items, int kv_heads, int sms, int splits) {
  struct Sm {
    double now = 0.0, left[2] = {0.0, 0.0};  // work left in its two slots
    double next() const {                    // when one of them is free
      const bool two = left[0] > 0.0 && left[1] > 0.0;
      const double w = two ? std::min(left[0], left[1]) / kShared : std::max(left[0], left[1]);
      return now + w;
    }
    void advance(double t) {
      const double done = (t - now) * (left[0] > 0.0 && left[1] > 0.0 ? kShared : 1.0);
      for (double& x : left) x = x - done > 1e-9 ? x - done : 0.0;
      now = t;
    }
  };
  std::vector<Sm> sm(sms);
  using Entry = std::pair<double, int>;
  std::priority_queue<Entry, std::vector<Entry>, std::greater<Entry>> busy;
  int64_t placed = 0;
  double end = 0.0;
  for (int64_t i = 0; i < items; ++i) {
    const double cost = static_cast<double>((key_tiles[i] + splits - 1) / splits) + kFixed + (splits > 1 ? kJoin : 0.0);
    for (int h = 0; h < kv_heads * splits; ++h, ++placed) {
      if (placed < 2 * sms) {  // the first CTAs: one on every SM, then a second
        sm[placed % sms].left[placed / sms] = cost;
        if (placed == 2 * sms - 1)
          for (int m = 0; m < sms; ++m) busy.push({sm[m].next(), m});
        continue;
      }
      const Entry e = busy.top();
      busy.pop();
      Sm& x = sm[e.second];
      x.advance(e.first);
      x.left[x.left[0] > 0.0 ? 1 : 0] = cost;
      busy.push({x.next(), e.second});
    }
  }
  for (Sm& x : sm)
    while (x.left[0] > 0.0 || x.left[1] > 0.0) {
      x.advance(x.next());
      end = std::max(end, x.now);
    }
  return end;
}

}  // namespace

int masked_splits(const int* key_tiles, int64_t items, int kv_heads, int sms) {
  // Two rounds of CTAs and more: a cut gains nothing that the order does not give (816 and 984 tiles
  // in 1 / 2 / 3 CTAs each: 129 / 152 / 180 and 508 / 530 / 561 us).  That holds where the longest tile is short beside
  // the whole; one count for all tiles does not suit a plan that mixes a prompt with single tokens over much
  // longer documents (a causal prompt of 6,400 tokens x 12 heads 103 us, with one token over 32,000 keys 273, that token
  // in a plan of its own 20): the header advises a plan for each kind.
  if (items == 0 || items * kv_heads >= 4 * static_cast<int64_t>(sms)) return 1;
  int best = 1;
  double best_time = masked_time(key_tiles, items, kv_heads, sms, 1);
  int64_t tiles = 0;
  for (int64_t i = 0; i < items; ++i) tiles += key_tiles[i];
  for (int s = 2; s <= kMaxSplits && s <= key_tiles[0]; ++s) {  // key_tiles[0]: the most
    // No launch of so much work ends sooner, and a finer cut only adds to it.
    const double bound = kv_heads * (tiles + items * s * (kFixed + kJoin)) / (2.0 * kShared * sms);
    if (bound >= 0.97 * best_time) break;
    const double t = masked_time(key_tiles, items, kv_heads, sms, s);
    if (t < 0.97 * best_time) {
      best = s;
      best_time = t;
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
  if (!f16 && cap && !bias && a.t.cap_out <= kFixedCap && a.fewest_keys >= kFixedKeys) {
    MaskedArgs fixed = a;
    int log2_keys = 10;
    while ((int64_t(1) << log2_keys) < a.most_keys) ++log2_keys;
    fixed.fixed = static_cast<float>(127 - kFixedValues - log2_keys) - a.t.cap_out;
    return launch<false, true, false, true>(mq, mk, mv, fixed, blocks, err, st);
  }
  return fn[f16][cap][bias](mq, mk, mv, a, blocks, err, st);
}

}  // namespace va
