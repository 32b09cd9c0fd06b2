// Attention of a few new tokens per document over the quantised key/value cache.
//
//   out_i = sum_j p_ij vs_j V_j / sum_j p_ij,   p_ij = exp(score_ij - max_j score_ij),
//   score_ij = cap tanh(scale ks_j (q_i . K_j) / cap) - slope |f(P_i) - f(j)|
// with K_j, V_j the integer or e4m3 codes and ks_j, vs_j their scales: a key's scale
// multiplies its scores, a value's scale its probability, so codes are never scaled.
//
// Bound by HBM where all SMs have work: every visible key costs 2 * (64 + 4) bytes per key head
// and 256 FLOP per query row.  The fragments, and the joining of warps and cluster, are va_rows.cuh's.  The operands
// are f16 because both code formats become f16 in one or two instructions a pair (bf16 took four or five, and the
// conversions are most of the loop).  Its range is met by powers of two.  A query row is scaled to a largest magnitude
// in [1, 2) and the factor goes to the scores: 16-bit elements stay exact down to 2^-14 of the largest, and to 2^-25
// of it below.  A weight (a probability times its value scale) is scaled by 2^(kTop - E) and split in two f16 parts,
// the second in the product's rows 8..15 at no further cost.
//   While every row sees the whole chunk and the warp's value scales so far lie within 2^kAlike, E is just above
//   the largest of them, for all rows: the key of a row's maximum has probability 1, so the row's largest
//   weight is at least 2^(E - 1 - kAlike).
//   From the first chunk on where this does not hold, each row has its own E, above its own largest weight: a
//   key that the row does not see, or that hardly counts in it, must not take the range from the others, whatever
//   the values' sizes (probabilities below 2^-126 are 0).
// Either way a scaled weight has steps of 2^-24 and the row's largest is 2^(kTop - 1 - kAlike) or more.
// The weights' maximum then stands between the scores and the product: scales that span 2^6 and more make the mixed
// batch below 38.5 us instead of 35, 16 x 32,000 x 16 key heads 224 instead of 202, one token 11.4 instead of 10.2.
//
// A cluster of CTAs shares one (document, key head, row block), or two documents' that divide its
// CTAs; a warp takes 64-key chunks in turn through a ring of its own in shared memory (cp.async, one chunk ahead), each
// warp with its own running maximum and sum, and the partial results meet in shared memory
// and then, through distributed shared memory, across the cluster in rank order: one
// launch, no workspace, no atomics, and the same bits on every run.
//
// Measured on B200: one token over 10,392 int8 tokens x 12 heads 9.5 us; 16 documents of 0 to 32,000 e4m3
// tokens, 22 rows, 4 key heads, cap and bias, 35 us; 16 documents of 32,000, cap and bias off, caches in turn, 51 us
// (5.4 TB/s), and x 16 key heads 179 us (6.2 TB/s = 0.95 of measured).  A warp's chunk takes about 2.5 us with 12 warps
// on the SM and 1.1 us with 4: some 900 instructions of conversions, score terms and softmax (58% of issue slots), not the loads.
// Masks are applied to chunks that some row does not see whole only, and scales lie in the order of the
// fragments.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "va_internal.h"
#include "va_ptx.cuh"
#include "va_rows.cuh"

namespace va {

namespace {

using namespace rows;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kChunk = 64;         // keys a warp takes at a time
constexpr int kTiles = kChunk / 8;
constexpr int kStages = 2;         // chunks of a warp in shared memory
constexpr int kCtasPerSm = 3;
constexpr int64_t kMostBlocks = 1 << 20;
constexpr int kMaxPaired = 256;    // documents that a CTA puts in order
constexpr int kTop = 14;       // weights are brought below 2^kTop
constexpr int kAlike = 6;
constexpr int kMinExp = -100;  // weights below 2^-100 lose precision

struct CacheAttnArgs {
  KvCacheRef c;
  AttnTerms t;
  int group;                // query heads per key head
  int row_blocks;           // row blocks a launch provides per document
  uint32_t frame_magic;     // floor(2^32 / frame)
  int64_t rows;
  const int32_t* offsets;
  const int32_t* lens;
  const int32_t* prefix;
  const float* slopes;
  HeadsRef q, out;
};

// Two code bytes of w -> f16x2, exactly.  kHigh: bytes 2 and 3, else 0 and 1.  int8 codes come
// with their sign bits flipped (flip): u = c + 128 under 0x64 is the f16 1024 + u.
template <bool kE4m3>
__device__ __forceinline__ uint32_t flip(uint32_t w) { return kE4m3 ? w : w ^ 0x80808080u; }
template <bool kE4m3, bool kHigh>
__device__ __forceinline__ uint32_t codes_to_f16x2(uint32_t w) {
  uint32_t r;
  if constexpr (kE4m3) {
    const uint16_t h = static_cast<uint16_t>(kHigh ? w >> 16 : w);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
  } else {
    const uint32_t t = prmt(w, 0x64646464u, kHigh ? 0x4342u : 0x4140u);  // bytes: u0, 64, u1, 64
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(t), "r"(0x64806480u));  // - (1024 + 128)
  }
  return r;
}

// 2^e: 0 below the normal range, infinity above.
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float(static_cast<uint32_t>(min(max(e + 127, 0), 255)) << 23); }
// The least e >= kMinExp with w < 2^e (128 for what is not finite).
__device__ __forceinline__ int exponent_above(uint32_t bits) {
  return min(max(static_cast<int>(bits >> 23) - 126, kMinExp), 128);
}

// A warp's ring of chunks in shared memory, filled by cp.async (16 bytes of codes, 4 of
// scales a copy: no alignment beyond the cache's own).  Code rows of 64 bytes; the
// 16-byte piece p of row r lies at piece p ^ (2 bit2(r)).
struct Chunk {
  uint8_t k[kChunk][kHeadDim];
  uint8_t v[kChunk][kHeadDim];
  float ks[kChunk], vs[kChunk];
};
// Place of a key's scales within 32: the two keys of a lane in the score fragments (tile_key's order) are
// neighbours.  Its own inverse.
__device__ __forceinline__ int scale_at(int key) { return key ^ ((key >> 1) & 1); }
// Rows past `last` repeat it (they are hidden, and the codes of any row held are finite).
__device__ __forceinline__ void load_chunk(Chunk& ch, const uint8_t* kc, const uint8_t* vc, const float* ks,
                                           const float* vs, int key0, int last, int lane) {
  const int row = lane >> 2, p = lane & 3;
  uint8_t* to = &ch.k[row][16 * (p ^ ((row >> 1) & 2))];  // bit 2 of 8 i + row is that of row
  if (key0 + kChunk - 1 <= last) {
    const int64_t at = (static_cast<int64_t>(key0) + row) * kHeadDim + 16 * p;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      cp16(to + 8 * i * kHeadDim, kc + at + 8 * i * kHeadDim);
      cp16(to + (kChunk + 8 * i) * kHeadDim, vc + at + 8 * i * kHeadDim);
    }
#pragma unroll
    for (int i = 0; i < kChunk; i += 32) {
      cp4(&ch.ks[i + scale_at(lane)], ks + key0 + i + lane);
      cp4(&ch.vs[i + scale_at(lane)], vs + key0 + i + lane);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int64_t at = static_cast<int64_t>(min(key0 + 8 * i + row, last)) * kHeadDim + 16 * p;
      cp16(to + 8 * i * kHeadDim, kc + at);
      cp16(to + (kChunk + 8 * i) * kHeadDim, vc + at);
    }
#pragma unroll
    for (int i = 0; i < kChunk; i += 32) {
      const int64_t key = min(key0 + i + lane, last);
      cp4(&ch.ks[i + scale_at(lane)], ks + key);
      cp4(&ch.vs[i + scale_at(lane)], vs + key);
    }
  }
}

// Two documents that share a cluster.  key: 0 without rows in this block of rows, else 1 + the length.
struct Pair {
  int doc[2], key[2], begin[2], tokens[2];
};
struct Documents {
  int key[kMaxPaired];
  Pair pair;
};
__device__ __forceinline__ bool good_document(const CacheAttnArgs& a, int32_t begin, int32_t end, int32_t len) {
  return begin >= 0 && end >= begin && end <= a.rows && len >= 0 && len <= a.c.capacity;
}
// The documents in order of falling keys: number `index` and, from the other end, its mirror image (itself in the
// middle of an odd count, and then key[1] is 0).  Every CTA counts for itself: at most 256 keys.
__device__ __forceinline__ Pair find_pair(Documents& sh, const CacheAttnArgs& a, int index, int block0, bool report,
                                          int* err) {
  int32_t begin[kMaxPaired / kThreads], tokens[kMaxPaired / kThreads];
  int key[kMaxPaired / kThreads];
#pragma unroll
  for (int i = 0; i < kMaxPaired / kThreads; ++i) {
    const int doc = i * kThreads + static_cast<int>(threadIdx.x);
    key[i] = -1;  // behind every document
    if (doc < a.c.documents) {
      begin[i] = __ldg(a.offsets + doc);
      const int32_t end = __ldg(a.offsets + doc + 1), len = __ldg(a.lens + doc);
      const bool ok = good_document(a, begin[i], end, len);
      if (!ok && report) report_error(err, kDevBadLengths);
      tokens[i] = ok ? end - begin[i] : 0;
      key[i] = block0 * kRowsPerBlock < tokens[i] * a.group ? len + 1 : 0;
    }
    sh.key[doc] = key[i];
  }
  if (threadIdx.x == 0) sh.pair.key[1] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMaxPaired / kThreads; ++i) {
    const int doc = i * kThreads + static_cast<int>(threadIdx.x);
    if (doc >= a.c.documents) break;
    int ahead = 0;
    for (int e = 0; e < a.c.documents; e += 4) {
      const int4 k = *reinterpret_cast<const int4*>(&sh.key[e]);
      ahead += (k.x > key[i] || (k.x == key[i] && e < doc)) + (k.y > key[i] || (k.y == key[i] && e + 1 < doc)) +
               (k.z > key[i] || (k.z == key[i] && e + 2 < doc)) + (k.w > key[i] || (k.w == key[i] && e + 3 < doc));
    }
    const int place = ahead == index ? 0 : ahead == a.c.documents - 1 - index ? 1 : -1;
    if (place >= 0) {
      sh.pair.doc[place] = doc;
      sh.pair.key[place] = key[i];
      sh.pair.begin[place] = begin[i];
      sh.pair.tokens[place] = tokens[i];
    }
  }
  __syncthreads();
  return sh.pair;
}
// CTAs of a cluster that the first of two documents gets: by their chunks, so that the slower one is soonest done.
__device__ __forceinline__ int share(int key0, int key1, int cluster) {
  if (key1 == 0) return cluster;
  const float w0 = static_cast<float>((key0 - 1) / kChunk + 1), w1 = static_cast<float>((key1 - 1) / kChunk + 1);
  const int n = min(max(static_cast<int>(cluster * w0 / (w0 + w1)), 1), cluster - 1);
  const int up = min(n + 1, cluster - 1);
  return fmaxf(w0 / up, w1 / (cluster - up)) < fmaxf(w0 / n, w1 / (cluster - n)) ? up : n;
}

struct Shared {
  union {
    Chunk ring[kWarps][kStages];
    Join<kWarps> join;  // once the block's last chunk is used
  };
  union {
    Documents docs;          // read out before this CTA arrives at its first cluster barrier
    Part part[kMaxCluster];  // [own row][number in the document's share], written after that barrier
  };
};
static_assert(kCtasPerSm * (sizeof(Shared) + 1024) <= 228 * 1024, "shared memory of an SM");

template <class T, bool kE4m3, bool kPaired>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    cache_attn_kernel(const __grid_constant__ CacheAttnArgs a, int cluster, int* err) {
  extern __shared__ uint4 smem_raw[];
  Shared& smem = *reinterpret_cast<Shared*>(smem_raw);
  Join<kWarps>& sh = smem.join;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  int rank = static_cast<int>(blockIdx.x) % cluster;
  int unit = static_cast<int>(blockIdx.x) / cluster;
  const int kvh = unit % a.c.kv_heads;
  unit /= a.c.kv_heads;
  const int block0 = unit % a.row_blocks;
  int doc = unit / a.row_blocks;

  // This CTA is number `rank` of the `splits` that share the document's keys; number 0 has rank `lead` in the
  // cluster.  All CTAs of the cluster walk `most_rows`, so that they meet the same barriers.
  int splits = cluster, lead = 0;
  int32_t begin, len;
  int tokens, most_rows;
  if constexpr (kPaired) {
    const Pair pair = find_pair(smem.docs, a, doc, block0, blockIdx.x == 0, err);
    if (pair.key[0] == 0) return;  // neither document has rows here (key[0] >= key[1])
    const int n = share(pair.key[0], pair.key[1], cluster);
    const bool second = rank >= n;
    splits = second ? cluster - n : n;
    lead = second ? n : 0;
    rank -= lead;
    doc = second ? pair.doc[1] : pair.doc[0];
    begin = second ? pair.begin[1] : pair.begin[0];
    tokens = second ? pair.tokens[1] : pair.tokens[0];
    len = (second ? pair.key[1] : pair.key[0]) - 1;
    most_rows = (pair.key[1] == 0 ? pair.tokens[0] : max(pair.tokens[0], pair.tokens[1])) * a.group;
  } else {
    begin = __ldg(a.offsets + doc);
    len = __ldg(a.lens + doc);
    const int32_t end = __ldg(a.offsets + doc + 1);
    if (!good_document(a, begin, end, len)) {  // the same for every CTA of the cluster: none of them waits
      if (threadIdx.x == 0) report_error(err, kDevBadLengths);
      return;
    }
    tokens = end - begin;
    most_rows = tokens * a.group;
  }
  const int q_rows = tokens * a.group;
  const int prefix = a.prefix ? max(__ldg(a.prefix + doc), 0) : 0;
  const int64_t head_base = (static_cast<int64_t>(doc) * a.c.kv_heads + kvh) * a.c.capacity;
  const uint8_t* kc = a.c.codes[0] + head_base * kHeadDim;
  const uint8_t* vc = a.c.codes[1] + head_base * kHeadDim;
  const float* ks = a.c.scales[0] + head_base;
  const float* vs = a.c.scales[1] + head_base;
  const T* qd = static_cast<const T*>(a.q.data);

  // Keys a token sees: the first `limit` of the document.
  auto limit_of = [&](int token) {
    if (!a.t.causal) return len;
    const int p = token + len - tokens;
    int64_t e = prefix;
    if (p >= 0) {
      const int64_t f = static_cast<int64_t>(frame_index(p, a.t.frame, a.frame_magic) + 1) * a.t.frame;
      e = max(e, f);
    }
    return static_cast<int>(min(e, static_cast<int64_t>(len)));
  };

  for (int rb = block0; rb * kRowsPerBlock < most_rows; rb += a.row_blocks) {
    // Every CTA of the cluster has started, and is done with the parts of the last block.
    if (cluster > 1) cluster_arrive();
    if (kPaired && rb * kRowsPerBlock >= q_rows) {  // only the pair's other document has rows left: finish_block's barriers
      cluster_wait();
      cluster_arrive();
      cluster_wait();
      continue;
    }
    const int r = rb * kRowsPerBlock + g;  // this lane's query row
    const bool valid = r < q_rows;
    const int token = valid ? r / a.group : tokens - 1;
    const int head = kvh * a.group + (valid ? r % a.group : 0);
    const int block_limit = limit_of(min(rb * kRowsPerBlock + kRowsPerBlock - 1, q_rows - 1) / a.group);
    const int limit = valid ? limit_of(token) : block_limit;
    const int fp = frame_index(token + len - tokens, a.t.frame, a.frame_magic);
    const float slope = a.slopes ? __ldg(a.slopes + head) * kLog2e : 0.0f;

    // The row's load, then the first chunks', go off together; the row is used while the chunks
    // arrive.
    RawRow raw;
    load_row(raw, qd + (begin + static_cast<int64_t>(token)) * a.q.token_stride + head * a.q.head_stride + 16 * c);
    const int chunks = (block_limit + kChunk - 1) / kChunk;
    const int stride = splits * kWarps;
    const int first = rank * kWarps + warp;
    Chunk* ring = smem.ring[warp];
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (first + i * stride < chunks) load_chunk(ring[i], kc, vc, ks, vs, (first + i * stride) * kChunk, len - 1, lane);
      cp_commit();
    }
    // Query row in fragment order: word s of the lane's 16 channels [16c, 16c + 16).
    uint32_t qa[4][4];
    float q_scale;
    {
      float x[16];
      unpack_row<T>(raw, x);
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (!valid) x[e] = 0.0f;
        top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t ex = min(max(top >> 23, 2u), 252u);  // a non-finite row stays non-finite
      q_scale = __uint_as_float(ex << 23);
      const float inv = __uint_as_float((254u - ex) << 23);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        qa[s][0] = f16x2_from_f32(x[4 * s] * inv, x[4 * s + 1] * inv);
        qa[s][2] = f16x2_from_f32(x[4 * s + 2] * inv, x[4 * s + 3] * inv);
        qa[s][1] = qa[s][3] = 0u;
      }
    }
    const float score_scale = q_scale * a.t.scale_log2, cap_scale = q_scale * a.t.cap_in;
    int w_exp = kMinExp;  // E: the row's weights so far are below 2^E

    float o[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    int stage = 0, ch = first;
    Chunk* cur = ring;
    auto fetch = [&] {
      cp_wait<kStages - 2>();
      __syncwarp();  // every lane's copies have landed, and the stage below is read out
      const int next = ch + (kStages - 1) * stride;
      const int to = stage == 0 ? kStages - 1 : stage - 1;
      if (next < chunks) load_chunk(ring[to], kc, vc, ks, vs, next * kChunk, len - 1, lane);
      cp_commit();
      cur = ring + stage;
      stage = stage + 1 == kStages ? 0 : stage + 1;
    };
    // Scores of 8 rows x 64 keys: lane (g, c) gets row g, columns 2c and 2c + 1 of each tile.
    auto score = [&](float(&x)[kTiles][2]) {
      float d[kTiles][4];
      uint32_t w[kTiles][4];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int kr = 8 * t + tile_key(g);
        const uint4 kw = *reinterpret_cast<const uint4*>(&cur->k[kr][16 * (c ^ ((kr >> 1) & 2))]);
        w[t][0] = flip<kE4m3>(kw.x), w[t][1] = flip<kE4m3>(kw.y), w[t][2] = flip<kE4m3>(kw.z), w[t][3] = flip<kE4m3>(kw.w);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[t][e] = 0.0f;
      }
      // Eight independent chains: a tile's four steps follow each other, the tiles do not.
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
          mma(__half(), d[t], qa[s], codes_to_f16x2<kE4m3, false>(w[t][s]), codes_to_f16x2<kE4m3, true>(w[t][s]));
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const float2 k_scale = *reinterpret_cast<const float2*>(&cur->ks[8 * t + 2 * c]);
#pragma unroll
        for (int e = 0; e < 2; ++e) x[t][e] = d[t][e] * (e ? k_scale.y : k_scale.x);
      }
    };
    // The row's maximum with this chunk.
    auto maximum = [&](const float(&x)[kTiles][2]) {
      float top = x[0][0];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) top = max3f(top, x[t][0], x[t][1]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      return fmaxf(m, top);
    };
    // A new maximum (alpha = 2^(m - m_new)) and a new E for the sums so far.
    auto rescale = [&](float m_new, float alpha, int e_new) {
      l *= alpha;
      // E falls only as alpha does, so the product stays in range.
      const float f = alpha * exp2i(max(min(w_exp - e_new, 127), -126));
      w_exp = e_new;
      // Accumulator rows g (elements 0, 1) and g + 8 (2, 3) are parts of query row g.
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= f;
      m = m_new;
    };
    // o += weights * values; weight(t, e) of the lane's keys, in order.
    auto add_values = [&](auto weight) {
#pragma unroll
      for (int u = 0; u < kTiles / 2; ++u) {
        uint32_t pa[4];
        uint2 vw[4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int t = 2 * u + half;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int kk = 8 * t + ((2 * c + e) ^ (c & 1));
            vw[2 * half + e] = *reinterpret_cast<const uint2*>(&cur->v[kk][(8 * g) ^ ((kk << 3) & 32)]);
          }
          const float2 w = weight(t);
          split2(__half(), w.x, w.y, pa[2 * half], pa[2 * half + 1]);
        }
#pragma unroll
        for (int word = 0; word < 2; ++word) {
          // Four channels of two keys each, interleaved in pairs.
          const uint32_t a0 = flip<kE4m3>(word ? vw[0].y : vw[0].x), a1 = flip<kE4m3>(word ? vw[1].y : vw[1].x);
          const uint32_t b0 = flip<kE4m3>(word ? vw[2].y : vw[2].x), b1 = flip<kE4m3>(word ? vw[3].y : vw[3].x);
          const uint32_t lo0 = prmt(a0, a1, 0x5140), hi0 = prmt(a0, a1, 0x7362);
          const uint32_t lo1 = prmt(b0, b1, 0x5140), hi1 = prmt(b0, b1, 0x7362);
          mma(__half(), o[4 * word + 0], pa, codes_to_f16x2<kE4m3, false>(lo0), codes_to_f16x2<kE4m3, false>(lo1));
          mma(__half(), o[4 * word + 1], pa, codes_to_f16x2<kE4m3, true>(lo0), codes_to_f16x2<kE4m3, true>(lo1));
          mma(__half(), o[4 * word + 2], pa, codes_to_f16x2<kE4m3, false>(hi0), codes_to_f16x2<kE4m3, false>(hi1));
          mma(__half(), o[4 * word + 3], pa, codes_to_f16x2<kE4m3, true>(hi0), codes_to_f16x2<kE4m3, true>(hi1));
        }
      }
    };

    // Chunks that every row sees whole, while the value scales are alike: one E for all rows.
    const int whole = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<unsigned>(limit))) / kChunk;
    uint32_t v_most = 0, v_least = 0x7f800000u;  // bits of the largest and the smallest value scale so far
    bool fetched = false;
    for (; ch < whole; ch += stride) {
      fetch();
      float x[kTiles][2];
      score(x);
      apply_terms<false>(x, a.t, score_scale, cap_scale, a.slopes != nullptr, slope, fp, ch * kChunk, limit, c, a.frame_magic);
      const float m_new = maximum(x);
      // NaN and infinity set no range; they reach the rows on their own.
      uint32_t most = 0, least = 0x7f800000u;
#pragma unroll
      for (int i = 0; i < kChunk; i += 32) {
        const uint32_t bits = __float_as_uint(cur->vs[i + lane]);
        if (bits < 0x7f800000u) most = max(most, bits), least = min(least, bits);
      }
      v_most = max(v_most, __reduce_max_sync(0xffffffffu, most));
      v_least = min(v_least, __reduce_min_sync(0xffffffffu, least));
      if (v_most > v_least + (static_cast<uint32_t>(kAlike) << 23)) {
        fetched = true;
        break;
      }
      const int e_new = exponent_above(v_most);
      if (__any_sync(0xffffffffu, m_new > m) || e_new != w_exp) rescale(m_new, m_new > m ? ex2(m - m_new) : 1.0f, e_new);
      const float base = m == -INFINITY ? 0.0f : m;
      const float v_scale = exp2i(kTop - w_exp);
#pragma unroll
      for (int i = 0; i < kChunk; i += 32) cur->vs[i + lane] *= v_scale;
      __syncwarp();
      add_values([&](int t) {
        const float2 v_sc = *reinterpret_cast<const float2*>(&cur->vs[8 * t + 2 * c]);
        const float p0 = ex2(x[t][0] - base), p1 = ex2(x[t][1] - base);
        l += p0;
        l += p1;
        return make_float2(p0 * v_sc.x, p1 * v_sc.y);
      });
    }
    // The others (one break of the above, the chunks with a mask): E by row.  In the units of m, the largest weight
    // so far is 2^(E - 1) or somewhat less.
    float w_run = exp2i(w_exp - 1);  // the lane's
    for (; ch < chunks; ch += stride) {
      if (!fetched) fetch();
      fetched = false;
      const int key0 = ch * kChunk;
      float x[kTiles][2];
      score(x);
      apply_terms<true>(x, a.t, score_scale, cap_scale, a.slopes != nullptr, slope, fp, key0, limit, c, a.frame_magic);
      const float m_new = maximum(x);
      const float base = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = m_new > m ? ex2(m - m_new) : 1.0f;  // 0 for the first keys
      // x becomes the weights, before E is known.
      float sum = 0.0f, w_top = 0.0f;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const float2 v_sc = *reinterpret_cast<const float2*>(&cur->vs[8 * t + 2 * c]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = ex2(x[t][e] - base);
          sum += p;
          // a hidden key's value scale may be anything (stale rows)
          x[t][e] = key0 + 8 * t + ((2 * c + e) ^ (c & 1)) < limit ? p * (e ? v_sc.y : v_sc.x) : 0.0f;
        }
        w_top = max3f(w_top, fabsf(x[t][0]), fabsf(x[t][1]));  // NaN is no maximum
      }
      w_run = fmaxf(w_run * alpha, w_top);
      w_top = fmaxf(w_run, __shfl_xor_sync(0xffffffffu, w_run, 1));
      w_top = fmaxf(w_top, __shfl_xor_sync(0xffffffffu, w_top, 2));
      const int e_new = exponent_above(__float_as_uint(w_top));
      if (__any_sync(0xffffffffu, m_new > m || e_new != w_exp)) rescale(m_new, alpha, e_new);
      l += sum;
      const float w_scale = exp2i(kTop - w_exp);
      add_values([&](int t) { return make_float2(x[t][0] * w_scale, x[t][1] * w_scale); });
    }
    cp_wait<0>();
    __syncthreads();  // every warp is done with its ring: the join buffers may cover it
    const float back = exp2i(w_exp - kTop);
    finish_block<T>(sh, smem.part, o, m, l, back, rb, q_rows, a.group, kvh, rank, splits, cluster, lead, begin,
                   a.out);
    __syncthreads();  // before the next block's loads and parts
  }
}

cudaLaunchConfig_t config(int64_t blocks, int cluster, cudaStream_t st, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = st;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = cluster;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// Clusters of a size that the current device holds at once.  The variants of the kernel are alike in
// what limits them: registers and shared memory, for kCtasPerSm CTAs.
cudaError_t clusters_held(int cluster, int* held) {
  static std::atomic<int> known[64][kMaxCluster + 1];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (*held = known[dev][cluster].load(std::memory_order_relaxed)) > 0) return e;
  auto kern = cache_attn_kernel<__half, true, true>;
  static std::atomic<uint64_t> ready{0};
  e = prepare_kernel(reinterpret_cast<const void*>(kern), sizeof(Shared), ready);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = config(cluster, cluster, nullptr, attr);
  e = cudaOccupancyMaxActiveClusters(held, kern, &cfg);
  if (e == cudaSuccess && dev < 64) known[dev][cluster].store(*held, std::memory_order_relaxed);
  return e;
}

template <class T, bool kE4m3, bool kPaired>
cudaError_t launch(const CacheAttnArgs& a, int cluster, int64_t blocks, int* err, cudaStream_t st) {
  auto kern = cache_attn_kernel<T, kE4m3, kPaired>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = prepare_kernel(reinterpret_cast<const void*>(kern), sizeof(Shared), ready);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = config(blocks, cluster, st, attr);
  return cudaLaunchKernelEx(&cfg, kern, a, cluster, err);
}

}  // namespace

cudaError_t launch_cache_attention(const KvCacheRef& c, const AttnTerms& t, int dtype, int64_t rows,
                                   const int32_t* offsets, const int32_t* lens, int max_tokens,
                                   const int32_t* prefix, const float* slopes, const HeadsRef& q,
                                   const HeadsRef& out, int sms, int* err, cudaStream_t st) {
  CacheAttnArgs a{};
  a.c = c;
  a.t = t;
  a.group = t.heads / t.kv_heads;
  a.row_blocks = std::max(1, static_cast<int>((static_cast<int64_t>(max_tokens) * a.group + kRowsPerBlock - 1) /
                                              kRowsPerBlock));
  a.frame_magic = static_cast<uint32_t>((1ull << 32) / static_cast<uint32_t>(std::max(2, t.frame)));
  a.rows = rows;
  a.offsets = offsets;
  a.lens = lens;
  a.prefix = prefix;
  a.slopes = slopes;
  a.q = q;
  a.out = out;
  // CTAs per (document, key head): the lengths are on the device, so by the capacity (at least one
  // chunk per warp) and by what the SMs hold at once, at most 8, or 16, which the GPU places less
  // easily, where that fits.  Letting the CTAs past a document's share of the work leave at once
  // gained nothing: a cluster still waits for all its places.
  const int64_t slots = kCtasPerSm * static_cast<int64_t>(sms), pairs = static_cast<int64_t>(c.documents) * c.kv_heads;
  const int64_t most = std::max<int64_t>(1, c.capacity / (kChunk * kWarps));
  const int64_t fit = std::max<int64_t>(1, std::min(slots / pairs, most));
  int cluster = static_cast<int>(fit >= kMaxCluster ? kMaxCluster : std::min<int64_t>(fit, 8));
  bool paired = false;  // two documents share a cluster
  int64_t shared_by = c.documents;  // clusters per key head and block of rows
  // From 8 documents on, a long and a short one share a cluster and divide its CTAs by their lengths, where that
  // is two to six each on average, the clusters all fit with hardly fewer CTAs, and a capacity of 8192 pays for the
  // sorting.  Measured (us, own clusters / shared, e4m3, 4 query heads a key head, caches in turn; lengths random /
  // equal): 64 documents x 2 key heads of up to 32,000 68 / 51, 88 / 90; 20 x 4 43 / 35, 58 / 59; 16 x 12 of up to
  // 9,000 32 / 28, 42 / 42; 16 x 4 of up to 32,000, where clusters of 10 are the largest that fit, 38 / 32, 47 / 51:
  // the lengths are on the device, so equal ones pay up to 8 % for what unequal ones gain.  Outside the rule
  // (sharing forced): 4 x 16 of up to 32,000 46 / 51, 54 / 64; 8 x 4 27 / 29, 33 / 44; 16 x 12 of up to 2,000 11.4 / 11.7,
  // 14.7 / 15.9.
  if (fit >= 2 && fit <= 6 && c.documents >= 8 && c.documents <= kMaxPaired && c.capacity >= 8192) {
    const int64_t both = (c.documents + 1) / 2;
    for (int s = 2 * static_cast<int>(fit); 3 * s >= 5 * fit && !paired; s -= 2) {
      int held = 0;
      const cudaError_t e = clusters_held(s, &held);
      if (e != cudaSuccess) return e;
      if (held < both * c.kv_heads) continue;
      paired = true;
      cluster = s;
      shared_by = both;
    }
  }
  // A generous max_tokens over many documents: CTAs past a thousand rounds take several blocks of rows instead.
  const int64_t units = shared_by * c.kv_heads * cluster;
  a.row_blocks = static_cast<int>(std::min<int64_t>(a.row_blocks, std::max<int64_t>(1, kMostBlocks / units)));
  const int64_t blocks = units * a.row_blocks;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  auto go = [&](auto type, auto e4m3) {
    return paired ? launch<decltype(type), e4m3.value, true>(a, cluster, blocks, err, st)
                  : launch<decltype(type), e4m3.value, false>(a, cluster, blocks, err, st);
  };
  if (c.e4m3) return dtype == kF16 ? go(__half(), std::true_type()) : go(__nv_bfloat16(), std::true_type());
  return dtype == kF16 ? go(__half(), std::false_type()) : go(__nv_bfloat16(), std::false_type());
}

}  // namespace va
