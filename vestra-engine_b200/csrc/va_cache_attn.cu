// Attention of a few new tokens per document over the quantised key/value cache.
//
//   out_i = sum_j p_ij vs_j V_j / sum_j p_ij,   p_ij = exp(score_ij - max_j score_ij),
//   score_ij = cap tanh(scale ks_j (q_i . K_j) / cap) - slope |f(P_i) - f(j)|
// with K_j, V_j the integer or e4m3 codes and ks_j, vs_j their scales: a key's scale
// multiplies its scores, a value's scale its probability, so codes are never scaled.
//
// Bound by HBM: every visible key costs 2 * (64 + 4) bytes per key head and 256 FLOP per
// query row.  A row block is 8 query rows of one key head (tokens x the heads that share
// it), so the products are m16n8k16 tensor-core instructions (mma.sync: the tcgen05 tile
// of 128 rows would be 94 % padding, and the operands come from registers): rows 0..7
// hold the high bf16 part of the row, rows 8..15 the rest, which makes the product of an
// f16 row, and of the F32 probabilities, good to 2^-16 at no further instruction.
//
// A cluster of CTAs shares one (document, key head, row block); its warps take 32-key
// chunks in turn straight from global memory into registers (one chunk ahead), each warp
// with its own running maximum and sum, and the partial results meet in shared memory
// and then, through distributed shared memory, across the cluster in rank order: one
// launch, no workspace, no atomics, and the same bits on every run.
//
// Operand layout: the channel order inside a product is free as long as both operands
// use the same, so lane (g, c) = (lane / 4, lane % 4) loads 16 consecutive code bytes
// [16c, 16c + 16) of key g of an 8-key tile (one 512-byte warp load), and its word s
// holds the lane's k indices of step s; the query row is loaded with the same
// order.  For the second product the key order is free: lane (g, c) loads channels [8g, 8g + 8)
// of the four keys whose probabilities it holds.
#include <algorithm>

#include <cooperative_groups.h>

#include "va_internal.h"
#include "va_ptx.cuh"

namespace va {

namespace {

constexpr int kHeadDim = 64;
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRowsPerBlock = 8;
constexpr int kChunk = 32;         // keys a warp takes at a time
constexpr int kMaxCluster = 16;
constexpr float kLog2e = 1.4426950408889634f;

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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

// Two code bytes of w -> bf16x2, exactly.  kHigh: bytes 2 and 3, else 0 and 1.
// int8 c: with the byte under 0x43, 0x4300 | (c & 0x7f) is the bf16 128 + (c & 127) and
//   0x4300 | (c & 0x80) is 128 or, for a negative code, 256: their difference is c.
// e4m3 s.eeee.mmm: moved under bf16's exponent the bits read as the value times 2^-120
//   (subnormals included), undone by an exact multiplication.  The NaN code reads as 480.
template <bool kE4m3, bool kHigh>
__device__ __forceinline__ uint32_t codes_to_bf16x2(uint32_t w) {
  if constexpr (kE4m3) {
    const uint32_t t = prmt(w, 0u, kHigh ? 0x3424u : 0x1404u);  // bytes: 0, c0, 0, c1
    const uint32_t u = ((t >> 4) & 0x07f007f0u) | (t & 0x80008000u);
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x7b807b80u));  // 2^120
    return r;
  } else {
    const uint32_t t = prmt(w, 0x43434343u, kHigh ? 0x4342u : 0x4140u);  // bytes: c0, 43, c1, 43
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(t & 0xff7fff7fu), "r"(t & 0xff80ff80u));
    return r;
  }
}

// x in two bf16 parts, packed with a neighbour's: hi = bf16(x), lo = bf16(x - hi).
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(x0, x1);
  lo = pack_bf16x2(x0 - __uint_as_float(hi << 16), x1 - __uint_as_float(hi & 0xffff0000u));
}

// floor(p / frame), magic = floor(2^32 / frame).
__device__ __forceinline__ int frame_index(int p, int frame, uint32_t magic) {
  if (frame == 1) return p;
  const uint32_t x = static_cast<uint32_t>(p < 0 ? -1 - p : p);
  uint32_t q = __umulhi(x, magic);  // x / frame or one less
  if (x - q * frame >= static_cast<uint32_t>(frame)) ++q;
  return p < 0 ? -1 - static_cast<int>(q) : static_cast<int>(q);
}

// One 32-key chunk in registers: lane (g, c) holds key 8t + g's bytes [16c, 16c + 16) for
// t = 0..3, and of each 16-key half u the value bytes [8g, 8g + 8) of keys 16u + {2c,
// 2c + 1, 8 + 2c, 9 + 2c}; scales of the keys whose scores it will hold.
struct Chunk {
  uint4 k[4];
  uint2 v[2][4];
  float ks[4][2], vs[4][2];
};

__device__ __forceinline__ void load_chunk(Chunk& ch, const uint8_t* kc, const uint8_t* vc, const float* ks,
                                           const float* vs, int key0, int last, int g, int c) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int64_t key = min(key0 + 8 * t + g, last);
    ch.k[t] = __ldcs(reinterpret_cast<const uint4*>(kc + key * kHeadDim + 16 * c));
    const int64_t j0 = min(key0 + 8 * t + 2 * c, last), j1 = min(key0 + 8 * t + 2 * c + 1, last);
    ch.ks[t][0] = __ldg(ks + j0), ch.ks[t][1] = __ldg(ks + j1);
    ch.vs[t][0] = __ldg(vs + j0), ch.vs[t][1] = __ldg(vs + j1);
    ch.v[t >> 1][2 * (t & 1)] = __ldcs(reinterpret_cast<const uint2*>(vc + j0 * kHeadDim + 8 * g));
    ch.v[t >> 1][2 * (t & 1) + 1] = __ldcs(reinterpret_cast<const uint2*>(vc + j1 * kHeadDim + 8 * g));
  }
}

struct Shared {
  float o[kWarps][kRowsPerBlock][kHeadDim];
  float m[kWarps][kRowsPerBlock], l[kWarps][kRowsPerBlock];
  // the CTA's result, read by the cluster
  float co[kRowsPerBlock][kHeadDim];
  float cm[kRowsPerBlock], cl[kRowsPerBlock];
};

__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

template <class T>
__device__ __forceinline__ float elem(const T* p);
template <>
__device__ __forceinline__ float elem(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <>
__device__ __forceinline__ float elem(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }

template <class T, bool kE4m3>
__global__ void __launch_bounds__(kThreads, 2)
    cache_attn_kernel(const __grid_constant__ CacheAttnArgs a, int splits, int* err) {
  __shared__ Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int rank = static_cast<int>(blockIdx.x) % splits;
  int unit = static_cast<int>(blockIdx.x) / splits;
  const int kvh = unit % a.c.kv_heads;
  unit /= a.c.kv_heads;
  const int block0 = unit % a.row_blocks;
  const int doc = unit / a.row_blocks;

  const int32_t begin = __ldg(a.offsets + doc), end = __ldg(a.offsets + doc + 1);
  const int32_t len = __ldg(a.lens + doc);
  const bool ok = begin >= 0 && end >= begin && end <= a.rows && len >= 0 && len <= a.c.capacity;
  if (!ok) {  // the same for every CTA of the cluster: none of them waits
    if (threadIdx.x == 0) report_error(err, kDevBadLengths);
    return;
  }
  const int tokens = end - begin;
  const int q_rows = tokens * a.group;
  const int prefix = a.prefix ? max(__ldg(a.prefix + doc), 0) : 0;
  const int64_t head_base = (static_cast<int64_t>(doc) * a.c.kv_heads + kvh) * a.c.capacity;
  const uint8_t* kc = a.c.codes[0] + head_base * kHeadDim;
  const uint8_t* vc = a.c.codes[1] + head_base * kHeadDim;
  const float* ks = a.c.scales[0] + head_base;
  const float* vs = a.c.scales[1] + head_base;
  const T* qd = static_cast<const T*>(a.q.data);
  T* od = static_cast<T*>(a.out.data);

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

  for (int rb = block0; rb * kRowsPerBlock < q_rows; rb += a.row_blocks) {
    const int r = rb * kRowsPerBlock + g;  // this lane's query row
    const bool valid = r < q_rows;
    const int token = valid ? r / a.group : tokens - 1;
    const int head = kvh * a.group + (valid ? r % a.group : 0);
    const int limit = valid ? limit_of(token) : 0;
    const int block_limit = limit_of(min(rb * kRowsPerBlock + kRowsPerBlock - 1, q_rows - 1) / a.group);
    const int fp = frame_index(token + len - tokens, a.t.frame, a.frame_magic);
    const float slope = a.slopes ? __ldg(a.slopes + head) * kLog2e : 0.0f;

    // Query row in fragment order: word s of the lane's 16 channels [16c, 16c + 16).
    uint32_t qa[4][4];
    {
      const T* p = qd + (begin + static_cast<int64_t>(token)) * a.q.token_stride + head * a.q.head_stride + 16 * c;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = valid ? elem(p + 4 * s + e) : 0.0f;
        split2(x[0], x[1], qa[s][0], qa[s][1]);
        split2(x[2], x[3], qa[s][2], qa[s][3]);
      }
    }

    float o[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    const int chunks = (block_limit + kChunk - 1) / kChunk;
    const int stride = splits * kWarps;
    int ch = rank * kWarps + warp;
    Chunk cur;
    if (ch < chunks) load_chunk(cur, kc, vc, ks, vs, ch * kChunk, len - 1, g, c);
    for (; ch < chunks; ch += stride) {
      const int key0 = ch * kChunk;
      // Scores of 8 rows x 32 keys: lane (g, c) gets row g, keys 8t + 2c and 8t + 2c + 1.
      float x[4][2];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t w[4] = {cur.k[t].x, cur.k[t].y, cur.k[t].z, cur.k[t].w};
#pragma unroll
        for (int s = 0; s < 4; ++s)
          mma_bf16(d, qa[s], codes_to_bf16x2<kE4m3, false>(w[s]), codes_to_bf16x2<kE4m3, true>(w[s]));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float dot = (d[e] + d[2 + e]) * cur.ks[t][e];
          float y;
          if (a.t.cap_out > 0.0f) {
            // cap log2(e) tanh(z) = cap log2(e) (1 - 2 / (1 + e^(2z)))
            y = a.t.cap_out * (1.0f - __fdividef(2.0f, 1.0f + ex2(dot * a.t.cap_in)));
          } else {
            y = dot * a.t.scale_log2;
          }
          const int key = key0 + 8 * t + 2 * c + e;
          if (a.slopes) {
            const int dist = fp - frame_index(key, a.t.frame, a.frame_magic);
            y -= slope * static_cast<float>(abs(dist));
          }
          x[t][e] = key < limit ? y : -INFINITY;
        }
      }
      float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1])),
                        fmaxf(fmaxf(x[2][0], x[2][1]), fmaxf(x[3][0], x[3][1])));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float m_new = fmaxf(m, top);
      if (__any_sync(0xffffffffu, m_new > m)) {
        const float alpha = m_new > m ? ex2(m - m_new) : 1.0f;  // 0 for the first keys
        l *= alpha;
        // Accumulator rows g (elements 0, 1) and g + 8 (2, 3) are parts of query row g.
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][e] *= alpha;
        m = m_new;
      }
      const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t pa[4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int t = 2 * u + half;
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = ex2(x[t][e] - base);
            l += p;
            // A hidden key's value scale may be anything (stale rows): not multiplied.
            w[e] = x[t][e] == -INFINITY ? 0.0f : p * cur.vs[t][e];
          }
          split2(w[0], w[1], pa[2 * half], pa[2 * half + 1]);
        }
#pragma unroll
        for (int word = 0; word < 2; ++word) {
          // Four channels of keys (2c, 2c + 1) and (8 + 2c, 9 + 2c), interleaved in pairs.
          const uint32_t a0 = word ? cur.v[u][0].y : cur.v[u][0].x, a1 = word ? cur.v[u][1].y : cur.v[u][1].x;
          const uint32_t b0 = word ? cur.v[u][2].y : cur.v[u][2].x, b1 = word ? cur.v[u][3].y : cur.v[u][3].x;
          const uint32_t lo0 = prmt(a0, a1, 0x5140), hi0 = prmt(a0, a1, 0x7362);
          const uint32_t lo1 = prmt(b0, b1, 0x5140), hi1 = prmt(b0, b1, 0x7362);
          mma_bf16(o[4 * word + 0], pa, codes_to_bf16x2<kE4m3, false>(lo0), codes_to_bf16x2<kE4m3, false>(lo1));
          mma_bf16(o[4 * word + 1], pa, codes_to_bf16x2<kE4m3, true>(lo0), codes_to_bf16x2<kE4m3, true>(lo1));
          mma_bf16(o[4 * word + 2], pa, codes_to_bf16x2<kE4m3, false>(hi0), codes_to_bf16x2<kE4m3, false>(hi1));
          mma_bf16(o[4 * word + 3], pa, codes_to_bf16x2<kE4m3, true>(hi0), codes_to_bf16x2<kE4m3, true>(hi1));
        }
      }
      if (ch + stride < chunks) load_chunk(cur, kc, vc, ks, vs, (ch + stride) * kChunk, len - 1, g, c);
    }
    // Row sums over the four lanes of a row; accumulator column 2c + e of tile n is
    // channel 8 (2c + e) + n (the value operand's column g holds channel 8g + n).
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) sh.o[warp][g][8 * (2 * c + e) + n] = o[n][e] + o[n][2 + e];
    if (c == 0) {
      sh.m[warp][g] = m;
      sh.l[warp][g] = l;
    }
    __syncthreads();
    // Join the warps: 512 outputs over 256 threads.
    for (int i = threadIdx.x; i < kRowsPerBlock * kHeadDim; i += kThreads) {
      const int row = i / kHeadDim, col = i % kHeadDim;
      float mt = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, sh.m[w][row]);
      float os = 0.0f, ls = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = sh.m[w][row] == -INFINITY ? 0.0f : ex2(sh.m[w][row] - mt);
        os += f * sh.o[w][row][col];
        ls += f * sh.l[w][row];
      }
      sh.co[row][col] = os;
      if (col == 0) {
        sh.cm[row] = mt;
        sh.cl[row] = ls;
      }
    }
    if (splits > 1) {
      cooperative_groups::this_cluster().sync();
    } else {
      __syncthreads();
    }
    // Join the cluster: CTA `rank` writes outputs rank, rank + splits, ... in blocks of 64
    // divided evenly.
    for (int i = rank * kThreads + threadIdx.x; i < kRowsPerBlock * kHeadDim; i += splits * kThreads) {
      const int row = i / kHeadDim, col = i % kHeadDim;
      const int rr = rb * kRowsPerBlock + row;
      if (rr >= q_rows) continue;
      float mt = -INFINITY, os = 0.0f, ls = 0.0f;
      if (splits > 1) {
        for (int p = 0; p < splits; ++p) mt = fmaxf(mt, ld_cluster(&sh.cm[row], p));
        for (int p = 0; p < splits; ++p) {
          const float mp = ld_cluster(&sh.cm[row], p);
          const float f = mp == -INFINITY ? 0.0f : ex2(mp - mt);
          os += f * ld_cluster(&sh.co[row][col], p);
          ls += f * ld_cluster(&sh.cl[row], p);
        }
      } else {
        os = sh.co[row][col];
        ls = sh.cl[row];
      }
      put(od + (begin + static_cast<int64_t>(rr / a.group)) * a.out.token_stride +
              static_cast<int64_t>(kvh * a.group + rr % a.group) * a.out.head_stride + col,
          ls == 0.0f ? 0.0f : os / ls);
    }
    // The next row block, or the exit, must not overwrite what a peer still reads.
    if (splits > 1) {
      cooperative_groups::this_cluster().sync();
    } else {
      __syncthreads();
    }
  }
}

template <class T, bool kE4m3>
cudaError_t launch(const CacheAttnArgs& a, int splits, int64_t blocks, int* err, cudaStream_t st) {
  auto kern = cache_attn_kernel<T, kE4m3>;
  if (splits > 8) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a, splits, err);
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
  const int64_t units = static_cast<int64_t>(c.documents) * c.kv_heads * a.row_blocks;
  // CTAs per unit: enough for two per SM, at least four chunks per warp of the capacity.
  const int64_t most = std::max<int64_t>(1, c.capacity / (4 * kChunk * kWarps));
  int splits = 1;
  while (splits < kMaxCluster && units * splits < 2 * sms && 2 * splits <= most) splits *= 2;
  const int64_t blocks = units * splits;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  if (c.e4m3)
    return dtype == kF16 ? launch<__half, true>(a, splits, blocks, err, st)
                         : launch<__nv_bfloat16, true>(a, splits, blocks, err, st);
  return dtype == kF16 ? launch<__half, false>(a, splits, blocks, err, st)
                       : launch<__nv_bfloat16, false>(a, splits, blocks, err, st);
}

}  // namespace va
