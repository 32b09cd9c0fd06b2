// Masked attention of tiles that hold only a few query rows (single tokens over long documents).
//
// The same operator as va_masked.cu's; a tcgen05 tile of 128 rows spends its softmax and its two
// cluster barriers on padding there, so the launch comes here when no tile has more than kMaxRows
// rows.  Bound by HBM: every visible key costs 256 bytes per key head and is used by at most 16
// rows.  Layout, score terms and joins as in va_rows.cuh; keys and values are the operands as they
// are (no conversion), the query row too (its low half rows are zero), and a probability keeps a
// high and a low part, so the result is closer to F32 than the tile kernel's.  f16's steps end at
// 2^-24, so there probabilities are lifted by 2^kLift, and the sums with them (it cancels in the quotient): each is
// off by at most 2^-22 of itself or 2^-40 of the row's largest.
//
// A cluster of CTAs shares one (tile, key head, 8-row block); its warps take 32-key chunks in turn
// through a ring of their own in shared memory (cp.async, one chunk ahead).  Measured on B200: one token
// over 10,392 keys x 12 heads 9.4 us (16.8 in the tile kernel; 3.4 TB/s), of which a launch without
// keys is 4: five or six chunks a warp, one after the other, and the cluster's join are the rest.
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
constexpr int kChunk = 32;  // keys a warp takes at a time
constexpr int kTiles = kChunk / 8;
constexpr int kStages = 2;  // chunks of a warp in shared memory
constexpr int kCtasPerSm = 3;
constexpr int kMaxRows = 16;

// Rows of 64 two-byte elements; the 16-byte piece p of row r lies at piece p ^ (r % 8).
struct Chunk {
  uint4 k[kChunk][8];
  uint4 v[kChunk][8];
};
struct Shared {
  union {
    Chunk ring[kWarps][kStages];
    Join<kWarps> join;  // once the block's last chunk is used
  };
  Part part[kMaxCluster];  // [own row][cluster rank]
};
static_assert(kCtasPerSm * (sizeof(Shared) + 1024) <= 228 * 1024, "shared memory of an SM");

struct RowsArgs {
  MaskedArgs m;
  HeadsRef q, k, v;
  int row_blocks, splits;
  uint32_t frame_magic;
};

// Rows past `last` repeat it: a hidden key's probability is 0 and its values stay a document's own.
__device__ __forceinline__ void load_chunk(Chunk& ch, const char* k, const char* v, int64_t k_step, int64_t v_step,
                                           int key0, int last, int lane) {
  const int row = lane >> 3, p = lane & 7;
#pragma unroll
  for (int i = 0; i < kChunk / 4; ++i) {
    const int r = 4 * i + row;
    const int64_t key = min(key0 + r, last);
    cp16(&ch.k[r][p ^ (r & 7)], k + key * k_step + 16 * p);
    cp16(&ch.v[r][p ^ (r & 7)], v + key * v_step + 16 * p);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) rows_attn_kernel(const __grid_constant__ RowsArgs a) {
  constexpr float kLift = std::is_same<T, __half>::value ? 15.0f : 0.0f;  // so a probability is at most 2^15
  extern __shared__ uint4 smem_raw[];
  Shared& smem = *reinterpret_cast<Shared*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const AttnTerms& t = a.m.t;
  const int group = a.m.group;
  const int rank = static_cast<int>(blockIdx.x) % a.splits;
  int unit = static_cast<int>(blockIdx.x) / a.splits;
  const int kvh = unit % t.kv_heads;
  unit /= t.kv_heads;
  const int rb = unit % a.row_blocks;
  const MaskedItem it = a.m.item[unit / a.row_blocks];
  const int q_rows = it.tokens * group;
  if (rb * kRowsPerBlock >= q_rows) return;  // the same for every CTA of the cluster
  if (a.splits > 1) cluster_arrive();

  auto limit_of = [&](int token) {
    if (!t.causal) return it.doc_keys;
    const int64_t f = static_cast<int64_t>(frame_index(it.first + token, t.frame, a.frame_magic) + 1) * t.frame;
    return static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(it.doc_keys),
                                                             max(f, static_cast<int64_t>(it.prefix)))));
  };
  const int r = rb * kRowsPerBlock + g;  // this lane's query row
  const bool valid = r < q_rows;
  const int token = valid ? r / group : it.tokens - 1;
  const int head = kvh * group + (valid ? r - token * group : 0);
  const int block_limit = limit_of(min(rb * kRowsPerBlock + kRowsPerBlock - 1, q_rows - 1) / group);
  const int limit = valid ? limit_of(token) : block_limit;
  const int fp = frame_index(it.first + token, t.frame, a.frame_magic);
  const float slope = a.m.slopes ? __ldg(a.m.slopes + head) : 0.0f;

  RawRow raw;
  load_row(raw, static_cast<const T*>(a.q.data) + (it.q_row + static_cast<int64_t>(token)) * a.q.token_stride +
                    head * a.q.head_stride + 16 * c);
  const char* k = reinterpret_cast<const char*>(static_cast<const T*>(a.k.data) + it.k_row * a.k.token_stride +
                                                kvh * a.k.head_stride);
  const char* v = reinterpret_cast<const char*>(static_cast<const T*>(a.v.data) + it.k_row * a.v.token_stride +
                                                kvh * a.v.head_stride);
  const int64_t k_step = a.k.token_stride * 2, v_step = a.v.token_stride * 2;
  const int last = it.doc_keys - 1;
  const int chunks = (block_limit + kChunk - 1) / kChunk;
  const int stride = a.splits * kWarps;
  const int first = rank * kWarps + warp;
  Chunk* ring = smem.ring[warp];
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (first + i * stride < chunks) load_chunk(ring[i], k, v, k_step, v_step, (first + i * stride) * kChunk, last, lane);
    cp_commit();
  }
  // The row in fragment order (16 channels [16c, 16c + 16)); no low part.
  uint32_t qa[4][4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const uint4 u = raw.u[s >> 1];
    qa[s][0] = valid ? (s & 1 ? u.z : u.x) : 0u;
    qa[s][2] = valid ? (s & 1 ? u.w : u.y) : 0u;
    qa[s][1] = qa[s][3] = 0u;
  }

  float o[8][4];
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  int stage = 0;
  for (int ch = first; ch < chunks; ch += stride) {
    cp_wait<kStages - 2>();
    __syncwarp();  // every lane's copies have landed, and the stage below is read out
    {
      const int next = ch + (kStages - 1) * stride;
      const int to = stage == 0 ? kStages - 1 : stage - 1;
      if (next < chunks) load_chunk(ring[to], k, v, k_step, v_step, next * kChunk, last, lane);
      cp_commit();
    }
    const Chunk& cur = ring[stage];
    stage = stage + 1 == kStages ? 0 : stage + 1;
    const int key0 = ch * kChunk;
    float x[kTiles][2], d[kTiles][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) d[i][e] = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 w[kTiles];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const int kr = 8 * i + tile_key(g);
        w[i] = cur.k[kr][(2 * c + h) ^ (kr & 7)];
      }
#pragma unroll
      for (int i = 0; i < kTiles; ++i) mma(T(), d[i], qa[2 * h], w[i].x, w[i].y);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) mma(T(), d[i], qa[2 * h + 1], w[i].z, w[i].w);
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) x[i][e] = d[i][e];
    apply_terms<true>(x, t, t.scale_log2, t.cap_in, a.m.slopes != nullptr, slope, fp, key0, limit, c, a.frame_magic);
    float top = x[0][0];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) top = max3f(top, x[i][0], x[i][1]);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float m_new = fmaxf(m, top);
    if (__any_sync(0xffffffffu, m_new > m)) {
      const float alpha = m_new > m ? ex2(m - m_new) : 1.0f;  // 0 for the first keys
      l *= alpha;
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= alpha;
      m = m_new;
    }
    const float base = (m == -INFINITY ? 0.0f : m) - kLift;
#pragma unroll
    for (int u = 0; u < kTiles / 2; ++u) {
      uint32_t pa[4];
      uint4 vw[4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = 2 * u + half;
        float p[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int kk = 8 * i + ((2 * c + e) ^ (c & 1));
          vw[2 * half + e] = cur.v[kk][g ^ (kk & 7)];
          p[e] = ex2(x[i][e] - base);
          l += p[e];
        }
        split2(T(), p[0], p[1], pa[2 * half], pa[2 * half + 1]);
      }
#pragma unroll
      for (int word = 0; word < 4; ++word) {
        auto pick = [&](const uint4& w) { return word == 0 ? w.x : word == 1 ? w.y : word == 2 ? w.z : w.w; };
        const uint32_t a0 = pick(vw[0]), a1 = pick(vw[1]), b0 = pick(vw[2]), b1 = pick(vw[3]);
        mma(T(), o[2 * word], pa, prmt(a0, a1, 0x5410), prmt(b0, b1, 0x5410));
        mma(T(), o[2 * word + 1], pa, prmt(a0, a1, 0x7632), prmt(b0, b1, 0x7632));
      }
    }
  }
  cp_wait<0>();
  __syncthreads();  // every warp is done with its ring: the join buffers may cover it
  finish_block<T>(smem.join, smem.part, o, m, l, 1.0f, rb, q_rows, group, kvh, rank, a.splits, a.splits, 0, it.q_row,
                  a.m.out);
}

template <class T>
cudaError_t launch(const RowsArgs& a, int64_t blocks, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = prepare_kernel(reinterpret_cast<const void*>(rows_attn_kernel<T>), sizeof(Shared), ready);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, rows_attn_kernel<T>, a);
}

}  // namespace

bool rows_form(int most_rows) { return most_rows <= kMaxRows; }

int rows_splits(int64_t units, int most_keys, int sms) {
  // As many CTAs as the SMs hold at once, at least one chunk per warp.
  const int64_t most = std::max<int64_t>(1, most_keys / (kChunk * kWarps));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kMaxCluster, most, kCtasPerSm * static_cast<int64_t>(sms) / units})));
}

cudaError_t launch_rows(const HeadsRef& q, const HeadsRef& k, const HeadsRef& v, const MaskedArgs& m, int most_rows,
                        int dtype, cudaStream_t st) {
  RowsArgs a{};
  a.m = m;
  a.q = q;
  a.k = k;
  a.v = v;
  a.row_blocks = (most_rows + kRowsPerBlock - 1) / kRowsPerBlock;
  a.splits = m.splits;
  a.frame_magic = static_cast<uint32_t>((1ull << 32) / static_cast<uint32_t>(std::max(2, m.t.frame)));
  const int64_t blocks = static_cast<int64_t>(m.items) * m.t.kv_heads * a.row_blocks * a.splits;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  return dtype == kF16 ? launch<__half>(a, blocks, st) : launch<__nv_bfloat16>(a, blocks, st);
}

}  // namespace va
