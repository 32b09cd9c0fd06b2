// Shared parts of the attention kernels for a few query rows per key head (va_cache_attn.cu over
// the quantised cache, va_rows_attn.cu over dense keys and values): fragment layout, score terms,
// and the joining of the warps and of the cluster.
//
// A row block is 8 query rows of one key head.  The products are m16n8k16 tensor-core instructions
// (mma.sync: a tcgen05 tile of 128 rows would be 94 % padding, and the operands come from
// registers): accumulator rows 0..7 hold the products of the operand's high part, rows 8..15 those
// of the rest.  Lane (g, c) = (lane / 4, lane % 4) of a warp holds row g.  Column n of an 8-key tile is
// key tile_key(n) of the tile.
//
// The channel order inside a product is free as long as both operands use the same, so a lane
// loads 16 consecutive channels [16c, 16c + 16) of one key, and its k indices of step s are channels
// 16c + 4s .. + 3; the query row is loaded with the same order.  For the second product the key order is
// free: a lane loads channels [8g, 8g + 8) of the keys whose probabilities it holds.
#pragma once

#include <type_traits>

#include "va_internal.h"
#include "va_ptx.cuh"
#include "va_stream.cuh"

namespace va {
namespace rows {

constexpr int kHeadDim = 64;
constexpr int kRowsPerBlock = 8;
constexpr int kMaxCluster = 16;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void mma(__half /*type*/, float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma(__nv_bfloat16 /*type*/, float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
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

// x in two f16 parts, packed with a neighbour's: hi = f16(x), lo = f16(x - hi).
__device__ __forceinline__ void split2(__half /*type*/, float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = f16x2_from_f32(x0, x1);
  const float2 h = __half22float2(*reinterpret_cast<__half2*>(&hi));
  lo = f16x2_from_f32(x0 - h.x, x1 - h.y);
}

// The same in bf16.
__device__ __forceinline__ void split2(__nv_bfloat16 /*type*/, float x0, float x1, uint32_t& hi, uint32_t& lo) {
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

// Key of column n of an 8-key tile: with this order a warp's loads of key rows and of value rows
// from swizzled shared memory meet no bank twice.
__device__ __forceinline__ int tile_key(int n) { return n ^ ((n >> 1) & 1); }

__device__ __forceinline__ void cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 16 consecutive two-byte elements.
struct RawRow {
  uint4 u[2];
};
__device__ __forceinline__ void load_row(RawRow& r, const void* p) {
  r.u[0] = __ldg(static_cast<const uint4*>(p));
  r.u[1] = __ldg(static_cast<const uint4*>(p) + 1);
}
template <class T>
__device__ __forceinline__ void unpack_row(const RawRow& r, float* x) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t w[4] = {r.u[h].x, r.u[h].y, r.u[h].z, r.u[h].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[8 * h + 2 * i] = f.x;
        x[8 * h + 2 * i + 1] = f.y;
      } else {
        x[8 * h + 2 * i] = __uint_as_float(w[i] << 16);
        x[8 * h + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
}
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }

// Scores of the lane's keys from their products (x, times the key's scale): scale or cap, distance
// bias, mask.  Each term over all scores of the lane under one branch, so that they overlap.
// score_scale = scale log2(e), cap_scale = 2 log2(e) scale / cap, both times what x lacks.
// kMask false: every row sees the whole chunk.
template <bool kMask, int kTiles>
__device__ __forceinline__ void apply_terms(float (&x)[kTiles][2], const AttnTerms& t, float score_scale, float cap_scale,
                                            bool biased, float slope, int frame_at, int key0, int limit, int c,
                                            uint32_t frame_magic) {
#define VA_EACH_SCORE(...)                                 \
  _Pragma("unroll") for (int i = 0; i < kTiles; ++i) {     \
    _Pragma("unroll") for (int e = 0; e < 2; ++e) {        \
      const int kk = 8 * i + ((2 * c + e) ^ (c & 1));      \
      __VA_ARGS__                                          \
    }                                                      \
  }
  if (t.cap_out > 0.0f) {
    // cap log2(e) tanh(z) = cap log2(e) (1 - 2 / (1 + e^(2z)))
    VA_EACH_SCORE((void)kk; x[i][e] = fmaf(-2.0f * t.cap_out, rcp(1.0f + ex2(x[i][e] * cap_scale)), t.cap_out);)
  } else {
    VA_EACH_SCORE((void)kk; x[i][e] *= score_scale;)
  }
  if (biased) {
    if (t.frame == 1) {
      const float ahead = static_cast<float>(frame_at - key0);  // tokens past the chunk's first
      VA_EACH_SCORE(x[i][e] = fmaf(-slope, fabsf(ahead - static_cast<float>(kk)), x[i][e]);)
    } else {
      VA_EACH_SCORE(const float dist = static_cast<float>(frame_at - frame_index(key0 + kk, t.frame, frame_magic));
                    x[i][e] = fmaf(-slope, fabsf(dist), x[i][e]);)
    }
  }
  if (kMask && __any_sync(0xffffffffu, key0 + 8 * kTiles > limit)) {
    VA_EACH_SCORE(x[i][e] = key0 + kk < limit ? x[i][e] : -INFINITY;)
  }
#undef VA_EACH_SCORE
}

// The warps' results of a row block.  Channel ch of a row lies at slot(ch): the order in which
// a lane's accumulators are neighbours; rows are padded against bank conflicts.
__device__ __forceinline__ int slot(int ch) { return (ch & 7) * 8 + (ch >> 3); }
template <int kWarps>
struct Join {
  float o[kWarps][kRowsPerBlock][kHeadDim + 8];
  float m[kWarps][kRowsPerBlock], l[kWarps][kRowsPerBlock];
};
// What the CTAs of a document send to the CTA that finishes a row: rows r, r + splits, ... go to
// CTA r % splits, so a CTA receives at most 16 (splits x rows) parts.
struct Part {
  float o[kHeadDim];
  float m, l;
};
// Stores v at this address of CTA `rank` of the cluster.
__device__ __forceinline__ void st_cluster(float* p, int rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr(smem_u32(p), rank)), "f"(v) : "memory");
}

// Joins the warps' results of a row block (o, m, l of every lane; `back` undoes a scaling of o) and
// the cluster's, and writes the block's rows.  base: output row of the first token; rb: the block.  The `splits` CTAs that share the
// document's keys stand in a cluster of `cluster` from rank `lead` on; the caller has arrived at the cluster's barrier once,
// and every CTA of the cluster takes part in two more phases here (or stands in for them).
template <class T, int kWarps>
__device__ __forceinline__ void finish_block(Join<kWarps>& sh, Part* parts, const float (&o)[8][4], float m, float l,
                                             float back, int rb, int q_rows, int group, int kvh, int rank, int splits,
                                             int cluster, int lead, int64_t base, const HeadsRef& out) {
  constexpr int kThreads = kWarps * 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  // Row sums over the four lanes of a row; accumulator column 2c + e of tile n is
  // channel 8 (2c + e) + n (the value operand's column g holds channel 8g + n).
  const int rows = min(kRowsPerBlock, q_rows - rb * kRowsPerBlock);
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (g < rows) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
      *reinterpret_cast<float2*>(&sh.o[warp][g][8 * n + 2 * c]) =
          make_float2((o[n][0] + o[n][2]) * back, (o[n][1] + o[n][3]) * back);
    if (c == 0) {
      sh.m[warp][g] = m;
      sh.l[warp][g] = l;
    }
  }
  __syncthreads();
  if (cluster > 1) cluster_wait();
  // Join the warps and hand each row to the CTA that finishes it.
  for (int i = threadIdx.x; i < rows * kHeadDim; i += kThreads) {
    const int row = i / kHeadDim, at = i % kHeadDim;
    float mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, sh.m[w][row]);
    float os = 0.0f, ls = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = sh.m[w][row] == -INFINITY ? 0.0f : ex2(sh.m[w][row] - mt);
      os += f * sh.o[w][row][at];
      ls += f * sh.l[w][row];
    }
    const int owner = row % splits;
    Part& to = parts[row / splits * splits + rank];
    st_cluster(&to.o[at], lead + owner, os);
    if (at == 0) {
      st_cluster(&to.m, lead + owner, mt);
      st_cluster(&to.l, lead + owner, ls);
    }
  }
  if (cluster > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  // This CTA's rows rank, rank + splits, ...: the cluster's parts in rank order.
  for (int i = threadIdx.x; rank + i / kHeadDim * splits < rows; i += kThreads) {
    const int own = i / kHeadDim, ch = i % kHeadDim;
    const Part* part = parts + own * splits;
    float mt = -INFINITY, os = 0.0f, ls = 0.0f;
    for (int p = 0; p < splits; ++p) mt = fmaxf(mt, part[p].m);
    for (int p = 0; p < splits; ++p) {
      const float f = part[p].m == -INFINITY ? 0.0f : ex2(part[p].m - mt);
      os += f * part[p].o[slot(ch)];
      ls += f * part[p].l;
    }
    const int rr = rb * kRowsPerBlock + rank + own * splits;
    put(static_cast<T*>(out.data) + (base + rr / group) * out.token_stride +
            static_cast<int64_t>(kvh * group + rr % group) * out.head_stride + ch,
        ls == 0.0f ? 0.0f : os / ls);
  }
}

}  // namespace rows
}  // namespace va
