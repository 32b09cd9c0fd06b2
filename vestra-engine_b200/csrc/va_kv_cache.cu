// The quantised key/value cache: writing (quantise) and reading back.
//
// Layout: codes [document][kv head][capacity][64] bytes, scales [document][kv head]
// [capacity] F32.  Head-major, so the tokens of one head are one stream of 64-byte rows.
//
// Write and read are bound by HBM: each input element is read once, each output written
// once.  Eight lanes own one (token, head): 8 channels each, one 16-byte load of 2-byte
// elements, the row's largest magnitude by three shuffles.  A warp's four groups take
// four consecutive tokens of one head, so its code rows are 256 consecutive bytes.
// Measured on B200 (16 heads, f16, e4m3): 22,322 tokens written 26.3 us (5.3 TB/s), 31,321 read back 34.7 us
// (5.7 TB/s = 0.86 of measured).
#include <algorithm>

#include "va_internal.h"
#include "va_ptx.cuh"

namespace va {

namespace {

constexpr int kHeadDim = 64;
constexpr int kThreads = 256;

// ------------------------------------------------------------------ documents of rows
// Document of `row`, or -1: the last b with offsets[b] <= row, if row < offsets[b + 1].
__device__ __forceinline__ int document_of(const int32_t* offsets, int documents, int row) {
  int lo = 0, hi = documents;  // offsets[lo] <= row < offsets[hi] when row is inside
  if (row < __ldg(offsets) || row >= __ldg(offsets + documents)) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(offsets + mid) <= row)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Checks every document's offsets and token range (one block's threads); a bad one is
// reported, and the kernels skip it by the same test.
__device__ __forceinline__ bool document_ok(int32_t begin, int32_t end, int64_t first, int64_t rows,
                                            int64_t capacity) {
  return begin >= 0 && end >= begin && end <= rows && first >= 0 && first + (end - begin) <= capacity;
}

// Eight elements as loaded (so that several loads fit in few registers), then as F32.
template <class T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ void load8(const T* p, Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float* v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[4 * i] = __uint_as_float(r.u[i].x), v[4 * i + 1] = __uint_as_float(r.u[i].y);
    v[4 * i + 2] = __uint_as_float(r.u[i].z), v[4 * i + 3] = __uint_as_float(r.u[i].w);
  }
}
__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16>& r, float* v) {
  const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const Raw8<__half>& r, float* v) {
  const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float* v);
template <>
__device__ __forceinline__ void store8(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <>
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) {
  uint4 u;
  u.x = pack_bf16x2(v[0], v[1]), u.y = pack_bf16x2(v[2], v[3]);
  u.z = pack_bf16x2(v[4], v[5]), u.w = pack_bf16x2(v[6], v[7]);
  *reinterpret_cast<uint4*>(p) = u;
}
template <>
__device__ __forceinline__ void store8(__half* p, const float* v) {
  uint4 u;
  u.x = f16x2_from_f32(v[0], v[1]), u.y = f16x2_from_f32(v[2], v[3]);
  u.z = f16x2_from_f32(v[4], v[5]), u.w = f16x2_from_f32(v[6], v[7]);
  *reinterpret_cast<uint4*>(p) = u;
}

template <class T>
__device__ __forceinline__ float finite_max();
template <>
__device__ __forceinline__ float finite_max<float>() { return 3.402823466e38f; }
template <>
__device__ __forceinline__ float finite_max<__nv_bfloat16>() { return 3.38953139e38f; }
template <>
__device__ __forceinline__ float finite_max<__half>() { return 65504.0f; }

// rint(x / s) exactly (half to even), s = amax / 127 rounded: the candidate from a
// multiplication by the reciprocal is off by at most one; r = x - c s is exact in one
// FMA (c s and x are multiples of half an ulp of s and the difference is at most about s),
// so comparing it with s / 2 settles the code, ties included.
__device__ __forceinline__ int int8_code(float x, float s, float inv) {
  float c = rintf(x * inv);
  const float r = fmaf(-c, s, x), h = 0.5f * s;
  const bool odd = static_cast<int>(c) & 1;
  if (r > h || (r == h && odd)) c += 1.0f;
  if (r < -h || (r == -h && odd)) c -= 1.0f;
  return static_cast<int>(fminf(fmaxf(c, -127.0f), 127.0f));
}

// (lo, hi) F32 -> two e4m3 codes, round to nearest even, saturating.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two e4m3 codes -> f16x2 (exact).
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(codes)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

struct KvArgs {
  KvCacheRef c;
  int64_t rows;
  const int32_t* offsets;
  const int32_t* edge;  // write: lens; read: first (or nullptr)
  HeadsRef x[2];        // k, v
};

// Codes and scale of one head's eight channels (the eight lanes of a group hold 64).
template <bool kE4m3>
__device__ __forceinline__ uint2 quantise(const float* v, uint32_t group_mask, float* scale_out) {
  // The largest magnitude as an integer maximum of the bit patterns, which order like the
  // values with infinities and NaN on top.
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(group_mask, top, o));
  uint2 u = make_uint2(0u, 0u);
  *scale_out = __uint_as_float(0x7fffffffu);  // NaN: a head with a non-finite value
  if (top >= 0x7f800000u) return u;
  if (kE4m3) {
    // amax = f 2^e, 1 <= f < 2: 2^(e - 8), or 2^(e - 7) when f > 1.75.
    const int e = static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u);
    const int ec = max(e, -126);
    *scale_out = __uint_as_float(static_cast<uint32_t>(ec + 127) << 23);
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - ec) << 23);
    u.x = e4m3x2(v[0] * inv, v[1] * inv) | (e4m3x2(v[2] * inv, v[3] * inv) << 16);
    u.y = e4m3x2(v[4] * inv, v[5] * inv) | (e4m3x2(v[6] * inv, v[7] * inv) << 16);
  } else {
    const float scale = fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), 1.17549435e-38f);
    *scale_out = scale;
    const float inv = __fdiv_rn(1.0f, scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u.x |= static_cast<uint32_t>(int8_code(v[i], scale, inv) & 255) << (8 * i);
      u.y |= static_cast<uint32_t>(int8_code(v[4 + i], scale, inv) & 255) << (8 * i);
    }
  }
  return u;
}

template <bool kE4m3>
__device__ __forceinline__ void dequantise(uint2 u, float scale, float top, float* v) {
  if (kE4m3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = e4m3x2_to_f32((i < 2 ? u.x : u.y) >> (16 * (i & 1)));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = static_cast<float>(static_cast<int8_t>(u.x >> (8 * i)));
      v[4 + i] = static_cast<float>(static_cast<int8_t>(u.y >> (8 * i)));
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = v[i] * scale;
    v[i] = y != y ? y : fminf(fmaxf(y, -top), top);  // fmin and fmax drop a NaN
  }
}

// An eight-lane group takes one row and kHeads heads of K and of V: all its loads are
// issued before the first is used.
template <class T, bool kE4m3, bool kWrite, int kHeads>
__global__ void __launch_bounds__(kThreads) kv_rows_kernel(const __grid_constant__ KvArgs a, int* err) {
  const int heads = a.c.kv_heads;
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    for (int b = threadIdx.x; b < a.c.documents; b += kThreads) {
      const int32_t begin = __ldg(a.offsets + b), end = __ldg(a.offsets + b + 1);
      const int64_t n = static_cast<int64_t>(end) - begin;
      const int64_t first = kWrite ? __ldg(a.edge + b) - n : (a.edge ? __ldg(a.edge + b) : 0);
      if (!document_ok(begin, end, first, a.rows, a.c.capacity)) report_error(err, kDevBadLengths);
    }
  }
  const int lane8 = threadIdx.x & 7;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 8) + (threadIdx.x >> 3);
  // The eight lanes of a group share the row; the group leaves together.
  if (row >= a.rows) return;
  const int h0 = blockIdx.y * kHeads;
  const int doc = document_of(a.offsets, a.c.documents, static_cast<int>(row));
  if (doc < 0) return;
  const int32_t begin = __ldg(a.offsets + doc), end = __ldg(a.offsets + doc + 1);
  const int64_t n = static_cast<int64_t>(end) - begin;
  const int64_t first = kWrite ? __ldg(a.edge + doc) - n : (a.edge ? __ldg(a.edge + doc) : 0);
  if (row < begin || row >= end || !document_ok(begin, end, first, a.rows, a.c.capacity)) return;
  const int64_t token = first + (row - begin);
  const int64_t slot0 = (static_cast<int64_t>(doc) * heads + h0) * a.c.capacity + token;
  const uint32_t group_mask = 0xffu << (threadIdx.x & 24);
  if (kWrite) {
    Raw8<T> raw[2][kHeads];
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (h0 + i < heads)
          load8<T>(static_cast<const T*>(a.x[w].data) + row * a.x[w].token_stride + (h0 + i) * a.x[w].head_stride + 8 * lane8,
                   raw[w][i]);
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (h0 + i < heads) {
          const int64_t slot = slot0 + i * a.c.capacity;
          float scale, v[8];
          unpack8(raw[w][i], v);
          const uint2 u = quantise<kE4m3>(v, group_mask, &scale);
          *reinterpret_cast<uint2*>(a.c.codes[w] + slot * kHeadDim + 8 * lane8) = u;
          if (lane8 == 0) a.c.scales[w][slot] = scale;
        }
  } else {
    uint2 u[2][kHeads];
    float scale[2][kHeads];
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (h0 + i < heads) {
          const int64_t slot = slot0 + i * a.c.capacity;
          u[w][i] = *reinterpret_cast<const uint2*>(a.c.codes[w] + slot * kHeadDim + 8 * lane8);
          scale[w][i] = a.c.scales[w][slot];
        }
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (h0 + i < heads) {
          float v[8];
          dequantise<kE4m3>(u[w][i], scale[w][i], finite_max<T>(), v);
          store8<T>(static_cast<T*>(a.x[w].data) + row * a.x[w].token_stride + (h0 + i) * a.x[w].head_stride + 8 * lane8, v);
        }
  }
}

// Two heads per group where one would give at least 8 blocks per SM: more loads in flight per
// group and half the document searches (four windows of 24,000 rows written 29.3 -> 26.3 us,
// 33,000 read 42.8 -> 34.7 us = 5.7 TB/s); a few blocks are served sooner by more, lighter groups (866
// rows written 4.8 us against 5.9).
template <class T, bool kWrite>
cudaError_t launch_rows(const KvArgs& a, int sms, int* err, cudaStream_t st) {
  const int64_t bx = std::max<int64_t>(1, (a.rows + kThreads / 8 - 1) / (kThreads / 8));
  if (bx > 0x7fffffff) return cudaErrorInvalidValue;
  const int per = bx * a.c.kv_heads >= 8 * static_cast<int64_t>(sms) ? 2 : 1;
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>((a.c.kv_heads + per - 1) / per));
  auto kern = a.c.e4m3 ? (per == 2 ? kv_rows_kernel<T, true, kWrite, 2> : kv_rows_kernel<T, true, kWrite, 1>)
                       : (per == 2 ? kv_rows_kernel<T, false, kWrite, 2> : kv_rows_kernel<T, false, kWrite, 1>);
  kern<<<grid, kThreads, 0, st>>>(a, err);
  return cudaGetLastError();
}

template <bool kWrite>
cudaError_t launch_kv(const KvArgs& a, int dtype, int sms, int* err, cudaStream_t st) {
  if (dtype == kF32) return launch_rows<float, kWrite>(a, sms, err, st);
  if (dtype == kF16) return launch_rows<__half, kWrite>(a, sms, err, st);
  return launch_rows<__nv_bfloat16, kWrite>(a, sms, err, st);
}

}  // namespace

cudaError_t launch_kv_write(const KvCacheRef& c, int dtype, int64_t rows, const int32_t* offsets,
                            const int32_t* lens, const HeadsRef& k, const HeadsRef& v, int sms,
                            int* err, cudaStream_t st) {
  return launch_kv<true>(KvArgs{c, rows, offsets, lens, {k, v}}, dtype, sms, err, st);
}

cudaError_t launch_kv_read(const KvCacheRef& c, int dtype, int64_t rows, const int32_t* offsets,
                           const int32_t* first, const HeadsRef& k, const HeadsRef& v, int sms,
                           int* err, cudaStream_t st) {
  return launch_kv<false>(KvArgs{c, rows, offsets, first, {k, v}}, dtype, sms, err, st);
}

}  // namespace va
