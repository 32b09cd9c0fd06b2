// Rotary positions over several axes (time, height, width), on q and k in one launch.
//
//   (x0, x1) -> (x0 cos a - x1 sin a, x1 cos a + x0 sin a),  a = position[axis] * freq
//
// One pass: every element is read once and written once, so the kernel is bound by HBM
// (or, for a handful of tokens, by the launch).  A block takes kRows token rows.  It
// first tabulates the rows' (cos, sin) per pair in shared memory, once for all heads of
// q and k (a 32-pair row is shared by 12 + 12 heads, so the trigonometry is 4 % of the
// pairs), then its threads walk (row, head, chunk) items: a chunk is V pairs, read and
// written as one or two vectors of up to 16 bytes.
//
// Angles: a position may be any int32 and the product with the frequency is needed
// modulo one turn, which F32 loses beyond a few thousand turns.  The frequency in turns
// is held in 64 bits, the product is formed and reduced to [-1/2, 1/2] in 64 bits, and
// the reduced angle goes to sincospi in F32 with the F32 rounding of the angle put back
// by one first-order step.
#include "va_internal.h"
#include "va_ptx.cuh"

namespace va {

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 4;
constexpr int kBatch = 4;  // items a thread has in flight

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// (cos, sin) of 2 pi t for t in turns, |t| <= 1/2 after the reduction.
__device__ __forceinline__ float2 turn_cos_sin(double t) {
  t -= rint(t);
  const float hi = static_cast<float>(t);
  const float lo = static_cast<float>(t - static_cast<double>(hi)) * 6.283185307179586f;
  float s, c;
  sincospif(2.0f * hi, &s, &c);
  return make_float2(fmaf(-s, lo, c), fmaf(c, lo, s));
}

// V pairs per chunk; kInter: pairs are neighbours (2i, 2i+1), one vector of 2V elements;
// otherwise two vectors of V elements, min_half a multiple of V.
template <class T, int V, bool kInter>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ RopeAxesArgs a) {
  extern __shared__ float2 cs[];  // [kRows][pairs]
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kRows), a.rows - row0));
  for (int i = threadIdx.x; i < rows * a.pairs; i += kThreads) {
    const int r = i / a.pairs, p = i - r * a.pairs;
    const int pos = __ldg(a.positions + (row0 + r) * a.axes + a.axis[p]);
    cs[i] = turn_cos_sin(static_cast<double>(pos) * a.turns[p]);
  }
  __syncthreads();

  const int chunks = a.pairs / V;
  const int heads = a.in[0].heads + a.in[1].heads;
  const int items = rows * heads * chunks;
  using Part = Vec<T, kInter ? 2 * V : V>;
  for (int i0 = threadIdx.x; i0 < items; i0 += kThreads * kBatch) {
    Part x0[kBatch], x1[kBatch];
    T* dst[kBatch];
    int pair[kBatch], row[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kThreads;
      if (i < items) {
        const int rh = i / chunks;
        row[b] = rh / heads;
        int h = rh - row[b] * heads;
        pair[b] = (i - rh * chunks) * V;
        const int which = h >= a.in[0].heads;
        if (which) h -= a.in[0].heads;
        const HeadsRef& in = a.in[which];
        const HeadsRef& out = a.out[which];
        const T* src = static_cast<const T*>(in.data) + (row0 + row[b]) * in.token_stride + h * in.head_stride;
        dst[b] = static_cast<T*>(out.data) + (row0 + row[b]) * out.token_stride + h * out.head_stride;
        x0[b] = *reinterpret_cast<const Part*>(src + a.first[pair[b]]);
        if (!kInter) x1[b] = *reinterpret_cast<const Part*>(src + a.second[pair[b]]);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kThreads;
      if (i < items) {
        const float2* t = cs + row[b] * a.pairs + pair[b];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 w = t[e];
          T& lo = kInter ? x0[b].v[(2 * e) % (kInter ? 2 * V : V)] : x0[b].v[e % (kInter ? 2 * V : V)];
          T& hi = kInter ? x0[b].v[(2 * e + 1) % (kInter ? 2 * V : V)] : x1[b].v[e % (kInter ? 2 * V : V)];
          const float p0 = to_f32(lo), p1 = to_f32(hi);
          lo = from_f32<T>(p0 * w.x - p1 * w.y);
          hi = from_f32<T>(p1 * w.x + p0 * w.y);
        }
        *reinterpret_cast<Part*>(dst[b] + a.first[pair[b]]) = x0[b];
        if (!kInter) *reinterpret_cast<Part*>(dst[b] + a.second[pair[b]]) = x1[b];
      }
    }
  }

  // Channels past the sections pass through (nothing to do in place).
  const int rest = a.head_dim - a.rotated;
  if (rest == 0) return;
  for (int i = threadIdx.x; i < rows * heads * rest; i += kThreads) {
    const int rh = i / rest, c = a.rotated + (i - rh * rest);
    const int r = rh / heads;
    int h = rh - r * heads;
    const int which = h >= a.in[0].heads;
    if (which) h -= a.in[0].heads;
    const HeadsRef& in = a.in[which];
    const HeadsRef& out = a.out[which];
    if (in.data == out.data) continue;
    static_cast<T*>(out.data)[(row0 + r) * out.token_stride + h * out.head_stride + c] =
        static_cast<const T*>(in.data)[(row0 + r) * in.token_stride + h * in.head_stride + c];
  }
}

template <class T, int V>
cudaError_t launch_v(const RopeAxesArgs& a, cudaStream_t st) {
  const int64_t blocks = (a.rows + kRows - 1) / kRows;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  const size_t smem = sizeof(float2) * kRows * a.pairs;
  if (a.pairing)
    rope_axes_kernel<T, V, true><<<static_cast<unsigned>(blocks), kThreads, smem, st>>>(a);
  else
    rope_axes_kernel<T, V, false><<<static_cast<unsigned>(blocks), kThreads, smem, st>>>(a);
  return cudaGetLastError();
}

// The widest chunk (in pairs) that every block, pointer and stride allows, at most
// 16 bytes a vector.
template <class T>
cudaError_t launch_t(const RopeAxesArgs& a, cudaStream_t st) {
  const int per_pair = a.pairing ? 2 : 1;  // elements of one vector per pair
  int v = 16 / static_cast<int>(sizeof(T)) / per_pair;
  for (; v > 1; v >>= 1) {
    bool ok = a.min_half % v == 0;
    for (int w = 0; w < 2; ++w) {
      if (a.in[w].heads == 0) continue;
      for (const HeadsRef* h : {&a.in[w], &a.out[w]}) {
        const int e = v * per_pair;
        ok = ok && reinterpret_cast<uintptr_t>(h->data) % (sizeof(T) * e) == 0 && h->token_stride % e == 0 &&
             h->head_stride % e == 0;
      }
    }
    if (ok) break;
  }
  switch (v) {
    case 8:
      if constexpr (sizeof(T) == 2) return launch_v<T, 8>(a, st);
    case 4:
      return launch_v<T, 4>(a, st);
    case 2:
      return launch_v<T, 2>(a, st);
    default:
      return launch_v<T, 1>(a, st);
  }
}

}  // namespace

cudaError_t launch_rope_axes(const RopeAxesArgs& a, int dtype, cudaStream_t st) {
  if (a.rows == 0 || a.in[0].heads + a.in[1].heads == 0) return cudaSuccess;
  if (dtype == kF32) return launch_t<float>(a, st);
  if (dtype == kF16) return launch_t<__half>(a, st);
  return launch_t<__nv_bfloat16>(a, st);
}

}  // namespace va
