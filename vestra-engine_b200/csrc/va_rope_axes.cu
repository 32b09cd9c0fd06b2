// Rotary positions over several axes (time, height, width), on q and k in one launch.
//
//   (x0, x1) -> (x0 cos a - x1 sin a, x1 cos a + x0 sin a),  a = position[axis] * freq
//
// One pass: every element is read once and written once, so the kernel is bound by HBM
// (or, for a handful of tokens, by the launch).  A thread owns one (head, chunk) of a few
// consecutive token rows, a chunk being V pairs held in one or two vectors of up to 16
// bytes: it issues all its rows' loads, then the block tabulates the rows' (cos, sin) per
// pair in shared memory, once for all heads of q and k (a 32-pair row is shared by 12 + 12
// heads, so the trigonometry is 4 % of the pairs and hides behind the loads), then the
// thread turns its chunks and writes them.  No index is divided inside the row loop.
// Measured on B200: 10,392 bf16 tokens of 12 + 12 heads 13.5 us out of L2, 16.8 from HBM (3.8 TB/s); 27,729 F32
// tokens of 16 + 4 heads 49.4 us (5.8 TB/s = 0.88 of measured); two tokens 2.7 us.
//
// Angles: a position may be any int32 and the product with the frequency is needed
// modulo one turn, which F32 loses beyond a few thousand turns.  The frequency in turns is
// held as a 64-bit binary fraction, so the product modulo 2^64 is the exact fraction of a
// turn in integer arithmetic (64-bit floating point made the table the block's longest
// chain); its upper 32 bits are the reduced angle, a signed fraction of a turn.
#include "va_internal.h"
#include "va_ptx.cuh"

namespace va {

namespace {

constexpr int kMaxThreads = 256;
// Rows per block: two where a row's chunk is two 16-byte vectors of 2-byte elements, else four.  Measured
// at 10,392 bf16 rows of 24 heads, inputs out of L2, for 2 / 4 / 8 rows: sections 16,24,24 (8-byte
// vectors) 18.9 / 16.7 / 23.5 us, sections 32,32 15.8 / 18.8 / 22.4, F32 (27,729 rows of 20 heads) 62.4 / 49.4 / 48.2.
template <class T, int V, bool kInter>
constexpr int rows_per_block() { return sizeof(T) == 2 && V == 8 && !kInter ? 2 : 4; }

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

template <class T, int N, bool kAligned = true>
struct alignas(kAligned ? sizeof(T) * N : sizeof(T)) Vec {
  T v[N];
};

// (cos, sin) of position * turns (2^-64 turns a unit).  For 16-bit elements sin.approx and cos.approx on
// [-pi, pi] (absolute error below 2^-21); for F32 sincospi of the F32 part of the angle, the rest put
// back by one first-order step.
template <class T>
__device__ __forceinline__ float2 turn_cos_sin(int position, uint64_t turns) {
  const int t = static_cast<int>((static_cast<uint64_t>(static_cast<int64_t>(position)) * turns) >> 32);
  float s, c;
  if constexpr (sizeof(T) == 2) {
    __sincosf(static_cast<float>(t) * 1.4629180792671596e-9f, &s, &c);  // 2 pi / 2^32
    return make_float2(c, s);
  } else {
    const float hi = static_cast<float>(t);
    // hi may be 2^31, which no int holds: the difference is taken in 64 bits
    const float lo = static_cast<float>(static_cast<int>(t - static_cast<int64_t>(hi))) * 1.4629180792671596e-9f;
    sincospif(hi * 4.656612873077393e-10f, &s, &c);  // 2^-31
    return make_float2(fmaf(-s, lo, c), fmaf(c, lo, s));
  }
}

// V pairs per chunk; kInter: pairs are neighbours (2i, 2i+1), one vector of 2V elements, or, where that is not
// aligned (kAligned false, V = 1), two loads of an element; otherwise two vectors of V elements.
template <class T, int V, bool kInter, bool kAligned>
__global__ void __launch_bounds__(kMaxThreads) rope_axes_kernel(const __grid_constant__ RopeAxesArgs a) {
  constexpr int kRows = rows_per_block<T, V, kInter>();
  extern __shared__ float4 table[];  // cosines [kRows][pairs], then sines: a chunk's are one vector each
  float* cosines = reinterpret_cast<float*>(table);
  float* sines = cosines + kRows * a.pairs;
  using Part = Vec<T, kInter ? 2 * V : V, kAligned>;
  constexpr int kVecs = kInter ? 1 : 2;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kRows), a.rows - row0));
  const int chunks = a.pairs / V;
  const int item = blockIdx.y * blockDim.x + threadIdx.x;
  const bool active = item < (a.in[0].heads + a.in[1].heads) * chunks;
  int h = active ? item / chunks : 0;
  const int pair = active ? (item - h * chunks) * V : 0;
  const int which = h >= a.in[0].heads;
  if (which) h -= a.in[0].heads;
  const int ch[2] = {a.first[pair], a.second[pair]};
  Part x[kRows][kVecs];
  if (active) {
    const T* src = static_cast<const T*>(a.in[which].data) + row0 * a.in[which].token_stride + h * a.in[which].head_stride;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (r < rows) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
          x[r][i] = *reinterpret_cast<const Part*>(src + r * a.in[which].token_stride + ch[i]);
      }
  }
  for (int i = threadIdx.x; i < rows * a.pairs; i += blockDim.x) {
    const int r = i / a.pairs, p = i - r * a.pairs;
    const int pos = __ldg(a.positions + (row0 + r) * a.axes + a.axis[p]);
    const float2 w = turn_cos_sin<T>(pos, a.turns[p]);
    cosines[i] = w.x;
    sines[i] = w.y;
  }
  __syncthreads();
  if (active) {
    T* dst = static_cast<T*>(a.out[which].data) + row0 * a.out[which].token_stride + h * a.out[which].head_stride;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r < rows) {
        constexpr int kWide = V < 4 ? V : 4;
        using Wide = Vec<float, kWide>;
        const Wide* tc = reinterpret_cast<const Wide*>(cosines + r * a.pairs + pair);
        const Wide* ts = reinterpret_cast<const Wide*>(sines + r * a.pairs + pair);
        Wide wc, ws;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (e % kWide == 0) wc = tc[e / kWide], ws = ts[e / kWide];
          const float2 w = make_float2(wc.v[e % kWide], ws.v[e % kWide]);
          T& lo = x[r][0].v[kInter ? 2 * e : e];
          T& hi = kInter ? x[r][0].v[2 * e + 1] : x[r][kVecs - 1].v[e];
          const float p0 = to_f32(lo), p1 = to_f32(hi);
          lo = from_f32<T>(p0 * w.x - p1 * w.y);
          hi = from_f32<T>(p1 * w.x + p0 * w.y);
        }
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
          *reinterpret_cast<Part*>(dst + r * a.out[which].token_stride + ch[i]) = x[r][i];
      }
    }
  }

  // Channels past the sections pass through (nothing to do in place).
  const int rest = a.head_dim - a.rotated;
  if (rest == 0 || blockIdx.y != 0) return;
  const int heads = a.in[0].heads + a.in[1].heads;
  for (int i = threadIdx.x; i < rows * heads * rest; i += blockDim.x) {
    const int rh = i / rest, c = a.rotated + (i - rh * rest);
    const int r = rh / heads;
    int hh = rh - r * heads;
    const int w = hh >= a.in[0].heads;
    if (w) hh -= a.in[0].heads;
    const HeadsRef& in = a.in[w];
    const HeadsRef& out = a.out[w];
    if (in.data == out.data) continue;
    static_cast<T*>(out.data)[(row0 + r) * out.token_stride + hh * out.head_stride + c] =
        static_cast<const T*>(in.data)[(row0 + r) * in.token_stride + hh * in.head_stride + c];
  }
}

template <class T, int V, bool kInter, bool kAligned = true>
cudaError_t launch(const RopeAxesArgs& a, cudaStream_t st) {
  constexpr int rows = rows_per_block<T, V, kInter>();
  const int64_t blocks = (a.rows + rows - 1) / rows;
  const int items = (a.in[0].heads + a.in[1].heads) * (a.pairs / V);
  // As few threads past the items as the warp size allows.
  const int parts = (items + kMaxThreads - 1) / kMaxThreads;
  const int threads = ((items + parts - 1) / parts + 31) / 32 * 32;
  if (blocks > 0x7fffffff || parts > 65535) return cudaErrorInvalidValue;
  const size_t smem = 2 * sizeof(float) * rows * a.pairs;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(parts));
  rope_axes_kernel<T, V, kInter, kAligned><<<grid, threads, smem, st>>>(a);
  return cudaGetLastError();
}

template <class T>
cudaError_t launch_t(const RopeAxesArgs& a, cudaStream_t st) {
  if (a.pairing) {
    switch (a.chunk) {
      case 4:
        if constexpr (sizeof(T) == 2) return launch<T, 4, true>(a, st);
        break;
      case 2:
        return launch<T, 2, true>(a, st);
      case 1:
        return launch<T, 1, true>(a, st);
      case 0:
        return launch<T, 1, true, false>(a, st);
    }
  } else {
    switch (a.chunk) {
      case 8:
        if constexpr (sizeof(T) == 2) return launch<T, 8, false>(a, st);
        break;
      case 4:
        return launch<T, 4, false>(a, st);
      case 2:
        return launch<T, 2, false>(a, st);
      case 1:
        return launch<T, 1, false>(a, st);
    }
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_rope_axes(const RopeAxesArgs& a, int dtype, cudaStream_t st) {
  if (a.rows == 0 || a.in[0].heads + a.in[1].heads == 0) return cudaSuccess;
  if (dtype == kF32) return launch_t<float>(a, st);
  if (dtype == kF16) return launch_t<__half>(a, st);
  return launch_t<__nv_bfloat16>(a, st);
}

}  // namespace va
