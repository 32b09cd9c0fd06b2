// Stand-in for the CUDA runtime and the kernels' launchers under va_stream.cu (argument checks and plans of
// the streaming operators), so that the C entry points run without a GPU.  Device memory is host memory.
// A copy from pageable memory is done when the stream is waited for, as the runtime allows it to be: until then
// the device holds what it held.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

#include "va_internal.h"

struct va_ctx {
  std::string error;
};

namespace {

struct Copy {
  char* dst;
  std::vector<char> data;
};
std::vector<Copy> pending;
int device = 0;

// What the launchers were given last.
struct Seen {
  int64_t launches, unfinished;  // launches, and copies that were not done at one of them
  int64_t items, most_keys;      // masked: work items, keys of the longest
  int64_t token_stride[2], head_stride[2];
  float slope[4];
  int64_t rope_chunk, rope_pairs;
  uint8_t rope_first[128], rope_second[128];
} seen;

void launched(const va::HeadsRef& a, const va::HeadsRef& b) {
  ++seen.launches;
  seen.unfinished += static_cast<int64_t>(pending.size());
  const va::HeadsRef* h[2] = {&a, &b};
  for (int i = 0; i < 2; ++i) {
    seen.token_stride[i] = h[i]->token_stride;
    seen.head_stride[i] = h[i]->head_stride;
  }
}

void finish_copies() {
  for (const Copy& c : pending) std::memcpy(c.dst, c.data.data(), c.data.size());
  pending.clear();
}

}  // namespace

extern "C" {

cudaError_t cudaGetDevice(int* d) { return *d = device, cudaSuccess; }
cudaError_t cudaSetDevice(int d) { return device = d, cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "fake"; }
cudaError_t cudaMalloc(void** p, size_t n) {
  *p = std::malloc(n);
  std::memset(*p, 0xee, n);
  return cudaSuccess;
}
cudaError_t cudaFree(void* p) { return std::free(p), cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* dst, const void* src, size_t n, cudaMemcpyKind, cudaStream_t) {
  const char* s = static_cast<const char*>(src);
  pending.push_back({static_cast<char*>(dst), std::vector<char>(s, s + n)});
  return cudaSuccess;
}
cudaError_t cudaMemcpy(void* dst, const void* src, size_t n, cudaMemcpyKind kind) {
  return cudaMemcpyAsync(dst, src, n, kind, nullptr);
}
cudaError_t cudaStreamSynchronize(cudaStream_t) { return finish_copies(), cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { return finish_copies(), cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }

void* fake_context() { return new va_ctx(); }
const char* fake_error(va_ctx* c) { return c->error.c_str(); }
int fake_pending() { return static_cast<int>(pending.size()); }
void fake_reset() {
  finish_copies();
  seen = Seen{};
}
const Seen* fake_seen() { return &seen; }

}  // extern "C"

namespace va {

CtxCore ctx_core(const va_ctx*) { return CtxCore{0, 148, nullptr}; }
int ctx_fail(va_ctx* c, int code, const char* msg) {
  c->error = msg;
  return code;
}
bool rows_form(int most_rows) { return most_rows <= 16; }
int rows_splits(int64_t, int, int) { return 1; }
int masked_splits(const int*, int64_t, int, int) { return 1; }
cudaError_t launch_rope_axes(const RopeAxesArgs& a, int, cudaStream_t) {
  launched(a.in[0], a.out[0]);
  seen.rope_chunk = a.chunk;
  seen.rope_pairs = a.pairs;
  std::memcpy(seen.rope_first, a.first, sizeof(a.first));
  std::memcpy(seen.rope_second, a.second, sizeof(a.second));
  return cudaSuccess;
}
cudaError_t launch_kv_write(const KvCacheRef&, int, int64_t, const int32_t*, const int32_t*, const HeadsRef& k,
                            const HeadsRef& v, int, int*, cudaStream_t) {
  launched(k, v);
  return cudaSuccess;
}
cudaError_t launch_kv_read(const KvCacheRef&, int, int64_t, const int32_t*, const int32_t*, const HeadsRef& k,
                           const HeadsRef& v, int, int*, cudaStream_t) {
  launched(k, v);
  return cudaSuccess;
}
cudaError_t launch_cache_attention(const KvCacheRef&, const AttnTerms&, int, int64_t, const int32_t*, const int32_t*,
                                   int, const int32_t*, const float*, const HeadsRef& q, const HeadsRef& out, int, int*,
                                   cudaStream_t) {
  launched(q, out);
  return cudaSuccess;
}
static void masked(const HeadsRef& q, const MaskedArgs& m) {
  launched(q, m.out);
  seen.items = m.items;
  seen.most_keys = m.item[0].keys;
  for (int h = 0; h < 4 && h < m.t.heads; ++h) seen.slope[h] = m.slopes ? m.slopes[h] : 0.0f;
}
cudaError_t launch_rows(const HeadsRef& q, const HeadsRef&, const HeadsRef&, const MaskedArgs& m, int, int, cudaStream_t) {
  masked(q, m);
  return cudaSuccess;
}
cudaError_t launch_masked(const HeadsRef& q, const HeadsRef&, const HeadsRef&, int64_t, int64_t, const MaskedArgs& m, int,
                          int*, cudaStream_t) {
  masked(q, m);
  return cudaSuccess;
}

}  // namespace va
