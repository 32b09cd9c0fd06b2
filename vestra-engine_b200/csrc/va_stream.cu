// C-ABI layer of the streaming-attention operators: argument checks, the plan of the masked
// attention (host work list), and the launches.  The kernels are in va_rope_axes.cu,
// va_masked.cu, va_rows_attn.cu, va_kv_cache.cu and va_cache_attn.cu.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <new>
#include <vector>

#include "../../include/vestra_attn.h"
#include "va_internal.h"

struct va_attn_plan {
  int device = 0;
  va::AttnTerms terms{};
  int group = 1, tile_tokens = 1, splits = 1;
  int fewest_keys = 0x7fffffff;
  int most_rows = 0;  // query rows of the fullest tile
  int64_t q_rows = 0, k_rows = 0;  // rows the documents reach to
  std::vector<va::MaskedItem> items;
  va::MaskedItem* dev_items = nullptr;
  float* dev_slopes = nullptr;
};

namespace {

constexpr double kLog2e = 1.4426950408889634;
constexpr int64_t kMaxRows = 0x7fffffff;
constexpr int64_t kMaxCapacity = int64_t(1) << 30;  // chunk arithmetic stays in 32 bits
constexpr int64_t kMaxDocKeys = int64_t(1) << 24;  // frame indices stay exact in F32
constexpr float kMaxSlope = 0x1p96f;  // times log2(e) and 2^30 tokens: inside F32

// Makes the context's device current for one call and puts the caller's back.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    err_ = cudaGetDevice(&prev_);
    if (err_ == cudaSuccess && prev_ != device) {
      err_ = cudaSetDevice(device);
      changed_ = err_ == cudaSuccess;
    }
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(prev_);
  }
  cudaError_t error() const { return err_; }

 private:
  int prev_ = 0;
  bool changed_ = false;
  cudaError_t err_;
};

int launched(va_ctx* c, cudaError_t e, const char* what) {
  if (e == cudaSuccess) return VA_OK;
  char msg[160];
  std::snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
  return va::ctx_fail(c, VA_ERR_CUDA, msg);
}

int bad(va_ctx* c, const char* msg) { return va::ctx_fail(c, VA_ERR_INVALID, msg); }

int elem_size(int dtype) { return dtype == VA_F32 ? 4 : 2; }

// int32 and F32 arrays that kernels read (nullptr passes).
bool words_ok(std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (reinterpret_cast<uintptr_t>(p) % 4) return false;
  return true;
}

// No two elements of [rows][heads][head_dim] share an address: either the heads lie inside a
// token's stride or the tokens inside a head's.  A stride that is never stepped over may be anything.
bool strides_ok(const va_heads* h, int head_dim, int64_t rows) {
  constexpr int64_t kMost = int64_t(1) << 30, kMostHead = int64_t(1) << 38;
  if (h->heads < 1) return false;
  if (rows == 0) return true;
  if (rows == 1) return h->heads == 1 || (h->head_stride >= head_dim && h->head_stride <= kMostHead);
  if (h->token_stride < head_dim || h->token_stride > kMost) return false;
  if (h->heads == 1) return true;
  if (h->head_stride < head_dim || h->head_stride > kMostHead) return false;
  const bool token_major = h->head_stride <= kMost && h->token_stride >= (h->heads - 1) * h->head_stride + head_dim;
  const bool head_major = h->head_stride >= (rows - 1) * h->token_stride + head_dim;
  return token_major || head_major;
}

// 16-byte vectors: aligned data, strides in whole vectors.
bool vector_ok(const va_heads* h, int64_t rows) {
  const int per = 16 / elem_size(h->dtype);
  return reinterpret_cast<uintptr_t>(h->data) % 16 == 0 && (rows <= 1 || h->token_stride % per == 0) &&
         (rows == 0 || h->heads == 1 || h->head_stride % per == 0);
}

va::HeadsRef ref(const va_heads* h, int64_t rows) {
  if (!h) return va::HeadsRef{nullptr, 0, 0, 0};
  constexpr int64_t kNoStep = 64;  // for kernels and tensor maps: a legal stride
  return va::HeadsRef{h->data, rows > 1 ? h->token_stride : kNoStep, h->heads > 1 ? h->head_stride : 0, h->heads};
}

const char* check_terms(const va_attn_terms* t) {
  if (!t) return "attention terms are missing";
  if (t->heads < 1 || t->heads > 128 || t->kv_heads < 1 || t->heads % t->kv_heads)
    return "heads must be 1..128 and a multiple of kv_heads";
  if (t->frame < 1) return "frame must be at least 1 token";
  if (t->causal != 0 && t->causal != 1) return "causal must be 0 or 1";
  // The capped score's error grows with the cap (about 2e-7 of it); the tanh polynomial's factors
  // (scale / cap)^6 have to stay inside F32.
  if (!(t->scale >= 0.0f && t->scale <= 100.0f)) return "scale must be 0 (default) or at most 100";
  if (!(t->score_cap == 0.0f || (t->score_cap >= 0.01f && t->score_cap <= 1000.0f)))
    return "score_cap must be 0 (none) or 0.01..1000";
  return nullptr;
}

va::AttnTerms make_terms(const va_attn_terms* t) {
  va::AttnTerms a{};
  a.heads = t->heads;
  a.kv_heads = t->kv_heads;
  a.causal = t->causal;
  a.frame = t->frame;
  const double scale = t->scale > 0.0f ? t->scale : 0.125;
  a.scale_log2 = static_cast<float>(scale * kLog2e);
  a.cap_in = t->score_cap > 0.0f ? static_cast<float>(2.0 * kLog2e * scale / t->score_cap) : 0.0f;
  a.cap_out = t->score_cap > 0.0f ? static_cast<float>(t->score_cap * kLog2e) : 0.0f;
  if (t->score_cap > 0.0f) {
    // tanh(z) = z (c0 + c1 z^2 + ...) for |z| <= 0.3 and |z| <= 0.6 (fits: va_masked.cu), z = scale x / cap
    static const double kTanh[7] = {0.9999988388472373, -0.3331002159727106, 0.126339459668236, 0.9999978512525337,
                                    -0.3331403919023951, 0.13057855946359676, -0.040929422032535266};
    const double z = scale / t->score_cap;
    double k = scale * kLog2e;
    for (int i = 0; i < 4; ++i, k *= z * z) {
      if (i < 3) a.cap_poly[i] = static_cast<float>(kTanh[i] * k);
      a.cap_poly[3 + i] = static_cast<float>(kTanh[3 + i] * k);
    }
    a.cap_range[0] = static_cast<float>(std::min(0.3 * t->score_cap, 77.0) / scale);
    a.cap_range[1] = static_cast<float>(std::min(0.6 * t->score_cap, 77.0) / scale);
  }
  return a;
}

int64_t floor_div(int64_t a, int64_t b) { return a >= 0 ? a / b : -1 - (-1 - a) / b; }

// The work list of a layout (host only).  Returns nullptr or what is wrong with it.
const char* build_plan(const va_attn_terms* t, int documents, const int64_t* qo, const int64_t* ko,
                       const int64_t* prefix, int sms, va_attn_plan* p) {
  if (const char* m = check_terms(t)) return m;
  if (documents < 1 || !qo || !ko) return "a plan needs at least one document and both offset arrays";
  if (qo[0] < 0 || ko[0] < 0) return "offsets start below 0";
  p->terms = make_terms(t);
  p->group = t->heads / t->kv_heads;
  p->tile_tokens = 128 / p->group;
  p->q_rows = qo[documents];
  p->k_rows = ko[documents];
  if (p->q_rows > kMaxRows || p->k_rows > kMaxRows) return "offsets reach past 2^31 rows";
  // Everything is checked, the number of tiles too, before the list is built.
  int64_t tiles = 0;
  for (int b = 0; b < documents; ++b) {
    if (qo[b + 1] < qo[b] || ko[b + 1] < ko[b] || qo[b + 1] > kMaxRows || ko[b + 1] > kMaxRows) return "offsets must ascend";
    if (ko[b + 1] - ko[b] > kMaxDocKeys) return "a document has more than 2^24 keys";
    if (qo[b + 1] - qo[b] > kMaxDocKeys) return "a document has more than 2^24 query rows";
    if (prefix && prefix[b] < 0) return "prefix must not be negative";
    tiles += (qo[b + 1] - qo[b] + p->tile_tokens - 1) / p->tile_tokens;
  }
  if (tiles > kMaxRows / t->kv_heads / 16) return "too many query tiles";
  p->items.reserve(static_cast<size_t>(tiles));
  for (int b = 0; b < documents; ++b) {
    const int64_t lq = qo[b + 1] - qo[b], lk = ko[b + 1] - ko[b];
    const int64_t pre = prefix ? prefix[b] : 0;
    for (int64_t i = 0; i < lq; i += p->tile_tokens) {
      va::MaskedItem it{};
      it.q_row = static_cast<int>(qo[b] + i);
      it.tokens = static_cast<int>(std::min<int64_t>(p->tile_tokens, lq - i));
      it.k_row = static_cast<int>(ko[b]);
      it.first = static_cast<int>(i + lk - lq);
      it.doc_keys = static_cast<int>(lk);
      it.prefix = static_cast<int>(std::min(pre, lk));
      // Keys the row at a position sees; the tile's last row sees most, its first fewest.
      auto limit = [&](int64_t at) {
        if (!t->causal) return it.doc_keys;
        const int64_t e = (floor_div(at, t->frame) + 1) * t->frame;
        return static_cast<int>(std::max<int64_t>(0, std::min<int64_t>(lk, std::max<int64_t>(e, it.prefix))));
      };
      it.keys = limit(static_cast<int64_t>(it.first) + it.tokens - 1);
      p->fewest_keys = std::min(p->fewest_keys, limit(it.first));
      p->most_rows = std::max(p->most_rows, it.tokens * p->group);
      p->items.push_back(it);
    }
  }
  // Longest first, so the last CTAs to start are the short ones; equal ones in row order, so
  // the tiles that read the same keys run together.
  std::stable_sort(p->items.begin(), p->items.end(),
                   [](const va::MaskedItem& a, const va::MaskedItem& b) { return a.keys > b.keys; });
  if (p->items.empty()) return nullptr;
  if (va::rows_form(p->most_rows)) {
    p->splits = va::rows_splits(static_cast<int64_t>(p->items.size()) * t->kv_heads * ((p->most_rows + 7) / 8),
                                p->items[0].keys, sms);
    return nullptr;
  }
  std::vector<int> key_tiles(p->items.size());
  for (size_t i = 0; i < key_tiles.size(); ++i) key_tiles[i] = (p->items[i].keys + 127) / 128;
  p->splits = va::masked_splits(key_tiles.data(), tiles, t->kv_heads, sms);
  return nullptr;
}

void free_plan(va_attn_plan* p) {
  if (!p) return;
  if (p->dev_items || p->dev_slopes) {
    DeviceScope scope(p->device);
    cudaFree(p->dev_items);
    cudaFree(p->dev_slopes);
  }
  delete p;
}

// On the legacy stream; from pageable memory the copy may still be under way on return (finish_uploads).
template <class T>
cudaError_t upload(T** dst, const T* src, size_t n) {
  cudaError_t e = cudaMalloc(reinterpret_cast<void**>(dst), n * sizeof(T));
  if (e == cudaSuccess) e = cudaMemcpy(*dst, src, n * sizeof(T), cudaMemcpyHostToDevice);
  return e;
}

// Waits for the uploads: a plan's first launch may be on a stream that does not wait for the legacy one.
cudaError_t finish_uploads() { return cudaStreamSynchronize(cudaStreamLegacy); }

const char* check_cache(const va_kv_cache* c) {
  if (!c) return "the cache is missing";
  if (c->documents < 1 || c->kv_heads < 1 || c->kv_heads > 128 || c->capacity < 1 || c->capacity > kMaxCapacity)
    return "cache needs documents >= 1, kv_heads 1..128 and capacity 1..2^30";
  if (c->format != VA_KV_INT8 && c->format != VA_KV_E4M3) return "unknown cache format";
  if (c->reserved != 0) return "reserved must be 0";
  for (const void* p : {static_cast<const void*>(c->k_codes), static_cast<const void*>(c->v_codes),
                        static_cast<const void*>(c->k_scales), static_cast<const void*>(c->v_scales)})
    if (!p || reinterpret_cast<uintptr_t>(p) % 16) return "cache buffers must be given and 16-byte aligned";
  return nullptr;
}

va::KvCacheRef cache_ref(const va_kv_cache* c) {
  va::KvCacheRef r{};
  r.documents = c->documents;
  r.kv_heads = c->kv_heads;
  r.e4m3 = c->format == VA_KV_E4M3;
  r.capacity = c->capacity;
  r.codes[0] = static_cast<uint8_t*>(c->k_codes);
  r.codes[1] = static_cast<uint8_t*>(c->v_codes);
  r.scales[0] = c->k_scales;
  r.scales[1] = c->v_scales;
  return r;
}

int cache_rows_call(va_ctx* c, const va_kv_cache* cache, int64_t rows, const int32_t* offsets, const int32_t* edge,
                    const va_heads* k, const va_heads* v) {
  if (const char* m = check_cache(cache)) return bad(c, m);
  if (!offsets || !k || !v) return bad(c, "offsets, k and v must be given");
  if (!words_ok({offsets, edge})) return bad(c, "offsets, lens and first must be 4-byte aligned");
  if (rows < 0 || rows > kMaxRows) return bad(c, "rows must be 0..2^31 - 1");
  if (k->dtype < VA_BF16 || k->dtype > VA_F32 || v->dtype != k->dtype) return bad(c, "k and v must have one type");
  for (const va_heads* h : {k, v}) {
    if (h->heads != cache->kv_heads) return bad(c, "k and v need the cache's kv_heads");
    if (rows > 0 && !h->data) return bad(c, "k and v data must be given");
    if (!strides_ok(h, 64, rows)) return bad(c, "k or v strides overlap");
    if (!vector_ok(h, rows)) return bad(c, "k and v need 16-byte aligned data and strides");
  }
  return VA_OK;
}

}  // namespace

namespace va {
// The widest vectors that every block (min_half: the gcd of their halves), pointer and stride allows, at most 16
// bytes.
int rope_chunk(const RopeAxesArgs& a, int min_half, int elem_bytes) {
  const int per_pair = a.pairing ? 2 : 1;  // elements of one vector per pair
  for (int v = 16 / elem_bytes / per_pair; v >= 1; v >>= 1) {
    bool ok = min_half % v == 0;
    for (int w = 0; w < 2; ++w) {
      if (a.in[w].heads == 0) continue;
      for (const HeadsRef* h : {&a.in[w], &a.out[w]}) {
        const int e = v * per_pair;
        ok = ok && reinterpret_cast<uintptr_t>(h->data) % (elem_bytes * e) == 0 && h->token_stride % e == 0 &&
             h->head_stride % e == 0;
      }
    }
    if (ok) return v;
  }
  return 0;  // pairing 1 only: there one pair is a vector of two elements already
}

cudaError_t prepare_kernel(const void* kernel, int smem_bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (ready.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
  // clusters of up to 16 CTAs
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
  return e;
}
}  // namespace va

extern "C" {

int va_rope_axes_device(va_ctx* c, const va_rope_axes* rope, int64_t rows, int head_dim,
                        const int32_t* positions, const va_heads* q, const va_heads* q_out,
                        const va_heads* k, const va_heads* k_out, void* stream) {
  if (!c) return VA_ERR_INVALID;
  if (!rope || !q || !q_out || (k == nullptr) != (k_out == nullptr))
    return bad(c, "rope, q and q_out must be given, k and k_out together or not at all");
  if (rope->axes < 1 || rope->axes > 4) return bad(c, "rope needs 1 to 4 axes");
  if (rope->layout != VA_ROPE_PER_AXIS && rope->layout != VA_ROPE_SHARED) return bad(c, "unknown rope layout");
  if (rope->pairing != 0 && rope->pairing != 1) return bad(c, "rope pairing must be 0 or 1");
  if (!std::isfinite(rope->base) || rope->base <= 0.0f) return bad(c, "rope base must be positive");
  if (head_dim < 2 || head_dim > 256 || head_dim % 2) return bad(c, "head_dim must be even, 2..256");
  int total = 0;
  for (int a = 0; a < rope->axes; ++a) {
    if (rope->section[a] < 2 || rope->section[a] % 2 || rope->section[a] > head_dim)
      return bad(c, "every rope section must be even, 2..head_dim");
    total += rope->section[a];
  }
  if (total > head_dim) return bad(c, "the rope sections exceed head_dim");
  if (rows < 0 || rows > kMaxRows) return bad(c, "rows must be 0..2^31 - 1");
  const va_heads* in[2] = {q, k};
  const va_heads* out[2] = {q_out, k_out};
  va::RopeAxesArgs a{};
  for (int w = 0; w < 2; ++w) {
    if (!in[w]) continue;
    if (in[w]->dtype < VA_BF16 || in[w]->dtype > VA_F32 || in[w]->dtype != q->dtype || out[w]->dtype != q->dtype)
      return bad(c, "rope tensors must have one type");
    if (in[w]->heads != out[w]->heads || in[w]->heads > 1024) return bad(c, "an output needs its input's heads, at most 1024");
    if (!strides_ok(in[w], head_dim, rows) || !strides_ok(out[w], head_dim, rows)) return bad(c, "rope strides overlap");
    if (rows > 0 && (!in[w]->data || !out[w]->data)) return bad(c, "rope data must be given");
    for (const va_heads* h : {in[w], out[w]})
      if (reinterpret_cast<uintptr_t>(h->data) % elem_size(h->dtype)) return bad(c, "rope data is not aligned to its type");
    if (in[w]->data == out[w]->data &&
        ((rows > 1 && in[w]->token_stride != out[w]->token_stride) || (in[w]->heads > 1 && in[w]->head_stride != out[w]->head_stride)))
      return bad(c, "an output on its input needs the same strides");
    a.in[w] = ref(in[w], rows);
    a.out[w] = ref(out[w], rows);
  }
  if (rows == 0) return VA_OK;
  if (!positions) return bad(c, "positions must be given");
  if (!words_ok({positions})) return bad(c, "positions must be 4-byte aligned");
  const bool shared = rope->layout == VA_ROPE_SHARED;
  int start = 0, n = 0, g = 0;
  auto gcd = [](int x, int y) {
    while (y) {
      const int t = x % y;
      x = y;
      y = t;
    }
    return x;
  };
  for (int ax = 0; ax < rope->axes; ++ax) {
    const int s = rope->section[ax];
    const int block = shared ? total : s, origin = shared ? 0 : start;
    for (int i = 0; i < s / 2; ++i, ++n) {
      const int j = shared ? n : i;
      a.first[n] = static_cast<uint8_t>(origin + (rope->pairing ? 2 * j : j));
      a.second[n] = static_cast<uint8_t>(origin + (rope->pairing ? 2 * j + 1 : j + block / 2));
      a.axis[n] = static_cast<uint8_t>(ax);
      const double turns = std::pow(static_cast<double>(rope->base), -2.0 * j / block) / 6.283185307179586476925;
      // 2^64 times the fraction of a turn (a product of 53 bits: exact), wrapping at 2^64
      const double scaled = (turns - std::floor(turns)) * 18446744073709551616.0;
      a.turns[n] = scaled < 18446744073709551615.0 ? static_cast<uint64_t>(scaled) : 0;
    }
    g = gcd(g, block / 2);
    start += s;
  }
  a.pairs = n;
  a.axes = rope->axes;
  a.head_dim = head_dim;
  a.rotated = total;
  a.pairing = rope->pairing;
  a.chunk = va::rope_chunk(a, g, elem_size(q->dtype));
  a.rows = rows;
  a.positions = positions;
  const va::CtxCore core = va::ctx_core(c);
  DeviceScope scope(core.device);
  if (scope.error() != cudaSuccess) return launched(c, scope.error(), "rope device");
  return launched(c, va::launch_rope_axes(a, q->dtype, static_cast<cudaStream_t>(stream)), "rope launch");
}

int va_attn_plan_shape(const va_attn_terms* terms, int documents, const int64_t* q_offsets,
                       const int64_t* k_offsets, const int64_t* prefix, int sms, int64_t* plan) {
  if (!plan || sms < 1) return VA_ERR_INVALID;
  try {
    va_attn_plan p;
    if (build_plan(terms, documents, q_offsets, k_offsets, prefix, sms, &p)) return VA_ERR_INVALID;
    int64_t tiles = 0;
    for (const va::MaskedItem& it : p.items) tiles += (it.keys + 127) / 128;
    plan[0] = static_cast<int64_t>(p.items.size()) * terms->kv_heads;
    plan[1] = p.splits;
    plan[2] = p.tile_tokens;
    plan[3] = tiles * terms->kv_heads;
    plan[4] = plan[0] * p.splits * (va::rows_form(p.most_rows) ? (p.most_rows + 7) / 8 : 1);
    return VA_OK;
  } catch (...) {
    return VA_ERR_CAPACITY;
  }
}

int va_attn_plan_create(va_ctx* c, const va_attn_terms* terms, int documents, const int64_t* q_offsets,
                        const int64_t* k_offsets, const int64_t* prefix, const float* slopes,
                        va_attn_plan** out) {
  if (!c || !out) return VA_ERR_INVALID;
  *out = nullptr;
  va_attn_plan* p = nullptr;
  try {
    p = new va_attn_plan();
    const va::CtxCore core = va::ctx_core(c);
    p->device = core.device;
    const char* m = build_plan(terms, documents, q_offsets, k_offsets, prefix, core.sms, p);
    std::vector<float> s;
    if (!m && slopes) {
      for (int h = 0; h < terms->heads && !m; ++h) {
        if (!(std::fabs(slopes[h]) <= kMaxSlope)) m = "slopes must be finite, at most 2^96";
        s.push_back(static_cast<float>(slopes[h] * kLog2e));
      }
    }
    if (m) {
      free_plan(p);
      return bad(c, m);
    }
    DeviceScope scope(core.device);
    cudaError_t e = scope.error();
    if (e == cudaSuccess && !p->items.empty()) e = upload(&p->dev_items, p->items.data(), p->items.size());
    if (e == cudaSuccess && slopes) e = upload(&p->dev_slopes, s.data(), s.size());
    if (e == cudaSuccess) e = finish_uploads();
    if (e != cudaSuccess) {
      free_plan(p);
      return launched(c, e, "attention plan upload");
    }
    *out = p;
    return VA_OK;
  } catch (...) {
    free_plan(p);
    return va::ctx_fail(c, VA_ERR_CAPACITY, "out of host memory for the attention plan");
  }
}

void va_attn_plan_destroy(va_attn_plan* plan) { free_plan(plan); }

int va_masked_attention_device(va_ctx* c, const va_attn_plan* p, const va_heads* q, const va_heads* k,
                               const va_heads* v, const va_heads* out, void* stream) {
  if (!c) return VA_ERR_INVALID;
  if (!p || !q || !k || !v || !out) return bad(c, "plan, q, k, v and out must be given");
  const va::CtxCore core = va::ctx_core(c);
  if (core.device != p->device) return bad(c, "the plan belongs to another device");
  if (q->dtype != VA_BF16 && q->dtype != VA_F16) return bad(c, "masked attention takes BF16 or F16");
  if (p->items.empty()) return VA_OK;
  const struct {
    const va_heads* h;
    int heads;
    int64_t rows;
  } ops[4] = {{q, p->terms.heads, p->q_rows},
              {k, p->terms.kv_heads, p->k_rows},
              {v, p->terms.kv_heads, p->k_rows},
              {out, p->terms.heads, p->q_rows}};
  for (const auto& o : ops) {
    if (o.rows == 0) continue;  // no document has a key: k and v are not touched
    if (o.h->dtype != q->dtype) return bad(c, "q, k, v and out must have one type");
    if (o.h->heads != o.heads) return bad(c, "q and out need the plan's heads, k and v its kv_heads");
    if (!o.h->data) return bad(c, "q, k, v and out data must be given");
    if (!strides_ok(o.h, 64, o.rows)) return bad(c, "strides overlap");
    if (!vector_ok(o.h, o.rows)) return bad(c, "data must be 16-byte aligned, strides multiples of 8 elements");
  }
  va::MaskedArgs a{};
  a.t = p->terms;
  a.group = p->group;
  a.tile_tokens = p->tile_tokens;
  a.items = static_cast<int>(p->items.size());
  a.splits = p->splits;
  a.fewest_keys = p->fewest_keys;
  a.most_keys = p->items[0].keys;
  a.item = p->dev_items;
  a.slopes = p->dev_slopes;
  a.out = ref(out, p->q_rows);
  DeviceScope scope(core.device);
  if (scope.error() != cudaSuccess) return launched(c, scope.error(), "attention device");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (va::rows_form(p->most_rows))
    return launched(c, va::launch_rows(ref(q, p->q_rows), ref(k, p->k_rows), ref(v, p->k_rows), a, p->most_rows, q->dtype, st), "masked attention launch");
  return launched(c, va::launch_masked(ref(q, p->q_rows), ref(p->k_rows ? k : q, p->k_rows), ref(p->k_rows ? v : q, p->k_rows), p->q_rows,
                                       p->k_rows, a, q->dtype, core.err, st),
                  "masked attention launch");
}

int va_kv_cache_write_device(va_ctx* c, const va_kv_cache* cache, int64_t rows, const int32_t* offsets,
                             const int32_t* lens, const va_heads* k, const va_heads* v, void* stream) {
  if (!c) return VA_ERR_INVALID;
  const int rc = cache_rows_call(c, cache, rows, offsets, lens, k, v);
  if (rc) return rc;
  if (!lens) return bad(c, "lens must be given");
  const va::CtxCore core = va::ctx_core(c);
  DeviceScope scope(core.device);
  if (scope.error() != cudaSuccess) return launched(c, scope.error(), "cache device");
  return launched(c, va::launch_kv_write(cache_ref(cache), k->dtype, rows, offsets, lens, ref(k, rows), ref(v, rows), core.sms, core.err,
                                         static_cast<cudaStream_t>(stream)),
                  "cache write launch");
}

int va_kv_cache_read_device(va_ctx* c, const va_kv_cache* cache, int64_t rows, const int32_t* offsets,
                            const int32_t* first, const va_heads* k, const va_heads* v, void* stream) {
  if (!c) return VA_ERR_INVALID;
  const int rc = cache_rows_call(c, cache, rows, offsets, first, k, v);
  if (rc) return rc;
  const va::CtxCore core = va::ctx_core(c);
  DeviceScope scope(core.device);
  if (scope.error() != cudaSuccess) return launched(c, scope.error(), "cache device");
  return launched(c, va::launch_kv_read(cache_ref(cache), k->dtype, rows, offsets, first, ref(k, rows), ref(v, rows), core.sms, core.err,
                                        static_cast<cudaStream_t>(stream)),
                  "cache read launch");
}

int va_cache_attention_device(va_ctx* c, const va_kv_cache* cache, const va_attn_terms* terms, int64_t rows,
                              const int32_t* offsets, const int32_t* lens, int max_tokens, const int32_t* prefix,
                              const float* slopes, const va_heads* q, const va_heads* out, void* stream) {
  if (!c) return VA_ERR_INVALID;
  if (const char* m = check_cache(cache)) return bad(c, m);
  if (const char* m = check_terms(terms)) return bad(c, m);
  if (terms->kv_heads != cache->kv_heads) return bad(c, "terms and cache differ in kv_heads");
  if (!offsets || !lens || !q || !out) return bad(c, "offsets, lens, q and out must be given");
  if (!words_ok({offsets, lens, prefix, slopes})) return bad(c, "offsets, lens, prefix and slopes must be 4-byte aligned");
  if (rows < 0 || rows > kMaxRows / terms->heads) return bad(c, "rows * heads must be below 2^31");
  if (max_tokens < 1) return bad(c, "max_tokens must be at least 1");
  if (q->dtype != VA_BF16 && q->dtype != VA_F16) return bad(c, "cache attention takes BF16 or F16");
  for (const va_heads* h : {q, out}) {
    if (h->dtype != q->dtype) return bad(c, "q and out must have one type");
    if (h->heads != terms->heads) return bad(c, "q and out need the terms' heads");
    if (rows > 0 && !h->data) return bad(c, "q and out data must be given");
    if (!strides_ok(h, 64, rows)) return bad(c, "strides overlap");
    if (!vector_ok(h, rows)) return bad(c, "data must be 16-byte aligned, strides multiples of 8 elements");
  }
  if (rows == 0) return VA_OK;
  const va::CtxCore core = va::ctx_core(c);
  DeviceScope scope(core.device);
  if (scope.error() != cudaSuccess) return launched(c, scope.error(), "cache attention device");
  const int most = static_cast<int>(std::min<int64_t>(max_tokens, rows));
  return launched(c, va::launch_cache_attention(cache_ref(cache), make_terms(terms), q->dtype, rows, offsets, lens,
                                                most, prefix, slopes, ref(q, rows), ref(out, rows), core.sms, core.err,
                                                static_cast<cudaStream_t>(stream)),
                  "cache attention launch");
}

}  // extern "C"
