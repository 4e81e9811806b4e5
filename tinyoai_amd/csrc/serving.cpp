// C ABI of the operators around a layer's attention: rotary positions, the
// paged key-value cache, attention over its pages and of packed prompts.
#include <cmath>
#include <exception>
#include <map>
#include <memory>
#include <mutex>
#include <vector>

#include "attend.h"
#include "experts.h"
#include "stream_scratch.h"
#include "tinyoai_hip.h"

using namespace tinyoai;

struct tinyoai_rope {
  int device = 0, hd = 0, rot = 0, interleaved = 0;
  float magnitude = 1.f;
  double *frequencies = nullptr;
  hipStream_t stream = nullptr;
  ~tinyoai_rope() {
    if (frequencies) hipFree(frequencies);
    if (stream) hipStreamDestroy(stream);
  }
};

struct tinyoai_kv_pages {
  int device = 0, layers = 0;
  KVPagesDev d{};  // of layer 0
  void *mem = nullptr;
  int64_t plane = 0, scales = 0;  // bytes of a layer's K or V, and of its scales
  hipStream_t stream = nullptr;
  StreamScratch scratch;
  ~tinyoai_kv_pages() {
    if (mem) hipFree(mem);
    if (stream) hipStreamDestroy(stream);
  }
};

namespace {

bool plain_type(int32_t dtype) { return dtype == FMT_F32 || dtype == FMT_F16 || dtype == FMT_BF16; }

// `rows` rows of `heads` heads of a buffer (of none: null, as empty arrays are), ld values apart.
int check_heads(const char *what, int32_t dtype, const void *p, int64_t ld, int32_t heads, int32_t hd, int32_t rows) {
  if (!plain_type(dtype)) return fail(TINYOAI_EINVAL, "unsupported %s type %d", what, dtype);
  if (!p && rows) return fail(TINYOAI_EINVAL, "%s is null", what);
  if (ld < (int64_t)heads * hd)
    return fail(TINYOAI_EINVAL, "%s rows of %d heads of %d are %lld apart", what, heads, hd, (long long)ld);
  if (ld > kRowValues) return fail(TINYOAI_EINVAL, "%s rows are %lld apart, more than %lld", what, (long long)ld, (long long)kRowValues);
  if (reinterpret_cast<uintptr_t>(p) % mx_width(dtype)) return fail(TINYOAI_EINVAL, "%s is not aligned to its type", what);
  return TINYOAI_OK;
}

bool head_width(int32_t hd) { return hd > 0 && hd <= kHeadDim && hd % 8 == 0; }

// The angle of a pair for a step of one position.
int frequencies(const tinyoai_rope_config &c, std::vector<double> &f) {
  const double pi2 = 6.283185307179586;
  f.resize(c.rot / 2);
  double first = 0, last = 0;
  if (c.scaling == TINYOAI_ROPE_YARN) {
    auto pair = [&](double turns) { return c.rot * std::log(c.context / (pi2 * turns)) / (2 * std::log(c.theta)); };
    first = std::fmax(std::floor(pair(c.high)), 0.0);
    last = std::fmin(std::ceil(pair(c.low)), c.rot - 1.0);
  }
  for (int i = 0; i < c.rot / 2; i++) {
    const double w = std::pow(c.theta, -2.0 * i / c.rot);
    double keep = 1;  // how much of the unscaled angle stays
    if (c.scaling == TINYOAI_ROPE_LINEAR) keep = 0;
    if (c.scaling == TINYOAI_ROPE_BANDS)
      keep = std::fmin(std::fmax((c.context * w / pi2 - c.low) / (c.high - c.low), 0.0), 1.0);
    if (c.scaling == TINYOAI_ROPE_YARN)
      keep = 1 - std::fmin(std::fmax((i - first) / std::fmax(last - first, 0.001), 0.0), 1.0);
    f[i] = w * keep + w / c.factor * (1 - keep);
  }
  return TINYOAI_OK;
}

int check_rope(const tinyoai_rope_config &c) {
  if (!head_width(c.head_dim) || c.rot <= 0 || c.rot > c.head_dim || c.rot % 2)
    return fail(TINYOAI_EINVAL, "invalid rotation of %d values of a head of %d", c.rot, c.head_dim);
  if (c.layout != TINYOAI_ROPE_HALF && c.layout != TINYOAI_ROPE_INTERLEAVED)
    return fail(TINYOAI_EINVAL, "unsupported rotary layout %d", c.layout);
  if (!(c.theta > 1) || !std::isfinite(c.theta)) return fail(TINYOAI_EINVAL, "invalid rotary base %g", c.theta);
  if (c.scaling < TINYOAI_ROPE_NONE || c.scaling > TINYOAI_ROPE_YARN)
    return fail(TINYOAI_EINVAL, "unsupported rotary scaling %d", c.scaling);
  if (c.scaling == TINYOAI_ROPE_NONE) return TINYOAI_OK;
  if (!(c.factor >= 1) || !std::isfinite(c.factor)) return fail(TINYOAI_EINVAL, "invalid rotary factor %g", c.factor);
  if (c.scaling == TINYOAI_ROPE_LINEAR) return TINYOAI_OK;
  if (c.context <= 0 || !(c.low > 0) || !(c.high > c.low) || !std::isfinite(c.high))
    return fail(TINYOAI_EINVAL, "invalid rotary scaling between %g and %g of %d positions", c.low, c.high, c.context);
  return TINYOAI_OK;
}

// The pages of a layer.
KVPagesDev layer_pages(const tinyoai_kv_pages &c, int layer) {
  KVPagesDev d = c.d;
  d.k += layer * 2 * c.plane;
  d.v = d.k + c.plane;
  d.kd = d.nb ? reinterpret_cast<uint16_t *>(static_cast<uint8_t *>(c.mem) + c.layers * 2 * c.plane + layer * 2 * c.scales) : nullptr;
  d.vd = d.nb ? d.kd + c.scales / 2 : nullptr;
  return d;
}

int check_layer(const tinyoai_kv_pages *c, int32_t layer) {
  if (!c) return fail(TINYOAI_EINVAL, "the paged cache is closed");
  if (layer < 0 || layer >= c->layers) return fail(TINYOAI_EINVAL, "layer %d of %d", layer, c->layers);
  return check_device(c->device, "paged cache");
}

int kv_rows(tinyoai_kv_pages *c, int32_t layer, int32_t dtype, const void *k, int64_t ldk, const void *v, int64_t ldv,
            const int32_t *slots, int32_t n, void *stream, hipError_t (*launch)(const KVRowsArgs &, hipStream_t)) {
  if (!c) return fail(TINYOAI_EINVAL, "the paged cache is closed");
  if (int rc = check_heads("k", dtype, k, ldk, c->d.kv_heads, c->d.hd, n)) return rc;
  if (int rc = check_heads("v", dtype, v, ldv, c->d.kv_heads, c->d.hd, n)) return rc;
  if ((!slots && n) || n < 0) return fail(TINYOAI_EINVAL, "invalid slots of %d rows", n);
  if (int rc = check_layer(c, layer)) return rc;
  if (!n) return TINYOAI_OK;
  const KVRowsArgs a{layer_pages(*c, layer), dtype, const_cast<void *>(k), const_cast<void *>(v), ldk, ldv, slots, n};
  const hipError_t e = launch(a, stream ? (hipStream_t)stream : c->stream);
  return e == hipSuccess ? TINYOAI_OK : hip_fail(e, "paged cache rows");
}

// Scratch of the calls without a handle on the current device; kept until the
// process ends (no destructor, which might run after the runtime's).
StreamScratch &attention_scratch() {
  static std::mutex mu;
  static std::map<int, StreamScratch *> *scratch = new std::map<int, StreamScratch *>;
  int device = 0;
  (void)hipGetDevice(&device);
  std::lock_guard<std::mutex> lock(mu);
  StreamScratch *&s = (*scratch)[device];
  if (!s) s = new StreamScratch;
  return *s;
}

}  // namespace

extern "C" {

int tinyoai_rope_open(const tinyoai_rope_config *config, tinyoai_rope **out) try {
  if (!out) return fail(TINYOAI_EINVAL, "invalid rotary arguments");
  *out = nullptr;
  if (!config) return fail(TINYOAI_EINVAL, "invalid rotary arguments");
  if (int rc = check_rope(*config)) return rc;
  std::vector<double> f;
  frequencies(*config, f);
  auto r = std::make_unique<tinyoai_rope>();
  r->hd = config->head_dim;
  r->rot = config->rot;
  r->interleaved = config->layout == TINYOAI_ROPE_INTERLEAVED;
  if (config->scaling == TINYOAI_ROPE_YARN) r->magnitude = (float)(0.1 * std::log(config->factor) + 1);
  hipError_t e = hipGetDevice(&r->device);
  if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
  e = hipStreamCreateWithFlags(&r->stream, hipStreamNonBlocking);
  if (e != hipSuccess) return hip_fail(e, "hipStreamCreate");
  const size_t bytes = f.size() * sizeof(double);
  e = device_alloc(&r->frequencies, bytes);
  if (e != hipSuccess) return fail(TINYOAI_ENOMEM, "hipMalloc(%zu): %s", bytes, hipGetErrorString(e));
  e = hipMemcpyAsync(r->frequencies, f.data(), bytes, hipMemcpyHostToDevice, r->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(r->stream);
  if (e != hipSuccess) return hip_fail(e, "rotary frequencies");
  *out = r.release();
  return TINYOAI_OK;
} catch (const std::exception &e) {
  return fail(TINYOAI_ENOMEM, "rotary positions: %s", e.what());
}

int tinyoai_rope_device(tinyoai_rope *r, int32_t dtype, const void *x_dev, int64_t ldx, int32_t n, int32_t heads,
                        const int32_t *positions_dev, int32_t out_dtype, void *out_dev, int64_t ldo, void *stream) {
  if (!r) return fail(TINYOAI_EINVAL, "the rotary positions are closed");
  if (n < 0 || heads <= 0 || (int64_t)heads * r->hd > kRowValues)
    return fail(TINYOAI_EINVAL, "invalid rotation of %d rows of %d heads", n, heads);
  if (int rc = check_heads("x", dtype, x_dev, ldx, heads, r->hd, n)) return rc;
  if (int rc = check_heads("out", out_dtype, out_dev, ldo, heads, r->hd, n)) return rc;
  if (!positions_dev && n) return fail(TINYOAI_EINVAL, "positions are null");
  if (n && x_dev == out_dev && (dtype != out_dtype || ldx != ldo))
    return fail(TINYOAI_EINVAL, "rows turned in place keep their type and distance");
  if (int rc = check_device(r->device, "rotary positions")) return rc;
  if (!n) return TINYOAI_OK;
  const hipError_t e = launch_rope(RopeArgs{r->frequencies, r->magnitude, r->hd, r->rot, r->interleaved, dtype, out_dtype, x_dev,
                                            ldx, n, heads, positions_dev, out_dev, ldo},
                                   stream ? (hipStream_t)stream : r->stream);
  return e == hipSuccess ? TINYOAI_OK : hip_fail(e, "rotary positions");
}

int tinyoai_rope_close(tinyoai_rope *r) {
  if (r) {
    hipStreamSynchronize(r->stream);
    delete r;
  }
  return TINYOAI_OK;
}

int tinyoai_kv_pages_open(int32_t type, int32_t layers, int32_t kv_heads, int32_t head_dim, int32_t page, int32_t pages,
                          tinyoai_kv_pages **out) try {
  if (!out) return fail(TINYOAI_EINVAL, "invalid paged cache arguments");
  *out = nullptr;
  if (!plain_type(type) && type != FMT_Q8_0) return fail(TINYOAI_EINVAL, "unsupported paged cache type %d", type);
  if (!head_width(head_dim) || kv_heads <= 0 || (int64_t)kv_heads * head_dim > kRowValues || layers <= 0)
    return fail(TINYOAI_EINVAL, "invalid paged cache of %d layers of %d heads of %d", layers, kv_heads, head_dim);
  if (page <= 0 || page > kPage || page & (page - 1) || pages <= 0 || (int64_t)page * pages > kPositions)
    return fail(TINYOAI_EINVAL, "invalid paged cache of %d pages of %d positions", pages, page);
  auto c = std::make_unique<tinyoai_kv_pages>();
  c->layers = layers;
  c->d.type = type;
  c->d.kv_heads = kv_heads;
  c->d.hd = head_dim;
  c->d.pages = pages;
  while (1 << c->d.page_log2 < page) c->d.page_log2++;
  c->d.pitch = type == FMT_Q8_0 ? (head_dim + 15) / 16 * 16 : head_dim * (int)mx_width(type);
  if (type == FMT_Q8_0)
    for (c->d.nb = 2; c->d.nb * 32 < head_dim; c->d.nb *= 2) {}
  const int64_t rows = (int64_t)pages * page * kv_heads;  // at most 2^54
  c->plane = rows * c->d.pitch;
  c->scales = (rows * c->d.nb * 2 + 255) / 256 * 256;
  c->plane = (c->plane + 255) / 256 * 256;
  const double bytes = 2.0 * layers * ((double)c->plane + (double)c->scales);
  if (bytes > 1e15) return fail(TINYOAI_ENOMEM, "paged cache of %.3g bytes", bytes);
  const size_t total = (size_t)layers * 2 * (size_t)(c->plane + c->scales) + 256;  // (zeros last)
  hipError_t e = hipGetDevice(&c->device);
  if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
  e = hipStreamCreateWithFlags(&c->stream, hipStreamNonBlocking);
  if (e != hipSuccess) return hip_fail(e, "hipStreamCreate");
  e = device_alloc(&c->mem, total);
  if (e != hipSuccess) return fail(TINYOAI_ENOMEM, "hipMalloc(%zu): %s", total, hipGetErrorString(e));
  c->d.k = static_cast<uint8_t *>(c->mem);
  c->d.zeros = c->d.k + (total - 256);
  e = hipMemsetAsync(c->mem, 0, total, c->stream);  // what no call has written reads as zeros
  if (e == hipSuccess) e = hipStreamSynchronize(c->stream);
  if (e != hipSuccess) return hip_fail(e, "paged cache");
  *out = c.release();
  return TINYOAI_OK;
} catch (const std::exception &e) {
  return fail(TINYOAI_ENOMEM, "paged cache: %s", e.what());
}

int tinyoai_kv_pages_write_device(tinyoai_kv_pages *c, int32_t layer, int32_t dtype, const void *k_dev, int64_t ldk,
                                  const void *v_dev, int64_t ldv, const int32_t *slots_dev, int32_t n, void *stream) {
  return kv_rows(c, layer, dtype, k_dev, ldk, v_dev, ldv, slots_dev, n, stream, launch_kv_write);
}

int tinyoai_kv_pages_read_device(tinyoai_kv_pages *c, int32_t layer, int32_t dtype, void *k_dev, int64_t ldk, void *v_dev,
                                 int64_t ldv, const int32_t *slots_dev, int32_t n, void *stream) {
  return kv_rows(c, layer, dtype, k_dev, ldk, v_dev, ldv, slots_dev, n, stream, launch_kv_read);
}

int tinyoai_kv_pages_attend_device(tinyoai_kv_pages *c, int32_t layer, int32_t dtype, const void *q_dev, int64_t ldq,
                                   int32_t heads, float scale, const int32_t *table_dev, int32_t width,
                                   const int32_t *lengths_dev, int32_t n, void *out_dev, int64_t ldo, void *stream) try {
  if (!c) return fail(TINYOAI_EINVAL, "the paged cache is closed");
  if (heads <= 0 || heads % c->d.kv_heads || (int64_t)heads * c->d.hd > kRowValues)
    return fail(TINYOAI_EINVAL, "%d query heads over %d key heads", heads, c->d.kv_heads);
  if (int rc = check_heads("q", dtype, q_dev, ldq, heads, c->d.hd, n)) return rc;
  if (int rc = check_heads("out", dtype, out_dev, ldo, heads, c->d.hd, n)) return rc;
  if (!std::isfinite(scale)) return fail(TINYOAI_EINVAL, "invalid scale %g", scale);
  if (n < 0 || width < 0 || ((!table_dev || !lengths_dev || !width) && n) || ((int64_t)width << c->d.page_log2) > kPositions)
    return fail(TINYOAI_EINVAL, "invalid page table of %d rows of %d", n, width);
  if ((int64_t)n * heads > kAttendRows) return fail(TINYOAI_EINVAL, "%d rows of %d heads exceed what one call takes", n, heads);
  if (int rc = check_layer(c, layer)) return rc;
  if (!n) return TINYOAI_OK;
  const AttendArgs a{layer_pages(*c, layer), dtype, q_dev, ldq, heads, scale, table_dev, width, lengths_dev, n, out_dev, ldo};
  hipStream_t st = stream ? (hipStream_t)stream : c->stream;
  return c->scratch.run(st, attend_scratch(a), [&](void *scratch) { return launch_attend(a, scratch, st); });
} catch (const std::exception &e) {
  return fail(TINYOAI_ENOMEM, "attention: %s", e.what());
}

int tinyoai_kv_pages_close(tinyoai_kv_pages *c) {
  if (c) {
    hipStreamSynchronize(c->stream);
    delete c;
  }
  return TINYOAI_OK;
}

int tinyoai_attention_device(int32_t dtype, const void *q_dev, int64_t ldq, int32_t heads, const void *k_dev, int64_t ldk,
                             const void *v_dev, int64_t ldv, int32_t kv_heads, int32_t head_dim, float scale, int32_t causal,
                             const int32_t *q_offsets_dev, const int32_t *k_offsets_dev, int32_t sequences, int32_t nq,
                             int32_t nk, void *out_dev, int64_t ldo, void *stream) try {
  if (!head_width(head_dim)) return fail(TINYOAI_EINVAL, "unsupported head width %d", head_dim);
  if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || (int64_t)heads * head_dim > kRowValues)
    return fail(TINYOAI_EINVAL, "%d query heads over %d key heads", heads, kv_heads);
  if (int rc = check_heads("q", dtype, q_dev, ldq, heads, head_dim, nq)) return rc;
  if (int rc = check_heads("k", dtype, k_dev, ldk, kv_heads, head_dim, nq ? nk : 0)) return rc;
  if (int rc = check_heads("v", dtype, v_dev, ldv, kv_heads, head_dim, nq ? nk : 0)) return rc;
  if (int rc = check_heads("out", dtype, out_dev, ldo, heads, head_dim, nq)) return rc;
  if (!std::isfinite(scale)) return fail(TINYOAI_EINVAL, "invalid scale %g", scale);
  if (((!q_offsets_dev || !k_offsets_dev || !sequences) && nq) || sequences < 0 || nq < 0 || nk < 0 || nq > kPositions || nk > kPositions)
    return fail(TINYOAI_EINVAL, "invalid offsets of %d sequences of %d queries and %d keys", sequences, nq, nk);
  if (((int64_t)nq / 128 + std::min(sequences, nq)) * heads >= 1 << 24)
    return fail(TINYOAI_EINVAL, "%d queries of %d sequences by %d heads exceed what one call takes", nq, sequences, heads);
  if (!nq) return TINYOAI_OK;
  const PromptArgs a{dtype, q_dev, k_dev, v_dev, ldq, ldk, ldv, heads, kv_heads, head_dim, scale, causal, q_offsets_dev,
                     k_offsets_dev, sequences, nq, nk, out_dev, ldo};
  const size_t bytes = prompt_scratch(a);
  hipStream_t st = (hipStream_t)stream;
  if (bytes) return attention_scratch().run(st, bytes, [&](void *scratch) { return launch_prompt(a, scratch, st); });
  const hipError_t e = launch_prompt(a, nullptr, st);
  return e == hipSuccess ? TINYOAI_OK : hip_fail(e, "attention");
} catch (const std::exception &e) {
  return fail(TINYOAI_ENOMEM, "attention: %s", e.what());
}

}  // extern "C"
