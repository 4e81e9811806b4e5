// C ABI of the mixture-of-experts operators: MXFP4 rows, expert routing,
// products grouped by expert and the weighted sum of the experts' rows.
#include "experts.h"

#include <algorithm>
#include <atomic>
#include <climits>
#include <exception>
#include <memory>
#include <vector>

#include "stream_scratch.h"
#include "tinyoai_hip.h"

// ---------------------------------------------------------------- products
bool mx_supported(const MxProduct &p) { return mx_few_supported(p) || mx_tiles_supported(p); }

size_t mx_scratch(const MxProduct &p) { return mx_few_supported(p) ? 0 : mx_tiles_scratch(p); }

hipError_t launch_mx_product(const MxProduct &p, void *scratch, hipStream_t st) {
  const hipError_t e = mx_few_supported(p) ? launch_mx_few(p, st) : launch_mx_tiles(p, scratch, st);
  if (e != hipSuccess || !p.w.infinite_rows || (p.xdtype != FMT_F32 && p.xdtype != FMT_F16)) return e;
  return launch_mx_infinite_rows(p, st);
}

namespace tinyoai {

// ---------------------------------------------------------------- scratch
namespace {
// Allowing this thread's allocations while a stream is captured.
struct RelaxedCapture {
  hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
  bool set = hipThreadExchangeStreamCaptureMode(&mode) == hipSuccess;
  ~RelaxedCapture() {
    if (set) hipThreadExchangeStreamCaptureMode(&mode);
  }
};
class ThreadEnd {
 public:
  ThreadStream add(int device) {
    if (!life_) life_ = std::make_shared<char>(0);
    if (std::find(devices_.begin(), devices_.end(), device) == devices_.end()) devices_.push_back(device);
    return ThreadStream{number_, life_};
  }
  ~ThreadEnd() {
    RelaxedCapture relaxed;
    for (int device : devices_)
      if (hipSetDevice(device) == hipSuccess) (void)hipStreamSynchronize(hipStreamPerThread);
  }

 private:
  static uint64_t next() {
    static std::atomic<uint64_t> n{1};
    return n++;
  }
  std::shared_ptr<char> life_;  // (released last)
  std::vector<int> devices_;
  const uint64_t number_ = next();
};
}  // namespace

// (made behind the thread's first call of the runtime, so it ends before the runtime's own record of the thread)
ThreadStream thread_stream(int device) {
  thread_local ThreadEnd end;
  return end.add(device);
}

StreamScratch::~StreamScratch() {
  pool_.clear([](void *p) { hipFree(p); });
  if (shared_done_) hipEventDestroy(shared_done_);
}

int StreamScratch::take(hipStream_t st, size_t bytes, ScratchPool::Lease *lease) {
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  hipGraph_t graph = nullptr;
  hipError_t e = hipStreamGetCaptureInfo_v2(st, &cap, &id, &graph, nullptr, nullptr);
  if (e != hipSuccess) return hip_fail(e, "hipStreamGetCaptureInfo");
  // (under capture nothing is given back to make room: hipFree waits for the device)
  const bool capturing = cap != hipStreamCaptureStatusNone;
  auto alloc = [capturing](size_t n) {
    RelaxedCapture relaxed;
    void *ptr = nullptr;
    if ((capturing ? hipMalloc(&ptr, n) : device_alloc(&ptr, n)) == hipSuccess) return ptr;
    (void)hipGetLastError();
    return static_cast<void *>(nullptr);
  };
  if (capturing) {
    ScratchPool::Record *made = nullptr;
    lease->ptr = pool_.captured(id, st, bytes, alloc, &made);
    hipUserObject_t owner = nullptr;
    if (made) {  // the graph's, and that of every executable graph made from it
      e = hipUserObjectCreate(&owner, made, ScratchPool::release, 1, hipUserObjectNoDestructorSync);
      if (e != hipSuccess) {
        ScratchPool::release(made);
        return hip_fail(e, "product scratch");
      }
      if ((e = hipGraphRetainUserObject(graph, owner, 1, hipGraphUserObjectMove)) != hipSuccess) {
        hipUserObjectRelease(owner, 1);
        return hip_fail(e, "product scratch");
      }
    }
  } else {
    ThreadStream thread{};
    if (st == hipStreamPerThread) {
      int device = 0;
      if ((e = hipGetDevice(&device)) != hipSuccess) return hip_fail(e, "hipGetDevice");
      thread = thread_stream(device);
    }
    *lease = pool_.eager(st, thread.number, bytes, alloc, thread.number ? &thread.life : nullptr);
  }
  if (!lease->ptr) return fail(TINYOAI_ENOMEM, "product scratch of %zu bytes", bytes);
  if (lease->shared) {
    RelaxedCapture relaxed;
    if (!shared_done_)
      e = hipEventCreateWithFlags(&shared_done_, hipEventDisableTiming);
    else
      e = hipStreamWaitEvent(st, shared_done_, 0);
    if (e != hipSuccess) return hip_fail(e, "product scratch");
  }
  return TINYOAI_OK;
}

hipError_t StreamScratch::give_back(hipStream_t st) {
  RelaxedCapture relaxed;
  return hipEventRecord(shared_done_, st);
}

// ---------------------------------------------------------------- matrices
ExpertMatrix::~ExpertMatrix() {
  if (mem) hipFree(mem);
  if (infinite) hipFree(infinite);
}

int check_matrices(int32_t dtype, int32_t experts, int64_t rows, int64_t cols, uint64_t nbytes, int64_t *each) {
  if (experts <= 0 || experts > kMxExperts || rows <= 0 || rows > (1 << 28) || cols <= 0 || cols > kMxCols)
    return fail(TINYOAI_EINVAL, "invalid matrix shape [%lld, %lld] of %d", (long long)rows, (long long)cols, experts);
  if (dtype != FMT_BF16 && dtype != FMT_MXFP4) return fail(TINYOAI_EINVAL, "unsupported expert tensor type %d", dtype);
  if (dtype == FMT_MXFP4 && cols % 32)
    return fail(TINYOAI_EINVAL, "rows of type %d must hold whole quant blocks (%lld values)", dtype, (long long)cols);
  *each = dtype == FMT_MXFP4 ? rows * (cols / 32) * 17 : rows * cols * 2;
  if (*each > INT64_MAX / experts || nbytes != (uint64_t)*each * experts)
    return fail(TINYOAI_EINVAL, "%d tensors [%lld, %lld] of type %d need %llu bytes, got %llu", experts, (long long)rows,
                (long long)cols, dtype, (unsigned long long)*each * experts, (unsigned long long)nbytes);
  return TINYOAI_OK;
}

int ExpertMatrix::upload(int32_t dtype, int32_t experts, int64_t rows, int64_t cols, const void *data, const void *up,
                         uint64_t nbytes, hipStream_t st) {
  int64_t each = 0;
  if (int rc = check_matrices(dtype, experts, rows, cols, nbytes, &each)) return rc;
  MxMat m{};
  m.fmt = dtype;
  m.experts = experts;
  m.rows = (int32_t)rows;
  m.cols = (int32_t)cols;
  m.gate = up != nullptr;
  m.tiles = (int32_t)(((rows + 15) / 16 * (up ? 2 : 1) + 3) / 4 * 4);
  m.chunks = (int32_t)((cols + mx_chunk_cols(dtype) - 1) / mx_chunk_cols(dtype));
  const size_t codes = (size_t)experts * mx_code_bytes(m), bytes = codes + (size_t)experts * mx_scale_bytes(m);
  hipError_t e = device_alloc(&mem, bytes);
  if (e != hipSuccess) return fail(TINYOAI_ENOMEM, "hipMalloc(%zu): %s", bytes, hipGetErrorString(e));
  m.codes = (const uint8_t *)mem;
  m.scales = (const uint8_t *)mem + codes;
  void *raw = nullptr;
  // behind the room for one matrix, a word for each: whether it holds an infinity
  const size_t at = ((size_t)each + 3) / 4 * 4, phases = m.gate + 1;
  std::vector<uint32_t> any(experts * phases);
  const size_t raw_bytes = at + any.size() * 4;
  e = device_alloc(&raw, raw_bytes);
  if (e != hipSuccess) return fail(TINYOAI_ENOMEM, "hipMalloc(%zu): %s", raw_bytes, hipGetErrorString(e));
  const std::unique_ptr<void, hipError_t (*)(void *)> free_raw(raw, hipFree);
  uint8_t *matrix = (uint8_t *)raw;
  uint32_t *any_dev = (uint32_t *)(matrix + at);
  auto copy = [&](size_t i) {  // (of pairs, expert after expert, both)
    return hipMemcpyAsync(raw, (const uint8_t *)(i % phases ? up : data) + i / phases * each, each, hipMemcpyHostToDevice, st);
  };
  auto fetch = [&](void *to, const void *from, size_t n) {
    const hipError_t f = hipMemcpyAsync(to, from, n, hipMemcpyDeviceToHost, st);
    return f == hipSuccess ? hipStreamSynchronize(st) : f;
  };
  e = hipMemsetAsync(mem, 0, bytes, st);  // rows and columns past the matrix are zeros
  if (e == hipSuccess) e = hipMemsetAsync(any_dev, 0, any.size() * 4, st);
  for (size_t i = 0; i < any.size(); i++) {
    if (e == hipSuccess) e = copy(i);
    if (e == hipSuccess) e = launch_mx_place(m, matrix, (int)(i / phases), (int)(i % phases), any_dev + i, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);  // the next copy takes the same buffer
  }
  if (e == hipSuccess) e = fetch(any.data(), any_dev, any.size() * 4);
  if (e != hipSuccess) return hip_fail(e, "expert upload");
  std::vector<int32_t> found;  // (expert, row) with an infinity
  for (size_t i = 0; i < any.size(); i += phases) {
    if (std::none_of(&any[i], &any[i] + phases, [](uint32_t v) { return v != 0; })) continue;
    std::vector<uint8_t> flags(rows);
    void *flags_dev = nullptr;
    e = device_alloc(&flags_dev, rows);
    if (e != hipSuccess) return fail(TINYOAI_ENOMEM, "hipMalloc(%lld): %s", (long long)rows, hipGetErrorString(e));
    e = hipMemsetAsync(flags_dev, 0, rows, st);
    for (size_t j = i; j < i + phases; j++) {
      if (e == hipSuccess) e = copy(j);
      if (e == hipSuccess) e = launch_mx_infinite(dtype, matrix, rows, cols, (uint8_t *)flags_dev, st);
      if (e == hipSuccess) e = hipStreamSynchronize(st);
    }
    if (e == hipSuccess) e = fetch(flags.data(), flags_dev, rows);
    hipFree(flags_dev);
    if (e != hipSuccess) return hip_fail(e, "expert upload");
    for (int64_t r = 0; r < rows; r++)
      if (flags[r]) found.insert(found.end(), {(int32_t)(i / phases), (int32_t)r});
  }
  if (!found.empty()) {
    if (found.size() / 2 > INT32_MAX) return fail(TINYOAI_EINVAL, "%zu rows with infinities", found.size() / 2);
    e = device_alloc(&infinite, found.size() * 4);
    if (e != hipSuccess) return fail(TINYOAI_ENOMEM, "hipMalloc(%zu): %s", found.size() * 4, hipGetErrorString(e));
    e = hipMemcpyAsync(infinite, found.data(), found.size() * 4, hipMemcpyHostToDevice, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    if (e != hipSuccess) return hip_fail(e, "expert upload");
    m.infinite = (const int32_t *)infinite;
    m.infinite_rows = (int32_t)(found.size() / 2);
  }
  d = m;
  return TINYOAI_OK;
}

int check_device(int device, const char *what) {
  int current = 0;
  const hipError_t e = hipGetDevice(&current);
  if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
  if (current != device)
    return fail(TINYOAI_EINVAL, "the %s lives on device %d, not the current %d", what, device, current);
  return TINYOAI_OK;
}

int check_mxfp4_rows(const void *codes, const void *scales) {
  if (reinterpret_cast<uintptr_t>(codes) % 16 || reinterpret_cast<uintptr_t>(scales) % 4)
    return fail(TINYOAI_EINVAL, "MXFP4 rows need codes on 16-byte and scales on 4-byte boundaries");
  return TINYOAI_OK;
}

int check_product(const MxProduct &p) {
  if (mx_supported(p)) return TINYOAI_OK;
  return fail(TINYOAI_EINVAL, "product of %d rows (of %d) by %d outputs exceeds what one call takes", p.n, p.x_rows, p.w.rows);
}

// A row-major [n][cols] buffer of F32, F16 or BF16 values.
static int check_rows(const char *what, int32_t dtype, const void *p, int64_t ld, int64_t cols) {
  if (dtype != FMT_F32 && dtype != FMT_F16 && dtype != FMT_BF16)
    return fail(TINYOAI_EINVAL, "unsupported %s type %d", what, dtype);
  if (!p) return fail(TINYOAI_EINVAL, "%s is null", what);
  if (ld < cols) return fail(TINYOAI_EINVAL, "%s rows of %lld values are %lld apart", what, (long long)cols, (long long)ld);
  if (reinterpret_cast<uintptr_t>(p) % mx_width(dtype)) return fail(TINYOAI_EINVAL, "%s is not aligned to its type", what);
  return TINYOAI_OK;
}

}  // namespace tinyoai

using namespace tinyoai;

struct tinyoai_experts {
  ExpertMatrix m;
  int device = 0;
  hipStream_t stream = nullptr;
  StreamScratch scratch;
  ~tinyoai_experts() {
    if (stream) hipStreamDestroy(stream);
  }
};

extern "C" {

int tinyoai_mxfp4_quantize_device(int32_t dtype, const void *x_dev, int64_t ldx, int64_t n, int64_t cols,
                                  uint8_t *codes_dev, uint8_t *scales_dev, void *stream) {
  if (n <= 0 || cols <= 0 || cols % 32 || n > INT32_MAX || cols > kMxCols)
    return fail(TINYOAI_EINVAL, "invalid MXFP4 shape [%lld, %lld]", (long long)n, (long long)cols);
  if (int rc = check_rows("x", dtype, x_dev, ldx, cols)) return rc;
  if (!codes_dev || !scales_dev) return fail(TINYOAI_EINVAL, "invalid MXFP4 rows");
  if (int rc = check_mxfp4_rows(codes_dev, scales_dev)) return rc;
  const hipError_t e = launch_mx_quantize(dtype, x_dev, ldx, n, cols, codes_dev, scales_dev, (hipStream_t)stream);
  return e == hipSuccess ? TINYOAI_OK : hip_fail(e, "MXFP4 quantisation");
}

int tinyoai_mxfp4_dequantize_device(const uint8_t *codes_dev, const uint8_t *scales_dev, int64_t n, int64_t cols,
                                    int32_t dtype, void *out_dev, int64_t ldo, void *stream) {
  if (n <= 0 || cols <= 0 || cols % 32 || n > INT32_MAX || cols > kMxCols)
    return fail(TINYOAI_EINVAL, "invalid MXFP4 shape [%lld, %lld]", (long long)n, (long long)cols);
  if (int rc = check_rows("out", dtype, out_dev, ldo, cols)) return rc;
  if (!codes_dev || !scales_dev) return fail(TINYOAI_EINVAL, "invalid MXFP4 rows");
  if (int rc = check_mxfp4_rows(codes_dev, scales_dev)) return rc;
  const hipError_t e = launch_mx_dequantize(codes_dev, scales_dev, n, cols, dtype, out_dev, ldo, (hipStream_t)stream);
  return e == hipSuccess ? TINYOAI_OK : hip_fail(e, "MXFP4 values");
}

int tinyoai_route_device(int32_t dtype, const void *logits_dev, int64_t ld, int32_t n, int32_t experts, int32_t k,
                         int32_t over_all, int32_t *ids_dev, float *weights_dev, int32_t *offsets_dev,
                         int32_t *tokens_dev, int32_t *positions_dev, void *stream) {
  if (n <= 0 || experts <= 0 || experts > kRouteExperts || k <= 0 || k > kRouteMost || k > experts ||
      (int64_t)n * k > (1 << 30))
    return fail(TINYOAI_EINVAL, "invalid routing of %d tokens to %d of %d experts", n, k, experts);
  if (int rc = check_rows("logits", dtype, logits_dev, ld, experts)) return rc;
  if (!ids_dev || !weights_dev || !offsets_dev || !tokens_dev || !positions_dev)
    return fail(TINYOAI_EINVAL, "invalid routing outputs");
  const hipError_t e = launch_route(RouteArgs{dtype, logits_dev, ld, n, experts, k, over_all, ids_dev, weights_dev,
                                              offsets_dev, tokens_dev, positions_dev},
                                    (hipStream_t)stream);
  return e == hipSuccess ? TINYOAI_OK : hip_fail(e, "routing");
}

int tinyoai_combine_device(int32_t dtype, const void *y_dev, int64_t ldy, int32_t y_rows, const int32_t *positions_dev,
                           const float *weights_dev, int32_t n, int32_t k, int64_t cols, int32_t out_dtype, void *out_dev,
                           int64_t ldo, void *stream) {
  if (n <= 0 || k <= 0 || y_rows < 0 || cols <= 0 || cols > INT32_MAX || (int64_t)n * k > (1 << 30) ||
      n * ((cols + 255) / 256) > INT32_MAX)
    return fail(TINYOAI_EINVAL, "invalid sum of %d rows for %d tokens", k, n);
  if (int rc = check_rows("y", dtype, y_dev, ldy, cols)) return rc;
  if (int rc = check_rows("out", out_dtype, out_dev, ldo, cols)) return rc;
  if (!positions_dev || !weights_dev) return fail(TINYOAI_EINVAL, "invalid positions or weights");
  const hipError_t e = launch_combine(CombineArgs{dtype, y_dev, ldy, y_rows, positions_dev, weights_dev, n, k, cols,
                                                  out_dtype, out_dev, ldo},
                                      (hipStream_t)stream);
  return e == hipSuccess ? TINYOAI_OK : hip_fail(e, "combine");
}

int tinyoai_experts_upload(int32_t dtype, int32_t experts, int64_t rows, int64_t cols, const void *data, const void *up,
                           uint64_t nbytes, tinyoai_experts **out) try {
  if (!out || !data) return fail(TINYOAI_EINVAL, "invalid expert upload arguments");
  *out = nullptr;
  int64_t each = 0;
  if (int rc = check_matrices(dtype, experts, rows, cols, nbytes, &each)) return rc;
  auto x = std::make_unique<tinyoai_experts>();
  hipError_t e = hipGetDevice(&x->device);
  if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
  e = hipStreamCreateWithFlags(&x->stream, hipStreamNonBlocking);
  if (e != hipSuccess) return hip_fail(e, "hipStreamCreate");
  if (int rc = x->m.upload(dtype, experts, rows, cols, data, up, nbytes, x->stream)) return rc;
  *out = x.release();
  return TINYOAI_OK;
} catch (const std::exception &e) {
  return fail(TINYOAI_ENOMEM, "expert upload: %s", e.what());
}

int tinyoai_experts_mul_device(tinyoai_experts *x, int32_t x_dtype, const void *x_dev, const uint8_t *x_scales_dev,
                               int64_t ldx, int32_t x_rows, const int32_t *offsets_dev, const int32_t *index_dev,
                               int32_t n, int32_t out_dtype, void *out_dev, int64_t ldo, void *stream) try {
  if (!x || !offsets_dev || n <= 0 || x_rows <= 0) return fail(TINYOAI_EINVAL, "invalid product arguments");
  const MxMat &m = x->m.d;
  if (x_dtype == FMT_MXFP4) {
    if (m.fmt != FMT_MXFP4) return fail(TINYOAI_EINVAL, "products of MXFP4 rows need MXFP4 experts, not type %d", m.fmt);
    if (!x_dev || !x_scales_dev) return fail(TINYOAI_EINVAL, "invalid MXFP4 rows");
    if (ldx != m.cols) return fail(TINYOAI_EINVAL, "MXFP4 rows of %d values, not %lld", m.cols, (long long)ldx);
    if (int rc = check_mxfp4_rows(x_dev, x_scales_dev)) return rc;
  } else {
    if (int rc = check_rows("x", x_dtype, x_dev, ldx, m.cols)) return rc;
    if (x_scales_dev) return fail(TINYOAI_EINVAL, "scales with x of type %d", x_dtype);
  }
  if (int rc = check_rows("out", out_dtype, out_dev, ldo, m.rows)) return rc;
  if (!index_dev && x_rows < n) return fail(TINYOAI_EINVAL, "%d rows of x for %d rows without an index", x_rows, n);
  if (int rc = check_device(x->device, "experts")) return rc;
  hipStream_t st = stream ? (hipStream_t)stream : x->stream;
  // (without an index, rows past n do not count; an MXFP4 buffer's layout has them)
  if (!index_dev && x_dtype != FMT_MXFP4) x_rows = n;
  const MxProduct p{m, x_dtype, x_dev, x_scales_dev, ldx, x_rows, offsets_dev, index_dev, n, out_dtype, out_dev, ldo};
  if (int rc = check_product(p)) return rc;
  return x->scratch.run(st, mx_scratch(p), [&](void *scratch) { return launch_mx_product(p, scratch, st); });
} catch (const std::exception &e) {
  return fail(TINYOAI_ENOMEM, "product: %s", e.what());
}

int tinyoai_experts_free(tinyoai_experts *x) {
  if (x) {
    hipStreamSynchronize(x->stream);
    delete x;
  }
  return TINYOAI_OK;
}

}  // extern "C"
