// Rows of keys and values to the slots of a paged cache, and back.
//
// An 8-bit block of 32 values x of a head (the last one may be shorter): its
// scale is d = fp16(fp32(max |x| / 127)), at most 65504, and each code the
// fp32 quotient x / d rounded to the nearest whole number, halfway ones to the
// even one, within -127 .. 127; a scale of zero has zero codes. A block with an
// infinity or NaN becomes NaN (scale NaN, zero codes). Other types round to the
// nearest.
//
// What bounds it: HBM (each value read once, what the pages hold written
// once). A thread takes eight values, so four lanes hold a block and exchange
// its largest magnitude by two lane moves. It keeps its place within the row
// and goes through rows, four at a time, whose loads all start before the first
// is used. Quotients come from the scale's reciprocal where that cannot change
// what they round to. 8192 bf16 rows of 8 heads of 128 (K and V) to 8-bit
// pages 14 us, and back 10: 101 MB at 3.9 TB/s with the launches (a thread a
// chunk, its loads alone and divisions throughout: 18 and 12).
#include <type_traits>

#include "attend.h"

namespace {

constexpr int kT = 256, kBatch = 4;

// Chunks of eight values that a head's row has room for: 8-bit rows in whole blocks.
__host__ __device__ inline int row_chunks(const KVPagesDev &c, bool write) {
  return c.type == FMT_Q8_0 && write ? (c.hd + 31) / 32 * 4 : c.hd / 8;
}

// How a launch's blocks are laid over n rows of `per` chunks: `side` rows next
// to each other (or `parts` blocks a row), `rows` rows a block.
struct Grid {
  int per, side, parts, rows;
  Grid(const KVRowsArgs &a, bool write) {
    per = a.c.kv_heads * row_chunks(a.c, write);
    side = per < kT ? kT / per : 1;
    parts = (per + kT - 1) / kT;
    // as many rows a thread, up to a batch, as leave the chip full
    const int64_t full = ((int64_t)a.n * parts + side * 1024 - 1) / (side * 1024);
    rows = side * (int)std::min<int64_t>(kBatch, full);
  }
};
// This thread's chunk of every row, and its row among those side by side.
struct Place {
  int head, chunk, row;
  bool in;
};
__device__ __forceinline__ Place place_of(const Grid &g, int chunks) {
  const int item = g.parts > 1 ? blockIdx.y * kT + threadIdx.x : threadIdx.x % g.per;
  const int row = g.parts > 1 ? 0 : threadIdx.x / g.per;
  return Place{item / chunks, item % chunks, row, item < g.per && row < g.side};
}

// x / d rounded to fp32 and then to the nearest whole number. x times the
// reciprocal is off by less than 2^-16 where that is below 128, and the fp32
// quotient by 2^-18, so both round alike but next to halfway points.
__device__ __forceinline__ void quantised8(const float (&x)[8], float d, int (&q)[8]) {
  const float inv = __fdiv_rn(1.f, d);
  bool close = false;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float t = x[j] * inv, r = rintf(t);
    close |= fabsf(t - r) > 0.5f - 0x1p-14f;
    q[j] = (int)fminf(fmaxf(r, -127.f), 127.f);
  }
  if (!close) return;
#pragma unroll
  for (int j = 0; j < 8; j++) q[j] = (int)fminf(fmaxf(rintf(__fdiv_rn(x[j], d)), -127.f), 127.f);
}

template <int D, int C>
__global__ __launch_bounds__(kT) void write_kernel(KVRowsArgs a, Grid grid) {
  const int chunks = C == FMT_Q8_0 ? (a.c.hd + 31) / 32 * 4 : a.c.hd / 8;
  // (the four lanes of an 8-bit block take the same branches: they hold one row's)
  const Place at = place_of(grid, chunks);
  if (!at.in) return;
  const bool value = blockIdx.z;
  const void *src = value ? a.v : a.k;
  uint8_t *dst = value ? a.c.v : a.c.k;
  const int64_t ld = value ? a.ldv : a.ldk;
  const int c = at.chunk * 8;
  float v[kBatch][8];
  int slot[kBatch];
#pragma unroll
  for (int j = 0; j < kBatch; j++) {
    const int64_t row = (int64_t)blockIdx.x * grid.rows + j * grid.side + at.row;
    slot[j] = -1;
#pragma unroll
    for (int i = 0; i < 8; i++) v[j][i] = 0.f;
    if (j * grid.side < grid.rows && row < a.n) {
      slot[j] = a.slots[row];
      if (c < a.c.hd) load8<D>(src, row * ld + (int64_t)at.head * a.c.hd + c, v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kBatch; j++) {
    if ((uint32_t)slot[j] >= (uint32_t)a.c.pages << a.c.page_log2) continue;
    const int64_t to = kv_row(a.c, slot[j], at.head);
    if constexpr (C == FMT_Q8_0) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) most = max(most, __float_as_uint(v[j][i]) & 0x7fffffffu);
      most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0xb1, 0xf, 0xf, false));  // lanes 1, 0, 3, 2
      most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0x4e, 0xf, 0xf, false));  // lanes 2, 3, 0, 1
      const bool bad = most >= 0x7f800000u;
      const uint16_t bits = bad ? 0x7e00 : __half_as_ushort(__float2half_rn(fminf(__fdiv_rn(__uint_as_float(most), 127.f), 65504.f)));
      const float d = hw_half(bits);
      uint32_t w[2] = {};
      if (!bad && d > 0.f) {
        int q[8];
        quantised8(v[j], d, q);
#pragma unroll
        for (int i = 0; i < 8; i++) w[i / 4] |= (uint32_t)(q[i] & 255) << (8 * (i % 4));
      }
      if (c < a.c.hd) *reinterpret_cast<uint2 *>(dst + to * a.c.pitch + c) = make_uint2(w[0], w[1]);
      if ((at.chunk & 3) == 0) (value ? a.c.vd : a.c.kd)[to * a.c.nb + at.chunk / 4] = bits;
    } else {
      store8<C>(dst + to * a.c.pitch, c, v[j]);
    }
  }
}

template <int D, int C>
__global__ __launch_bounds__(kT) void read_kernel(KVRowsArgs a, Grid grid) {
  const Place at = place_of(grid, a.c.hd / 8);
  if (!at.in) return;
  const bool value = blockIdx.z;
  void *dst = value ? a.v : a.k;
  const int64_t ld = value ? a.ldv : a.ldk;
  const int c = at.chunk * 8;
  float v[kBatch][8], d[kBatch];
  uint2 w[kBatch];
  int64_t row[kBatch];
  int slot[kBatch];
#pragma unroll
  for (int j = 0; j < kBatch; j++) {
    row[j] = (int64_t)blockIdx.x * grid.rows + j * grid.side + at.row;
    if (j * grid.side >= grid.rows || row[j] >= a.n) row[j] = -1;
    slot[j] = row[j] < 0 ? -1 : a.slots[row[j]];
  }
#pragma unroll
  for (int j = 0; j < kBatch; j++) {
    w[j] = make_uint2(0, 0), d[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) v[j][i] = 0.f;
    if ((uint32_t)slot[j] >= (uint32_t)a.c.pages << a.c.page_log2) continue;
    const int64_t from = kv_row(a.c, slot[j], at.head);
    const uint8_t *src = (value ? a.c.v : a.c.k) + from * a.c.pitch;
    if constexpr (C == FMT_Q8_0) {
      d[j] = hw_half((value ? a.c.vd : a.c.kd)[from * a.c.nb + at.chunk / 4]);
      w[j] = *reinterpret_cast<const uint2 *>(src + c);
    } else {
      load8<C>(src, c, v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kBatch; j++) {
    if (row[j] < 0) continue;
    if constexpr (C == FMT_Q8_0)
#pragma unroll
      for (int i = 0; i < 8; i++) v[j][i] = (float)(int8_t)((i < 4 ? w[j].x : w[j].y) >> (8 * (i % 4))) * d[j];
    store8<D>(dst, row[j] * ld + (int64_t)at.head * a.c.hd + c, v[j]);
  }
}

template <typename F>
void for_cache(int type, const F &call) {
  if (type == FMT_Q8_0) call(std::integral_constant<int, FMT_Q8_0>());
  else for_type(type, call);
}

// launch(the grid's shape, the blocks of a launch)
template <typename F>
hipError_t over_rows(const KVRowsArgs &a, bool write, const F &launch) {
  const Grid g(a, write);
  // a launch's threads, of K and of V, number below 2^32
  const int64_t most = ((int64_t)1 << 22) / g.parts * g.rows;
  for (int64_t first = 0; first < a.n; first += most) {
    KVRowsArgs part = a;
    part.n = (int32_t)std::min<int64_t>(a.n - first, most);
    part.slots += first;
    part.k = static_cast<char *>(a.k) + first * a.ldk * (int64_t)mx_width(a.dtype);
    part.v = static_cast<char *>(a.v) + first * a.ldv * (int64_t)mx_width(a.dtype);
    launch(part, g, dim3((unsigned)((part.n + g.rows - 1) / g.rows), (unsigned)g.parts, 2));
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_write(const KVRowsArgs &a, hipStream_t st) {
  return over_rows(a, true, [&](const KVRowsArgs &part, const Grid &g, dim3 grid) {
    for_type(a.dtype, [&](auto d) {
      for_cache(a.c.type, [&](auto c) {
        hipLaunchKernelGGL((write_kernel<decltype(d)::value, decltype(c)::value>), grid, dim3(kT), 0, st, part, g);
      });
    });
  });
}

hipError_t launch_kv_read(const KVRowsArgs &a, hipStream_t st) {
  return over_rows(a, false, [&](const KVRowsArgs &part, const Grid &g, dim3 grid) {
    for_type(a.dtype, [&](auto d) {
      for_cache(a.c.type, [&](auto c) {
        hipLaunchKernelGGL((read_kernel<decltype(d)::value, decltype(c)::value>), grid, dim3(kT), 0, st, part, g);
      });
    });
  });
}
