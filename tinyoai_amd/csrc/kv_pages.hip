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
// its largest magnitude by two lane moves.
#include <type_traits>

#include "attend.h"

namespace {

constexpr int kT = 256;

// Chunks of eight values that a head's row has room for: 8-bit rows in whole blocks.
__host__ __device__ inline int row_chunks(const KVPagesDev &c) {
  return c.type == FMT_Q8_0 ? (c.hd + 31) / 32 * 4 : c.hd / 8;
}

struct Item {
  int row, head, chunk;
};
__device__ __forceinline__ Item item_of(uint32_t i, uint32_t chunks, uint32_t heads) {
  const uint32_t rh = i / chunks;
  return Item{(int)(rh / heads), (int)(rh % heads), (int)(i % chunks)};
}

__device__ __forceinline__ int quantised(float x, float d) {
  return (int)fminf(fmaxf(rintf(__fdiv_rn(x, d)), -127.f), 127.f);
}

template <int D, int C>
__global__ __launch_bounds__(kT) void write_kernel(KVRowsArgs a, int64_t first, int64_t items) {
  const int64_t at = first + (int64_t)blockIdx.x * kT + threadIdx.x;
  const int chunks = row_chunks(a.c);
  const int per = a.c.kv_heads * chunks;
  const int row = (int)(at / per);
  const Item it = item_of((uint32_t)(at - (int64_t)row * per), chunks, a.c.kv_heads);
  // (the four lanes of an 8-bit block take the same branches: they hold one row's)
  if (at >= items) return;
  const int slot = a.slots[row];
  if ((uint32_t)slot >= (uint32_t)a.c.pages << a.c.page_log2) return;
  const int head = it.head;
  const void *src = blockIdx.y ? a.v : a.k;
  uint8_t *dst = blockIdx.y ? a.c.v : a.c.k;
  const int64_t to = kv_row(a.c, slot, head);
  float v[8] = {};
  const int c = it.chunk * 8;
  if (c < a.c.hd) load8<D>(src, row * (blockIdx.y ? a.ldv : a.ldk) + (int64_t)head * a.c.hd + c, v);
  if constexpr (C == FMT_Q8_0) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
    most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0xb1, 0xf, 0xf, false));  // lanes 1, 0, 3, 2
    most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0x4e, 0xf, 0xf, false));  // lanes 2, 3, 0, 1
    const bool bad = most >= 0x7f800000u;
    const uint16_t bits = bad ? 0x7e00 : __half_as_ushort(__float2half_rn(fminf(__fdiv_rn(__uint_as_float(most), 127.f), 65504.f)));
    const float d = hw_half(bits);
    uint32_t w[2] = {};
    if (!bad && d > 0.f) {
#pragma unroll
      for (int j = 0; j < 8; j++) w[j / 4] |= (uint32_t)(quantised(v[j], d) & 255) << (8 * (j % 4));
    }
    if (c < a.c.hd) *reinterpret_cast<uint2 *>(dst + to * a.c.pitch + c) = make_uint2(w[0], w[1]);
    if ((it.chunk & 3) == 0) (blockIdx.y ? a.c.vd : a.c.kd)[to * a.c.nb + it.chunk / 4] = bits;
  } else {
    store8<C>(dst + to * a.c.pitch, c, v);
  }
}

template <int D, int C>
__global__ __launch_bounds__(kT) void read_kernel(KVRowsArgs a, int64_t first, int64_t items) {
  const int64_t at = first + (int64_t)blockIdx.x * kT + threadIdx.x;
  if (at >= items) return;
  const int chunks = a.c.hd / 8;
  const int per = a.c.kv_heads * chunks;
  const int row = (int)(at / per);
  const Item it = item_of((uint32_t)(at - (int64_t)row * per), chunks, a.c.kv_heads);
  const int slot = a.slots[row], head = it.head, c = it.chunk * 8;
  void *dst = blockIdx.y ? a.v : a.k;
  const int64_t to = row * (blockIdx.y ? a.ldv : a.ldk) + (int64_t)head * a.c.hd + c;
  float v[8] = {};
  if ((uint32_t)slot < (uint32_t)a.c.pages << a.c.page_log2) {
    const int64_t from = kv_row(a.c, slot, head);
    const uint8_t *src = (blockIdx.y ? a.c.v : a.c.k) + from * a.c.pitch;
    if constexpr (C == FMT_Q8_0) {
      const float d = hw_half((blockIdx.y ? a.c.vd : a.c.kd)[from * a.c.nb + it.chunk / 4]);
      const uint2 w = *reinterpret_cast<const uint2 *>(src + c);
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = (float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j % 4))) * d;
    } else {
      load8<C>(src, c, v);
    }
  }
  store8<D>(dst, to, v);
}

template <typename F>
void for_cache(int type, const F &call) {
  if (type == FMT_Q8_0) call(std::integral_constant<int, FMT_Q8_0>());
  else for_type(type, call);
}

template <typename F>
hipError_t over_items(int64_t items, const F &launch) {
  constexpr int64_t kMost = (int64_t)kT << 22;  // a launch's threads, of K and of V, number below 2^32
  for (int64_t first = 0; first < items; first += kMost) {
    const int64_t n = items - first < kMost ? items - first : kMost;
    launch(dim3((unsigned)((n + kT - 1) / kT), 2), first);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_write(const KVRowsArgs &a, hipStream_t st) {
  const int64_t items = (int64_t)a.n * a.c.kv_heads * row_chunks(a.c);
  return over_items(items, [&](dim3 grid, int64_t first) {
    for_type(a.dtype, [&](auto d) {
      for_cache(a.c.type, [&](auto c) {
        hipLaunchKernelGGL((write_kernel<decltype(d)::value, decltype(c)::value>), grid, dim3(kT), 0, st, a, first, items);
      });
    });
  });
}

hipError_t launch_kv_read(const KVRowsArgs &a, hipStream_t st) {
  const int64_t items = (int64_t)a.n * a.c.kv_heads * (a.c.hd / 8);
  return over_items(items, [&](dim3 grid, int64_t first) {
    for_type(a.dtype, [&](auto d) {
      for_cache(a.c.type, [&](auto c) {
        hipLaunchKernelGGL((read_kernel<decltype(d)::value, decltype(c)::value>), grid, dim3(kT), 0, st, a, first, items);
      });
    });
  });
}
