// Operators around a layer's attention: rotary positions, the paged key-value
// cache, the attention of new tokens over its pages and of packed prompts:
// their arguments, the pages' layout in HBM and the launch interfaces.
//
// Pages: K and V of a layer are planes of their own, and a page holds one head
// after another, each head's positions together: [pages][kv_heads][page] rows
// of `pitch` bytes (a head's values, rounded up to 16 bytes with zeros). What a
// block attends to, a head's positions of a page, is then one contiguous run.
// 8-bit pages (Q8_0) hold a byte a value and, in planes of their own with the
// same order, the fp16 scales of a row's blocks of 32 values (the last block
// may be shorter), `nb` of them, a power of two from 2 on.
#pragma once

#include "mx.h"

constexpr int kHeadDim = 256;   // of a head, at most; a multiple of 8
constexpr int kPage = 1024;     // positions of a page, at most; a power of two
constexpr int64_t kRowValues = 1 << 22;   // of a buffer's row, at most
constexpr int64_t kPositions = 1 << 30;   // of a pool, a table's row or a packed buffer, at most
constexpr int64_t kAttendRows = 1 << 22;  // query heads of all of a call's new tokens, at most

struct KVPagesDev {
  int32_t type;                 // FMT_F32, FMT_F16, FMT_BF16 or FMT_Q8_0
  int32_t kv_heads, hd;
  int32_t page_log2;            // positions of a page
  int32_t pages;
  int32_t pitch, nb;            // bytes of a row, its scales (0: none)
  uint8_t *k, *v;               // of the call's layer
  uint16_t *kd, *vd;            // scales
  const uint8_t *zeros;         // 256 bytes: what positions that do not count read
};

// The row of (slot, head): of a plane in rows, so `pitch` bytes or `nb` scales each.
__host__ __device__ inline int64_t kv_row(const KVPagesDev &c, int slot, int head) {
  const int page = slot >> c.page_log2, at = slot & ((1 << c.page_log2) - 1);
  return ((((int64_t)page * c.kv_heads + head) << c.page_log2) + at);
}

// n rows [kv_heads][hd] of K and of V to (write) or from their slots; rows of
// slots outside the pool are left out.
struct KVRowsArgs {
  KVPagesDev c;
  int32_t dtype;
  void *k, *v;
  int64_t ldk, ldv;
  const int32_t *slots;
  int32_t n;
};
hipError_t launch_kv_write(const KVRowsArgs &a, hipStream_t st);
hipError_t launch_kv_read(const KVRowsArgs &a, hipStream_t st);

// One new token of each of n sequences over its pages.
struct AttendArgs {
  KVPagesDev c;
  int32_t dtype;                // of q and out
  const void *q;
  int64_t ldq;
  int32_t heads;
  float scale;
  const int32_t *table;         // [n][width]
  int32_t width;
  const int32_t *lengths;
  int32_t n;
  void *out;
  int64_t ldo;
};
// Bytes of scratch (0: none) that launch_attend takes.
size_t attend_scratch(const AttendArgs &a);
hipError_t launch_attend(const AttendArgs &a, void *scratch, hipStream_t st);

// Packed sequences: queries q_offsets[s] .. q_offsets[s + 1] - 1 over keys
// k_offsets[s] .. k_offsets[s + 1] - 1.
struct PromptArgs {
  int32_t dtype;
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  int32_t heads, kv_heads, hd;
  float scale;
  int32_t causal;
  const int32_t *q_offsets, *k_offsets;
  int32_t sequences, nq, nk;
  void *out;
  int64_t ldo;
};
// Bytes of scratch (0: none) that launch_prompt takes.
size_t prompt_scratch(const PromptArgs &a);
hipError_t launch_prompt(const PromptArgs &a, void *scratch, hipStream_t st);

// Rows of heads turned by their positions.
struct RopeArgs {
  const double *frequencies;    // [rot / 2], radians a position
  float magnitude;
  int32_t hd, rot, interleaved;
  int32_t dtype, out_dtype;
  const void *x;
  int64_t ldx;
  int32_t n, heads;
  const int32_t *positions;
  void *out;
  int64_t ldo;
};
hipError_t launch_rope(const RopeArgs &a, hipStream_t st);

// Eight values of a row from value i on (any alignment of the type's), as fp32.
template <int D>
__device__ __forceinline__ void load8(const void *x, int64_t i, float (&v)[8]) {
  if constexpr (D == FMT_F32) {
    const f32x4_any *p = reinterpret_cast<const f32x4_any *>(static_cast<const float *>(x) + i);
    const f32x4_any a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const u32x4_any w = *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(x) + i);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint16_t h = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
      v[j] = D == FMT_F16 ? hw_half(h) : bf16_to_float(h);
    }
  }
}
// Eight values rounded to the nearest, stored from value i on.
template <int D>
__device__ __forceinline__ void store8(void *x, int64_t i, const float (&v)[8]) {
  if constexpr (D == FMT_F32) {
    f32x4_any *p = reinterpret_cast<f32x4_any *>(static_cast<float *>(x) + i);
    p[0] = f32x4_any{v[0], v[1], v[2], v[3]};
    p[1] = f32x4_any{v[4], v[5], v[6], v[7]};
  } else {
    u32x4_any w;
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = mx_narrow(D, v[2 * j]) | (uint32_t)mx_narrow(D, v[2 * j + 1]) << 16;
    *reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(x) + i) = w;
  }
}
// call(std::integral_constant<int, type>) for a type of F32, F16 and BF16.
template <typename F>
inline void for_type(int dtype, const F &call) {
  if (dtype == FMT_F32) call(std::integral_constant<int, FMT_F32>());
  else if (dtype == FMT_F16) call(std::integral_constant<int, FMT_F16>());
  else call(std::integral_constant<int, FMT_BF16>());
}

// LDS rows of C chunks of 16 bytes; chunk c of row r at place c ^ swizzle, so
// that the lanes of a read that go together hit distinct banks. K (by rows): 16
// consecutive rows, one chunk. V (transposed): 4 consecutive rows, 4 chunks
// (fp32: one row, consecutive dims: none needed).
template <int C>
__device__ __forceinline__ int k_place(int r, int c) {
  if constexpr (C % 16 == 0) return c ^ (r & 15);
  else if constexpr (C == 8) return c ^ ((r >> 1) & 7);
  else if constexpr (C % 4 == 0) return c ^ ((r >> 2) & 3);
  else return c ^ ((r >> 3) & 1);
}
// (rows of ten chunks: four rows in a row are kept two apart instead, v_row)
template <int C>
__device__ __forceinline__ int v_row(int r) { return C == 10 ? (r & ~7) | (r & 3) << 1 | ((r >> 2) & 1) : r; }
template <int C>
__device__ __forceinline__ int v_key(int r) { return C == 10 ? (r & ~7) | ((r >> 1) & 3) | (r & 1) << 2 : r; }  // its inverse
template <int C>
__device__ __forceinline__ int v_place(int r, int c) {
  if constexpr (C % 16 == 0) return c ^ ((r & 3) << 2 | ((r >> 2) & 3));
  else if constexpr (C == 8) return c ^ (((r >> 1) & 1) << 2 | ((r >> 2) & 3));
  else return c;
}

// The value of lane l % 32.
__device__ __forceinline__ float lower_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]);
}
// As lds_dma16 and lds_dma4 (or from an address per lane), for a descriptor or a
// place in LDS that a lane read has just put into scalar registers: the
// hardware wants five wait states between that and the load, and the compiler,
// which sees to it elsewhere, does not look into inline assembly.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t lds_byte) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "{m0}"(lds_byte) : "memory");
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t lds_byte) {
  asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "{m0}"(lds_byte) : "memory");
}
__device__ __forceinline__ void dma16_at(const void *p, uint32_t lds_byte) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "{m0}"(lds_byte) : "memory");
}
__device__ __forceinline__ void dma4_at(const void *p, uint32_t lds_byte) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, off" ::"v"(p), "{m0}"(lds_byte) : "memory");
}

// Over lanes l and l ^ 32, and (quarters) l, l ^ 16, l ^ 32 and l ^ 48.
__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float quarters_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarters_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
