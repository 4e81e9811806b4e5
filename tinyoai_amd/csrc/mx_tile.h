// Device parts that the matrix-core products of mx.h share: operands, the
// planes of X and their places in LDS.
#pragma once

#include <type_traits>

#include "mx.h"
#include "mx_rule.h"

// bf16 planes that hold a type's values exactly (MXFP4: none).
__host__ __device__ inline int mx_planes(int dtype) { return dtype == FMT_F32 ? 3 : dtype == FMT_F16 ? 2 : 1; }

// What the rules see of a product.
inline tinyoai_rule::Sizes mx_sizes(const MxProduct &p) {
  return {p.w.fmt == FMT_BF16, p.xdtype == FMT_MXFP4 ? 0 : mx_planes(p.xdtype), p.w.gate != 0, p.offsets != nullptr,
          p.w.experts, p.n, p.w.rows, p.w.cols};
}

namespace tinyoai_mx {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

template <int WF>
constexpr int mx_cols() { return WF == FMT_MXFP4 ? 128 : 64; }

__device__ __forceinline__ f32x4 mfma_bf16(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_bf16_32(uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// MXFP4 times MXFP4: a's scale is byte A of sa, b's byte B of sb.
template <int A, int B>
__device__ __forceinline__ f32x16 mfma_mx_32(uint4 a, uint4 b, f32x16 c, uint32_t sa, uint32_t sb) {
  const i32x8 x = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, y = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, A, (int)sa, B, (int)sb);
}
template <int A>
__device__ __forceinline__ f32x4 mfma_mx(uint4 a, uint4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 x = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, y = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, A, (int)sa, 0, (int)sb);
}
// Eight codes times 2^(exponent of s - 127) as bf16, exact within bf16's range.
__device__ __forceinline__ uint4 fp4_bf16(uint32_t c, float s) {
  auto two = [](bf16x2 v) { return __builtin_bit_cast(uint32_t, v); };
  return make_uint4(two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)), two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
                    two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)), two(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3)));
}

// A value's planes as fp32 bit patterns whose low halves are zero: what is
// left after a plane has eight bits fewer, and the difference is exact (but a
// plane's bits below 2^-133, bf16's smallest, are lost). An
// infinity or NaN is all in the first plane.
template <int P>
__device__ __forceinline__ void planes_of(float v, uint32_t (&h)[P]) {
  uint32_t u = __float_as_uint(v);
  if constexpr (P == 1) {
    h[0] = u;  // a bf16 value
  } else {
    const uint32_t mag = u & 0x7fffffffu;
    if (mag > 0x7f800000u) u |= 0x00400000u;  // the half kept must not read as an infinity
    h[0] = u & 0xffff0000u;
    const bool finite = mag < 0x7f800000u;
    float rest = finite ? v - __uint_as_float(h[0]) : 0.f;
#pragma unroll
    for (int i = 1; i < P; i++) {
      h[i] = __float_as_uint(rest) & 0xffff0000u;
      rest -= __uint_as_float(h[i]);
    }
  }
}
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {  // a's below b's
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// Raw bits of eight values of row `src` from column k on; zeros past `cols`.
// XT: the type.
template <int XT>
struct Raw8 {
  uint4 a[XT == FMT_F32 ? 2 : 1];
};
template <int XT>
__device__ __forceinline__ Raw8<XT> load_x8(const MxProduct &p, int64_t src, int k) {
  using V = std::conditional_t<XT == FMT_F32, uint32_t, uint16_t>;
  const V *s = static_cast<const V *>(p.x) + src * p.ldx + k;
  Raw8<XT> r;
  if (k + 8 <= p.w.cols) {
#pragma unroll
    for (int j = 0; j < (XT == FMT_F32 ? 2 : 1); j++) {
      const u32x4_any v = reinterpret_cast<const u32x4_any *>(s)[j];
      r.a[j] = make_uint4(v.x, v.y, v.z, v.w);
    }
  } else {
    V v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = k + j < p.w.cols ? s[j] : V(0);
    memcpy(&r, v, sizeof r);
  }
  return r;
}
// Their planes, each as eight bf16 values.
template <int XT>
__device__ __forceinline__ void planes8(const Raw8<XT> &r, uint4 (&out)[XT == FMT_F32 ? 3 : XT == FMT_F16 ? 2 : 1]) {
  if constexpr (XT == FMT_BF16) {
    out[0] = r.a[0];
  } else {
    constexpr int P = XT == FMT_F32 ? 3 : 2;
    uint32_t w[XT == FMT_F32 ? 8 : 4], h[8][P];
    memcpy(w, &r, sizeof w);
#pragma unroll
    for (int j = 0; j < 8; j++)
      planes_of<P>(XT == FMT_F32 ? __uint_as_float(w[j]) : hw_half((uint16_t)(w[j / 2] >> (16 * (j & 1)))), h[j]);
#pragma unroll
    for (int pl = 0; pl < P; pl++)
      out[pl] = make_uint4(high_halves(h[0][pl], h[1][pl]), high_halves(h[2][pl], h[3][pl]), high_halves(h[4][pl], h[5][pl]),
                           high_halves(h[6][pl], h[7][pl]));
  }
}

// The few-row kernel's X in LDS: for each column chunk and virtual column v,
// the chunk's values in 16-byte pieces, piece c at a place that depends on v,
// so that the 16 columns' reads of one piece hit distinct banks.
template <int WF>
__device__ __forceinline__ int few_x_at(int v, int c) {
  return WF == FMT_MXFP4 ? v * 256 + ((c ^ (v & 15)) << 4) : v * 128 + ((c ^ ((v >> 1) & 7)) << 4);
}
}  // namespace tinyoai_mx
