// MXFP4 rows: quantisation, the values that the codes stand for, and the
// placing of GGUF matrices into the tiles of mx.h.
//
// Quantisation of a block of 32 values x: with a = max |x|, the scale is 2^e,
// e = floor(log2 a) - 2 (2 is the exponent of 6, the largest code) within
// [-127, 127], and each code is x / 2^e rounded to the nearest, halfway cases
// to the code with a zero fraction bit, at most 6. A block of zeros takes e =
// -127; a block with an infinity or NaN takes the NaN scale and zero codes.
//
// What bounds it: HBM (each value read once, 17 bytes written for 32 of
// them). Eight values a lane: four lanes hold a block, whose largest
// magnitude they exchange by two lane moves; sixteen a row's 128 columns, and
// a wave four rows', which lie together in the codes. 8192 bf16 rows of 6912
// columns to MXFP4 and back: 54 us, 286 MB at 5.3 TB/s (a copy: 4.6).
#include <type_traits>

#include "mx.h"

namespace {

constexpr int kT = 256;

// Eight values of a row.
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

// An item: eight values of a row's 128 columns `unit` (zeros past cols).
template <int D>
__global__ __launch_bounds__(kT) void quantize_kernel(const void *x, int64_t ldx, int64_t n, int64_t cols, uint32_t *codes,
                                                      uint32_t *scales) {
  const int64_t unit = blockIdx.y, first = unit * n * 16;
  // (the 16 lanes of a row stay together: their number is a multiple of 16)
  for (int64_t i = blockIdx.x * (int64_t)kT + threadIdx.x; i < n * 16; i += (int64_t)gridDim.x * kT) {
    const int64_t c = unit * 128 + (i & 15) * 8;
    float v[8] = {};
    if (c < cols) load8<D>(x, (i >> 4) * ldx + c, v);
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
    most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0xb1, 0xf, 0xf, false));  // lanes 1, 0, 3, 2
    most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0x4e, 0xf, 0xf, false));  // lanes 2, 3, 0, 1
    const bool bad = most >= 0x7f800000u;
    // the scale byte: the largest's exponent field less 2, 0 (2^-127) at least
    const uint32_t s = bad ? 255u : max((int)(most >> 23) - 2, 0);
    // (the conversion takes the scale's exponent alone; nearest, ties to even, at most 6)
    const float scale = __uint_as_float(s << 23);
    uint32_t word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], scale, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], scale, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], scale, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], scale, 3);
    codes[first + i] = bad ? 0u : word;
    // lane 0 of 16 writes the word of four blocks' scales
    const uint32_t s1 = __shfl(s, (threadIdx.x & 48) + 4), s2 = __shfl(s, (threadIdx.x & 48) + 8),
                   s3 = __shfl(s, (threadIdx.x & 48) + 12);
    if ((i & 15) == 0) scales[(first + i) >> 4] = s | s1 << 8 | s2 << 16 | s3 << 24;
  }
}

template <int D>
__global__ __launch_bounds__(kT) void dequantize_kernel(const uint32_t *codes, const uint8_t *scales, int64_t n,
                                                        int64_t cols, void *out, int64_t ldo) {
  const int64_t unit = blockIdx.y, first = unit * n * 16;
  for (int64_t i = blockIdx.x * (int64_t)kT + threadIdx.x; i < n * 16; i += (int64_t)gridDim.x * kT) {
    const int64_t c = unit * 128 + (i & 15) * 8;
    if (c >= cols) continue;
    const uint32_t word = codes[first + i];
    const float s = mx_scale(scales[(first + i) >> 2]);
    float v[8];
    auto two = [&](auto sel) {
      const auto w = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.f, decltype(sel)::value);
      v[2 * decltype(sel)::value] = w[0] * s;
      v[2 * decltype(sel)::value + 1] = w[1] * s;
    };
    two(std::integral_constant<int, 0>());
    two(std::integral_constant<int, 1>());
    two(std::integral_constant<int, 2>());
    two(std::integral_constant<int, 3>());
    const int64_t o = (i >> 4) * ldo + c;
    if constexpr (D == FMT_F32) {
      f32x4_any *p = reinterpret_cast<f32x4_any *>(static_cast<float *>(out) + o);
      p[0] = f32x4_any{v[0], v[1], v[2], v[3]};
      p[1] = f32x4_any{v[4], v[5], v[6], v[7]};
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; j++) w[j] = mx_narrow(D, v[2 * j]) | (uint32_t)mx_narrow(D, v[2 * j + 1]) << 16;
      *reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(out) + o) = u32x4_any{w[0], w[1], w[2], w[3]};
    }
  }
}

// GGUF rows -> tiles. MXFP4 blocks are {scale, 16 bytes}, byte j the codes of
// values j (low) and j + 16; BF16 rows are plain values.
__global__ __launch_bounds__(kT) void place_mxfp4_kernel(MxMat m, uint8_t *codes, uint8_t *scales, const uint8_t *raw,
                                                         int phase, uint32_t *any) {
  const int64_t nb = m.cols / 32, total = m.rows * nb;
  for (int64_t i = blockIdx.x * (int64_t)kT + threadIdx.x; i < total; i += (int64_t)gridDim.x * kT) {
    const int row = mx_stored_row(m, (int)(i / nb), phase), col = (int)(i % nb) * 32;
    const uint8_t *src = raw + i * 17;
    uint8_t *dst = codes + mx_code_at(m, row, col);
    for (int j = 0; j < 8; j++) {
      const uint32_t a = src[1 + 2 * j], b = src[2 + 2 * j];
      dst[j] = (uint8_t)((a & 15) | (b & 15) << 4);
      dst[j + 8] = (uint8_t)((a >> 4) | (b >> 4) << 4);
    }
    scales[mx_scale_at(m, row, col)] = src[0];
    if (mx_infinite(src)) *any = 1;
  }
}
__global__ __launch_bounds__(kT) void place_bf16_kernel(MxMat m, uint8_t *codes, const uint16_t *raw, int phase, uint32_t *any) {
  const int64_t total = (int64_t)m.rows * m.cols;
  for (int64_t i = blockIdx.x * (int64_t)kT + threadIdx.x; i < total; i += (int64_t)gridDim.x * kT) {
    const int row = mx_stored_row(m, (int)(i / m.cols), phase), col = (int)(i % m.cols);
    *reinterpret_cast<uint16_t *>(codes + mx_code_at(m, row, col)) = raw[i];
    if (mx_infinite(raw[i])) *any = 1;
  }
}

__global__ __launch_bounds__(kT) void read_kernel(MxMat m, int64_t offset, int64_t n, float *out) {
  for (int64_t i = blockIdx.x * (int64_t)kT + threadIdx.x; i < n; i += (int64_t)gridDim.x * kT) {
    const int64_t e = offset + i;
    out[i] = mx_value(m, 0, (int)(e / m.cols), (int)(e % m.cols));
  }
}

int blocks_for(int64_t items) { return (int)std::max<int64_t>(1, std::min<int64_t>((items + kT - 1) / kT, 16384)); }
// A 128-column unit of all rows for each y (2^15 at most).
dim3 grid_for(int64_t n, int64_t cols) {
  return dim3((unsigned)std::min<int64_t>((n * 16 + kT - 1) / kT, 1 << 20), (unsigned)((cols + 127) / 128));
}

}  // namespace

hipError_t launch_mx_quantize(int dtype, const void *x, int64_t ldx, int64_t n, int64_t cols, uint8_t *codes,
                              uint8_t *scales, hipStream_t st) {
  const dim3 grid = grid_for(n, cols);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kT), 0, st, x, ldx, n, cols, reinterpret_cast<uint32_t *>(codes),
                       reinterpret_cast<uint32_t *>(scales));
  };
  if (dtype == FMT_F32) go(quantize_kernel<FMT_F32>);
  else if (dtype == FMT_F16) go(quantize_kernel<FMT_F16>);
  else go(quantize_kernel<FMT_BF16>);
  return hipGetLastError();
}

hipError_t launch_mx_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t n, int64_t cols, int dtype, void *out,
                                int64_t ldo, hipStream_t st) {
  const dim3 grid = grid_for(n, cols);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kT), 0, st, reinterpret_cast<const uint32_t *>(codes), scales, n, cols, out,
                       ldo);
  };
  if (dtype == FMT_F32) go(dequantize_kernel<FMT_F32>);
  else if (dtype == FMT_F16) go(dequantize_kernel<FMT_F16>);
  else go(dequantize_kernel<FMT_BF16>);
  return hipGetLastError();
}

hipError_t launch_mx_place(const MxMat &m, const uint8_t *raw, int expert, int phase, uint32_t *any, hipStream_t st) {
  uint8_t *codes = const_cast<uint8_t *>(m.codes) + expert * mx_code_bytes(m);
  uint8_t *scales = const_cast<uint8_t *>(m.scales) + expert * mx_scale_bytes(m);
  if (m.fmt == FMT_MXFP4)
    hipLaunchKernelGGL(place_mxfp4_kernel, dim3(blocks_for((int64_t)m.rows * m.cols / 32)), dim3(kT), 0, st, m, codes,
                       scales, raw, phase, any);
  else
    hipLaunchKernelGGL(place_bf16_kernel, dim3(blocks_for((int64_t)m.rows * m.cols)), dim3(kT), 0, st, m, codes,
                       reinterpret_cast<const uint16_t *>(raw), phase, any);
  return hipGetLastError();
}

hipError_t launch_mx_read(const MxMat &m, int64_t offset, int64_t n, float *out, hipStream_t st) {
  hipLaunchKernelGGL(read_kernel, dim3(blocks_for(n)), dim3(kT), 0, st, m, offset, n, out);
  return hipGetLastError();
}
