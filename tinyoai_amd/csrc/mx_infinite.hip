// Rows of expert matrices that hold infinities (bf16 ones, or MXFP4 values past
// fp32's range).
//
// fp32 and fp16 rows are multiplied as planes (mx_tile.h), and an infinity
// times a plane that is zero would make NaN of an infinite output. Such rows
// are few, if there are any: the upload lists them, and once a product has run
// their outputs are formed again, a wave for each, with the values of X as they
// are. (Every one is an infinity or NaN, but for a gate's zero; the order of
// the sum does not matter.) Nothing is launched for other matrices.
#include <algorithm>

#include "mx.h"

namespace {

constexpr int kT = 256;

__global__ __launch_bounds__(kT) void infinite_kernel(int fmt, const uint8_t *raw, int64_t items, int64_t per, uint8_t *flags) {
  for (int64_t i = blockIdx.x * (int64_t)kT + threadIdx.x; i < items; i += (int64_t)gridDim.x * kT)
    if (fmt == FMT_BF16 ? mx_infinite(reinterpret_cast<const uint16_t *>(raw)[i]) : mx_infinite(raw + i * 17)) flags[i / per] = 1;
}

__global__ __launch_bounds__(kT) void infinite_rows_kernel(MxProduct p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = blockIdx.x; i < p.w.infinite_rows; i += gridDim.x) {
    const int e = p.w.infinite[2 * i], o = p.w.infinite[2 * i + 1];
    int r_lo = 0, r_hi = p.n;
    if (p.offsets) {
      r_lo = min(max(p.offsets[e], 0), p.n);
      r_hi = min(max(p.offsets[e + 1], r_lo), p.n);
    }
    for (int64_t r = r_lo + (int64_t)blockIdx.y * (kT / 64) + wave; r < r_hi; r += (int64_t)gridDim.y * (kT / 64)) {
      const int64_t src = p.index ? p.index[r] : r;
      if (src < 0 || src >= p.x_rows) continue;  // (zeros already)
      float sum[2] = {0.f, 0.f};
      for (int phase = 0; phase <= p.w.gate; phase++) {
        const int row = mx_stored_row(p.w, o, phase);
        for (int k = lane; k < p.w.cols; k += 64)
          sum[phase] = fmaf(mx_load(p.xdtype, p.x, src * p.ldx + k), mx_value(p.w, e, row, k), sum[phase]);
        sum[phase] = wave_sum(sum[phase]);
      }
      if (lane == 0) mx_store(p.odtype, p.out, r * p.ldo + o, p.w.gate ? mx_gate(sum[0], sum[1]) : sum[0]);
    }
  }
}

}  // namespace

hipError_t launch_mx_infinite(int fmt, const uint8_t *raw, int64_t rows, int64_t cols, uint8_t *flags, hipStream_t st) {
  const int64_t per = fmt == FMT_MXFP4 ? cols / 32 : cols, items = rows * per;
  const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + kT - 1) / kT, 16384));
  hipLaunchKernelGGL(infinite_kernel, dim3(blocks), dim3(kT), 0, st, fmt, raw, items, per, flags);
  return hipGetLastError();
}

hipError_t launch_mx_infinite_rows(const MxProduct &p, hipStream_t st) {
  const dim3 grid((unsigned)std::min(p.w.infinite_rows, 4096), (unsigned)std::min((p.n + 3) / 4, 64));
  hipLaunchKernelGGL(infinite_rows_kernel, grid, dim3(kT), 0, st, p);
  return hipGetLastError();
}
