// Products of rows with expert matrices (mx.h): the vector-unit kernel.
//
// y[r][o] = sum over k of x[r][k] * w[o][k] in fp32 multiply-adds. A block
// takes 16 rows and 64 outputs of one group, 32 columns at a time through LDS
// as fp32 values; a thread forms four sums (of pairs: eight).
#include "mx.h"

namespace {

constexpr int kRows = 16, kOut = 64, kK = 32, kT = 256;

__device__ __forceinline__ float x_value(const MxProduct &p, int64_t row, int col) {
  if (p.xdtype != FMT_MXFP4) return mx_load(p.xdtype, p.x, row * p.ldx + col);
  const int64_t units = (p.w.cols + 127) / 128;
  const uint32_t byte = static_cast<const uint8_t *>(p.x)[row * units * 64 + col / 2];
  return mx_code((byte >> (4 * (col & 1))) & 15) * mx_scale(p.xscales[row * units * 4 + col / 32]);
}

__global__ __launch_bounds__(kT) void product_kernel(MxProduct p) {
  __shared__ float xs[kRows][kK + 1], ws[2][kOut][kK + 1];
  const int tid = threadIdx.x, o0 = blockIdx.y * kOut;
  // the group and rows of this block's tile
  int tile = blockIdx.x, e = 0, r0 = 0, r1 = p.n;
  if (p.offsets) {
    for (e = 0; e < p.w.experts; e++) {
      r0 = min(max(p.offsets[e], 0), p.n);
      r1 = min(max(p.offsets[e + 1], r0), p.n);
      const int tiles = (r1 - r0 + kRows - 1) / kRows;
      if (tile < tiles) break;
      tile -= tiles;
    }
    if (e == p.w.experts) return;
  }
  r0 += tile * kRows;
  const int tr = tid >> 4, to = (tid & 15) * 4;  // this thread's row and outputs
  float acc[2][4] = {};
  for (int k0 = 0; k0 < p.w.cols; k0 += kK) {
    __syncthreads();
    for (int i = tid; i < kRows * kK; i += kT) {
      const int r = r0 + i / kK, k = k0 + i % kK;
      float v = 0.f;
      if (r < r1 && k < p.w.cols) {
        const int64_t src = p.index ? p.index[r] : r;
        if (src >= 0 && src < p.x_rows) v = x_value(p, src, k);
      }
      xs[i / kK][i % kK] = v;
    }
    for (int phase = 0; phase <= p.w.gate; phase++)
      for (int i = tid; i < kOut * kK; i += kT) {
        const int o = o0 + i / kK, k = k0 + i % kK;
        ws[phase][i / kK][i % kK] = o < p.w.rows && k < p.w.cols ? mx_value(p.w, e, mx_stored_row(p.w, o, phase), k) : 0.f;
      }
    __syncthreads();
    for (int phase = 0; phase <= p.w.gate; phase++)
      for (int k = 0; k < kK; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[phase][j] = fmaf(xs[tr][k], ws[phase][to + j][k], acc[phase][j]);
  }
  const int r = r0 + tr;
  if (r >= r1) return;
  const bool none = p.index && (p.index[r] < 0 || p.index[r] >= p.x_rows);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if (o0 + to + j >= p.w.rows) break;
    float v = p.w.gate ? mx_gate(acc[0][j], acc[1][j]) : acc[0][j];
    if (none) v = 0.f;  // whatever the matrix holds
    mx_store(p.odtype, p.out, r * p.ldo + o0 + to + j, v);
  }
}

}  // namespace

size_t mx_scratch(const MxProduct &p) { return 0; }

hipError_t launch_mx_product(const MxProduct &p, void *scratch, hipStream_t st) {
  if (mx_few_supported(p)) return launch_mx_few(p, st);
  const int tiles = (p.n + kRows - 1) / kRows + (p.offsets ? p.w.experts : 0);
  hipLaunchKernelGGL(product_kernel, dim3(tiles, (p.w.rows + kOut - 1) / kOut), dim3(kT), 0, st, p);
  return hipGetLastError();
}
