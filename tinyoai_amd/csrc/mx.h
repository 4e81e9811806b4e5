// Expert matrices and MXFP4 operands: their layouts in HBM, and the launch
// interfaces of the kernels that make and multiply them.
//
// MXFP4: blocks of 32 values share one scale byte s (the value 2^(s - 127);
// 255: NaN); a code's bits are sign, two exponent bits and one fraction bit:
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives.
//
// Matrices are stored in the order in which the matrix cores take them, so a
// wave's loads are contiguous and need no address arithmetic per lane. Rows
// are cut into tiles of 16, columns into chunks. Sixteen tiles form a group (the
// last one may have fewer, a multiple of four), and a group holds its tiles'
// first chunk, then their second, and so on: what a block of many rows loads
// for a step is contiguous (a tile's chunks one after another put a step's 16
// loads on the same few memory channels). One tile's chunk is
//   MXFP4: 128 columns, 1 KB: lane l's 16 bytes are the codes of row l % 16,
//          columns 32 (l / 16) .. + 31, two a byte, the earlier one low. The
//          scales of four tiles' chunk, in an array of their own and in the
//          same order, are 256 bytes: lane l's word holds tile t's scale of
//          row l % 16 and block l / 16 in byte t;
//   BF16:  64 columns, 2 KB: lane l's 16 bytes of half j are the values of
//          row l % 16, columns 16 (l / 16) + 8 j .. + 7.
// Rows and columns past the matrix hold zeros. Of a (gate, up) pair, the gate
// rows are the even tiles and the up rows the odd ones: one lane then holds
// both halves of four consecutive outputs.
//
// Rows of quantised activations: for each 128 columns, 64 bytes of codes (two
// a byte, the earlier one low) of every row, one row after another, and in an
// array of their own 4 scale bytes of every row; zeros past the last column.
// (What a block loads for a step is contiguous: with whole rows together, loads
// took 64 bytes each from as many lines, and came at 14.5 TB/s instead of 24.6.)
#pragma once

#include "kernels.h"

enum : int32_t { FMT_MXFP4 = 39 };

constexpr int64_t kMxCols = 1 << 22;  // of a matrix or MXFP4 row, at most
constexpr int kMxExperts = 65535;     // (blocks of a grid's second dimension)

struct MxMat {
  const uint8_t *codes, *scales;
  int32_t fmt;              // FMT_MXFP4 or FMT_BF16
  int32_t experts, rows, cols;
  int32_t gate;             // (gate, up) pairs
  int32_t tiles;            // row tiles of an expert, a multiple of four
  int32_t chunks;           // column chunks
  int32_t infinite_rows;    // (expert, output row) with an infinity in the matrix (of a pair, in either)
  const int32_t *infinite;  // [infinite_rows][2]
};

__host__ __device__ inline int mx_chunk_cols(int fmt) { return fmt == FMT_MXFP4 ? 128 : 64; }
__host__ __device__ inline int mx_chunk_bytes(int fmt) { return fmt == FMT_MXFP4 ? 1024 : 2048; }
__host__ __device__ inline int64_t mx_code_bytes(const MxMat &m) {  // of one expert
  return (int64_t)m.tiles * m.chunks * mx_chunk_bytes(m.fmt);
}
__host__ __device__ inline int64_t mx_scale_bytes(const MxMat &m) {
  return m.fmt == FMT_MXFP4 ? (int64_t)m.tiles / 4 * m.chunks * 256 : 0;
}
// Where a tile's chunk begins, and its scale quad's (bytes within an expert).
__host__ __device__ inline int mx_group_tiles(const MxMat &m, int tile) {
  const int left = m.tiles - (tile & ~15);
  return left < 16 ? left : 16;
}
__host__ __device__ inline int64_t mx_tile_at(const MxMat &m, int tile, int chunk) {
  return ((int64_t)(tile >> 4) * 16 * m.chunks + (int64_t)chunk * mx_group_tiles(m, tile) + (tile & 15)) * mx_chunk_bytes(m.fmt);
}
__host__ __device__ inline int64_t mx_quad_at(const MxMat &m, int tile, int chunk) {
  return ((int64_t)(tile >> 4) * 4 * m.chunks + (int64_t)chunk * (mx_group_tiles(m, tile) / 4) + ((tile & 15) >> 2)) * 256;
}
// The byte of value (row of the stored tiles, column) within an expert.
__host__ __device__ inline int64_t mx_code_at(const MxMat &m, int row, int col) {
  const int cc = mx_chunk_cols(m.fmt), k = col % cc;
  const int64_t at = mx_tile_at(m, row >> 4, col / cc);
  if (m.fmt == FMT_MXFP4) return at + ((k >> 5) * 16 + (row & 15)) * 16 + (k & 31) / 2;
  return at + ((k >> 3) & 1) * 1024 + ((k >> 4) * 16 + (row & 15)) * 16 + (k & 7) * 2;
}
__host__ __device__ inline int64_t mx_scale_at(const MxMat &m, int row, int col) {
  return mx_quad_at(m, row >> 4, col / 128) + (((col & 127) >> 5) * 16 + (row & 15)) * 4 + ((row >> 4) & 3);
}
// The stored row of output row `row` (phase 1: its up row).
__host__ __device__ inline int mx_stored_row(const MxMat &m, int row, int phase) {
  return m.gate ? (row >> 4) * 32 + phase * 16 + (row & 15) : row;
}

__device__ __forceinline__ float mx_scale(uint32_t s) {  // 2^(s - 127), 2^-127 a subnormal
  return __uint_as_float(s == 255 ? 0x7fc00000u : s ? s << 23 : 0x00400000u);
}
__device__ __forceinline__ float mx_code(uint32_t c) {
  const uint32_t m = c & 7;
  const float v = m < 2 ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126) << 23 | (m & 1) << 22);
  return c & 8 ? -v : v;
}
// Whether a raw bf16 value, or one of a raw MXFP4 block's, is an infinity in
// fp32: codes 4 and 6 (2 and 4) times 2^127, 6 times 2^126.
__device__ __forceinline__ bool mx_infinite(uint16_t bf16) { return (bf16 & 0x7fff) == 0x7f80; }
__device__ __forceinline__ bool mx_infinite(const uint8_t *block) {
  const uint32_t s = block[0], least = s == 254 ? 4 : 6;
  bool inf = false;
  if (s == 254 || s == 253)
    for (int j = 1; j <= 16; j++) inf |= (block[j] & 7u) >= least || (block[j] >> 4 & 7u) >= least;
  return inf;
}
// Value (row of the stored tiles, column) of expert e.
__device__ __forceinline__ float mx_value(const MxMat &m, int e, int row, int col) {
  const uint8_t *p = m.codes + e * mx_code_bytes(m) + mx_code_at(m, row, col);
  if (m.fmt == FMT_BF16) return bf16_to_float(*reinterpret_cast<const uint16_t *>(p));
  return mx_code((*p >> (4 * (col & 1))) & 15) * mx_scale(m.scales[e * mx_scale_bytes(m) + mx_scale_at(m, row, col)]);
}

__device__ __forceinline__ float mx_load(int dtype, const void *p, int64_t i) {
  if (dtype == FMT_F32) return static_cast<const float *>(p)[i];
  const uint16_t h = static_cast<const uint16_t *>(p)[i];
  return dtype == FMT_F16 ? hw_half(h) : bf16_to_float(h);
}
__device__ __forceinline__ uint16_t mx_narrow(int dtype, float v) {  // to the nearest, ties to even
  return dtype == FMT_F16 ? __half_as_ushort(__float2half_rn(v)) : __builtin_bit_cast(uint16_t, (__bf16)v);
}
__device__ __forceinline__ void mx_store(int dtype, void *p, int64_t i, float v) {
  if (dtype == FMT_F32) static_cast<float *>(p)[i] = v;
  else static_cast<uint16_t *>(p)[i] = mx_narrow(dtype, v);
}
// g / (1 + e^-g) * u (stablelm.go:371-373), off by ten half-units in the last
// place at most where the gate is a normal number: e^x is 2^t (1 + r ln 2), t the rounded x log2 e
// and r what it lacks, by the hardware's 2^t and reciprocal, one unit each (64
// experts' pairs times 16384 MXFP4 rows, K = 2560, 167 us with expf and a
// division, 155 so). The hardware's reciprocal is zero where it would be
// subnormal, from 1 + e^x = 2^126 on: past t = 64 both terms are taken 2^-64
// times as large, and the quotient with them. |x| is held at 200, where that
// e^x is infinite or zero too.
__device__ __forceinline__ float mx_gate(float g, float u) {
  const float x = fminf(fmaxf(-g, -200.f), 200.f), t = x * 1.44269502f;
  const float r = fmaf(x, 1.92596303e-8f, fmaf(x, 1.44269502f, -t));  // log2 e = 1.44269502 + 1.93e-8
  const bool far = t > 64.f;
  const float one = far ? 0x1p-64f : 1.f;
  const float e = __builtin_amdgcn_exp2f(far ? t - 64.f : t);
  return g * __builtin_amdgcn_rcpf(fmaf(e, fmaf(r, 0.693147182f, 1.f), one)) * one * u;
}

// Sixteen (eight) bytes at an address of a value's alignment alone: the card
// loads and stores them as it does aligned ones, so rows of any length move in
// whole pieces (the sum of 8192 tokens' 4 bf16 rows of 2563 columns 41 us, 104
// value by value; 1322 x 7237 fp32 outputs of an MXFP4 product, K = 1024, 25 and 34).
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

__host__ __device__ inline size_t mx_width(int dtype) { return dtype == FMT_F32 ? 4 : 2; }

// out[r] = x[index ? index[r] : r] * W[e]^T for the rows r of [offsets[e],
// offsets[e + 1]) (clamped to [0, n)), for every expert e; offsets null: all
// n rows with the one matrix. An index outside [0, x_rows) gives a row of
// zeros. Rows of no group stay as they are.
struct MxProduct {
  MxMat w;
  int32_t xdtype;           // FMT_F32, FMT_F16, FMT_BF16, or FMT_MXFP4 (x: code rows, xscales: scale rows)
  const void *x;
  const uint8_t *xscales;
  int64_t ldx;              // values (not for FMT_MXFP4)
  int32_t x_rows;
  const int32_t *offsets, *index;
  int32_t n;
  int32_t odtype;
  void *out;
  int64_t ldo;
};

// Rows of one expert's GGUF tensor (raw, on the device) into its tiles; phase
// 1: the up rows of pairs. *any becomes 1 if one of its values is an infinity.
hipError_t launch_mx_place(const MxMat &m, const uint8_t *raw, int expert, int phase, uint32_t *any, hipStream_t st);
// flags[row] = 1 for the rows of a raw matrix with an infinity.
hipError_t launch_mx_infinite(int fmt, const uint8_t *raw, int64_t rows, int64_t cols, uint8_t *flags, hipStream_t st);
// The outputs of the rows p.w.infinite, after the product of fp32 or fp16 rows.
hipError_t launch_mx_infinite_rows(const MxProduct &p, hipStream_t st);
// Values [offset, offset + n) of a single matrix, row-major.
hipError_t launch_mx_read(const MxMat &m, int64_t offset, int64_t n, float *out, hipStream_t st);
hipError_t launch_mx_quantize(int dtype, const void *x, int64_t ldx, int64_t n, int64_t cols, uint8_t *codes,
                              uint8_t *scales, hipStream_t st);
hipError_t launch_mx_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t n, int64_t cols, int dtype, void *out,
                                int64_t ldo, hipStream_t st);
// The product, with mx_scratch bytes of scratch; mx_supported: within what the
// kernels address.
bool mx_supported(const MxProduct &p);
size_t mx_scratch(const MxProduct &p);
hipError_t launch_mx_product(const MxProduct &p, void *scratch, hipStream_t st);
// A few rows (or a few for each expert) on the streaming kernel.
bool mx_few_supported(const MxProduct &p);
hipError_t launch_mx_few(const MxProduct &p, hipStream_t st);
// Many rows on LDS tiles.
bool mx_tiles_supported(const MxProduct &p);
size_t mx_tiles_scratch(const MxProduct &p);
hipError_t launch_mx_tiles(const MxProduct &p, void *scratch, hipStream_t st);

struct RouteArgs {
  int32_t dtype;
  const void *logits;
  int64_t ld;
  int32_t n, experts, k, over_all;
  int32_t *ids;
  float *weights;
  int32_t *offsets, *tokens, *positions;
};
constexpr int kRouteExperts = 1024, kRouteMost = 32;
hipError_t launch_route(const RouteArgs &a, hipStream_t st);

struct CombineArgs {
  int32_t dtype;
  const void *y;
  int64_t ldy;
  int32_t y_rows;
  const int32_t *positions;
  const float *weights;
  int32_t n, k;
  int64_t cols;
  int32_t odtype;
  void *out;
  int64_t ldo;
};
hipError_t launch_combine(const CombineArgs &a, hipStream_t st);
