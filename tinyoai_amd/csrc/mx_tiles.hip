// Products of many rows with expert matrices (mx.h) on LDS tiles.
//
// A block forms BM rows of one group times BN stored matrix rows; both
// operands go straight to LDS (buffer loads to LDS, rows picked by the index
// on the way), a ring of stages ahead of the products, and each wave holds MF x
// NF tiles of 32 x 32 sums. The matrix is the first operand, so a lane ends with
// four runs of four outputs of a row, and of a pair with both halves; the sums
// go through LDS so that whole rows of a wave's outputs are stored together
// (as they are, a store would take 16-byte pieces of 32 rows). (16 x 16 sums
// reach the same rate on paper; a wave alone on its SIMD kept them at half of it,
// these at 0.9.)
//
// What bounds it, by measurement: 1999 fp32 rows times 6912 x 2560 MXFP4, 181 us,
// the matrix cores, busy 78% of the time (212 GFLOP of plane products, 1.17
// PFLOP/s; a large library bf16 product reaches 1.22). 8192 MXFP4 rows times 13824
// x 2560, 200 us, 2.9 PFLOP/s: cores busy 40%; the 453 MB of fp32 outputs alone
// take 66 us at the rate of a fill, and only the CU's other block hides them
// (one 256 x 256 block a CU of the same wave tiles 235 us, of larger ones 258).
// 16384 MXFP4 rows of 64 experts' pairs, 1728 x 2560, 145 us: cores busy 33%, groups'
// last row tiles and the gate on top. 4096 bf16 rows, 8 BF16 experts of 2560 x
// 1728, 48 us: cores busy 60%, 0.76 PFLOP/s, one round of 160 blocks for 256 CUs.
//
// Long rows: the sums of runs of columns go to totals (RUNS; mx_rule.h).
//
//   planes of X (1, 2 or 3, bf16; mx_tile.h) times BF16, or times MXFP4 codes
//   that become bf16 times their scale as a wave reads them (exact): 64
//   columns a step, four v_mfma_f32_32x32x16_bf16. Lane (row, h) takes columns
//   32 b + 16 h + 8 t .. + 7 of its row for product 2 b + t;
//   MXFP4 times MXFP4: 128 columns a step, two
//   v_mfma_scale_f32_32x32x64_f8f6f4; lane (row, h) takes block 2 j + h for
//   product j.
//
// X rows in LDS: the step's 16-byte pieces of a row, piece c at a place that
// depends on the row, so that 16 rows' reads of one piece hit distinct banks.
//
// Groups: the row tiles of all groups are numbered in a row; a wave finds its
// tile's group from the offsets, 64 experts at a time by lane moves. Tiles go
// to the XCDs in runs of bands, kBand row tiles by all matrix tiles, so that
// the blocks that run together on an XCD share both operands through its L2.
#include <algorithm>

#include "mx_tile.h"

namespace {

using namespace tinyoai_mx;
using namespace tinyoai_rule;

constexpr int kBand = 8;
// Offsets within a buffer are below 2^31; kNone and what is added to it, and
// kPast and what it is added to, are past it. (Their sum is 0: the load takes
// the buffer's first bytes, for a step that is not multiplied.)
constexpr uint32_t kNone = 0x80000000u, kPast = 0x80000000u;
constexpr int64_t kExtent = (int64_t)1 << 31;

struct TileArgs {
  MxProduct p;
  int ks;                  // parts of the columns; part i's sums go to p.out + i * part_stride
  int64_t part_stride;
  const uint16_t *planes;  // XM > 0: bf16 planes of X, plane_stride values apart, rows of ldp values
  int64_t plane_stride;
  int64_t ldp;
  const int32_t *index;    // X's row in `planes` (MXFP4: in x) of each output row; null: rows as they come
};

template <int WF, int XM, int BM, int BN, int WAVES>
struct Shape {
  static constexpr bool Q = XM == 0;
  static constexpr int P = Q ? 1 : XM;
  static constexpr int kCols = Q ? 128 : 64;                                     // columns of a step
  static constexpr int kX = BM * (Q ? 64 : 128);                                 // bytes of a plane
  static constexpr int kXS = !Q ? 0 : BM < 64 ? 256 : BM * 4;                    // of the scale words
  static constexpr int kW = BN / 16 * (Q ? 1024 : WF == FMT_BF16 ? 2048 : 512);  // of the codes
  static constexpr int kWS = WF == FMT_MXFP4 ? BN / 64 * 256 : 0;
  static constexpr int kStage = P * kX + kXS + kW + kWS;
  // A step's loads of 1 KB, and how many of them a wave makes (every wave the
  // same number: where there are fewer, some repeat others')
  static constexpr int LX = kX / 1024, LW = kW / 1024, LXS = kXS / 256, LWS = BN / 64;
  static constexpr int NX = (LX + WAVES - 1) / WAVES, NXS = Q ? 1 : 0, NW = (LW + WAVES - 1) / WAVES, NWS = WF == FMT_MXFP4 ? 1 : 0;
  static constexpr int kLoads = P * NX + NXS + NW + NWS;
  static_assert((LX % WAVES == 0 || WAVES % LX == 0) && (LW % WAVES == 0 || WAVES % LW == 0), "loads of every wave");
  static_assert(BN % 64 == 0 && BN <= 256 && LXS <= WAVES && LWS <= WAVES, "whole scale quads");
};

// This block's group and first row, from its number among all row tiles;
// false: there is no such tile. The tile number comes from the block's place
// in the whole grid, whose size only the offsets give.
template <int BM>
__device__ __forceinline__ bool find_tile(const MxProduct &p, int lane, int ntiles, int block, int &e, int &r0, int &r1, int &nt) {
  auto place = [&](int mtiles, int &mt) {
    const int64_t total = (int64_t)mtiles * ntiles, per = (total + 7) / 8;
    const int64_t t = (block & 7) * per + (block >> 3);
    if ((block >> 3) >= per || t >= total) return false;
    const int64_t band = (int64_t)kBand * ntiles, b = t / band;
    const int wide = min(kBand, mtiles - (int)b * kBand), in = (int)(t - b * band);
    nt = in / wide;
    mt = (int)b * kBand + in - nt * wide;
    return true;
  };
  int mt;
  if (!p.offsets) {
    e = 0;
    if (!place((p.n + BM - 1) / BM, mt)) return false;
    r0 = mt * BM;
    r1 = p.n;
    return true;
  }
  auto tiles_of = [&](int i, int &lo, int &hi) {
    lo = hi = 0;
    if (i < p.w.experts) {
      lo = min(max(p.offsets[i], 0), p.n);
      hi = min(max(p.offsets[i + 1], lo), p.n);
    }
    return (hi - lo + BM - 1) / BM;
  };
  int total = 0, lo, hi;
  for (int b = 0; b < p.w.experts; b += 64) total += tiles_of(b + lane, lo, hi);
#pragma unroll
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
  if (!place(total, mt)) return false;
  for (int b = 0; b < p.w.experts; b += 64) {
    const int n = tiles_of(b + lane, lo, hi);
    int end = n;  // tiles of this lane's expert and the lanes below
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(end, o);
      if (lane >= o) end += v;
    }
    const uint64_t mask = __ballot(mt < end);
    if (mask) {
      const int l = __ffsll((unsigned long long)mask) - 1;
      e = b + l;
      r0 = __shfl(lo, l) + (mt - __shfl(end - n, l)) * BM;
      r1 = __shfl(hi, l);
      return true;
    }
    mt -= __shfl(end, 63);
  }
  return false;
}

template <int WF, int XM, int BM, int BN, int WAVES, int WM, int STAGES, bool RUNS>
__global__ __launch_bounds__(WAVES * 64, WAVES == 4 ? 2 : 1) void tile_kernel(TileArgs g) {
  using S = Shape<WF, XM, BM, BN, WAVES>;
  constexpr bool Q = S::Q;
  constexpr int P = S::P, WN = WAVES / WM, MF = BM / 32 / WM, NF = BN / 32 / WN;
  static_assert(MF * WM * 32 == BM && NF * WN * 32 == BN && (NF % 2 == 0 || NF == 1), "scale quads");
  extern __shared__ __align__(16) uint8_t lds[];
  const MxProduct &p = g.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  const int wm = wave / WN, wn = wave - wm * WN;

  int e, r0, r1, nt;
  if (!find_tile<BM>(p, lane, (p.w.tiles * 16 + BN - 1) / BN, blockIdx.x, e, r0, r1, nt)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  r0 = __builtin_amdgcn_readfirstlane(r0);
  r1 = __builtin_amdgcn_readfirstlane(r1);
  nt = __builtin_amdgcn_readfirstlane(nt);
  const int t0 = nt * (BN / 16), steps = (p.w.cols + S::kCols - 1) / S::kCols;
  // (products cut over the columns take the smallest tiles; the others' range of
  // steps stays plain: 1999 fp32 rows times 6912 x 2560 193 us, 199 otherwise)
  constexpr bool kParts = BM == 32;
  const int part = kParts ? blockIdx.y : 0;
  const int first_step = kParts ? steps * part / g.ks : 0, end_step = kParts ? steps * (part + 1) / g.ks : steps;
  constexpr int CB = WF == FMT_MXFP4 ? 1024 : 2048;
  constexpr int kRun = (Q ? kRunMx : kRunBf16) / S::kCols;  // steps

  // Buffers: X from its first row (no index: from the tile's), the matrix from
  // the block's first tile; past them reads zeros.
  // (MXFP4 rows: a step's columns of all rows lie together, and each step has
  // a buffer of its own)
  const int64_t xrow = g.index ? 0 : r0;
  const int64_t xld = Q ? 64 : g.ldp * 2;  // bytes
  const int64_t xrows = g.index ? p.x_rows : min(BM, r1 - r0);
  __amdgpu_buffer_rsrc_t rx[P];
#pragma unroll
  for (int i = 0; i < P; i++)
    rx[i] = plane_rsrc(reinterpret_cast<const uint8_t *>(g.planes + i * g.plane_stride) + xrow * xld, Q ? 0 : xrows * xld);
  const int gt = mx_group_tiles(p.w, t0), tg = t0 & 15, wtiles = min(BN / 16, gt - tg);
  const __amdgpu_buffer_rsrc_t rw =
      plane_rsrc(p.w.codes + e * mx_code_bytes(p.w) + mx_tile_at(p.w, t0, 0), ((int64_t)(p.w.chunks - 1) * gt + wtiles) * CB);
  const __amdgpu_buffer_rsrc_t rws =
      plane_rsrc(p.w.scales + e * mx_scale_bytes(p.w) + mx_quad_at(p.w, t0, 0),
                 WF == FMT_MXFP4 ? ((int64_t)(p.w.chunks - 1) * (gt / 4) + (wtiles + 3) / 4) * 256 : 0);

  // This lane's offsets at the first step.
  auto source = [&](int row) -> uint32_t {  // of X's row in the buffer, in rows; kNone: no row
    const int r = r0 + row;
    if (row >= BM || r >= r1) return kNone;
    if (!g.index) return (uint32_t)row;
    const int src = g.index[r];
    return src >= 0 && src < p.x_rows ? (uint32_t)src : kNone;
  };
  uint32_t xoff[S::NX], woff[S::NW], xsoff = kNone, wsoff = kNone;
#pragma unroll
  for (int i = 0; i < S::NX; i++) {
    const int row = (wave + WAVES * i) % S::LX * (Q ? 16 : 8) + (Q ? lane >> 2 : lane >> 3);
    const uint32_t piece = Q ? (lane & 3) ^ ((row >> 2) & 3) : (lane & 7) ^ ((row >> 1) & 7);
    const uint32_t src = source(row);
    xoff[i] = src == kNone ? kNone : src * (uint32_t)xld + piece * 16;
  }
  if constexpr (Q) {
    const uint32_t src = source((wave % S::LXS) * 64 + lane);
    xsoff = src == kNone ? kNone : src * 4;
  }
#pragma unroll
  for (int i = 0; i < S::NW; i++) {
    const int piece = (wave + WAVES * i) % S::LW * 64 + lane;  // of 16 bytes
    constexpr int per = Q ? 64 : WF == FMT_BF16 ? 128 : 32;  // pieces of a tile's step
    woff[i] = piece / per < wtiles ? (uint32_t)(piece / per) * CB + (uint32_t)(piece % per) * 16 : kNone;
  }
  if constexpr (WF == FMT_MXFP4)
    if (wave % S::LWS < wtiles / 4) wsoff = (uint32_t)(wave % S::LWS) * 256 + lane * 4;

  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)lds;
  constexpr uint32_t kXS0 = P * S::kX, kW0 = kXS0 + S::kXS, kWS0 = kW0 + S::kW;
  auto issue = [&](int kb, int slot) {
    const bool in = kb < end_step;
    const uint32_t base = lds0 + slot * S::kStage;
    if constexpr (Q) {
      const int64_t first = in ? (int64_t)kb * p.x_rows + xrow : 0;  // row, of the step's
      const auto xc = plane_rsrc(static_cast<const uint8_t *>(p.x) + first * 64, in ? xrows * 64 : 0);
#pragma unroll
      for (int j = 0; j < S::NX; j++) lds_dma16(xc, xoff[j], base + (wave + WAVES * j) % S::LX * 1024);
      lds_dma4(plane_rsrc(p.xscales + first * 4, in ? xrows * 4 : 0), xsoff, base + kXS0 + wave % S::LXS * 256);
    } else {
      const uint32_t kx = in ? (uint32_t)kb * 128 : kPast;
#pragma unroll
      for (int i = 0; i < P; i++)
#pragma unroll
        for (int j = 0; j < S::NX; j++) lds_dma16(rx[i], xoff[j] + kx, base + i * S::kX + (wave + WAVES * j) % S::LX * 1024);
    }
    constexpr bool kHalf = WF == FMT_MXFP4 && !Q;  // a step is half a chunk
    const uint32_t chunk = kHalf ? kb >> 1 : kb;
    const uint32_t kw = in ? chunk * (uint32_t)(gt * CB) + (kHalf ? (kb & 1) * 512 : 0) : kPast;
#pragma unroll
    for (int j = 0; j < S::NW; j++) lds_dma16(rw, woff[j] + kw, base + kW0 + (wave + WAVES * j) % S::LW * 1024);
    if constexpr (WF == FMT_MXFP4)
      lds_dma4(rws, wsoff + (in ? chunk * (uint32_t)(gt * 64) : kPast), base + kWS0 + wave % S::LWS * 256);
  };

  // (a single tile has four sums, added at a run's end: each product would wait
  // for the one before)
  constexpr int NA = MF * NF == 1 ? 4 : 1;
  f32x16 acc[MF][NF], more[NA];
  std::conditional_t<BM == 32, double, float> total[RUNS ? MF : 1][RUNS ? NF : 1][16];
#pragma unroll
  for (int v = 0; v < 16; v++) {
#pragma unroll
    for (int f = 0; f < MF; f++)
#pragma unroll
      for (int n = 0; n < NF; n++) {
        acc[f][n][v] = 0.f;
        if constexpr (RUNS) total[f][n][v] = 0;
      }
#pragma unroll
    for (int a = 0; a < NA; a++) more[a][v] = 0.f;
  }
  auto joined = [&](int f, int n, int v) {
    if constexpr (NA > 1) return (more[0][v] + more[1][v]) + (more[2][v] + more[3][v]);
    else return acc[f][n][v];
  };
  auto end_run = [&] {  // the run's sums to the totals
#pragma unroll
    for (int v = 0; v < 16; v++) {
#pragma unroll
      for (int f = 0; f < MF; f++)
#pragma unroll
        for (int n = 0; n < NF; n++) {
          total[f][n][v] += joined(f, n, v);
          acc[f][n][v] = 0.f;
        }
#pragma unroll
      for (int a = 0; a < NA; a++) more[a][v] = 0.f;
    }
  };
  const int xr = wm * MF * 32 + l32;            // this lane's row of the wave's first row tile
  const int wt = (lane & 31) >> 4, l16 = lane & 15;  // its matrix row: of the pair's tile wt, row l16
  const int mine = 8 * wt + (NF == 1 ? 16 * (wn & 1) : 0);  // where a scale word has the byte of this lane's row in tile 0

  // A step's operands go through registers in two halves, each read from LDS
  // while the products of the half before it run: a wave meets the barrier
  // between them, so neither it nor the reads leave the matrix cores waiting.
  struct Half {
    uint4 x[MF][P][Q ? 1 : 2];
    uint4 w[WF == FMT_BF16 || Q ? NF : 1][Q ? 1 : 2];
    uint2 c[WF == FMT_MXFP4 && !Q ? NF : 1];  // codes
    uint32_t sw[(NF + 1) / 2], sx[Q ? MF : 1];
  };
  auto read = [&](Half &H, int kb, int slot, int b) {
    const uint8_t *st = lds + slot * S::kStage;
#pragma unroll
    for (int f = 0; f < MF; f++) {
      const int row = xr + f * 32;
      if constexpr (Q) {
        H.x[f][0][0] = *reinterpret_cast<const uint4 *>(st + row * 64 + (((2 * b + h) ^ ((row >> 2) & 3)) << 4));
        H.sx[f] = *reinterpret_cast<const uint32_t *>(st + kXS0 + row * 4);
      } else {
#pragma unroll
        for (int i = 0; i < P; i++)
#pragma unroll
          for (int t = 0; t < 2; t++)
            H.x[f][i][t] = *reinterpret_cast<const uint4 *>(st + i * S::kX + row * 128 + (((4 * b + 2 * h + t) ^ ((row >> 1) & 7)) << 4));
      }
    }
#pragma unroll
    for (int n = 0; n < NF; n++) {
      const int tile = (wn * NF + n) * 2 + wt;
      if constexpr (Q)
        H.w[n][0] = *reinterpret_cast<const uint4 *>(st + kW0 + tile * 1024 + (2 * b + h) * 256 + l16 * 16);
      else if constexpr (WF == FMT_BF16)
#pragma unroll
        for (int t = 0; t < 2; t++)
          H.w[n][t] = *reinterpret_cast<const uint4 *>(st + kW0 + tile * 2048 + t * 1024 + ((2 * b + h) * 16 + l16) * 16);
      else
        H.c[n] = *reinterpret_cast<const uint2 *>(st + kW0 + tile * 512 + b * 256 + l16 * 16 + h * 8);
    }
    if constexpr (WF == FMT_MXFP4)
#pragma unroll
      for (int n = 0; n < (NF + 1) / 2; n++)  // the word of four tiles' scales of this row and block
        H.sw[n] = *reinterpret_cast<const uint32_t *>(st + kWS0 + (wn * NF / 2 + n) * 256 +
                                                      ((Q ? 2 * b + h : (kb & 1) * 2 + b) * 16 + l16) * 4);
  };
  auto multiply = [&](const Half &H, auto half) {
    constexpr int b = decltype(half)::value;
    if constexpr (Q) {
#pragma unroll
      for (int n = 0; n < NF; n += 2) {
        const uint32_t sw = H.sw[n / 2] >> mine;  // bytes 0 and 2: the tile of this lane's row of tiles n and n + 1
#pragma unroll
        for (int f = 0; f < MF; f++) {
          const uint32_t sx = H.sx[f] >> (8 * h);  // bytes 0 and 2: blocks h, 2 + h
          f32x16 &to = NA > 1 ? more[b] : acc[f][n];
          to = mfma_mx_32<0, 2 * b>(H.w[n][0], H.x[f][0][0], to, sw, sx);
          if constexpr (NF > 1)
            acc[f][n + 1] = mfma_mx_32<2, 2 * b>(H.w[n + 1][0], H.x[f][0][0], acc[f][n + 1], sw, sx);
        }
      }
    } else {
      uint4 w[NF][2];
#pragma unroll
      for (int n = 0; n < NF; n++) {
        if constexpr (WF == FMT_BF16) {
          w[n][0] = H.w[n][0];
          w[n][1] = H.w[n][1];
        } else {
          // the tile's scale byte in an exponent's place; the conversion takes no other bit
          const uint32_t sw = H.sw[n / 2] >> mine;
          const float sc = __uint_as_float(n & 1 ? sw << 7 : sw << 23);
          w[n][0] = fp4_bf16(H.c[n].x, sc);
          w[n][1] = fp4_bf16(H.c[n].y, sc);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < P; i++)
#pragma unroll
          for (int f = 0; f < MF; f++)
#pragma unroll
            for (int n = 0; n < NF; n++) {
              f32x16 &to = NA > 1 ? more[(t * P + i) % NA] : acc[f][n];
              to = mfma_bf16_32(w[n][t], H.x[f][i][t], to);
            }
    }
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; i++) issue(first_step + i, i);
  wait_vmcnt<S::kLoads *(STAGES - 2)>();
  __syncthreads();
  Half A, B;
  read(A, first_step, 0, 0);
  issue(first_step + STAGES - 1, STAGES - 1);
  for (int kb = first_step, slot = 0; kb < end_step; kb++) {
    const int next = slot + 1 == STAGES ? 0 : slot + 1;
    read(B, kb, slot, 1);
    multiply(A, std::integral_constant<int, 0>());
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<S::kLoads *(STAGES - 2)>();  // this wave's loads of kb + 1 (later steps' may be in flight)
    __syncthreads();                        // every wave's; and all are past their reads of kb
    // (past the last step: zeros. One bf16 plane and BF16 values: the next loads
    // after the reads, 2% faster; otherwise before, 2 to 3%)
    constexpr bool kReadFirst = WF == FMT_BF16 && XM == 1;
    if constexpr (kReadFirst) read(A, kb + 1, next, 0);
    issue(kb + STAGES, slot);
    if constexpr (!kReadFirst) read(A, kb + 1, next, 0);
    multiply(B, std::integral_constant<int, 1>());
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (RUNS)
      if ((kb + 1) % kRun == 0) end_run();
    slot = next;
  }
  if constexpr (RUNS) {
    end_run();
#pragma unroll
    for (int v = 0; v < 16; v++)
#pragma unroll
      for (int f = 0; f < MF; f++)
#pragma unroll
        for (int n = 0; n < NF; n++) acc[f][n][v] = (float)total[f][n][v];
  } else if constexpr (NA > 1) {
#pragma unroll
    for (int v = 0; v < 16; v++) acc[0][0][v] = joined(0, 0, v);
  }
  wait_vmcnt<0>();  // nothing may land in LDS any more
  __syncthreads();

  // Lane: row l32 of row tile f; sum v of tile n is of matrix row 8 (v / 4) +
  // 4 h + v % 4. The wave's outputs of a row tile as rows in its part of LDS,
  // then to memory a whole row's at a time.
  const int C = p.w.gate ? NF * 16 : NF * 32, pitch = C + 4;
  float *outs = reinterpret_cast<float *>(lds) + wave * (32 * (NF * 32 + 4));
  const bool wide = p.odtype == FMT_F32;
  const int V = wide ? 4 : 8, lanes = C / V, at = lane % lanes * V;  // outputs of a lane, lanes of a row
  const int o = (p.w.gate ? (t0 + wn * NF * 2) / 2 : t0 + wn * NF * 2) * 16 + at;
#pragma unroll
  for (int f = 0; f < MF; f++) {
    const int first = r0 + wm * MF * 32 + f * 32;
    if (first >= r1) break;
    bool none = false;  // the index names no row: zeros, whatever the matrix holds
    if (p.index && first + l32 < r1) {
      const int src = p.index[first + l32];
      none = src < 0 || src >= p.x_rows;
    }
    const uint32_t zeros = (uint32_t)__ballot(none);
#pragma unroll
    for (int n = 0; n < NF; n++)
#pragma unroll
      for (int u = 0; u < 4; u++) {
        if (p.w.gate && u >= 2) continue;
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = p.w.gate ? mx_gate(acc[f][n][u * 4 + i], acc[f][n][(u * 4 + i + 8) & 15]) : acc[f][n][u * 4 + i];
        *reinterpret_cast<f32x4 *>(outs + l32 * pitch + n * (p.w.gate ? 16 : 32) + u * 8 + h * 4) = v;
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 4
    for (int i = 0; i < 32; i += 64 / lanes) {
      const int row = i + lane / lanes, r = first + row;
      if (r >= r1 || o >= p.w.rows) continue;
      const bool zero = zeros >> row & 1;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        if (j && wide) continue;
        const f32x4 a = *reinterpret_cast<const f32x4 *>(outs + row * pitch + at + j);
#pragma unroll
        for (int k = 0; k < 4; k++) v[j + k] = zero ? 0.f : a[k];
      }
      const int64_t to = part * g.part_stride + r * p.ldo + o;
      if (o + V <= p.w.rows) {
        if (wide) {
          __builtin_nontemporal_store(f32x4_any{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4_any *>(static_cast<float *>(p.out) + to));
        } else {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; k++) w[k] = mx_narrow(p.odtype, v[2 * k]) | (uint32_t)mx_narrow(p.odtype, v[2 * k + 1]) << 16;
          __builtin_nontemporal_store(u32x4_any{w[0], w[1], w[2], w[3]}, reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(p.out) + to));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (k < V && o + k < p.w.rows) mx_store(p.odtype, p.out, to + k, v[k]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// X's rows (those that the index names, in order) as planes of bf16, columns
// past `cols` zeros up to ldp.
template <int XT>
__global__ __launch_bounds__(256) void planes_kernel(MxProduct p, const int32_t *index, int rows, uint16_t *planes,
                                                     int64_t plane_stride, int64_t ldp) {
  const int64_t per = ldp / 8, total = per * rows;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, c = i - r * per;
    constexpr int P = XT == FMT_F32 ? 3 : XT == FMT_F16 ? 2 : 1;
    const int64_t src = index ? index[r] : r;
    if (src < 0 || src >= p.x_rows) continue;  // (the product's outputs of such a row are zeros)
    uint4 h[P];
    planes8<XT>(load_x8<XT>(p, src, (int)c * 8), h);
#pragma unroll
    for (int j = 0; j < P; j++) *reinterpret_cast<uint4 *>(planes + j * plane_stride + r * ldp + c * 8) = h[j];
  }
}

// The sums of the parts, in order.
__global__ __launch_bounds__(256) void join_kernel(const float *parts, int ks, int64_t values, float *out) {
  const int64_t i = (blockIdx.x * (int64_t)256 + threadIdx.x) * 4;
  if (i >= values) return;
  f32x4_any sum = {0.f, 0.f, 0.f, 0.f};
  if (i + 4 <= values) {
#pragma unroll 8
    for (int k = 0; k < ks; k++) sum += *reinterpret_cast<const f32x4_any *>(parts + k * values + i);
    *reinterpret_cast<f32x4_any *>(out + i) = sum;
  } else {
    for (int64_t j = i; j < values; j++) {
      float s = 0.f;
      for (int k = 0; k < ks; k++) s += parts[k * values + j];
      out[j] = s;
    }
  }
}

int64_t padded_cols(const MxProduct &p) { return (p.w.cols + 63) / 64 * 64; }
// bf16 rows that the tiles can read where they are (of an index, any of them
// from one buffer).
bool direct(const MxProduct &p) {
  return p.xdtype == FMT_BF16 && p.w.cols % 64 == 0 && p.ldx % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 &&
         (p.index ? p.x_rows : 256) * p.ldx * 2 <= kExtent;
}
// Else the planes are of X's rows, or of the rows that the index names where
// those are fewer or X's would not be one buffer.
bool gathered(const MxProduct &p) {
  return p.index && (p.n < p.x_rows || p.x_rows * padded_cols(p) * 2 > kExtent);
}
// (without an index, X may have more rows than are multiplied)
int plane_rows(const MxProduct &p) { return !p.index || gathered(p) ? p.n : p.x_rows; }

template <int WF, int XM, int BM, int BN, int WAVES, int WM, int STAGES, bool RUNS = false>
hipError_t launch(TileArgs &g, hipStream_t st) {
  using S = Shape<WF, XM, BM, BN, WAVES>;
  const MxProduct &p = g.p;
  constexpr int rows = WAVES * 32 * (BN / (WAVES / WM) + 4) * 4;  // the waves' outputs
  constexpr int bytes = STAGES * S::kStage > rows ? STAGES * S::kStage : rows;
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  const auto kernel = &tile_kernel<WF, XM, BM, BN, WAVES, WM, STAGES, RUNS>;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (attr != hipSuccess) return attr;
  // row tiles there can be: one more for each group than its rows fill
  const int64_t groups = tinyoai_rule::groups(mx_sizes(p));
  const int64_t mtiles = p.offsets ? (p.n + groups * (BM - 1)) / BM : (p.n + BM - 1) / BM;
  const int64_t blocks = (mtiles * ((p.w.tiles * 16 + BN - 1) / BN) + 7) / 8 * 8;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, BM == 32 ? g.ks : 1), dim3(WAVES * 64), bytes, st, g);
  return hipGetLastError();
}

}  // namespace

static int parts_of(const MxProduct &p) {
  return p.odtype == FMT_F32 && p.ldo == p.w.rows ? parts(mx_sizes(p), device_cu_count()) : 1;
}
static size_t planes_bytes(const MxProduct &p) {
  if (p.xdtype == FMT_MXFP4 || direct(p)) return 0;
  return (size_t)mx_planes(p.xdtype) * plane_rows(p) * padded_cols(p) * 2;  // (a multiple of 128)
}

size_t mx_tiles_scratch(const MxProduct &p) {
  const int ks = parts_of(p);
  return planes_bytes(p) + (ks > 1 ? (size_t)ks * p.n * p.w.rows * 4 : 0);
}

// A step's columns of MXFP4 rows are one buffer, as a block's 256 matrix rows
// are (kMxCols columns at most); the threads of a launch number below 2^32, with
// the smallest tiles too.
bool mx_tiles_supported(const MxProduct &p) {
  const int64_t groups = tinyoai_rule::groups(mx_sizes(p));
  return (p.xdtype != FMT_MXFP4 || (int64_t)p.x_rows * 64 <= kExtent) &&
         (p.n + groups * 31) / 32 * (((int64_t)p.w.tiles * 16 + 127) / 128) < (int64_t)1 << 24;
}

hipError_t launch_mx_tiles(const MxProduct &p, void *scratch, hipStream_t st) {
  TileArgs g{p};
  g.index = p.index;
  g.ks = parts_of(p);
  if (g.ks > 1) {
    g.p.out = static_cast<uint8_t *>(scratch) + planes_bytes(p);
    g.part_stride = (int64_t)p.n * p.w.rows;
  }
  if (p.xdtype != FMT_MXFP4) {
    if (direct(p)) {
      g.planes = static_cast<const uint16_t *>(p.x);
      g.ldp = p.ldx;
    } else {
      g.planes = static_cast<const uint16_t *>(scratch);
      g.ldp = padded_cols(p);
      const int rows = plane_rows(p);
      const int32_t *index = gathered(p) ? p.index : nullptr;
      if (index) g.index = nullptr;
      g.plane_stride = rows * g.ldp;
      const int64_t items = rows * g.ldp / 8;
      const dim3 grid((unsigned)std::min<int64_t>((items + 255) / 256, 1 << 16));
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p, index, rows, static_cast<uint16_t *>(scratch), g.plane_stride, g.ldp);
      };
      if (p.xdtype == FMT_F32) go(planes_kernel<FMT_F32>);
      else if (p.xdtype == FMT_F16) go(planes_kernel<FMT_F16>);
      else go(planes_kernel<FMT_BF16>);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  const int planes = p.xdtype == FMT_MXFP4 ? 0 : mx_planes(p.xdtype);
  const Tile t = tile(mx_sizes(p), g.ks, device_cu_count());
  auto go = [&](auto wf, auto xm) {
    constexpr int WF = decltype(wf)::value, XM = decltype(xm)::value;
    constexpr bool B = WF == FMT_BF16, Q = XM == 0;
    if constexpr (B && XM == 1)
      if (t.bm == 256) return launch<WF, XM, 256, 256, 8, 4, 2>(g, st);
    if constexpr (Q)
      if (t.bm == 128) return launch<WF, XM, 128, 256, 4, 2, 3>(g, st);
    auto of = [&](auto runs) {
      constexpr bool R = decltype(runs)::value;
      if constexpr (B)
        if (t.bm == 128) return launch<WF, XM, 128, 256, 8, 2, XM == 1 ? 3 : 2, R>(g, st);
      if (t.bm == 64 && t.bn == 256) return launch<WF, XM, 64, 256, 4, 1, Q ? 3 : 2, R>(g, st);
      if (t.bm == 64) return launch<WF, XM, 64, 128, 4, 2, Q || (XM == 1 && !B) ? 6 : XM == 3 ? 2 : 3, R>(g, st);
      return launch<WF, XM, 32, 128, 4, 1, Q ? 6 : B ? 5 - XM : XM == 1 ? 8 : 4, R>(g, st);
    };
    return t.runs ? of(std::true_type()) : of(std::false_type());
  };
  using std::integral_constant;
  hipError_t e;
  if (p.w.fmt == FMT_BF16) {
    const integral_constant<int, FMT_BF16> wf;
    e = planes == 1   ? go(wf, integral_constant<int, 1>())
        : planes == 2 ? go(wf, integral_constant<int, 2>())
                      : go(wf, integral_constant<int, 3>());
  } else {
    const integral_constant<int, FMT_MXFP4> wf;
    e = planes == 0   ? go(wf, integral_constant<int, 0>())
        : planes == 1 ? go(wf, integral_constant<int, 1>())
        : planes == 2 ? go(wf, integral_constant<int, 2>())
                      : go(wf, integral_constant<int, 3>());
  }
  if (e != hipSuccess || g.ks == 1) return e;
  hipLaunchKernelGGL(join_kernel, dim3((unsigned)((g.part_stride + 1023) / 1024)), dim3(256), 0, st,
                     static_cast<const float *>(g.p.out), g.ks, g.part_stride, static_cast<float *>(p.out));
  return hipGetLastError();
}
