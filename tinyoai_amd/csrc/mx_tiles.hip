// Products of many rows with expert matrices (mx.h) on LDS tiles.
//
// A block forms BM rows of one group times BN = 256 stored matrix rows; both
// operands go straight to LDS (buffer loads to LDS, rows picked by the index
// on the way), a ring of stages ahead of the products, and each wave holds MF x
// NF tiles of 16 x 16 sums. What bounds it: the matrix cores. The matrix is
// the first operand, so a lane ends with four consecutive outputs of a row.
//
//   planes of X (1, 2 or 3, bf16; mx_tile.h) times BF16, or times MXFP4 codes
//   that become bf16 times their scale as a wave reads them (exact): 64
//   columns a step, v_mfma_f32_16x16x32_bf16. Lane l of an operand holds the
//   step's columns 16 (l / 16) .. + 15 of its row, eight for each of the two
//   products;
//   MXFP4 times MXFP4: 128 columns a step, one
//   v_mfma_scale_f32_16x16x128_f8f6f4 a tile.
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

constexpr int kT = 256, kBand = 8;
constexpr uint32_t kNone = 0x80000000u, kPast = 0x40000000u;

struct TileArgs {
  MxProduct p;
  const uint16_t *planes;  // XM > 0: bf16 planes of X, plane_stride values apart, rows of ldp values
  int64_t plane_stride;
  int64_t ldp;
  int mtiles;  // row tiles there can be
};

template <int WF, int XM, int BM, int BN>
struct Shape {
  static constexpr bool Q = XM == 0;
  static constexpr int P = Q ? 1 : XM;
  static constexpr int kCols = Q ? 128 : 64;                                     // columns of a step
  static constexpr int kX = BM * (Q ? 64 : 128), kXS = Q ? BM * 4 : 0;           // bytes of a plane, of the scale words
  static constexpr int kW = BN / 16 * (Q ? 1024 : WF == FMT_BF16 ? 2048 : 512);  // of the codes
  static constexpr int kWS = WF == FMT_MXFP4 ? BN / 64 * 256 : 0;
  static constexpr int kStage = P * kX + kXS + kW + kWS;
  // wave loads of a step
  static constexpr int NX = kX / 4096, NXS = Q ? 1 : 0, NW = kW / 4096, NWS = WF == FMT_MXFP4 ? 1 : 0;
  static constexpr int kLoads = P * NX + NXS + NW + NWS;
  static_assert(kX % 4096 == 0 && kW % 4096 == 0 && BN % 64 == 0 && BN <= 256, "whole loads of every wave");
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

template <int WF, int XM, int BM, int BN, int WM, int STAGES>
__global__ __launch_bounds__(kT, 2) void tile_kernel(TileArgs g) {
  using S = Shape<WF, XM, BM, BN>;
  constexpr bool Q = S::Q;
  constexpr int P = S::P, WN = 4 / WM, MF = BM / 16 / WM, NF = BN / 16 / WN;
  static_assert(MF * WM * 16 == BM && NF * WN * 16 == BN && NF % 4 == 0, "whole scale quads a wave");
  extern __shared__ __align__(16) uint8_t lds[];
  const MxProduct &p = g.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, q = lane >> 4;
  const int wm = wave / WN, wn = wave - wm * WN;

  int e, r0, r1, nt;
  if (!find_tile<BM>(p, lane, (p.w.tiles * 16 + BN - 1) / BN, blockIdx.x, e, r0, r1, nt)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  r0 = __builtin_amdgcn_readfirstlane(r0);
  r1 = __builtin_amdgcn_readfirstlane(r1);
  nt = __builtin_amdgcn_readfirstlane(nt);
  const int t0 = nt * (BN / 16), steps = (p.w.cols + S::kCols - 1) / S::kCols;
  constexpr int CB = WF == FMT_MXFP4 ? 1024 : 2048;

  // Buffers: X from its first row (no index: from the tile's), the matrix from
  // the block's first tile; past them reads zeros.
  const int64_t xrow = p.index ? 0 : r0;
  const int64_t xld = Q ? (int64_t)p.w.chunks * 64 : g.ldp * 2;  // bytes
  const int64_t xrows = p.index ? p.x_rows : min(BM, p.x_rows - r0);
  __amdgpu_buffer_rsrc_t rx[P];
#pragma unroll
  for (int i = 0; i < P; i++)
    rx[i] = plane_rsrc(Q ? static_cast<const uint8_t *>(p.x) + xrow * xld
                         : reinterpret_cast<const uint8_t *>(g.planes + i * g.plane_stride) + xrow * xld,
                       xrows * xld);
  const __amdgpu_buffer_rsrc_t rxs = plane_rsrc(Q ? p.xscales + xrow * p.w.chunks * 4 : p.w.codes, Q ? xrows * p.w.chunks * 4 : 0);
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
    if (!p.index) return (uint32_t)row;
    const int src = p.index[r];
    return src >= 0 && src < p.x_rows ? (uint32_t)src : kNone;
  };
  uint32_t xoff[S::NX], woff[S::NW], xsoff = kNone, wsoff = kNone;
#pragma unroll
  for (int i = 0; i < S::NX; i++) {
    const int row = (wave + 4 * i) * (Q ? 16 : 8) + (Q ? lane >> 2 : lane >> 3);
    const uint32_t piece = Q ? (lane & 3) ^ ((row >> 2) & 3) : (lane & 7) ^ ((row >> 1) & 7);
    const uint32_t src = source(row);
    xoff[i] = src == kNone ? kNone : src * (uint32_t)xld + piece * 16;
  }
  if constexpr (Q) {  // (waves past BM / 64 repeat the others' loads)
    const uint32_t src = source((wave % (BM / 64)) * 64 + lane);
    xsoff = src == kNone ? kNone : src * (uint32_t)(p.w.chunks * 4);
  }
#pragma unroll
  for (int i = 0; i < S::NW; i++) {
    const int piece = (wave + 4 * i) * 64 + lane;  // of 16 bytes
    constexpr int per = Q ? 64 : WF == FMT_BF16 ? 128 : 32;  // pieces of a tile's step
    woff[i] = piece / per < wtiles ? (uint32_t)(piece / per) * CB + (uint32_t)(piece % per) * 16 : kNone;
  }
  if constexpr (WF == FMT_MXFP4)
    if (wave % (BN / 64) < wtiles / 4) wsoff = (uint32_t)(wave % (BN / 64)) * 256 + lane * 4;

  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)lds;
  constexpr uint32_t kXS0 = P * S::kX, kW0 = kXS0 + S::kXS, kWS0 = kW0 + S::kW;
  auto issue = [&](int kb, int slot) {
    const bool in = kb < steps;
    const uint32_t base = lds0 + slot * S::kStage, mine = base + wave * 1024;
    const uint32_t kx = in ? (uint32_t)kb * (Q ? 64 : 128) : kPast;
#pragma unroll
    for (int i = 0; i < P; i++)
#pragma unroll
      for (int j = 0; j < S::NX; j++) lds_dma16(rx[i], xoff[j] + kx, mine + i * S::kX + j * 4096);
    if constexpr (Q) lds_dma4(rxs, xsoff + (in ? (uint32_t)kb * 4 : kPast), base + kXS0 + (wave % (BM / 64)) * 256);
    constexpr bool kHalf = WF == FMT_MXFP4 && !Q;  // a step is half a chunk
    const uint32_t chunk = kHalf ? kb >> 1 : kb;
    const uint32_t kw = in ? chunk * (uint32_t)(gt * CB) + (kHalf ? (kb & 1) * 512 : 0) : kPast;
#pragma unroll
    for (int j = 0; j < S::NW; j++) lds_dma16(rw, woff[j] + kw, mine + kW0 + j * 4096);
    if constexpr (WF == FMT_MXFP4)
      lds_dma4(rws, wsoff + (in ? chunk * (uint32_t)(gt * 64) : kPast), base + kWS0 + (wave % (BN / 64)) * 256);
  };

  f32x4 acc[MF][NF];
#pragma unroll
  for (int f = 0; f < MF; f++)
#pragma unroll
    for (int n = 0; n < NF; n++) acc[f][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int xr = wm * MF * 16 + l16;  // this lane's row of the wave's first row tile
  auto compute = [&](int kb, int slot) {
    const uint8_t *st = lds + slot * S::kStage;
    if constexpr (Q) {
      uint4 x[MF];
      uint32_t sx[MF];
#pragma unroll
      for (int f = 0; f < MF; f++) {
        const int row = xr + f * 16;
        x[f] = *reinterpret_cast<const uint4 *>(st + row * 64 + ((q ^ ((row >> 2) & 3)) << 4));
        sx[f] = *reinterpret_cast<const uint32_t *>(st + kXS0 + row * 4) >> (8 * q);
      }
#pragma unroll
      for (int n4 = 0; n4 < NF / 4; n4++) {
        const uint32_t sw = *reinterpret_cast<const uint32_t *>(st + kWS0 + (wn * NF / 4 + n4) * 256 + lane * 4);
        uint4 w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = *reinterpret_cast<const uint4 *>(st + kW0 + (wn * NF + n4 * 4 + i) * 1024 + lane * 16);
#pragma unroll
        for (int f = 0; f < MF; f++) {
          acc[f][n4 * 4 + 0] = mfma_mx<0>(w[0], x[f], acc[f][n4 * 4 + 0], sw, sx[f]);
          acc[f][n4 * 4 + 1] = mfma_mx<1>(w[1], x[f], acc[f][n4 * 4 + 1], sw, sx[f]);
          acc[f][n4 * 4 + 2] = mfma_mx<2>(w[2], x[f], acc[f][n4 * 4 + 2], sw, sx[f]);
          acc[f][n4 * 4 + 3] = mfma_mx<3>(w[3], x[f], acc[f][n4 * 4 + 3], sw, sx[f]);
        }
      }
    } else {
      uint4 w[NF][2];
      if constexpr (WF == FMT_BF16) {
#pragma unroll
        for (int n = 0; n < NF; n++)
#pragma unroll
          for (int j = 0; j < 2; j++) w[n][j] = *reinterpret_cast<const uint4 *>(st + kW0 + (wn * NF + n) * 2048 + j * 1024 + lane * 16);
      } else {
        // lane (row, q): block q / 2 of the step's two, its bytes 8 (q % 2) .. + 7
        const int at = (q >> 1) * 256 + l16 * 16 + (q & 1) * 8;
        const int sl = ((kb & 1) * 2 + (q >> 1)) * 16 + l16;  // where the chunk's scale word of this row and block is
#pragma unroll
        for (int n4 = 0; n4 < NF / 4; n4++) {
          const uint32_t sw = *reinterpret_cast<const uint32_t *>(st + kWS0 + (wn * NF / 4 + n4) * 256 + sl * 4);
          // the tile's scale byte in an exponent's place; the conversion takes no other bit
          const uint32_t sc[4] = {sw << 23, sw << 15, sw << 7, sw >> 1};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint2 c = *reinterpret_cast<const uint2 *>(st + kW0 + (wn * NF + n4 * 4 + i) * 512 + at);
            w[n4 * 4 + i][0] = fp4_bf16(c.x, __uint_as_float(sc[i]));
            w[n4 * 4 + i][1] = fp4_bf16(c.y, __uint_as_float(sc[i]));
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < P; i++) {
          uint4 x[MF];
#pragma unroll
          for (int f = 0; f < MF; f++) {
            const int row = xr + f * 16;
            x[f] = *reinterpret_cast<const uint4 *>(st + i * S::kX + row * 128 + (((2 * q + j) ^ ((row >> 1) & 7)) << 4));
          }
#pragma unroll
          for (int f = 0; f < MF; f++)
#pragma unroll
            for (int n = 0; n < NF; n++) acc[f][n] = mfma_bf16(w[n][j], x[f], acc[f][n]);
        }
    }
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; i++) issue(i, i);
  int slot = 0;
  for (int kb = 0; kb < steps; kb++) {
    wait_vmcnt<S::kLoads *(STAGES - 2)>();  // this wave's loads of kb (later steps' may be in flight)
    __syncthreads();
    issue(kb + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
    compute(kb, slot);
    slot = slot + 1 == STAGES ? 0 : slot + 1;
  }
  wait_vmcnt<0>();  // nothing may land in LDS after the block

  // Lane: row l16 of row tile f, outputs 4 q .. + 3 of tile n.
  const bool vec = p.ldo % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % (p.odtype == FMT_F32 ? 16 : 8) == 0;
#pragma unroll
  for (int f = 0; f < MF; f++) {
    const int r = r0 + xr + f * 16;
    if (r >= r1) continue;
    bool none = false;
    if (p.index) {
      const int src = p.index[r];
      none = src < 0 || src >= p.x_rows;
    }
    const int64_t row = r * p.ldo;
    auto put = [&](int tile, f32x4 v) {
      const int o = tile * 16 + 4 * q;
      if (none) v = f32x4{0.f, 0.f, 0.f, 0.f};  // whatever the matrix holds
      if (vec && o + 3 < p.w.rows) {
        if (p.odtype == FMT_F32)
          *reinterpret_cast<f32x4 *>(static_cast<float *>(p.out) + row + o) = v;
        else
          *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + row + o) =
              make_uint2(mx_narrow(p.odtype, v[0]) | (uint32_t)mx_narrow(p.odtype, v[1]) << 16,
                         mx_narrow(p.odtype, v[2]) | (uint32_t)mx_narrow(p.odtype, v[3]) << 16);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (o + i < p.w.rows) mx_store(p.odtype, p.out, row + o + i, v[i]);
      }
    };
    if (p.w.gate) {
#pragma unroll
      for (int n = 0; n < NF; n += 2) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = mx_gate(acc[f][n][i], acc[f][n + 1][i]);
        put((t0 + wn * NF + n) / 2, v);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NF; n++) put(t0 + wn * NF + n, acc[f][n]);
    }
  }
}

// X's rows as planes of bf16, columns past `cols` zeros up to ldp.
template <int XT>
__global__ __launch_bounds__(256) void planes_kernel(MxProduct p, uint16_t *planes, int64_t plane_stride, int64_t ldp) {
  const int64_t per = ldp / 8, total = per * p.x_rows;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, c = i - r * per;
    constexpr int P = XT == FMT_F32 ? 3 : XT == FMT_F16 ? 2 : 1;
    uint4 h[P];
    planes8<XT>(load_x8<XT>(p, r, (int)c * 8), h);
#pragma unroll
    for (int j = 0; j < P; j++) *reinterpret_cast<uint4 *>(planes + j * plane_stride + r * ldp + c * 8) = h[j];
  }
}

int64_t padded_cols(const MxProduct &p) { return (p.w.cols + 63) / 64 * 64; }
// bf16 rows that the tiles can read where they are.
bool direct(const MxProduct &p) {
  return p.xdtype == FMT_BF16 && p.w.cols % 64 == 0 && p.ldx % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0;
}

template <int WF, int XM, int BM, int BN, int WM, int STAGES>
hipError_t launch(TileArgs &g, hipStream_t st) {
  using S = Shape<WF, XM, BM, BN>;
  const MxProduct &p = g.p;
  constexpr int bytes = STAGES * S::kStage;
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  static bool set = false;
  const auto kernel = &tile_kernel<WF, XM, BM, BN, WM, STAGES>;
  if (!set) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return e;
    set = true;
  }
  // row tiles there can be: one more for each group than its rows fill
  const int64_t groups = p.offsets ? std::min(p.w.experts, p.n) : 1;
  const int64_t mtiles = p.offsets ? (p.n + groups * (BM - 1)) / BM : (p.n + BM - 1) / BM;
  const int64_t blocks = (mtiles * ((p.w.tiles * 16 + BN - 1) / BN) + 7) / 8 * 8;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kT), bytes, st, g);
  return hipGetLastError();
}

}  // namespace

size_t mx_tiles_scratch(const MxProduct &p) {
  if (p.xdtype == FMT_MXFP4 || direct(p)) return 0;
  return (size_t)mx_planes(p.xdtype) * p.x_rows * padded_cols(p) * 2;
}

// Offsets within a buffer stay below 2^31 bytes: X where an index may name any
// of its rows (else the tile's rows alone), a block's 256 matrix rows.
bool mx_tiles_supported(const MxProduct &p) {
  const int64_t ld = p.xdtype == FMT_MXFP4 ? (int64_t)p.w.chunks * 64 : direct(p) ? p.ldx * 2 : padded_cols(p) * 2;
  return (p.index ? p.x_rows : 256) * ld < kPast && (int64_t)p.w.chunks * mx_chunk_bytes(p.w.fmt) * 16 < kPast;
}

hipError_t launch_mx_tiles(const MxProduct &p, void *scratch, hipStream_t st) {
  TileArgs g{p};
  if (p.xdtype != FMT_MXFP4) {
    if (direct(p)) {
      g.planes = static_cast<const uint16_t *>(p.x);
      g.ldp = p.ldx;
    } else {
      g.planes = static_cast<const uint16_t *>(scratch);
      g.ldp = padded_cols(p);
      g.plane_stride = p.x_rows * g.ldp;
      const int64_t items = p.x_rows * g.ldp / 8;
      const dim3 grid((unsigned)std::min<int64_t>((items + 255) / 256, 1 << 16));
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p, static_cast<uint16_t *>(scratch), g.plane_stride, g.ldp);
      };
      if (p.xdtype == FMT_F32) go(planes_kernel<FMT_F32>);
      else if (p.xdtype == FMT_F16) go(planes_kernel<FMT_F16>);
      else go(planes_kernel<FMT_BF16>);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  const int xm = p.xdtype == FMT_MXFP4 ? 0 : mx_planes(p.xdtype);
  if (p.w.fmt == FMT_MXFP4) {
    if (xm == 0) return launch<FMT_MXFP4, 0, 128, 256, 2, 3>(g, st);
    if (xm == 1) return launch<FMT_MXFP4, 1, 128, 256, 2, 3>(g, st);
    if (xm == 2) return launch<FMT_MXFP4, 2, 128, 256, 2, 3>(g, st);
    return launch<FMT_MXFP4, 3, 64, 256, 1, 2>(g, st);
  }
  if (xm == 1) return launch<FMT_BF16, 1, 128, 256, 2, 3>(g, st);
  if (xm == 2) return launch<FMT_BF16, 2, 64, 256, 1, 2>(g, st);
  return launch<FMT_BF16, 3, 64, 256, 1, 2>(g, st);
}
