// Products of a few rows with expert matrices (mx.h): one decode step.
//
// y[r][o] = sum over k of x[r][k] w[o][k]. What bounds it: each matrix that
// some row needs is read once from HBM. The waves of a block share the
// columns: a wave holds its columns of X in registers, as operands of the
// matrix cores, and streams its columns of one tile of 16 matrix rows after
// another (pairs: of two), each chunk's registers loaded again for the next
// tile once it is multiplied; a load takes 1 KB of a tile as it is stored. So
// nothing but sums goes through LDS: the waves' parts of a tile meet there.
// (With X in LDS, every wave whole tiles of its own, a block had to stage the
// rows in parts, and eight waves fitted a CU: 16 tokens' gate and up of 32
// experts, 1728 x 2560, took 43 us; now 38, 131 MB at 3.5 TB/s, 31 where the
// matrices were read just before. One fp32 row times 6912 x 2560: 5.6 us, 1.7
// TB/s, most of it the launch's ramp.)
//
// fp32 and fp16 rows keep all their bits: a value is the sum of three (fp16:
// two) bf16 planes, truncations of what is left (exact but for what lies below
// bf16's smallest, 2^-133), and each plane is an operand column of its own, so P
// planes of m rows fill m * P of the 16 columns that v_mfma_f32_16x16x32_bf16
// multiplies anyway; the planes' sums are added at the end. MXFP4 codes times
// their block's scale are exact in bf16 (past its range infinite). MXFP4 rows take v_mfma_scale_f32_16x16x128_f8f6f4, both operands as
// they are stored.
#include <algorithm>

#include "mx_tile.h"

namespace {

using namespace tinyoai_mx;

constexpr uint32_t kNone = 0x80000000u;  // past every buffer

// LDS written by the wave is read by its other lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ uint4 load16(__amdgpu_buffer_rsrc_t r, uint32_t at) {
  const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0);
  return make_uint4(v.x, v.y, v.z, v.w);
}

struct FewArgs {
  MxProduct p;
  int units;  // tiles (pairs: of both) of an expert
  int per;    // units of a block
  int64_t x_bytes;
};

// CT: column tiles (16 operand columns). NC: column chunks of a wave, at most.
template <int WF, int XM, bool GATE, int kWaves, int CT, int NC>
__global__ __launch_bounds__(kWaves * 64) void few_kernel(FewArgs g) {
  constexpr int NT = GATE ? 2 : 1, P = XM == 0 ? 1 : XM, NJ = WF == FMT_MXFP4 ? 4 : 2;
  constexpr int kChunk = mx_cols<WF>();
  constexpr int kRows = 16 * CT / P;            // rows of X at once
  constexpr int kRed = kWaves * NT * CT * 256;  // sums of a unit
  constexpr int kT = kWaves * 64;
  // Units ahead (as many as the registers hold): two of pairs (16 tokens' fp32
  // pairs of 32 experts 34.2 us with one, 31.7 so; of plain ones no gain).
  constexpr int D = NC == 3 && XM != 0 && GATE ? 2 : 1;
  constexpr int kStaged = XM >= 2 ? kWaves * CT * 16 * kChunk / 4 : 0;  // floats; half of each wave's planes of a chunk
  __shared__ __align__(16) float red[2][kRed > kStaged ? kRed : kStaged];
  const MxProduct &p = g.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int e = blockIdx.y, l16 = lane & 15, q = lane >> 4;
  int r_lo = 0, r_hi = p.n;
  if (p.offsets) {
    r_lo = min(max(p.offsets[e], 0), p.n);
    r_hi = min(max(p.offsets[e + 1], r_lo), p.n);
  }
  const int chunks = p.w.chunks, c0 = chunks * wave / kWaves, nc = chunks * (wave + 1) / kWaves - c0;
  const __amdgpu_buffer_rsrc_t rx = plane_rsrc(static_cast<const uint8_t *>(p.x), g.x_bytes);
  const __amdgpu_buffer_rsrc_t rxs = plane_rsrc(p.xscales, XM == 0 ? (int64_t)p.x_rows * chunks * 4 : 0);
  const int u0 = blockIdx.x * g.per, u1 = min(u0 + g.per, g.units);

  // A unit's part of this wave; chunks past it read zeros (an offset past the buffer).
  struct Tile {
    uint4 w[NC][NT][WF == FMT_MXFP4 ? 1 : 2];
    uint32_t s[NC];  // the scale quad's words
  };
  const __amdgpu_buffer_rsrc_t rw = plane_rsrc(p.w.codes + e * mx_code_bytes(p.w), mx_code_bytes(p.w));
  const __amdgpu_buffer_rsrc_t rs = plane_rsrc(p.w.scales + e * mx_scale_bytes(p.w), mx_scale_bytes(p.w));
  auto fetch = [&](Tile &f, int u, int i) {
    const bool real = u < u1 && i < nc;
    const int tile = real ? u * NT : 0, c = real ? c0 + i : 0;
    const uint32_t at = (uint32_t)mx_tile_at(p.w, tile, c), sat = (uint32_t)mx_quad_at(p.w, tile, c);
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int j = 0; j < (WF == FMT_BF16 ? 2 : 1); j++)
        f.w[i][t][j] = load16(rw, real ? at + t * mx_chunk_bytes(WF) + j * 1024 + lane * 16 : kNone);
    if constexpr (WF == FMT_MXFP4)
      f.s[i] = __builtin_amdgcn_raw_buffer_load_b32(rs, real ? (int)(sat + lane * 4) : (int)kNone, 0, 0);
  };

  for (int r0 = r_lo + blockIdx.z * kRows; r0 < r_hi; r0 += gridDim.z * kRows) {
    const int m = min(kRows, r_hi - r0);
    Tile ring[D];
#pragma unroll
    for (int d = 0; d < D; d++)
#pragma unroll
      for (int i = 0; i < NC; i++) fetch(ring[d], u0 + d, i);
    __builtin_amdgcn_sched_barrier(0);
    // X: operand column v = plane * m + row of column tile v / 16; columns
    // past the planes, and rows that the index does not name, are zeros.
    uint4 x[NC][CT][XM == 0 ? 1 : NJ];
    uint32_t xs[XM == 0 ? NC : 1][CT];
    auto source = [&](int r) {  // the row of X, or -1
      const int src = p.index ? p.index[r0 + r] : r0 + r;
      return src < p.x_rows ? src : -1;
    };
    if constexpr (XM <= 1) {  // as they are stored
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
        const int v = ct * 16 + l16, src = v < m ? source(v) : -1;
#pragma unroll
        for (int i = 0; i < NC; i++) {
          const bool in = src >= 0 && i < nc;
          if constexpr (XM == 0) {
            const uint32_t at = (uint32_t)(c0 + i) * (uint32_t)p.x_rows + (uint32_t)src;
            x[i][ct][0] = load16(rx, in ? at * 64 + q * 16 : kNone);
            xs[i][ct] = __builtin_amdgcn_raw_buffer_load_b32(rxs, in ? (int)(at * 4) : (int)kNone, 0, 0);
          } else {
#pragma unroll
            for (int j = 0; j < NJ; j++) {
              const int k = (c0 + i) * kChunk + (NJ * q + j) * 8;
              x[i][ct][j] = load16(rx, in && k < p.w.cols ? (uint32_t)src * (uint32_t)(p.ldx * 2) + k * 2 : kNone);
            }
          }
        }
      }
    } else {
      // The wave's columns of the rows, four values a lane, cut into planes
      // and through its part of LDS into the operand's places.
      constexpr int kQuads = kChunk / 4, kItems = (kRows * kQuads + 63) / 64, kBytes = XM == 3 ? 4 : 2;
      uint8_t *mine = reinterpret_cast<uint8_t *>(red) + wave * (CT * 16 * kChunk * 2);
      uint32_t raw[NC][kItems][XM == 3 ? 4 : 2];
#pragma unroll
      for (int it = 0; it < kItems; it++) {
        const int item = it * 64 + lane, r = item / kQuads, src = r < m ? source(r) : -1;
#pragma unroll
        for (int i = 0; i < NC; i++) {
          const int k = (c0 + i) * kChunk + item % kQuads * 4;
          const uint32_t at = src >= 0 && i < nc && k < p.w.cols ? ((uint32_t)src * (uint32_t)p.ldx + k) * kBytes : kNone;
          if constexpr (XM == 3) {
            const uint4 w = load16(rx, at);
            raw[i][it][0] = w.x, raw[i][it][1] = w.y, raw[i][it][2] = w.z, raw[i][it][3] = w.w;
          } else {
            const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(rx, (int)at, 0, 0);
            raw[i][it][0] = w.x, raw[i][it][1] = w.y;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NC; i++) {
        if (i >= nc) {
#pragma unroll
          for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int j = 0; j < NJ; j++) x[i][ct][j] = make_uint4(0, 0, 0, 0);
          continue;
        }
#pragma unroll
        for (int it = 0; it < kItems; it++) {
          if (it * 64 >= m * kQuads) break;
          const int item = it * 64 + lane, r = item / kQuads, c = item % kQuads;
          uint32_t h[4][P];
#pragma unroll
          for (int j = 0; j < 4; j++)
            planes_of<P>(XM == 3 ? __uint_as_float(raw[i][it][j & (XM == 3 ? 3 : 1)])
                                 : hw_half((uint16_t)(raw[i][it][j / 2] >> (16 * (j & 1)))), h[j]);
          if (r < m)
#pragma unroll
            for (int pl = 0; pl < P; pl++)
              *reinterpret_cast<uint2 *>(mine + few_x_at<WF>(pl * m + r, c / 2) + (c & 1) * 8) =
                  make_uint2(high_halves(h[0][pl], h[1][pl]), high_halves(h[2][pl], h[3][pl]));
        }
        wave_sync();
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
          const int v = ct * 16 + l16;
#pragma unroll
          for (int j = 0; j < NJ; j++) {
            x[i][ct][j] = *reinterpret_cast<const uint4 *>(mine + few_x_at<WF>(v, NJ * q + j));
            if (v >= m * P) x[i][ct][j] = make_uint4(0, 0, 0, 0);
          }
        }
        wave_sync();
      }
      __syncthreads();  // the sums take this LDS
    }
    if constexpr (XM == 0) {
#pragma unroll
      for (int i = 0; i < NC; i++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) xs[i][ct] >>= 8 * q;
    }

    auto unit = [&](Tile &f, int u, int buf) {
      f32x4 acc[NT][CT];
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) acc[t][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NC; i++) {
        if (i >= nc) break;
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t s = f.s[i] >> (8 * ((u * NT) & 3));  // this tile's byte (and the next one's above it)
        if constexpr (XM == 0) {
#pragma unroll
          for (int ct = 0; ct < CT; ct++) {
            acc[0][ct] = mfma_mx<0>(f.w[i][0][0], x[i][ct][0], acc[0][ct], s, xs[i][ct]);
            if constexpr (GATE) acc[1][ct] = mfma_mx<1>(f.w[i][1][0], x[i][ct][0], acc[1][ct], s, xs[i][ct]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < NT; t++) {
            uint4 w[NJ];
            if constexpr (WF == FMT_BF16) {
              w[0] = f.w[i][t][0];
              w[1] = f.w[i][t][1];
            } else {
              // the scale's byte in the exponent's place; the conversion takes no other bit of it
              const float sc = __uint_as_float(t ? s << 15 : s << 23);
              w[0] = fp4_bf16(f.w[i][t][0].x, sc);
              w[1] = fp4_bf16(f.w[i][t][0].y, sc);
              w[2] = fp4_bf16(f.w[i][t][0].z, sc);
              w[3] = fp4_bf16(f.w[i][t][0].w, sc);
            }
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
              for (int ct = 0; ct < CT; ct++) acc[t][ct] = mfma_bf16(w[j], x[i][ct][j], acc[t][ct]);
          }
        }
        fetch(f, u + D, i);
      }
      // [wave][tile][operand column][16 matrix rows]
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
          *reinterpret_cast<f32x4 *>(&red[buf][((wave * NT + t) * CT + ct) * 256 + l16 * 16 + 4 * q]) = acc[t][ct];
    };
    auto finish = [&](int u, int buf) {  // the waves' and planes' sums of the unit
      for (int i = tid; i < m * 16; i += kT) {
        const int o = i & 15, r = i >> 4, out = u * 16 + o;
        if (out >= p.w.rows) continue;
        float v[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
          v[t] = 0.f;
#pragma unroll
          for (int pl = P - 1; pl >= 0; pl--)  // the smallest first
#pragma unroll
            for (int w = 0; w < kWaves; w++) v[t] += red[buf][(w * NT + t) * CT * 256 + (pl * m + r) * 16 + o];
        }
        float y = GATE ? mx_gate(v[0], v[NT - 1]) : v[0];
        if (p.index) {
          const int src = p.index[r0 + r];
          if (src < 0 || src >= p.x_rows) y = 0.f;  // whatever the matrix holds
        }
        mx_store(p.odtype, p.out, (int64_t)(r0 + r) * p.ldo + out, y);
      }
    };
    // (the sums' buffer of two units ago is free once every wave is past the
    // barrier of the unit between)
    for (int u = u0; u < u1; u += D)
#pragma unroll
      for (int d = 0; d < D; d++) {
        if (u + d >= u1) break;
        unit(ring[d], u + d, (u + d) & 1);
        __syncthreads();
        finish(u + d, (u + d) & 1);
      }
    __syncthreads();  // X of the next rows takes the sums' LDS
  }
}

int64_t x_bytes(const MxProduct &p) {
  if (p.xdtype == FMT_MXFP4) return (int64_t)p.x_rows * p.w.chunks * 64;
  return ((int64_t)(p.x_rows - 1) * p.ldx + p.w.cols) * (int64_t)mx_width(p.xdtype);
}

template <int WF, int XM, bool GATE, int kWaves, int CT, int NC>
hipError_t launch(FewArgs &g, hipStream_t st) {
  const MxProduct &p = g.p;
  g.units = (p.w.rows + 15) / 16;
  // A block a CU, each with units of its own (two in turn would both bring X:
  // 6912 x 2560 MXFP4 times an fp32 row 8.9 us instead of 6.0); two with MXFP4
  // rows of groups, which cost little and are uneven (16 tokens' gate and up of
  // 32 experts 21.9 us instead of 23.6).
  const int64_t blocks = (int64_t)device_cu_count() * (XM == 0 && p.offsets ? 2 : 1);
  g.per = (int)std::max<int64_t>(1, (tinyoai_rule::groups(mx_sizes(p)) * g.units + blocks - 1) / blocks);
  // a group's rows past the first kRows have blocks of their own
  const int rows = 16 * CT / (XM == 0 ? 1 : XM);
  const dim3 grid((g.units + g.per - 1) / g.per, p.offsets ? p.w.experts : 1, std::min((p.n + rows - 1) / rows, p.offsets ? 4 : 1));
  hipLaunchKernelGGL((few_kernel<WF, XM, GATE, kWaves, CT, NC>), grid, dim3(kWaves * 64), 0, st, g);
  return hipGetLastError();
}

}  // namespace

// Whether the few-row kernel takes the product: by its sizes (mx_rule.h), and X
// comes in whole 16-byte pieces, and offsets within X and a matrix fit 31 bits.
bool mx_few_supported(const MxProduct &p) {
  const bool pieces = p.xdtype == FMT_MXFP4 || (p.w.cols % 8 == 0 && p.ldx * mx_width(p.xdtype) % 16 == 0 &&
                                                reinterpret_cast<uintptr_t>(p.x) % 16 == 0);
  return pieces && x_bytes(p) < kNone && mx_code_bytes(p.w) < kNone && tinyoai_rule::few_rows(mx_sizes(p));
}

hipError_t launch_mx_few(const MxProduct &p, hipStream_t st) {
  FewArgs g{p};
  g.x_bytes = x_bytes(p);
  const tinyoai_rule::Few form = tinyoai_rule::few_form(mx_sizes(p));
  const bool two = form.column_tiles == 2;
  using std::integral_constant;
  auto go = [&](auto wf, auto xm) {
    constexpr int WF = decltype(wf)::value, XM = decltype(xm)::value;
    auto gated = [&](auto waves, auto ct, auto nc) {
      constexpr int K = decltype(waves)::value, CT = decltype(ct)::value, N = decltype(nc)::value;
      if constexpr (K == 8 || XM == 0)
        if (p.w.gate) return launch<WF, XM, true, K, CT, N>(g, st);
      return launch<WF, XM, false, K, CT, N>(g, st);
    };
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> both;
    const integral_constant<int, 3> three;
    const integral_constant<int, 4> four;
    const integral_constant<int, 8> eight;
    if (form.waves == 16) return gated(integral_constant<int, 16>(), one, four);
    if (form.wave_chunks == 4) return two ? gated(eight, both, four) : gated(eight, one, four);
    return two ? gated(eight, both, three) : gated(eight, one, three);
  };
  const int xm = p.xdtype == FMT_MXFP4 ? 0 : mx_planes(p.xdtype);
  if (p.w.fmt == FMT_MXFP4) {
    const integral_constant<int, FMT_MXFP4> wf;
    return xm == 0   ? go(wf, integral_constant<int, 0>())
           : xm == 1 ? go(wf, integral_constant<int, 1>())
           : xm == 2 ? go(wf, integral_constant<int, 2>())
                     : go(wf, integral_constant<int, 3>());
  }
  const integral_constant<int, FMT_BF16> wf;
  return xm == 1 ? go(wf, integral_constant<int, 1>()) : xm == 2 ? go(wf, integral_constant<int, 2>()) : go(wf, integral_constant<int, 3>());
}
