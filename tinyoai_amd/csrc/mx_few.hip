// Products of a few rows with expert matrices (mx.h): one decode step.
//
// y[r][o] = sum over k of x[r][k] w[o][k]. What bounds it: each matrix that
// some row needs is read once from HBM, so a wave streams 1 KB (BF16: 2 KB) of
// one tile of 16 matrix rows an instruction, in the order of the matrix
// cores' operand, several loads ahead; the rows of X, which every wave of a
// block shares, sit in LDS.
//
// fp32 and fp16 rows keep all their bits: a value is the exact sum of three
// (fp16: two) bf16 planes, truncations of what is left, and each plane is an
// operand column of its own, so P planes of m rows fill m * P of the 16
// columns that v_mfma_f32_16x16x32_bf16 multiplies anyway; the planes' sums
// are added at the end. MXFP4 codes times their block's scale are exact in
// bf16. MXFP4 rows take v_mfma_scale_f32_16x16x128_f8f6f4, both operands as
// they are stored.
#include <algorithm>

#include "mx_tile.h"

namespace {

using namespace tinyoai_mx;

constexpr int kT = 512, kWaves = 8, kCols = 4;  // column tiles: 64 virtual columns
constexpr int kAhead = 4;                       // chunks in flight a wave

struct FewArgs {
  MxProduct p;
  int ksplit, kshift;  // waves that share a unit's columns: 1, 2, 4 or 8; its logarithm
  int units;     // tiles (pairs: of both) of an expert
  int per;       // units of a block, a multiple of kWaves / ksplit
  int seg;       // column chunks in LDS at once
  int rows;      // rows of X at once (rows * planes <= 16 * kCols)
};

// X's bytes in LDS for one chunk of columns and one virtual column.
template <int WF, int XM>
constexpr int chunk_bytes() { return XM == 0 ? 68 : mx_cols<WF>() * 2; }

template <int WF>
struct Raw {
  uint4 w[WF == FMT_MXFP4 ? 1 : 2];
};
template <int WF, int NT>
struct Fetch {
  Raw<WF> t[NT];
  uint32_t s;  // the scale quad's word
};

template <int WF, int XM, bool GATE>
__global__ __launch_bounds__(kT) void few_kernel(FewArgs g) {
  constexpr int NT = GATE ? 2 : 1, P = XM == 0 ? 1 : XM;
  constexpr int kUnitCols = mx_cols<WF>();  // columns of a chunk
  extern __shared__ __align__(16) uint8_t lds[];
  const MxProduct &p = g.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int e = blockIdx.y;
  int r_lo = 0, r_hi = p.n;
  if (p.offsets) {
    r_lo = min(max(p.offsets[e], 0), p.n);
    r_hi = min(max(p.offsets[e + 1], r_lo), p.n);
  }
  const int G = kWaves / g.ksplit, part = wave % g.ksplit, u0 = blockIdx.x * g.per + wave / g.ksplit;
  const int u_end = min((int)(blockIdx.x + 1) * g.per, g.units);
  const int passes = (min(g.per, g.units - (int)blockIdx.x * g.per) + G - 1) / G;  // groups of G units
  const int chunks = p.w.chunks, nseg = (chunks + g.seg - 1) / g.seg;
  const uint8_t *codes = p.w.codes + e * mx_code_bytes(p.w), *scales = p.w.scales + e * mx_scale_bytes(p.w);
  const int l16 = lane & 15, q = lane >> 4;

  for (int r0 = r_lo; r0 < r_hi; r0 += g.rows) {
    const int m = min(g.rows, r_hi - r0), V = m * P, nct = (V + 15) / 16;
    // The wave's chunks of segment sg: [lo, hi), as places in the segment.
    auto range = [&](int sg, int &lo, int &hi) {
      const int n = min(g.seg, chunks - sg * g.seg);
      lo = n * part >> g.kshift;
      hi = n * (part + 1) >> g.kshift;
    };
    // Loads run kAhead chunks ahead of the products, over segments and units.
    // Each run of chunks starts at the ring's first slot; the slots past its
    // end load nothing (a buffer of no bytes).
    int fu = u0, fs = 0, fi, fhi;
    range(0, fi, fhi);
    int fleft = max((fhi - fi + kAhead - 1) / kAhead * kAhead, kAhead);
    auto fetch = [&](Fetch<WF, NT> &f) {
      const bool real = fu < u_end && fi < fhi;
      const int tile = (real ? fu : 0) * NT, c = real ? fs * g.seg + fi : 0;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const __amdgpu_buffer_rsrc_t r =
            plane_rsrc(codes + mx_tile_at(p.w, tile + t, c), real ? mx_chunk_bytes(WF) : 0);
#pragma unroll
        for (int j = 0; j < (WF == FMT_BF16 ? 2 : 1); j++) {
          const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, lane * 16 + j * 1024, 0, 0);
          f.t[t].w[j] = make_uint4(v.x, v.y, v.z, v.w);
        }
      }
      if constexpr (WF == FMT_MXFP4)
        f.s = __builtin_amdgcn_raw_buffer_load_b32(plane_rsrc(scales + mx_quad_at(p.w, tile, c), real ? 256 : 0),
                                                   lane * 4, 0, 0);
      fi++;
      if (--fleft == 0) {
        if (++fs == nseg) fs = 0, fu += G;
        range(fs, fi, fhi);
        fleft = max((fhi - fi + kAhead - 1) / kAhead * kAhead, kAhead);
      }
    };
    Fetch<WF, NT> ring[kAhead];
    auto prime = [&]() {
#pragma unroll
      for (int i = 0; i < kAhead; i++) fetch(ring[i]);
    };

    for (int ps = 0; ps < passes; ps++) {
      const int u = u0 + ps * G;
      f32x4 acc[NT][kCols];
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int c = 0; c < kCols; c++) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int sg = 0; sg < nseg; sg++) {
        if (nseg > 1 || ps == 0) {  // X's columns of the segment into LDS
          __syncthreads();
          const int k0 = sg * g.seg * kUnitCols, count = min(g.seg, chunks - sg * g.seg) * kUnitCols;
          stage_few<WF, XM, kT>(p, lds, r0, m, V, k0, count, g.seg, tid, [&]() {
            if (ps + sg == 0) prime();  // the ring's first loads behind X's
          });
          __syncthreads();
        }
        int lo, hi;
        range(sg, lo, hi);
        const bool mine = u < u_end;
        const int shift = 8 * ((u * NT) & 3);  // this tile's byte of the scale words
        auto consume = [&](const Fetch<WF, NT> &f, int c) {
          const uint32_t fs = f.s >> shift;
          const uint8_t *xs = lds + (size_t)c * V * (XM == 0 ? 64 : kUnitCols * 2);
          if constexpr (XM == 0) {  // both operands MXFP4
            const uint32_t *ss = reinterpret_cast<const uint32_t *>(lds + (size_t)g.seg * V * 64) + c * V;
#pragma unroll
            for (int ct = 0; ct < kCols; ct++) {
              if (ct >= nct) break;
              const int v = min(ct * 16 + l16, V - 1);
              const uint4 x = *reinterpret_cast<const uint4 *>(xs + v * 64 + ((q ^ ((v >> 2) & 3)) << 4));
              const uint32_t sx = ss[v] >> (8 * q);
              acc[0][ct] = mfma_mx<0>(f.t[0].w[0], x, acc[0][ct], fs, sx);
              if constexpr (GATE) acc[1][ct] = mfma_mx<1>(f.t[1].w[0], x, acc[1][ct], fs, sx);
            }
          } else {
            constexpr int NJ = WF == FMT_MXFP4 ? 4 : 2;
            uint4 w[NT][NJ];
#pragma unroll
            for (int t = 0; t < NT; t++) {
              if constexpr (WF == FMT_BF16) {
                w[t][0] = f.t[t].w[0];
                w[t][1] = f.t[t].w[1];
              } else {
                // the scale's byte in the exponent's place; the conversion takes no other bit of it
                const float sc = __uint_as_float(t ? fs << 15 : fs << 23);
                w[t][0] = fp4_bf16(f.t[t].w[0].x, sc);
                w[t][1] = fp4_bf16(f.t[t].w[0].y, sc);
                w[t][2] = fp4_bf16(f.t[t].w[0].z, sc);
                w[t][3] = fp4_bf16(f.t[t].w[0].w, sc);
              }
            }
#pragma unroll
            for (int ct = 0; ct < kCols; ct++) {
              if (ct >= nct) break;
              const int v = min(ct * 16 + l16, V - 1);
#pragma unroll
              for (int j = 0; j < NJ; j++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(xs + few_x_at<WF>(v, NJ * q + j));
#pragma unroll
                for (int t = 0; t < NT; t++) acc[t][ct] = mfma_bf16(w[t][j], x, acc[t][ct]);
              }
            }
          }
        };
        int c = lo;
        do {
#pragma unroll
          for (int i = 0; i < kAhead; i++) {
            if (mine && c + i < hi) consume(ring[i], c + i);
            fetch(ring[i]);
          }
          c += kAhead;
        } while (c < hi);
      }
      // [wave][tile][virtual column][16 matrix rows], in the LDS past X
      float *red = reinterpret_cast<float *>(lds + few_x_bytes<WF, XM>(g.seg, V));
      const int V16 = nct * 16;
      if (ps) __syncthreads();
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int ct = 0; ct < kCols; ct++)
          if (ct < nct)
            *reinterpret_cast<f32x4 *>(red + ((wave * NT + t) * V16 + ct * 16 + l16) * 16 + 4 * q) = acc[t][ct];
      __syncthreads();
      for (int i = tid; i < G * m * 16; i += kT) {
        const int o = i & 15, r = (i >> 4) % m, gu = (i >> 4) / m;
        const int unit = blockIdx.x * g.per + ps * G + gu, out = unit * 16 + o;
        if (unit >= u_end || out >= p.w.rows) continue;
        float v[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
          v[t] = 0.f;
          for (int s = 0; s < g.ksplit; s++)
#pragma unroll
            for (int pl = P - 1; pl >= 0; pl--)  // the smallest first
              v[t] += red[(((gu * g.ksplit + s) * NT + t) * V16 + pl * m + r) * 16 + o];
        }
        float y = GATE ? mx_gate(v[0], v[NT - 1]) : v[0];
        if (p.index) {
          const int src = p.index[r0 + r];
          if (src < 0 || src >= p.x_rows) y = 0.f;
        }
        mx_store(p.odtype, p.out, (int64_t)(r0 + r) * p.ldo + out, y);
      }
    }
    __syncthreads();
  }
}

template <int WF, int XM, bool GATE>
hipError_t launch(FewArgs &g, int active, hipStream_t st) {
  constexpr int P = XM == 0 ? 1 : XM;
  constexpr size_t kLds = 160 * 1024;
  const MxProduct &p = g.p;
  const int cus = device_cu_count();
  g.units = (p.w.rows + 15) / 16;
  // Enough waves for the chip: a unit's columns go to more of them where units are few.
  g.ksplit = 1;
  while (g.ksplit < 8 && (int64_t)active * g.units * g.ksplit < (int64_t)cus * 12 && p.w.chunks >= 2 * g.ksplit) g.ksplit *= 2;
  g.kshift = g.ksplit == 8 ? 3 : g.ksplit / 2;
  const int G = kWaves / g.ksplit;
  const int64_t blocks = (int64_t)active * ((g.units + G - 1) / G);
  const int runs = (int)std::max<int64_t>(1, std::min<int64_t>(blocks / (cus * 2), 16));
  g.per = G * runs;
  const int most = p.offsets ? p.n : std::min(p.n, 16 * kCols / P);
  g.rows = std::min(16 * kCols / P, most);
  const int V = g.rows * P, V16 = (V + 15) / 16 * 16;
  const size_t red = (size_t)kWaves * (GATE ? 2 : 1) * V16 * 64;
  g.seg = p.w.chunks;
  while (few_x_bytes<WF, XM>(g.seg, V) + red > kLds) g.seg = (g.seg + 1) / 2;
  const size_t bytes = few_x_bytes<WF, XM>(g.seg, V) + red;
  static bool set = false;
  if (!set) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&few_kernel<WF, XM, GATE>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds);
    if (e != hipSuccess) return e;
    set = true;
  }
  hipLaunchKernelGGL((few_kernel<WF, XM, GATE>), dim3((g.units + g.per - 1) / g.per, p.offsets ? p.w.experts : 1), dim3(kT),
                     bytes, st, g);
  return hipGetLastError();
}

}  // namespace

// Whether the few-row kernel takes the product: its rows fill no more than
// kCols column tiles.
bool mx_few_supported(const MxProduct &p) {
  const int planes = mx_planes(p.xdtype);
  const int active = p.offsets ? std::min(p.w.experts, p.n) : 1;
  return (int64_t)p.n * planes <= (int64_t)active * 16 * kCols;
}

hipError_t launch_mx_few(const MxProduct &p, hipStream_t st) {
  FewArgs g{p};
  const int active = p.offsets ? std::min(p.w.experts, p.n) : 1;
  auto go = [&](auto wf, auto xm) {
    constexpr int WF = decltype(wf)::value, XM = decltype(xm)::value;
    return p.w.gate ? launch<WF, XM, true>(g, active, st) : launch<WF, XM, false>(g, active, st);
  };
  using std::integral_constant;
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
