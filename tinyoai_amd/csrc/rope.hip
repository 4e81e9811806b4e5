// Rotary positions: pair i of a head turns by a = position * frequency[i],
//   y1 = m (x1 cos a - x2 sin a),  y2 = m (x2 cos a + x1 sin a),
// its values i and i + rot / 2 of the head (half layout) or 2 i and 2 i + 1
// (interleaved); values from rot on are copied. The angle is formed and taken
// into [-pi, pi] in float64 (an fp32 angle of position 100000 is off by 0.004),
// its sine and cosine and the products in fp32.
//
// What bounds it: HBM, each value read and written once. A block takes a few
// rows, so that their angles' sines and cosines, one a thread, serve all of the
// rows' heads. A thread keeps its place within the head (a unit: sixteen values
// of eight pairs in the half layout, eight values in a row in the interleaved
// one, or eight values to copy) and goes through rows and heads, two at a
// time, whose loads start before the first is used (at first before the angles
// are formed). 8192 rows of 40 bf16 heads of 128: 38 us, 168 MB at 4.4 TB/s (a
// copy on this card: 4.9); four at a time 42, one row's loads at a time, with
// divisions for its place, 80.
#include <type_traits>

#include "attend.h"

namespace {

constexpr int kT = 256;

struct Turn {
  float c, s;
};

template <int D, int O, bool INTER>
__global__ __launch_bounds__(kT) void rope_kernel(RopeArgs a, int rows, int heads) {
  constexpr int B = 2;                // units of a thread in flight
  constexpr int P = INTER ? 4 : 8;    // pairs of a unit
  constexpr int L = INTER ? 1 : 2;    // loads of a unit
  __shared__ Turn turn[kT];           // [rows][rot / 2]
  const int half = a.rot / 2, r0 = blockIdx.x * rows, h0 = blockIdx.y * heads;
  const int nr = min(rows, a.n - r0), nh = min(heads, a.heads - h0);
  const int pairs = (half + P - 1) / P, units = pairs + (a.hd - a.rot + 7) / 8;
  const int side = kT / units;        // heads that the block takes side by side
  const int unit = threadIdx.x % units, lane_head = threadIdx.x / units;
  const bool turns = unit < pairs;
  const int first = turns ? unit * P : 0;                            // the unit's first pair
  const int at0 = turns ? INTER ? 2 * first : first : a.rot + (unit - pairs) * 8, at1 = at0 + half;
  // its values at each place, less than eight at the end of a head's part
  const int count = turns ? min(INTER ? 2 * (half - first) : half - first, 8) : min(a.hd - at0, 8);
  const bool whole = count == 8;
  float v[B][L][8];
  // Of the next B (row, heads side by side): where they are, from row `nr` on none.
  int row[B], head[B], next_row = 0, next_head = 0;
  auto load = [&]() {
#pragma unroll
    for (int j = 0; j < B; j++) {
      row[j] = next_row, head[j] = next_head + lane_head;
      next_head += side;
      if (next_head >= nh) next_head = 0, next_row++;
      if (lane_head >= side || head[j] >= nh) head[j] = -1;
      if (row[j] >= nr || head[j] < 0) continue;
      const int64_t from = (r0 + row[j]) * a.ldx + (int64_t)(h0 + head[j]) * a.hd;
      if (whole) {
        load8<D>(a.x, from + at0, v[j][0]);
        if (L == 2 && turns) load8<D>(a.x, from + at1, v[j][L - 1]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          v[j][0][e] = e < count ? mx_load(D, a.x, from + at0 + e) : 0.f;
          if (L == 2) v[j][L - 1][e] = e < count && turns ? mx_load(D, a.x, from + at1 + e) : 0.f;
        }
      }
    }
  };
  load();
  for (int i = threadIdx.x; i < nr * half; i += kT) {
    const double angle = (double)a.positions[r0 + i / half] * a.frequencies[i % half];
    const double whole_turns = rint(angle * 0.15915494309189535);
    const float t = (float)fma(-whole_turns, 2.4492935982947064e-16, fma(-whole_turns, 6.283185307179586, angle));
    float s, c;
    sincosf(t, &s, &c);
    turn[i] = Turn{c * a.magnitude, s * a.magnitude};
  }
  __syncthreads();
  for (;;) {
#pragma unroll
    for (int j = 0; j < B; j++) {
      if (row[j] >= nr || head[j] < 0) continue;
      const int64_t to = (r0 + row[j]) * a.ldo + (int64_t)(h0 + head[j]) * a.hd;
      const Turn *t = turn + row[j] * half + first;
      if (turns) {
#pragma unroll
        for (int p = 0; p < P; p++) {
          float &x1 = INTER ? v[j][0][2 * p % 8] : v[j][0][p], &x2 = INTER ? v[j][0][(2 * p + 1) % 8] : v[j][L - 1][p];
          const Turn w = t[min(p, half - 1 - first)];  // (past the last pair: of no value)
          const float y1 = x1 * w.c - x2 * w.s, y2 = x2 * w.c + x1 * w.s;
          x1 = y1, x2 = y2;
        }
      }
      if (whole) {
        store8<O>(a.out, to + at0, v[j][0]);
        if (L == 2 && turns) store8<O>(a.out, to + at1, v[j][L - 1]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (e < count) {
            mx_store(O, a.out, to + at0 + e, v[j][0][e]);
            if (L == 2 && turns) mx_store(O, a.out, to + at1 + e, v[j][L - 1][e]);
          }
      }
    }
    if (next_row >= nr) break;
    load();
  }
}

}  // namespace

hipError_t launch_rope(const RopeArgs &a, hipStream_t st) {
  // rows a block, while there are blocks for the chip; the heads of few rows over several blocks
  const int rows = std::max(1, std::min({kT / (a.rot / 2), 8, a.n / 1024}));
  const int64_t most = (int64_t)rows << 23;  // a launch's threads number below 2^32
  for (int64_t first = 0; first < a.n; first += most) {
    RopeArgs part = a;
    part.n = (int32_t)std::min<int64_t>(a.n - first, most);
    part.x = static_cast<const char *>(a.x) + first * a.ldx * (int64_t)mx_width(a.dtype);
    part.out = static_cast<char *>(a.out) + first * a.ldo * (int64_t)mx_width(a.out_dtype);
    part.positions += first;
    const int64_t blocks = (part.n + rows - 1) / rows;
    int parts = (int)(1024 / blocks);
    parts = parts < 1 ? 1 : parts > a.heads ? a.heads : parts;
    const int heads = (a.heads + parts - 1) / parts;
    const dim3 grid((unsigned)blocks, (unsigned)((a.heads + heads - 1) / heads));
    for_type(a.dtype, [&](auto d) {
      for_type(a.out_dtype, [&](auto o) {
        constexpr int D = decltype(d)::value, O = decltype(o)::value;
        if (a.interleaved) hipLaunchKernelGGL((rope_kernel<D, O, true>), grid, dim3(kT), 0, st, part, rows, heads);
        else hipLaunchKernelGGL((rope_kernel<D, O, false>), grid, dim3(kT), 0, st, part, rows, heads);
      });
    });
  }
  return hipGetLastError();
}
