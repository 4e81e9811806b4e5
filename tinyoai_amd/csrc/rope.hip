// Rotary positions: pair i of a head turns by a = position * frequency[i],
//   y1 = m (x1 cos a - x2 sin a),  y2 = m (x2 cos a + x1 sin a),
// its values i and i + rot / 2 of the head (half layout) or 2 i and 2 i + 1
// (interleaved); values from rot on are copied. The angle is formed and taken
// into [-pi, pi] in float64 (an fp32 angle of position 100000 is off by 0.004),
// its sine and cosine and the products in fp32.
//
// What bounds it: HBM, each value read and written once. A block takes a few
// rows, so that their angles' sines and cosines, one a thread, serve all of the
// rows' heads; a thread then takes eight pairs of a head at a time (both
// halves, so a row may be turned in place).
#include <type_traits>

#include "attend.h"

namespace {

constexpr int kT = 256;

struct Turn {
  float c, s;
};

template <int D, int O>
__global__ __launch_bounds__(kT) void rope_kernel(RopeArgs a, int rows, int heads) {
  __shared__ Turn turn[kT];  // [rows][rot / 2]
  const int half = a.rot / 2, r0 = blockIdx.x * rows, h0 = blockIdx.y * heads;
  const int nr = min(rows, a.n - r0), nh = min(heads, a.heads - h0);
  for (int i = threadIdx.x; i < nr * half; i += kT) {
    const double angle = (double)a.positions[r0 + i / half] * a.frequencies[i % half];
    const double turns = rint(angle * 0.15915494309189535);
    const float t = (float)fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, angle));
    float s, c;
    sincosf(t, &s, &c);
    turn[i] = Turn{c * a.magnitude, s * a.magnitude};
  }
  __syncthreads();
  const int pairs = (half + 7) / 8, rest = (a.hd - a.rot + 7) / 8, units = pairs + rest;
  const int items = nr * nh * units;
  for (int i = threadIdx.x; i < items; i += kT) {
    const int u = i % units, rh = i / units, row = rh / nh, head = h0 + rh % nh;
    const int64_t from = (int64_t)(r0 + row) * a.ldx + (int64_t)head * a.hd, to = (int64_t)(r0 + row) * a.ldo + (int64_t)head * a.hd;
    if (u >= pairs) {
      const int c = a.rot + (u - pairs) * 8;
      if (c + 8 <= a.hd) {
        float v[8];
        load8<D>(a.x, from + c, v);
        store8<O>(a.out, to + c, v);
      } else {
        for (int j = c; j < a.hd; j++) mx_store(O, a.out, to + j, mx_load(D, a.x, from + j));
      }
      continue;
    }
    const int p = u * 8;
    const Turn *t = turn + row * half + p;
    if (p + 8 <= half) {
      const int at0 = a.interleaved ? 2 * p : p, at1 = a.interleaved ? 2 * p + 8 : p + half;
      float v[2][8];
      load8<D>(a.x, from + at0, v[0]);
      load8<D>(a.x, from + at1, v[1]);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        float &x1 = a.interleaved ? v[j / 4][2 * (j % 4)] : v[0][j], &x2 = a.interleaved ? v[j / 4][2 * (j % 4) + 1] : v[1][j];
        const float y1 = x1 * t[j].c - x2 * t[j].s, y2 = x2 * t[j].c + x1 * t[j].s;
        x1 = y1, x2 = y2;
      }
      store8<O>(a.out, to + at0, v[0]);
      store8<O>(a.out, to + at1, v[1]);
    } else {
      for (int j = 0; p + j < half; j++) {
        const int i1 = a.interleaved ? 2 * (p + j) : p + j, i2 = a.interleaved ? i1 + 1 : i1 + half;
        const float x1 = mx_load(D, a.x, from + i1), x2 = mx_load(D, a.x, from + i2);
        mx_store(O, a.out, to + i1, x1 * t[j].c - x2 * t[j].s);
        mx_store(O, a.out, to + i2, x2 * t[j].c + x1 * t[j].s);
      }
    }
  }
}

}  // namespace

hipError_t launch_rope(const RopeArgs &a, hipStream_t st) {
  const int rows = a.rot / 2 >= kT / 2 ? 1 : kT / (a.rot / 2);
  const int64_t blocks = (a.n + rows - 1) / rows;
  // a few rows' heads over several blocks, as many as fill the chip
  int parts = (int)(512 / blocks);
  parts = parts < 1 ? 1 : parts > a.heads ? a.heads : parts;
  const int heads = (a.heads + parts - 1) / parts;
  const dim3 grid((unsigned)blocks, (unsigned)((a.heads + heads - 1) / heads));
  for_type(a.dtype, [&](auto d) {
    for_type(a.out_dtype, [&](auto o) {
      hipLaunchKernelGGL((rope_kernel<decltype(d)::value, decltype(o)::value>), grid, dim3(kT), 0, st, a, rows, heads);
    });
  });
  return hipGetLastError();
}
