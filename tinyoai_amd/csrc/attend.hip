// Attention of one new token of each sequence over its pages:
//   s_j = scale q . k_j,  o = sum_j 2^(s_j' - m) v_j / sum_j 2^(s_j' - m),
// s' = s log2 e and m the running maximum, in one pass over the positions
// (softmax weights are then single 2^x instructions). Positions from the
// sequence's length on, and those of table entries outside the pool, are not
// read; a sequence without positions gets zeros.
//
// A block of four waves takes one key head, up to G of its query heads and a
// range of positions; the ranges' unnormalised records {m, sum, o} are joined
// in order by a second kernel. A row's lanes hold eight values each, rows are
// spread over the lanes, and every group of lanes keeps a maximum and sums of
// its own, so nothing is exchanged but the parts of the scores until the end.
#include <type_traits>

#include "attend.h"

namespace {

constexpr int kT = 256, kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

template <int C>
struct Row8 {  // eight values of a row as they lie in the pages
  uint4 a[C == FMT_F32 ? 2 : 1];
};

template <int C>
__device__ __forceinline__ void load_row(Row8<C> &r, const uint8_t *p) {
  if constexpr (C == FMT_Q8_0) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    r.a[0].x = w.x, r.a[0].y = w.y;
  } else {
#pragma unroll
    for (int i = 0; i < (C == FMT_F32 ? 2 : 1); i++) r.a[i] = reinterpret_cast<const uint4 *>(p)[i];
  }
}
template <int C>
__device__ __forceinline__ void values(const Row8<C> &r, float (&v)[8]) {
  uint32_t w[8] = {r.a[0].x, r.a[0].y, r.a[0].z, r.a[0].w};
  if constexpr (C == FMT_F32) w[4] = r.a[1].x, w[5] = r.a[1].y, w[6] = r.a[1].z, w[7] = r.a[1].w;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    if constexpr (C == FMT_F32) v[j] = __uint_as_float(w[j]);
    else if constexpr (C == FMT_Q8_0) v[j] = (float)(int8_t)(w[j / 4] >> (8 * (j % 4)));
    else if constexpr (C == FMT_F16) v[j] = hw_half((uint16_t)(w[j / 2] >> (16 * (j & 1))));
    else v[j] = bf16_to_float((uint16_t)(w[j / 2] >> (16 * (j & 1))));
  }
}

struct Plan {
  int chunk, splits;  // positions of a block, blocks along the longest sequence
  int groups;         // query heads of a key head over blocks
  float *records;     // [n][heads][splits][hd + 2]
};

__device__ __forceinline__ void store_out(const AttendArgs &a, int seq, int head, int d, float v) {
  mx_store(a.dtype, a.out, seq * a.ldo + (int64_t)head * a.c.hd + d, v);
}

template <int C, int G>
__global__ __launch_bounds__(kT) void attend_kernel(AttendArgs a, Plan p) {
  constexpr int U = 4;
  __shared__ float part[kWaves][G][kHeadDim + 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hd = a.c.hd, group = a.heads / a.c.kv_heads;
  const int split = blockIdx.y, seq = blockIdx.x / (a.c.kv_heads * p.groups);
  const int kvh = blockIdx.x / p.groups % a.c.kv_heads, g0 = blockIdx.x % p.groups * G;
  const int length = min(a.lengths[seq], (int)min((int64_t)a.width << a.c.page_log2, (int64_t)INT32_MAX));
  const int start = split * p.chunk, end = min(length, start + p.chunk);
  if (start >= end && (split || length > 0)) return;
  const int row_lanes = 1 << (hd > 128 ? 5 : hd > 64 ? 4 : hd > 32 ? 3 : hd > 16 ? 2 : hd > 8 ? 1 : 0);
  const int rows = 64 / row_lanes, mine = lane / row_lanes, c = lane % row_lanes * 8;
  const bool in = c < hd;
  float q[G][8];
#pragma unroll
  for (int g = 0; g < G; g++) {
    const int head = kvh * group + min(g0 + g, group - 1);
    const int64_t at = seq * a.ldq + (int64_t)head * hd + c;
#pragma unroll
    for (int j = 0; j < 8; j++) q[g][j] = 0.f;
    if (in) {
      if (a.dtype == FMT_F32) load8<FMT_F32>(a.q, at, q[g]);
      else if (a.dtype == FMT_F16) load8<FMT_F16>(a.q, at, q[g]);
      else load8<FMT_BF16>(a.q, at, q[g]);
    }
  }
  const float scale = a.scale * kLog2e;
  float m[G], l[G], acc[G][8];
#pragma unroll
  for (int g = 0; g < G; g++) {
    m[g] = -INFINITY, l[g] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) acc[g][j] = 0.f;
  }
  const int *table = a.table + (int64_t)seq * a.width;
  constexpr int kValue = C == FMT_F32 ? 4 : C == FMT_Q8_0 ? 1 : 2;
  for (int t0 = start + wave * rows * U; t0 < end; t0 += kWaves * rows * U) {
    Row8<C> k[U], v[U];
    float dk[U], dv[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int t = t0 + u * rows + mine;
      const int page = t < end ? table[t >> a.c.page_log2] : -1;
      ok[u] = (uint32_t)page < (uint32_t)a.c.pages;
      k[u] = v[u] = Row8<C>{};
      dk[u] = dv[u] = 0.f;
      if (ok[u] && in) {
        const int64_t row = kv_row(a.c, page << a.c.page_log2 | (t & ((1 << a.c.page_log2) - 1)), kvh);
        load_row<C>(k[u], a.c.k + row * a.c.pitch + c * kValue);
        load_row<C>(v[u], a.c.v + row * a.c.pitch + c * kValue);
        if constexpr (C == FMT_Q8_0) {
          dk[u] = hw_half(a.c.kd[row * a.c.nb + c / 32]);
          dv[u] = hw_half(a.c.vd[row * a.c.nb + c / 32]);
        }
      }
    }
    float s[U][G];
#pragma unroll
    for (int u = 0; u < U; u++) {
      float x[8];
      values<C>(k[u], x);
#pragma unroll
      for (int g = 0; g < G; g++) {
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) d = fmaf(q[g][j], x[j], d);
        if constexpr (C == FMT_Q8_0) d *= dk[u];
        s[u][g] = d;
      }
    }
    for (int off = row_lanes / 2; off; off /= 2)
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int g = 0; g < G; g++) s[u][g] += __shfl_xor(s[u][g], off);
#pragma unroll
    for (int g = 0; g < G; g++) {
      float top = m[g];
#pragma unroll
      for (int u = 0; u < U; u++) {
        s[u][g] = ok[u] ? s[u][g] * scale : -INFINITY;
        top = fmaxf(top, s[u][g]);
      }
      const float ref = top == -INFINITY ? 0.f : top, fade = exp2_hw(m[g] - ref);
      m[g] = top;
      l[g] *= fade;
#pragma unroll
      for (int j = 0; j < 8; j++) acc[g][j] *= fade;
#pragma unroll
      for (int u = 0; u < U; u++) {
        s[u][g] = exp2_hw(s[u][g] - ref);
        l[g] += s[u][g];
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      float x[8];
      values<C>(v[u], x);
#pragma unroll
      for (int g = 0; g < G; g++) {
        const float w = C == FMT_Q8_0 ? s[u][g] * dv[u] : s[u][g];
#pragma unroll
        for (int j = 0; j < 8; j++) acc[g][j] = fmaf(w, x[j], acc[g][j]);
      }
    }
  }
  // the wave's groups of lanes, then the waves
  for (int off = row_lanes; off < 64; off *= 2)
#pragma unroll
    for (int g = 0; g < G; g++) {
      const float other = __shfl_xor(m[g], off), top = fmaxf(m[g], other), ref = top == -INFINITY ? 0.f : top;
      const float fade = exp2_hw(m[g] - ref), fade2 = exp2_hw(other - ref);
      m[g] = top;
      l[g] = l[g] * fade + __shfl_xor(l[g], off) * fade2;
#pragma unroll
      for (int j = 0; j < 8; j++) acc[g][j] = acc[g][j] * fade + __shfl_xor(acc[g][j], off) * fade2;
    }
#pragma unroll
  for (int g = 0; g < G; g++) {
    if (lane == 0) part[wave][g][0] = m[g], part[wave][g][1] = l[g];
    if (mine == 0 && in)
#pragma unroll
      for (int j = 0; j < 8; j++) part[wave][g][2 + c + j] = acc[g][j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * hd; i += kT) {
    const int g = i / hd, d = i % hd, head = kvh * group + g0 + g;
    if (g0 + g >= group) break;
    float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) top = fmaxf(top, part[w][g][0]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float fade = exp2_hw(part[w][g][0] - ref);
      sum += part[w][g][1] * fade;
      o += part[w][g][2 + d] * fade;
    }
    if (p.splits == 1) {
      store_out(a, seq, head, d, sum == 0.f ? 0.f : o / sum);
    } else {
      float *rec = p.records + (((int64_t)seq * a.heads + head) * p.splits + split) * (hd + 2);
      if (d == 0) rec[0] = top, rec[1] = sum;
      rec[2 + d] = o;
    }
  }
}

__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a, Plan p) {
  const int seq = blockIdx.x / a.heads, head = blockIdx.x % a.heads, hd = a.c.hd;
  const int length = min(a.lengths[seq], (int)min((int64_t)a.width << a.c.page_log2, (int64_t)INT32_MAX));
  const int splits = length > 0 ? (length - 1) / p.chunk + 1 : 0;
  const float *rec = p.records + (int64_t)blockIdx.x * p.splits * (hd + 2);
  float top = -INFINITY;
  for (int s = 0; s < splits; s++) top = fmaxf(top, rec[(int64_t)s * (hd + 2)]);
  const float ref = top == -INFINITY ? 0.f : top;
  for (int d = threadIdx.x; d < hd; d += 256) {
    float sum = 0.f, o = 0.f;
    for (int s = 0; s < splits; s++) {
      const float *r = rec + (int64_t)s * (hd + 2);
      const float fade = exp2_hw(r[0] - ref);
      sum += r[1] * fade;
      o += r[2 + d] * fade;
    }
    store_out(a, seq, head, d, sum == 0.f ? 0.f : o / sum);
  }
}

int heads_per_block(const AttendArgs &a) {
  const int group = a.heads / a.c.kv_heads;
  return group >= 4 ? 4 : group >= 2 ? 2 : 1;
}

Plan plan_of(const AttendArgs &a) {
  Plan p{};
  const int group = a.heads / a.c.kv_heads, g = heads_per_block(a);
  p.groups = (group + g - 1) / g;
  const int64_t most = std::min<int64_t>((int64_t)a.width << a.c.page_log2, INT32_MAX), rows = (int64_t)a.n * a.c.kv_heads * p.groups;
  // blocks for the chip several times over, of 256 positions at least
  int64_t chunk = std::max<int64_t>(256, most * rows / 4096);
  chunk = std::max<int64_t>(chunk, (most + 255) / 256);
  p.chunk = (int)std::min<int64_t>((chunk + 63) / 64 * 64, (int64_t)1 << 30);
  p.splits = (int)((most + p.chunk - 1) / p.chunk);
  return p;
}

}  // namespace

size_t attend_scratch(const AttendArgs &a) {
  const Plan p = plan_of(a);
  return p.splits == 1 ? 0 : (size_t)a.n * a.heads * p.splits * (a.c.hd + 2) * 4;
}

hipError_t launch_attend(const AttendArgs &a, void *scratch, hipStream_t st) {
  Plan p = plan_of(a);
  p.records = static_cast<float *>(scratch);
  const dim3 grid((unsigned)(a.n * a.c.kv_heads * p.groups), (unsigned)p.splits);
  auto go = [&](auto c) {
    constexpr int C = decltype(c)::value;
    switch (heads_per_block(a)) {
      case 1: hipLaunchKernelGGL((attend_kernel<C, 1>), grid, dim3(kT), 0, st, a, p); break;
      case 2: hipLaunchKernelGGL((attend_kernel<C, 2>), grid, dim3(kT), 0, st, a, p); break;
      default: hipLaunchKernelGGL((attend_kernel<C, 4>), grid, dim3(kT), 0, st, a, p);
    }
  };
  if (a.c.type == FMT_Q8_0) go(std::integral_constant<int, FMT_Q8_0>());
  else for_type(a.c.type, go);
  if (p.splits > 1) hipLaunchKernelGGL(attend_join_kernel, dim3((unsigned)(a.n * a.heads)), dim3(256), 0, st, a, p);
  return hipGetLastError();
}
