// Expert routing: each token's k best experts, their softmax weights, and the
// (token, choice) slots sorted by expert; and the weighted sum that brings the
// experts' rows back to their tokens.
//
// A logit of -inf or NaN is never chosen; -0 and +0 are equal, and ties go to
// the lower expert. With m the token's largest logit, the weights are
// exp(l - m) over the sum of the chosen ones, or of all (m = +inf: its experts
// share the weight).
//
// What bounds it: latency, at a few tokens; the scan of the slots otherwise. A
// wave holds a token's logits in registers and takes k maxima by lane moves.
// The sort is a counting sort without a histogram in memory, so it needs no
// workspace: the block of expert e counts the slots of lower experts and of
// its own, then places its own in slot order.
#include "mx.h"

namespace {

// The order of logits as unsigned numbers; 0: never chosen.
__device__ __forceinline__ uint32_t rank_of(float v) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <typename F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, F f) {
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));   // lanes 1, 0, 3, 2
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));   // lanes 2, 3, 0, 1
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // row_half_mirror
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror 8
  const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
  const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  return f(f(a, b), f(c, d));
}

// One token by one wave: lane l holds experts l + 64 i. Its choices go to
// ids_out (LDS or global) as well as to the arguments' arrays.
template <int EI>
__device__ __forceinline__ void choose(const RouteArgs &a, int token, int lane, int32_t *ids_out) {
  float v[EI];
  uint32_t key[EI];
#pragma unroll
  for (int i = 0; i < EI; i++) {
    const int e = lane + 64 * i;
    v[i] = e < a.experts ? mx_load(a.dtype, a.logits, token * a.ld + e) : -INFINITY;
    key[i] = rank_of(v[i]);
  }
  int my_id = -1;  // lane j: choice j
  float my_v = 0.f, most = 0.f;
  for (int j = 0; j < a.k; j++) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < EI; i++)
      if (key[i] > best) best = key[i], at = i;
    const uint32_t top = wave_reduce(best, [](uint32_t x, uint32_t y) { return max(x, y); });
    if (!top) break;
    const uint32_t id =
        wave_reduce(best == top ? (uint32_t)(lane + 64 * at) : ~0u, [](uint32_t x, uint32_t y) { return min(x, y); });
    const uint32_t bits = top & 0x80000000u ? top & 0x7fffffffu : ~top;
    if (j == 0) most = __uint_as_float(bits);
    if (lane == j) my_id = (int)id, my_v = __uint_as_float(bits);
#pragma unroll
    for (int i = 0; i < EI; i++)
      if (lane + 64 * i == (int)id) key[i] = 0;
  }
  auto power = [&](float l) { return l == most ? 1.f : expf(l - most); };
  const float mine = my_id >= 0 ? power(my_v) : 0.f;
  float total = mine;
  if (a.over_all) {
    total = 0.f;
#pragma unroll
    for (int i = 0; i < EI; i++) total += v[i] > -INFINITY ? power(v[i]) : 0.f;
  }
  total = wave_sum(total);
  if (lane < a.k) {
    const int64_t slot = (int64_t)token * a.k + lane;
    a.ids[slot] = my_id;
    a.weights[slot] = my_id >= 0 ? mine / total : 0.f;
    if (ids_out) ids_out[slot] = my_id;
    else if (my_id < 0) a.positions[slot] = -1;
  }
}

template <int EI>
__global__ __launch_bounds__(256) void choose_kernel(RouteArgs a) {
  const int token = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (token < a.n) choose<EI>(a, token, threadIdx.x & 63, nullptr);
}

// Block e: offsets[e + 1] and expert e's rows.
constexpr int kSortT = 1024, kSortWaves = kSortT / 64;
__global__ __launch_bounds__(kSortT) void sort_kernel(RouteArgs a) {
  __shared__ uint32_t counts[3][kSortWaves];
  const int e = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slots = a.n * a.k, per = ((slots + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int lo = min(wave * per, slots), hi = min(lo + per, slots);
  uint32_t below = 0, own = 0, valid = 0;
  for (int s = lo + lane; s < hi; s += 64 * 8) {
    int id[8];
#pragma unroll
    for (int j = 0; j < 8; j++) id[j] = s + 64 * j < hi ? a.ids[s + 64 * j] : -1;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      below += id[j] >= 0 && id[j] < e;
      own += id[j] == e;
      valid += id[j] >= 0;
    }
  }
  auto sum = [](uint32_t x, uint32_t y) { return x + y; };
  below = wave_reduce(below, sum);
  own = wave_reduce(own, sum);
  valid = wave_reduce(valid, sum);
  if (lane == 0) counts[0][wave] = below, counts[1][wave] = own, counts[2][wave] = valid;
  __syncthreads();
  uint32_t base = 0, before = 0, all = 0, total = 0;
  for (int w = 0; w < kSortWaves; w++) {
    base += counts[0][w];
    before += w < wave ? counts[1][w] : 0;
    all += counts[1][w];
    total += counts[2][w];
  }
  if (threadIdx.x == 0) {
    if (e == 0) a.offsets[0] = 0;
    a.offsets[e + 1] = (int32_t)(base + all);
  }
  // rows past the last: no token
  for (int64_t r = total + (int64_t)e * kSortT + threadIdx.x; r < slots; r += (int64_t)gridDim.x * kSortT) a.tokens[r] = -1;
  if (!own) return;
  int32_t row = (int32_t)(base + before);
  for (int s0 = lo; s0 < hi; s0 += 64 * 8) {
    int id[8];
#pragma unroll
    for (int j = 0; j < 8; j++) id[j] = s0 + 64 * j + lane < hi ? a.ids[s0 + 64 * j + lane] : -1;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint64_t mask = __ballot(id[j] == e);
      if (id[j] == e) {
        const int s = s0 + 64 * j + lane;
        const int r = row + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        a.tokens[r] = s / a.k;
        a.positions[s] = r;
      }
      row += __popcll(mask);
    }
  }
}

// A few tokens: both steps in one block.
constexpr int kFewSlots = 256, kFewTokens = 32;
template <int EI>
__global__ __launch_bounds__(1024) void route_few_kernel(RouteArgs a) {
  __shared__ int32_t ids[kFewSlots];
  const int tid = threadIdx.x, slots = a.n * a.k;
  for (int t = tid >> 6; t < a.n; t += 16) choose<EI>(a, t, tid & 63, ids);
  __syncthreads();
  // thread e: the slots of experts below e; a slot's row: those and its own expert's earlier ones
  for (int e = tid; e <= a.experts; e += 1024) {
    int below = 0;
    for (int s = 0; s < slots; s++) below += (uint32_t)ids[s] < (uint32_t)e;  // (-1: no expert, above all)
    a.offsets[e] = below;
  }
  if (tid < slots) {
    const int id = ids[tid];
    int row = 0;
    for (int s = 0; s < slots; s++) {
      const int o = ids[s];
      row += (uint32_t)o < (uint32_t)id || (o == id && s < tid);
    }
    // slots without an expert come last, in order: their rows hold no token
    a.tokens[row] = id >= 0 ? tid / a.k : -1;
    a.positions[tid] = id >= 0 ? row : -1;
  }
}

template <int EI>
void launch(const RouteArgs &a, hipStream_t st) {
  if (a.n <= kFewTokens && a.n * a.k <= kFewSlots) {
    hipLaunchKernelGGL(route_few_kernel<EI>, dim3(1), dim3(1024), 0, st, a);
    return;
  }
  hipLaunchKernelGGL(choose_kernel<EI>, dim3((a.n + 3) / 4), dim3(256), 0, st, a);
  hipLaunchKernelGGL(sort_kernel, dim3(a.experts), dim3(kSortT), 0, st, a);
}

// ---------------------------------------------------------------- combine
// out[t] = sum over j of weights[t][j] * y[positions[t][j]], j in order, in
// fp32; positions outside [0, y_rows) add nothing. Bound: HBM (each row of y
// once). A thread forms V consecutive columns, the loads of four choices in
// flight.
template <int D, int V>
__device__ __forceinline__ void load_row(const void *y, int64_t i, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = mx_load(D, y, i);
  } else if constexpr (D == FMT_F32) {
    const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(y) + i);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
    const uint2 a = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(y) + i);
    const uint32_t h[4] = {a.x & 0xffff, a.x >> 16, a.y & 0xffff, a.y >> 16};
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = D == FMT_F16 ? hw_half((uint16_t)h[j]) : __uint_as_float(h[j] << 16);
  }
}

template <int D, int V>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
  const int64_t per = (a.cols + V - 1) / V, total = per * a.n;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / per, c = (i - t * per) * V;
    float sum[V] = {};
    for (int j0 = 0; j0 < a.k; j0 += 4) {
      float v[4][V], w[4];
      bool ok[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int64_t slot = t * a.k + min(j0 + j, a.k - 1);
        const int p = a.positions[slot];
        w[j] = a.weights[slot];
        ok[j] = j0 + j < a.k && p >= 0 && p < a.y_rows;
        if (ok[j]) load_row<D, V>(a.y, p * a.ldy + c, v[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int q = 0; q < V; q++)
          if (ok[j]) sum[q] = fmaf(w[j], v[j][q], sum[q]);
    }
    const int64_t o = t * a.ldo + c;
    if constexpr (V == 1) {
      mx_store(a.odtype, a.out, o, sum[0]);
    } else if (a.odtype == FMT_F32) {
      *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + o) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    } else {
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + o) =
          make_uint2(mx_narrow(a.odtype, sum[0]) | (uint32_t)mx_narrow(a.odtype, sum[1]) << 16,
                     mx_narrow(a.odtype, sum[2]) | (uint32_t)mx_narrow(a.odtype, sum[3]) << 16);
    }
  }
}

}  // namespace

hipError_t launch_route(const RouteArgs &a, hipStream_t st) {
  if (a.experts <= 64) launch<1>(a, st);
  else if (a.experts <= 128) launch<2>(a, st);
  else if (a.experts <= 256) launch<4>(a, st);
  else if (a.experts <= 512) launch<8>(a, st);
  else launch<16>(a, st);
  return hipGetLastError();
}

hipError_t launch_combine(const CombineArgs &a, hipStream_t st) {
  auto quads = [](const void *p, int64_t ld, int dtype) {
    const size_t w = mx_width(dtype) * 4;
    return reinterpret_cast<uintptr_t>(p) % w == 0 && ld % 4 == 0;
  };
  const bool vec = a.cols % 4 == 0 && quads(a.y, a.ldy, a.dtype) && quads(a.out, a.ldo, a.odtype);
  const int64_t items = a.n * (vec ? a.cols / 4 : a.cols);
  const dim3 grid((unsigned)std::min<int64_t>((items + 255) / 256, 1 << 20));
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a); };
  if (a.dtype == FMT_F32) vec ? go(combine_kernel<FMT_F32, 4>) : go(combine_kernel<FMT_F32, 1>);
  else if (a.dtype == FMT_F16) vec ? go(combine_kernel<FMT_F16, 4>) : go(combine_kernel<FMT_F16, 1>);
  else vec ? go(combine_kernel<FMT_BF16, 4>) : go(combine_kernel<FMT_BF16, 1>);
  return hipGetLastError();
}
