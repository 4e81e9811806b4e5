// Expert routing: each token's k best experts, their softmax weights, and the
// (token, choice) slots sorted by expert; and the weighted sum that brings the
// experts' rows back to their tokens.
//
// A logit of -inf or NaN is never chosen; -0 and +0 are equal, and ties go to
// the lower expert. With m the token's largest logit, the weights are
// exp(l - m) over the sum of the chosen ones, or of all (m = +inf: its experts
// share the weight).
//
// What bounds it: latency, at a few tokens (one launch of one block); the k
// maxima of each token otherwise. A wave holds a token's logits in registers
// and takes the maxima by lane moves. The sort is a counting sort; it needs no
// workspace. Up to a few thousand slots, the block of expert e counts the slots
// of lower experts and of its own, then places its own in slot order (two
// launches). Beyond, each block of tokens leaves how many slots it has for each
// expert in `tokens`; the next launch sums the blocks before each, places the
// block's slots and writes `positions`, and a third one writes `tokens` from
// them (16384 tokens to 8 of 128 experts: 53 us with a block for each expert,
// each over all slots, 23 us so, 14 of them the choices' lane moves).
// 16 tokens to 4 of 64 experts: 5.9 us.
#include <algorithm>

#include "mx.h"
#include "mx_rule.h"

namespace {

using namespace tinyoai_rule;

// The order of logits as unsigned numbers; 0: never chosen.
__device__ __forceinline__ uint32_t rank_of(float v) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The wave's largest value, and sum (0 is neutral for both).
template <typename F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, F f) {
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true));   // row_shr 1
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true));   // row_shr 2
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true));   // row_shr 4
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true));   // row_shr 8: lane 15 has its row's
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));  // row_bcast 15 to rows 1 and 3
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));  // row_bcast 31 to rows 2 and 3
  return __builtin_amdgcn_readlane(v, 63);
}

// One token by one wave: lane l holds experts l + 64 i. Its choices go to
// ids_out (LDS) as well as to the arguments' arrays, and are counted in LDS.
template <int EI>
__device__ __forceinline__ void choose(const RouteArgs &a, int token, int lane, int32_t *ids_out, uint32_t *counts) {
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
#pragma unroll
    for (int i = 0; i < EI; i++) best = max(best, key[i]);
    const uint32_t top = wave_reduce(best, [](uint32_t x, uint32_t y) { return max(x, y); });
    if (!top) break;
    // of the experts with this logit the lowest: the first group of 64 with one, its first lane
    uint32_t id = 0;
#pragma unroll
    for (int i = EI - 1; i >= 0; i--) {
      const uint64_t mask = __ballot(key[i] == top);
      if (mask) id = (uint32_t)(64 * i + __ffsll((unsigned long long)mask) - 1);
    }
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
    if (counts && my_id >= 0) atomicAdd(&counts[my_id], 1u);  // (in LDS: the sum does not depend on the order)
  }
}

template <int EI>
__global__ __launch_bounds__(256) void choose_kernel(RouteArgs a) {
  const int token = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (token < a.n) choose<EI>(a, token, threadIdx.x & 63, nullptr, nullptr);
}

// Block e: offsets[e + 1] and expert e's rows.
constexpr int kSortT = 1024, kSortWaves = kSortT / 64;
static_assert(kSortSlots == kSortT * 8, "a round of loads");
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

// Many slots. Block b has the tokens [n b / nb, n (b + 1) / nb), whose slots are
// no fewer than the experts: its row of the table of counts is in `tokens`.
constexpr int kBlockT = 1024;
__device__ __forceinline__ int first_token(const RouteArgs &a, int b, int nb) { return (int)((int64_t)a.n * b / nb); }

template <int EI>
__global__ __launch_bounds__(kBlockT) void choose_count_kernel(RouteArgs a) {
  __shared__ uint32_t counts[64 * EI];
  const int tid = threadIdx.x, b = blockIdx.x, lo = first_token(a, b, gridDim.x), hi = first_token(a, b + 1, gridDim.x);
  for (int e = tid; e < a.experts; e += kBlockT) counts[e] = 0;
  __syncthreads();
  for (int t = lo + (tid >> 6); t < hi; t += kBlockT / 64) choose<EI>(a, t, tid & 63, nullptr, counts);
  __syncthreads();
  for (int e = tid; e < a.experts; e += kBlockT) a.tokens[(int64_t)b * a.experts + e] = (int32_t)counts[e];
}

// BITS: those of an expert's number.
template <int BITS>
__global__ __launch_bounds__(kBlockT) void place_kernel(RouteArgs a) {
  constexpr int kW = kBlockT / 64;
  __shared__ int before[kBlockT], all[kBlockT], ends[kW];
  __shared__ int count[kW][1 << BITS];  // a round's slots of each wave and expert
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x, nb = gridDim.x, E = a.experts;
  // Columns of the table: thread (part, e) the rows part, part + parts, ...
  const int parts = kBlockT / E;
  const int e = tid % E, part = tid / E;
  int mine = 0, total = 0;
  if (part < parts) {
    for (int r0 = part; r0 < nb; r0 += parts * 16) {
      int v[16];
#pragma unroll
      for (int j = 0; j < 16; j++) v[j] = r0 + j * parts < nb ? a.tokens[(int64_t)(r0 + j * parts) * E + e] : 0;
#pragma unroll
      for (int j = 0; j < 16; j++) {
        total += v[j];
        mine += r0 + j * parts < b ? v[j] : 0;
      }
    }
    before[tid] = mine;
    all[tid] = total;
  }
  __syncthreads();
  mine = total = 0;
  if (tid < E)
    for (int p = 0; p < parts; p++) {
      mine += before[p * E + tid];
      total += all[p * E + tid];
    }
  // the experts' ends, by waves
  int end = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(end, o);
    if (lane >= o) end += v;
  }
  if (lane == 63) ends[wave] = end;
  __syncthreads();
  for (int w = 0; w < wave; w++) end += ends[w];
  if (tid < E) {
    before[tid] = end - total + mine;  // the next row of expert tid for this block
    if (b == 0) {
      a.offsets[tid + 1] = end;
      if (tid == 0) a.offsets[0] = 0;
    }
  }
  const int64_t lo = (int64_t)first_token(a, b, nb) * a.k, hi = (int64_t)first_token(a, b + 1, nb) * a.k;
  for (int64_t s0 = lo; s0 < hi; s0 += kBlockT) {
    for (int i = tid; i < kW << BITS; i += kBlockT) (&count[0][0])[i] = 0;
    __syncthreads();
    const int id = s0 + tid < hi ? a.ids[s0 + tid] : -1;
    // the lanes with this slot's expert
    uint64_t same = __ballot(id >= 0);
#pragma unroll
    for (int i = 0; i < BITS; i++) {
      const uint64_t ones = __ballot(id >> i & 1);
      same &= id >> i & 1 ? ones : ~ones;
    }
    const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
    if (id >= 0 && rank == 0) count[wave][id] = __popcll(same);
    __syncthreads();
    int row = -1;
    if (id >= 0) {
      row = before[id] + rank;
      for (int w = 0; w < wave; w++) row += count[w][id];
    }
    if (s0 + tid < hi) a.positions[s0 + tid] = row;
    __syncthreads();
    if (tid < E) {
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kW; w++) sum += count[w][tid];
      before[tid] += sum;
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(256) void tokens_kernel(RouteArgs a) {
  const int slots = a.n * a.k, total = a.offsets[a.experts];
  for (int s = blockIdx.x * 256 + threadIdx.x; s < slots; s += gridDim.x * 256) {
    const int row = a.positions[s];
    if (row >= 0) a.tokens[row] = s / a.k;
    if (s >= total) a.tokens[s] = -1;
  }
}

// A few tokens: both steps in one block.
template <int EI>
__global__ __launch_bounds__(1024) void route_few_kernel(RouteArgs a) {
  __shared__ __align__(16) int32_t ids[kFewSlots];
  const int tid = threadIdx.x, slots = a.n * a.k, quads = (slots + 3) / 4;
  if (tid < 4 && slots + tid < kFewSlots) ids[slots + tid] = -1;
  for (int t = tid >> 6; t < a.n; t += 16) choose<EI>(a, t, tid & 63, ids, nullptr);
  __syncthreads();
  // thread e: the slots of experts below e (-1, no expert, is above all); a
  // slot's row: those and its own expert's earlier ones
  const bool offset = tid <= a.experts, slot = tid < slots;
  if (offset || slot) {
    const uint32_t id = slot ? (uint32_t)ids[tid] : 0;
    uint32_t below = 0, row = 0;
#pragma unroll 4
    for (int i = 0; i < quads; i++) {
      const uint4 q = reinterpret_cast<const uint4 *>(ids)[i];
      const uint32_t o[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        below += o[j] < (uint32_t)tid;
        row += o[j] < id || (o[j] == id && 4 * i + j < tid);
      }
    }
    if (offset) a.offsets[tid] = (int32_t)below;
    if (slot) {
      // slots without an expert come last, in order: their rows hold no token
      a.tokens[row] = (int32_t)id >= 0 ? tid / a.k : -1;
      a.positions[tid] = (int32_t)id >= 0 ? (int32_t)row : -1;
    }
  }
  if (tid == 0 && a.experts == 1024) {  // the one offset past the threads
    int total = 0;
    for (int s = 0; s < slots; s++) total += ids[s] >= 0;
    a.offsets[1024] = total;
  }
}

template <int EI>
void launch(const RouteArgs &a, hipStream_t st) {
  const Sort path = sort_path(a.n, a.k);
  if (path == Sort::one_block) {
    hipLaunchKernelGGL(route_few_kernel<EI>, dim3(1), dim3(1024), 0, st, a);
    return;
  }
  const int slots = a.n * a.k;
  if (path == Sort::by_expert) {
    hipLaunchKernelGGL(choose_kernel<EI>, dim3((a.n + 3) / 4), dim3(256), 0, st, a);
    hipLaunchKernelGGL(sort_kernel, dim3(a.experts), dim3(kSortT), 0, st, a);
    return;
  }
  // (a block's slots are no fewer than the experts; kSortSlots leaves several)
  const int blocks = std::min(device_cu_count(), a.n / ((a.experts + a.k - 1) / a.k));
  hipLaunchKernelGGL(choose_count_kernel<EI>, dim3(blocks), dim3(kBlockT), 0, st, a);
  constexpr int kBits = EI == 1 ? 6 : EI == 2 ? 7 : EI == 4 ? 8 : EI == 8 ? 9 : 10;
  hipLaunchKernelGGL(place_kernel<kBits>, dim3(blocks), dim3(kBlockT), 0, st, a);
  hipLaunchKernelGGL(tokens_kernel, dim3(std::min((slots + 255) / 256, 4096)), dim3(256), 0, st, a);
}

// ---------------------------------------------------------------- combine
// out[t] = sum over j of weights[t][j] * y[positions[t][j]], j in order, in
// fp32; positions outside [0, y_rows) add nothing. Bound: HBM (each row of y
// once: 8192 tokens of 8 bf16 rows of 2560 columns, 378 MB, in 79 us, 4.8 TB/s).
// A thread forms V consecutive columns (16 bytes of y; those of a row's last
// thread one by one), the loads of four choices in flight.
template <int D, int V>
__device__ __forceinline__ void load_row(const void *y, int64_t i, int n, float (&v)[V]) {
  if (n < V) {
#pragma unroll
    for (int q = 0; q < V; q++) v[q] = q < n ? mx_load(D, y, i + q) : 0.f;
  } else if constexpr (D == FMT_F32) {
    const f32x4_any a = *reinterpret_cast<const f32x4_any *>(static_cast<const float *>(y) + i);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
    const u32x4_any w = *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(y) + i);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint16_t h = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
      v[j] = D == FMT_F16 ? hw_half(h) : bf16_to_float(h);
    }
  }
}

template <int D>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a, int per) {
  constexpr int V = D == FMT_F32 ? 4 : 8;
  const int t = blockIdx.x / per;  // per: blocks of a token
  const int64_t c = ((int64_t)(blockIdx.x - t * per) * 256 + threadIdx.x) * V;
  if (c >= a.cols) return;
  const int n = (int)min(a.cols - c, (int64_t)V);
  float sum[V] = {};
  for (int j0 = 0; j0 < a.k; j0 += 4) {
    float v[4][V], w[4];
    bool ok[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t slot = (int64_t)t * a.k + min(j0 + j, a.k - 1);
      const int p = a.positions[slot];
      w[j] = a.weights[slot];
      ok[j] = j0 + j < a.k && p >= 0 && p < a.y_rows;
      if (ok[j]) load_row<D, V>(a.y, p * a.ldy + c, n, v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int q = 0; q < V; q++)
        if (ok[j]) sum[q] = fmaf(w[j], v[j][q], sum[q]);
  }
  const int64_t o = t * a.ldo + c;
  if (n < V) {
#pragma unroll
    for (int q = 0; q < V; q++)
      if (q < n) mx_store(a.odtype, a.out, o + q, sum[q]);
  } else if (a.odtype == FMT_F32) {
#pragma unroll
    for (int q = 0; q < V; q += 4)
      *reinterpret_cast<f32x4_any *>(static_cast<float *>(a.out) + o + q) = f32x4_any{sum[q], sum[q + 1], sum[q + 2], sum[q + 3]};
  } else {
    uint32_t h[V / 2];
#pragma unroll
    for (int q = 0; q < V / 2; q++) h[q] = mx_narrow(a.odtype, sum[2 * q]) | (uint32_t)mx_narrow(a.odtype, sum[2 * q + 1]) << 16;
    if constexpr (V == 8) *reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(a.out) + o) = u32x4_any{h[0], h[1], h[2], h[3]};
    else *reinterpret_cast<u32x2_any *>(static_cast<uint16_t *>(a.out) + o) = u32x2_any{h[0], h[1]};
  }
}

}  // namespace

hipError_t launch_route(const RouteArgs &a, hipStream_t st) {
  switch (lane_experts(a.experts)) {
    case 1: launch<1>(a, st); break;
    case 2: launch<2>(a, st); break;
    case 4: launch<4>(a, st); break;
    case 8: launch<8>(a, st); break;
    default: launch<16>(a, st);
  }
  return hipGetLastError();
}

hipError_t launch_combine(const CombineArgs &a, hipStream_t st) {
  const int64_t threads = a.dtype == FMT_F32 ? (a.cols + 3) / 4 : (a.cols + 7) / 8;
  const int per = (int)((threads + 255) / 256);  // at most 2^23
  // A launch's threads number below 2^32: many tokens in several. (Blocks that
  // take several parts in turn cost more, since positions and weights no longer
  // come by scalar loads: 8192 tokens of 8 rows of 2560 columns 96 us instead
  // of 78.)
  if ((int64_t)per * a.n > 1 << 23) {
    const int first = (1 << 23) / per;
    CombineArgs part = a;
    part.n = first;
    if (const hipError_t e = launch_combine(part, st); e != hipSuccess) return e;
    part.n = a.n - first;
    part.positions += (int64_t)first * a.k;
    part.weights += (int64_t)first * a.k;
    part.out = static_cast<char *>(a.out) + first * a.ldo * (int64_t)mx_width(a.odtype);
    return launch_combine(part, st);
  }
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)(per * a.n)), dim3(256), 0, st, a, per); };
  if (a.dtype == FMT_F32) go(combine_kernel<FMT_F32>);
  else if (a.dtype == FMT_F16) go(combine_kernel<FMT_F16>);
  else go(combine_kernel<FMT_BF16>);
  return hipGetLastError();
}
