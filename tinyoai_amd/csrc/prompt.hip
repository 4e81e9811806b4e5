// Attention of packed prompts: query i of a sequence's nq sees its keys j <=
// i + nk - nq (causal; all of them otherwise), grouped heads, online softmax in
// fp32 base 2. A query that sees nothing gets zeros; rows of sequences' other
// queries are not touched.
//
// On the matrix cores, both products transposed, so that a lane's column is
// one query throughout and softmax statistics, rescaling and the final division
// need no exchange but one of a maximum between the two halves of a wave:
//   S^T = K Q^T   (32 keys x 32 queries a tile; A = K rows, B = Q rows)
//   O^T += V^T P  (32 dims x 32 queries; A = V^T, B = the softmax weights, in
//                  the very registers that S^T left them in)
// Lane l of S^T's tile holds, for query l % 32, the keys 8 (v / 4) + 4 (l / 32)
// + v % 4. 16-bit values: 32x32x16 products; the eight keys of a step of O^T
// are the lane's values 8 h .. 8 h + 7, so V^T is read with that order of keys,
// by transposed LDS reads (each 16 lanes read 4 keys x 16 dims, and a lane gets
// its dim of the four keys). fp32 values: 32x32x2 products, each value of S^T a
// step, V read as it lies.
//
// What bounds it: at length the power the card gives. 8192 queries and keys, 32
// over 8 bf16 heads of 128, all seen: 1.03 to 1.07 ms, 1028 to 1065 TFLOP/s by the
// card; 16381 fp16 tokens of 32 heads of 80, causal: 1.50 to 1.60 ms, 860 to 915 (a
// library product of 8192^3: 1160 to 1207). There the clock falls to 1.6 to 1.9 GHz, and fewer cycles (products
// scheduled between their operands' reads and the weights) do not change the
// time, fewer bytes do: 64 queries a wave for heads up to 64 (829 -> 882). At few
// thousand queries it is the longest block's chain of tiles, 1.3 to 2 us each
// (64 keys by 128 queries). Few queries over many keys: the keys are cut into
// parts whose sums a second kernel joins (296 queries over 12000 keys 81 -> 58
// us), or over groups of waves in a block (19 over 449 in fp32 61 -> 16).
// fp32: 140 TFLOP/s at heads of 128 (a library product: 154).
//
// 16-bit weights are rounded to their type before the product with V, and summed
// as rounded. Errors against 64 bits are 1.2 to 1.4 times those of results that
// are only rounded themselves; a second plane for the rest of the weights would
// double the products with V.
#include <type_traits>

#include "attend.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Groups of __builtin_amdgcn_sched_group_barrier, which orders the instructions around it.
constexpr int kVector = 0x2, kProducts = 0x8, kReads = 0x100, kExponents = 0x400;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

template <int D>
__device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
  if constexpr (D == FMT_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int D>
__device__ __forceinline__ uint32_t pack2(float a, float b) {  // to the nearest, ties to even
  if constexpr (D == FMT_F16) return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  else return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}
// Whether one of the values in 16 bytes is an infinity or NaN.
template <int D>
__device__ __forceinline__ bool not_finite(uint4 w) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if constexpr (D == FMT_F32) {
      bad |= (x[j] & 0x7f800000u) == 0x7f800000u;
    } else {
      constexpr uint32_t e = D == FMT_F16 ? 0x7c00u : 0x7f80u;
      bad |= (x[j] & e) == e || (x[j] >> 16 & e) == e;
    }
  }
  return bad;
}

template <int D>
__device__ __forceinline__ uint4 only_finite(uint4 w) {  // zeros for the others
  auto one = [](uint32_t u) {
    if constexpr (D == FMT_F32) return (u & 0x7f800000u) == 0x7f800000u ? 0u : u;
    constexpr uint32_t e = D == FMT_F16 ? 0x7c00u : 0x7f80u;
    return ((u & e) == e ? 0u : u & 0xffffu) | ((u >> 16 & e) == e ? 0u : u & 0xffff0000u);
  };
  return make_uint4(one(w.x), one(w.y), one(w.z), one(w.w));
}
// c plus both halves of a pair.
template <int D>
__device__ __forceinline__ float plus2(uint32_t a, float c) {
  if constexpr (D == FMT_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), f16x2{(_Float16)1.f, (_Float16)1.f}, c, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a), bf16x2{(__bf16)1.f, (__bf16)1.f}, c, false);
}
// The sequence of query tile `tile` (tiles of QB queries, a sequence's last
// ones first), its queries and keys.
struct Where {
  int tile;            // within the sequence; -1: none
  int q0, nq, k0, nk;  // first rows and numbers
};
template <int QB>
__device__ __forceinline__ Where find(const PromptArgs &a, int tile) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < a.sequences; s0 += 64) {
    const int s = s0 + lane;
    int q0 = 0, nq = 0, k0 = 0, nk = 0;
    if (s < a.sequences) {
      q0 = min(max(a.q_offsets[s], 0), a.nq);
      nq = max(min(a.q_offsets[s + 1], a.nq) - q0, 0);
      k0 = min(max(a.k_offsets[s], 0), a.nk);
      nk = max(min(a.k_offsets[s + 1], a.nk) - k0, 0);
    }
    int upto = (nq + QB - 1) / QB;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      if (off >= a.sequences) break;  // (past them nothing is added up)
      const int x = __shfl_up(upto, off);
      if (lane >= off) upto += x;
    }
    const uint64_t past = __ballot(before + upto > tile && s < a.sequences);
    if (past) {
      const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
      return Where{before + __builtin_amdgcn_readlane(upto, l) - 1 - tile, __builtin_amdgcn_readlane(q0, l),
                   __builtin_amdgcn_readlane(nq, l), __builtin_amdgcn_readlane(k0, l), __builtin_amdgcn_readlane(nk, l)};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return Where{-1, 0, 0, 0, 0};
}

// Which block does what. Blocks go over the eight XCDs in turn, and an XCD takes
// the same heads of every tile, so that the blocks that it runs share their keys
// in its L2 (all heads of some tiles to an XCD: 8192 queries and keys, 32 over 8
// heads of 128, 1100 instead of 1060 us). Tiles come longest first.
struct Order {
  int tiles, split;
};
__device__ __forceinline__ void block_of(const PromptArgs &a, const Order &o, int block, int &head, int &tile, int &part) {
  const int ways = a.heads % 8 == 0 ? 8 : 1, heads = a.heads / ways, j = block / ways;
  head = block % ways * heads + j % heads;
  tile = j / heads / o.split;
  part = j / heads % o.split;
}

// The chunk that place `p` of a tile's plane holds: C chunks a row, a row's
// chunks exchanged by k_place or v_place (both are their own inverse).
template <int D, int C, bool VT>
__device__ __forceinline__ int chunk_at(int row, int p) {
  return !VT ? k_place<C>(row, p) : D == FMT_F32 ? p : v_place<C>(row, p);
}

// QG * KG waves: QG groups of QN times 32 queries by KG groups of keys, which take the
// sequence's tiles of KEYS keys in turn and whose sums are joined at the end.
// KS: steps of 16 dims. DMA: K and V go straight into LDS (rows on 16-byte
// boundaries), else through registers.
template <int D, int KS, int QN, int QG, int KG, int KEYS, int STAGES, bool DMA>
struct Prompt {
  static constexpr bool F32 = D == FMT_F32;
  static constexpr int HD = KS * 16;
  static constexpr int T = 64 * QG * KG, QB = 32 * QN * QG;
  static constexpr int V = F32 ? 4 : 8;              // values of a chunk
  static constexpr int C = HD / V;                   // chunks of a row
  static constexpr int DT = (HD + 31) / 32;          // 32-dim tiles of O^T
  static constexpr int PLANE = KEYS * C;             // chunks of a tile's K or V
  static constexpr int QS = F32 ? 2 * KS : KS;       // operands of a query
  // Dims past a row's end in the last tile: chunks that an fp32 read may touch
  // there; of 16-bit values a column of ones takes the first of them, which
  // makes the matrix cores add up the softmax weights.
  static constexpr int SPAN = DT * 32 / V - C;
  static constexpr bool ONES = !F32 && SPAN > 0;
  static constexpr int JOIN = KG > 1 ? QG * KG * (DT * 16 + 2) * 16 : 0;  // chunks that the groups' sums take
  static constexpr int TILES = STAGES * KG * 2 * PLANE + SPAN;
  static constexpr int LDS = TILES > JOIN ? TILES : JOIN;
  static_assert(LDS * 16 <= 160 * 1024, "LDS of a CU");
  typedef std::conditional_t<F32, float, uint16_t> Value;
};

// With several parts, a block takes one of that many equal runs of its tile's
// keys and leaves unnormalised records for prompt_join_kernel.
struct Parts {
  Order order;
  float2 *stats;   // [tile][head][part][query] {reference, sum}
  float *values;   // [tile][head][part][query][hd]
};

template <int D, int KS, int QN, int QG, int KG, int KEYS, int STAGES, bool DMA>
__global__ __launch_bounds__(64 * QG * KG) __attribute__((amdgpu_waves_per_eu(KS > 8 ? 1 : D != FMT_F32 && KS == 5 && QG == 4 && DMA ? 3 : 2)))
void prompt_kernel(PromptArgs a, Parts parts) {
  using P = Prompt<D, KS, QN, QG, KG, KEYS, STAGES, DMA>;
  static_assert(QN == 1 || KG == 1, "one or the other");
  using Value = typename P::Value;
  constexpr bool F32 = P::F32;
  constexpr int V = P::V, C = P::C, DT = P::DT, PLANE = P::PLANE, QS = P::QS, HALVES = KEYS / 32;
  // The reference moves only when a score exceeds it by kLeap (in powers of two).
  // Weights lie higher by 2^kLift: in fp16 the largest is 2^15, and those below
  // 2^-36 of it (24.9 nats), the half of its smallest, vanish. Without that, 131071
  // keys 17.4 nats below one lost all of their 0.36%. The lift cancels in the division.
  constexpr bool HALF = D == FMT_F16;
  constexpr float kLeap = HALF ? 4.f : 8.f, kLift = HALF ? 11.f : 0.f;
  __shared__ __align__(16) uint4 lds[P::LDS];
  uint16_t *ones = reinterpret_cast<uint16_t *>(lds + P::TILES - P::SPAN);  // 1, 0, 0, 0; 0, 0, 0, 0
  if (P::ONES && threadIdx.x < 8) ones[threadIdx.x] = threadIdx.x ? 0 : D == FMT_F16 ? 0x3c00 : 0x3f80;

  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), qg = wave % QG, kg = wave / QG;
  int head, tile, part_at;
  block_of(a, parts.order, blockIdx.x, head, tile, part_at);
  const int split = parts.order.split;
  const Where w = find<P::QB>(a, tile);
  if (w.tile < 0) return;
  const int kvh = head / (a.heads / a.kv_heads);
  const int qb = w.tile * P::QB, qw = qb + qg * 32 * QN, mine = qw + col;  // within the sequence; mine + 32 n of set n
  const int shift = w.nk - w.nq;
  // the last key that this lane's queries, the wave's and the block's last ones
  // see, and the first ones'
  int last[QN];
#pragma unroll
  for (int n = 0; n < QN; n++) last[n] = a.causal ? min(mine + 32 * n, w.nq - 1) + shift : w.nk - 1;
  const int last_wave = a.causal ? min(qw + 32 * QN - 1, w.nq - 1) + shift : w.nk - 1;
  const int last_block = a.causal ? min(qb + P::QB - 1, w.nq - 1) + shift : w.nk - 1;
  const int first_wave = a.causal ? qw + shift : w.nk - 1;
  const int first_block = a.causal ? qb + shift : w.nk - 1;

  // Q^T as B operands: query l % 32, dims 16 step + 8 g .. + 7 (fp32: a chunk 8
  // step + 4 g .. + 3, one value a product). A negative scale turns their signs.
  uint4 q[QN][QS];
#pragma unroll
  for (int n = 0; n < QN; n++) {
    const Value *p = static_cast<const Value *>(a.q) + (w.q0 + min(mine + 32 * n, w.nq - 1)) * a.ldq + (int64_t)head * a.hd;
    const uint32_t sign = a.scale < 0.f ? F32 ? 0x80000000u : 0x80008000u : 0u;
#pragma unroll
    for (int s = 0; s < QS; s++) {
      const int d = (2 * s + g) * V;
      q[n][s] = make_uint4(0, 0, 0, 0);
      if (d < a.hd) {
        const u32x4_any x = *reinterpret_cast<const u32x4_any *>(p + d);
        q[n][s] = make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign);
      }
    }
  }
  f32x16 o[QN][DT];
#pragma unroll
  for (int n = 0; n < QN; n++)
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
      for (int v = 0; v < 16; v++) o[n][t][v] = 0.f;
  // Softmax weights are 2^(s scale - ref). sum: of the lane's own keys.
  float ref[QN], sum[QN];
#pragma unroll
  for (int n = 0; n < QN; n++) ref[n] = -INFINITY, sum[n] = 0.f;
  const float scale = fmaxf(fabsf(a.scale) * kLog2e, 1e-37f);  // (of zero: all weights alike)

  // ---- staging. A group's QG waves load its tile, K by their first half and V by the other.
  constexpr int PARTS = QG == 1 ? 1 : QG / 2;              // waves of a plane
  constexpr int N = PLANE / 64 / PARTS, NS = QG == 1 ? 2 * N : N;  // loads of a wave
  static_assert(PLANE % (64 * PARTS) == 0, "whole loads");
  const Value *kp = static_cast<const Value *>(a.k) + (int64_t)w.k0 * a.ldk + (int64_t)kvh * a.hd;
  const Value *vp = static_cast<const Value *>(a.v) + (int64_t)w.k0 * a.ldv + (int64_t)kvh * a.hd;
  const bool second = QG > 1 && qg >= PARTS;               // (uniform: this wave loads V)
  const int part = QG == 1 ? 0 : qg % PARTS;
  constexpr uint32_t kNone = 0x80000000u;
  uint32_t voff[NS];                                       // bytes from the tile's first row
#pragma unroll
  for (int j = 0; j < NS; j++) {
    const bool vt = QG == 1 ? j >= N : second;
    const int e = (part * N + j % N) * 64 + lane, r = vt && !F32 ? v_key<C>(e / C) : e / C, c = vt ? chunk_at<D, C, true>(r, e % C) : chunk_at<D, C, false>(r, e % C);
    const int64_t ld = vt ? a.ldv : a.ldk;
    voff[j] = c * V < a.hd ? (uint32_t)((r * ld + c * V) * (int)sizeof(Value)) : kNone;
  }
  uint4 staged[DMA ? 1 : NS];
  // One of this wave's loads of the tile from key t0 on, or all; between the
  // products of a tile they cost no time of their own (eight in a row do, as
  // their addresses take).
  constexpr bool SPREAD = DMA && QG > 1 && STAGES == 2 && !F32 && NS == QS;
  auto source = [&](int t0) {
    const int left = min(max(w.nk - t0, 0), KEYS);
    const int64_t ld = second ? a.ldv : a.ldk;
    const Value *at = (second ? vp : kp) + (int64_t)t0 * ld;
    const uint32_t bytes = left ? (uint32_t)(((left - 1) * ld + a.hd) * (int)sizeof(Value)) : 0u;
    return plane_rsrc(uniform_ptr(reinterpret_cast<const uint8_t *>(at)), __builtin_amdgcn_readfirstlane((int)bytes));
  };
  auto load_one = [&](__amdgpu_buffer_rsrc_t from, int stage, int j) {
    const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4 *)(lds) +
                        (((stage * KG + kg) * 2 + second) * PLANE + part * N * 64) * 16 + j * 1024;
    // (as dma16, but without a clobber: reads of the tile at work may pass it)
    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff[j]), "s"(from), "{m0}"(__builtin_amdgcn_readfirstlane(to)));
  };
  auto load = [&](int t0, int stage) {  // the tile from key t0 on
    const int left = min(max(w.nk - t0, 0), KEYS);
    auto plane = [&](const Value *base, int64_t ld, int j0, bool vt) {
      const Value *at = base + (int64_t)t0 * ld;
      const uint32_t bytes = left ? (uint32_t)(((left - 1) * ld + a.hd) * (int)sizeof(Value)) : 0u;
      if constexpr (DMA) {
        const __amdgpu_buffer_rsrc_t rsrc = plane_rsrc(uniform_ptr(reinterpret_cast<const uint8_t *>(at)), __builtin_amdgcn_readfirstlane((int)bytes));
        const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4 *)(lds) +
                            (((stage * KG + kg) * 2 + vt) * PLANE + part * N * 64) * 16;
#pragma unroll
        for (int j = 0; j < N; j++) dma16(rsrc, voff[j0 + j], __builtin_amdgcn_readfirstlane(to + j * 1024));
      } else {
#pragma unroll
        for (int j = 0; j < N; j++) {
          staged[j0 + j] = make_uint4(0, 0, 0, 0);
          if (voff[j0 + j] < bytes) {
            const u32x4_any x = *reinterpret_cast<const u32x4_any *>(reinterpret_cast<const uint8_t *>(at) + voff[j0 + j]);
            staged[j0 + j] = make_uint4(x.x, x.y, x.z, x.w);
          }
        }
      }
    };
    if constexpr (QG == 1) {
      plane(kp, a.ldk, 0, false);
      plane(vp, a.ldv, N, true);
    } else {
      plane(second ? vp : kp, second ? a.ldv : a.ldk, 0, second);
    }
  };
  auto store = [&](int stage) {  // (not DMA)
#pragma unroll
    for (int j = 0; j < NS; j++) {
      const bool vt = QG == 1 ? j >= N : second;
      lds[((stage * KG + kg) * 2 + vt) * PLANE + (part * N + j % N) * 64 + lane] = staged[j];
    }
  };

  // this block's rounds of KG tiles
  int round = 0, rounds = last_block < 0 ? 0 : (last_block / KEYS + KG) / KG;
  if (split > 1) {
    const int each = (rounds + split - 1) / split;
    round = min(part_at * each, rounds);
    rounds = min(round + each, rounds);
  }
  const int round0 = round;
  bool bad = false;
  if (round < rounds) {
    load((round * KG + kg) * KEYS, 0);
    if constexpr (!DMA) store(0);
  }
  for (; round < rounds; round++) {
    const int t0 = (round * KG + kg) * KEYS, stage = STAGES == 2 ? (round - round0) & 1 : 0;
    if constexpr (DMA) wait_vmcnt<0>();
    __syncthreads();
    const bool more = round + 1 < rounds;
    if (STAGES == 2 && more && !SPREAD) load(t0 + KG * KEYS, stage ^ 1);
    const bool active = qw < w.nq && t0 <= last_wave;
    __amdgpu_buffer_rsrc_t from;
    if constexpr (SPREAD) {  // (of no bytes past the last tile: zeros, that nobody reads)
      from = source(more ? t0 + KG * KEYS : w.nk);
      if (!active)
#pragma unroll
        for (int j = 0; j < NS; j++) load_one(from, stage ^ 1, j);
    }
    const uint4 *ks = lds + (stage * KG + kg) * 2 * PLANE;
    uint4 *vs = lds + ((stage * KG + kg) * 2 + 1) * PLANE;
    // A key that some query of the block does not see: its weight there is 0,
    // and 0 times an infinity or NaN would be one too. Such values are left out
    // of the products here and added to the queries that see them at the end.
    if (a.causal && ((round + 1) * KG) * KEYS - 1 > first_block) {
      bool found = false;
      for (int e = qg * 64 + lane; e < PLANE; e += 64 * QG) {
        uint4 x = vs[e];
        if (not_finite<D>(x)) vs[e] = only_finite<D>(x), found = true;
      }
      bad |= found;
      __syncthreads();
    }
    if (active) {
      f32x16 s[QN][HALVES];
#pragma unroll
      for (int n = 0; n < QN; n++)
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
          for (int v = 0; v < 16; v++) s[n][h][v] = 0.f;
#pragma unroll
      for (int st = 0; st < QS; st++) {
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
          const int r = h * 32 + col;
          const uint4 x = ks[r * C + k_place<C>(r, 2 * st + g)];
#pragma unroll
          for (int n = 0; n < QN; n++) {
            const uint4 y = q[n][st];
            if constexpr (F32) {
              s[n][h] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.x), __uint_as_float(y.x), s[n][h], 0, 0, 0);
              s[n][h] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.y), __uint_as_float(y.y), s[n][h], 0, 0, 0);
              s[n][h] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.z), __uint_as_float(y.z), s[n][h], 0, 0, 0);
              s[n][h] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.w), __uint_as_float(y.w), s[n][h], 0, 0, 0);
            } else {
              s[n][h] = mfma<D>(x, y, s[n][h]);
            }
          }
        }
        if constexpr (SPREAD) load_one(from, stage ^ 1, st);
      }
      if constexpr (!F32 && KS != 5) {  // operands come some products ahead
        constexpr int M = QS * HALVES, AHEAD = M < 6 ? M : 6;
        __builtin_amdgcn_sched_group_barrier(kReads, AHEAD, 0);
#pragma unroll
        for (int i = 0; i < M - AHEAD; i++) {
          __builtin_amdgcn_sched_group_barrier(kProducts, QN, 0);
          __builtin_amdgcn_sched_group_barrier(kReads, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kProducts, AHEAD * QN, 0);
      }
      if (t0 + KEYS - 1 > first_wave) {  // some of the wave's queries do not see the whole tile
#pragma unroll
        for (int n = 0; n < QN; n++)
#pragma unroll
          for (int h = 0; h < HALVES; h++)
#pragma unroll
            for (int v = 0; v < 16; v++)
              if (t0 + h * 32 + (v >> 2) * 8 + g * 4 + (v & 3) > last[n]) s[n][h][v] = -INFINITY;
      }
      float top[QN];
      bool leap = false;
#pragma unroll
      for (int n = 0; n < QN; n++) {
        top[n] = s[n][0][0];
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
          for (int v = 0; v < 16; v++) top[n] = fmaxf(top[n], s[n][h][v]);
        top[n] = halves_max(top[n]) * scale;
        leap |= top[n] > ref[n] + kLeap;  // (at first always: -inf + 8 is -inf)
      }
      if (__any(leap)) {
#pragma unroll
        for (int n = 0; n < QN; n++) {
          const float next = fmaxf(ref[n], top[n]), fade = next == -INFINITY ? 1.f : exp2_hw(ref[n] - next);
          ref[n] = next;
          sum[n] *= fade;
#pragma unroll
          for (int t = 0; t < DT; t++)
#pragma unroll
            for (int v = 0; v < 16; v++) o[n][t][v] *= fade;
        }
      }
      float base[QN];
#pragma unroll
      for (int n = 0; n < QN; n++) base[n] = ref[n] == -INFINITY ? 0.f : kLift - ref[n];
      if constexpr (F32) {
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
          for (int v = 0; v < 16; v++) {
            const int r = h * 32 + (v >> 2) * 8 + g * 4 + (v & 3);
#pragma unroll
            for (int n = 0; n < QN; n++) {
              const float p = exp2_hw(fmaf(s[n][h][v], scale, base[n]));
              sum[n] += p;
#pragma unroll
              for (int t = 0; t < DT; t++)
                o[n][t] = __builtin_amdgcn_mfma_f32_32x32x2f32(reinterpret_cast<const float *>(vs + r * C)[t * 32 + col], p, o[n][t], 0, 0, 0);
            }
          }
      } else {
        // A step's eight weights, and its operands of V: those of the next step
        // are formed and read while one step's products run.
        constexpr int STEPS = HALVES * 2;
        auto weights = [&](int n, int i) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int v = 8 * (i & 1) + 2 * j;
            w[j] = pack2<D>(exp2_hw(fmaf(s[n][i >> 1][v], scale, base[n])), exp2_hw(fmaf(s[n][i >> 1][v + 1], scale, base[n])));
            if constexpr (!P::ONES) sum[n] = plus2<D>(w[j], sum[n]);
          }
          return make_uint4(w[0], w[1], w[2], w[3]);
        };
        auto operands = [&](int i, uint4(&x)[DT]) {
          const int r0 = (i >> 1) * 32 + (i & 1) * 16 + g * 4 + (lane & 15) / 4;
#pragma unroll
          for (int t = 0; t < DT; t++) {
            const int d = t * 32 + (lane >> 4 & 1) * 16 + (lane & 3) * 4;
            auto read = [&](int r) {
              const uint16_t *at = reinterpret_cast<const uint16_t *>(vs + (v_row<C>(r) * C + v_place<C>(r, d / 8))) + d % 8;
              if (P::ONES && t == DT - 1 && (lane & 16)) at = ones + ((lane & 3) ? 4 : 0);
              return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)at));
            };
            const uint2 lo = read(r0), hi = read(r0 + 8);
            x[t] = make_uint4(lo.x, lo.y, hi.x, hi.y);
          }
        };
        // (KS 5: in turn, which leaves registers for a third wave a SIMD: 1620 against 1680 us for 16381 tokens of 32 heads of 80)
        if constexpr (KS == 5) {
#pragma unroll
          for (int i = 0; i < STEPS; i++) {
            uint4 x[DT];
            const uint4 p = weights(0, i);
            operands(i, x);
#pragma unroll
            for (int t = 0; t < DT; t++) o[0][t] = mfma<D>(x[t], p, o[0][t]);
          }
        } else {
          uint4 x[2][DT], p[2][QN];
          operands(0, x[0]);
#pragma unroll
          for (int n = 0; n < QN; n++) p[0][n] = weights(n, 0);
#pragma unroll
          for (int i = 0; i < STEPS; i++) {
            __builtin_amdgcn_sched_barrier(0);
            if (i + 1 < STEPS) {
              operands(i + 1, x[(i + 1) & 1]);
#pragma unroll
              for (int n = 0; n < QN; n++) p[(i + 1) & 1][n] = weights(n, i + 1);
            }
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
              for (int n = 0; n < QN; n++) o[n][t] = mfma<D>(x[i & 1][t], p[i & 1][n], o[n][t]);
            if (i + 1 < STEPS) {
              __builtin_amdgcn_sched_group_barrier(kReads, 2 * DT, 0);
#pragma unroll
              for (int t = 0; t < DT * QN; t++) {
                __builtin_amdgcn_sched_group_barrier(kProducts, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kVector, 16 / DT, 0);
                __builtin_amdgcn_sched_group_barrier(kExponents, 8 / DT, 0);
              }
            }
          }
        }
      }
    }
    if constexpr (STAGES == 1) {
      if (more) {
        if constexpr (!DMA) load(t0 + KG * KEYS, 0);
        __syncthreads();
        if constexpr (DMA) load(t0 + KG * KEYS, 0);
      }
    }
    if constexpr (!DMA) {
      if (more) store(STAGES == 2 ? stage ^ 1 : 0);
    }
  }
  if constexpr (SPREAD) wait_vmcnt<0>();  // (the zeros' place is the groups' next)
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int n = 0; n < QN; n++) {
    if constexpr (P::ONES) sum[n] = lower_half(o[n][DT - 1][8]);  // row 16 of the last tile: lanes 0 .. 31's value 8
    else sum[n] = halves_sum(sum[n]);
  }
  Value *out = static_cast<Value *>(a.out) + (w.q0 + mine) * a.ldo + (int64_t)head * a.hd;
  // Of a part: this lane's query in the records.
  const int64_t record = (((int64_t)tile * a.heads + head) * split + part_at) * P::QB + qg * 32 * QN + col;
  const int fixed0 = max(first_block / (KG * KEYS), round0) * (KG * KEYS);
  auto finish = [&](int n, int t, f32x16 x, float inv) {
    if (mine + 32 * n >= w.nq) return;
    const int fixed1 = min(last[n], rounds * KG * KEYS - 1);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int d = t * 32 + j * 8 + g * 4;
      if (d >= a.hd) continue;
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = x[4 * j + i] * inv;
      if (bad)
        for (int r = fixed0; r <= fixed1; r++)
          for (int i = 0; i < 4; i++) {
            const float u = mx_load(D, vp, r * a.ldv + d + i);
            if ((__float_as_uint(u) & 0x7f800000u) == 0x7f800000u) y[i] += u;
          }
      if (split > 1) *reinterpret_cast<f32x4_any *>(parts.values + (record + 32 * n) * a.hd + d) = f32x4_any{y[0], y[1], y[2], y[3]};
      else if constexpr (F32) *reinterpret_cast<f32x4_any *>(out + 32 * n * a.ldo + d) = f32x4_any{y[0], y[1], y[2], y[3]};
      else *reinterpret_cast<u32x2_any *>(out + 32 * n * a.ldo + d) = u32x2_any{pack2<D>(y[0], y[1]), pack2<D>(y[2], y[3])};
    }
  };
  // what the sums are multiplied by, and a part's reference and sum
  auto ending = [&](int n, float top, float all, bool leader) {
    if (split == 1) return all == 0.f ? 0.f : 1.f / all;
    if (leader && g == 0 && mine + 32 * n < w.nq) parts.stats[record + 32 * n] = make_float2(top, all);
    return 1.f;
  };
  if constexpr (KG == 1) {
#pragma unroll
    for (int n = 0; n < QN; n++) {
      const float inv = ending(n, ref[n], sum[n], true);
#pragma unroll
      for (int t = 0; t < DT; t++) finish(n, t, o[n][t], inv);
    }
  } else {
    // [wave][reference, sum, values][lane]; a group of keys joins every KG-th tile of its queries'
    float *f = reinterpret_cast<float *>(lds) + lane;
    constexpr int W = (DT * 16 + 2) * 64;
    f[wave * W] = ref[0];
    f[wave * W + 64] = sum[0];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
      for (int v = 0; v < 16; v++) f[wave * W + (2 + t * 16 + v) * 64] = o[0][t][v];
    __syncthreads();
    float top = -INFINITY, fade[KG], all = 0.f;
#pragma unroll
    for (int i = 0; i < KG; i++) top = fmaxf(top, f[(i * QG + qg) * W]);
#pragma unroll
    for (int i = 0; i < KG; i++) {
      fade[i] = top == -INFINITY ? 0.f : exp2_hw(f[(i * QG + qg) * W] - top);
      all += fade[i] * f[(i * QG + qg) * W + 64];
    }
    const float inv = ending(0, top, all, kg == 0);
    for (int t = kg; t < DT; t += KG) {
      f32x16 x;
#pragma unroll
      for (int v = 0; v < 16; v++) {
        x[v] = 0.f;
#pragma unroll
        for (int i = 0; i < KG; i++) x[v] += fade[i] * f[(i * QG + qg) * W + (2 + t * 16 + v) * 64];
      }
      finish(0, t, x, inv);
    }
  }
}

}  // namespace

namespace {

// The parts of a query, joined in order; four dims a thread.
template <int QB>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs a, Parts p) {
  const int tile = blockIdx.x / a.heads, head = blockIdx.x % a.heads, split = p.order.split;
  const Where w = find<QB>(a, tile);
  if (w.tile < 0) return;
  const int wide = a.hd / 4;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < QB * wide; i += gridDim.y * 256) {
    const int row = i / wide, d = i % wide * 4, mine = w.tile * QB + row;
    if (mine >= w.nq) return;
    const int64_t first = ((int64_t)tile * a.heads + head) * split * QB + row;
    float top = -INFINITY, sum = 0.f;
    for (int s = 0; s < split; s++) top = fmaxf(top, p.stats[first + s * QB].x);
    float o[4] = {};
#pragma unroll 4
    for (int s = 0; s < split; s++) {
      const float2 x = p.stats[first + s * QB];
      const f32x4_any v = *reinterpret_cast<const f32x4_any *>(p.values + (first + s * QB) * a.hd + d);
      const float fade = top == -INFINITY ? 0.f : exp2_hw(x.x - top);
      sum += fade * x.y;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] += fade * v[j];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int j = 0; j < 4; j++) mx_store(a.dtype, a.out, (w.q0 + mine) * a.ldo + (int64_t)head * a.hd + d + j, o[j] * inv);
  }
}

// How a call is run: query groups, key groups of a block, parts of the keys.
struct Shape {
  int qg, kg, split, qn = 1;
  int queries() const { return 32 * qg * qn; }  // of a block
};
int64_t tiles_of(const PromptArgs &a, int qb) {  // at most: every sequence's last tile may be a part
  return a.nq / qb + std::min<int64_t>(a.sequences, a.nq);
}
// Two blocks of 128 queries a CU are 512. Fewer than 256 leave CUs idle: there
// the keys are cut, into parts of 1024 at least where they are long (a join costs
// 7 us), else over a block's waves (512 queries of 32 heads of 80: 10.7 us).
Shape shape_of(const PromptArgs &a) {
  Shape s{4, 1, 1};
  const int64_t blocks = tiles_of(a, 128) * a.heads, keys = a.nk / std::max(1, std::min(a.sequences, a.nk));
  if (a.dtype != FMT_F32 && a.hd <= 64 && tiles_of(a, 256) * a.heads >= 512) s.qn = 2;
  if (blocks >= 256) return s;
  if (a.dtype == FMT_F32) {
    s = Shape{1, a.hd > 128 ? 2 : 4, 1};
    const int64_t few = tiles_of(a, 32) * a.heads;
    s.split = (int)std::min(512 / few, (keys + 32 * s.kg - 1) / (32 * s.kg));
  } else if (keys >= 2048 && blocks <= 256) {
    s.split = (int)std::min(512 / blocks, keys / 1024);
  } else if (a.nq <= 32) {
    s = Shape{1, 4, 1};
  } else if (a.hd <= 128) {
    s = Shape{2, 4, 1};
  }
  if (s.split < 1) s.split = 1;
  return s;
}

template <int D, int KS, int QN, int QG, int KG, int KEYS, int STAGES>
void launch(const PromptArgs &a, const Parts &p, bool dma, hipStream_t st) {
  const dim3 grid((unsigned)(p.order.tiles * p.order.split * a.heads)), block(64 * QG * KG);
  if (dma) hipLaunchKernelGGL((prompt_kernel<D, KS, QN, QG, KG, KEYS, STAGES, true>), grid, block, 0, st, a, p);
  else hipLaunchKernelGGL((prompt_kernel<D, KS, QN, QG, KG, KEYS, STAGES, false>), grid, block, 0, st, a, p);
}

bool aligned16(const void *p, int64_t ld, int width) { return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * width)) % 16 == 0; }

}  // namespace

size_t prompt_scratch(const PromptArgs &a) {
  const Shape s = shape_of(a);
  return s.split == 1 ? 0 : (size_t)tiles_of(a, s.queries()) * a.heads * s.split * s.queries() * (a.hd + 2) * 4;
}

hipError_t launch_prompt(const PromptArgs &a, void *scratch, hipStream_t st) {
  const int width = (int)mx_width(a.dtype);
  const bool dma = aligned16(a.k, a.ldk, width) && aligned16(a.v, a.ldv, width);
  const Shape s = shape_of(a);
  const int64_t tiles = tiles_of(a, s.queries());
  Parts p{{(int)tiles, s.split}, nullptr, static_cast<float *>(scratch)};
  if (s.split > 1) p.stats = reinterpret_cast<float2 *>(p.values + tiles * a.heads * s.split * s.queries() * a.hd);
  auto go = [&](auto d, auto k) {
    constexpr int D = decltype(d)::value, KS = decltype(k)::value;
    constexpr bool wide = KS > 8;
    if constexpr (D == FMT_F32) {
      if (s.qg == 1) launch<D, KS, 1, 1, wide ? 2 : 4, 32, KS <= 4 ? 2 : 1>(a, p, dma, st);
      else launch<D, KS, 1, 4, 1, 32, wide ? 1 : 2>(a, p, dma, st);
    } else {
      if (s.qg == 1) launch<D, KS, 1, 1, 4, 32, wide ? 1 : 2>(a, p, dma, st);
      else if (s.qg == 2) launch<D, KS, 1, wide ? 4 : 2, wide ? 1 : 4, 32, 2>(a, p, dma, st);
      else if (s.qn == 2) launch<D, KS, KS <= 4 ? 2 : 1, 4, 1, wide ? 32 : 64, 2>(a, p, dma, st);
      else launch<D, KS, 1, 4, 1, wide ? 32 : 64, 2>(a, p, dma, st);
    }
  };
  for_type(a.dtype, [&](auto d) {
    if (a.hd <= 32) go(d, std::integral_constant<int, 2>());
    else if (a.hd <= 64) go(d, std::integral_constant<int, 4>());
    else if (a.hd <= 80) go(d, std::integral_constant<int, 5>());
    else if (a.hd <= 96) go(d, std::integral_constant<int, 6>());
    else if (a.hd <= 128) go(d, std::integral_constant<int, 8>());
    else go(d, std::integral_constant<int, 16>());
  });
  if (s.split > 1) {
    const dim3 grid((unsigned)(tiles * a.heads), (unsigned)((s.queries() * a.hd / 4 + 255) / 256));
    if (s.qg == 1) hipLaunchKernelGGL((prompt_join_kernel<32>), grid, dim3(256), 0, st, a, p);
    else hipLaunchKernelGGL((prompt_join_kernel<128>), grid, dim3(256), 0, st, a, p);
  }
  return hipGetLastError();
}
