// Attention of one new token of each sequence over its pages:
//   s_j = scale q . k_j,  o = sum_j 2^(s_j' - m) v_j / sum_j 2^(s_j' - m),
// s' = s log2 e and m a running reference, in one pass over the positions
// (softmax weights are then single 2^x instructions). Positions from the
// sequence's length on, and those of table entries outside the pool, are not
// read; a sequence without positions gets zeros.
//
// What bounds it: HBM, every key and value read once. A row of K meets few
// queries (the heads that share it), but both products still go to the matrix
// cores, transposed as in the prompts' kernel, with the queries as the 16
// columns of a 16 x 16 tile:
//   S^T = K Q^T,  O^T += V^T P.
// Their time is far below the loads', columns that no head fills included, and
// K and V then need no lane of their own: the pages' rows, which lie one after
// another, go to LDS by DMA as they lie, and fragments are read from there.
//
// The queries and the weights keep fp32 accuracy as planes: sums of two or
// three values of the matrix cores' type (fp16 for an fp16 cache, the queries
// scaled by a power of two; bf16 for bf16 and 8-bit ones, whose codes bf16 holds
// exactly: scores and weights take the blocks' scales in fp32). An fp32 cache
// multiplies on the fp32 matrix instructions. An infinity of a 16-bit cache meets
// every plane, and a plane may be zero or of the other sign: it gives NaN where
// the value itself gives an infinity or no weight. Sums that are not finite tell,
// and such a piece, where its rows hold an infinity, is done again in plain fp32
// (64 requests of 3000 positions, 32 over 8 fp16 heads of 128: 154 us, with an
// infinity in two pages 1.29 ms, with a NaN there 224 us; the test costs less than 1%).
//
// Lengths are known on the device alone, so the waves deal out the work
// themselves: all positions of all pairs (of a sequence and up to 16 query heads
// of a key head) in a row, in units of 32, and each wave takes an equal run of
// them. It goes through its run in tiles of 32 positions (fp32: 16), whatever
// pairs they belong to, in its own two LDS buffers, K's and V's: the next K is
// in flight during the softmax and the product with V, the next V during the
// scores. Waves never meet. A pair that lies within one run goes out at once;
// the pieces of others leave unnormalised records {m, sum, o}, two a wave at
// most, which a second kernel joins in order.
//
// Two contexts of 131071 positions (8 fp16 key heads of 64): 104 us, 5.2 TB/s (a
// copy on this card: 4.9). 64 requests of up to 4096 (32 over 8 bf16 heads of
// 128): 31 to 45 us with the lengths drawn, 28 the floor of their mean. 8-bit
// pages, 32 requests of up to 2048 (22 heads of 128, fp32 queries): 28 to 35 us,
// bound by the codes' and planes' vector work (660 instructions a tile). One
// request of 700 positions (32 heads of 80): 11 us, two launches' latencies. With
// ranges of a fixed length for each block instead of equal runs for each wave the
// first took 112 (1024 blocks' worth) to 157 us, the second 46 to 81.
#include <type_traits>

#include "attend.h"
#include "mx_tile.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ void store4(int dtype, void *p, int64_t i, f32x4 v) {
  if (dtype == FMT_F32) {
    *reinterpret_cast<f32x4_any *>(static_cast<float *>(p) + i) = f32x4_any{v[0], v[1], v[2], v[3]};
  } else {
    const u32x2_any w = {mx_narrow(dtype, v[0]) | (uint32_t)mx_narrow(dtype, v[1]) << 16, mx_narrow(dtype, v[2]) | (uint32_t)mx_narrow(dtype, v[3]) << 16};
    *reinterpret_cast<u32x2_any *>(static_cast<uint16_t *>(p) + i) = w;
  }
}

constexpr int kUnit = 32;  // positions: what the work is dealt out by

struct Plan {
  int waves;            // of the launch
  int qtiles, columns;  // tiles of 16 query heads of a key head; heads of a tile, at most
  int by_pair;          // how `ends` is kept: for each pair, else for each wave
  // Scratch. What the join has to do for the pair that ends in a wave's run
  // (its last piece is that wave's first): `from` is the wave with its first
  // piece, which lies in its place `place`; last -1: nothing.
  struct End {
    int seq, pair, from, place, last;
  } * ends;
  // The pieces: [wave][0: its first, 1: its last][head of the tile], {m, sum} and o[hd].
  float2 *stats;
  float *values;
};

// CT: the cache's type; KS: steps of 32 dims; PL: planes of the queries (3: fp32, 1:
// as the matrix cores take them, 2: the other 16-bit type; fp32 caches: any type).
template <int CT, int KS, int PL>
struct Attend {
  static constexpr bool F32 = CT == FMT_F32, Q8 = CT == FMT_Q8_0, F16 = CT == FMT_F16;
  // The queries' type. It is the instance's: with a branch on the argument where
  // they are read, the compiler left their address undefined behind one of its
  // sides, and a wave's next pairs read theirs from there.
  static constexpr int QT = PL == 3 ? FMT_F32 : PL == 1 ? (Q8 ? FMT_BF16 : CT) : F16 ? FMT_BF16 : FMT_F16;
  static constexpr int WAVES = KS == 8 ? 2 : 4;
  static constexpr int ROWS = F32 ? 16 : 32;                // positions of a tile
  static constexpr int C = KS * (F32 ? 8 : Q8 ? 2 : 4);     // chunks of a row in LDS
  static constexpr int NB = KS == 1 ? 2 : KS == 3 ? 4 : KS; // scales of a row
  static constexpr int PLANE = ROWS * C;                    // chunks
  static constexpr int N = (PLANE + 63) / 64;               // loads of a plane
  static constexpr int NSC = Q8 ? (16 * NB + 63) / 64 : 0;  // of its scales
  static constexpr int SCALES = NSC * 16;                   // chunks
  static constexpr int SIDE = N * 64 + SCALES;              // chunks of a tile's K or V
  static constexpr int LOADS = N + NSC;                     // of a side
  static constexpr int DT = KS * 2;                         // 16-dim tiles of O^T
  static constexpr int PP = PL == 3 ? 3 : 2;                // planes of the weights
  static constexpr int LDS = WAVES * 2 * SIDE;
  static_assert(LDS * 16 <= 160 * 1024, "LDS of a CU");
  static_assert(LOADS < 64, "loads in flight");
};

// The planes of eight values, packed; their sum is the value to 8 (bf16) or 11
// bits a plane. WEIGHTS: never infinite (a NaN gives one in any case), which
// spares the tests that keep an infinity from becoming one.
template <int CT, bool WEIGHTS, int P>
__device__ __forceinline__ void planes_of8(const float (&v)[8], uint4 (&out)[P]) {
  if constexpr (CT == FMT_F16) {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; j++) rest[j] = v[j];
#pragma unroll
    for (int p = 0; p < P; p++) {
      f16x8 h;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        float x = rest[j];
        asm volatile("" : "+v"(x));  // one value, rounded once: not a product's own rounding here and its value below
        h[j] = (_Float16)x;
        rest[j] = x - (float)h[j];
      }
      out[p] = __builtin_bit_cast(uint4, h);
    }
  } else {
    uint32_t h[8][P];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if constexpr (WEIGHTS) {
        float rest = v[j];
#pragma unroll
        for (int p = 0; p < P; p++) {
          h[j][p] = __float_as_uint(rest) & 0xffff0000u;
          rest -= __uint_as_float(h[j][p]);
        }
      } else {
        tinyoai_mx::planes_of<P>(v[j], h[j]);
      }
    }
#pragma unroll
    for (int p = 0; p < P; p++)
      out[p] = make_uint4(tinyoai_mx::high_halves(h[0][p], h[1][p]), tinyoai_mx::high_halves(h[2][p], h[3][p]),
                          tinyoai_mx::high_halves(h[4][p], h[5][p]), tinyoai_mx::high_halves(h[6][p], h[7][p]));
  }
}
template <int CT>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
  if constexpr (CT == FMT_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Eight codes as bf16, exactly.
__device__ __forceinline__ uint4 codes_bf16(uint32_t lo, uint32_t hi) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; j++) v[j] = (float)(int8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
  auto two = [&](int j) { return tinyoai_mx::high_halves(__float_as_uint(v[j]), __float_as_uint(v[j + 1])); };
  return make_uint4(two(0), two(2), two(4), two(6));
}

template <int CT, int KS, int PL>
__global__ __launch_bounds__(KS == 8 ? 128 : 256) __attribute__((amdgpu_waves_per_eu(KS == 1 ? 4 : KS == 2 ? 3 : KS == 8 ? 1 : 2)))
void attend_kernel(AttendArgs a, Plan plan) {
  using A = Attend<CT, KS, PL>;
  constexpr bool F32 = A::F32, Q8 = A::Q8, F16 = A::F16;
  constexpr int WAVES = A::WAVES, ROWS = A::ROWS, C = A::C, NB = A::NB, N = A::N, DT = A::DT, PP = A::PP;
  constexpr float kLeap = 8.f;              // the reference moves only when a score exceeds it by 2^8
  constexpr float kLift = F16 ? 7.f : 0.f;  // fp16 weights lie higher by 2^7, their smallest planes in range
  __shared__ __align__(16) uint4 lds[A::LDS];

  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hd = a.c.hd, group = a.heads / a.c.kv_heads, lg = a.c.page_log2;
  const int64_t most = (int64_t)a.width << lg;
  uint4 *mine = lds + wave * 2 * A::SIDE;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4 *)(mine);

  // Where this lane's pieces of a tile lie: row of the tile, byte within the row.
  constexpr uint32_t kNone = 0x80000000u;
  uint32_t koff[N], voff[N];
#pragma unroll
  for (int j = 0; j < N; j++) {
    const int e = j * 64 + lane, r = e / C, p = e % C;
    const int kc = k_place<C>(r, p), vc = F32 ? p ^ ((r >> 2 & 1) << 2) : v_place<C>(r, p);
    koff[j] = r < ROWS && kc * 16 < a.c.pitch ? (uint32_t)(r * a.c.pitch + kc * 16) : kNone;
    voff[j] = r < ROWS && vc * 16 < a.c.pitch ? (uint32_t)(r * a.c.pitch + vc * 16) : kNone;
  }

  // The units of a sequence; a lane each of 64 sequences at a time.
  const int per = a.c.kv_heads * plan.qtiles;
  int first = 0, len = 0;  // the window's first sequence; of the lane's: its length
  uint32_t upto = 0;       // and the units up to its end (64 of the longest: 2^31)
  auto units_of = [&](int length) { return max((length + kUnit - 1) / kUnit, 1); };  // (one to write zeros)
  auto length_of = [&](int s) { return s < a.n ? (int)min((int64_t)max(a.lengths[s], 0), most) : -1; };
  auto window = [&]() {
    len = length_of(first + lane);
    upto = len < 0 ? 0u : (uint32_t)units_of(len);
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const uint32_t x = __shfl_up(upto, off);
      if (lane >= off) upto += x;
    }
  };
  auto uniform = [](int64_t x) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
  };
  window();
  auto upto_of = [&](int l) { return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)upto, l); };
  int64_t all_units = upto_of(63);
  if (a.n > 64) {
    double sum = 0;  // (exact: below 2^53)
    for (int s = 64 + lane; s < a.n; s += 64) sum += units_of(length_of(s));
    all_units += (int64_t)wave_total_d(sum);
  }
  // The wave's run of the T units, u .. u + left - 1, and where it is.
  const int64_t T = uniform(all_units * per);
  const int G = (int)min(T, (int64_t)plan.waves), b = blockIdx.x * WAVES + wave;
  if (b >= G) {
    if (!plan.by_pair && lane == 0) plan.ends[b].last = -1;
    return;
  }
  int64_t u = uniform(b * T / G), left = uniform((b + 1) * T / G) - u;
  int at, length, units, pair, unit;  // the sequence within the window, its length and units, the pair and unit within it
  {
    const int64_t at_units = uniform(u / per);
    int64_t before = 0;  // units before the window
    while (at_units >= before + upto_of(63)) before += upto_of(63), first += 64, window();
    at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(before + upto > at_units)));
    length = __builtin_amdgcn_readlane(len, at);
    units = units_of(length);
    const int64_t local = uniform(u - (before + upto_of(at) - units) * per);
    pair = __builtin_amdgcn_readfirstlane((int)(local / units));
    unit = __builtin_amdgcn_readfirstlane((int)(local % units));
  }
  // A piece of the run: positions start .. end - 1 of a pair; place -1: all of it.
  struct Piece {
    int seq, kvh, q0, start, end, place;
  };
  bool begun = false;
  auto next_piece = [&](Piece &p) {
    while (left > 0) {
      const int count = __builtin_amdgcn_readfirstlane((int)min((int64_t)(units - unit), left));
      p = Piece{first + at, pair / plan.qtiles, pair % plan.qtiles * 16, unit * kUnit, min(length, (unit + count) * kUnit),
                count == units ? -1 : begun ? 1 : 0};
      if (unit + count == units) {  // the pair's end
        Plan::End e{p.seq, pair, 0, 0, -1};
        if (count < units) {
          const int64_t f = u - unit;  // its first unit, in the run of wave ceil((f + 1) G / T) - 1
          e.from = (int)(((f + 1) * G + T - 1) / T - 1);
          e.place = e.from * T / G == f ? 0 : 1;
          e.last = b;
        }
        if (lane == 0 && (plan.by_pair || e.last >= 0)) plan.ends[plan.by_pair ? p.seq * per + pair : b] = e;
      }
      if (!begun && !plan.by_pair && (unit + count < units || count == units) && lane == 0) plan.ends[b].last = -1;
      begun = true;
      u += count, left -= count;
      unit = 0;
      if (++pair == per && left > 0) {
        pair = 0;
        if (++at == 64) at = 0, first += 64, window();
        length = __builtin_amdgcn_readlane(len, at);
        units = units_of(length);
      }
      if (p.end > p.start) return true;
      if (p.q0 + col < group)  // nothing to attend to
        for (int d = g * 4; d < hd; d += 16) {
          const int64_t to = p.seq * a.ldo + (int64_t)(p.kvh * group + p.q0 + col) * hd + d;
          store4(a.dtype, a.out, to, f32x4{0.f, 0.f, 0.f, 0.f});
        }
    }
    return false;
  };
  Piece now, next;
  if (!next_piece(now)) return;
  next = now;

  // Table entries of the piece whose loads are started: a lane each from page `wb` on.
  int wb = 0, entry = -1;
  auto entries = [&](const Piece &p, int page) {
    wb = page;
    entry = ((int64_t)(wb + lane) << lg) < p.end ? a.table[(int64_t)p.seq * a.width + wb + lane] : -1;
  };
  // Starts the loads of K or V of a piece's tile from position t0 on; returns which of its positions count.
  auto issue = [&](const Piece &p, int t0, auto value) {
    const int we = p.end, kvh = p.kvh;
    constexpr bool VT = decltype(value)::value;
    if (((t0 + ROWS - 1) >> lg) - wb >= 64) entries(p, t0 >> lg);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + (VT ? A::SIDE * 16 : 0));
    const uint32_t(&off)[N] = VT ? voff : koff;
    const uint8_t *base = VT ? a.c.v : a.c.k;
    const uint16_t *scales = VT ? a.c.vd : a.c.kd;
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): what was read of this buffer has arrived
    if ((1 << lg) >= ROWS) {             // within one page
      const int page = __builtin_amdgcn_readlane(entry, (t0 >> lg) - wb);
      const int count = __builtin_amdgcn_readfirstlane((uint32_t)page < (uint32_t)a.c.pages ? min(we - t0, ROWS) : 0);
      const int64_t row = kv_row(a.c, (count ? page : 0) << lg | (t0 & ((1 << lg) - 1)), kvh);
      const __amdgpu_buffer_rsrc_t rows = plane_rsrc(uniform_ptr(base + row * a.c.pitch), count * a.c.pitch);
#pragma unroll
      for (int j = 0; j < N; j++) dma16(rows, off[j], __builtin_amdgcn_readfirstlane(to + j * 1024));
      if constexpr (Q8) {
        const __amdgpu_buffer_rsrc_t sc = plane_rsrc(uniform_ptr(reinterpret_cast<const uint8_t *>(scales + row * NB)), count * NB * 2);
#pragma unroll
        for (int j = 0; j < A::NSC; j++) dma4(sc, (j * 64 + lane) * 4, __builtin_amdgcn_readfirstlane(to + N * 1024 + j * 256));
      }
      return count >= 32 ? 0xffffffffu : (1u << count) - 1u;
    }
    // rows of several pages: an address per lane
    auto row_of = [&](int r, bool &ok) {
      const int t = t0 + r, page = __shfl(entry, (t >> lg) - wb);
      ok = r < ROWS && t < we && (uint32_t)page < (uint32_t)a.c.pages;
      return ok ? kv_row(a.c, page << lg | (t & ((1 << lg) - 1)), kvh) - r : 0;  // the row before the tile's first, were it one run
    };
#pragma unroll
    for (int j = 0; j < N; j++) {
      bool ok;
      const int64_t row = row_of((j * 64 + lane) / C, ok) * a.c.pitch;
      dma16_at(ok && off[j] != kNone ? base + row + off[j] : a.c.zeros, __builtin_amdgcn_readfirstlane(to + j * 1024));
    }
    if constexpr (Q8) {
#pragma unroll
      for (int j = 0; j < A::NSC; j++) {
        const int e = j * 64 + lane;  // a pair of scales
        bool ok;
        const int64_t row = row_of(e * 2 / NB, ok) * NB;
        dma4_at(ok ? (const void *)(scales + row + e * 2) : a.c.zeros, __builtin_amdgcn_readfirstlane(to + N * 1024 + j * 256));
      }
    }
    bool ok;
    row_of(lane & 31, ok);
    return (uint32_t)__ballot(ok);
  };
  // The scales of rows 16 h + 4 g .. + 3 (of a tile's K or V): [row][block].
  auto scales_of = [&](const uint4 *at, int h, float (&d)[4 * NB]) {
    const uint4 *from = at + (h * 16 + g * 4) * NB / 8;
#pragma unroll
    for (int i = 0; i < NB / 2; i++) {
      const uint4 x = from[i];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; j++) d[8 * i + 2 * j] = hw_half((uint16_t)w[j]), d[8 * i + 2 * j + 1] = hw_half((uint16_t)(w[j] >> 16));
    }
  };

  // Q^T as B operands: column l % 16, dims 32 step + 8 g .. + 7 (fp32: 16 step + 4 g .. + 3).
  constexpr int QS = F32 ? 2 * KS : KS;
  uint4 q[QS][F32 ? 1 : PL];
  float scale;
  auto queries = [&](const Piece &pc) {
    scale = a.scale * kLog2e;
    const bool live = pc.q0 + col < group;
    const int64_t from = pc.seq * a.ldq + (int64_t)(pc.kvh * group + min(pc.q0 + col, group - 1)) * hd;
    if constexpr (F32) {
#pragma unroll
      for (int s = 0; s < QS; s++) {
        const int d = s * 16 + g * 4;
        float v[4] = {};
        if (live && d < hd)
#pragma unroll
          for (int j = 0; j < 4; j++) v[j] = mx_load(a.dtype, a.q, from + d + j);
        q[s][0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      }
    } else if constexpr (PL == 1) {  // the cache's own type
#pragma unroll
      for (int s = 0; s < QS; s++) {
        const int d = s * 32 + g * 8;
        q[s][0] = make_uint4(0, 0, 0, 0);
        if (live && d < hd) {
          const u32x4_any x = *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(a.q) + from + d);
          q[s][0] = make_uint4(x.x, x.y, x.z, x.w);
        }
      }
    } else {
      float v[QS][8];
      float big = 0.f;
#pragma unroll
      for (int s = 0; s < QS; s++) {
        const int d = s * 32 + g * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) v[s][j] = 0.f;
        if (live && d < hd) load8<A::QT>(a.q, from + d, v[s]);
#pragma unroll
        for (int j = 0; j < 8; j++) big = fmaxf(big, fabsf(v[s][j]));
      }
      if constexpr (F16) {  // the row's largest below 2^15
        big = quarters_max(big);
        int e = 0;
        if (big > 0.f && big < INFINITY) e = 15 - ((int)(__float_as_uint(big) >> 23) - 126);
        e = min(max(e, -120), 120);
#pragma unroll
        for (int s = 0; s < QS; s++)
#pragma unroll
          for (int j = 0; j < 8; j++) v[s][j] = ldexpf(v[s][j], e);
        scale = ldexpf(scale, -e);
      }
#pragma unroll
      for (int s = 0; s < QS; s++) planes_of8<CT, false>(v[s], q[s]);
    }
  };

  f32x4 o[DT];
  float ref, sum;
  auto reset = [&]() {
    ref = -INFINITY, sum = 0.f;
#pragma unroll
    for (int t = 0; t < DT; t++) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  // ---- pieces with infinities (16-bit caches)
  // A copy of x that the compiler does not know: addresses of a path that is hardly ever
  // taken are formed there, and not kept in registers throughout the loop.
  auto anew = [](int x) {
    asm volatile("" : "+v"(x));
    return x;
  };
  // The row of a piece's position t; -1: it does not count.
  auto row_at = [&](const Piece &p, int t) {
    const int page = a.table[(int64_t)p.seq * a.width + (t >> lg)];
    return (uint32_t)page < (uint32_t)a.c.pages ? kv_row(a.c, page << lg | (t & ((1 << lg) - 1)), p.kvh) : (int64_t)-1;
  };
  auto holds_infinity = [&](const Piece &p) {
    constexpr uint32_t kInf = F16 ? 0x7c00u : 0x7f80u;
    bool found = false;
#pragma unroll 1
    for (int t = p.start + anew(lane); t < p.end; t += 64) {
      const int64_t row = row_at(p, t);
      if (row < 0) continue;
#pragma unroll 1
      for (int at = 0; at < hd * 2; at += 16)
        for (const uint8_t *side : {a.c.k, a.c.v}) {
          const uint4 x = *reinterpret_cast<const uint4 *>(side + row * a.c.pitch + at);
          for (uint32_t w : {x.x, x.y, x.z, x.w}) found |= (w & 0x7fffu) == kInf || (w >> 16 & 0x7fffu) == kInf;
        }
    }
    return __any(found) != 0;
  };
  // The piece's sums by the formula, position after position; lane g of a column takes every fourth eight dims of a score.
  auto in_fp32 = [&](const Piece &p) {
    reset();
    const int part = anew(g);
    const int64_t from = p.seq * a.ldq + (int64_t)(p.kvh * group + min(p.q0 + anew(col), group - 1)) * hd;
#pragma unroll 1
    for (int t = p.start; t < p.end; t++) {
      const int64_t row = row_at(p, t);
      if (row < 0) continue;
      float x = 0.f;
#pragma unroll 1
      for (int d = part * 8; d < hd; d += 32) {
        float k[8], q[8];
        load8<CT>(a.c.k + row * a.c.pitch, d, k);
        load8<A::QT>(a.q, from + d, q);
#pragma unroll
        for (int j = 0; j < 8; j++) x = fmaf(q[j], k[j], x);
      }
      x = quarters_sum(x) * (a.scale * kLog2e);
      const float next = fmaxf(ref, x), base = next == -INFINITY ? 0.f : next;
      const float fade = exp2_hw(ref - base), w = exp2_hw(x - base);
      ref = next;
      sum = sum * fade + (part == 0 ? w : 0.f);
#pragma unroll
      for (int i = 0; i < DT; i++) {
        const int d = i * 16 + part * 4;
        if (d >= hd) continue;
        const uint2 v = *reinterpret_cast<const uint2 *>(a.c.v + row * a.c.pitch + d * 2);
        const uint16_t h[4] = {(uint16_t)v.x, (uint16_t)(v.x >> 16), (uint16_t)v.y, (uint16_t)(v.y >> 16)};
#pragma unroll
        for (int j = 0; j < 4; j++) o[i][j] = fmaf(w, F16 ? hw_half(h[j]) : bf16_to_float(h[j]), o[i][j] * fade);
      }
    }
    ref += kLift;  // (what these weights do not have)
  };
  reset();
  entries(now, now.start >> lg);
  uint32_t seen = issue(now, now.start, std::false_type());
  issue(now, now.start, std::true_type());
  queries(now);
  const uint4 *ks = mine, *vs = mine + A::SIDE;
  for (int t0 = now.start;;) {
    // K has landed (V may be in flight), later V (the next K may be)
    wait_vmcnt<A::LOADS>();
    constexpr int H = ROWS / 16;
    // scores of the positions 16 h + 4 g + i
    float s[H][4];
#pragma unroll
    for (int h = 0; h < H; h++) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      const int r = h * 16 + col;
      float d[Q8 ? 4 * NB : 1];
      if constexpr (Q8) scales_of(ks + N * 64, h, d);
#pragma unroll
      for (int st = 0; st < QS; st++) {
        if constexpr (F32) {
          const uint4 k = ks[r * C + k_place<C>(r, 4 * st + g)];
          const uint4 y = q[st][0];
          x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.x), __uint_as_float(y.x), x, 0, 0, 0);
          x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.y), __uint_as_float(y.y), x, 0, 0, 0);
          x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.z), __uint_as_float(y.z), x, 0, 0, 0);
          x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.w), __uint_as_float(y.w), x, 0, 0, 0);
        } else if constexpr (Q8) {
          const uint2 w = reinterpret_cast<const uint2 *>(ks + r * C + k_place<C>(r, 2 * st + (g >> 1)))[g & 1];
          const uint4 k = codes_bf16(w.x, w.y);
          f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = 0; p < PL; p++) y = mfma16<CT>(k, q[st][p], y);
#pragma unroll
          for (int i = 0; i < 4; i++) x[i] = fmaf(d[i * NB + st], y[i], x[i]);
        } else {
          const uint4 k = ks[r * C + k_place<C>(r, 4 * st + g)];
#pragma unroll
          for (int p = 0; p < PL; p++) x = mfma16<CT>(k, q[st][p], x);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) s[h][i] = x[i] * scale;
    }
    // the tile after this one: of the piece, or the next one's first
    const bool ends = t0 + ROWS >= now.end;
    int t1 = t0 + ROWS;
    bool more = true;
    if (!ends) {
      next = now;
    } else if ((more = next_piece(next))) {
      t1 = next.start;
      entries(next, t1 >> lg);
    }
    uint32_t next_seen = 0;
    if (more) next_seen = issue(next, t1, std::false_type());
    if (seen != (ROWS == 32 ? 0xffffffffu : (1u << ROWS) - 1u)) {
#pragma unroll
      for (int h = 0; h < H; h++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (!(seen >> (h * 16 + g * 4 + i) & 1)) s[h][i] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
      for (int i = 0; i < 4; i++) top = fmaxf(top, s[h][i]);
    top = quarters_max(top);
    if (__any(top > ref + kLeap)) {  // (at first always: -inf + 8 is -inf)
      const float next = fmaxf(ref, top), fade = next == -INFINITY ? 1.f : exp2_hw(ref - next);
      ref = next;
      sum *= fade;
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[t][i] *= fade;
    }
    const float base = ref == -INFINITY ? 0.f : kLift - ref;
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[h][i] = exp2_hw(s[h][i] + base);
        sum += s[h][i];
      }
    if (more) wait_vmcnt<A::LOADS>();
    else wait_vmcnt<0>();
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = g * 4 + i;
        const float *row = reinterpret_cast<const float *>(vs + r * C);
#pragma unroll
        for (int t = 0; t < DT; t++)
          o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(row[(t * 16 + col) ^ ((r >> 2 & 1) << 4)], s[0][i], o[t], 0, 0, 0);
      }
    } else {
      float w[8] = {s[0][0], s[0][1], s[0][2], s[0][3], s[H - 1][0], s[H - 1][1], s[H - 1][2], s[H - 1][3]};
      uint4 p[PP];
      float dv[Q8 ? 2 : 1][Q8 ? 4 * NB : 1];
      if constexpr (Q8) {
        scales_of(vs + N * 64, 0, dv[0]);
        scales_of(vs + N * 64, 1, dv[1]);
      } else {
        planes_of8<CT, true>(w, p);
      }
#pragma unroll
      for (int t = 0; t < DT; t++) {
        uint4 v;
        if constexpr (Q8) {
          if (t % 2 == 0) {  // a block of 32 dims: its scales go to the weights
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = w[j] * dv[j >> 2][(j & 3) * NB + t / 2];
            planes_of8<CT, true>(x, p);
          }
          const int k = (lane & 15) >> 1, r = (k >> 2) * 16 + g * 4 + (k & 3);
          const uint2 *chunk = reinterpret_cast<const uint2 *>(vs + r * C + v_place<C>(r, t)) + (lane & 1);
          const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)chunk);
          v = codes_bf16(x.x, x.y);
        } else {
          const int d = t * 16 + (lane & 3) * 4, r = g * 4 + (lane & 15) / 4;
          auto read = [&](int row) {
            const uint16_t *chunk = reinterpret_cast<const uint16_t *>(vs + row * C + v_place<C>(row, d / 8));
            return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(chunk + d % 8)));
          };
          const uint2 lo = read(r), hi = read(r + 16);
          v = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
#pragma unroll
        for (int i = 0; i < PP; i++) o[t] = mfma16<CT>(v, p[i], o[t]);
      }
    }
    if (more) issue(next, t1, std::true_type());
    if (ends) {
      const int head = now.q0 + col;  // of the key head's
      if constexpr (!F32 && !Q8) {
        f32x4 nan = {sum * 0.f, 0.f, 0.f, 0.f};  // where a sum is not finite, else zeros
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) nan[i] = fmaf(o[t][i], 0.f, nan[i]);
        const bool odd = head < group && nan[0] + nan[1] + (nan[2] + nan[3]) != 0.f;
        if (__builtin_expect(__any(odd) != 0, 0) && holds_infinity(now)) in_fp32(now);
      }
      sum = quarters_sum(sum);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (head < group) {
        if (now.place < 0) {
          const int64_t to = now.seq * a.ldo + (int64_t)(now.kvh * group + head) * hd;
#pragma unroll
          for (int t = 0; t < DT; t++)
            if (t * 16 + g * 4 < hd) store4(a.dtype, a.out, to + t * 16 + g * 4, o[t] * inv);
        } else {
          const int64_t at = (int64_t)(b * 2 + now.place) * plan.columns + col;
          if (g == 0) plan.stats[at] = make_float2(ref - kLift, sum);
#pragma unroll
          for (int t = 0; t < DT; t++)
            if (t * 16 + g * 4 < hd) *reinterpret_cast<f32x4 *>(plan.values + at * hd + t * 16 + g * 4) = o[t];
        }
      }
      if (!more) break;
      reset();
      queries(next);
    }
    seen = next_seen;
    now = next;
    t0 = t1;
  }
}

// The pieces of a pair that has several, of one head: o = sum_i 2^(m_i - m) o_i
// / sum_i 2^(m_i - m) sum_i. What bounds it is latency: the factors of 256
// pieces at a time come by one load a thread, and their rows four dims a thread,
// several pieces side by side; these groups' sums are then added in order.
constexpr int kJoin = 256;
__global__ __launch_bounds__(kJoin) void attend_join_kernel(AttendArgs a, Plan p) {
  __shared__ float fades[kJoin], red[2][4];
  __shared__ f32x4 part[kJoin];
  const Plan::End e = p.ends[blockIdx.x];
  if (e.last < 0) return;
  const int group = a.heads / a.c.kv_heads, hd = a.c.hd, col = blockIdx.y, q = e.pair % p.qtiles * 16 + col;
  if (q >= group) return;
  const int tid = threadIdx.x, wave = tid >> 6, pieces = e.last - e.from + 1;
  auto piece = [&](int i) { return (int64_t)((e.from + i) * 2 + (i ? 0 : e.place)) * p.columns + col; };
  int lanes = 2;  // of a row
  while (lanes * 4 < hd) lanes *= 2;
  const int side = tid / lanes, sides = kJoin / lanes, d = tid % lanes * 4;
  float top = -INFINITY, sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < pieces; i0 += kJoin) {
    const float2 x = i0 + tid < pieces ? p.stats[piece(i0 + tid)] : make_float2(-INFINITY, 0.f);
    const int end = min(pieces - i0, kJoin);
    constexpr int B = 4;  // rows that come together with the factors
    f32x4 rows[B];
#pragma unroll
    for (int j = 0; j < B; j++)
      rows[j] = d < hd && side + j * sides < end ? *reinterpret_cast<const f32x4 *>(p.values + piece(i0 + side + j * sides) * hd + d) : f32x4{0.f, 0.f, 0.f, 0.f};
    const float w = wave_max(x.x);
    if ((tid & 63) == 0) red[0][wave] = w;
    __syncthreads();
    const float next = fmaxf(fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])), top);
    const float base = next == -INFINITY ? 0.f : next, fade = exp2_hw(top - base);
    top = next;
    const float mine = exp2_hw(x.x - base), part_sum = wave_sum(mine * x.y);
    fades[tid] = mine;
    if ((tid & 63) == 0) red[1][wave] = part_sum;
    __syncthreads();
    sum = sum * fade + ((red[1][0] + red[1][1]) + (red[1][2] + red[1][3]));
    o *= fade;
    if (d < hd) {
#pragma unroll
      for (int j = 0; j < B; j++)
        if (side + j * sides < end) o += fades[side + j * sides] * rows[j];
#pragma unroll 4
      for (int i = side + B * sides; i < end; i += sides) o += fades[i] * *reinterpret_cast<const f32x4 *>(p.values + piece(i0 + i) * hd + d);
    }
    __syncthreads();
  }
  part[tid] = o;
  __syncthreads();
  if (side || d >= hd) return;
  for (int i = 1; i < sides; i++) o += part[i * lanes + tid];
  store4(a.dtype, a.out, e.seq * a.ldo + (int64_t)(e.pair / p.qtiles * group + q) * hd + d, o * (sum == 0.f ? 0.f : 1.f / sum));
}

// Blocks of a CU, as their registers allow (attend_kernel's bounds).
constexpr int waves_of(int steps) { return steps == 8 ? 2 : 4; }
constexpr int resident(int steps) { return steps == 1 ? 4 : steps == 2 ? 3 : 2; }
int steps_of(int hd) { return hd <= 32 ? 1 : hd <= 64 ? 2 : hd <= 96 ? 3 : hd <= 128 ? 4 : 8; }

Plan plan_of(const AttendArgs &a) {
  Plan p{};
  const int group = a.heads / a.c.kv_heads;
  p.qtiles = (group + 15) / 16;
  p.columns = std::min(group, 16);
  // one round of blocks; no more than there are units in full tables
  const int64_t most = ((int64_t)a.width << a.c.page_log2) / kUnit + 1, pairs = (int64_t)a.n * a.c.kv_heads * p.qtiles;
  const int each = waves_of(steps_of(a.c.hd));
  p.waves = (int)std::min<int64_t>(256 * resident(steps_of(a.c.hd)) * each, (pairs * most + each - 1) / each * each);
  p.by_pair = pairs <= p.waves;
  return p;
}

}  // namespace

size_t attend_scratch(const AttendArgs &a) {
  const Plan p = plan_of(a);
  return (size_t)p.waves * (32 + (size_t)2 * p.columns * (a.c.hd + 2) * 4);
}

hipError_t launch_attend(const AttendArgs &a, void *scratch, hipStream_t st) {
  Plan p = plan_of(a);
  p.values = static_cast<float *>(scratch);
  p.stats = reinterpret_cast<float2 *>(p.values + (size_t)p.waves * 2 * p.columns * a.c.hd);
  p.ends = reinterpret_cast<Plan::End *>(p.stats + (size_t)p.waves * 2 * p.columns);
  auto go = [&](auto c, auto k, auto planes) {
    using A = Attend<decltype(c)::value, decltype(k)::value, decltype(planes)::value>;
    hipLaunchKernelGGL((attend_kernel<decltype(c)::value, decltype(k)::value, decltype(planes)::value>),
                       dim3((unsigned)(p.waves / A::WAVES)), dim3(64 * A::WAVES), 0, st, a, p);
  };
  auto by_planes = [&](auto c, auto k) {
    constexpr int CT = decltype(c)::value;
    if constexpr (CT == FMT_F32) {
      go(c, k, std::integral_constant<int, 3>());
    } else {
      if (a.dtype == FMT_F32) go(c, k, std::integral_constant<int, 3>());
      else if (a.dtype == (CT == FMT_Q8_0 ? FMT_BF16 : CT)) go(c, k, std::integral_constant<int, 1>());
      else go(c, k, std::integral_constant<int, 2>());
    }
  };
  auto by_width = [&](auto c) {
    switch (steps_of(a.c.hd)) {
      case 1: by_planes(c, std::integral_constant<int, 1>()); break;
      case 2: by_planes(c, std::integral_constant<int, 2>()); break;
      case 3: by_planes(c, std::integral_constant<int, 3>()); break;
      case 4: by_planes(c, std::integral_constant<int, 4>()); break;
      default: by_planes(c, std::integral_constant<int, 8>());
    }
  };
  if (a.c.type == FMT_Q8_0) by_width(std::integral_constant<int, FMT_Q8_0>());
  else for_type(a.c.type, by_width);
  const int joins = p.by_pair ? a.n * a.c.kv_heads * p.qtiles : p.waves;
  hipLaunchKernelGGL(attend_join_kernel, dim3((unsigned)joins, (unsigned)p.columns), dim3(kJoin), 0, st, a, p);
  return hipGetLastError();
}
