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

constexpr int kT = 256;     // four waves
constexpr int kQ = 128;     // queries of a block, 32 a wave
constexpr int kKeys = 64;   // keys of a tile
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

// LDS rows of C chunks of 16 bytes; chunk c of row r at place c ^ swizzle, so
// that the lanes of a read that go together hit distinct banks. K (by rows): 16
// consecutive rows, one chunk. V (transposed): 4 consecutive rows, 4 chunks
// (fp32: one row, consecutive dims: none needed).
template <int C>
__device__ __forceinline__ int k_place(int r, int c) {
  if constexpr (C % 16 == 0) return c ^ (r & 15);
  else if constexpr (C == 8) return c ^ ((r >> 1) & 7);
  else if constexpr (C % 4 == 0) return c ^ ((r >> 2) & 3);
  else return c ^ ((r >> 3) & 1);
}
template <int C>
__device__ __forceinline__ int v_place(int r, int c) {
  if constexpr (C % 16 == 0) return c ^ ((r & 3) << 2 | ((r >> 2) & 3));
  else if constexpr (C == 8) return c ^ (((r >> 1) & 1) << 2 | ((r >> 2) & 3));
  else return c;
}

// The sequence of query tile `tile` (tiles of kQ queries, a sequence's last
// ones first), its queries and keys.
struct Where {
  int tile;            // within the sequence; -1: none
  int q0, nq, k0, nk;  // first rows and numbers
};
__device__ __forceinline__ Where find(const PromptArgs &a, int tile) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < a.sequences; s0 += 64) {
    const int s = s0 + lane;
    int first = 0, n = 0;
    if (s < a.sequences) {
      first = min(max(a.q_offsets[s], 0), a.nq);
      n = max(min(a.q_offsets[s + 1], a.nq) - first, 0);
    }
    const int tiles = (n + kQ - 1) / kQ;
    int upto = tiles;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const int x = __shfl_up(upto, off);
      if (lane >= off) upto += x;
    }
    const uint64_t past = __ballot(before + upto > tile);
    if (past) {
      const int l = __builtin_ctzll(past);
      Where w;
      w.tile = before + __shfl(upto, l) - 1 - tile;
      w.q0 = __shfl(first, l), w.nq = __shfl(n, l);
      const int k0 = min(max(a.k_offsets[s0 + l], 0), a.nk);
      w.k0 = k0, w.nk = max(min(a.k_offsets[s0 + l + 1], a.nk) - k0, 0);
      return w;
    }
    before += __shfl(upto, 63);
  }
  return Where{-1, 0, 0, 0, 0};
}

// KS: steps of 16 dims. T: the chunks (16 bytes) of a row.
template <int D, int KS>
__global__ __launch_bounds__(kT) void prompt_kernel(PromptArgs a) {
  constexpr bool F32 = D == FMT_F32;
  constexpr int HD = KS * 16;
  constexpr int V = F32 ? 4 : 8;          // values of a chunk
  constexpr int C = HD / V;               // chunks of a row
  constexpr int DT = (HD + 31) / 32;      // 32-dim tiles of O^T
  constexpr int KEYS = F32 && KS > 8 ? 32 : kKeys;
  constexpr int HALVES = KEYS / 32;
  constexpr int LOADS = (KEYS * C + kT - 1) / kT;
  constexpr float kLeap = 8.f;            // the reference moves only when a score exceeds it by 2^8
  typedef std::conditional_t<F32, float, uint16_t> Value;
  // (the transposed reads of a row's last tile may go past the row)
  __shared__ __align__(16) uint4 ks[KEYS * C];
  __shared__ __align__(16) uint4 vs[KEYS * C + DT * 32 / V - C];

  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Blocks go over the XCDs in turn: an XCD takes the same heads of every tile,
  // so the blocks it runs share their keys in its L2.
  int head, tile;
  if (a.heads % 8 == 0) {
    const int j = blockIdx.x / 8;
    head = blockIdx.x % 8 * (a.heads / 8) + j % (a.heads / 8);
    tile = j / (a.heads / 8);
  } else {
    head = blockIdx.x % a.heads;
    tile = blockIdx.x / a.heads;
  }
  const Where w = find(a, tile);
  if (w.tile < 0) return;
  const int kvh = head / (a.heads / a.kv_heads);
  const int qb = w.tile * kQ, qw = qb + wave * 32, mine = qw + col;  // within the sequence
  const int shift = w.nk - w.nq;
  // the last key that this lane's query, the wave's and the block's last ones see
  const int last = a.causal ? min(mine, w.nq - 1) + shift : w.nk - 1;
  const int last_wave = a.causal ? min(qw + 31, w.nq - 1) + shift : w.nk - 1;
  const int last_block = a.causal ? min(qb + kQ - 1, w.nq - 1) + shift : w.nk - 1;
  const int first_wave = a.causal ? qw + shift : w.nk - 1;  // of the wave's first query

  // Q^T as B operands: query l % 32, dims 16 step + 8 g .. + 7 (fp32: of a
  // chunk 8 step + 4 g .. + 3, one value a product).
  uint4 q[F32 ? 2 * KS : KS];
  {
    const Value *p = static_cast<const Value *>(a.q) + (w.q0 + min(mine, w.nq - 1)) * a.ldq + (int64_t)head * a.hd;
#pragma unroll
    for (int s = 0; s < (F32 ? 2 * KS : KS); s++) {
      const int d = (2 * s + g) * V;
      q[s] = make_uint4(0, 0, 0, 0);
      if (d < a.hd) {
        const u32x4_any x = *reinterpret_cast<const u32x4_any *>(p + d);
        q[s] = make_uint4(x.x, x.y, x.z, x.w);
      }
    }
  }
  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; t++)
#pragma unroll
    for (int v = 0; v < 16; v++) o[t][v] = 0.f;
  float ref = -INFINITY, sum = 0.f;  // of this lane's query; sum: of the lane's own keys
  const float scale = a.scale * kLog2e;

  const Value *kp = static_cast<const Value *>(a.k) + (int64_t)w.k0 * a.ldk + (int64_t)kvh * a.hd;
  const Value *vp = static_cast<const Value *>(a.v) + (int64_t)w.k0 * a.ldv + (int64_t)kvh * a.hd;
  const int tiles = last_block / KEYS + 1;  // (last_block < 0: no key, tiles <= 0 or all masked)
  uint4 kr[LOADS], vr[LOADS];
  auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const int e = tid + kT * i, r = t0 + e / C, d = e % C * V;
      kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      if (e < KEYS * C && r < w.nk && d < a.hd) {
        const u32x4_any x = *reinterpret_cast<const u32x4_any *>(kp + r * a.ldk + d);
        const u32x4_any y = *reinterpret_cast<const u32x4_any *>(vp + r * a.ldv + d);
        kr[i] = make_uint4(x.x, x.y, x.z, x.w);
        vr[i] = make_uint4(y.x, y.y, y.z, y.w);
      }
    }
  };
  if (last_block >= 0) load(0);
  for (int tile_k = 0; last_block >= 0 && tile_k < tiles; tile_k++) {
    const int t0 = tile_k * KEYS;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const int e = tid + kT * i, r = e / C, c = e % C;
      if (KEYS * C % kT == 0 || e < KEYS * C) {
        ks[r * C + k_place<C>(r, c)] = kr[i];
        vs[r * C + (F32 ? c : v_place<C>(r, c))] = vr[i];
      }
    }
    if (tile_k + 1 < tiles) load(t0 + KEYS);
    __syncthreads();
    if (qw >= w.nq || t0 > last_wave) continue;
    const bool masked = t0 + KEYS - 1 > first_wave || t0 + KEYS > w.nk;

    f32x16 s[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; h++) {
#pragma unroll
      for (int v = 0; v < 16; v++) s[h][v] = 0.f;
      const int r = h * 32 + col;
#pragma unroll
      for (int st = 0; st < (F32 ? 2 * KS : KS); st++) {
        const uint4 x = ks[r * C + k_place<C>(r, 2 * st + g)];
        if constexpr (F32) {
          s[h] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.x), __uint_as_float(q[st].x), s[h], 0, 0, 0);
          s[h] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.y), __uint_as_float(q[st].y), s[h], 0, 0, 0);
          s[h] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.z), __uint_as_float(q[st].z), s[h], 0, 0, 0);
          s[h] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x.w), __uint_as_float(q[st].w), s[h], 0, 0, 0);
        } else {
          s[h] = mfma<D>(x, q[st], s[h]);
        }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int h = 0; h < HALVES; h++)
#pragma unroll
      for (int v = 0; v < 16; v++) {
        s[h][v] *= scale;
        if (masked && t0 + h * 32 + (v >> 2) * 8 + g * 4 + (v & 3) > last) s[h][v] = -INFINITY;
        top = fmaxf(top, s[h][v]);
      }
    top = fmaxf(top, __shfl_xor(top, 32));
    if (__any(top > ref + kLeap || (ref == -INFINITY && top > ref))) {
      const float next = fmaxf(ref, top), fade = next == -INFINITY ? 1.f : exp2_hw(ref - next);
      ref = next;
      sum *= fade;
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[t][v] *= fade;
    }
    const float base = ref == -INFINITY ? 0.f : ref;
#pragma unroll
    for (int h = 0; h < HALVES; h++)
#pragma unroll
      for (int v = 0; v < 16; v++) {
        s[h][v] = exp2_hw(s[h][v] - base);
        sum += s[h][v];
      }
    // A key that some query of the tile does not see: its weight there is 0,
    // and 0 times an infinity or NaN would be one too. Such values are left out
    // of the products and added to the queries that see them.
    bool bad = false;
    if (masked && a.causal) {
      for (int e = lane; e < KEYS * C; e += 64) bad |= not_finite<D>(vs[e]);
      bad = __any(bad);
    }
    auto product = [&](auto clean) {
      constexpr bool CLEAN = decltype(clean)::value;
#pragma unroll
      for (int h = 0; h < HALVES; h++) {
        if constexpr (F32) {
#pragma unroll
          for (int v = 0; v < 16; v++) {
            const int r = h * 32 + (v >> 2) * 8 + g * 4 + (v & 3);
#pragma unroll
            for (int t = 0; t < DT; t++) {
              float x = reinterpret_cast<const float *>(vs + r * C)[t * 32 + col];
              if (CLEAN && (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) x = 0.f;
              o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[h][v], o[t], 0, 0, 0);
            }
          }
        } else {
#pragma unroll
          for (int st = 0; st < 2; st++) {
            uint4 pw;
            pw.x = pack2<D>(s[h][8 * st], s[h][8 * st + 1]);
            pw.y = pack2<D>(s[h][8 * st + 2], s[h][8 * st + 3]);
            pw.z = pack2<D>(s[h][8 * st + 4], s[h][8 * st + 5]);
            pw.w = pack2<D>(s[h][8 * st + 6], s[h][8 * st + 7]);
            const int r0 = h * 32 + st * 16 + g * 4 + (lane & 15) / 4;
#pragma unroll
            for (int t = 0; t < DT; t++) {
              const int d = t * 32 + (lane >> 4 & 1) * 16 + (lane & 3) * 4;
              auto read = [&](int r) {
                const uint4 *chunk = vs + (r * C + v_place<C>(r, d / 8));
                return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(reinterpret_cast<const uint16_t *>(chunk) + d % 8));
              };
              const uint2 lo = __builtin_bit_cast(uint2, read(r0)), hi = __builtin_bit_cast(uint2, read(r0 + 8));
              uint4 x = make_uint4(lo.x, lo.y, hi.x, hi.y);
              if constexpr (CLEAN) {
                constexpr uint32_t e = D == FMT_F16 ? 0x7c00u : 0x7f80u;
                auto finite = [](uint32_t u) {
                  return ((u & e) == e ? 0u : u & 0xffffu) | ((u >> 16 & e) == e ? 0u : u & 0xffff0000u);
                };
                x = make_uint4(finite(x.x), finite(x.y), finite(x.z), finite(x.w));
              }
              o[t] = mfma<D>(x, pw, o[t]);
            }
          }
        }
      }
    };
    if (!bad) {
      product(std::false_type());
    } else {
      product(std::true_type());
      for (int r = 0; r < KEYS && t0 + r <= last; r++)
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
          for (int v = 0; v < 16; v++) {
            const int d = t * 32 + (v >> 2) * 8 + g * 4 + (v & 3);
            if (d >= HD) continue;
            const Value raw = reinterpret_cast<const Value *>(vs + (r * C + (F32 ? d / V : v_place<C>(r, d / V))))[d % V];
            float x;
            if constexpr (F32) x = raw;
            else x = D == FMT_F16 ? hw_half(raw) : bf16_to_float(raw);
            if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) o[t][v] += x;
          }
    }
  }
  sum += __shfl_xor(sum, 32);
  if (mine >= w.nq) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  Value *out = static_cast<Value *>(a.out) + (w.q0 + mine) * a.ldo + (int64_t)head * a.hd;
#pragma unroll
  for (int t = 0; t < DT; t++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int d = t * 32 + j * 8 + g * 4;
      if (d >= a.hd) continue;
      const float x = o[t][4 * j] * inv, y = o[t][4 * j + 1] * inv, z = o[t][4 * j + 2] * inv, u = o[t][4 * j + 3] * inv;
      if constexpr (F32) *reinterpret_cast<f32x4_any *>(out + d) = f32x4_any{x, y, z, u};
      else *reinterpret_cast<u32x2_any *>(out + d) = u32x2_any{pack2<D>(x, y), pack2<D>(z, u)};
    }
}

}  // namespace

hipError_t launch_prompt(const PromptArgs &a, hipStream_t st) {
  // at most: every sequence's last tile may be a part
  const int64_t tiles = a.nq / kQ + std::min<int64_t>(a.sequences, a.nq);
  const dim3 grid((unsigned)(tiles * a.heads));
  auto go = [&](auto d, auto k) {
    hipLaunchKernelGGL((prompt_kernel<decltype(d)::value, decltype(k)::value>), grid, dim3(kT), 0, st, a);
  };
  for_type(a.dtype, [&](auto d) {
    if (a.hd <= 32) go(d, std::integral_constant<int, 2>());
    else if (a.hd <= 64) go(d, std::integral_constant<int, 4>());
    else if (a.hd <= 80) go(d, std::integral_constant<int, 5>());
    else if (a.hd <= 96) go(d, std::integral_constant<int, 6>());
    else if (a.hd <= 128) go(d, std::integral_constant<int, 8>());
    else go(d, std::integral_constant<int, 16>());
  });
  return hipGetLastError();
}
