// Attention over a sliding-window cache: softmax(scale * q . K) V over the positions that a query sees
// (cache_device.hpp). Queries of the same stream and key/value head share the cache rows: a row of the
// matrix products is a (token, query head) pair, head fastest.
//
// One pass over the keys with the softmax's running maximum m and sum l per row, in 32 bits, in the base
// of two. For a tile of keys S^T = K Q^T and O^T += V^T P^T, both on MFMA 16x16: with the rows of the
// products on the lanes (lane % 16), the maximum, the sum and the rescaling are per lane, and the four keys
// (4 (lane / 16) + i) that a lane holds of each 16 x 16 block of S^T are, rounded, the operand that P^T
// wants. The order of the keys within a product's depth does not matter as long as both operands agree.
#pragma once

#include "cache_device.hpp"

#include <type_traits>

namespace stamd {

struct AttentionView {
  const char* q;
  char* out;
  int64_t q_token, q_head, out_token, out_head;  // strides in bytes
  float scale;       // times log2(e)
  int group;         // query heads per key/value head
  int rows;          // most rows of a (stream, key/value head): max_tokens * group
  int splits;        // workgroups along the keys
  float2* part_ml;   // splits > 1: partial (m, l) [stream][kv head][row][split]
  float* part_o;     // and output [stream][kv head][row][split][dim]
  int out_layout;    // 0: strides above; 1, 2: the projections' operand layouts (act_index), out_ld columns
  int out_ld;
};

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// The keys that some query of the tokens ta .. tb (positions) sees, as a list: first the sinks, then the
// ring's positions lo .. tb. j is an index into the list.
struct KeyList {
  int sinks, total;     // entries
  int offset, ring, slots_sinks;  // ring slot of the first ring entry
  int64_t lo;
  __device__ __forceinline__ void init(const CacheView& c, int64_t ta, int64_t tb) {
    sinks = (int)min((int64_t)c.sinks, tb + 1);
    lo = max((int64_t)c.sinks, ta - c.window + 1);
    const int64_t ringed = tb - lo + 1;
    total = sinks + (ringed > 0 ? (int)ringed : 0);
    offset = ringed > 0 ? ring_offset(c, lo) : 0;
    ring = c.ring;
    slots_sinks = c.sinks;
  }
  // Offsets of n rows, `step` apart, of the `count` entries from j0 on: in units of slots, row i of the lane at entry
  // min(j0 + min(i * step + sub, count - 1), total - 1). Where the entries are consecutive slots, and their
  // offsets within 32 bits of the first (near), the lane's part `part` = sub * unit is given.
  template <int N>
  __device__ __forceinline__ void offsets(int j0, int step, int sub, int count, bool near, uint32_t unit, uint32_t part,
                                          uint64_t (&at)[N]) const {
    int o = offset + j0 - sinks;
    o = o >= ring ? o - ring : o;
    if (near && j0 >= sinks && j0 + count <= total && o + count <= ring) {
#pragma unroll
      for (int i = 0; i < N; i++) at[i] = (uint64_t)(slots_sinks + o + i * step) * unit + part;
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) at[i] = (uint64_t)slot(min(j0 + min(i * step + sub, count - 1), total - 1)) * unit;
    }
  }
  __device__ __forceinline__ int slot(int j) const {
    const int o = offset + j - sinks;
    return j < sinks ? j : slots_sinks + (o >= ring ? o - ring : o);
  }
};
// What one query at position t sees of a list: sinks up to t, ring entries in (newest - window, newest].
struct Seen {
  int t, newest;
  __device__ __forceinline__ void init(const KeyList& k, int64_t position) {
    t = (int)min(position, (int64_t)1 << 30);
    newest = (int)max(position - k.lo, (int64_t)-1);
  }
  // No short circuits: they compile to a tree of branches for each of a lane's keys.
  __device__ __forceinline__ bool operator()(const KeyList& k, int window, int j) const {
    const int e = j - k.sinks;
    const bool ringed = (e <= newest) & (e > newest - window), sink = j <= t;
    return (j < k.total) & ((e < 0) ? sink : ringed);
  }
};

// A tile of K and V rows in LDS, the elements that the MFMAs take: FP32, or 16 bits. Rows are D elements
// (the head dimension padded with zeros to 64, 128 or 256) in 16-byte chunks; chunk c of row r is stored
// at c ^ swizzle(r), which spreads over the banks what 16 lanes read at once: one chunk of 16 rows (K),
// 32 bytes of 16 rows (V, transposed 16-bit reads), 64 bytes of four rows (V, FP32); and what 16 lanes write of
// 4-bit rows, every fourth chunk of four rows.
template <int M, int D>
struct TileLayout {
  static constexpr int kElem = M == kTF32 ? 4 : 2;
  static constexpr int kRow = D * kElem, kChunks = kRow / 16;
  __device__ static __forceinline__ int key_chunk(int r, int c) { return c ^ (kChunks == 8 ? (r >> 1) & 7 : r & 15); }
  __device__ static __forceinline__ int value_chunk(int r, int c) {
    if constexpr (M == kTF32) return c ^ (((r >> 2) & 3) << 2);
    else if constexpr (kChunks == 8) return c ^ (((r >> 1) & 3) << 1);
    else return c ^ ((r & 7) << 1 | (r >> 1 & 1));
  }
};

// How rows of cache type C come in 16-byte loads: E elements each, L lanes per row.
template <int C, int D>
struct RowLoad {
  static constexpr int E = C == kTF32 ? 4 : C == kTInt4 ? 32 : 8;
  static constexpr int L = D / E;
};

// Eight codes of a 4-bit row and their (scale, minimum) as FP16 values. code + 1024 (or + 64 for the codes in
// bits 4 and 12 of a half) is made by an OR, the constant subtracted exactly. term 0: minimum + scale * code
// rounded once, to FP16; term 1: what that rounding left, from the FP32 value.
template <int kTerm>
__device__ __forceinline__ word4_t dequant8_f16(unsigned w, half2_t sz) {
  const half2_t big = {(_Float16)1024.f, (_Float16)1024.f}, mid = {(_Float16)64.f, (_Float16)64.f};
  const half2_t s = {sz[0], sz[0]}, z = {sz[1], sz[1]};
  auto value = [&](half2_t code) {
    const half2_t v = code * s + z;
    if constexpr (kTerm == 0) return __builtin_bit_cast(unsigned, v);
    const float a = (float)code[0] * (float)sz[0] + (float)sz[1], b = (float)code[1] * (float)sz[0] + (float)sz[1];
    return pack_f16(a - (float)v[0], b - (float)v[1]);
  };
  // The constants in registers: as literals, of which an instruction takes one, AND and OR are two instructions.
  unsigned low_mask = 0x000f000fu, high_mask = 0x00f000f0u, low_one = 0x64006400u, high_one = 0x54005400u;
  asm("" : "+s"(low_mask), "+s"(high_mask));
  asm("" : "+v"(low_one), "+v"(high_one));
  auto low = [&](unsigned x) { return value(__builtin_bit_cast(half2_t, (x & low_mask) | low_one) - big); };
  auto high = [&](unsigned x) { return value(__builtin_bit_cast(half2_t, (x & high_mask) | high_one) - mid); };
  return word4_t{low(w), high(w), low(w >> 8), high(w >> 8)};
}
__device__ __forceinline__ void dequant8_f32(unsigned w, float s, float z, float4_t (&out)[2]) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    out[j >> 1][(j & 1) * 2] = z + s * (float)((w >> (4 * j)) & 15u);
    out[j >> 1][(j & 1) * 2 + 1] = z + s * (float)((w >> (16 + 4 * j)) & 15u);
  }
}

// One 16-byte load of row r, lane position p of the row's L, as the chunks of the LDS tile: calls
// put(chunk, value) for each. `keep`: whether the lane's elements are inside the head. kTerm: of 4-bit rows.
template <int C, int M, int kTerm = 0, typename Put>
__device__ __forceinline__ void expand(word4_t w, unsigned params, int p, bool keep, Put&& put) {
  if constexpr (C == kTInt4) params = keep ? params : 0u;  // zeros, whatever the codes
  else w = keep ? w : word4_t{0, 0, 0, 0};
  if constexpr (C == M) {
    put(p, w);
  } else if constexpr (C == kTInt4) {
    const half2_t sz = __builtin_bit_cast(half2_t, params);
    if constexpr (M == kTF32) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float4_t f[2];
        dequant8_f32(w[i], (float)sz[0], (float)sz[1], f);
        put(p * 8 + 2 * i, __builtin_bit_cast(word4_t, f[0]));
        put(p * 8 + 2 * i + 1, __builtin_bit_cast(word4_t, f[1]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) put(p * 4 + i, dequant8_f16<kTerm>(w[i], sz));
    }
  } else {
    static_assert(M == kTF32);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      put(p * 2 + i, __builtin_bit_cast(word4_t, float4_t{low16<C>(w[2 * i]), high16<C>(w[2 * i]), low16<C>(w[2 * i + 1]),
                                                          high16<C>(w[2 * i + 1])}));
    }
  }
}
// Whether a chunk of the tile holds a value that is not finite.
template <int M>
__device__ __forceinline__ bool not_finite(word4_t w) {
  constexpr unsigned e = M == kTF32 ? 0x7f800000u : M == kTF16 ? 0x7c00u : 0x7f80u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (M == kTF32) bad |= (w[i] & e) == e;
    else bad |= (w[i] & e) == e || ((w[i] >> 16) & e) == e;
  }
  return bad;
}

template <int M>
struct Mfma {
  // Two 16-byte fragments (4 FP32 or 8 16-bit elements of depth per lane): D += A B^T.
  __device__ static __forceinline__ float4_t mul(word4_t a, word4_t b, float4_t d) {
    if constexpr (M == kTF16) {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), d, 0, 0, 0);
    } else if constexpr (M == kTB16) {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8_t, a), __builtin_bit_cast(bhalf8_t, b), d, 0, 0,
                                                     0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) d = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_to_float(a[i]), bits_to_float(b[i]), d, 0, 0, 0);
      return d;
    }
  }
};

typedef __attribute__((address_space(3))) char lds_char;
template <typename T>
__device__ __forceinline__ T lds_load(const char* p) {
  return *(const __attribute__((address_space(3))) T*)p;
}
template <typename T>
__device__ __forceinline__ void lds_put(char* p, T v) {
  *(__attribute__((address_space(3))) T*)p = v;
}
// Four 16-bit elements of one column and four consecutive rows: 16 lanes read a 4 x 16 block, lane i at
// row i / 4, elements 4 (i % 4) ..; lane i receives column i.
__device__ __forceinline__ word2_t lds_column4(const char* p) {
  return __builtin_bit_cast(word2_t,
                            __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)p));
}
// 16 bytes per lane straight to LDS, lane i's to to + 16 i (`to` is the wave's), and the wait for such loads.
__device__ __forceinline__ void load_to_lds(const char* from, char* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// FP16 queries over 4-bit rows: the rounding of the dequantised values to FP16 is as large as the output's own,
// twice (K and V), and the weights' a third. Keys in two FP16 terms and weights in two leave one of the three
// (the output of 4 x 1024 tokens 1.9 times as far from exact as its own rounding without, 1.35 with).
template <int A, int C>
constexpr bool two_terms() {
  return A == kTF16 && C == kTInt4;
}

// The type that the MFMAs take: FP32 for FP32 queries (every cache type widens to it exactly), else the
// queries' own; 4-bit rows become FP16 for bfloat16 queries too, whose eight significant bits FP16 holds
// once the row is scaled by a power of two.
template <int A, int C>
constexpr int mfma_type() {
  return A == kTF32 ? kTF32 : C == kTInt4 ? kTF16 : A;
}

// The queries' fragments of one block of 16 rows, lane % 16 the row: 16 bytes per step of kStep dims.
// factor: what a logit in the base of two is of the products.
template <int A, int M, int D>
struct QueryBlock {
  static constexpr int kStep = M == kTF32 ? 16 : 32, kSteps = D / kStep;
  word4_t f[kSteps];
  float factor;
  __device__ __forceinline__ void load(const char* row, int dim, float scale, int g, bool valid) {
    factor = scale;
    constexpr int per = kStep / 4;  // dims of a lane per step
    if constexpr (A == M) {
#pragma unroll
      for (int s = 0; s < kSteps; s++) {
        const int d = s * kStep + g * per;
        const word4_t w = load_global<word4_t>(row + (d < dim ? d : 0) * (A == kTF32 ? 4 : 2));
        f[s] = valid && d < dim ? w : word4_t{0, 0, 0, 0};
      }
    } else {  // bfloat16 to FP16
      float x[kSteps][8], top = 0.f;
#pragma unroll
      for (int s = 0; s < kSteps; s++) {
        const int d = s * kStep + g * per;
        const bool in = valid && d < dim;
        const word4_t w = load_global<word4_t>(row + (d < dim ? d : 0) * 2);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          x[s][2 * i] = in ? low16<kTB16>(w[i]) : 0.f;
          x[s][2 * i + 1] = in ? high16<kTB16>(w[i]) : 0.f;
          top = fmaxf(top, fmaxf(fabsf(x[s][2 * i]), fabsf(x[s][2 * i + 1])));
        }
      }
      top = pair32_max(pair16_max(top));
      // 2^e with e the exponent of the row's largest value; rows of zeros, and rows that are not finite,
      // stay as they are.
      const unsigned e = (float_to_bits(top) >> 23) & 255u;
      const bool plain = e == 0 || e >= 254;
      const float down = plain ? 1.f : bits_to_float((254u - e) << 23);
      factor = plain ? scale : scale * bits_to_float(e << 23);
#pragma unroll
      for (int s = 0; s < kSteps; s++)
#pragma unroll
        for (int i = 0; i < 4; i++) f[s][i] = pack_f16(x[s][2 * i] * down, x[s][2 * i + 1] * down);
    }
  }
};

// Products of one tile with a block of 16 rows, for a wave. kt and vt: the tile's K and V in LDS.
// kFine: 16-bit weights in two terms (w and what its rounding left), so that the output's own rounding is
// the only one that counts; twice the products with V. U: the head's dimensions that are multiplied, in steps of 32.
template <int M, int D, int U, int KT, bool kFine>
struct TileMath {
  using T = TileLayout<M, D>;
  static constexpr int kBlocks = KT / 16;
  // S^T of the tile for MB blocks of rows. Each depth's products go over all blocks: independent sums.
  // kMore: added to what s holds.
  template <bool kMore, int MB, typename Q>
  __device__ static __forceinline__ void logits(const char* kt, const Q (&q)[MB], float4_t (&s)[MB][kBlocks], int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int step = 0; step < Q::kSteps; step++) {
#pragma unroll
      for (int kb = 0; kb < kBlocks; kb++) {
        const int r = kb * 16 + (lane & 15);
        const word4_t k = lds_load<word4_t>(kt + r * T::kRow + T::key_chunk(r, step * 4 + g) * 16);
#pragma unroll
        for (int u = 0; u < MB; u++)
          s[u][kb] = Mfma<M>::mul(k, q[u].f[step], step == 0 && !kMore ? float4_t{0.f, 0.f, 0.f, 0.f} : s[u][kb]);
      }
    }
    // Six reads ahead of the products, then one per MB of them: left alone, the compiler waits for most reads
    // where it makes them (a prompt of 8192 tokens 271 -> 267 us).
    if constexpr (M != kTF32 && MB > 1) {
      constexpr int kReads = Q::kSteps * kBlocks, kAhead = kReads < 6 ? kReads : 6;
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int i = 0; i < kReads - kAhead; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, MB, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, MB * kAhead, 0);
    }
  }
  // The V operand of 16 dims (block db) and one depth of P: 32 keys (blocks 2 d, 2 d + 1), FP32 16 keys.
  __device__ static __forceinline__ word4_t values(const char* vt, int depth, int db, int lane) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (M == kTF32) {
      word4_t v;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int r = depth * 16 + g * 4 + e;
        v[e] = lds_load<unsigned>(vt + r * T::kRow + T::value_chunk(r, db * 4 + (i >> 2)) * 16 + (i & 3) * 4);
      }
      return v;
    } else {
      word2_t h[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int r = depth * 32 + e * 16 + g * 4 + (i >> 2);
        h[e] = lds_column4(vt + r * T::kRow + T::value_chunk(r, db * 2 + ((i & 3) >> 1)) * 16 + (i & 1) * 8);
      }
      return word4_t{h[0][0], h[0][1], h[1][0], h[1][1]};
    }
  }
  static constexpr int kDepth = M == kTF32 ? 16 : 32, kDepths = KT / kDepth;
  // Tiles that are not seen whole and hold values of V that are not finite: this adds such values to the
  // outputs of the rows that see them, before clear makes them zeros, which the products then add nothing
  // for.
  template <int MB, typename Sees>
  __device__ static __forceinline__ void add_odd(const char* vt, float4_t (&o)[MB][U / 16 + 1], int lane, Sees&& sees) {
    const int g = lane >> 4;
#pragma unroll 1
    for (int r = 0; r < KT; r++) {
      bool seen[MB];
#pragma unroll
      for (int u = 0; u < MB; u++) seen[u] = sees(u, r);
#pragma unroll
      for (int db = 0; db < U / 16; db++) {
        float v[4];
        if constexpr (M == kTF32) {
          const float4_t x = lds_load<float4_t>(vt + r * T::kRow + T::value_chunk(r, db * 4 + g) * 16);
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = x[i];
        } else {
          const word2_t x = lds_load<word2_t>(vt + r * T::kRow + T::value_chunk(r, db * 2 + (g >> 1)) * 16 + (g & 1) * 8);
#pragma unroll
          for (int i = 0; i < 2; i++) {
            v[2 * i] = low16<M>(x[i]);
            v[2 * i + 1] = high16<M>(x[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float bad = v[i] - v[i] == 0.f ? 0.f : v[i];
#pragma unroll
          for (int u = 0; u < MB; u++) o[u][db][i] += seen[u] ? bad : 0.f;
        }
      }
    }
  }
  // Whether the thread's share of a tile of V holds a value that is not finite.
  template <int kThreads>
  __device__ static __forceinline__ bool any_odd(const char* vt, int thread) {
    bool found = false;
#pragma unroll 1
    for (int at = thread * 16; at < KT * T::kRow; at += kThreads * 16) found |= not_finite<M>(lds_load<word4_t>(vt + at));
    return found;
  }
  template <int kThreads>
  __device__ static __forceinline__ void clear(char* vt, int thread) {
#pragma unroll 1
    for (int at = thread * 16; at < KT * T::kRow; at += kThreads * 16) {
      word4_t w = lds_load<word4_t>(vt + at);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (M == kTF32) {
          w[i] = (w[i] & 0x7f800000u) == 0x7f800000u ? 0u : w[i];
        } else {
          constexpr unsigned e = M == kTF16 ? 0x7c00u : 0x7f80u;
          w[i] = ((w[i] & e) == e ? 0u : w[i] & 0xffffu) | (((w[i] >> 16) & e) == e ? 0u : w[i] & 0xffff0000u);
        }
      }
      lds_put(vt + at, w);
    }
  }
  // O^T += V^T P^T of the tile, P = exp2(s factor - base), each depth's weights made right before its products. The
  // last block of O is the rows' sums: for 16-bit products those of the rounded weights, by a product with
  // ones (every element is the row's whole sum), for FP32 the lane's own share in four parts.
  template <int MB, typename Q>
  __device__ static __forceinline__ void outputs(const char* vt, const float4_t (&s)[MB][kBlocks], const Q (&q)[MB],
                                                 const float (&base)[MB], float4_t (&o)[MB][U / 16 + 1], int lane) {
#pragma unroll
    for (int depth = 0; depth < kDepths; depth++) {
      word4_t w[MB], rest[MB];
#pragma unroll
      for (int u = 0; u < MB; u++) {
        float p[kDepth / 4];
#pragma unroll
        for (int i = 0; i < kDepth / 4; i++)
          p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][depth * (kDepth / 16) + i / 4][i % 4], q[u].factor, -base[u]));
        if constexpr (M == kTF32) {
          const float4_t x = {p[0], p[1], p[2], p[3]};
          w[u] = __builtin_bit_cast(word4_t, x);
          o[u][U / 16] += x;
        } else {
          constexpr unsigned one = M == kTF16 ? 0x3c003c00u : 0x3f803f80u;
          const word4_t ones = {one, one, one, one};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            w[u][i] = pack16<M>(p[2 * i], p[2 * i + 1]);
            if constexpr (kFine) rest[u][i] = pack16<M>(p[2 * i] - low16<M>(w[u][i]), p[2 * i + 1] - high16<M>(w[u][i]));
          }
          o[u][U / 16] = Mfma<M>::mul(ones, w[u], o[u][U / 16]);
          if constexpr (kFine) o[u][U / 16] = Mfma<M>::mul(ones, rest[u], o[u][U / 16]);
        }
      }
#pragma unroll
      for (int d = 0; d < U / 16; d++) {
        const word4_t v = values(vt, depth, d, lane);
#pragma unroll
        for (int u = 0; u < MB; u++) o[u][d] = Mfma<M>::mul(v, w[u], o[u][d]);
        if constexpr (kFine) {
#pragma unroll
          for (int u = 0; u < MB; u++) o[u][d] = Mfma<M>::mul(v, rest[u], o[u][d]);
        }
      }
    }
  }
  // A row's sum of weights, from the last block of its O.
  __device__ static __forceinline__ float row_sum(const float4_t& x) {
    if constexpr (M == kTF32) return pair32_add(pair16_add((x[0] + x[1]) + (x[2] + x[3])));
    else return x[0];
  }
  // Entries that a row does not see: minus infinity.
  template <int MB, typename See>
  __device__ static __forceinline__ void mask(float4_t (&s)[MB][kBlocks], const See (&seen)[MB], const KeyList& keys, int window,
                                              int j0, int lane) {
    const int j = j0 + (lane >> 4) * 4;
#pragma unroll
    for (int u = 0; u < MB; u++) {
      if (j0 >= keys.sinks) {
        const int age = seen[u].newest + keys.sinks - j;
#pragma unroll
        for (int kb = 0; kb < kBlocks; kb++) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float x = s[u][kb][i];
            s[u][kb][i] = (unsigned)(age - kb * 16 - i) < (unsigned)window ? x : -INFINITY;
          }
        }
      } else {
#pragma unroll
        for (int kb = 0; kb < kBlocks; kb++) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float x = s[u][kb][i];
            s[u][kb][i] = seen[u](keys, window, j + kb * 16 + i) ? x : -INFINITY;
          }
        }
      }
    }
  }
};

// The maxima m that the weights exp2(s factor - m) of MB blocks of 16 rows are relative to, s a tile's products
// (masked ones -inf). A row's moves only when its logits pass it by more than 2^8: the weights stay below 256
// then, far from any type's limit, and almost every tile is spared the rescaling of O (one that follows every
// maximum ran for most tiles, as one of 16 rows nearly always has a new one: a prompt of 8192 tokens 360 -> 320 us
// together with the scaling inside the exponential). factor > 0, so the largest product is the largest logit.
// base: m, or 0 for rows without a logit so far.
template <int MB, int N, int ND, typename Q>
__device__ __forceinline__ void move_maxima(const float4_t (&s)[MB][N], const Q (&q)[MB], float (&m)[MB], float (&base)[MB],
                                            float4_t (&o)[MB][ND]) {
  float top[MB];
  bool any = false;
#pragma unroll
  for (int u = 0; u < MB; u++) {
    top[u] = s[u][0][0];
#pragma unroll
    for (int kb = 0; kb < N; kb++) {
#pragma unroll
      for (int i = 0; i < 4; i++) top[u] = fmaxf(top[u], s[u][kb][i]);
    }
    top[u] = pair32_max(pair16_max(top[u])) * q[u].factor;
    any |= top[u] > m[u] + 8.f;  // -inf has no weights yet: any logit passes it
  }
  if (__ballot(any)) {
#pragma unroll
    for (int u = 0; u < MB; u++) {
      const bool move = top[u] > m[u] + 8.f;
      // O of a row without weights may hold infinities that were added apart: it keeps them.
      const float alpha = !move || m[u] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[u] - top[u]);
#pragma unroll
      for (int d = 0; d < ND; d++) o[u][d] *= alpha;
      m[u] = move ? top[u] : m[u];
    }
  }
#pragma unroll
  for (int u = 0; u < MB; u++) base[u] = m[u] == -INFINITY ? 0.f : m[u];
}

// Keys of a wave's tile: 16 KB of K and V, or what one MFMA depth needs.
template <int M, int D>
constexpr int wave_tile() {
  return M == kTF32 ? (D == 64 ? 32 : 16) : (D == 64 ? 64 : 32);
}

// 16 bytes of a cache row. kNT: non-temporal, for caches that the Infinity Cache does not hold: each row is read
// once per call then, and keeping it would cost more than it gives.
template <bool kNT>
__device__ __forceinline__ word4_t load_row(const char* p) {
  typedef const __attribute__((address_space(1))) word4_t* global;
  return kNT ? __builtin_nontemporal_load((global)p) : *(global)p;
}

// The address of a pair of 16-byte (four FP32 or eight 16-bit) elements of the output row of (token row,
// head h), elements d ..: four consecutive FP32 elements are consecutive in every layout.
template <int A>
__device__ __forceinline__ void store_out(const AttentionView& a, int row, int h, int dim, int d, const float (&x)[4]) {
  if (A == kTF32 && a.out_layout) {
    const int n = h * dim + d;
    const size_t at = a.out_layout == 1 ? ((((size_t)(row >> 4) * (a.out_ld >> 4) + (n >> 4)) * 64 + (row & 15) + 16 * ((n & 15) >> 2)) * 4)
                                        : (((((size_t)(row >> 4) * (a.out_ld >> 5) + (n >> 5)) * 2 + ((n >> 2) & 1)) * 64 + (row & 15) +
                                            16 * ((n & 31) >> 3)) * 4);
    store_global(a.out + at * 4, float4_t{x[0], x[1], x[2], x[3]});
    return;
  }
  char* p = a.out + row * a.out_token + h * a.out_head + (int64_t)d * (A == kTF32 ? 4 : 2);
  if constexpr (A == kTF32) store_global(p, float4_t{x[0], x[1], x[2], x[3]});
  else store_global(p, word2_t{pack16<A>(x[0], x[1]), pack16<A>(x[2], x[3])});
}

// Few rows over many keys (decoding, short pieces): bound by reading the cache once. Workgroup (split,
// kv head, row tile; stream): MB blocks of 16 rows. Its waves take the keys' tiles in turn, each
// with LDS of its own and no barrier in the loop; the next tile is in flight in registers while one is
// computed. At the end the waves' (m, l, O) are merged through LDS. With splits > 1 the workgroup's own
// are written instead, and cache_combine merges them.
//
// Measured, bfloat16, 32 heads on 8 of 128, single tokens: 64 streams and a window of 4096 166 us (6.45 TB/s); one
// stream, FP16, a window of 131,072 89 us (6.0 TB/s, with the merge of its splits); 64 streams over 8191 rows of 4
// bits 130 us (5.1 TB/s): those are bound by the instructions that unpack a row, 1.7 per element.
//
// A masked key's weight is an exact zero, but zero times a value that is not finite is NaN: tiles that are
// not seen whole look for such values as they are staged, and where there is one they are added apart, for
// the rows that see them (TileMath::add_odd).
template <int A, int C, int D, int MB, int kWaves, bool kNT>
__global__ __launch_bounds__(64 * kWaves, 2 * 4 / kWaves) void cache_attention(CacheView c, RowsView r, AttentionView a) {
  constexpr int M = mfma_type<A, C>();
  constexpr int KT = wave_tile<M, D>();
  using T = TileLayout<M, D>;
  using R = RowLoad<C, D>;
  // (FP16 weights are far finer than a bfloat16 output.)
  using X = TileMath<M, D, D, KT, M != kTF32 && M == A>;
  constexpr int kPerLoad = 64 / R::L;                                // rows of one load of the wave
  constexpr int kLoads = (KT + kPerLoad - 1) / kPerLoad;
  static_assert(KT % kPerLoad == 0);
  constexpr int kTile = KT * T::kRow;
  constexpr int kMerge = MB * 16 * (D + 4) * 4;                      // a wave's O in the merge
  constexpr int kWaveLds = 2 * kTile > kMerge ? 2 * kTile : kMerge;
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kWaveLds];
  __shared__ float ml[kWaves][2][MB * 16];

  const int split = blockIdx.x % a.splits, head = blockIdx.x / a.splits % c.kv_heads;
  const int tile_of_rows = blockIdx.x / a.splits / c.kv_heads, b = blockIdx.y;
  const int64_t start = uniform64(c.positions[b]);
  int first, n;
  stream_rows(r, b, first, n);
  first = __builtin_amdgcn_readfirstlane(first);
  n = __builtin_amdgcn_readfirstlane(n);
  const int row0 = tile_of_rows * MB * 16, rows = n * a.group;
  if (start < 0 || row0 >= rows) return;
  const int last_row = min(row0 + MB * 16, rows) - 1;
  const int64_t ta = start + row0 / a.group, tb = start + last_row / a.group;
  KeyList keys;
  keys.init(c, ta, tb);

  const int wave = wave_id(), lane = lane_id(), g = lane >> 4;
  char* kt = lds + wave * kWaveLds;
  char* vt = kt + kTile;

  // Loads of the tile that starts at list entry j0; entries past the end repeat the last.
  const int p = lane % R::L, sub = lane / R::L;
  const bool keep = p * R::E < c.dim;
  const int64_t base_row = b * c.stream_stride + head * c.head_stride;
  const char* kbase = c.keys + base_row * c.row_bytes;
  const char* vbase = c.values + base_row * c.row_bytes;
  const char* kpbase = C == kTInt4 ? reinterpret_cast<const char*>(c.key_params) + base_row * (c.row_bytes / 4) : nullptr;
  const char* vpbase = C == kTInt4 ? reinterpret_cast<const char*>(c.value_params) + base_row * (c.row_bytes / 4) : nullptr;
  const uint32_t slot_bytes = c.slot_stride * c.row_bytes, chunk = keep ? p * 16 : 0, pair = keep ? p : 0;
  const bool near = slot_bytes < 1u << 25;  // a tile's rows within 32 bits of its first
  struct Loaded {
    word4_t kw[kLoads], vw[kLoads];
    unsigned kp[kLoads], vp[kLoads];
  };
  // The loads have one place and no condition: a branch around them, or two forms of them, makes the compiler
  // move what they return, which waits for it. Those past the last tile repeat it.
  const uint32_t part = sub * slot_bytes;
  auto load = [&](int j0, Loaded& t) {
    uint64_t at[kLoads];
    keys.offsets(j0, kPerLoad, sub, KT, near, slot_bytes, part, at);
#pragma unroll
    for (int i = 0; i < kLoads; i++) t.kw[i] = load_row<kNT>(kbase + at[i] + chunk);
#pragma unroll
    for (int i = 0; i < kLoads; i++) t.vw[i] = load_row<kNT>(vbase + at[i] + chunk);
    if constexpr (C == kTInt4) {
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const uint64_t params = at[i] / 16 * 4 + pair * 4;  // 16 bytes of codes have 4 of scale and minimum
        t.kp[i] = load_global<unsigned>(kpbase + params);
        t.vp[i] = load_global<unsigned>(vpbase + params);
      }
    }
  };

  const int tiles = (keys.total + KT - 1) / KT, per = (tiles + a.splits - 1) / a.splits;
  const int t1 = min((split + 1) * per, tiles);
  int tile = split * per + wave;
  // 4-bit tiles are a quarter of the bytes: two of them in flight per wave.
  constexpr int kSets = C == kTInt4 ? 2 : 1;
  Loaded loaded[kSets];
#pragma unroll
  for (int i = 0; i < kSets; i++) load(min(tile + i * kWaves, tiles - 1) * KT, loaded[i]);

  QueryBlock<A, M, D> q[MB];
  Seen seen[MB];
  float m[MB];
  float4_t o[MB][D / 16 + 1];  // and the sums of the weights
#pragma unroll
  for (int u = 0; u < MB; u++) {
    const int row = min(row0 + u * 16 + (lane & 15), last_row);
    const int token = row / a.group, h = head * a.group + row - token * a.group;
    q[u].load(a.q + (first + token) * a.q_token + h * a.q_head, c.dim, a.scale, g, row0 + u * 16 + (lane & 15) <= last_row);
    seen[u].init(keys, start + token);
    m[u] = -INFINITY;
#pragma unroll
    for (int d = 0; d <= D / 16; d++) o[u][d] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  // List entries that every row sees: from whole_from on, up to whole_to (ring entries).
  const int whole_from = keys.sinks + max((int)(tb - keys.lo) - c.window + 1, 0);
  const int whole_to = keys.sinks + max((int)max(ta - keys.lo, (int64_t)-1) + 1, 0);
  const int whole_sinks = (int)min((int64_t)keys.sinks, ta + 1);

  auto step = [&](int tile, Loaded& in) {
    const int j0 = tile * KT;
    // Whole: every row sees the tile's every entry.
    const bool whole = (j0 >= whole_from && j0 + KT <= whole_to) || j0 + KT <= whole_sinks ||
                       (whole_sinks == keys.sinks && whole_from == keys.sinks && j0 + KT <= whole_to);
    wave_sync();
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      const int row = i * kPerLoad + sub;
      expand<C, M>(in.kw[i], in.kp[i], p, keep, [&](int ch, word4_t w) { lds_put(kt + row * T::kRow + T::key_chunk(row, ch) * 16, w); });
      expand<C, M>(in.vw[i], in.vp[i], p, keep, [&](int ch, word4_t w) { lds_put(vt + row * T::kRow + T::value_chunk(row, ch) * 16, w); });
    }
    wave_sync();
    if (!whole && __ballot(X::template any_odd<64>(vt, lane))) {
      X::add_odd(vt, o, lane, [&](int u, int e) { return seen[u](keys, c.window, j0 + e); });
      wave_sync();
      X::template clear<64>(vt, lane);
      wave_sync();
    }
    float4_t s[MB][X::kBlocks];
    float base[MB];
    if constexpr (two_terms<A, C>()) {
      X::template logits<false>(kt, q, s, lane);
      wave_sync();
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const int row = i * kPerLoad + sub;
        expand<C, M, 1>(in.kw[i], in.kp[i], p, keep, [&](int ch, word4_t w) { lds_put(kt + row * T::kRow + T::key_chunk(row, ch) * 16, w); });
      }
      wave_sync();
    }
    load(min(tile + kSets * kWaves, t1 - 1) * KT, in);
    X::template logits<two_terms<A, C>()>(kt, q, s, lane);
    if (!whole) X::mask(s, seen, keys, c.window, j0, lane);
    move_maxima(s, q, m, base, o);
    X::outputs(vt, s, q, base, o, lane);
  };
  for (; tile < t1; tile += kSets * kWaves) {
    step(tile, loaded[0]);
    if constexpr (kSets > 1) {
      if (tile + kWaves < t1) step(tile + kWaves, loaded[1]);
    }
  }

  // Merge of the four waves.
#pragma unroll
  for (int u = 0; u < MB; u++) {
    const float l = X::row_sum(o[u][D / 16]);
    if (g == 0) {
      ml[wave][0][u * 16 + (lane & 15)] = m[u];
      ml[wave][1][u * 16 + (lane & 15)] = l;
    }
  }
  __syncthreads();
  float* merge = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int u = 0; u < MB; u++) {
    const int row = u * 16 + (lane & 15);
    float top = ml[0][0][row];
#pragma unroll
    for (int w = 1; w < kWaves; w++) top = fmaxf(top, ml[w][0][row]);
    const float f = m[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[u] - top);
#pragma unroll
    for (int d = 0; d < D / 16; d++) {
      const float4_t x = o[u][d] * f;
      *(float4_t*)(merge + (wave * MB * 16 + row) * (D + 4) + d * 16 + g * 4) = x;
    }
  }
  __syncthreads();
  const int quads = c.dim / 4;
  for (int i = threadIdx.x; i < (last_row - row0 + 1) * quads; i += 64 * kWaves) {
    const int row = i / quads, d = (i - row * quads) * 4;
    float top = ml[0][0][row], sum = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; w++) top = fmaxf(top, ml[w][0][row]);
    float4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float mw = ml[w][0][row];
      sum += mw == -INFINITY ? ml[w][1][row] : ml[w][1][row] * __builtin_amdgcn_exp2f(mw - top);
      x += *(const float4_t*)(merge + (w * MB * 16 + row) * (D + 4) + d);
    }
    if (a.splits > 1) {
      const size_t at = (((size_t)b * c.kv_heads + head) * a.rows + row0 + row) * a.splits + split;
      if (d == 0) a.part_ml[at] = make_float2(top, sum);
      store_global(a.part_o + at * c.dim + d, x);
    } else {
      const int token = (row0 + row) / a.group, h = head * a.group + row0 + row - token * a.group;
      const float inv = 1.f / sum;
      const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
      store_out<A>(a, first + token, h, c.dim, d, y);
    }
  }
}

// op over the lanes that share lane % L, in every lane: rotations within rows of 16, then swaps across rows.
template <int L, typename Op>
__device__ __forceinline__ float over_groups(float v, Op&& op) {
  if constexpr (L <= 2) v = op(v, dpp_get<0x4E>(v));   // lane ^ 2
  if constexpr (L <= 4) v = op(v, dpp_get<0x124>(v));  // row_ror:4: any two of lane % 4
  if constexpr (L <= 8) v = op(v, dpp_get<0x128>(v));  // row_ror:8
  float a, b;
  if constexpr (L <= 16) {
    swap_halves<false>(v, a, b);
    v = op(a, b);
  }
  if constexpr (L <= 32) {
    swap_halves<true>(v, a, b);
    v = op(a, b);
  }
  return v;
}
template <int C, int D>
constexpr int vector_loads() {  // loads of K (and of V) in flight per wave
  return C == kTInt4 ? 2 : 8;
}
// One new token per stream with FP32 queries, at most four query heads per cache head: products of so few rows
// would leave most of an FP32 MFMA's 16 idle (16 streams, 16 heads of 64, a window of 512 in 4 bits: 15.7 us,
// bound by them), so they are made by vector instructions, without LDS in the loop: 9.2 us, and 12.0 over FP32
// rows, 5.6 TB/s. A row of the cache is shared by L lanes, E elements each; every group of
// L lanes takes keys of its own, with its own (m, l, O), and the groups and waves are merged at the end. Each
// load's registers are loaded again as soon as they are used. The loop is bound by the cache's bytes where rows
// have 16 bits or more, by the unpacking of 4-bit ones; small calls by the launch and the merge.
template <int C, int D, int R, int kWaves, bool kNT>
__global__ __launch_bounds__(64 * kWaves) void cache_attention_vector(CacheView c, RowsView r, AttentionView a) {
  using Row = RowLoad<C, D>;
  constexpr int E = Row::E, L = Row::L, kGroups = 64 / L, NB = vector_loads<C, D>(), KT = NB * kGroups;
  __shared__ __attribute__((aligned(16))) float merge[kWaves][R][D];
  __shared__ float ml[kWaves][2][R];
  const int split = blockIdx.x % a.splits, head = blockIdx.x / a.splits, b = blockIdx.y;
  const int64_t start = uniform64(c.positions[b]);
  int first, n;
  stream_rows(r, b, first, n);
  first = __builtin_amdgcn_readfirstlane(first);
  n = __builtin_amdgcn_readfirstlane(n);
  if (start < 0 || n == 0) return;
  KeyList keys;
  keys.init(c, start, start);
  const int wave = wave_id(), lane = lane_id(), p = lane % L, sub = lane / L;
  const bool keep = p * E < c.dim;
  const int64_t base_row = b * c.stream_stride + head * c.head_stride;
  const uint32_t slot_bytes = c.slot_stride * c.row_bytes, chunk = keep ? p * 16 : 0, part = sub * slot_bytes;
  const bool near = slot_bytes < 1u << 25;
  const char* const kbase = c.keys + base_row * c.row_bytes + chunk;
  const char* const vbase = c.values + base_row * c.row_bytes + chunk;
  const int64_t pbase = C == kTInt4 ? base_row * (c.row_bytes / 4) + (keep ? p * 4 : 0) : 0;
  const char* const kpbase = reinterpret_cast<const char*>(c.key_params) + pbase;
  const char* const vpbase = reinterpret_cast<const char*>(c.value_params) + pbase;

  // The queries' elements that meet this lane's.
  float q[R][E];
#pragma unroll
  for (int u = 0; u < R; u++) {
    const char* row = a.q + first * a.q_token + (head * a.group + min(u, a.group - 1)) * a.q_head + (keep ? p * E * 4 : 0);
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4_t x = load_global<float4_t>(row + e * 4);
#pragma unroll
      for (int i = 0; i < 4; i++) q[u][e + i] = keep ? x[i] * a.scale : 0.f;
    }
  }
  word4_t kw[NB], vw[NB];
  unsigned kp[NB], vp[NB];
  uint64_t at[NB];
  auto load_keys = [&] {
#pragma unroll
    for (int i = 0; i < NB; i++) {
      kw[i] = load_row<kNT>(kbase + at[i]);
      if constexpr (C == kTInt4) kp[i] = load_global<unsigned>(kpbase + at[i] / 16 * 4);
    }
  };
  auto load_values = [&] {
#pragma unroll
    for (int i = 0; i < NB; i++) {
      vw[i] = load_row<kNT>(vbase + at[i]);
      if constexpr (C == kTInt4) vp[i] = load_global<unsigned>(vpbase + at[i] / 16 * 4);
    }
  };
  // The elements of a load.
  auto widen = [&](word4_t w, unsigned params, float (&x)[E]) {
    if constexpr (C == kTF32) {
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = bits_to_float(w[i]);
    } else if constexpr (C == kTInt4) {
      const half2_t sz = __builtin_bit_cast(half2_t, params);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float4_t f[2];
        dequant8_f32(w[i], (float)sz[0], (float)sz[1], f);
#pragma unroll
        for (int e = 0; e < 8; e++) x[8 * i + e] = f[e >> 2][e & 3];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[2 * i] = low16<C>(w[i]);
        x[2 * i + 1] = high16<C>(w[i]);
      }
    }
  };

  const int tiles = (keys.total + KT - 1) / KT, per = (tiles + a.splits - 1) / a.splits;
  const int t1 = min((split + 1) * per, tiles);
  int tile = split * per + wave;
  keys.offsets(min(tile, tiles - 1) * KT, kGroups, sub, KT, near, slot_bytes, part, at);
  load_keys();
  load_values();
  float m[R], l[R], o[R][E];
#pragma unroll
  for (int u = 0; u < R; u++) {
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) o[u][e] = 0.f;
  }
  for (; tile < t1; tile += kWaves) {
    const int j0 = tile * KT;
    // Entries past the end (of the last tile) weigh nothing, and their loads' repeated rows count as zeros.
    const bool whole = j0 + KT <= keys.total;
    keys.offsets(min(tile + kWaves, t1 - 1) * KT, kGroups, sub, KT, near, slot_bytes, part, at);
    float s[R][NB];
#pragma unroll
    for (int i = 0; i < NB; i++) {
      float x[E];
      widen(kw[i], kp[i], x);
#pragma unroll
      for (int u = 0; u < R; u++) {
        float d[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < E; e++) d[e & 1] = __builtin_fmaf(q[u][e], x[e], d[e & 1]);
        s[u][i] = group_sum(d[0] + d[1], L);
      }
    }
    load_keys();
    if (!whole) {
#pragma unroll
      for (int i = 0; i < NB; i++) {
        const bool in = j0 + i * kGroups + sub < keys.total;
#pragma unroll
        for (int u = 0; u < R; u++) {
          const float x = s[u][i];
          s[u][i] = in ? x : -INFINITY;
        }
#pragma unroll
        for (int w = 0; w < 4; w++) vw[i][w] = in ? vw[i][w] : 0u;
        if constexpr (C == kTInt4) vp[i] = in ? vp[i] : 0u;
      }
    }
    float top[R], base[R];
    bool any = false;
#pragma unroll
    for (int u = 0; u < R; u++) {
      top[u] = s[u][0];
#pragma unroll
      for (int i = 1; i < NB; i++) top[u] = fmaxf(top[u], s[u][i]);
      any |= top[u] > m[u] + 8.f;
    }
    if (__ballot(any)) {  // as in move_maxima
#pragma unroll
      for (int u = 0; u < R; u++) {
        const bool move = top[u] > m[u] + 8.f;
        const float alpha = !move || m[u] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[u] - top[u]);
        l[u] *= alpha;
#pragma unroll
        for (int e = 0; e < E; e++) o[u][e] *= alpha;
        m[u] = move ? top[u] : m[u];
      }
    }
#pragma unroll
    for (int u = 0; u < R; u++) {
      base[u] = m[u] == -INFINITY ? 0.f : m[u];
#pragma unroll
      for (int i = 0; i < NB; i++) {
        s[u][i] = __builtin_amdgcn_exp2f(s[u][i] - base[u]);
        l[u] += s[u][i];
      }
    }
#pragma unroll
    for (int i = 0; i < NB; i++) {
      float x[E];
      widen(vw[i], vp[i], x);
#pragma unroll
      for (int u = 0; u < R; u++) {
#pragma unroll
        for (int e = 0; e < E; e++) o[u][e] = __builtin_fmaf(s[u][i], x[e], o[u][e]);
      }
    }
    load_values();
  }

  // The wave's groups, then the waves.
#pragma unroll
  for (int u = 0; u < R; u++) {
    const float top = over_groups<L>(m[u], [](float a, float b) { return fmaxf(a, b); });
    const float f = m[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[u] - top);
    const auto add = [](float a, float b) { return a + b; };
    const float sum = over_groups<L>(m[u] == -INFINITY ? l[u] : l[u] * f, add);
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float y = over_groups<L>(o[u][e] * f, add);
      if (sub == 0) merge[wave][u][p * E + e] = y;
    }
    if (lane == 0) {
      ml[wave][0][u] = top;
      ml[wave][1][u] = sum;
    }
  }
  __syncthreads();
  const int quads = c.dim / 4;
  for (int i = threadIdx.x; i < a.group * quads; i += 64 * kWaves) {
    const int u = i / quads, d = (i - u * quads) * 4;
    float top = ml[0][0][u], sum = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; w++) top = fmaxf(top, ml[w][0][u]);
    float4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float mw = ml[w][0][u], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - top);
      sum += mw == -INFINITY ? ml[w][1][u] : ml[w][1][u] * f;
      x += *(const float4_t*)(&merge[w][u][d]) * f;
    }
    if (a.splits > 1) {
      const size_t to = (((size_t)b * c.kv_heads + head) * a.rows + u) * a.splits + split;
      if (d == 0) a.part_ml[to] = make_float2(top, sum);
      store_global(a.part_o + to * c.dim + d, x);
    } else {
      const float inv = 1.f / sum;
      const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
      store_out<kTF32>(a, first, head * a.group + u, c.dim, d, y);
    }
  }
}

// Many rows (prompts, long pieces): bound by the matrix products. Workgroup (kv head, row tile; stream):
// waves of MB blocks of 16 rows each. The tile of keys is the workgroup's, staged once for its rows:
// two tiles of LDS, so that one is computed while the next one's loads are in flight (straight to LDS where the
// rows need no conversion), and one barrier per tile. Row tiles of one (stream, kv head) follow each other in the
// grid at steps of kv_heads, those that see most keys first: with eight heads, or a multiple, each XCD's L2 holds
// one head's keys.
//
// Measured, 32 heads on 8 of 128: 8192 tokens, bfloat16, a window of 2048 264 us (910 TF/s of the 1107 that a large
// matrix product reaches): the exponentials and packing between the two products share the issue slots with them,
// and two workgroups per CU overlap most of it. Tiles of 32 keys 316 us, of 128 517; waves of 16 rows 422; eight
// waves 288. Four streams of 1024 FP16 tokens over 4-bit rows, window 4096: 465 us; K in two terms is half as many
// products again. Ragged pieces of up to 333 tokens (19 streams, head dimension 80) 51 us: about 2 us for each tile
// of a workgroup's chain of 13 and some 20 us before and after it, with fewer workgroups than the chip holds.
template <int M, int D>
constexpr int rows_tile() {
  return M == kTF32 ? 4096 / D : D == 256 ? 32 : 64;
}
// Waves of a workgroup: eight where rows are converted on their way (which costs the less per row the more rows
// share it; half of the threads take K, half V), else four, two workgroups per CU. Head dimension 256 leaves
// registers for four waves on a CU.
constexpr int rows_waves(int type, int stored, int dim) { return type == stored || dim > 128 ? 4 : 8; }
constexpr int rows_threads(int type, int stored, int dim) { return 64 * rows_waves(type, stored, dim); }
constexpr int rows_per_cu(int type, int stored, int dim) { return dim > 128 ? 1 : 8 / rows_waves(type, stored, dim); }
template <int A, int C, int D, int U, int MB>
__global__ __launch_bounds__(rows_threads(A, C, D), rows_per_cu(A, C, D))
void cache_attention_rows(CacheView c, RowsView r, AttentionView a) {
  constexpr int M = mfma_type<A, C>();
  constexpr int KT = rows_tile<M, D>();
  using T = TileLayout<M, D>;
  using R = RowLoad<C, D>;
  constexpr bool kTwo = two_terms<A, C>();  // both terms of K are staged
  using X = TileMath<M, D, U, KT, kTwo>;
  constexpr bool kDirect = C == M;
  constexpr int kWaves = rows_waves(A, C, D), kThreads = 64 * kWaves, kRows = kWaves * MB * 16;
  constexpr int kLoaders = kDirect ? kThreads : kThreads / 2;  // of one of K and V
  constexpr int kPerLoad = kLoaders / R::L;  // rows of one load of theirs
  constexpr int kLoads = (KT + kPerLoad - 1) / kPerLoad;
  constexpr int kTile = KT * T::kRow;
  static_assert(!kDirect || KT % kPerLoad == 0);
  __shared__ __attribute__((aligned(16))) char lds[2][kTwo ? 3 : 2][kTile];

  const int split = blockIdx.x % a.splits, head = blockIdx.x / a.splits % c.kv_heads, b = blockIdx.y;
  const int64_t start = uniform64(c.positions[b]);
  int first, n;
  stream_rows(r, b, first, n);
  first = __builtin_amdgcn_readfirstlane(first);
  n = __builtin_amdgcn_readfirstlane(n);
  const int rows = n * a.group, tiles_of_rows = (rows + kRows - 1) / kRows;
  const int tile_of_rows = tiles_of_rows - 1 - (int)(blockIdx.x / a.splits / c.kv_heads);
  if (start < 0 || tile_of_rows < 0) return;
  const int row0 = tile_of_rows * kRows, last_row = min(row0 + kRows, rows) - 1;
  KeyList keys;
  keys.init(c, start + row0 / a.group, start + last_row / a.group);

  const int loader = threadIdx.x % kLoaders, p = loader % R::L, sub = loader / R::L;
  const bool is_v = threadIdx.x >= kLoaders;  // of those that load to registers
  const bool keep = p * R::E < c.dim;
  const int64_t base_row = b * c.stream_stride + head * c.head_stride;
  const char* kbase = c.keys + base_row * c.row_bytes;
  const char* vbase = c.values + base_row * c.row_bytes;
  const char* kpbase = C == kTInt4 ? reinterpret_cast<const char*>(c.key_params) + base_row * (c.row_bytes / 4) : nullptr;
  const char* vpbase = C == kTInt4 ? reinterpret_cast<const char*>(c.value_params) + base_row * (c.row_bytes / 4) : nullptr;
  const uint32_t slot_bytes = c.slot_stride * c.row_bytes, chunk = keep ? p * 16 : 0, pair = keep ? p : 0;
  const bool near = slot_bytes < 1u << 25;  // a tile's rows within 32 bits of its first
  word4_t raw[kLoads];
  unsigned params[kLoads];
  const char* const base = is_v ? vbase : kbase;
  const char* const pbase = is_v ? vpbase : kpbase;
  const uint32_t part = min(sub, KT - 1) * slot_bytes;
  const int wave = wave_id(), lane = lane_id(), g = lane >> 4;
  // The loads of the tile at entry j0: rows that need no conversion go straight to LDS, others to registers.
  auto load = [&](int j0, int buffer) {
    uint64_t at[kLoads];
    keys.offsets(j0, kPerLoad, sub, KT, near, slot_bytes, part, at);
    if constexpr (kDirect) {
      // A wave's load fills 64 consecutive chunks of the tile: the lane fetches the one that belongs there.
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const int row = i * kPerLoad + sub, to = (i * kThreads + wave * 64) * 16;
        const int kc = T::key_chunk(row, p), vc = T::value_chunk(row, p);
        if (kc * R::E < c.dim) load_to_lds(kbase + at[i] + kc * 16, lds[buffer][0] + to);
        if (vc * R::E < c.dim) load_to_lds(vbase + at[i] + vc * 16, lds[buffer][1] + to);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        raw[i] = load_global<word4_t>(base + at[i] + chunk);
        if constexpr (C == kTInt4) params[i] = load_global<unsigned>(pbase + at[i] / 16 * 4 + pair * 4);  // 4 bytes of 16
      }
    }
  };
  // Waits for the loads and stages what came to registers; look: whether any value of V is not finite.
  auto stage = [&](int buffer, bool look) {
    if constexpr (kDirect) {
      wait_loads();
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const int row = i * kPerLoad + sub;
        if (KT % kPerLoad != 0 && row >= KT) break;
        if (!is_v) {
          expand<C, M>(raw[i], params[i], p, keep, [&](int ch, word4_t w) { lds_put(lds[buffer][0] + row * T::kRow + T::key_chunk(row, ch) * 16, w); });
          if constexpr (kTwo)
            expand<C, M, 1>(raw[i], params[i], p, keep, [&](int ch, word4_t w) { lds_put(lds[buffer][2] + row * T::kRow + T::key_chunk(row, ch) * 16, w); });
        } else {
          expand<C, M>(raw[i], params[i], p, keep, [&](int ch, word4_t w) { lds_put(lds[buffer][1] + row * T::kRow + T::value_chunk(row, ch) * 16, w); });
        }
      }
    }
    if (!look) return false;
    __syncthreads();
    return X::template any_odd<kThreads>(lds[buffer][1], threadIdx.x);
  };
  if (kDirect && c.dim < D) {  // the padding, which no load writes
    for (int at = threadIdx.x * 16; at < (int)sizeof(lds); at += kThreads * 16) lds_put(&lds[0][0][0] + at, word4_t{0, 0, 0, 0});
    __syncthreads();
  }

  const int all_tiles = (keys.total + KT - 1) / KT, per = (all_tiles + a.splits - 1) / a.splits;
  const int begin = min(split * per, all_tiles), tiles = min(begin + per, all_tiles);  // this split's: begin .. tiles - 1
  if (begin < tiles) load(begin * KT, begin & 1);
  QueryBlock<A, M, U> q[MB];
  Seen seen[MB];
  float m[MB];
  float4_t o[MB][U / 16 + 1];  // and the sums of the weights
  const int wave_row0 = row0 + wave * MB * 16, wave_last = min(wave_row0 + MB * 16 - 1, last_row);
#pragma unroll
  for (int u = 0; u < MB; u++) {
    const int row = min(wave_row0 + u * 16 + (lane & 15), last_row);
    const int token = row / a.group, h = head * a.group + row - token * a.group;
    q[u].load(a.q + (first + token) * a.q_token + h * a.q_head, c.dim, a.scale, g, wave_row0 + u * 16 + (lane & 15) <= last_row);
    seen[u].init(keys, start + token);
    m[u] = -INFINITY;
#pragma unroll
    for (int d = 0; d <= U / 16; d++) o[u][d] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  // What some of the wave's rows see of the ring's entries: nothing before some_from or from some_to on.
  const bool idle = wave_row0 > last_row;
  const int64_t ta = start + min(wave_row0, last_row) / a.group, tb = start + wave_last / a.group;
  const int newest_a = (int)max(ta - keys.lo, (int64_t)-1), newest_b = (int)max(tb - keys.lo, (int64_t)-1);
  const int some_from = keys.sinks + max(newest_a - c.window + 1, 0);
  const int some_to = newest_b < 0 ? (int)min((int64_t)keys.sinks, tb + 1) : keys.sinks + newest_b + 1;
  // All of the workgroup's rows see the entries [all_from, all_to). Other tiles are looked through for values
  // that are not finite (cache_attention).
  const int all_from = keys.sinks + max(keys.total - keys.sinks - c.window, 0);
  const int all_to = keys.sinks + (int)max(start + row0 / a.group - keys.lo, (int64_t)-1) + 1;
  auto partial = [&](int j0) { return !(j0 >= all_from && j0 + KT <= all_to); };
  bool odd = false;
  if (begin < tiles) odd = __syncthreads_or(stage(begin & 1, partial(begin * KT))) != 0;

  // One tile. kWhole: all of the workgroup's rows see all of it.
  auto step = [&](int tile, auto kWhole) {
    const int j0 = tile * KT, buffer = tile & 1, other = buffer ^ 1;
    const char* kt = lds[buffer][0];
    char* vt = lds[buffer][1];
    bool none = false;
    if constexpr (!kWhole) {
      none = idle || j0 >= some_to || (j0 >= keys.sinks && j0 + KT <= some_from);
      if (odd) {
        if (!none) X::add_odd(vt, o, lane, [&](int u, int e) { return seen[u](keys, c.window, j0 + e); });
        __syncthreads();
        X::template clear<kThreads>(vt, threadIdx.x);
        __syncthreads();
      }
    }
    float4_t s[MB][X::kBlocks];
    float base[MB];
    if (!none) {
      X::template logits<false>(kt, q, s, lane);
      if constexpr (kTwo) X::template logits<true>(lds[buffer][2], q, s, lane);
    }
    // The next tile's loads, after the reads of K: the compiler lets no LDS read pass a load to LDS before it has
    // arrived, and the next ones are V's, behind the maxima. Loads to registers have no condition around them, and
    // repeat the last tile: with one, or in two forms, the compiler moves what they return and waits for it.
    if (!kDirect || tile + 1 < tiles) load(min(tile + 1, tiles - 1) * KT, other);
    if (!none) {
      if constexpr (!kWhole) X::mask(s, seen, keys, c.window, j0, lane);
      move_maxima(s, q, m, base, o);
      X::outputs(vt, s, q, base, o, lane);
    }
    if (tile + 1 < tiles) {
      const bool look = partial(j0 + KT), found = stage(other, look);
      if (look) odd = __syncthreads_or(found) != 0;
      else {
        odd = false;
        __syncthreads();
      }
    }
  };
  // The tiles seen whole are one run: a loop of their own, in which nothing branches around the products (a
  // branch around the masks alone cost a register move per logit).
  const int run_from = max(min((all_from + KT - 1) / KT, tiles), begin), run_to = max(run_from, min(all_to / KT, tiles));
  int tile = begin;
  for (int round = 0; round < 2; round++) {
    const int until = round ? tiles : run_from;
    for (; tile < until; tile++) step(tile, std::false_type{});
    for (; tile < run_to; tile++) step(tile, std::true_type{});
  }

#pragma unroll
  for (int u = 0; u < MB; u++) {
    const float sum = X::row_sum(o[u][U / 16]), inv = 1.f / sum;
    const int row = wave_row0 + u * 16 + (lane & 15);
    if (row <= last_row && a.splits > 1) {
      const size_t at = (((size_t)b * c.kv_heads + head) * a.rows + row) * a.splits + split;
      if (g == 0) a.part_ml[at] = make_float2(m[u], sum);
#pragma unroll
      for (int d = 0; d < U / 16; d++)
        if (d * 16 + g * 4 < c.dim) store_global(a.part_o + at * c.dim + d * 16 + g * 4, o[u][d]);
    } else if (row <= last_row) {
      const int token = row / a.group, h = head * a.group + row - token * a.group;
#pragma unroll
      for (int d = 0; d < U / 16; d++) {
        const float y[4] = {o[u][d][0] * inv, o[u][d][1] * inv, o[u][d][2] * inv, o[u][d][3] * inv};
        if (d * 16 + g * 4 < c.dim) store_out<A>(a, first + token, h, c.dim, d * 16 + g * 4, y);
      }
    }
  }
}

constexpr int kMaxSplits = 64;

// The splits of each row merged: workgroup (row, kv head, stream), 64 lanes of four elements times four
// shares of the splits, joined in a fixed order. Its few reads are in L2: bound by the launch and two round trips,
// 4.6 us of the 89 that one stream's window of 131,072 takes.
template <int A>
__global__ __launch_bounds__(256) void cache_combine(CacheView c, RowsView r, AttentionView a) {
  __shared__ float weight[kMaxSplits];
  __shared__ float4_t part[4][64];
  const int row = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
  int first, n;
  stream_rows(r, b, first, n);
  if (c.positions[b] < 0 || row >= n * a.group) return;
  const size_t at = (((size_t)b * c.kv_heads + head) * a.rows + row) * a.splits;
  const int lane = lane_id(), wave = wave_id();
  const float2 ml = lane < a.splits ? a.part_ml[at + lane] : make_float2(-INFINITY, 0.f);
  const float top = wave_top(ml.x);
  const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
  const float sum = wave_total(ml.x == -INFINITY ? ml.y : ml.y * w);
  if (wave == 0) weight[lane] = w;
  __syncthreads();
  const int d = lane * 4;
  float4_t x = {0.f, 0.f, 0.f, 0.f};
  if (d < c.dim) {
#pragma unroll 4
    for (int s = wave; s < a.splits; s += 4) {
      const float4_t v = load_global<float4_t>(a.part_o + (at + s) * c.dim + d);
      if (weight[s] != 0.f) x += v * weight[s];
    }
  }
  part[wave][lane] = x;
  __syncthreads();
  if (wave == 0 && d < c.dim) {
    x = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
    const float inv = 1.f / sum;
    const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
    const int token = row / a.group, h = head * a.group + row - token * a.group;
    store_out<A>(a, first + token, h, c.dim, d, y);
  }
}

}  // namespace stamd
