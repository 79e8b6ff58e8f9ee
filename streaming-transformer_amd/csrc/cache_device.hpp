// The sliding-window cache as its operators' kernels see it, on gfx950. A cache holds, for each stream
// and key/value head, `sinks` rows for the positions 0 .. sinks - 1 and a ring of `ring` rows for the
// positions after them: position p lives in slot p (p < sinks) or sinks + (p - sinks) mod ring. A query
// at position t sees the positions p <= t with p < sinks or p > t - window. A call brings up to
// max_tokens new tokens per stream, and ring >= window + max_tokens - 1, so that no row that one of its
// queries sees has been overwritten by another of its tokens: all queries of a call read the cache as it
// is after the append, whatever number of tokens they came in with.
//
// Rows are FP32, FP16, bfloat16 or 4-bit: codes 0 .. 15 and, for each 32 values, an FP16 pair (scale,
// minimum); a code stands for minimum + scale * code. In each 32-bit word of eight codes element 2j is
// in bits 4j .. and element 2j + 1 in bits 16 + 4j ..: masked with 0x000f000f after a shift by 4j, the two
// halves of the word are two consecutive elements, ready for packed FP16 arithmetic.
#pragma once

#include "step_device.hpp"

#include <cstdint>

namespace stamd {

enum CacheType : int { kTF32 = 0, kTF16 = 1, kTB16 = 2, kTInt4 = 3 };

constexpr int kQuantGroup = 32;   // values of a row that share a (scale, minimum) pair
constexpr int kMaxHeadDim = 256;

struct CacheView {
  char *keys, *values;              // rows of row_bytes
  uint32_t *key_params, *value_params;  // 4-bit rows: head_dim / 32 words, scale in the low half
  int64_t stream_stride, head_stride;   // in rows
  uint32_t slot_stride;                 // in rows
  uint32_t row_bytes;
  const int64_t* positions;         // [streams] position of the stream's first new token; < 0: no part in the call
  int streams, kv_heads, dim, window, sinks, ring;
};

struct RowsView {
  const int32_t* offsets;  // [streams + 1] first row of each stream, or null: max_tokens rows each
  int tokens, max_tokens;
};

// Rows [first, first + n) of stream b, clamped to the rows that the call has.
__device__ __forceinline__ void stream_rows(const RowsView& r, int b, int& first, int& n) {
  if (r.offsets) {
    first = min(max(r.offsets[b], 0), r.tokens);
    n = min(min(r.offsets[b + 1], r.tokens) - first, r.max_tokens);
    n = max(n, 0);
  } else {
    first = b * r.max_tokens;
    n = r.max_tokens;
  }
}

// The ring slot of position p >= sinks. A 64-bit remainder only where the position needs it.
__device__ __forceinline__ int ring_offset(const CacheView& c, int64_t p) {
  const int64_t x = p - c.sinks;
  return x <= 0x7fffffff ? (int)((uint32_t)x % (uint32_t)c.ring) : (int)(x % c.ring);
}

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));
typedef unsigned word2_t __attribute__((ext_vector_type(2)));
typedef unsigned word4_t __attribute__((ext_vector_type(4)));
typedef float float4_t __attribute__((ext_vector_type(4)));

// Loads and stores through the global address space (a flat access would also count on the LDS counter).
template <typename T>
__device__ __forceinline__ T load_global(const void* p) {
  return *(const __attribute__((address_space(1))) T*)p;
}
template <typename T>
__device__ __forceinline__ void store_global(void* p, T v) {
  *(__attribute__((address_space(1))) T*)p = v;
}

__device__ __forceinline__ float bits_to_float(unsigned u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ unsigned float_to_bits(float f) { return __builtin_bit_cast(unsigned, f); }
// Two FP32 values rounded (nearest even) to a pair of 16-bit ones.
__device__ __forceinline__ unsigned pack_f16(float a, float b) {
  return __builtin_bit_cast(unsigned, half2_t{(_Float16)a, (_Float16)b});
}
__device__ __forceinline__ unsigned pack_b16(float a, float b) {
  typedef __bf16 bhalf2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, bhalf2_t{(__bf16)a, (__bf16)b});
}
template <int T>
__device__ __forceinline__ unsigned pack16(float a, float b) {
  if constexpr (T == kTF16) return pack_f16(a, b);
  else return pack_b16(a, b);
}
// The two values of a 16-bit pair.
template <int T>
__device__ __forceinline__ float low16(unsigned u) {
  if constexpr (T == kTF16) return (float)__builtin_bit_cast(_Float16, (unsigned short)u);
  else return bits_to_float(u << 16);
}
template <int T>
__device__ __forceinline__ float high16(unsigned u) {
  if constexpr (T == kTF16) return (float)__builtin_bit_cast(_Float16, (unsigned short)(u >> 16));
  else return bits_to_float(u & 0xffff0000u);
}

// Orders a wave's LDS accesses among its lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Eight consecutive elements of type T (FP32, FP16 or bfloat16) as loaded, and as FP32 values.
template <int T>
struct Eight {
  word4_t w[T == kTF32 ? 2 : 1];
  __device__ __forceinline__ void load(const char* p) {
    w[0] = load_global<word4_t>(p);
    if constexpr (T == kTF32) w[1] = load_global<word4_t>(p + 16);
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    if constexpr (T == kTF32) {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = bits_to_float(w[i >> 2][i & 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const unsigned u = w[0][i];
        x[2 * i] = low16<T>(u);
        x[2 * i + 1] = high16<T>(u);
      }
    }
  }
};
template <int T>
__device__ __forceinline__ void store_eight(char* p, const float (&x)[8]) {
  if constexpr (T == kTF32) {
    store_global(p, float4_t{x[0], x[1], x[2], x[3]});
    store_global(p + 16, float4_t{x[4], x[5], x[6], x[7]});
  } else {
    store_global(p, word4_t{pack16<T>(x[0], x[1]), pack16<T>(x[2], x[3]), pack16<T>(x[4], x[5]), pack16<T>(x[6], x[7])});
  }
}

}  // namespace stamd
