// Queries, keys and values of new tokens on their way from the projection to the attention, in one pass:
// RMS norm of each query and key head (x / sqrt(mean(x^2) + eps) * gain), rotation of its first rope_dims
// elements by the position's angles, and the append of keys and values to the cache in its own type.
#pragma once

#include "cache_device.hpp"

namespace stamd {

struct AppendView {
  const char *q, *k, *v;
  char* q_out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;  // strides in bytes
  const float *q_gain, *k_gain;  // [head_dim] or null
  const double* inv_freq;        // [rope_dims / 2] radians per position, or null
  const float2* rope;            // [tokens][rope_dims / 2] (cos, sin), or null
  float epsilon;
  int q_heads, rope_dims;
  int halves;                    // pairs (i, i + rope_dims / 2) instead of (2i, 2i + 1)
  int lane_shift;                // log2 of the lanes that share a head
};

constexpr int kAppendThreads = 256;

// Eight values of one row to the cache, x of elements e0 .. e0 + 7 in each lane; lanes of four share a
// 4-bit group. The 4-bit form: minimum and scale = (maximum - minimum) / 15, both rounded to FP16 (the
// format), then code = round((x - minimum) / scale) of the rounded pair, so that a code is the nearest one
// that the format has. A group with a value that is not finite gets a pair of NaN and reads as NaN.
template <int C>
__device__ __forceinline__ void store_cache(char* row, uint32_t* params, int e0, bool active, const float (&x)[8]) {
  if constexpr (C != kTInt4) {
    if (active) store_eight<C>(row + (size_t)e0 * (C == kTF32 ? 4 : 2), x);
  } else {
    float low = x[0], high = x[0], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      low = fminf(low, x[i]);
      high = fmaxf(high, x[i]);
      sum += x[i] - x[i];  // 0, or NaN where a value is not finite
    }
    low = fminf(low, dpp_get<0xB1>(low));
    low = fminf(low, dpp_get<0x4E>(low));
    high = fmaxf(high, dpp_get<0xB1>(high));
    high = fmaxf(high, dpp_get<0x4E>(high));
    sum = dpp_add<0xB1>(sum);
    sum = dpp_add<0x4E>(sum);
    const _Float16 scale = (_Float16)((high - low) / 15.f + sum), zero = (_Float16)(low + sum);
    const float s = (float)scale, z = (float)zero;
    unsigned word = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float code = s > 0.f ? fminf(fmaxf(rintf((x[i] - z) / s), 0.f), 15.f) : 0.f;
      word |= (unsigned)code << ((i >> 1) * 4 + (i & 1) * 16);
    }
    if (active) {
      store_global(row + e0 / 2, word);
      if ((e0 & 31) == 0)
        store_global(params + e0 / 32, __builtin_bit_cast(unsigned, half2_t{scale, zero}));
    }
  }
}

// One workgroup per token. A head is shared by G = 2^lane_shift lanes, eight elements (16 bytes, 32 of
// FP32) each, and the workgroup's 256 / G groups walk the token's query, key and value heads; four heads
// of a group are loaded before the first is used. The angles are the token's, so they are computed once
// (one pair per thread, the product with the position in 64 bits, which far positions need; the turn's
// fraction then has 24 bits to spare for FP32) while the first heads are in flight.
template <int A, int C>
__global__ __launch_bounds__(kAppendThreads) void cache_append(CacheView c, RowsView r, AppendView a) {
  __shared__ float2 turn[kMaxHeadDim / 2];
  __shared__ float swap[kAppendThreads * 8];
  constexpr int es = A == kTF32 ? 4 : 2;
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  int b, index;
  if (r.offsets) {
    int before = 0;  // streams that end at or before this row
    for (int i = lane; i < (c.streams + 63 & ~63); i += 64)
      before += __builtin_popcountll(__ballot(i < c.streams && r.offsets[min(i, c.streams - 1) + 1] <= row));
    if (before >= c.streams) return;
    int first, n;
    stream_rows(r, before, first, n);
    b = before;
    index = row - first;
    if (index < 0 || index >= n) return;
  } else {
    b = row / r.max_tokens;
    index = row - b * r.max_tokens;
  }
  const int64_t start = c.positions[b];
  if (start < 0) return;
  const int64_t position = start + index;

  const int G = 1 << a.lane_shift, groups = kAppendThreads >> a.lane_shift;
  const int group = threadIdx.x >> a.lane_shift, e0 = (threadIdx.x & (G - 1)) * 8;
  const bool active = e0 < c.dim;
  const int at = active ? e0 : 0;  // lanes past the head load its first elements
  const int heads = a.q_heads + 2 * c.kv_heads;
  const int half = a.rope_dims / 2;
  auto source = [&](int h) -> const char* {
    if (h < a.q_heads) return a.q + row * a.q_token + h * a.q_head + at * es;
    h -= a.q_heads;
    if (h < c.kv_heads) return a.k + row * a.k_token + h * a.k_head + at * es;
    return a.v + row * a.v_token + (h - c.kv_heads) * a.v_head + at * es;
  };
  constexpr int kAhead = 4;
  Eight<A> raw[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; u++) raw[u].load(source(min(group + u * groups, heads - 1)));

  for (int j = threadIdx.x; j < half; j += kAppendThreads) {
    if (a.rope) {
      turn[j] = a.rope[(size_t)row * half + j];
    } else {
      const double turns = (double)position * a.inv_freq[j] * 0.15915494309189535;  // 1 / (2 pi)
      const float x = 2.f * (float)(turns - rint(turns));
      turn[j] = make_float2(cospif(x), sinpif(x));
    }
  }
  float gq[8], gk[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    gq[i] = a.q_gain ? a.q_gain[at + i] : 1.f;
    gk[i] = a.k_gain ? a.k_gain[at + i] : 1.f;
  }
  __syncthreads();
  const int slot = position < c.sinks ? (int)position : c.sinks + ring_offset(c, position);
  const int64_t cache_row = b * c.stream_stride + (int64_t)slot * c.slot_stride;
  float* mine = swap + threadIdx.x * 8;                       // this lane's elements
  const float* head = swap + (threadIdx.x & ~(G - 1)) * 8;    // its head's

  for (int base = 0;; base += kAhead * groups) {
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      // All groups walk the same number of heads: those past the last one load it and store nothing.
      if (base + u * groups >= heads) return;
      const int h = base + u * groups + group;
      const bool mineh = active && h < heads;
      const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + c.kv_heads;
      float x[8];
      raw[u].values(x);
      if (!active) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = 0.f;
      }
      if (!is_v && (is_q ? a.q_gain : a.k_gain)) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss += x[i] * x[i];
        ss = group_sum(ss, G);
        const float scale = 1.f / sqrtf(ss / (float)c.dim + a.epsilon);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = x[i] * scale * (is_q ? gq[i] : gk[i]);
      }
      if (!a.halves) {
        if (!is_v) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int j = e0 / 2 + i;
            if (j < half) {
              const float2 t = turn[j];
              const float x0 = x[2 * i], x1 = x[2 * i + 1];
              x[2 * i] = x0 * t.x - x1 * t.y;
              x[2 * i + 1] = x0 * t.y + x1 * t.x;
            }
          }
        }
      } else if (half) {
        // Partners are half a rotation's width apart: through LDS, within the wave.
        *(float4*)mine = make_float4(x[0], x[1], x[2], x[3]);
        *(float4*)(mine + 4) = make_float4(x[4], x[5], x[6], x[7]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int e = e0 + i;
          y[i] = head[e < half ? e + half : e < 2 * half ? e - half : e];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (!is_v) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int e = e0 + i;
            if (e < 2 * half) {
              const float2 t = turn[e < half ? e : e - half];
              x[i] = e < half ? x[i] * t.x - y[i] * t.y : y[i] * t.y + x[i] * t.x;
            }
          }
        }
      }
      if (is_q) {
        if (mineh) store_eight<A>(a.q_out + row * a.out_token + h * a.out_head + (int64_t)e0 * es, x);
      } else {
        const int kv = min(h, heads - 1) - a.q_heads - (is_v ? c.kv_heads : 0);
        const int64_t to = cache_row + kv * c.head_stride;
        uint32_t* params = is_v ? c.value_params : c.key_params;
        store_cache<C>((is_v ? c.values : c.keys) + to * c.row_bytes, params + (C == kTInt4 ? to * (c.dim / 32) : 0), e0,
                       mineh, x);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++) raw[u].load(source(min(base + (kAhead + u) * groups + group, heads - 1)));
  }
}

}  // namespace stamd
