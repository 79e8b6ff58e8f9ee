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
  float epsilon, inv_dim;
  int q_heads, rope_dims;
  int halves;                    // pairs (i, i + rope_dims / 2) instead of (2i, 2i + 1)
  int lane_shift;                // log2 of the lanes that share a head
};

constexpr int kAppendThreads = 256;

__device__ __forceinline__ void lds_put4(float* p, float a, float b, float c, float d) {
  *(__attribute__((address_space(3))) float4_t*)p = float4_t{a, b, c, d};
}

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

// A team of kTeam threads per token: the workgroup for few tokens, a wave for many (four tokens per workgroup,
// and no barrier), a quarter of a wave where those have few heads (then the teams of a wave return apart, and
// nothing crosses them). A head is shared by G = 2^lane_shift lanes, eight elements (16 bytes, 32 of FP32) each, and
// the team's kTeam / G groups walk the token's query, key and value heads, four of a group in flight. A lane's
// elements are the same of every head, so its gains and angles stay in registers. The angles are computed once
// per token (a pair per lane; the product with the position in 64 bits, which far positions need: the turn's
// fraction then has 24 bits to spare for FP32) while the first heads are in flight. Pairs (i, i + half)
// are exchanged through the wave's own LDS, 16 bytes at a time where half is a multiple of 8.
//
// Measured, 32 heads on 8 of 128, bfloat16: 16,384 tokens 89 us, 4.5 TB/s, bound by the bytes (a large copy reaches
// 4.8); 256 tokens 6.3 us, one token 4.2: the launch and the chain of dependent loads (stream, position, heads).
// Loading heads, frequencies and gains before the stream is looked up cost 0.8 us: loads return in order, so the
// lookup then waits for them.
template <int A, int C, int kTeam>
__global__ __launch_bounds__(kAppendThreads) void cache_append(CacheView c, RowsView r, AppendView a) {
  constexpr int kTeams = kAppendThreads / kTeam, kAhead = 4;
  constexpr int es = A == kTF32 ? 4 : 2;
  __shared__ float2 turns[kTeams][kMaxHeadDim / 2];
  __shared__ __attribute__((aligned(16))) float swaps[kAppendThreads / 64][2][64 * 4];
  const int wave = wave_id(), lane = lane_id();
  const int thread = threadIdx.x % kTeam;  // of the team
  float2* const turn = turns[threadIdx.x / kTeam];
  const int row = blockIdx.x * kTeams + (kTeam == 64 ? wave : threadIdx.x / kTeam);
  if (kTeams > 1 && row >= r.tokens) return;
  int b, index;
  if (r.offsets) {
    int before = 0;  // streams that end at or before this row
    if constexpr (kTeam < 64) {
      for (int i = thread; i < c.streams; i += kTeam) before += r.offsets[i + 1] <= row;
      before = (int)group_sum((float)before, kTeam);
    } else {
      for (int i = lane; i < ((c.streams + 63) & ~63); i += 64)
        before += __builtin_popcountll(__ballot(i < c.streams && r.offsets[min(i, c.streams - 1) + 1] <= row));
      before = __builtin_amdgcn_readfirstlane(before);
    }
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

  const int G = 1 << a.lane_shift, groups = kTeam >> a.lane_shift;
  const int group = thread >> a.lane_shift, e0 = (thread & (G - 1)) * 8;
  const bool active = e0 < c.dim;
  const int at = active ? e0 : 0;  // lanes past the head load its first elements
  const int heads = a.q_heads + 2 * c.kv_heads;
  const int half = a.rope_dims / 2;
  const char* const q = a.q + row * a.q_token + at * es;
  const char* const k = a.k + row * a.k_token + at * es;
  const char* const v = a.v + row * a.v_token + at * es;
  const int64_t q_head = a.q_head, k_head = a.k_head, v_head = a.v_head;
  const int q_heads = a.q_heads, k_end = a.q_heads + c.kv_heads;
  auto source = [=](int h) {  // by value: selects of the arguments' addresses would put them into scratch memory
    const int64_t qo = h * q_head, ko = (h - q_heads) * k_head, vo = (h - k_end) * v_head;
    const char* const kv = h < k_end ? k + ko : v + vo;
    return h < q_heads ? q + qo : kv;
  };
  Eight<A> raw[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; u++) raw[u].load(source(min(group + u * groups, heads - 1)));

  for (int j = thread; j < half; j += kTeam) {
    if (a.rope) {
      turn[j] = a.rope[(size_t)row * half + j];
    } else {
      const double turned = (double)position * a.inv_freq[j] * 0.15915494309189535;  // 1 / (2 pi)
      const float x = 2.f * (float)(turned - rint(turned));
      turn[j] = make_float2(cospif(x), sinpif(x));
    }
  }
  float gq[8], gk[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    gq[i] = a.q_gain ? a.q_gain[at + i] : 1.f;
    gk[i] = a.k_gain ? a.k_gain[at + i] : 1.f;
  }
  if constexpr (kTeam <= 64) wave_sync();
  else __syncthreads();
  // Element i of the lane is rotated with its partner y: x cos - y sin (first of its pair) or x cos + y sin.
  // Elements that do not rotate: cos 1, and no partner.
  float co[8], si[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int e = e0 + i, j = a.halves ? (e < half ? e : e - half) : e / 2;
    const bool rotates = e < 2 * half, second = a.halves ? e >= half : i & 1;
    const float2 x = turn[rotates ? j : 0];
    co[i] = rotates ? x.x : 1.f;
    si[i] = !rotates ? 0.f : second ? x.y : -x.y;
  }
  const int slot = position < c.sinks ? (int)position : c.sinks + ring_offset(c, position);
  const int64_t cache_row = b * c.stream_stride + (int64_t)slot * c.slot_stride;
  const int block = e0 / 8, half_block = half / 8;  // of the head, in lanes
  const bool rotate_block = e0 < 2 * half;
  const int partner = lane + (!rotate_block ? 0 : block < half_block ? half_block : -half_block);
  float(*const swap)[64 * 4] = swaps[wave];

  for (int base = 0;; base += kAhead * groups) {
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      // All groups walk the same number of heads: those past the last one load it and store nothing.
      if (base + u * groups >= heads) return;
      const int h = base + u * groups + group;
      const bool mine = active && h < heads;
      const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + c.kv_heads;
      float x[8];
      raw[u].values(x);
      if (!active) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = 0.f;
      }
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) ss += x[i] * x[i];
      ss = group_sum(ss, G);
      // The reciprocal root to 1 ulp by the instruction (its argument, at least epsilon, is a normal number).
      const float scale = __builtin_amdgcn_rsqf(__builtin_fmaf(ss, a.inv_dim, a.epsilon));
      const bool normed = !is_v && (is_q ? a.q_gain : a.k_gain);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float y = x[i] * scale * (is_q ? gq[i] : gk[i]);
        x[i] = normed ? y : x[i];
      }
      if (half) {
        float y[8];
        if (!a.halves) {
#pragma unroll
          for (int i = 0; i < 8; i++) y[i] = x[i ^ 1];
        } else {
          lds_put4(swap[0] + lane * 4, x[0], x[1], x[2], x[3]);
          lds_put4(swap[1] + lane * 4, x[4], x[5], x[6], x[7]);
          wave_sync();
          if (half % 8 == 0) {
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = swap[i >> 2][partner * 4 + (i & 3)];
          } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int e = e0 + i, pe = e < half ? e + half : e < 2 * half ? e - half : e;
              y[i] = swap[(pe >> 2) & 1][((lane & ~(G - 1)) + pe / 8) * 4 + (pe & 3)];
            }
          }
          wave_sync();
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          // What does not rotate stays as it is, infinities too.
          const float z = x[i] * co[i] + y[i] * si[i];
          x[i] = !is_v && e0 + i < 2 * half ? z : x[i];
        }
      }
      if (is_q) {
        if (mine) store_eight<A>(a.q_out + row * a.out_token + h * a.out_head + (int64_t)e0 * es, x);
      } else {
        const int kv = min(h, heads - 1) - a.q_heads - (is_v ? c.kv_heads : 0);
        const int64_t to = cache_row + kv * c.head_stride;
        uint32_t* params = is_v ? c.value_params : c.key_params;
        store_cache<C>((is_v ? c.values : c.keys) + to * c.row_bytes, params + (C == kTInt4 ? to * (c.dim / 32) : 0), e0,
                       mine, x);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++) raw[u].load(source(min(base + (kAhead + u) * groups + group, heads - 1)));
  }
}

}  // namespace stamd
