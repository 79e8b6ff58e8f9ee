// The cache operators (include/st_runtime.h: st_qk_norm_rope_append, st_window_attention): checks of the
// arguments, the choice of kernels, and the C entry points. Every check is made on the host before any
// device work; nothing here synchronizes, allocates or copies, so the calls can be captured into a graph.
#include "cache_api.hpp"
#include "cache_append.hpp"
#include "cache_attention.hpp"

#include <atomic>
#include <cmath>

namespace stamd {

namespace {

void require(bool ok, const char* message) {
  if (!ok) throw Error(ST_ERR_INVALID, message);
}

int elem_bytes(int dtype) { return dtype == ST_TYPE_F32 ? 4 : 2; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The library's kernels are gfx950 code: looked up once per device.
void check_device() {
  static std::atomic<bool> known[64];
  int device = 0;
  HIP_CHECK(hipGetDevice(&device));
  if (device < 64 && known[device].load(std::memory_order_relaxed)) return;
  hipDeviceProp_t prop;
  HIP_CHECK(hipGetDeviceProperties(&prop, device));
  if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0)
    throw Error(ST_ERR_DEVICE, std::string("Supported target is gfx950; found ") + prop.gcnArchName);
  if (device < 64) known[device].store(true, std::memory_order_relaxed);
}

void check_types(int dtype, int cache) {
  require(dtype == ST_TYPE_F32 || dtype == ST_TYPE_F16 || dtype == ST_TYPE_BF16, "Unknown element type");
  require(dtype == ST_TYPE_F32 || dtype == cache || cache == ST_TYPE_INT4,
          "16-bit queries need a cache of their own type or of 4 bits");
}

// Strides of [token][head][head_dim] in bytes, checked for 16-byte accesses.
void byte_strides(const void* data, const int64_t (&strides)[2], int dtype, int64_t& token, int64_t& head) {
  const int es = elem_bytes(dtype);
  require(data != nullptr, "Null argument");
  require(aligned(data, 16), "Rows must start at multiples of 16 bytes");
  constexpr int64_t most = (int64_t)1 << 40;
  require(strides[0] > -most && strides[0] < most && strides[1] > -most && strides[1] < most, "Stride out of range");
  require(strides[0] * es % 16 == 0 && strides[1] * es % 16 == 0, "Rows must start at multiples of 16 bytes");
  token = strides[0] * es;
  head = strides[1] * es;
}

void check_heads(const st_kv_cache* cache, const st_new_rows* rows, int q_heads) {
  require(q_heads >= 1 && q_heads <= 65535 && q_heads % cache->kv_heads == 0,
          "Query heads must be a multiple of the cache's heads");
  require((int64_t)rows->max_tokens * q_heads <= (int64_t)1 << 30, "Too many rows in one call");
}

// Head dimension of the kernels: the smallest that holds it.
int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// cache_attention_rows is taken where it has kManyWaves waves, three eighths of what the chip holds, by itself or
// split along the keys into shares of kManyKeys or more. us of cache_attention (split) / cache_attention_rows, 32
// heads on 8, head dimension 128, bfloat16: 128 tokens and a window of 1024, one stream 25 / 35 (128 waves), four
// 35 / 36 (512), 16 123 / 57 (2048); window 8192, one stream 57 / 46 (128 waves x 8 splits), four 159 / 105 (512 x
// 4), 16 613 / 306; one stream of 512 tokens 155 / 100. 12 on 3 of 64, FP16, window 512: 1186 tokens 17 / 18 (456),
// 2400 32 / 20 (912); window 22 10 / 9, 18 / 9. Over 4-bit rows, eight streams, window 2048: 32 tokens 41 / 54 (512
// waves x 2), 128 tokens 100 / 83 (1024).
// Rows per (stream, cache head) above which: a wave of theirs has 32, so fewer leave waves idle, and FP32 products
// or converted rows cost those that work more. 64 streams, window 1024, 32 rows 52 / 55, 36 rows 65 / 52; 4-bit 96
// rows 92 / 97, 128 rows 115 / 95; FP32 (32 streams, window 512) 64 rows 71 / 103, 128 rows 130 / 114.
constexpr int kManyRows = 32, kManyRowsSlow = 96;
constexpr int kManyWaves = 768, kManySplit = 2048, kManyKeys = 1024;
// The Infinity Cache: a larger cache is read with non-temporal loads where each row is read once. 1.07 GB of bfloat16 by
// 64 streams' single tokens 186 us without, 166 with; 0.6 GB of 4-bit rows 165 / 155.
constexpr size_t kStreamBytes = (size_t)256 << 20;

struct Plan {
  bool many;   // cache_attention_rows
  int vector;  // rows of cache_attention_vector; 0, and not many: cache_attention
  int blocks;  // blocks of 16 rows in a workgroup (many: in a wave)
  int waves;   // of a workgroup
  int tiles;   // row tiles of a (stream, kv head)
  int splits;
  bool stream;  // non-temporal loads (decoding)
};
Plan plan_attention(const CacheView& c, const RowsView& r, int q_heads, int dtype, int stored) {
  Plan p{};
  const int rows = r.max_tokens * (q_heads / c.kv_heads), padded = padded_dim(c.dim);
  const int64_t pairs = (int64_t)c.streams * c.kv_heads;
  // Most keys of a tile of rows: its tokens' windows together.
  const auto keys_of = [&](int tile) {
    return (int64_t)c.sinks + c.window + std::min(r.max_tokens, (tile - 1) / (q_heads / c.kv_heads) + 2) - 1;
  };
  if (rows > (dtype != ST_TYPE_F32 && dtype == stored ? kManyRows : kManyRowsSlow)) {
    const int waves = rows_waves(dtype, stored, padded), blocks = padded == 256 ? 1 : 2, tile = 16 * blocks * waves;
    p.tiles = (rows + tile - 1) / tile;
    const int64_t base = pairs * p.tiles;
    const int64_t splits = std::min<int64_t>({kManySplit / (base * waves), keys_of(tile) / kManyKeys, kMaxSplits});
    if (base * waves >= kManyWaves || (splits >= 4 && base * waves * splits >= kManyWaves)) {
      p.many = true;
      p.blocks = blocks;
      p.splits = (int)std::max<int64_t>(1, splits);
      return p;
    }
  }
  p.blocks = rows > 16 && padded < 256 ? 2 : 1;  // head dimension 256: one block's registers fill the file
  p.tiles = (rows + 16 * p.blocks - 1) / (16 * p.blocks);
  const int group = q_heads / c.kv_heads;
  // Four query heads over 4-bit rows, 32 elements of each to a lane, do not fit into registers.
  if (dtype == ST_TYPE_F32 && r.max_tokens == 1 && group <= (stored == ST_TYPE_INT4 ? 2 : 4)) p.vector = group == 3 ? 4 : group;
  const int64_t keys = keys_of(16 * p.blocks);
  p.stream = 2 * pairs * keys * c.row_bytes > (int64_t)kStreamBytes;
  // Workgroups beside the splits.
  const int64_t base = pairs * p.tiles;
  // cache_attention_vector's workgroups end with a merge of all their lanes, which costs most over 4-bit rows (32
  // groups of two lanes), so many short windows take two waves. us of eight / two, 8 heads of 64: 4-bit, 512 pairs
  // 128 keys 12 / 9, 512 keys 17 / 15, 2048 keys 30 / 38; 1024 pairs 21 / 10, 31 / 16, 55 / 40; 4096 pairs 77 / 28,
  // 112 / 51, 208 / 151. FP32, 512 pairs 7.7 / 8.1, 23 / 24; 1024 pairs 128 keys 16 / 14, 512 keys 42 / 44; 4096
  // pairs 51 / 44, 161 / 166.
  const bool two = stored == ST_TYPE_INT4 ? pairs >= (keys <= 1024 ? 512 : 1024) : pairs >= 1024 && keys <= 256;
  // cache_attention: eight waves a CU, in one workgroup, or in two where there are more than one round of those. us of
  // eight / four, bfloat16, 32 heads on 8 of 128: 32 streams (256 workgroups), window 64 8.0 / 7.6, 512 15 / 19, 1024
  // 25 / 29; 64 streams, 64 13 / 8.0, 256 22 / 18, 1024 49 / 47, 4096 168 / 167; 256 streams, 128 60 / 39, 1024 179 /
  // 166; 4 bits 58 / 34, 105 / 85.
  p.waves = p.vector ? (two ? 2 : 8) : p.blocks == 1 && padded < 256 && base <= 256 ? 8 : 4;
  const int64_t room = padded == 256 || p.waves == 8 || p.vector ? 256 : 512;
  const int64_t share = p.waves * 32 * 2;  // fewest keys of a split: two tiles for each wave
  // As many as the chip holds at once and no more, since a second round costs more than idle CUs: us of 3 / 4 splits,
  // 37 streams, two heads (222 / 296 workgroups for 256 CUs), window 3438 28 / 35, head dimension 256 52 / 72, 4-bit
  // (8192) 32 / 45; 1 / 2 splits, 75 streams, window 2048 29 / 39, 8192 118 / 132.
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({room / base, keys / share, kMaxSplits}));
  return p;
}

size_t workspace_of(const CacheView& c, const RowsView& r, int q_heads, const Plan& p) {
  if (p.splits == 1) return 0;
  return (size_t)c.streams * q_heads * r.max_tokens * p.splits * (8 + (size_t)c.dim * 4);
}

// Tokens from which a wave takes one, else a workgroup. us of a workgroup / a wave each, bfloat16, 32 heads on 8 of
// 128: 256 tokens 7.0 / 12.5, 512 9.3 / 13.1, 1024 14.3 / 13.7, 2048 23.8 / 18.7, 4096 39.6 / 26.2; FP32, 16 on 16 of
// 64: 256 tokens 6.1 / 8.5, 1024 11.3 / 10.0, 2048 18.5 / 14.4.
constexpr int kWaveTokens = 1024;
// Few heads (queries', keys' and values' at 8 elements a lane: kFewLanes lanes, twice that from kManyTokens on) leave
// most of a wave idle: 16 lanes a token then. us of 16 / 64 lanes, bfloat16: 32,768 tokens, two heads on one of 64 (32
// lanes) 18 / 43, four on two of 128 (128) 38 / 69, eight on two (192) 46 / 72, 32 on 8 (768) 179 / 166; 4096 tokens
// 6.6 / 8.8, 12 / 13, 15 / 14, 39 / 26.
constexpr int kFewLanes = 128, kFewTokens = 4096, kManyTokens = 16384;

template <int A, int C>
void launch_append(const CacheView& c, const RowsView& r, const AppendView& a, hipStream_t stream) {
  const int lanes = (a.q_heads + 2 * c.kv_heads) << a.lane_shift;
  if (r.tokens >= kFewTokens && a.lane_shift <= 4 && lanes <= (r.tokens >= kManyTokens ? 2 * kFewLanes : kFewLanes))
    hipLaunchKernelGGL((cache_append<A, C, 16>), dim3((r.tokens + 15) / 16), dim3(kAppendThreads), 0, stream, c, r, a);
  else if (r.tokens < kWaveTokens) hipLaunchKernelGGL((cache_append<A, C, 256>), dim3(r.tokens), dim3(kAppendThreads), 0, stream, c, r, a);
  else hipLaunchKernelGGL((cache_append<A, C, 64>), dim3((r.tokens + 3) / 4), dim3(kAppendThreads), 0, stream, c, r, a);
}

template <int A, int C>
void launch_attention(const CacheView& c, const RowsView& r, const AttentionView& a, const Plan& p, hipStream_t stream) {
  const dim3 grid((unsigned)(p.splits * c.kv_heads * p.tiles), c.streams);
  auto go = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, stream, c, r, a); };
  auto form = [&](auto D) {
    constexpr int d = decltype(D)::value;
    if constexpr (d == 128) {  // head dimensions up to 96 in the same tiles, with a quarter of the products less
      if (p.many && c.dim <= 96) return go(cache_attention_rows<A, C, d, 96, 2>, rows_threads(A, C, d));
    }
    if (p.many) return go(cache_attention_rows<A, C, d, d, d == 256 ? 1 : 2>, rows_threads(A, C, d));
    auto few = [&](auto NT) {
      constexpr bool nt = decltype(NT)::value;
      if constexpr (A == kTF32) {
        auto rows = [&](auto R) {
          constexpr int n = decltype(R)::value;
          if (p.waves == 2) go(cache_attention_vector<C, d, n, 2, nt>, 128);
          else go(cache_attention_vector<C, d, n, 8, nt>, 512);
        };
        if (p.vector == 1) return rows(std::integral_constant<int, 1>{});
        if (p.vector == 2) return rows(std::integral_constant<int, 2>{});
        if constexpr (C != kTInt4) {
          if (p.vector == 4) return rows(std::integral_constant<int, 4>{});
        }
      }
      if constexpr (d < 256) {
        if (p.waves == 8) return go(cache_attention<A, C, d, 1, 8, nt>, 512);
      }
      go(cache_attention<A, C, d, 1, 4, nt>, 256);
    };
    if constexpr (d < 256) {
      if (p.blocks == 2) return go(cache_attention<A, C, d, 2, 4, false>, 256);
    }
    if (p.stream) few(std::true_type{});
    else few(std::false_type{});
  };
  const int padded = padded_dim(c.dim);
  if (padded == 64) form(std::integral_constant<int, 64>{});
  else if (padded == 128) form(std::integral_constant<int, 128>{});
  else form(std::integral_constant<int, 256>{});
  HIP_CHECK(hipGetLastError());
  if (p.splits > 1) {
    hipLaunchKernelGGL((cache_combine<A>), dim3(a.rows, c.kv_heads, c.streams), dim3(256), 0, stream, c, r, a);
    HIP_CHECK(hipGetLastError());
  }
}

// go(type of the queries, type of the cache) for the pairs that check_types lets through.
template <typename Go>
void by_types(int dtype, int cache, Go&& go) {
  using std::integral_constant;
  integral_constant<int, kTF32> f32;
  integral_constant<int, kTF16> f16;
  integral_constant<int, kTB16> b16;
  integral_constant<int, kTInt4> int4;
  if (dtype == ST_TYPE_F32) {
    if (cache == ST_TYPE_F32) go(f32, f32);
    else if (cache == ST_TYPE_F16) go(f32, f16);
    else if (cache == ST_TYPE_BF16) go(f32, b16);
    else go(f32, int4);
  } else if (dtype == ST_TYPE_F16) {
    if (cache == ST_TYPE_F16) go(f16, f16);
    else go(f16, int4);
  } else {
    if (cache == ST_TYPE_BF16) go(b16, b16);
    else go(b16, int4);
  }
}

}  // namespace

CacheView cache_view(const st_kv_cache* s) {
  require(s != nullptr, "Null argument");
  require(s->dtype == ST_TYPE_F32 || s->dtype == ST_TYPE_F16 || s->dtype == ST_TYPE_BF16 || s->dtype == ST_TYPE_INT4,
          "Unknown cache type");
  require(s->streams >= 1 && s->streams <= 65535 && s->kv_heads >= 1 && s->kv_heads <= 65535,
          "A cache needs 1 to 65535 streams and heads");
  require(s->head_dim >= 8 && s->head_dim <= kMaxHeadDim && s->head_dim % 8 == 0,
          "The head dimension must be a multiple of 8 up to 256");
  require(s->dtype != ST_TYPE_INT4 || s->head_dim % kQuantGroup == 0,
          "A 4-bit cache needs a head dimension that is a multiple of 32");
  require(s->window >= 1 && s->sinks >= 0 && s->ring >= s->window && (int64_t)s->sinks + s->ring <= (int64_t)1 << 30,
          "A cache needs window >= 1, sinks >= 0, ring >= window and at most 2^30 slots");
  require(s->keys && s->values && s->positions, "Null argument");
  require(aligned(s->keys, 16) && aligned(s->values, 16) && aligned(s->positions, 8), "Misaligned cache");
  if (s->dtype == ST_TYPE_INT4)
    require(s->key_params && s->value_params && aligned(s->key_params, 4) && aligned(s->value_params, 4),
            "A 4-bit cache needs its scales and minimums");
  CacheView c{};
  c.keys = static_cast<char*>(s->keys);
  c.values = static_cast<char*>(s->values);
  c.key_params = static_cast<uint32_t*>(s->key_params);
  c.value_params = static_cast<uint32_t*>(s->value_params);
  c.positions = s->positions;
  c.streams = s->streams;
  c.kv_heads = s->kv_heads;
  c.dim = s->head_dim;
  c.window = s->window;
  c.sinks = s->sinks;
  c.ring = s->ring;
  c.row_bytes = s->dtype == ST_TYPE_INT4 ? s->head_dim / 2 : s->head_dim * elem_bytes(s->dtype);
  int64_t slot = s->slot_stride;
  c.stream_stride = s->stream_stride;
  c.head_stride = s->head_stride;
  if (!slot && !c.stream_stride && !c.head_stride) {
    slot = 1;
    c.head_stride = (int64_t)s->sinks + s->ring;
    c.stream_stride = c.head_stride * s->kv_heads;
  }
  constexpr int64_t most = (int64_t)1 << 40;
  require(slot >= 1 && slot * c.row_bytes < ((int64_t)1 << 32) && c.head_stride >= 0 && c.head_stride < most &&
              c.stream_stride >= 0 && c.stream_stride < most && (s->kv_heads == 1 || c.head_stride > 0) &&
              (s->streams == 1 || c.stream_stride > 0),
          "Cache strides out of range");
  c.slot_stride = (uint32_t)slot;
  return c;
}

RowsView rows_view(const st_kv_cache* s, const st_new_rows* rows) {
  require(rows != nullptr, "Null argument");
  require(rows->tokens >= 0 && rows->tokens <= 1 << 30 && rows->max_tokens >= 1,
          "A call needs tokens between 0 and 2^30 and max_tokens >= 1");
  require(rows->max_tokens <= s->ring - s->window + 1, "More new tokens than the ring has rows beside the window");
  require(rows->offsets || (int64_t)s->streams * rows->max_tokens == rows->tokens,
          "Without offsets every stream brings max_tokens rows");
  require(!rows->offsets || aligned(rows->offsets, 4), "Misaligned offsets");
  return RowsView{rows->offsets, rows->tokens, rows->max_tokens};
}

void append_rows(const st_kv_cache* cache, const st_new_rows* rows, const st_append_args* args, hipStream_t stream) {
  const CacheView c = cache_view(cache);
  const RowsView r = rows_view(cache, rows);
  require(args != nullptr, "Null argument");
  check_types(args->dtype, cache->dtype);
  check_heads(cache, rows, args->q_heads);
  AppendView a{};
  a.q = static_cast<const char*>(args->q);
  a.k = static_cast<const char*>(args->k);
  a.v = static_cast<const char*>(args->v);
  a.q_out = static_cast<char*>(args->q_out);
  if (r.tokens == 0) return;
  byte_strides(args->q, args->q_strides, args->dtype, a.q_token, a.q_head);
  byte_strides(args->k, args->k_strides, args->dtype, a.k_token, a.k_head);
  byte_strides(args->v, args->v_strides, args->dtype, a.v_token, a.v_head);
  byte_strides(args->q_out, args->out_strides, args->dtype, a.out_token, a.out_head);
  require((a.out_token || r.tokens == 1) && (a.out_head || args->q_heads == 1), "Output rows overlap");
  a.q_gain = args->q_gain;
  a.k_gain = args->k_gain;
  a.epsilon = args->epsilon;
  require((!a.q_gain && !a.k_gain) || (std::isfinite(a.epsilon) && a.epsilon >= 1e-37f), "A norm needs an epsilon of at least 1e-37");
  a.inv_dim = 1.f / (float)c.dim;
  a.q_heads = args->q_heads;
  a.rope_dims = args->rope_dims;
  require(a.rope_dims >= 0 && a.rope_dims <= c.dim && a.rope_dims % 2 == 0,
          "Rotated dimensions must be even and at most the head dimension");
  require(args->rope_halves == 0 || args->rope_halves == 1, "rope_halves must be 0 or 1");
  require(a.rope_dims == 0 || (args->inv_freq != nullptr) != (args->rope != nullptr),
          "A rotation needs either its frequencies or its table");
  a.halves = args->rope_halves;
  a.inv_freq = args->inv_freq;
  a.rope = reinterpret_cast<const float2*>(args->rope);
  while ((8 << a.lane_shift) < c.dim) a.lane_shift++;
  check_device();
  by_types(args->dtype, cache->dtype, [&](auto A, auto C) { launch_append<decltype(A)::value, decltype(C)::value>(c, r, a, stream); });
  HIP_CHECK(hipGetLastError());
}

size_t attention_workspace(const st_kv_cache* cache, const st_new_rows* rows, int q_heads, int dtype) {
  const CacheView c = cache_view(cache);
  const RowsView r = rows_view(cache, rows);
  check_types(dtype, cache->dtype);
  check_heads(cache, rows, q_heads);
  return workspace_of(c, r, q_heads, plan_attention(c, r, q_heads, dtype, cache->dtype));
}

void attend_rows(const st_kv_cache* cache, const st_new_rows* rows, const st_attention_args* args, hipStream_t stream,
                 int out_layout, int out_ld) {
  const CacheView c = cache_view(cache);
  const RowsView r = rows_view(cache, rows);
  require(args != nullptr, "Null argument");
  check_types(args->dtype, cache->dtype);
  check_heads(cache, rows, args->q_heads);
  require(std::isfinite(args->scale) && args->scale > 0, "The scale must be positive and finite");
  if (r.tokens == 0) return;
  AttentionView a{};
  a.q = static_cast<const char*>(args->q);
  a.out = static_cast<char*>(args->out);
  byte_strides(args->q, args->q_strides, args->dtype, a.q_token, a.q_head);
  byte_strides(args->out, args->out_strides, args->dtype, a.out_token, a.out_head);
  require((a.out_token || r.tokens == 1) && (a.out_head || args->q_heads == 1), "Output rows overlap");
  a.scale = args->scale * 1.44269504088896341f;  // log2(e): the kernels' exponentials are powers of two
  a.group = args->q_heads / c.kv_heads;
  a.rows = r.max_tokens * a.group;
  a.out_layout = out_layout;
  a.out_ld = out_ld;
  const Plan p = plan_attention(c, r, args->q_heads, args->dtype, cache->dtype);
  a.splits = p.splits;
  const size_t need = workspace_of(c, r, args->q_heads, p);
  if (need) {
    require(args->workspace && aligned(args->workspace, 16) && args->workspace_bytes >= need, "Workspace too small or misaligned");
    a.part_o = static_cast<float*>(args->workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)c.streams * args->q_heads * r.max_tokens * p.splits * c.dim);
  }
  check_device();
  by_types(args->dtype, cache->dtype, [&](auto A, auto C) { launch_attention<decltype(A)::value, decltype(C)::value>(c, r, a, p, stream); });
}

}  // namespace stamd

extern "C" {

int st_qk_norm_rope_append(const st_kv_cache* cache, const st_new_rows* rows, const st_append_args* args, void* stream) {
  return stamd::guarded([&] { stamd::append_rows(cache, rows, args, static_cast<hipStream_t>(stream)); });
}

int st_window_attention_workspace(const st_kv_cache* cache, const st_new_rows* rows, int32_t q_heads, int32_t dtype,
                                  size_t* bytes) {
  return stamd::guarded([&] {
    if (!bytes) throw stamd::Error(ST_ERR_INVALID, "Null argument");
    *bytes = stamd::attention_workspace(cache, rows, q_heads, dtype);
  });
}

int st_window_attention(const st_kv_cache* cache, const st_new_rows* rows, const st_attention_args* args, void* stream) {
  return stamd::guarded([&] { stamd::attend_rows(cache, rows, args, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
