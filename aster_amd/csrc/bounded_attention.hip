// C ABI of the attention of a bounded cache: sliding windows beside which the first tokens
// stay visible, and attention that gathers each key's softmax weight. Argument checks,
// workspace layout and the choice of kernels (decode_bounded.hip, prefill.hip,
// chunk_weights.hip).
#include <algorithm>
#include <mutex>

#include "bounded_common.h"

namespace astr {
namespace attn {
namespace {

constexpr int kIdsPerWave = 64;  // block ids a decode wave holds, one a lane

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Compute units of the current device (256 when no device is visible).
int device_cus() {
  static std::mutex mu;
  static int cus[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  std::lock_guard<std::mutex> lock(mu);
  if (cus[dev] == 0) {
    int v = 0;
    cus[dev] = (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) ==
                    hipSuccess && v > 0)
                   ? v
                   : 256;
  }
  return cus[dev];
}

// The shape of a call, and what its launches take of the workspace.
struct Shape {
  int32_t num_seqs, num_q_heads, num_kv_heads, head_dim, max_context, window, sinks;
  int32_t num_q_tokens, max_q_len;  // 0: one query token per sequence, no offsets
  int32_t terms;                    // f16 terms of a query (chunks' weights)
  bool weights;
};
struct Plan {
  int32_t waves, part_blocks, parts;     // decode
  int64_t score_stride;
  int32_t column_pieces, column_tiles;   // chunks' weights
  size_t o_bytes, ml_bytes, score_bytes, column_bytes, prefill_bytes;
  size_t decode() const { return o_bytes + ml_bytes + score_bytes; }
  // the decode launches and the chunks' follow one another on the stream and share the bytes
  size_t total() const { return std::max(decode(), prefill_bytes + column_bytes); }
};

// Blocks of the longest row's visible list at most.
int64_t visible_blocks(const Shape& s) {
  const int64_t all = ((int64_t)s.max_context + kBlockTokens - 1) / kBlockTokens;
  if (s.window <= 0) return all;
  const int64_t seen = ((int64_t)s.window + kBlockTokens - 1) / kBlockTokens + 1 +
                       ((int64_t)s.sinks + kBlockTokens - 1) / kBlockTokens;
  return std::min(all + 1, seen);  // (a block of sinks and window keys is listed twice)
}

constexpr int64_t kMostPieces = 32;  // of a chunk's columns

// Partials of the prefill launch's split units: what a call of this shape may use.
constexpr size_t kPrefillPartials = (size_t)64 << 20;

Plan plan_call(const Shape& s) {
  Plan p{};
  const int64_t blocks = std::max<int64_t>(visible_blocks(s), 1);
  const int64_t units = std::max<int64_t>((int64_t)s.num_seqs * s.num_kv_heads, 1);
  const int64_t cus = device_cus();
  // A workgroup of 16 waves (8 at head dim 256, where the LDS holds no more stages) has the
  // CU to itself, two of 8 share it and hide each other's first loads and last merge: 16 where
  // every CU takes several units (128 rows, window 4096: 164 us a call against 167 with 8 waves and
  // 174 with 4), 8 where it takes one or none (48 rows, 4 KV heads, window 1024: 15.3 against
  // 17.8 and 20.2).
  p.waves = units > cus ? wide_waves(s.head_dim, s.weights && s.terms == 2) : 8;
  // pieces: of 64 blocks a wave at most, and enough of them to give every CU 16 waves
  int64_t parts = (blocks + (int64_t)p.waves * kIdsPerWave - 1) / ((int64_t)p.waves * kIdsPerWave);
  const int64_t want = 16 * cus / (units * p.waves);
  const int64_t most = blocks / (8 * p.waves);  // (eight blocks a wave are worth a launch more)
  parts = std::max(parts, std::min(want, most));
  parts = std::max<int64_t>(parts, 1);
  p.part_blocks = (int32_t)((blocks + parts - 1) / parts);
  p.parts = (int32_t)((blocks + p.part_blocks - 1) / p.part_blocks);
  if (p.parts > 1) {
    const size_t slots = (size_t)s.num_seqs * s.num_q_heads * p.parts;
    p.o_bytes = align256(slots * s.head_dim * sizeof(float));
    p.ml_bytes = align256(slots * 2 * sizeof(float));
  }
  if (s.weights) {
    p.score_stride = ((int64_t)s.max_context + kBlockTokens - 1) / kBlockTokens * kBlockTokens;
    p.score_bytes = align256((size_t)s.num_seqs * s.num_q_heads * p.score_stride * sizeof(float));
  }
  if (s.max_q_len > 1) {
    p.prefill_bytes = kPrefillPartials;
    if (s.weights) {
      const int64_t group = s.num_q_heads / s.num_kv_heads;
      // pieces of the column tiles for eight workgroups a CU, of 16 tiles at least
      const int64_t keys = kWaves * (s.head_dim == 256 ? 32 : 64);
      const int64_t units = (int64_t)s.num_seqs * s.num_kv_heads * ((s.max_context + keys - 1) / keys);
      const int64_t columns = ((int64_t)s.max_q_len * group + 31) / 32;
      int64_t pieces = std::min<int64_t>(8 * cus / std::max<int64_t>(units, 1), columns / 16);
      pieces = std::max<int64_t>(std::min<int64_t>(pieces, kMostPieces), 1);
      p.column_tiles = (int32_t)((columns + pieces - 1) / pieces);
      p.column_pieces = (int32_t)((columns + p.column_tiles - 1) / p.column_tiles);
      const size_t tiles = ((size_t)s.num_q_tokens * group / 32 + s.num_seqs) * s.num_kv_heads;
      p.column_bytes = align256(tiles * (32 * 8 + (size_t)s.terms * s.head_dim * 64));
      if (p.column_pieces > 1)
        p.column_bytes += align256((size_t)s.num_seqs * s.num_kv_heads * p.column_pieces *
                                   p.score_stride * sizeof(float));
    }
  }
  return p;
}

bool sane(const Shape& s) {
  return s.num_seqs >= 0 && s.num_q_heads >= 1 && s.num_kv_heads >= 1 && s.head_dim >= 1 &&
         s.max_context >= 0 && s.window >= 0 && s.sinks >= 0 && s.num_q_tokens >= 0 &&
         s.max_q_len >= 0 && s.num_q_heads % s.num_kv_heads == 0;
}

struct Call {
  const astr_paged_kv* cache;
  const void* query;
  int32_t q_dtype;
  int64_t q_tok, q_head;
  void* out;
  int64_t o_tok, o_head;
  const int32_t* query_start_loc;
  int32_t num_query_tokens, max_query_len;
  const int32_t* block_tables;
  int32_t block_table_stride;
  const int32_t* context_lens;
  int32_t num_seqs, num_q_heads, max_context_len;
  float scale;
  int32_t window, sinks;
  const astr_key_weights* weights;
  void* workspace;
  size_t workspace_bytes;
  int32_t* err_flag;
  void* stream;
};

int bounded_attention(const Call& c) {
  const astr_paged_kv* cache = c.cache;
  if (cache == nullptr || c.err_flag == nullptr)
    return fail(ASTR_EINVAL, "cache descriptor and err_flag are required");
  if (c.num_seqs < 0 || c.num_q_heads < 1 || c.max_context_len < 0 || c.block_table_stride < 0)
    return fail(ASTR_EINVAL, "num_seqs/max_context_len/block_table_stride must be >= 0 and "
                             "num_q_heads >= 1");
  if (c.num_seqs == 0) return 0;
  if (c.num_seqs > 65535) return fail(ASTR_EUNSUPPORTED, "more than 65535 sequences per launch");
  const bool packed = c.query_start_loc != nullptr;
  if (packed && (c.num_query_tokens < 0 || c.max_query_len < 0))
    return fail(ASTR_EINVAL, "num_query_tokens and max_query_len must be >= 0");
  if (packed && c.num_query_tokens == 0) return 0;
  if (c.query == nullptr || c.out == nullptr || c.block_tables == nullptr || c.context_lens == nullptr)
    return fail(ASTR_EINVAL, "query, out, block_tables and context_lens are required");
  if (!(c.scale > 0.f) || !std::isfinite(c.scale))
    return fail(ASTR_EINVAL, "attention scale must be finite and positive");
  if (c.window < 0 || c.sinks < 0) return fail(ASTR_EINVAL, "window and sinks must be >= 0");
  if (cache->block_size != kBlockTokens)
    return fail(ASTR_EUNSUPPORTED, "block_size %d != 16", cache->block_size);
  if (cache->code_format != ASTR_KV_INT8 && cache->code_format != ASTR_KV_FP8_E4M3FN &&
      cache->code_format != ASTR_KV_FP8_E5M2)
    return fail(ASTR_EUNSUPPORTED, "code format %d is not int8 / fp8 e4m3fn / fp8 e5m2",
                cache->code_format);
  if (cache->num_kv_heads < 1 || c.num_q_heads % cache->num_kv_heads != 0)
    return fail(ASTR_EINVAL, "num_q_heads %d must be a multiple of num_kv_heads %d", c.num_q_heads,
                cache->num_kv_heads);
  if (cache->num_kv_heads > 65535)
    return fail(ASTR_EUNSUPPORTED, "more than 65535 KV heads per launch");
  const int group = c.num_q_heads / cache->num_kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8 && group != 16)
    return fail(ASTR_EUNSUPPORTED, "GQA group size %d not supported", group);
  if (cache->head_dim != 64 && cache->head_dim != 128 && cache->head_dim != 256)
    return fail(ASTR_EUNSUPPORTED, "head_dim %d not in {64,128,256}", cache->head_dim);
  if (cache->num_blocks < 1) return fail(ASTR_EINVAL, "cache has no blocks");
  if ((int64_t)c.max_context_len > (int64_t)c.block_table_stride * kBlockTokens)
    return fail(ASTR_EINVAL, "max_context_len %d exceeds block table capacity %lld",
                c.max_context_len, (long long)c.block_table_stride * kBlockTokens);
  if (c.q_dtype != ASTR_F32 && c.q_dtype != ASTR_F16 && c.q_dtype != ASTR_BF16)
    return fail(ASTR_EUNSUPPORTED, "query dtype %d is not f32/f16/bf16", c.q_dtype);
  const int64_t esize = c.q_dtype == ASTR_F32 ? 4 : 2;
  if (!aligned16(c.query) || !aligned16(c.out) || (c.q_tok * esize) % 16 ||
      (c.q_head * esize) % 16 || (c.o_tok * esize) % 16 || (c.o_head * esize) % 16)
    return fail(ASTR_EINVAL, "query/out rows must be 16-byte aligned");
  if (!aligned16(cache->k_codes) || !aligned16(cache->v_codes) ||
      cache->code_block_stride % 16 || cache->code_head_stride % 16 ||
      !aligned16(cache->k_scales) || !aligned16(cache->v_scales) ||
      cache->scale_block_stride % 4 || cache->scale_head_stride % 4)
    return fail(ASTR_EINVAL, "cache code and scale blocks must be 16-byte aligned");
  if (cache->key_valid != nullptr && !aligned16(cache->key_valid))
    return fail(ASTR_EINVAL, "cache key_valid must be 16-byte aligned");
  const astr_key_weights* w = c.weights;
  if (w != nullptr) {
    if (w->values == nullptr || w->num_rows < 1 || w->capacity < 0)
      return fail(ASTR_EINVAL, "key weights have no rows");
    if (!aligned16(w->values) || w->row_stride % 4 || w->head_stride % 4)
      return fail(ASTR_EINVAL, "key weight rows must be 16-byte aligned");
    if (w->capacity < c.max_context_len)
      return fail(ASTR_EINVAL, "key weights of %d tokens do not hold max_context_len %d",
                  w->capacity, c.max_context_len);
  }
  const Shape shape{c.num_seqs, c.num_q_heads, cache->num_kv_heads, cache->head_dim,
                    c.max_context_len, c.window, c.sinks, packed ? c.num_query_tokens : 0,
                    packed ? c.max_query_len : 0, c.q_dtype == ASTR_F32 ? 2 : 1, w != nullptr};
  const Plan plan = plan_call(shape);
  const size_t need = plan.total();
  if (need > 0 && (c.workspace == nullptr || c.workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(c.workspace) & 255u) != 0))
    return fail(ASTR_EINVAL, "a 256-byte aligned workspace of %zu bytes is required (%zu given)",
                need, c.workspace_bytes);
  if (plan.parts > INT32_MAX / 2 || (int64_t)c.max_context_len > INT32_MAX - 4096)
    return fail(ASTR_EUNSUPPORTED, "max_context_len %d too large", c.max_context_len);

  SinkChunkArgs chunk{};
  AttnArgs& base = chunk;
  base.q = c.query;
  base.q_tok = c.q_tok;
  base.q_head = c.q_head;
  base.out = c.out;
  base.o_tok = c.o_tok;
  base.o_head = c.o_head;
  base.cache = *cache;
  base.block_tables = c.block_tables;
  base.bt_stride = c.block_table_stride;
  base.context_lens = c.context_lens;
  base.q_start = c.query_start_loc;
  base.num_q_tokens = packed ? c.num_query_tokens : c.num_seqs;
  base.max_q_len = packed ? c.max_query_len : 1;
  base.causal = 1;
  base.num_seqs = c.num_seqs;
  base.num_q_heads = c.num_q_heads;
  base.qk_scale_log2 = c.scale * kLog2e;
  base.window = c.window;
  base.err_flag = c.err_flag;

  BoundedArgs a{};
  static_cast<AttnArgs&>(a) = base;
  a.sinks = c.sinks;
  a.max_context = c.max_context_len;
  a.group = group;
  a.part_blocks = plan.part_blocks;
  a.max_parts = plan.parts;
  a.total_waves = plan.waves;
  // (rows of one sliding window are about equally long; one workgroup a CU or less starts at once)
  const int64_t units = (int64_t)c.num_seqs * cache->num_kv_heads;
  a.longest_first = w != nullptr && c.num_seqs <= 128 && units > device_cus() && units <= 4 * device_cus();
  char* ws = static_cast<char*>(c.workspace);
  a.ws_o = reinterpret_cast<float*>(ws);
  a.ws_ml = reinterpret_cast<float*>(ws + plan.o_bytes);
  a.score_stride = plan.score_stride;
  if (w != nullptr) {
    a.kw = KeyWeights{w->values, w->row_stride, w->head_stride, w->rows, w->num_rows, w->capacity};
    a.scores = reinterpret_cast<float*>(ws + plan.o_bytes + plan.ml_bytes);
  }
  hipStream_t s = static_cast<hipStream_t>(c.stream);
  const bool chunks = packed && c.max_query_len >= 2;
  // The chunk kernels take every row, without a decode launch, where each must carry
  // max_query_len tokens (an offset array that says otherwise is served all the same), and where
  // rows of one token would see few keys and take a place per CU at most: 12 ragged prompts over
  // an FP8 cache, window 256, 46.9 us a call against 48.5 with a launch that finds no row; 300
  // tokens beside 7 rows of one (8 KV heads of 128, window 256) 24.9 against 31.7, beside 31 rows
  // 26.9 against 31.8.
  const int64_t seen = c.window > 0 ? std::min<int64_t>(c.max_context_len, (int64_t)c.window + c.sinks)
                                    : c.max_context_len;
  const bool only_chunks = chunks && c.q_dtype != ASTR_F32 &&
                           !(cache->head_dim == 256 && group == 16) &&
                           ((int64_t)c.num_seqs * c.max_query_len == c.num_query_tokens ||
                            (seen <= 512 && units <= device_cus()));
  if (!only_chunks) {
    const int rc = launch_bounded(a, c.q_dtype, s);
    if (rc != 0 || !chunks) return rc;
  }
  chunk.pf_min_rows = only_chunks ? 1 : 2;
  chunk.max_context = c.max_context_len;
  chunk.pf_ws = static_cast<float*>(c.workspace);
  chunk.pf_bytes = plan.prefill_bytes;
  chunk.sinks = c.sinks;
  if (w != nullptr) a.column_ws = reinterpret_cast<float*>(ws + plan.prefill_bytes);
  chunk.column_ws = a.column_ws;
  const int rc = launch_prefill_sinks(chunk, c.q_dtype, s);
  if (rc != 0 || w == nullptr) return rc;
  a.min_rows = chunk.pf_min_rows;
  a.column_pieces = plan.column_pieces;
  a.column_tiles = plan.column_tiles;
  return launch_chunk_weights(a, c.q_dtype, s);
}

}  // namespace
}  // namespace attn
}  // namespace astr

extern "C" size_t astr_paged_attention_i8_bounded_workspace_bytes(
    int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t q_dtype, int32_t num_query_tokens, int32_t max_query_len, int32_t max_context_len,
    int32_t window, int32_t sinks, int32_t key_weights) {
  using namespace astr::attn;
  const Shape s{num_seqs, num_q_heads, num_kv_heads, head_dim, max_context_len, window, sinks,
                num_query_tokens, max_query_len, q_dtype == ASTR_F32 ? 2 : 1, key_weights != 0};
  return sane(s) && num_seqs > 0 ? plan_call(s).total() : 0;
}

extern "C" int astr_paged_attention_i8_sinks(
    const astr_paged_kv* cache, const void* query, int32_t q_dtype, int64_t q_token_stride,
    int64_t q_head_stride, void* out, int64_t out_token_stride, int64_t out_head_stride,
    const int32_t* query_start_loc, int32_t num_query_tokens, int32_t max_query_len,
    const int32_t* block_tables, int32_t block_table_stride, const int32_t* context_lens,
    int32_t num_seqs, int32_t num_q_heads, int32_t max_context_len, float scale, int32_t window,
    int32_t sinks, void* workspace, size_t workspace_bytes, int32_t* err_flag, void* stream) {
  astr::CallRange range("astr_paged_attention_i8_sinks");
  if (window < 1 || sinks < 1)
    return astr::fail(ASTR_EINVAL, "sinks stay visible beside a window: both must be >= 1");
  return astr::attn::bounded_attention(
      {cache, query, q_dtype, q_token_stride, q_head_stride, out, out_token_stride,
       out_head_stride, query_start_loc, num_query_tokens, max_query_len, block_tables,
       block_table_stride, context_lens, num_seqs, num_q_heads, max_context_len, scale, window,
       sinks, nullptr, workspace, workspace_bytes, err_flag, stream});
}

extern "C" int astr_paged_attention_i8_key_weights(
    const astr_paged_kv* cache, const void* query, int32_t q_dtype, int64_t q_token_stride,
    int64_t q_head_stride, void* out, int64_t out_token_stride, int64_t out_head_stride,
    const int32_t* query_start_loc, int32_t num_query_tokens, int32_t max_query_len,
    const int32_t* block_tables, int32_t block_table_stride, const int32_t* context_lens,
    int32_t num_seqs, int32_t num_q_heads, int32_t max_context_len, float scale,
    const astr_key_weights* weights, void* workspace, size_t workspace_bytes, int32_t* err_flag,
    void* stream) {
  astr::CallRange range("astr_paged_attention_i8_key_weights");
  if (weights == nullptr) return astr::fail(ASTR_EINVAL, "key weights are required");
  return astr::attn::bounded_attention(
      {cache, query, q_dtype, q_token_stride, q_head_stride, out, out_token_stride,
       out_head_stride, query_start_loc, num_query_tokens, max_query_len, block_tables,
       block_table_stride, context_lens, num_seqs, num_q_heads, max_context_len, scale, 0, 0,
       weights, workspace, workspace_bytes, err_flag, stream});
}
