// Arguments and launchers of the operators that keep a paged cache bounded (gfx950):
// attention in which the first tokens stay visible beside a sliding window, and attention
// that adds up each key's softmax weight.
#pragma once

#include "attention_common.h"

namespace astr {
namespace attn {

// The weights gathered per key: row `rows[s]` (s without `rows`) of sequence s, KV head h,
// key t at values[row * row_stride + h * head_stride + t], t < capacity.
struct KeyWeights {
  float* values;
  int64_t row_stride, head_stride;
  const int32_t* rows;
  int32_t num_rows, capacity;
};

struct BoundedArgs : AttnArgs {
  int32_t sinks;        // keys [0, sinks) stay visible beside the window
  int32_t max_context;  // host bound of context_lens
  int32_t group;        // query heads per KV head
  int32_t longest_first;  // decode with key weights: rows in the order of their lengths
  // decode: a row's visible blocks in pieces of part_blocks (AttnArgs), at most max_parts
  KeyWeights kw;
  // base-2 scores of every key, [num_seqs * num_kv_heads * group][score_stride]; weights only
  float* scores;
  int64_t score_stride;
  // chunks (key weights, chunk_weights.hip): their workspace; the pieces of the column tiles and
  // their length
  float* column_ws;
  int32_t min_rows;  // fewest queries of a row the chunk kernels take
  int32_t column_pieces, column_tiles;
};

// What sequence `seq` sees: keys [0, sinks) in blocks [0, sink_blocks) and keys [kv_begin,
// ctx) in blocks [first_blk, last_blk), as one list of blocks. No sink block of its own
// where the window reaches the sinks. A block that holds keys of both is listed twice, each
// time with the bounds of one.
struct VisibleList {
  int ctx, kv_begin, sink_end, sink_blocks, first_blk, blocks;
  __device__ __forceinline__ int block(int f) const {
    return f < sink_blocks ? f : first_blk + f - sink_blocks;
  }
  __device__ __forceinline__ int lo(int f) const { return f < sink_blocks ? 0 : kv_begin; }
  __device__ __forceinline__ int hi(int f) const { return f < sink_blocks ? sink_end : ctx; }
};

// A length outside the table or past the host's bound is reported and cut.
__device__ __forceinline__ int bounded_ctx(const BoundedArgs& a, int ctx, bool report) {
  const int64_t table = (int64_t)a.bt_stride * kBlockTokens;
  const int cap = (int)(table < a.max_context ? table : a.max_context);
  if (ctx < 0 || ctx > cap) {
    if (report) atomicOr(a.err_flag, ASTR_FLAG_BAD_INDEX);
    ctx = ctx < 0 ? 0 : cap;
  }
  return ctx;
}

__device__ __forceinline__ VisibleList visible_list(const BoundedArgs& a, int ctx) {
  VisibleList v;
  v.ctx = ctx;
  const int begin = a.window > 0 && ctx > a.window ? ctx - a.window : 0;
  const bool apart = a.sinks < begin;
  v.kv_begin = apart ? begin : 0;
  v.sink_end = apart ? a.sinks : 0;
  v.sink_blocks = (v.sink_end + kBlockTokens - 1) / kBlockTokens;
  v.first_blk = v.kv_begin / kBlockTokens;
  v.blocks = v.sink_blocks + (ctx + kBlockTokens - 1) / kBlockTokens - v.first_blk;
  return v;
}

// The weights' row of sequence `seq`, or -1 (reported) where its number is out of range.
__device__ __forceinline__ int64_t weight_row(const BoundedArgs& a, int seq, bool report) {
  const int row = a.kw.rows != nullptr ? a.kw.rows[seq] : seq;
  if ((unsigned)row >= (unsigned)a.kw.num_rows) {
    if (report) atomicOr(a.err_flag, ASTR_FLAG_BAD_INDEX);
    return -1;
  }
  return row;
}

// What the attention launch leaves of each query column (token, head of the group) of a chunk for
// the sums over the columns (chunk_weights.hip): {factor, lse}, with score = factor * k_scale *
// (codes . operand) in base 2 and an lse of +inf where the column adds no weight, and the f16
// operands in MFMA order. In tiles of 32 columns: those of sequence s begin at q0 * G / 32 + s, of
// `tiles` per KV head. Behind them the column pieces' sums, one row of score_stride keys per
// (sequence, KV head) and piece.
struct ColumnWs {
  typedef float pair_t __attribute__((ext_vector_type(2)));
  pair_t* cols;
  half8_t* ops;
  float* sums;
  int64_t tiles;
  int group;
  __host__ __device__ ColumnWs(const AttnArgs& a, float* base, int op_halves) {
    group = a.num_q_heads / a.cache.num_kv_heads;
    tiles = (int64_t)a.num_q_tokens * group / 32 + a.num_seqs;
    const int64_t columns = tiles * a.cache.num_kv_heads * 32;
    cols = reinterpret_cast<pair_t*>(base);
    ops = reinterpret_cast<half8_t*>(cols + columns);
    sums = reinterpret_cast<float*>(ops + columns * (op_halves / 8));
  }
  // the first tile of (seq, kvh), whose queries begin at q0
  __device__ int64_t tile0(int seq, int kvh, int q0) const {
    return (int64_t)kvh * tiles + (int64_t)q0 * group / 32 + seq;
  }
};
// A column's log2 of the sum over its keys; +inf where it saw none or its scores are not finite.
__device__ __forceinline__ float column_lse(float m, float l) {
  return l > 0.f ? m + __builtin_amdgcn_logf(l) : INFINITY;
}

template <int KF> int launch_bounded_kf(const BoundedArgs& a, int32_t q_dtype, hipStream_t stream);
template <int KF> int launch_chunk_weights_kf(const BoundedArgs& a, int32_t q_dtype, hipStream_t stream);
// the chunked-prefill kernels with sinks or key weights (prefill.hip)
struct SinkChunkArgs : ChunkArgs {
  int32_t sinks;
  float* column_ws;  // ColumnWs of a call with key weights, else null
};
template <int KF> int launch_prefill_sinks_kf(const SinkChunkArgs& a, int32_t q_dtype, hipStream_t stream);
#define ASTR_DECLARE_BOUNDED(KF)                                                             \
  template <> int launch_bounded_kf<KF>(const BoundedArgs&, int32_t, hipStream_t);           \
  template <> int launch_chunk_weights_kf<KF>(const BoundedArgs&, int32_t, hipStream_t);     \
  template <> int launch_prefill_sinks_kf<KF>(const SinkChunkArgs&, int32_t, hipStream_t);
ASTR_DECLARE_BOUNDED(kInt8)
ASTR_DECLARE_BOUNDED(kE4M3)
ASTR_DECLARE_BOUNDED(kE5M2)
#undef ASTR_DECLARE_BOUNDED

#define ASTR_BY_FORMAT(name, Args)                                               \
  inline int name(const Args& a, int32_t q_dtype, hipStream_t stream) {          \
    switch (a.cache.code_format) {                                               \
      case kInt8: return name##_kf<kInt8>(a, q_dtype, stream);                   \
      case kE4M3: return name##_kf<kE4M3>(a, q_dtype, stream);                   \
      default: return name##_kf<kE5M2>(a, q_dtype, stream);                     \
    }                                                                            \
  }
ASTR_BY_FORMAT(launch_bounded, BoundedArgs)
ASTR_BY_FORMAT(launch_chunk_weights, BoundedArgs)
ASTR_BY_FORMAT(launch_prefill_sinks, SinkChunkArgs)
#undef ASTR_BY_FORMAT

// Waves of the decode kernel's widest workgroup: as many as the LDS holds stages for, and the
// registers (fp32 queries with key weights do not fit the 128 of 16 waves).
constexpr int wide_waves(int head_dim, bool fp32_weights) {
  return head_dim == 256 || fp32_weights ? 8 : 16;
}

}  // namespace attn
}  // namespace astr
