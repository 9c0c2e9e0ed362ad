// Eviction from the paged cache by gathered weight (gfx950): of a row's real tokens (padding
// counts for nothing) the first `sinks` and the last `recent` stay, and of the others the
// heaviest per (layer, KV head), `keep` in all, equal weights lowest index first. They move
// to the front in their order, codes, scales and weights bit for bit.
//
// Two launches. select_kernel: one workgroup per (KV head, layer, row) finds the weight of the
// last token that stays by a radix select over the weights' bits (histograms of 11, 11 and 10
// bits in LDS, most significant first), then lists the tokens that stay, in order, and moves
// their weights. move_kernel: one (KV head, K or V, layer, row) per workgroup row, 16 bytes a
// lane. In place a token's destination lies at or before its source, and tokens before the
// source's: a workgroup goes through them in order, a batch of rows loaded before any of it is
// stored. Into other pages the batches are independent workgroups.
#include "attention_common.h"

namespace astr {
namespace attn {
namespace {

constexpr int kThreads = 1024, kBlockWaves = kThreads / kWave;
constexpr int kBins = 2048;

struct EvictArgs {
  astr_paged_kv cache;  // layer 0
  int64_t code_layer, scale_layer;
  float* weights;  // layer 0
  int64_t w_row, w_layer, w_head;
  const int32_t* rows;
  const int32_t* dst_rows;
  int32_t num_rows, capacity;
  const int32_t* tables;
  const int32_t* dst_tables;  // in place without
  int32_t t_stride, d_stride;
  const int32_t* context_lens;
  int32_t num_seqs, max_context, keep, sinks, recent;
  int32_t* kept;      // [num_seqs][layers][kv heads][keep], -1 behind the last
  int32_t* new_lens;  // [num_seqs]
  int32_t* err_flag;
};

// A weight's bits, ordered as the weights are (-0 as 0); NaN below every number. Never 0.
__device__ __forceinline__ uint32_t ordered(float w) {
  if (w != w) return 1u;
  const uint32_t b = __builtin_bit_cast(uint32_t, w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ int lanes_below(uint64_t mask, int lane) {
  return __builtin_popcountll(mask & ((1ull << lane) - 1));
}

// A token row's length as given, within its table, the weights' capacity and the host's bound.
__device__ __forceinline__ int evict_ctx(const EvictArgs& a, int seq, bool report) {
  const int64_t table = (int64_t)a.t_stride * kBlockTokens;
  int cap = (int)(table < a.max_context ? table : a.max_context);
  cap = min(cap, a.capacity);
  const int ctx = a.context_lens[seq];
  if (ctx < 0 || ctx > cap) {
    if (report) atomicOr(a.err_flag, ASTR_FLAG_BAD_INDEX);
    return ctx < 0 ? 0 : cap;
  }
  return ctx;
}

__device__ __forceinline__ int64_t row_of(const EvictArgs& a, const int32_t* rows, int seq, bool report) {
  const int row = rows != nullptr ? rows[seq] : seq;
  if ((unsigned)row >= (unsigned)a.num_rows) {
    if (report) atomicOr(a.err_flag, ASTR_FLAG_BAD_INDEX);
    return -1;
  }
  return row;
}

__global__ __launch_bounds__(kThreads) void select_kernel(EvictArgs a) {
  __shared__ int hist[kBins];
  __shared__ int wave_a[kBlockWaves], wave_b[kBlockWaves];
  __shared__ int found[3];
  const int head = blockIdx.x, layer = blockIdx.y, seq = blockIdx.z;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int layers = gridDim.y, heads = gridDim.x;
  const bool reporter = head == 0 && layer == 0 && threadIdx.x == 0;
  const int n = evict_ctx(a, seq, reporter);
  const int64_t src_row = row_of(a, a.rows, seq, reporter);
  const int64_t dst_row = row_of(a, a.dst_rows, seq, reporter);
  int32_t* const kept = a.kept + (((int64_t)seq * layers + layer) * heads + head) * a.keep;
  if (src_row < 0 || dst_row < 0) {  // nothing moves
    for (int i = threadIdx.x; i < a.keep; i += kThreads) kept[i] = -1;
    if (reporter) a.new_lens[seq] = 0;
    return;
  }
  const float* const w = a.weights + src_row * a.w_row + layer * a.w_layer + head * a.w_head;
  float* const w_dst = a.weights + dst_row * a.w_row + layer * a.w_layer + head * a.w_head;
  const int32_t* const table = a.tables + (int64_t)seq * a.t_stride;
  const uint8_t* const valid = a.cache.key_valid;
  auto real = [&](int t) __attribute__((always_inline)) -> bool {
    if (valid == nullptr) return true;
    const int id = table[t / kBlockTokens];
    return (unsigned)id < (unsigned)a.cache.num_blocks &&
           valid[(int64_t)id * kBlockTokens + t % kBlockTokens] != 0;
  };

  // ---- how many real tokens there are, and which ones stay for their place: those before
  // `sink_end` and from `recent_begin` on
  int count = n, sink_end = min(a.sinks, n), recent_begin = max(0, n - a.recent);
  if (valid != nullptr) {
    count = 0;
    for (int t0 = 0; t0 < n; t0 += kThreads) {
      const int t = t0 + (int)threadIdx.x;
      const uint64_t b = __ballot(t < n && real(t));
      if (lane == 0) wave_a[wave] = __builtin_popcountll(b);
      __syncthreads();
      for (int i = 0; i < kBlockWaves; ++i) count += wave_a[i];
      __syncthreads();
    }
    if (threadIdx.x == 0) {
      found[0] = a.sinks == 0 ? 0 : n;
      found[1] = a.recent == 0 ? n : 0;
    }
    int base = 0;
    for (int t0 = 0; t0 < n; t0 += kThreads) {
      const int t = t0 + (int)threadIdx.x;
      const bool is = t < n && real(t);
      const uint64_t b = __ballot(is);
      if (lane == 0) wave_a[wave] = __builtin_popcountll(b);
      __syncthreads();
      int rank = base + lanes_below(b, lane);
      for (int i = 0; i < kBlockWaves; ++i) {
        if (i < wave) rank += wave_a[i];
        base += wave_a[i];
      }
      if (is && rank + 1 == a.sinks) found[0] = t + 1;
      if (is && rank == count - a.recent) found[1] = t;
      __syncthreads();
    }
    sink_end = found[0];
    recent_begin = found[1];
    __syncthreads();
  }
  const int keep = min(a.keep, count);
  auto fixed = [&](int t) __attribute__((always_inline)) -> bool {
    return t < sink_end || t >= recent_begin;
  };

  // ---- the bits of the lightest of the heaviest: `threshold`, of which `ties` stay
  uint32_t threshold = 0;
  int ties = 0;
  if (keep < count) {
    // those of the others that stay (sinks + recent <= keep < count: the two do not overlap)
    int need = keep - a.sinks - a.recent;
    uint32_t prefix = 0, known = 0;  // bits known so far, and their mask
    threshold = 0xffffffffu;
    if (need > 0) {
      const int shifts[3] = {21, 10, 0};
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = shifts[pass], bins = pass == 2 ? 1024 : 2048;
        for (int i = threadIdx.x; i < kBins; i += kThreads) hist[i] = 0;
        __syncthreads();
        for (int t = threadIdx.x; t < n; t += kThreads) {
          if (fixed(t) || !real(t)) continue;
          const uint32_t u = ordered(w[t]);
          if ((u & known) == prefix) atomicAdd(&hist[u >> shift & (bins - 1)], 1);
        }
        __syncthreads();
        // counts from the top: thread i holds bins 2 i' and 2 i' + 1, i' = kThreads - 1 - i
        const int i2 = 2 * (kThreads - 1 - (int)threadIdx.x);
        const int hi = hist[i2 + 1], lo = hist[i2];
        int incl = hi + lo;
        for (int off = 1; off < kWave; off <<= 1) {
          const int v = __shfl_up(incl, off, kWave);
          if (lane >= off) incl += v;
        }
        if (lane == kWave - 1) wave_a[wave] = incl;
        __syncthreads();
        for (int i = 0; i < wave; ++i) incl += wave_a[i];
        const int above = incl - hi - lo;
        if (above < need && incl >= need) {  // one thread
          const bool in_hi = above + hi >= need;
          found[0] = in_hi ? i2 + 1 : i2;
          found[1] = need - (in_hi ? above : above + hi);
        }
        __syncthreads();
        prefix |= (uint32_t)found[0] << shift;
        known |= (uint32_t)(bins - 1) << shift;
        need = found[1];
        __syncthreads();
      }
      threshold = prefix;
      ties = need;
    }
  }

  // ---- the tokens that stay, in order
  int base_more = 0, base_ties = 0;
  for (int t0 = 0; t0 < n; t0 += kThreads) {
    const int t = t0 + (int)threadIdx.x;
    float weight = 0.f;
    bool more = false, tie = false;
    if (t < n && real(t)) {
      weight = w[t];
      const uint32_t u = ordered(weight);
      more = keep == count || fixed(t) || u > threshold;
      tie = !more && u == threshold;
    }
    const uint64_t bm = __ballot(more), bt = __ballot(tie);
    if (lane == 0) {
      wave_a[wave] = __builtin_popcountll(bm);
      wave_b[wave] = __builtin_popcountll(bt);
    }
    __syncthreads();
    int m = base_more + lanes_below(bm, lane), e = base_ties + lanes_below(bt, lane);
    for (int i = 0; i < kBlockWaves; ++i) {
      if (i < wave) {
        m += wave_a[i];
        e += wave_b[i];
      }
      base_more += wave_a[i];
      base_ties += wave_b[i];
    }
    if (more || (tie && e < ties)) {
      const int at = m + min(e, ties);
      if (at < keep) {  // (always, unless key_valid or the weights change under the kernel)
        kept[at] = t;
        w_dst[at] = weight;  // at <= t: in place, read by now
      }
    }
    __syncthreads();
  }
  for (int i = keep + (int)threadIdx.x; i < a.keep; i += kThreads) kept[i] = -1;
  if (reporter) a.new_lens[seq] = keep;
}

// IN_PLACE: one workgroup goes through all batches of its rows, else blockIdx.x names one.
template <int D, bool IN_PLACE>
__global__ __launch_bounds__(kThreads) void move_kernel(EvictArgs a) {
  constexpr int kLanes = D / 16, kRows = kThreads / kLanes;  // lanes a row, rows a batch
  const int heads = a.cache.num_kv_heads, layers = gridDim.y;
  const int batches = (a.keep + kRows - 1) / kRows;
  const int first = IN_PLACE ? 0 : blockIdx.x % batches;
  const int which = IN_PLACE ? blockIdx.x : blockIdx.x / batches;
  const int head = which >> 1, layer = blockIdx.y, seq = blockIdx.z;
  const bool value = which & 1;
  const int32_t* const kept = a.kept + (((int64_t)seq * layers + layer) * heads + head) * a.keep;
  const int32_t* const src_table = a.tables + (int64_t)seq * a.t_stride;
  const int32_t* const dst_table = IN_PLACE ? src_table : a.dst_tables + (int64_t)seq * a.d_stride;
  int8_t* const codes = (value ? a.cache.v_codes : a.cache.k_codes) + layer * a.code_layer +
                        head * a.cache.code_head_stride;
  float* const scales = (value ? a.cache.v_scales : a.cache.k_scales) + layer * a.scale_layer +
                        head * a.cache.scale_head_stride;
  const int row = threadIdx.x / kLanes, part = threadIdx.x % kLanes;
  const int new_len = a.new_lens[seq];
  bool bad = false;
  for (int batch = first; batch < (IN_PLACE ? batches : first + 1); ++batch) {
    const int j = batch * kRows + row;
    if (batch * kRows >= new_len) break;
    const int t = j < new_len ? kept[j] : -1;
    int src = -1, dst = -1;
    if (t >= 0) {
      src = src_table[t / kBlockTokens];
      dst = dst_table[j / kBlockTokens];
      if ((unsigned)src >= (unsigned)a.cache.num_blocks ||
          (unsigned)dst >= (unsigned)a.cache.num_blocks) {
        bad = true;
        src = -1;
      } else if (IN_PLACE && t == j) {
        src = -1;  // stays where it is
      }
    }
    uint4 v;
    float s = 0.f;
    if (src >= 0) {
      v = *reinterpret_cast<const uint4*>(codes + src * a.cache.code_block_stride +
                                          t % kBlockTokens * D + part * 16);
      if (part == 0) s = scales[src * a.cache.scale_block_stride + t % kBlockTokens];
    }
    if constexpr (IN_PLACE) {
      wait_vmcnt<0>();  // every load of the batch has returned before a store of it goes out
      __syncthreads();
    }
    if (src >= 0) {
      *reinterpret_cast<uint4*>(codes + dst * a.cache.code_block_stride + j % kBlockTokens * D +
                                part * 16) = v;
      if (part == 0) scales[dst * a.cache.scale_block_stride + j % kBlockTokens] = s;
    }
    if (a.cache.key_valid != nullptr && which == 0 && layer == 0 && part == 0 && t >= 0 &&
        (unsigned)dst < (unsigned)a.cache.num_blocks)
      a.cache.key_valid[(int64_t)dst * kBlockTokens + j % kBlockTokens] = 1;
  }
  if (bad) atomicOr(a.err_flag, ASTR_FLAG_BAD_INDEX);
}

template <int D>
void launch_move(const EvictArgs& a, int layers, hipStream_t stream) {
  constexpr int kRows = kThreads / (D / 16);
  const uint32_t units = 2u * (uint32_t)a.cache.num_kv_heads;
  if (a.dst_tables == nullptr) {
    hipLaunchKernelGGL((move_kernel<D, true>), dim3(units, layers, a.num_seqs), dim3(kThreads), 0,
                       stream, a);
  } else {
    const uint32_t batches = (uint32_t)((a.keep + kRows - 1) / kRows);
    hipLaunchKernelGGL((move_kernel<D, false>), dim3(units * batches, layers, a.num_seqs),
                       dim3(kThreads), 0, stream, a);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace attn
}  // namespace astr

extern "C" int astr_kv_evict(const astr_paged_kv* cache, int32_t num_layers,
                             int64_t code_layer_stride, int64_t scale_layer_stride,
                             const astr_key_weights* weights, int64_t weight_layer_stride,
                             const int32_t* dst_weight_rows, const int32_t* block_tables,
                             int32_t block_table_stride, const int32_t* dst_block_tables,
                             int32_t dst_block_table_stride, const int32_t* context_lens,
                             int32_t num_seqs, int32_t max_context_len, int32_t keep,
                             int32_t sinks, int32_t recent, int32_t* kept, int32_t* new_lens,
                             int32_t* err_flag, void* stream) {
  astr::CallRange range("astr_kv_evict");
  using namespace astr;
  using namespace astr::attn;
  if (cache == nullptr || weights == nullptr || err_flag == nullptr)
    return fail(ASTR_EINVAL, "cache descriptor, key weights and err_flag are required");
  if (num_seqs < 0 || num_layers < 1 || max_context_len < 0 || block_table_stride < 0 ||
      dst_block_table_stride < 0)
    return fail(ASTR_EINVAL, "num_seqs/max_context_len/strides must be >= 0 and num_layers >= 1");
  if (keep < 1 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > keep)
    return fail(ASTR_EINVAL, "keep %d must be >= 1 and hold the %d sinks and %d recent tokens", keep,
                sinks, recent);
  if (num_seqs == 0) return 0;
  if (num_seqs > 65535 || num_layers > 65535)
    return fail(ASTR_EUNSUPPORTED, "more than 65535 sequences or layers per launch");
  if (block_tables == nullptr || context_lens == nullptr || kept == nullptr || new_lens == nullptr ||
      weights->values == nullptr)
    return fail(ASTR_EINVAL, "block_tables, context_lens, kept, new_lens and weights are required");
  if (cache->block_size != kBlockTokens)
    return fail(ASTR_EUNSUPPORTED, "block_size %d != 16", cache->block_size);
  if (cache->num_blocks < 1 || cache->num_kv_heads < 1)
    return fail(ASTR_EINVAL, "cache has no blocks or no heads");
  if (weights->num_rows < 1 || weights->capacity < 0)
    return fail(ASTR_EINVAL, "key weights have no rows");
  if ((int64_t)max_context_len > (int64_t)block_table_stride * kBlockTokens)
    return fail(ASTR_EINVAL, "max_context_len %d exceeds block table capacity %lld", max_context_len,
                (long long)block_table_stride * kBlockTokens);
  if (weights->capacity < max_context_len)
    return fail(ASTR_EINVAL, "key weights of %d tokens do not hold max_context_len %d",
                weights->capacity, max_context_len);
  if (dst_block_tables != nullptr && (int64_t)dst_block_table_stride * kBlockTokens < keep &&
      (int64_t)dst_block_table_stride * kBlockTokens < max_context_len)
    return fail(ASTR_EINVAL, "destination tables hold fewer tokens than stay");
  if (!aligned16(cache->k_codes) || !aligned16(cache->v_codes) || cache->code_block_stride % 16 ||
      cache->code_head_stride % 16 || code_layer_stride % 16)
    return fail(ASTR_EINVAL, "cache code blocks must be 16-byte aligned");
  EvictArgs a{};
  a.cache = *cache;
  a.code_layer = code_layer_stride;
  a.scale_layer = scale_layer_stride;
  a.weights = weights->values;
  a.w_row = weights->row_stride;
  a.w_layer = weight_layer_stride;
  a.w_head = weights->head_stride;
  a.rows = weights->rows;
  a.dst_rows = dst_weight_rows != nullptr ? dst_weight_rows : weights->rows;
  a.num_rows = weights->num_rows;
  a.capacity = weights->capacity;
  a.tables = block_tables;
  a.dst_tables = dst_block_tables;
  a.t_stride = block_table_stride;
  a.d_stride = dst_block_table_stride;
  a.context_lens = context_lens;
  a.num_seqs = num_seqs;
  a.max_context = max_context_len;
  a.keep = keep;
  a.sinks = sinks;
  a.recent = recent;
  a.kept = kept;
  a.new_lens = new_lens;
  a.err_flag = err_flag;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int D = cache->head_dim;
  if (D != 64 && D != 128 && D != 256)
    return fail(ASTR_EUNSUPPORTED, "head_dim %d not in {64,128,256}", D);
  const int64_t batches = ((int64_t)keep * (D / 16) + kThreads - 1) / kThreads;
  if (2 * batches * cache->num_kv_heads > INT32_MAX)
    return fail(ASTR_EUNSUPPORTED, "keep %d too large for one launch", keep);
  hipLaunchKernelGGL(select_kernel, dim3(cache->num_kv_heads, num_layers, num_seqs), dim3(kThreads),
                     0, s, a);
  if (D == 64) launch_move<64>(a, num_layers, s);
  else if (D == 128) launch_move<128>(a, num_layers, s);
  else launch_move<256>(a, num_layers, s);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : hip_fail(err, "kv_evict launch");
}
