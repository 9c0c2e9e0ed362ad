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
#include <climits>

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

// What a select workgroup works on.
struct Segment {
  int n;                   // tokens
  int64_t src_row, dst_row;  // -1: nothing moves
  const float* w;
  float* w_dst;
  const int32_t* table;
  int32_t* kept;
  bool reporter;           // of the row's faults and length
  __device__ __forceinline__ explicit Segment(const EvictArgs& a) {
    const int head = blockIdx.x, layer = blockIdx.y, seq = blockIdx.z;
    reporter = head == 0 && layer == 0 && threadIdx.x == 0;
    n = evict_ctx(a, seq, reporter);
    src_row = row_of(a, a.rows, seq, reporter);
    dst_row = row_of(a, a.dst_rows, seq, reporter);
    w = a.weights + src_row * a.w_row + layer * a.w_layer + head * a.w_head;
    w_dst = a.weights + dst_row * a.w_row + layer * a.w_layer + head * a.w_head;
    table = a.tables + (int64_t)seq * a.t_stride;
    kept = a.kept + (((int64_t)seq * gridDim.y + layer) * gridDim.x + head) * a.keep;
  }
  __device__ __forceinline__ bool real(const EvictArgs& a, int t) const {
    const int id = table[t / kBlockTokens];
    return (unsigned)id < (unsigned)a.cache.num_blocks &&
           a.cache.key_valid[(int64_t)id * kBlockTokens + t % kBlockTokens] != 0;
  }
  // Ends a segment of which `keep` tokens stay.
  template <int T>
  __device__ __forceinline__ void finish(const EvictArgs& a, int keep) const {
    for (int i = keep + (int)threadIdx.x; i < a.keep; i += T) kept[i] = -1;
    if (reporter) a.new_lens[blockIdx.z] = keep;
  }
};

// One pass of the radix select by T threads: hist holds the counts of the digit's values; finds
// the value of the `need`-th largest and how many of that value are among the `need`: found[0],
// found[1]. Every thread calls it, after a barrier.
template <int T>
__device__ __forceinline__ void find_digit(const int* hist, int need, int* wave_sum, int* found) {
  constexpr int kPer = kBins / T;  // consecutive bins a thread holds, from the top down
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int bin0 = kPer * (T - 1 - (int)threadIdx.x);
  int c[kPer], incl = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    c[i] = hist[bin0 + i];
    incl += c[i];
  }
  int above = -incl;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int v = __shfl_up(incl, off, kWave);
    if (lane >= off) incl += v;
  }
  if (lane == kWave - 1) wave_sum[wave] = incl;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < T / kWave; ++i) incl += i < wave ? wave_sum[i] : 0;
  above += incl;
  if (above < need && incl >= need) {  // one thread
    int bin = bin0 + kPer - 1;
#pragma unroll
    for (int i = kPer - 1; i > 0; --i)
      if (bin == bin0 + i && above + c[i] < need) {
        above += c[i];
        --bin;
      }
    found[0] = bin;
    found[1] = need - above;
  }
  __syncthreads();
}

// Segments of up to R * T tokens: thread i holds the bits of tokens i, i + T, ... in registers,
// read once; order comes from one prefix over the counts of all (round, wave) pairs.
// Bound by the chain of barriers and LDS round trips of a segment and by its registers, of which
// R a thread: the fewer threads, the cheaper a barrier, the fewer tokens a thread, the more
// segments a CU holds. 8 prompts of 1500 to 9000 tokens, 16 layers, 8 heads: 40 us with 512 threads
// (47 with 256, 57 with 1024; 58 with loads behind a branch per lane, 72 when every pass read the
// weights again); the same prompts at 2200 to 4000 tokens: 22 us with 256 threads, 23 with 512.
template <int T, int R>
__global__ __launch_bounds__(T) void select_held_kernel(EvictArgs a) {
  constexpr int kWavesT = T / kWave, kPairs = R * kWavesT;
  __shared__ __attribute__((aligned(16))) int hist[kBins];
  __shared__ int count_a[kPairs], count_b[kPairs];
  __shared__ int wave_sum[kWavesT], found[2], total;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const Segment g(a);
  if (g.src_row < 0 || g.dst_row < 0) return g.finish<T>(a, 0);
  const int n = g.n, pairs = (n + T - 1) / T * kWavesT;

  // The exclusive prefix of counts[round * kWavesT + wave] in place, by one wave; the sum in
  // `total` where asked.
  auto scan = [&](int* counts, int by, bool sum) __attribute__((always_inline)) {
    if (wave != by) return;
    int base = 0;
    for (int c0 = 0; c0 < pairs; c0 += kWave) {
      const int v = c0 + lane < pairs ? counts[c0 + lane] : 0;
      int incl = v;
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) {
        const int u = __shfl_up(incl, off, kWave);
        if (lane >= off) incl += u;
      }
      if (c0 + lane < pairs) counts[c0 + lane] = base + incl - v;
      base += __shfl(incl, kWave - 1, kWave);
    }
    if (sum && lane == 0) total = base;
  };

  // Loads go out kBatch at a time, of clamped tokens and without a branch per lane: behind one,
  // each waits for the load before it.
  constexpr int kBatch = 8;
  static_assert(R % kBatch == 0, "");
  auto token = [&](int i) __attribute__((always_inline)) -> int { return min(i * T + (int)threadIdx.x, n - 1); };
  uint32_t u[R];  // 0: no token, or a padding one
#pragma unroll
  for (int b = 0; b < R; b += kBatch) {
    if (b * T < n) {  // (uniform, as every such test below)
      float w[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) w[i] = g.w[token(b + i)];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) u[b + i] = (b + i) * T + (int)threadIdx.x < n ? ordered(w[i]) : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) u[b + i] = 0;
    }
  }
  uint64_t fixed = 0;  // bit i: token i stays for its place
  int count = n;
  if (a.cache.key_valid != nullptr) {
#pragma unroll
    for (int b = 0; b < R; b += kBatch) {
      if (b * T < n) {
        int id[kBatch];
        uint8_t valid[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) id[i] = g.table[token(b + i) / kBlockTokens];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const bool in = (unsigned)id[i] < (unsigned)a.cache.num_blocks;
          valid[i] = a.cache.key_valid[in ? (int64_t)id[i] * kBlockTokens + token(b + i) % kBlockTokens : 0];
          valid[i] = in ? valid[i] : 0;
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          u[b + i] = valid[i] != 0 ? u[b + i] : 0u;
          const uint64_t m = __ballot(u[b + i] != 0);
          if (lane == 0 && (b + i) * T < n) count_a[(b + i) * kWavesT + wave] = __builtin_popcountll(m);
        }
      }
    }
    __syncthreads();
    scan(count_a, 0, true);
    __syncthreads();
    count = total;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i * T < n) {
        const uint64_t b = __ballot(u[i] != 0);
        const int rank = count_a[i * kWavesT + wave] + lanes_below(b, lane);
        fixed |= (uint64_t)(u[i] != 0 && (rank < a.sinks || rank >= count - a.recent)) << i;
      }
    }
    __syncthreads();  // count_a is written again
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int t = i * T + (int)threadIdx.x;
      fixed |= (uint64_t)(t < n && (t < a.sinks || t >= n - a.recent)) << i;
    }
  }
  const int keep = min(a.keep, count);

  // ---- the bits of the lightest of the heaviest, of which `ties` stay
  uint32_t threshold = 0;
  int ties = 0;
  if (keep < count) {
    // those of the others that stay (sinks + recent <= keep < count: the two do not overlap)
    int need = keep - a.sinks - a.recent;
    threshold = 0xffffffffu;
    if (need > 0) {
      uint32_t prefix = 0, known = 0;
#pragma unroll 1
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
#pragma unroll
        for (int i = 0; i < kBins / T / 4 + (kBins / T < 4); ++i)
          if ((i * T + (int)threadIdx.x) * 4 < kBins)
            *reinterpret_cast<int4_t*>(hist + (i * T + (int)threadIdx.x) * 4) = int4_t{0, 0, 0, 0};
        __syncthreads();
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (u[i] != 0 && !(fixed >> i & 1) && (u[i] & known) == prefix)
            atomicAdd(&hist[u[i] >> shift & (bins - 1)], 1);
        __syncthreads();
        find_digit<T>(hist, need, wave_sum, found);
        prefix |= (uint32_t)found[0] << shift;
        known |= (uint32_t)(bins - 1) << shift;
        need = found[1];
      }
      threshold = prefix;
      ties = need;
    }
  }

  // ---- the tokens that stay, in order
  const bool all = keep == count;
  auto more_of = [&](int i) __attribute__((always_inline)) -> bool {
    return u[i] != 0 && (all || (fixed >> i & 1) || u[i] > threshold);
  };
  auto tie_of = [&](int i) __attribute__((always_inline)) -> bool {
    return u[i] == threshold && !more_of(i) && u[i] != 0;
  };
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i * T < n) {
      const uint64_t bm = __ballot(more_of(i)), bt = __ballot(tie_of(i));
      if (lane == 0) {
        count_a[i * kWavesT + wave] = __builtin_popcountll(bm);
        count_b[i * kWavesT + wave] = __builtin_popcountll(bt);
      }
    }
  }
  __syncthreads();
  scan(count_a, 0, false);
  scan(count_b, 1, false);
  __syncthreads();
  // in place, a weight's destination may be another thread's source: all are read before any is
  // stored (u becomes the weight's own bits)
  int at[R];
#pragma unroll
  for (int b = 0; b < R; b += kBatch) {
    if (b * T < n) {
      float w[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) w[i] = g.w[token(b + i)];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const bool more = more_of(b + i), tie = tie_of(b + i);
        const uint64_t bm = __ballot(more), bt = __ballot(tie);
        const int pair = min((b + i) * kWavesT + wave, pairs - 1);  // (behind the pairs nothing stays)
        const int m = count_a[pair] + lanes_below(bm, lane);
        const int e = count_b[pair] + lanes_below(bt, lane);
        at[b + i] = more || (tie && e < ties) ? m + min(e, ties) : INT_MAX;
        u[b + i] = __builtin_bit_cast(uint32_t, w[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) at[b + i] = INT_MAX;
    }
  }
  wait_vmcnt<0>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (at[i] < keep) {  // (and so below a.keep)
      g.kept[at[i]] = i * T + (int)threadIdx.x;
      g.w_dst[at[i]] = __builtin_bit_cast(float, u[i]);
    }
  }
  g.finish<T>(a, keep);
}

// Segments of any length: every pass reads the weights again.
__global__ __launch_bounds__(kThreads) void select_kernel(EvictArgs a) {
  __shared__ int hist[kBins];
  __shared__ int wave_a[kBlockWaves], wave_b[kBlockWaves];
  __shared__ int found[2];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const Segment g(a);
  if (g.src_row < 0 || g.dst_row < 0) return g.finish<kThreads>(a, 0);
  const int n = g.n;
  const float* const w = g.w;
  const bool masks = a.cache.key_valid != nullptr;
  auto real = [&](int t) __attribute__((always_inline)) -> bool { return !masks || g.real(a, t); };

  // ---- how many real tokens there are, and which ones stay for their place: those before
  // `sink_end` and from `recent_begin` on
  int count = n, sink_end = min(a.sinks, n), recent_begin = max(0, n - a.recent);
  if (masks) {
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
        find_digit<kThreads>(hist, need, wave_a, found);
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
        g.kept[at] = t;
        g.w_dst[at] = weight;  // at <= t: in place, read by now
      }
    }
    __syncthreads();
  }
  g.finish<kThreads>(a, keep);
}

// Rows of a batch: kMoveDepth a thread, whose three loads in a row (the token, its pages, its
// bytes) are on their way together.
constexpr int kMoveDepth = 4;
template <int D>
constexpr int move_rows() { return kMoveDepth * kThreads / (D / 16); }

// IN_PLACE: one workgroup goes through all batches of its rows, else blockIdx.x names one.
template <int D, bool IN_PLACE>
__global__ __launch_bounds__(kThreads) void move_kernel(EvictArgs a) {
  constexpr int kLanes = D / 16;           // a row's
  constexpr int kRows = move_rows<D>(), kStep = kThreads / kLanes;
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
    if (batch * kRows >= new_len) break;
    int t[kMoveDepth], src[kMoveDepth], dst[kMoveDepth];
    typedef uint32_t word4_t __attribute__((ext_vector_type(4)));
    word4_t v[kMoveDepth];
    float s[kMoveDepth];
#pragma unroll
    for (int i = 0; i < kMoveDepth; ++i) {
      const int j = batch * kRows + i * kStep + row;
      t[i] = j < new_len ? kept[j] : -1;
    }
#pragma unroll
    for (int i = 0; i < kMoveDepth; ++i) {
      const int j = batch * kRows + i * kStep + row;
      src[i] = dst[i] = -1;
      v[i] = word4_t{0, 0, 0, 0};
      s[i] = 0.f;
      if (t[i] >= 0) {
        src[i] = src_table[t[i] / kBlockTokens];
        dst[i] = dst_table[j / kBlockTokens];
      }
    }
#pragma unroll
    for (int i = 0; i < kMoveDepth; ++i) {
      const int j = batch * kRows + i * kStep + row;
      if (t[i] >= 0 && ((unsigned)src[i] >= (unsigned)a.cache.num_blocks ||
                        (unsigned)dst[i] >= (unsigned)a.cache.num_blocks)) {
        bad = true;
        src[i] = -1;
      }
      if (IN_PLACE && t[i] == j) src[i] = -1;  // stays where it is
      if (src[i] >= 0) {
        v[i] = *reinterpret_cast<const word4_t*>(codes + src[i] * a.cache.code_block_stride +
                                               t[i] % kBlockTokens * D + part * 16);
        if (part == 0) s[i] = scales[src[i] * a.cache.scale_block_stride + t[i] % kBlockTokens];
      }
    }
    if constexpr (IN_PLACE) {
      wait_vmcnt<0>();  // every load of the batch has returned before a store of it goes out
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kMoveDepth; ++i) {
      const int j = batch * kRows + i * kStep + row;
      if (src[i] >= 0) {
        *reinterpret_cast<word4_t*>(codes + dst[i] * a.cache.code_block_stride +
                                  j % kBlockTokens * D + part * 16) = v[i];
        if (part == 0) scales[dst[i] * a.cache.scale_block_stride + j % kBlockTokens] = s[i];
      }
      if (a.cache.key_valid != nullptr && which == 0 && layer == 0 && part == 0 && t[i] >= 0 &&
          (unsigned)dst[i] < (unsigned)a.cache.num_blocks)
        a.cache.key_valid[(int64_t)dst[i] * kBlockTokens + j % kBlockTokens] = 1;
    }
  }
  if (bad) atomicOr(a.err_flag, ASTR_FLAG_BAD_INDEX);
}

template <int D>
void launch_move(const EvictArgs& a, int layers, hipStream_t stream) {
  constexpr int kRows = move_rows<D>();
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
  const dim3 segments(cache->num_kv_heads, num_layers, num_seqs);
  if (max_context_len <= 8 * 256)
    hipLaunchKernelGGL((select_held_kernel<256, 8>), segments, dim3(256), 0, s, a);
  else if (max_context_len <= 16 * 256)
    hipLaunchKernelGGL((select_held_kernel<256, 16>), segments, dim3(256), 0, s, a);
  else if (max_context_len <= 24 * 512)
    hipLaunchKernelGGL((select_held_kernel<512, 24>), segments, dim3(512), 0, s, a);
  else if (max_context_len <= 32 * kThreads)
    hipLaunchKernelGGL((select_held_kernel<kThreads, 32>), segments, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL(select_kernel, segments, dim3(kThreads), 0, s, a);
  if (D == 64) launch_move<64>(a, num_layers, s);
  else if (D == 128) launch_move<128>(a, num_layers, s);
  else launch_move<256>(a, num_layers, s);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : hip_fail(err, "kv_evict launch");
}
