// Key weights of prompt chunks over the paged cache (gfx950): for the rows of a step with
// two or more query tokens, each key's softmax weight summed over the row's queries that see
// it (k <= p) and the heads of its group,
//   A[k] += sum_{p >= k} sum_g exp(s_pgk - lse_pg),   lse_pg = log sum_{k <= p} exp(s_pgk).
//
// Two passes over the scores, which are formed twice (2 D operations each, cheaper than 4
// bytes written and read per score): the first keeps 32 (token, head) columns per wave and
// streams the keys (64 per step, converted once to f16 operands in LDS for the workgroup's
// 128 columns) under a running maximum and sum; the second keeps 64 keys per wave and streams
// the columns, whose f16 operands, factor and lse the first left in the workspace in the
// order the second's lanes read them. In both, v_mfma_f32_32x32x16_f16 gives lane (c, h) the
// scores of column c and keys 8 x + 4 h + y (element 4 x + y), so that the first pass reduces
// over keys, and the second over columns until its end, without crossing lanes. Sums in fp32,
// in an order that depends on the sizes alone.
//
// Scores: K codes exact in f16 against one f16 term of a 16-bit query (exact, scaled by a
// power of two per column) or two of an fp32 one (22 bits), fp32 accumulation.
#include <climits>

#include "bounded_common.h"

namespace astr {
namespace attn {
namespace {

#ifndef ASTR_KF
#define ASTR_KF 0
#endif
constexpr int KF = ASTR_KF;  // this translation unit's code format

typedef float float16v_t __attribute__((ext_vector_type(16)));
typedef float float2_t __attribute__((ext_vector_type(2)));

constexpr int kStepKeys = kWaves * kBlockTokens;

// The f16 operand of one 32-column tile: lane (c, h) holds column c's d = 16 cc + 8 h + [0, 8).
template <typename QT, int D>
struct ColumnOp {
  static constexpr int kTerms = sizeof(QT) == 4 ? 2 : 1;
  static constexpr int kChunks = D / 16;
  half8_t op[kTerms][kChunks];
};

// Workspace places of column tile `tile` of a (sequence, KV head): the tiles of sequence s
// begin at q0 * G / 32 + s, of `tiles` per KV head.
struct ColumnPlace {
  int64_t tile0;
  __device__ ColumnPlace(const BoundedArgs& a, int seq, int kvh, int q0)
      : tile0((int64_t)kvh * tiles(a) + (int64_t)q0 * a.group / 32 + seq) {}
  __host__ __device__ static int64_t tiles(const BoundedArgs& a) {
    return (int64_t)a.num_q_tokens * a.group / 32 + a.num_seqs;
  }
};

// The workspace: per column {factor, lse}, per piece and column {m, l}, the operands, and the
// column pieces' sums, one row of score_stride keys per (sequence, KV head) and piece.
struct ChunkWs {
  float2_t* cols;
  float2_t* ml;
  half8_t* ops;
  float* sums;
  int64_t columns;
  __host__ __device__ ChunkWs(const BoundedArgs& a, int op_halves) {
    columns = ColumnPlace::tiles(a) * a.cache.num_kv_heads * 32;
    cols = reinterpret_cast<float2_t*>(a.chunk_ws);
    ml = cols + columns;
    ops = reinterpret_cast<half8_t*>(ml + a.chunk_pieces * columns);
    sums = reinterpret_cast<float*>(ops + columns * (op_halves / 8));
  }
};
template <typename QT, int D>
__host__ __device__ ChunkWs chunk_ws(const BoundedArgs& a) {
  return ChunkWs(a, ColumnOp<QT, D>::kTerms * D);
}

struct ChunkRow {
  int q0, n, ctx, pos0;
};
// The row's queries and length; n = 0 where it is not a chunk. (The attention launch of the same
// call reports what is out of range.)
__device__ __forceinline__ ChunkRow chunk_row(const BoundedArgs& a, int seq) {
  ChunkRow r;
  r.n = seq_queries(a, seq, r.q0);
  r.ctx = bounded_ctx(a, a.context_lens[seq], false);
  if (r.n < a.min_rows || r.ctx < r.n) r.n = 0;
  r.pos0 = r.ctx - r.n;
  return r;
}

__device__ __forceinline__ float log_sum(float m, float l) {
  return l > 0.f ? m + __builtin_amdgcn_logf(l) : INFINITY;
}

// The workgroup's piece and tile. Workgroups are dealt to the 8 XCDs in turn, and under the causal
// mask a piece's or a tile's number says how much of it there is: pieces side by side left some
// XCDs little to do (2000 tokens, first pass: 67 us, 51 with them apart), and so does a number
// of tiles that 8 divides, against which each piece's tiles begin one later.
__device__ __forceinline__ void unit_of(int pieces, int& piece, int& tile) {
  const int tiles = gridDim.x / pieces;
  piece = blockIdx.x / tiles;
  tile = (blockIdx.x % tiles + piece) % tiles;
}

template <int D>
struct StatsLds {
  uint4 k[2][2 * (D / 16) * kWave];
  __attribute__((aligned(16))) float ks[2][kStepKeys];
  __attribute__((aligned(16))) uint32_t pad[2][kStepKeys / 4];
};

template <typename QT, int D>
__global__ __launch_bounds__(256, 2) void chunk_stats_kernel(BoundedArgs a) {
  using Op = ColumnOp<QT, D>;
  __shared__ StatsLds<D> L;
  // the latest tokens, which see the most keys, first
  int piece, ctile;
  unit_of(a.chunk_pieces, piece, ctile);
  ctile = (int)(gridDim.x / a.chunk_pieces) - 1 - ctile;
  const int kvh = blockIdx.y, seq = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int G = a.group;
  const ChunkRow row = chunk_row(a, seq);
  const int f0 = ctile * 128;
  if (f0 >= row.n * G) return;
  const int gs = __builtin_ctz(G);  // (a power of two)
  // the keys that the workgroup's last column sees, its piece of them
  const int last_tok = min(row.n - 1, (f0 + 127) >> gs);
  const int blocks = (row.pos0 + last_tok) / kBlockTokens + 1;
  const int b0 = piece * a.chunk_steps * kWaves;
  const int b1 = min(blocks, b0 + a.chunk_steps * kWaves);
  const int nsteps = b1 > b0 ? (b1 - b0 + kWaves - 1) / kWaves : 0;

  const ChunkWs ws = chunk_ws<QT, D>(a);
  const int64_t tile = ColumnPlace(a, seq, kvh, row.q0).tile0 + ctile * 4 + wave;
  const bool used = f0 + wave * 32 < row.n * G;  // the wave's tile has a place
  if (nsteps == 0 && piece > 0) {  // past the keys that the workgroup's columns see
    if (used && lane < 32) ws.ml[piece * ws.columns + tile * 32 + lane] = float2_t{-FLT_MAX, 0.f};
    return;
  }

  // ---- the wave's columns: rows read whole (lane `part` of D / 8 takes eight elements), their
  // f16 terms through LDS into the operand's order, and into the workspace. (Read by operand
  // lanes, 16 bytes of 64 rows at a time, the rows of a CU's 16 waves did not stay in its cache:
  // 15 us before the first step of a 2000-token prompt.)
  const int h = lane >> 5;
  const int f = f0 + wave * 32 + (lane & 31);
  const bool valid = f < row.n * G;
  const int pos = row.pos0 + (valid ? f >> gs : last_tok);
  Op q;
  float factor;
  {
    constexpr int kLanes = D / 8, kRows = kWave / kLanes, kLoads = 32 / kRows;
    static_assert(kWaves * Op::kChunks * kWave * 16 <= sizeof(L.k), "a term's operands fit the buffers");
    static_assert(kWaves * 32 * sizeof(float) <= sizeof(L.ks), "the factors fit theirs");
    struct alignas(8 * sizeof(QT) > 16 ? 16 : 8 * sizeof(QT)) Run {
      QT e[8];
    };
    const int part = lane % kLanes, sub = lane / kLanes;
    half8_t* const terms = reinterpret_cast<half8_t*>(L.k) + wave * Op::kChunks * kWave;
    float* const factors = reinterpret_cast<float*>(L.ks) + wave * 32;
    constexpr int kBatch = kLoads < 8 ? kLoads : 8;  // rows on their way together
#pragma unroll
    for (int t = 0; t < Op::kTerms; ++t) {  // (fp32 queries read their rows for each term)
#pragma unroll
      for (int i0 = 0; i0 < kLoads; i0 += kBatch) {
        Run run[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int fi = min(f0 + wave * 32 + (i0 + i) * kRows + sub, row.n * G - 1);
          run[i] = *reinterpret_cast<const Run*>(static_cast<const QT*>(a.q) +
                                                 (int64_t)(row.q0 + (fi >> gs)) * a.q_tok +
                                                 (int64_t)(kvh * G + (fi & (G - 1))) * a.q_head + 8 * part);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int c = (i0 + i) * kRows + sub;
          float x[8], mx = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = to_float<QT>(run[i].e[e]);
            mx = vmax(mx, fabsf(x[e]));  // NaN-propagating
          }
#pragma unroll
          for (int b = 1; b < kLanes; b <<= 1) mx = vmax(mx, shfl_xor(mx, b));
          // a column that is not finite enters as zeros, of no weight: its lse comes out infinite
          const bool finite = __builtin_isfinite(mx);
          int ex = 15;
          if (finite && mx > 0.f) frexpf(mx, &ex);
          ex = max(ex - 15, -126);
          const float down = finite && f0 + wave * 32 + c < row.n * G ? ldexpf(1.f, -ex) : 0.f;
          half8_t term;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float v = down == 0.f ? 0.f : x[e] * down;  // exact
            if constexpr (Op::kTerms == 2) asm volatile("" : "+v"(v));  // one value for both terms
            const _Float16 hi = (_Float16)v;
            term[e] = t == 0 ? hi : (_Float16)(v - (float)hi);
          }
          terms[(part / 2) * kWave + 32 * (part % 2) + c] = term;
          if (part == 0)
            factors[c] = finite ? ldexpf(1.f, ex) * a.qk_scale_log2 * code_scale<KF>() : __builtin_nanf("");
        }
      }
      __builtin_amdgcn_wave_barrier();  // a wave's LDS accesses complete in order
#pragma unroll
      for (int cc = 0; cc < Op::kChunks; ++cc) q.op[t][cc] = terms[cc * kWave + lane];
      factor = valid ? factors[lane & 31] : 0.f;
      __builtin_amdgcn_wave_barrier();
    }
  }
  if (piece == 0 && used) {
#pragma unroll
    for (int t = 0; t < Op::kTerms; ++t)
#pragma unroll
      for (int cc = 0; cc < Op::kChunks; ++cc)
        ws.ops[((tile * Op::kTerms + t) * Op::kChunks + cc) * kWave + lane] = q.op[t][cc];
  }
  __syncthreads();  // the buffers are the keys' from here on

  // ---- the keys
  const int32_t* bt = a.block_tables + (int64_t)seq * a.bt_stride;
  const bool masks = a.cache.key_valid != nullptr;
  uint4 rk[D / 64];
  float rks = 0.f;
  uint32_t rpad = 0x01010101u;
  auto load_step = [&](int i) __attribute__((always_inline)) {
    int id = bt[min(b0 + i * kWaves + wave, b1 - 1)];
    if ((unsigned)id >= (unsigned)a.cache.num_blocks) id = 0;
    const int8_t* kp = a.cache.k_codes + id * a.cache.code_block_stride +
                       kvh * a.cache.code_head_stride + (lane & 15) * D + (lane >> 4) * 16;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) rk[c] = *reinterpret_cast<const uint4*>(kp + 64 * c);
    rks = a.cache.k_scales[id * a.cache.scale_block_stride + kvh * a.cache.scale_head_stride +
                           (lane & 15)];
    if (masks)
      rpad = *reinterpret_cast<const uint32_t*>(a.cache.key_valid + (int64_t)id * kBlockTokens +
                                                4 * (lane & 3));
  };
  auto convert = [&](int buf) __attribute__((always_inline)) {
    uint4* kd = L.k[buf] + (wave / 2) * Op::kChunks * kWave + 16 * (wave % 2) + (lane & 15);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      uint4* e = kd + (4 * c + (lane >> 4)) * kWave;
      half2_t p[8];
      codes_to_f16<KF>(rk[c].x, p[0], p[1]);
      codes_to_f16<KF>(rk[c].y, p[2], p[3]);
      codes_to_f16<KF>(rk[c].z, p[4], p[5]);
      codes_to_f16<KF>(rk[c].w, p[6], p[7]);
      auto word = [&](int j) { return __builtin_bit_cast(uint32_t, p[j]); };
      e[0] = uint4{word(0), word(1), word(2), word(3)};
      e[32] = uint4{word(4), word(5), word(6), word(7)};
    }
    if (lane < 16) L.ks[buf][16 * wave + lane] = rks;
    if (lane < 4) L.pad[buf][4 * wave + lane] = rpad;
  };

  float m = -FLT_MAX, l = 0.f;
  if (nsteps > 0) {
    load_step(0);
    convert(0);
    if (nsteps > 1) load_step(1);
  }
  __syncthreads();
  // every column of the wave sees the keys below `inner`
  const int inner = row.pos0 + min(row.n - 1, (f0 + wave * 32) >> gs) + 1;
  for (int i = 0; i < nsteps; ++i) {
    const int buf = i & 1;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int kb = (b0 + i * kWaves) * kBlockTokens + 32 * kt;
      float16v_t s;
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = 0.f;
      const uint4* kp = L.k[buf] + kt * Op::kChunks * kWave + lane;
#pragma unroll
      for (int cc = 0; cc < Op::kChunks; ++cc) {
        const half8_t kop = __builtin_bit_cast(half8_t, kp[cc * kWave]);
#pragma unroll
        for (int t = 0; t < Op::kTerms; ++t)
          s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kop, q.op[t][cc], s, 0, 0, 0);
      }
      bool padded = false;
      if (masks) {
        const uint4 pw = *reinterpret_cast<const uint4*>(&L.pad[buf][8 * kt + 4 * (lane & 1)]);
        padded = __ballot(pw.x != 0x01010101u || pw.y != 0x01010101u || pw.z != 0x01010101u ||
                          pw.w != 0x01010101u) != 0;
      }
      float4_t ks[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        ks[x] = *reinterpret_cast<const float4_t*>(&L.ks[buf][32 * kt + 8 * x + 4 * h]) * factor;
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] *= ks[j / 4][j % 4];
      if (kb + 32 > inner || kb + 32 > b1 * kBlockTokens || padded) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t pad = L.pad[buf][8 * kt + 2 * x + h];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int key = kb + 8 * x + 4 * h + y;
            const bool seen = key <= pos && key < b1 * kBlockTokens && (pad >> (8 * y) & 0xffu) != 0;
            s[4 * x + y] = seen ? s[4 * x + y] : -INFINITY;
          }
        }
      }
      float mu = s[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) mu = fmaxf(mu, s[j]);
      if (__ballot(mu > m + kRescaleSlack) != 0) {
        const float mn = fmaxf(m, mu);
        l *= __builtin_amdgcn_exp2f(m - mn);
        m = mn;
      }
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) part += __builtin_amdgcn_exp2f(s[j] - m);
      l += part;
    }
    if (i + 1 < nsteps) {
      convert(buf ^ 1);
      if (i + 2 < nsteps) load_step(i + 2);
    }
    __syncthreads();
  }
  const float mo = shfl_xor(m, 32), lo = shfl_xor(l, 32);
  const float mm = fmaxf(m, mo);
  const float ll = l * __builtin_amdgcn_exp2f(m - mm) + lo * __builtin_amdgcn_exp2f(mo - mm);
  const float kept_factor = __builtin_isfinite(factor) ? factor : 0.f;
  if (used && lane < 32) {
    const int64_t at = tile * 32 + lane;
    if (a.chunk_pieces == 1) {
      ws.cols[at] = float2_t{kept_factor, valid ? log_sum(mm, ll) : INFINITY};
    } else {
      if (piece == 0) ws.cols[at][0] = kept_factor;
      ws.ml[piece * ws.columns + at] = float2_t{mm, valid ? ll : 0.f};
    }
  }
}

// The pieces' states joined (a piece past a column's keys left l = 0).
__global__ __launch_bounds__(256) void chunk_lse_kernel(BoundedArgs a) {
  const ChunkWs ws(a, 0);
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= ws.columns) return;
  float m = -FLT_MAX;
  for (int p = 0; p < a.chunk_pieces; ++p) m = fmaxf(m, ws.ml[p * ws.columns + at][0]);
  float l = 0.f;
  for (int p = 0; p < a.chunk_pieces; ++p) {
    const float2_t s = ws.ml[p * ws.columns + at];
    l = fmaf(s[1], __builtin_amdgcn_exp2f(s[0] - m), l);
  }
  ws.cols[at][1] = log_sum(m, l);
}

// The first column tile with a token that sees key k0.
__device__ __forceinline__ int column_first(const ChunkRow& row, int k0, int group) {
  return max(0, k0 - row.pos0) * group / 32;
}

// Adds what a key gathered.
__device__ __forceinline__ void add_key(const BoundedArgs& a, const ChunkRow& row, const int32_t* bt,
                                        int64_t wrow, int kvh, int key, float v) {
  if (key >= a.kw.capacity) return;
  if (a.cache.key_valid != nullptr) {
    const int id = bt[key / kBlockTokens];
    if ((unsigned)id < (unsigned)a.cache.num_blocks &&
        a.cache.key_valid[(int64_t)id * kBlockTokens + key % kBlockTokens] == 0)
      v = 0.f;  // a padding key
  }
  v = __builtin_isfinite(v) ? v : 0.f;  // a key whose own scale is not finite
  float* w = a.kw.values + wrow * a.kw.row_stride + kvh * a.kw.head_stride + key;
  *w = (key >= row.pos0 ? 0.f : *w) + v;
}

// Keys of one wave: 64 in two tiles, 32 at head dim 256 (the operands fill the registers). The
// workgroup's waves take consecutive keys and go through the same columns.
template <int D>
constexpr int column_sum_keys() { return D == 256 ? 32 : 64; }

template <typename QT, int D>
__global__ __launch_bounds__(256, 2) void column_sum_kernel(BoundedArgs a) {
  using Op = ColumnOp<QT, D>;
  constexpr int KT = column_sum_keys<D>(), NT = KT / 32;
  const int kvh = blockIdx.y, seq = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int h = lane >> 5;
  const int G = a.group, gs = __builtin_ctz(G);
  const ChunkRow row = chunk_row(a, seq);
  int piece, ktile;
  unit_of(a.column_pieces, piece, ktile);
  piece = a.column_pieces - 1 - piece;  // (every key is seen by the last)
  const int k0 = (ktile * kWaves + wave) * KT;
  if (row.n == 0 || k0 >= row.ctx) return;
  // the column tiles from the first token that sees key k0 on, the workgroup's piece of them
  const int first = max(column_first(row, k0, G), piece * a.column_tiles);
  const int tiles = min((row.n * G + 31) / 32,
                        piece == a.column_pieces - 1 ? INT_MAX : (piece + 1) * a.column_tiles);
  if (first >= tiles) return;
  const int64_t wrow = weight_row(a, seq, false);
  if (wrow < 0) return;

  // ---- the wave's keys, as operands in its registers: lane (key, h)
  const int32_t* bt = a.block_tables + (int64_t)seq * a.bt_stride;
  const int last_blk = (row.ctx - 1) / kBlockTokens;
  half8_t kop[NT][Op::kChunks];
  float4_t ks[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int key = k0 + 32 * t + (lane & 31);
    int id = bt[min(key / kBlockTokens, last_blk)];
    if ((unsigned)id >= (unsigned)a.cache.num_blocks) id = 0;
    const int8_t* kp = a.cache.k_codes + id * a.cache.code_block_stride +
                       kvh * a.cache.code_head_stride + (key % kBlockTokens) * D + 8 * h;
#pragma unroll
    for (int cc = 0; cc < Op::kChunks; ++cc) {
      const uint2 w = *reinterpret_cast<const uint2*>(kp + 16 * cc);
      half2_t p0, p1, p2, p3;
      codes_to_f16<KF>(w.x, p0, p1);
      codes_to_f16<KF>(w.y, p2, p3);
      kop[t][cc] = half8_t{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
    }
    // the factors of keys 8 x + 4 h + [0, 4)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int kx = k0 + 32 * t + 8 * x + 4 * h;
      int ix = bt[min(kx / kBlockTokens, last_blk)];
      if ((unsigned)ix >= (unsigned)a.cache.num_blocks) ix = 0;
      ks[t][x] = *reinterpret_cast<const float4_t*>(
          a.cache.k_scales + ix * a.cache.scale_block_stride + kvh * a.cache.scale_head_stride +
          kx % kBlockTokens);
    }
  }

  // ---- the columns
  const ChunkWs ws = chunk_ws<QT, D>(a);
  const int64_t tile0 = ColumnPlace(a, seq, kvh, row.q0).tile0;
  float sum[NT][16];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) sum[t][j] = 0.f;
  half8_t q[Op::kChunks];  // (a second term is read when the first has been used)
  float2_t col = {0.f, INFINITY};
  auto load_term = [&](int c, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int cc = 0; cc < Op::kChunks; ++cc)
      q[cc] = ws.ops[(((tile0 + c) * Op::kTerms + t) * Op::kChunks + cc) * kWave + lane];
  };
  auto load = [&](int c) __attribute__((always_inline)) {
    load_term(c, 0);
    col = ws.cols[(tile0 + c) * 32 + (lane & 31)];
  };
  load(first);
  for (int c = first; c < tiles; ++c) {
    float16v_t s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 16; ++j) s[t][j] = 0.f;
#pragma unroll
    for (int x = 0; x < Op::kTerms; ++x) {
      if (x > 0) load_term(c, x);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int cc = 0; cc < Op::kChunks; ++cc)
          s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kop[t][cc], q[cc], s[t], 0, 0, 0);
    }
    const float factor = col[0], lse = col[1];
    const int pos = row.pos0 + min(row.n - 1, (c * 32 + (lane & 31)) >> gs);
    if (c + 1 < tiles) load(c + 1);
    if (row.pos0 + (c * 32 >> gs) < k0 + KT - 1) {  // some column does not see some key
      asm volatile("");  // keeps this a branch: if-converted, the other tiles would pay for it
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int32_t before = pos - (k0 + 32 * t + 8 * (j / 4) + 4 * h + j % 4);  // < 0: not seen
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][j] * ks[t][j / 4][j % 4], factor, -lse));
          sum[t][j] += __builtin_bit_cast(float, __builtin_bit_cast(int32_t, p) & ~(before >> 31));
        }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sum[t][j] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][j] * ks[t][j / 4][j % 4], factor, -lse));
    }
  }
  // ---- over the columns: lane 32 h + 16 t + j keeps the sum of key 32 t + 8 (j / 4) + 4 h + j % 4
  float v = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float x = group_sum<16>(sum[t][j]);
      x += shfl_xor(x, 16);
      v = (lane & 31) == 16 * t + j ? x : v;
    }
  const int j = lane & 15, t = lane >> 4 & 1;
  const int key = k0 + 32 * t + 8 * (j / 4) + 4 * h + j % 4;
  if (t < NT && key < row.ctx) {
    if (a.column_pieces == 1)
      add_key(a, row, bt, wrow, kvh, key, v);
    else
      ws.sums[(((int64_t)seq * a.cache.num_kv_heads + kvh) * a.column_pieces + piece) * a.score_stride +
              key] = v;
  }
}

// The column pieces' sums joined, a key per thread.
__global__ __launch_bounds__(256) void column_join_kernel(BoundedArgs a, int op_halves, int keys) {
  const int kvh = blockIdx.y, seq = blockIdx.z;
  const ChunkRow row = chunk_row(a, seq);
  const int key = blockIdx.x * 256 + threadIdx.x;
  if (row.n == 0 || key >= row.ctx) return;
  const int64_t wrow = weight_row(a, seq, false);
  if (wrow < 0) return;
  const float* sums = ChunkWs(a, op_halves).sums +
                      ((int64_t)seq * a.cache.num_kv_heads + kvh) * a.column_pieces * a.score_stride + key;
  // the pieces that hold tiles which see the key's tile of keys
  const int first = column_first(row, key / keys * keys, a.group);
  const int tiles = (row.n * a.group + 31) / 32;
  float v = 0.f;
  for (int p = min(first / a.column_tiles, a.column_pieces - 1); p < a.column_pieces; ++p)
    if (p * a.column_tiles < tiles) v += sums[p * a.score_stride];
  add_key(a, row, a.block_tables + (int64_t)seq * a.bt_stride, wrow, kvh, key, v);
}

template <typename QT, int D>
int launch(const BoundedArgs& a, hipStream_t stream) {
  const uint32_t hkv = (uint32_t)a.cache.num_kv_heads, seqs = (uint32_t)a.num_seqs;
  const int64_t ctiles = ((int64_t)a.max_q_len * a.group + 127) / 128;
  if (ctiles * a.chunk_pieces > INT32_MAX) return fail(ASTR_EUNSUPPORTED, "chunk too long");
  hipLaunchKernelGGL((chunk_stats_kernel<QT, D>),
                     dim3((uint32_t)(ctiles * a.chunk_pieces), hkv, seqs), dim3(256), 0, stream, a);
  if (a.chunk_pieces > 1) {
    const int64_t columns = ChunkWs(a, 0).columns;
    hipLaunchKernelGGL(chunk_lse_kernel, dim3((uint32_t)((columns + 255) / 256)), dim3(256), 0,
                       stream, a);
  }
  constexpr int KT = column_sum_keys<D>();
  const int64_t ktiles = ((int64_t)a.max_context + kWaves * KT - 1) / (kWaves * KT);
  hipLaunchKernelGGL((column_sum_kernel<QT, D>), dim3((uint32_t)(ktiles * a.column_pieces), hkv, seqs),
                     dim3(256), 0, stream, a);
  if (a.column_pieces > 1)
    hipLaunchKernelGGL(column_join_kernel, dim3((uint32_t)((a.max_context + 255) / 256), hkv, seqs),
                       dim3(256), 0, stream, a, ColumnOp<QT, D>::kTerms * D, KT);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : hip_fail(err, "key weights (chunks) launch");
}

template <typename QT>
int launch_type(const BoundedArgs& a, hipStream_t s) {
  switch (a.cache.head_dim) {
    case 64: return launch<QT, 64>(a, s);
    case 128: return launch<QT, 128>(a, s);
    case 256: return launch<QT, 256>(a, s);
    default: return fail(ASTR_EUNSUPPORTED, "head_dim %d not in {64,128,256}", a.cache.head_dim);
  }
}

}  // namespace

template <>
int launch_chunk_weights_kf<KF>(const BoundedArgs& a, int32_t q_dtype, hipStream_t stream) {
  switch (q_dtype) {
    case ASTR_F32: return launch_type<float>(a, stream);
    case ASTR_F16: return launch_type<_Float16>(a, stream);
    default: return launch_type<bf16_t>(a, stream);
  }
}

}  // namespace attn
}  // namespace astr
