// Key weights of prompt chunks over the paged cache (gfx950): for the rows of a step with
// two or more query tokens, each key's softmax weight summed over the row's queries that see
// it (k <= p) and the heads of its group,
//   A[k] += sum_{p >= k} sum_g exp(s_pgk - lse_pg),   lse_pg = log sum_{k <= p} exp(s_pgk).
//
// Two passes over the scores, which are formed twice (2 D operations each, cheaper than 4
// bytes written and read per score): the first keeps 32 (token, head) columns per wave and
// streams the keys (64 per step, converted once to f16 operands in LDS for the workgroup's
// 128 columns) under a running maximum and sum; the second keeps KT keys per wave and streams
// the columns, whose f16 operands, factor and lse the first left in the workspace in the
// order the second's lanes read them. In both, v_mfma_f32_32x32x16_f16 gives lane (c, h) the
// scores of column c and keys 8 x + 4 h + y (element 4 x + y), so that the first pass reduces
// over keys, and the second over columns until its end, without crossing lanes. Sums in fp32,
// in an order that depends on the sizes alone.
//
// Scores: K codes exact in f16 against one f16 term of a 16-bit query (exact, scaled by a
// power of two per column) or two of an fp32 one (22 bits), fp32 accumulation.
#include <type_traits>

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

// The workspace: per column {factor, lse}, per piece and column {m, l}, the operands.
struct ChunkWs {
  float2_t* cols;
  float2_t* ml;
  half8_t* ops;
  int64_t columns;
  __host__ __device__ explicit ChunkWs(const BoundedArgs& a) {
    columns = ColumnPlace::tiles(a) * a.cache.num_kv_heads * 32;
    cols = reinterpret_cast<float2_t*>(a.chunk_ml);
    ml = cols + columns;
    ops = reinterpret_cast<half8_t*>(ml + a.chunk_pieces * columns);
  }
};

struct ChunkRow {
  int q0, n, ctx, pos0;
};
// The row's queries and length; n = 0 where it is not a chunk. (The attention launch of the same
// call reports what is out of range.)
__device__ __forceinline__ ChunkRow chunk_row(const BoundedArgs& a, int seq) {
  ChunkRow r;
  r.n = seq_queries(a, seq, r.q0);
  r.ctx = bounded_ctx(a, a.context_lens[seq], false);
  if (r.n < 2 || r.ctx < r.n) r.n = 0;
  r.pos0 = r.ctx - r.n;
  return r;
}

__device__ __forceinline__ float log_sum(float m, float l) {
  return l > 0.f ? m + __builtin_amdgcn_logf(l) : INFINITY;
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
  const int piece = blockIdx.x % a.chunk_pieces, ctile = blockIdx.x / a.chunk_pieces;
  const int kvh = blockIdx.y, seq = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int G = a.group;
  const ChunkRow row = chunk_row(a, seq);
  const int f0 = ctile * 128;
  if (f0 >= row.n * G) return;
  // the keys that the workgroup's last column sees, its piece of them
  const int last_tok = min(row.n - 1, (f0 + 127) / G);
  const int blocks = (row.pos0 + last_tok) / kBlockTokens + 1;
  const int b0 = piece * a.chunk_steps * kWaves;
  const int b1 = min(blocks, b0 + a.chunk_steps * kWaves);
  const int nsteps = b1 > b0 ? (b1 - b0 + kWaves - 1) / kWaves : 0;

  // ---- the wave's columns
  const int f = f0 + wave * 32 + (lane & 31), h = lane >> 5;
  const bool valid = f < row.n * G;
  const int tok = valid ? f / G : last_tok, head = kvh * G + (valid ? f % G : 0);
  const int pos = row.pos0 + tok;
  Op q;
  float factor;
  {
    const QT* qp = static_cast<const QT*>(a.q) + (int64_t)(row.q0 + tok) * a.q_tok +
                   (int64_t)head * a.q_head + 8 * h;
    float x[D / 16][8];
    float mx = 0.f;
#pragma unroll
    for (int cc = 0; cc < D / 16; ++cc) {
      struct alignas(16) Run {
        QT e[8];
      };
      const Run run = *reinterpret_cast<const Run*>(qp + 16 * cc);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[cc][i] = valid ? to_float<QT>(run.e[i]) : 0.f;
        mx = vmax(mx, fabsf(x[cc][i]));  // NaN-propagating
      }
    }
    mx = vmax(mx, shfl_xor(mx, 32));
    // a column that is not finite enters as zeros, of no weight: its lse comes out infinite
    const bool finite = __builtin_isfinite(mx);
    int ex = 15;
    if (finite && mx > 0.f) frexpf(mx, &ex);
    ex = max(ex - 15, -126);
#pragma unroll
    for (int cc = 0; cc < D / 16; ++cc)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = finite ? ldexpf(x[cc][i], -ex) : 0.f;
        const _Float16 hi = (_Float16)v;
        q.op[0][cc][i] = hi;
        if constexpr (Op::kTerms == 2) q.op[1][cc][i] = (_Float16)(v - (float)hi);
      }
    factor = finite ? ldexpf(1.f, ex) * a.qk_scale_log2 * code_scale<KF>() : __builtin_nanf("");
    factor = valid ? factor : 0.f;
  }
  const ChunkWs ws(a);
  const int64_t tile = ColumnPlace(a, seq, kvh, row.q0).tile0 + ctile * 4 + wave;
  const bool used = f0 + wave * 32 < row.n * G;  // the wave's tile has a place
  if (piece == 0 && used) {
#pragma unroll
    for (int t = 0; t < Op::kTerms; ++t)
#pragma unroll
      for (int cc = 0; cc < Op::kChunks; ++cc)
        ws.ops[((tile * Op::kTerms + t) * Op::kChunks + cc) * kWave + lane] = q.op[t][cc];
  }

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
  const int inner = row.pos0 + min(row.n - 1, (f0 + wave * 32) / G) + 1;
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
  const ChunkWs ws(a);
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

// Keys of one workgroup: 64 in two tiles, 32 at head dim 256 (the operands fill the registers).
template <int D>
constexpr int column_sum_keys() { return D == 256 ? 32 : 64; }

template <typename QT, int D>
__global__ __launch_bounds__(256, 2) void column_sum_kernel(BoundedArgs a) {
  using Op = ColumnOp<QT, D>;
  constexpr int KT = column_sum_keys<D>(), NT = KT / 32;
  __shared__ float red[kWaves][KT];
  const int kvh = blockIdx.y, seq = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int h = lane >> 5;
  const int G = a.group;
  const ChunkRow row = chunk_row(a, seq);
  const int k0 = blockIdx.x * KT;
  if (row.n == 0 || k0 >= row.ctx) return;
  const int64_t wrow = weight_row(a, seq, false);
  if (wrow < 0) return;

  // ---- the workgroup's keys, as operands in every wave's registers: lane (key, h)
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

  // ---- the column tiles from the first token that sees key k0 on, dealt to the waves
  const ChunkWs ws(a);
  const int64_t tile0 = ColumnPlace(a, seq, kvh, row.q0).tile0;
  const int tiles = (row.n * G + 31) / 32;
  const int first = max(0, k0 - row.pos0) * G / 32;
  float sum[NT][16];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) sum[t][j] = 0.f;
  Op q;
  float2_t col = {0.f, INFINITY};
  auto load = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < Op::kTerms; ++t)
#pragma unroll
      for (int cc = 0; cc < Op::kChunks; ++cc)
        q.op[t][cc] = ws.ops[(((tile0 + c) * Op::kTerms + t) * Op::kChunks + cc) * kWave + lane];
    col = ws.cols[(tile0 + c) * 32 + (lane & 31)];
  };
  if (first + wave < tiles) load(first + wave);
  for (int c = first + wave; c < tiles; c += kWaves) {
    float16v_t s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[t][j] = 0.f;
#pragma unroll
      for (int x = 0; x < Op::kTerms; ++x)
#pragma unroll
        for (int cc = 0; cc < Op::kChunks; ++cc)
          s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kop[t][cc], q.op[x][cc], s[t], 0, 0, 0);
    }
    const float factor = col[0], lse = col[1];
    const int pos = row.pos0 + min(row.n - 1, (c * 32 + (lane & 31)) / G);
    const bool edge = row.pos0 + c * 32 / G < k0 + KT - 1;  // some column does not see some key
    if (c + kWaves < tiles) load(c + kWaves);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][j] * ks[t][j / 4][j % 4], factor, -lse));
        if (edge) p = k0 + 32 * t + 8 * (j / 4) + 4 * h + j % 4 <= pos ? p : 0.f;
        sum[t][j] += p;
      }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float v = group_sum<16>(sum[t][j]);
      v += shfl_xor(v, 16);
      if ((lane & 31) == 0) red[wave][32 * t + 8 * (j / 4) + 4 * h + j % 4] = v;
    }
  __syncthreads();
  const int key = k0 + threadIdx.x;
  if ((int)threadIdx.x < KT && key < row.ctx && key < a.kw.capacity) {
    float v = red[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += red[w][threadIdx.x];
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
}

template <typename QT, int D>
int launch(const BoundedArgs& a, hipStream_t stream) {
  const uint32_t hkv = (uint32_t)a.cache.num_kv_heads, seqs = (uint32_t)a.num_seqs;
  const int64_t ctiles = ((int64_t)a.max_q_len * a.group + 127) / 128;
  if (ctiles * a.chunk_pieces > INT32_MAX) return fail(ASTR_EUNSUPPORTED, "chunk too long");
  hipLaunchKernelGGL((chunk_stats_kernel<QT, D>),
                     dim3((uint32_t)(ctiles * a.chunk_pieces), hkv, seqs), dim3(256), 0, stream, a);
  if (a.chunk_pieces > 1) {
    const int64_t columns = ChunkWs(a).columns;
    hipLaunchKernelGGL(chunk_lse_kernel, dim3((uint32_t)((columns + 255) / 256)), dim3(256), 0,
                       stream, a);
  }
  constexpr int KT = column_sum_keys<D>();
  hipLaunchKernelGGL((column_sum_kernel<QT, D>), dim3((uint32_t)((a.max_context + KT - 1) / KT), hkv, seqs),
                     dim3(256), 0, stream, a);
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
