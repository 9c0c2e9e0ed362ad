// Key weights of prompt chunks over the paged cache (gfx950): for the rows of a step with
// two or more query tokens, each key's softmax weight summed over the row's queries that see
// it (k <= p) and the heads of its group,
//   A[k] += sum_{p >= k} sum_g exp(s_pgk - lse_pg),   lse_pg = log sum_{k <= p} exp(s_pgk).
//
// The scores are formed twice (2 D operations each, cheaper than 4 bytes written and read per
// score): by the attention launch, which keeps 32 (token, head) columns per wave and streams the
// keys, and leaves each column's f16 operands, factor and lse in the workspace; then here, where a
// wave keeps 64 keys and streams the columns in the order in which its lanes read them.
// v_mfma_f32_32x32x16_f16 gives lane (c, h) the scores of column c and keys 8 x + 4 h + y (element
// 4 x + y), so that the sums over columns cross lanes at the end alone. Sums in fp32, in an order
// that depends on the sizes alone. A prompt of 2000
// tokens, 32/8 heads of 128: 80 us of attention, 44 of sums, 7 of their join (with a pass of its own
// for the lse, another 51).
//
// Scores: K codes exact in f16 against one f16 term of a 16-bit query or two of an fp32 one (22
// bits), fp32 accumulation.
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

// The f16 operand of one 32-column tile: lane (c, h) holds column c's d = 16 cc + 8 h + [0, 8).
template <typename QT, int D>
struct ColumnOp {
  static constexpr int kTerms = sizeof(QT) == 4 ? 2 : 1;
  static constexpr int kChunks = D / 16;
  half8_t op[kTerms][kChunks];
};

struct ChunkRow {
  int q0, n, ctx, pos0;
};
// The row's queries and length; n = 0 where it is not a chunk. (The attention launch of the same
// call reports offsets out of range.)
__device__ __forceinline__ ChunkRow chunk_row(const BoundedArgs& a, int seq, bool report) {
  ChunkRow r;
  r.n = seq_queries(a, seq, r.q0);
  r.ctx = bounded_ctx(a, a.context_lens[seq], report);
  if (r.n < a.min_rows || r.ctx < r.n) r.n = 0;
  r.pos0 = r.ctx - r.n;
  return r;
}

// The workgroup's piece and tile. Workgroups are dealt to the 8 XCDs in turn, and under the causal
// mask a piece's or a tile's number says how much of it there is: with a number of tiles that 8
// divides each XCD would take the same few tiles of every piece, so that each piece's tiles begin
// one later (a prompt of 2000 tokens, 32/8 heads of 128: 53 -> 44 us).
__device__ __forceinline__ void unit_of(int pieces, int& piece, int& tile) {
  const int tiles = gridDim.x / pieces;
  piece = blockIdx.x / tiles;
  tile = (blockIdx.x % tiles + piece) % tiles;
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
  const ChunkRow row = chunk_row(a, seq, kvh == 0 && blockIdx.x == 0 && threadIdx.x == 0);
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
  const ColumnWs ws(a, a.column_ws, Op::kTerms * D);
  const int64_t tile0 = ws.tile0(seq, kvh, row.q0);
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
  const ChunkRow row = chunk_row(a, seq, false);
  const int key = blockIdx.x * 256 + threadIdx.x;
  if (row.n == 0 || key >= row.ctx) return;
  const int64_t wrow = weight_row(a, seq, false);
  if (wrow < 0) return;
  const float* sums = ColumnWs(a, a.column_ws, op_halves).sums +
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
