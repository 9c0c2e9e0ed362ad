// Paged decode attention of a bounded cache (gfx950): rows of one query token at position
// p = ctx - 1, which see
//   keys k > p - window, and k < sinks  (window > 0), or every key;
// with WEIGHTS each key's softmax weight, summed over the heads of its group, is added to
// the weights kept per key and KV head:
//   A[k] += sum_g exp(s_gk - lse_g),  lse_g = log sum_k exp(s_gk).
//
// One workgroup of NW waves takes a (sequence, KV head), or one of the equal pieces of its
// visible blocks; wave w the blocks w, w + NW, ... of them, each 16-token block staged in
// LDS by direct global -> LDS loads, two ahead, and through the MFMAs for all heads of the
// group at once, so that each K/V byte is read from HBM once. The waves' states merge in
// LDS, the pieces' in a second launch (one row's blocks alone cannot fill the GPU).
// The scores do not stay on the chip: with WEIGHTS they are stored as they are formed (4
// bytes a key and head, against 2 D + 8 of its codes and scales) and read again, from the
// cache, once lse is known; reading the keys again instead would double the call's bytes.
//
// Queries of 16 bits: int8 codes meet three int8 terms of the query (exact products, 22
// bits of the query), FP8 codes an f16 query (two f16 terms of an fp32 one); the softmax weights
// enter the output's products rounded to f16 where the output is bf16, else as two f16 terms (22
// bits; one term, 2^-12 beside an f16 output's own 2^-12, saved 3 % of a call: 48 rows of FP8 codes
// 15.2 us, now 15.6). The sums are fp32, before that rounding.
#include <climits>

#include "bounded_common.h"

namespace astr {
namespace attn {
namespace {

#ifndef ASTR_KF
#define ASTR_KF 0
#endif
constexpr int KF = ASTR_KF;  // this translation unit's code format

constexpr int kTileTokens = 1024;  // keys whose weights one workgroup of the second launch adds

// The group's query columns as B operands, built once per workgroup (four elements a lane and
// wave at a time) and read by every wave: for all of them the arithmetic is 500 instructions,
// as much as four blocks take, and 16 waves share a CU. Lane (qg, r) holds elements d = 16 qg + 64 h + [0, 16) of head r.
//   int8 codes: three int8 terms of q * kQRange / max|q| (query_terms: 22 bits of the query)
//   FP8 codes: f16 terms of the column scaled by the power of two that brings its largest
//     element into [2^14, 2^15): one of 16-bit queries (exact; below 2^-28 of that maximum to
//     2^-39 of it), two of fp32 ones (22 bits)
template <typename QT, int D>
struct SharedQuery {
  static constexpr int kTerms = KF == kInt8 ? 3 : sizeof(QT) == 4 ? 2 : 1;
  static constexpr int kPer = KF == kInt8 ? 1 : 2;  // operands of 64 elements of a term
  static constexpr int kOps = kTerms * kPer * (D / 64);
  int4_t op[kOps][kWave];
  float factor[16];  // of the columns' scores; NaN for a column that is not finite
  __device__ static constexpr int at(int term, int h, int sub) { return (term * (D / 64) + h) * kPer + sub; }
};

// Elements 4 w + [0, 4) of chunk h of the columns (`own`), from the lane's elements of all
// chunks (`raw`, for the column's maximum). Cross-lane.
template <typename QT, int D>
__device__ __forceinline__ void share_query(const QueryColumn<QT, D>& raw, const QT (&own)[4], int h,
                                            int w, bool valid, float scale, int lane,
                                            SharedQuery<QT, D>& q) {
  float mx = 0.f;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    const QT* e = reinterpret_cast<const QT*>(raw.w[c]);
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = vmax(mx, fabsf(to_float<QT>(e[i])));  // NaN-propagating
  }
  mx = vmax(mx, shfl_xor(mx, 16));
  mx = vmax(mx, shfl_xor(mx, 32));
  mx = valid ? mx : 0.f;
  const bool finite = __builtin_isfinite(mx);
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = valid && finite ? to_float<QT>(own[i]) : 0.f;
  float factor;
  if constexpr (KF == kInt8) {
    factor = scale * (mx / (float)kQRange);
    // kQRange / mx overflows for mx below 2^-114: such columns are lifted by 2^64 (exact)
    const float up = mx > 0.f && mx < 0x1p-64f ? 0x1p64f : 1.f;
    const float inv = finite && mx > 0.f ? (float)kQRange / (mx * up) : 0.f;
    uint32_t b[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const QueryTerms t = query_terms(x[i] * up, inv);
      b[0][i] = __builtin_bit_cast(uint32_t, t.hi);
      b[1][i] = __builtin_bit_cast(uint32_t, t.lo);
      b[2][i] = __builtin_bit_cast(uint32_t, t.lo2);
    }
#pragma unroll
    for (int t = 0; t < 3; ++t)
      reinterpret_cast<uint32_t*>(&q.op[q.at(t, h, 0)][lane])[w] = low_bytes(b[t]);
  } else {
    int ex = 15;
    if (finite && mx > 0.f) frexpf(mx, &ex);
    ex = max(ex - 15, -126);
    factor = ldexpf(1.f, ex) * scale * code_scale<KF>();
    half4_t op[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = ldexpf(x[i], -ex);
      op[0][i] = (_Float16)v;
      op[1][i] = (_Float16)(v - (float)op[0][i]);
    }
#pragma unroll
    for (int t = 0; t < SharedQuery<QT, D>::kTerms; ++t)
      reinterpret_cast<uint2*>(&q.op[q.at(t, h, w / 2)][lane])[w % 2] =
          __builtin_bit_cast(uint2, op[t]);
  }
  if (h == 0 && w == 0 && lane < 16) q.factor[lane] = finite ? factor : __builtin_nanf("");
}

// The unit 2^e of the V scales: weights enter the output's products as p * (v_scale * 2^-e)
// in f16, the accumulators hold the output times 2^-e. The first block's largest scale sets
// it to [2^4, 2^5) units, and a block with one above 2^7 sets it anew: p <= 2^kRescaleSlack
// keeps the products' weights at 2^15 or less, and above f16's smallest step (2^-24) down to
// 2^-28 of the largest.
struct VUnit {
  int e;
  float inv, limit;
};

// One staged block through the MFMAs. Lane (qg, r) holds the scores of keys 4 qg + j for
// head r; those of keys outside [lo, hi) and of padding keys are -inf. Returns them.
template <typename QT, int D>
__device__ __forceinline__ float4_t bounded_block(const char* st,
                                              const int4_t (&q)[SharedQuery<QT, D>::kOps],
                                              float cf, int tok_base, int lo, int hi, bool gvalid, int r,
                                              int qg, float4_t (&acc)[D / 16], float& m, float& l,
                                              VUnit& vu, bool& bad_score, bool masks) {
  using S = Stage<D>;
  using Q = SharedQuery<QT, D>;
  constexpr int KCH = D / 64, VB = D / 16, NPV = D / 16;
  const float4_t vs = *reinterpret_cast<const float4_t*>(st + S::kS + 64 + 16 * qg) * code_scale<KF>();
  const float4_t ks = *reinterpret_cast<const float4_t*>(st + S::kS + 16 * qg);
  const float screened = *reinterpret_cast<const float*>(st + S::kS + 64 + 4 * r);
  float4_t s4;
  if constexpr (KF == kInt8) {
    int4_t si = {0, 0, 0, 0}, sf = {0, 0, 0, 0};
    int4_t kop[KCH];
#pragma unroll
    for (int h = 0; h < KCH; ++h)
      kop[h] = *reinterpret_cast<const int4_t*>(st + S::kK + k_chunk<D>(r, qg + 4 * h));
#pragma unroll
    for (int h = 0; h < KCH; ++h) si = __builtin_amdgcn_mfma_i32_16x16x64_i8(kop[h], q[Q::at(0, h, 0)], si, 0, 0, 0);
#pragma unroll
    for (int h = 0; h < KCH; ++h) sf = __builtin_amdgcn_mfma_i32_16x16x64_i8(kop[h], q[Q::at(2, h, 0)], sf, 0, 0, 0);
    si = si << 7;
#pragma unroll
    for (int h = 0; h < KCH; ++h) si = __builtin_amdgcn_mfma_i32_16x16x64_i8(kop[h], q[Q::at(1, h, 0)], si, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) s4[j] = __builtin_fmaf((float)sf[j], 1.f / 128.f, (float)si[j]);
  } else {
    s4 = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < KCH; ++h) {
      const uint4 c = *reinterpret_cast<const uint4*>(st + S::kK + k_chunk<D>(r, qg + 4 * h));
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        half2_t p0, p1, p2, p3;
        codes_to_f16<KF>(sub ? c.z : c.x, p0, p1);
        codes_to_f16<KF>(sub ? c.w : c.y, p2, p3);
        const half8_t kop = {p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
#pragma unroll
        for (int t = 0; t < Q::kTerms; ++t)
          s4 = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              kop, __builtin_bit_cast(half8_t, q[Q::at(t, h, sub)]), s4, 0, 0, 0);
      }
    }
  }
  // the conversions of MFMA results stay ahead of the branches below: sunk into their blocks,
  // they have been issued without the wait states an MFMA result needs
  asm volatile("" : "+v"(s4[0]), "+v"(s4[1]), "+v"(s4[2]), "+v"(s4[3]));

  if (__builtin_expect(__ballot(screened * code_scale<KF>() > vu.limit) != 0, 0)) {
    float top = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
    top = fmaxf(top, shfl_xor(top, 16));
    top = fmaxf(top, shfl_xor(top, 32));
    int x = 5;
    if (__builtin_isfinite(top) && top > 0.f) frexpf(top, &x);
    x = min(max(x - 5, -120), 120);
    const float down = ldexpf(1.f, max(vu.e - x, -250));  // (a first block's accumulators are 0)
#pragma unroll
    for (int n = 0; n < NPV; ++n) acc[n] *= down;
    vu = VUnit{x, ldexpf(1.f, -x), ldexpf(1.f, x + 7)};
  }

  bool padded = false;
  if (masks) padded = __ballot(*reinterpret_cast<const uint32_t*>(st + S::kF + 4 * qg) != 0x01010101u) != 0;
  float sc[4];
  bool nonfinite = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) sc[j] = s4[j] * (ks[j] * cf);
  if (tok_base < lo || tok_base + kBlockTokens > hi || padded) {
    const int tok0 = tok_base + 4 * qg;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool seen = tok0 + j >= lo && tok0 + j < hi && (!masks || st[S::kF + 4 * qg + j] != 0);
      nonfinite |= gvalid && seen && !__builtin_isfinite(sc[j]);
      sc[j] = seen ? sc[j] : -INFINITY;
    }
  } else {
    const float most = vmax(vmax(sc[0], sc[1]), vmax(sc[2], sc[3]));
    const float least = vmin(vmin(sc[0], sc[1]), vmin(sc[2], sc[3]));
    nonfinite = gvalid && !(__builtin_isfinite(most) && __builtin_isfinite(least));
  }
  if (__builtin_expect(__ballot(nonfinite) != 0, 0)) bad_score = true;
  float tmax = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
  if (__builtin_expect(__ballot(gvalid && tmax > m + kRescaleSlack) != 0, 0)) {
    tmax = fmaxf(tmax, shfl_xor(tmax, 16));
    tmax = fmaxf(tmax, shfl_xor(tmax, 32));
    const float mn = fmaxf(m, tmax);
    const float alpha = __builtin_amdgcn_exp2f(m - mn);
    l *= alpha;
#pragma unroll
    for (int n = 0; n < NPV; ++n) acc[n] *= alpha;
    m = mn;
  }
  constexpr int kTerms = __is_same(QT, bf16_t) ? 1 : 2;
  half4_t pop[kTerms];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float p = __builtin_amdgcn_exp2f(sc[j] - m);
    l += p;
    float w = p * (vs[j] * vu.inv);
    // (one rounding of the product for both terms: a multiply that rounds to f16 by itself would
    // now and then give a first term that the second does not fit)
    if constexpr (kTerms == 2) asm volatile("" : "+v"(w));
    pop[0][j] = (_Float16)w;
    if constexpr (kTerms == 2) pop[1][j] = (_Float16)(w - (float)pop[0][j]);
  }
  uint32_t vw[4][VB / 4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const char* rowp = st + S::kV + (4 * qg + j) * D + r * VB;
    struct alignas(VB) Run {
      uint32_t w[VB / 4];
    };
    const Run run = *reinterpret_cast<const Run*>(rowp);
#pragma unroll
    for (int i = 0; i < VB / 4; ++i) vw[j][i] = run.w[i];
  }
  // O^T += V^T P^T (row i of MFMA n is d = VB i + n)
#pragma unroll
  for (int n = 0; n < NPV; ++n) {
    const uint32_t col[4] = {vw[0][n / 4], vw[1][n / 4], vw[2][n / 4], vw[3][n / 4]};
    half4_t vop;
    switch (n % 4) {
      case 0: vop = v_operand<0, KF>(col); break;
      case 1: vop = v_operand<1, KF>(col); break;
      case 2: vop = v_operand<2, KF>(col); break;
      default: vop = v_operand<3, KF>(col); break;
    }
#pragma unroll
    for (int t = 0; t < kTerms; ++t)
      acc[n] = __builtin_amdgcn_mfma_f32_16x16x16f16(vop, pop[t], acc[n], 0, 0, 0);
  }
  return float4_t{sc[0], sc[1], sc[2], sc[3]};
}

// The scores (base 2) of four keys from t on for up to eight heads from g0 on, on their way
// together (one head at a time, the second launch of a row of 8192 keys took 6.3 us instead of 5.0).
struct KeyScores {
  static constexpr int kHeads = 8;
  float4_t s[kHeads];
  __device__ __forceinline__ void load(const BoundedArgs& a, const float* scores, int g0, int t) {
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (g0 + i < a.group)  // (uniform)
        s[i] = *reinterpret_cast<const float4_t*>(scores + (g0 + i) * a.score_stride + t);
  }
  // Adds their weights; lse (base 2) of the group's heads, +inf where one adds none.
  __device__ __forceinline__ void add(const BoundedArgs& a, const float* lse, int g0, float4_t& sum) const {
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (g0 + i < a.group) {
        const float e = lse[g0 + i];
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += e == INFINITY ? 0.f : __builtin_amdgcn_exp2f(s[i][j] - e);
      }
  }
};

// Adds the weights of keys t to t + 3, as far as they lie below t1, of one (sequence, KV head): its
// scores at `scores` (one row per head, a.score_stride apart), those of the first heads in `first`.
// The row's newest key starts at 0.
__device__ __forceinline__ void add_keys(const BoundedArgs& a, const KeyScores& first, const float* scores,
                                         const float* lse, float* weights, int ctx, int t, int t1) {
  float4_t sum = {0.f, 0.f, 0.f, 0.f};
  first.add(a, lse, 0, sum);
  if (a.group > KeyScores::kHeads) {
    KeyScores more;
    more.load(a, scores, KeyScores::kHeads, t);
    more.add(a, lse, KeyScores::kHeads, sum);
  }
  if (t + 4 <= min(t1, ctx - 1)) {
    *reinterpret_cast<float4_t*>(weights + t) += sum;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (t + j < t1) weights[t + j] = (t + j == ctx - 1 ? 0.f : weights[t + j]) + sum[j];
  }
}

__device__ __forceinline__ int row_parts(const BoundedArgs& a, const VisibleList& v) {
  const int parts = (v.blocks + a.part_blocks - 1) / a.part_blocks;
  return parts < 1 ? 1 : parts;  // <= max_parts: v comes of a length within max_context
}

// log2 of the sum over keys; +inf where the head saw none or its scores are not finite: it
// adds no weights.
__device__ __forceinline__ float log_sum(float m, float l) {
  return l > 0.f ? m + __builtin_amdgcn_logf(l) : INFINITY;
}

// The row that is `nth` by length, the longest first (of equal ones the lowest): a grid that deals
// out few workgroups per CU then does not end on a long row alone (64 rows of 128 to 4096 tokens,
// 8 KV heads, bf16: 85 us instead of 90). At most kOrderRows rows; every thread calls it.
constexpr int kOrderRows = 128;
__device__ __forceinline__ int nth_longest(const BoundedArgs& a, int nth, char* lds) {
  int* const len = reinterpret_cast<int*>(lds);  // kOrderRows lengths, then the row
  const int t = threadIdx.x;
  if (t < kOrderRows) len[t] = t < a.num_seqs ? a.context_lens[t] : INT_MIN;
  __syncthreads();
  if (t < a.num_seqs) {
    const int mine = len[t];
    int rank = 0;
#pragma unroll 1
    for (int j = 0; j < a.num_seqs; j += 4) {
      const int4_t v = *reinterpret_cast<const int4_t*>(len + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) rank += v[i] > mine || (v[i] == mine && j + i < t);
    }
    if (rank == nth) len[kOrderRows] = t;
  }
  __syncthreads();
  const int seq = __builtin_amdgcn_readfirstlane(len[kOrderRows]);
  __syncthreads();  // the stages take the lengths' place
  return seq;
}

template <int D, int NW>
struct BoundedLds {
  static constexpr int kStageBytes = NW * Stage<D>::kBytes;
  // a wave's outputs of a head: four lanes' runs of D / 4, each padded by four floats against
  // bank conflicts (with single stores at stride D / 4, 1.8 us of a 12.3 us call); groups of 16
  // heads, which would then take more LDS than the stages, go without the padding
  __device__ static constexpr int run(int group) { return group == 16 ? D / 4 : D / 4 + 4; }
  static constexpr int kMergeBytes =
      NW * (16 * (D + 2) > 8 * (D + 16) + 32 ? 16 * (D + 2) : 8 * (D + 16) + 32) * 4;
  static constexpr int kBytes = 2 * kStageBytes > kMergeBytes ? 2 * kStageBytes : kMergeBytes;
};

template <typename QT, int D, int NW, bool WEIGHTS>
__global__ __launch_bounds__(NW * kWave) void bounded_decode_kernel(BoundedArgs a) {
  static_assert(D == 64 || D == 128 || D == 256, "head_dim");
  using S = Stage<D>;
  using L = BoundedLds<D, NW>;
  constexpr int NPV = D / 16, VB = D / 16;
  static_assert(L::kBytes + sizeof(SharedQuery<QT, D>) + 64 <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) char lds[L::kBytes];
  __shared__ SharedQuery<QT, D> query;
  __shared__ float lse[16];

  const int part = blockIdx.x, kvh = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int r = lane & 15, qg = lane >> 4;
  const int seq = WEIGHTS && a.longest_first ? nth_longest(a, blockIdx.z, lds) : blockIdx.z;
  const int G = a.group;
  const bool gvalid = r < G;
  const int tok = decode_token(a, seq);
  if (tok < 0) return;  // not a decode row
  QueryColumn<QT, D> raw;
  const QT* const qp = query_col_ptr<QT>(a, tok, kvh * G + (gvalid ? r : 0), qg);
  load_query_column<QT, D>(qp, raw);
  constexpr int kQuads = D / 16;  // of a lane; wave w builds those w, w + NW, ...
  struct alignas(4 * sizeof(QT)) Quad {
    QT e[4];
  } own[(kQuads + NW - 1) / NW];
#pragma unroll
  for (int i = 0; i < (kQuads + NW - 1) / NW; ++i) {
    const int quad = min(wave + i * NW, kQuads - 1);
    own[i] = *reinterpret_cast<const Quad*>(qp + 64 * (quad / 4) + 4 * (quad % 4));
  }
  const bool reporter = part == 0 && kvh == 0 && threadIdx.x == 0;
  const VisibleList v = visible_list(a, bounded_ctx(a, a.context_lens[seq], reporter));
  const int parts = row_parts(a, v);
  if (part >= parts) return;
  const int f0 = part * a.part_blocks + wave;
  const int f1 = min(v.blocks, (part + 1) * a.part_blocks);
  const int nbw = f0 < f1 ? (f1 - f0 + NW - 1) / NW : 0;  // at most 64 (host)
  const int32_t* bt = a.block_tables + (int64_t)seq * a.bt_stride;
  const int ids = lane < nbw ? bt[v.block(f0 + NW * lane)] : 0;
  // a block outside the arena: the wave reports it and reads nothing
  const bool bad_index = __ballot(lane < nbw && (unsigned)ids >= (unsigned)a.cache.num_blocks) != 0;
  const int nblk = bad_index ? 0 : nbw;

  char* const st0 = lds + wave * S::kBytes;
  char* const st1 = lds + L::kStageBytes + wave * S::kBytes;
  if (0 < nblk) stage_block<D>(a, __builtin_amdgcn_readlane(ids, 0), kvh, lane, st0);
  if (1 < nblk) stage_block<D>(a, __builtin_amdgcn_readlane(ids, 1), kvh, lane, st1);

  // (the blocks' loads are on their way)
#pragma unroll
  for (int i = 0; i < (kQuads + NW - 1) / NW; ++i) {
    const int quad = wave + i * NW;
    if (quad < kQuads)
      share_query<QT, D>(raw, own[i].e, quad / 4, quad % 4, gvalid, a.qk_scale_log2, lane, query);
  }
  __syncthreads();
  int4_t q[SharedQuery<QT, D>::kOps];
#pragma unroll
  for (int i = 0; i < SharedQuery<QT, D>::kOps; ++i) q[i] = query.op[i][lane];
  const float cf = query.factor[r];
  float4_t acc[NPV];
#pragma unroll
  for (int n = 0; n < NPV; ++n) acc[n] = float4_t{0.f, 0.f, 0.f, 0.f};
  float m = gvalid ? -FLT_MAX : 0.f, l = 0.f;  // finite: a block without a visible key adds 0
  VUnit vu{0, 1.f, -1.f};
  bool bad_score = false;
  const bool masks = a.cache.key_valid != nullptr;
  const int64_t unit = (int64_t)seq * a.cache.num_kv_heads + kvh;
  float* const srow = WEIGHTS ? a.scores + (unit * G + (gvalid ? r : 0)) * a.score_stride : nullptr;

  auto step = [&](int i, char* st) __attribute__((always_inline)) {
    // block i has landed once only the next one's loads may be on their way, and (WEIGHTS) the
    // score store issued after them: vector-memory operations complete in order (a padding load
    // among the younger ones makes this wait longer). Stores ahead of the next loads instead made
    // every block wait for the one before's (16 rows of 32768 tokens, 64 heads: 1 % of the launch).
    if (i + 1 >= nblk) wait_vmcnt<0>();
    else if (WEIGHTS && i > 0) wait_vmcnt<S::kLoads + 1>();
    else wait_vmcnt<S::kLoads>();
    const int f = f0 + NW * i;
    const int base = v.block(f) * kBlockTokens;
    const float4_t sc = bounded_block<QT, D>(st, q, cf, base, v.lo(f), v.hi(f), gvalid, r, qg, acc, m, l,
                                             vu, bad_score, masks);
    if (i + 2 < nblk) stage_block<D>(a, __builtin_amdgcn_readlane(ids, i + 2), kvh, lane, st);
    if constexpr (WEIGHTS) {
      asm volatile("" ::: "memory");  // the store stays behind the loads
      if (gvalid) *reinterpret_cast<float4_t*>(srow + base + 4 * qg) = sc;
    }
  };
  for (int i = 0; i < nblk; i += 2) {
    step(i, st0);
    if (i + 1 >= nblk) break;
    step(i + 1, st1);
  }
  if (bad_index) {
    if (lane == 0) atomicOr(a.err_flag, ASTR_FLAG_BAD_INDEX);
    if (WEIGHTS && gvalid)  // its keys add no weight
      for (int i = 0; i < nbw; ++i)
        *reinterpret_cast<float4_t*>(srow + v.block(f0 + NW * i) * kBlockTokens + 4 * qg) =
            float4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  }
  if (bad_score && lane == 0) atomicOr(a.err_flag, ASTR_FLAG_NONFINITE_SCORE);

  // ---- the waves' states, in LDS (over the stages: every wave has read its own)
  l += shfl_xor(l, 16);
  l += shfl_xor(l, 32);
  const float up = ldexpf(1.f, vu.e);
  __syncthreads();
  float* const sm = reinterpret_cast<float*>(lds);  // [NW][16]
  float* const sl = sm + NW * 16;
  const int run = L::run(G);
  float* const so = sl + NW * 16;  // [NW][G][4][run]
  if (gvalid) {
    if (qg == 0) {
      sm[wave * 16 + r] = m;
      sl[wave * 16 + r] = l;
    }
    float* o = so + ((wave * G + r) * 4 + qg) * run;  // d = D / 4 qg + t
#pragma unroll
    for (int t = 0; t < D / 4; t += 4)
      *reinterpret_cast<float4_t*>(o + t) =
          float4_t{acc[t % VB][t / VB], acc[(t + 1) % VB][(t + 1) / VB],
                   acc[(t + 2) % VB][(t + 2) / VB], acc[(t + 3) % VB][(t + 3) / VB]} * up;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += NW * kWave) {
    const int g = i / D, d = i % D;
    const float* o = so + (g * 4 + d / (D / 4)) * run + d % (D / 4);
    float M = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w * 16 + g]);
    float Lg = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w * 16 + g] - M);
      Lg = fmaf(sl[w * 16 + g], f, Lg);
      O = fmaf(o[w * G * 4 * run], f, O);
    }
    const int h = kvh * G + g;
    if (parts == 1) {
      static_cast<QT*>(a.out)[(int64_t)tok * a.o_tok + (int64_t)h * a.o_head + d] =
          from_float<QT>(O / fmaxf(Lg, FLT_MIN));
      if (WEIGHTS && d == 0) lse[g] = log_sum(M, Lg);
    } else {
      const int64_t at = ((int64_t)seq * a.num_q_heads + h) * a.max_parts + part;
      a.ws_o[at * D + d] = O;
      if (d == 0) {
        a.ws_ml[at * 2] = M;
        a.ws_ml[at * 2 + 1] = Lg;
      }
    }
  }
  if constexpr (WEIGHTS) {
    if (parts > 1) return;
    const int64_t row = weight_row(a, seq, reporter);
    if (reporter && v.ctx > a.kw.capacity) atomicOr(a.err_flag, ASTR_FLAG_BAD_INDEX);
    __threadfence_block();  // the scores, which other waves of the workgroup stored
    __syncthreads();
    if (row < 0) return;
    const float* const scores = a.scores + unit * G * a.score_stride;
    float* const weights = a.kw.values + row * a.kw.row_stride + kvh * a.kw.head_stride;
    const int t1 = min(v.ctx, a.kw.capacity);
    for (int t = 4 * threadIdx.x; t < t1; t += 4 * NW * kWave) {
      KeyScores first;
      first.load(a, scores, 0, t);
      add_keys(a, first, scores, lse, weights, v.ctx, t, t1);
    }
  }
}

// The second launch, for rows of several pieces: the pieces' states merged into the output
// (the first workgroup of a (sequence, KV head)), and the weights of kTileTokens keys each.
template <typename QT, int D, bool WEIGHTS>
__global__ __launch_bounds__(256) void bounded_merge_kernel(BoundedArgs a) {
  __shared__ float top[16], sum[16], lse[16];
  const int tile = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int tok = decode_token(a, seq);
  if (tok < 0) return;
  const VisibleList v = visible_list(a, bounded_ctx(a, a.context_lens[seq], false));
  const int parts = row_parts(a, v);
  if (parts <= 1 || (tile > 0 && tile * kTileTokens >= v.ctx)) return;
  const int G = a.group;
  const int64_t head0 = (int64_t)seq * a.num_q_heads + kvh * G;
  static_assert(kTileTokens == 4 * 256, "four keys a thread");
  const int t = tile * kTileTokens + 4 * (int)threadIdx.x;
  const float* const scores = WEIGHTS ? a.scores + head0 * a.score_stride : nullptr;
  KeyScores first;  // on their way while lse is worked out
  if (WEIGHTS && t < v.ctx) first.load(a, scores, 0, t);
  for (int g = wave; g < G; g += kWaves) {
    const float* ml = a.ws_ml + (head0 + g) * a.max_parts * 2;
    float M = -FLT_MAX;
    for (int p = lane; p < parts; p += kWave) M = fmaxf(M, ml[2 * p]);
    M = wave_max(M);
    float Lg = 0.f;
    for (int p = lane; p < parts; p += kWave)
      Lg = fmaf(ml[2 * p + 1], __builtin_amdgcn_exp2f(ml[2 * p] - M), Lg);
    Lg = wave_sum(Lg);
    if (lane == 0) {
      top[g] = M;
      sum[g] = Lg;
      lse[g] = log_sum(M, Lg);
    }
  }
  __syncthreads();
  if (tile == 0) {
    for (int i = threadIdx.x; i < G * D; i += 256) {
      const int g = i / D, d = i % D;
      const int64_t at = (head0 + g) * a.max_parts;
      float O = 0.f;
#pragma unroll 4
      for (int p = 0; p < parts; ++p)
        O = fmaf(a.ws_o[(at + p) * D + d], __builtin_amdgcn_exp2f(a.ws_ml[(at + p) * 2] - top[g]), O);
      static_cast<QT*>(a.out)[(int64_t)tok * a.o_tok + (int64_t)(kvh * G + g) * a.o_head + d] =
          from_float<QT>(O / fmaxf(sum[g], FLT_MIN));
    }
  }
  if constexpr (WEIGHTS) {
    const bool reporter = tile == 0 && kvh == 0 && threadIdx.x == 0;
    const int64_t row = weight_row(a, seq, reporter);
    if (reporter && v.ctx > a.kw.capacity) atomicOr(a.err_flag, ASTR_FLAG_BAD_INDEX);
    const int t1 = min(v.ctx, a.kw.capacity);
    if (row >= 0 && t < t1)
      add_keys(a, first, scores, lse, a.kw.values + row * a.kw.row_stride + kvh * a.kw.head_stride, v.ctx,
               t, t1);
  }
}

template <typename QT, int D, int NW, bool WEIGHTS>
int launch(const BoundedArgs& a, hipStream_t stream) {
  const dim3 grid((uint32_t)a.max_parts, (uint32_t)a.cache.num_kv_heads, (uint32_t)a.num_seqs);
  hipLaunchKernelGGL((bounded_decode_kernel<QT, D, NW, WEIGHTS>), grid, dim3(NW * kWave), 0, stream, a);
  if (a.max_parts > 1) {
    const int tiles = WEIGHTS ? (a.max_context + kTileTokens - 1) / kTileTokens : 1;
    hipLaunchKernelGGL((bounded_merge_kernel<QT, D, WEIGHTS>), dim3((uint32_t)tiles, grid.y, grid.z),
                       dim3(256), 0, stream, a);
  }
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : hip_fail(err, "paged_attention (bounded decode) launch");
}

template <typename QT, int D>
int launch_dim(const BoundedArgs& a, hipStream_t s) {
  const bool weights = a.kw.values != nullptr;
  // total_waves: the workgroup's waves
  if constexpr (wide_waves(D, sizeof(QT) == 4) == 16) {
    if (a.total_waves == 16 && weights) return launch<QT, D, 16, true>(a, s);
  }
  if constexpr (wide_waves(D, false) == 16) {
    if (a.total_waves == 16 && !weights) return launch<QT, D, 16, false>(a, s);
  }
  if (a.total_waves == 8) return weights ? launch<QT, D, 8, true>(a, s) : launch<QT, D, 8, false>(a, s);
  return weights ? launch<QT, D, 4, true>(a, s) : launch<QT, D, 4, false>(a, s);
}

template <typename QT>
int launch_type(const BoundedArgs& a, hipStream_t s) {
  switch (a.cache.head_dim) {
    case 64: return launch_dim<QT, 64>(a, s);
    case 128: return launch_dim<QT, 128>(a, s);
    case 256: return launch_dim<QT, 256>(a, s);
    default: return fail(ASTR_EUNSUPPORTED, "head_dim %d not in {64,128,256}", a.cache.head_dim);
  }
}

}  // namespace

template <>
int launch_bounded_kf<KF>(const BoundedArgs& a, int32_t q_dtype, hipStream_t stream) {
  switch (q_dtype) {
    case ASTR_F32: return launch_type<float>(a, stream);
    case ASTR_F16: return launch_type<_Float16>(a, stream);
    default: return launch_type<bf16_t>(a, stream);
  }
}

}  // namespace attn
}  // namespace astr
