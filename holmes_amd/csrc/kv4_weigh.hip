// What attention has given each token of a 4-bit cache: over the rows i of a key head that see token j
//
//   w_j = prior_j + sum_i exp(scale q_i.k_j - lse_i)
//
// with lse_i the log of the row's sum of exponentials, as the attention before left it.  One product and no softmax: only
// the keys are read, and each token's sum stays with the wave that has the token, so nothing is added in an order that changes.
#include "kv4_attend.hpp"

namespace hck {
namespace {

struct WeighArgs {
  AttendArgs a;  // of which: pool, q, table, lengths, starts, strides, shapes
  const float *row_lse, *prior;
  float* weights;
  int64_t prior_seq, prior_head;
  int prior_places;
  float scale2, rest;  // scale log2 e in 32 bits, and what its rounding left over, divided by scale
};

// A row's share of the exponents: what comes off, in units of log 2, and a factor near 1 for what rounding took from
// that and from scale log2 e (counted where the score is the row's lse, near which weights are large).
struct RowTerm {
  float off, factor;
  int seen;
};
__device__ __forceinline__ RowTerm row_term(const WeighArgs& W, const Rows& R, int h, int row) {
  RowTerm r = {0.f, 1.f, 0};
  if (row >= R.rows) return r;
  const int64_t at = (int64_t)(R.q0 + row / W.a.group) * ((int64_t)W.a.heads * W.a.group) + h * W.a.group + row % W.a.group;
  const float lse = W.row_lse[at];
  r.off = lse * kLog2e;
  r.seen = lse == -INFINITY ? 0 : R.seen(W.a, row);  // such a row gave nothing
  if (fabsf(lse) < INFINITY) {
    const float low = __builtin_fmaf(lse, kLog2e, -r.off) + lse * 1.9259629911266174e-8f;  // (log2 e in two parts)
    r.factor = 1.f + kLn2 * (lse * W.rest - low);
  }
  return r;
}

// 64 tokens of a key head to a wave; 16 rows at a time.
template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void k_weigh(WeighArgs W) {
  using L = Kv4<D>;
  constexpr int kSteps = D / 32;
  constexpr bool kHalf = __is_same(T, _Float16);
  const AttendArgs& A = W.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % A.heads, u = blockIdx.x / A.heads * kWaves + wave, b = blockIdx.y;
  if (u >= 2 * A.cols) return;
  const int here = u * kUnit, mine = here + g * 16 + m;  // the token that the lane writes
  float* to = W.weights + ((int64_t)b * A.heads + h) * ((int64_t)A.cols * kPageTokens) + mine;
  const Rows R(A, b);
  if (here >= R.length) {
    *to = 0.f;
    return;
  }
  const int pg = A.table[b * A.table_stride + (u >> 1)];
  const bool there = pg >= 0 && pg < A.pages;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  if (there) {
    const uint8_t* page = A.pool + ((int64_t)pg * A.heads + h) * L::kBytes;
    const uint8_t* codes = page + (u & 1) * (32 * D);
    typedef uint32_t words __attribute__((ext_vector_type(kSteps)));
    words c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = *reinterpret_cast<const words*>(codes + i * (8 * D) + lane * (D / 8));
    const uint32_t scales =
        *reinterpret_cast<const uint32_t*>(page + L::kKScales + (u & 1) * (64 * L::kRuns) + g * (D / 4) / kRun * 64 + m * 4);
    bf16x8 k[4][kSteps];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t byte = (scales >> (8 * i)) & 0xffu;
      const float sc = byte == kNanByte ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        k[i][s] = operand(cvt<0>(c[i][s], sc), cvt<1>(c[i][s], sc), cvt<2>(c[i][s], sc), cvt<3>(c[i][s], sc));
    }
    // rows that see a token of these: from the first query that does
    const int skip = A.causal ? (int)((int64_t)max(0, here - (R.length - R.nq)) * A.group / 16) : 0;
    for (int tile = skip; tile * 16 < R.rows; ++tile) {
      const int row = tile * 16 + m;
      const bool live = row < R.rows;
      const T* qp = (const T*)A.q + (R.q0 + (live ? row / A.group : 0)) * A.q_ts +
                    (int64_t)(h * A.group + (live ? row % A.group : 0)) * A.q_hs + g * (D / 4);
      f32x4 s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < kSteps; ++d) {
        u32x4 raw = {0, 0, 0, 0};
        if (live) raw = reinterpret_cast<const Loose16*>(qp + 8 * d)->v;
        bf16x8 head, rest;
        query_parts<T>(raw, head, rest);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[i] = mfma(head, k[i][d], s[i]);
          if constexpr (kHalf) s[i] = mfma(rest, k[i][d], s[i]);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const RowTerm t = row_term(W, R, h, tile * 16 + 4 * g + r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], W.scale2, -t.off));
          acc[i] = __builtin_fmaf(here + 16 * i + m < t.seen ? p : 0.f, t.factor, acc[i]);
        }
      }
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float all = over_g(acc[i], [](float a, float c) { return a + c; });
    sum = g == i ? all : sum;
  }
  if (mine >= R.length) sum = 0.f;
  else if (W.prior && mine < W.prior_places) sum += W.prior[b * W.prior_seq + h * W.prior_head + mine];
  *to = sum;
}

}  // namespace
}  // namespace hck

extern "C" int hck_kv4_weigh(const void* pool, int64_t pages, int kv_heads, int head_dim, int type, const void* queries,
                             int64_t tokens, int group, int64_t q_token_stride, int64_t q_head_stride, const int32_t* table,
                             int64_t table_stride, int table_columns, const int32_t* lengths, const int32_t* starts, int seqs,
                             int most, int causal, double scale, const float* lse, const float* prior, int64_t prior_seq_stride,
                             int64_t prior_head_stride, int prior_places, float* weights, void* stream) {
  if (hck::kv4_bytes(head_dim) == 0 || (type != HCK_BF16 && type != HCK_F16)) return HCK_ERR_UNSUPPORTED;
  if (!pool || pages < 1 || kv_heads < 1 || kv_heads > 65535 || tokens < 0 || tokens > INT32_MAX || group < 1 || seqs < 0 ||
      seqs > 65535 || most < 0 || table_columns < 0 || table_columns >= 1 << 23 || prior_places < 0 ||
      !((float)scale > 0.f && scale <= 0x1p126) || (int64_t)most * group > INT32_MAX || (int64_t)kv_heads * group > INT32_MAX)
    return HCK_ERR_ARG;
  if (!starts && tokens != seqs) return HCK_ERR_ARG;
  if (seqs == 0 || table_columns == 0) return HCK_OK;
  if (!table || !lengths || !weights || (tokens && (!queries || !lse)) || (prior_places && !prior)) return HCK_ERR_ARG;
  hck::WeighArgs W = {};
  hck::AttendArgs& A = W.a;
  A.pool = (const uint8_t*)pool, A.q = queries, A.table = table, A.lengths = lengths, A.starts = starts;
  A.q_ts = q_token_stride, A.q_hs = q_head_stride, A.tokens = tokens, A.pages = pages, A.table_stride = table_stride;
  A.cols = table_columns, A.heads = kv_heads, A.group = group, A.causal = causal != 0, A.seqs = seqs;
  A.tiles = most, A.size = group;
  W.row_lse = lse, W.prior = prior, W.weights = weights, W.prior_seq = prior_seq_stride, W.prior_head = prior_head_stride;
  W.prior_places = prior ? prior_places : 0;
  const double scale2 = scale * 1.4426950408889634;
  W.scale2 = (float)scale2, W.rest = (float)((scale2 - W.scale2) / scale);
  const int64_t groups = ((int64_t)table_columns * 2 + hck::kWaves - 1) / hck::kWaves * kv_heads;
  if (groups > INT32_MAX) return HCK_ERR_ARG;
  const dim3 grid((unsigned)groups, seqs);
  hipStream_t s = (hipStream_t)stream;
  if (head_dim == 128) {
    if (type == HCK_BF16) hck::k_weigh<__bf16, 128><<<grid, 256, 0, s>>>(W);
    else hck::k_weigh<_Float16, 128><<<grid, 256, 0, s>>>(W);
  } else {
    if (type == HCK_BF16) hck::k_weigh<__bf16, 64><<<grid, 256, 0, s>>>(W);
    else hck::k_weigh<_Float16, 64><<<grid, 256, 0, s>>>(W);
  }
  HCK_CHECK_LAUNCH();
  return HCK_OK;
}
