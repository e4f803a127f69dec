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
  float* parts;  // with more than one: [part][seq][head][place]
  int64_t prior_seq, prior_head;
  int prior_places, split, units;  // split: parts that the rows of 256 tokens are cut into; units: of a wave, with few rows
  float scale2, rest;  // scale log2 e in 32 bits, and what its rounding left over, divided by scale
};

// A row's share of the exponents: what comes off, in units of log 2, and a factor, near 1 for scores of ordinary size, for what
// rounding took from that and from scale log2 e (counted where the score is the row's lse, near which weights are large).  Its
// exponent is within 45 up to |lse| = 2^28, and kept within 64 beyond, where half a step of lse itself is e^16 or more: so
// that no row's share is negative, or 0 times an infinity.
struct RowTerm {
  float off, factor;
  int seen;
};
__device__ __forceinline__ float row_lse(const WeighArgs& W, const Rows& R, int h, int row) {
  return W.row_lse[(int64_t)(R.q0 + row / W.a.group) * ((int64_t)W.a.heads * W.a.group) + h * W.a.group + row % W.a.group];
}
__device__ __forceinline__ RowTerm row_term(const WeighArgs& W, const Rows& R, int row, float lse) {
  RowTerm r = {lse * kLog2e, 1.f, lse == -INFINITY ? 0 : R.seen(W.a, row)};  // a row of -inf gave nothing
  if (fabsf(lse) < INFINITY) {
    const float low = __builtin_fmaf(lse, kLog2e, -r.off) + lse * 1.9259629911266174e-8f;  // (log2 e in two parts)
    r.factor = __builtin_amdgcn_exp2f(fminf(fmaxf(lse * W.rest - low, -64.f), 64.f));
  }
  return r;
}

// Sums over pairs of lanes LANES apart, of a in the first of each two groups of so many lanes, of b in the second.
template <int LANES>
__device__ __forceinline__ float beside(float a, float b) {
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
  if constexpr (LANES == 32) {
    const auto p = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
  } else {
    const auto p = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
}

// Up to 16 rows: a wave takes units of 64 tokens in turn, the next one's keys in flight, with the rows' operands and terms in its
// registers throughout.  The product's 16 rows are the left operand, so a lane has one token of each 16 and four of its rows.
// Bound by the keys' bytes: 32 histories of 2000 to 24576 tokens, 8 key heads of 128, 178 MB with the weights, 40 us, 4.4 TB/s; with
// one unit a wave, and nothing in flight behind the lookup of its page, 82 us, with loads through the caches 56 where these took 53.
template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void k_weigh_few(WeighArgs W) {
  using L = Kv4<D>;
  constexpr int kSteps = D / 32;
  constexpr bool kHalf = __is_same(T, _Float16);
  const AttendArgs& A = W.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % A.heads, b = blockIdx.y;
  int u = blockIdx.x / A.heads * (kWaves * W.units) + wave;
  const int u1 = min(u + kWaves * W.units, 2 * A.cols);
  if (u >= u1) return;
  const int* table = A.table + b * A.table_stride;
  int pg = table[u >> 1];  // (a column of the table, whatever the length)
  const Rows R(A, b);
  const int line = b * A.heads + h;
  float* to = W.weights + (int64_t)line * A.cols * kPageTokens + lane;
  const float* prior = W.prior + b * W.prior_seq + h * W.prior_head + lane;

  typedef uint32_t words __attribute__((ext_vector_type(kSteps)));
  words codes[4];
  uint32_t scales = 0;
  float old = 0.f;
  auto there = [&](int pg) { return pg >= 0 && pg < A.pages; };
  auto load = [&](int u, int pg) {  // unit u, of a page that is page 0 where it is none
    const uint8_t* page = A.pool + ((int64_t)(there(pg) ? pg : 0) * A.heads + h) * L::kBytes;
    const uint8_t* at = page + (u & 1) * (32 * D) + lane * (D / 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) codes[i] = __builtin_nontemporal_load(reinterpret_cast<const words*>(at + i * (8 * D)));
    scales = *reinterpret_cast<const uint32_t*>(page + L::kKScales + (u & 1) * (64 * L::kRuns) + g * (D / 4) / kRun * 64 + m * 4);
    const int j = u * kUnit + lane;
    old = W.prior && j < W.prior_places ? prior[u * kUnit] : 0.f;
  };
  if (u * kUnit >= R.length) {
    for (; u < u1; u += kWaves) to[u * kUnit] = 0.f;
    return;
  }
  pg = __builtin_amdgcn_readfirstlane(pg);
  int next = u + kWaves < u1 ? table[(u + kWaves) >> 1] : 0;
  load(u, pg);

  bf16x8 q[kSteps], rest[kSteps];
  u32x4 raw[kSteps] = {};
  float lse[4] = {};
  if (R.rows > 0) {  // (a lane without a row has the first one's values, which see nothing; loads under a condition each would wait each)
    const int row = m < R.rows ? m : 0;
    const T* qp = (const T*)A.q + (R.q0 + row / A.group) * A.q_ts + (int64_t)(h * A.group + row % A.group) * A.q_hs + g * (D / 4);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) raw[s] = reinterpret_cast<const Loose16*>(qp + 8 * s)->v;
#pragma unroll
    for (int r = 0; r < 4; ++r) lse[r] = row_lse(W, R, h, min(4 * g + r, R.rows - 1));
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) query_parts<T>(raw[s], q[s], rest[s]);
  RowTerm t[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) t[r] = row_term(W, R, 4 * g + r, 4 * g + r < R.rows ? lse[r] : -INFINITY);

  for (; u < u1; u += kWaves) {
    const int here = u * kUnit;
    if (here >= R.length) {
      to[here] = 0.f;
      continue;
    }
    const bool seen = there(pg);
    words now[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) now[i] = codes[i];
    const uint32_t bytes = scales;
    float total = old;
    pg = __builtin_amdgcn_readfirstlane(next);
    if (u + 2 * kWaves < u1) next = table[(u + 2 * kWaves) >> 1];
    if (u + kWaves < u1 && here + kWaves * kUnit < R.length) load(u + kWaves, pg);
    if (seen) {
      float part[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t byte = (bytes >> (8 * i)) & 0xffu;
        const float sc = byte == kNanByte ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < kSteps; ++d) {
          const bf16x8 k = operand(cvt<0>(now[i][d], sc), cvt<1>(now[i][d], sc), cvt<2>(now[i][d], sc), cvt<3>(now[i][d], sc));
          s = mfma(q[d], k, s);
          if constexpr (kHalf) s = mfma(rest[d], k, s);
        }
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], W.scale2, -t[r].off));
          sum = __builtin_fmaf(here + 16 * i + m < t[r].seen ? p : 0.f, t[r].factor, sum);
        }
        part[i] = sum;
      }
      // over the four lanes of a token, and lane (m, g) gets token 16 g + m: the halves' sums of two 16s side by side, then the 16s'
      total += beside<16>(beside<32>(part[0], part[2]), beside<32>(part[1], part[3]));
    }
    to[here] = here + lane < R.length ? total : 0.f;
  }
}

// Many rows: the keys of 64 tokens stay in a wave's registers as the right operand, 32 tokens to a product, and the rows pass
// by, 64 at a time through LDS for the four waves of 256 tokens.  A lane has one token (two in all) and 16 of 32 rows, so its
// sums need no other lane until the end; what comes off a row's scores is read from LDS, four rows at a time.  Rows that come
// in parts (few tokens, many rows) leave sums of their own, which k_weigh_join adds in order.
//
// A sum over many rows is taken over 64 of them and then over those, with what each addition of the latter loses carried on.
//
// What bounds it: per 64 rows and 64 tokens 32 matrix instructions (1024 cycles) and 192 vector ones, 64 of them exponentials (1024), and a
// barrier.  4096 tokens and queries, 32 query heads over 8 key heads of 128: 70 GFLOP in 88 us and 5 for the join, 750 TFLOP/s.
constexpr int kStage = 64, kBlock = kUnit * kWaves;  // rows at a time, tokens of a workgroup
constexpr int kMostRows = INT32_MAX - 256;            // of a sequence and key head: whole stages are counted in 31 bits

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void k_weigh_many(WeighArgs W) {
  using L = Kv4<D>;
  constexpr int kSteps = D / 16, kPieces = D / 8, kEach = kStage * kPieces / (64 * kWaves), kApart = 64 * kWaves / kPieces;
  constexpr bool kHalf = __is_same(T, _Float16);
  constexpr int kParts = kHalf ? 2 : 1;
  __shared__ u32x4 s_q[2][kParts][kStage * kPieces];
  __shared__ alignas(16) float s_off[2][kStage], s_factor[2][kStage];
  __shared__ alignas(16) int s_seen[2][kStage];
  __shared__ int s_least[2][2];
  const AttendArgs& A = W.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, half = lane >> 5;
  // (the tokens that most rows see first)
  const int h = blockIdx.x % A.heads, part = blockIdx.x / A.heads % W.split, block = blockIdx.x / A.heads / W.split, b = blockIdx.y;
  const Rows R(A, b);
  const int first = block * kBlock, here = first + wave * kUnit;
  const int64_t width = (int64_t)A.cols * kPageTokens, line = (int64_t)b * A.heads + h;
  if (first >= R.length) {
    const int j = first + threadIdx.x;
    if (W.split == 1 && j < width) W.weights[line * width + j] = 0.f;
    return;
  }
  int pg = -1;
  if (here < R.length) pg = A.table[b * A.table_stride + here / kPageTokens];
  const bool there = pg >= 0 && pg < A.pages;

  bf16x8 k[2][kSteps];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int t = (here & (kPageTokens - 1)) + 32 * x + n;  // within the page
    const uint8_t* page = A.pool + ((int64_t)(there ? pg : 0) * A.heads + h) * L::kBytes;
#pragma unroll
    for (int p = 0; p < 2; ++p) {  // dims (2 p + half) D / 4 ..
      typedef uint32_t words __attribute__((ext_vector_type(D / 32)));
      const words c = *reinterpret_cast<const words*>(page + L::key_code(t, (2 * p + half) * (D / 4)));
      const int byte = page[L::key_scale(t, (2 * p + half) * (D / 4) / kRun)];
      const float sc = __uint_as_float(byte == kNanByte ? 0x7fc00000u : (uint32_t)byte << 23);
#pragma unroll
      for (int s = 0; s < D / 32; ++s)
        k[x][p * (D / 32) + s] = operand(cvt<0>(c[s], sc), cvt<1>(c[s], sc), cvt<2>(c[s], sc), cvt<3>(c[s], sc));
    }
  }

  // the part's rows, from the first query that sees one of the workgroup's tokens
  const int skip = A.causal ? (int)min((int64_t)R.rows, (int64_t)max(0, first - (R.length - R.nq)) * A.group) / kStage * kStage : 0;
  const int stages = (R.rows - skip + kStage - 1) / kStage, each = (stages + W.split - 1) / W.split;
  const int from = skip + min(part * each, stages) * kStage, to = min(R.rows, skip + min((part + 1) * each, stages) * kStage);

  // A thread brings pieces of rows kApart apart; row = query * group + head goes on by additions.
  const int piece = threadIdx.x % kPieces, row0 = threadIdx.x / kPieces;
  int qo = (from + row0) % A.group;
  const T* next = (const T*)A.q + (R.q0 + (int64_t)((from + row0) / A.group)) * A.q_ts + (int64_t)(h * A.group + qo) * A.q_hs + piece * 8;
  const int step_o = kApart % A.group;
  const int64_t step = (kApart / A.group) * A.q_ts + step_o * A.q_hs, wrap = A.q_ts - A.group * A.q_hs;
  u32x4 raw[kEach];
  auto bring = [&](int at) {  // rows at .. at + kStage - 1
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      raw[j] = u32x4{0, 0, 0, 0};
      if (at + row0 + j * kApart < to) raw[j] = reinterpret_cast<const Loose16*>(next)->v;
      next += step, qo += step_o;
      if (qo >= A.group) qo -= A.group, next += wrap;
    }
  };
  auto place = [](int row, int p) { return row * kPieces + (p ^ (D == 128 ? row & 15 : (row >> 1) & 7)); };
  auto put = [&](int buf) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int at = place(row0 + j * kApart, piece);
      if constexpr (kHalf) {
        bf16x8 head, rest;
        query_parts<T>(raw[j], head, rest);
        s_q[buf][0][at] = __builtin_bit_cast(u32x4, head);
        s_q[buf][kParts - 1][at] = __builtin_bit_cast(u32x4, rest);
      } else {
        s_q[buf][0][at] = raw[j];
      }
    }
  };
  float lse = 0.f;
  auto terms = [&](int buf, int at) {  // one wave, whose lanes have the rows' lse
    const RowTerm t = row_term(W, R, at + lane, at + lane < to ? lse : -INFINITY);
    const int seen = at + lane < to ? t.seen : 0;
    s_off[buf][lane] = t.off, s_factor[buf][lane] = t.factor, s_seen[buf][lane] = seen;
    int least = seen;
    for (int d = 1; d < 32; d *= 2) least = min(least, __shfl_xor(least, d));
    if (n == 0) s_least[buf][half] = least;
  };

  // The sums over 64 rows.  PARTLY: some of them do not see some of the wave's tokens.
  float now[2];
  auto stage = [&](int buf, auto PARTLY) {
    now[0] = now[1] = 0.f;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      f32x16 c[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) c[0][i] = c[1][i] = 0.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int at = place(32 * y + n, (2 * (s / (D / 32)) + half) * (D / 32) + s % (D / 32));
        const bf16x8 q = __builtin_bit_cast(bf16x8, s_q[buf][0][at]);
#pragma unroll
        for (int x = 0; x < 2; ++x) c[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q, k[x][s], c[x], 0, 0, 0);
        if constexpr (kHalf) {
          const bf16x8 r = __builtin_bit_cast(bf16x8, s_q[buf][kParts - 1][at]);
#pragma unroll
          for (int x = 0; x < 2; ++x) c[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(r, k[x][s], c[x], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // rows 8 i + 4 half ..
        const int r = 32 * y + 8 * i + 4 * half;
        const f32x4 off = *reinterpret_cast<const f32x4*>(&s_off[buf][r]);
        const f32x4 factor = *reinterpret_cast<const f32x4*>(&s_factor[buf][r]);
        typedef int i32x4 __attribute__((ext_vector_type(4)));
        i32x4 seen;
        if constexpr (decltype(PARTLY)::value) seen = *reinterpret_cast<const i32x4*>(&s_seen[buf][r]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(c[x][4 * i + e], W.scale2, -off[e]));
            if constexpr (decltype(PARTLY)::value) p = here + 32 * x + n < seen[e] ? p : 0.f;
            now[x] = __builtin_fmaf(p, factor[e], now[x]);
          }
      }
    }
  };

  float sum[2] = {0.f, 0.f}, lost[2] = {0.f, 0.f};
  if (from < to) {
    bring(from);
    if (wave == 0) lse = row_lse(W, R, h, min(from + lane, R.rows - 1));
    put(0);
    if (wave == 0) terms(0, from);
  }
  __syncthreads();
  for (int at = from, buf = 0; at < to; at += kStage, buf ^= 1) {
    const bool more = at + kStage < to, mine = wave == ((at / kStage) & (kWaves - 1));
    if (more) {
      bring(at + kStage);
      if (mine) lse = row_lse(W, R, h, min(at + kStage + lane, R.rows - 1));
    }
    if (there) {
      if (here + kUnit <= __builtin_amdgcn_readfirstlane(min(s_least[buf][0], s_least[buf][1]))) stage(buf, std::false_type());
      else stage(buf, std::true_type());
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float add = now[x] - lost[x], all = sum[x] + add;
        lost[x] = fabsf(all) < INFINITY ? (all - sum[x]) - add : 0.f;
        sum[x] = all;
      }
    }
    if (more) {
      put(buf ^ 1);
      if (mine) terms(buf ^ 1, at + kStage);
    }
    __syncthreads();
  }
  const float s0 = over_half(sum[0], [](float a, float c) { return a + c; });
  const float s1 = over_half(sum[1], [](float a, float c) { return a + c; });
  float total = half ? s1 : s0;
  const int mine = here + lane;
  if (mine >= width) return;
  if (W.split > 1) {
    W.parts[((int64_t)part * A.seqs * A.heads + line) * width + mine] = total;
    return;
  }
  if (mine >= R.length) total = 0.f;
  else if (W.prior && mine < W.prior_places) total += W.prior[b * W.prior_seq + h * W.prior_head + mine];
  W.weights[line * width + mine] = total;
}

// The parts' sums, what was there before, and zeros behind the end.
__global__ __launch_bounds__(256) void k_weigh_join(WeighArgs W) {
  const AttendArgs& A = W.a;
  const int h = blockIdx.y, b = blockIdx.z, j = blockIdx.x * 256 + threadIdx.x;
  const int64_t width = (int64_t)A.cols * kPageTokens, line = (int64_t)b * A.heads + h;
  if (j >= width) return;
  float total = 0.f;
  if (j < min((int64_t)max(A.lengths[b], 0), width)) {
    for (int p = 0; p < W.split; ++p) total += W.parts[((int64_t)p * A.seqs * A.heads + line) * width + j];
    if (W.prior && j < W.prior_places) total += W.prior[b * W.prior_seq + h * W.prior_head + j];
  }
  W.weights[line * width + j] = total;
}

// How a call is run, from what the host knows of it.
struct WeighWay {
  bool many;
  int split, units;
  int64_t blocks;
  WeighWay(int64_t seqs, int heads, int group, int most, int cols) {
    const int64_t rows = (int64_t)most * group;
    many = rows > kFew;
    // More units a wave share the rows' loading, fewer even the work out (32 histories of 2000 to 24576 tokens: 2 58 us, 3 52,
    // 4 51, 8 53); no more than leave 8 waves for every SIMD.
    units = (int)std::min<int64_t>(4, std::max<int64_t>(1, (int64_t)cols * 2 * heads * seqs / (32 * kComputeUnits)));
    blocks = ((int64_t)cols * kPageTokens + kBlock - 1) / kBlock;
    // Parts of four stages at the least, and workgroups that get shorter from the first tokens on, for
    // every compute unit to end at about the same time (4096 tokens and queries, 32/8 heads: 93 us with 9 parts or 17, 104 with 33,
    // 115 at the best with parts of the same length).
    split = many ? (int)std::min<int64_t>((rows + 4 * kStage - 1) / (4 * kStage), (4 * kComputeUnits) / std::max<int64_t>(1, blocks * heads * seqs) + 1) : 1;
  }
  size_t bytes(int64_t seqs, int heads, int cols) const {
    return split > 1 ? (size_t)split * seqs * heads * cols * kPageTokens * sizeof(float) : 0;
  }
};

template <typename T, int D>
int launch(const WeighArgs& W, const WeighWay& way, hipStream_t s) {
  const AttendArgs& A = W.a;
  if (!way.many) {
    const int64_t groups = ((int64_t)A.cols * 2 + kWaves * W.units - 1) / (kWaves * W.units) * A.heads;
    if (!fits_grid(groups, 64 * kWaves)) return HCK_ERR_ARG;
    k_weigh_few<T, D><<<dim3((unsigned)groups, A.seqs), 64 * kWaves, 0, s>>>(W);
  } else {
    const int64_t groups = way.blocks * way.split * A.heads;
    if (!fits_grid(groups, 64 * kWaves)) return HCK_ERR_ARG;
    k_weigh_many<T, D><<<dim3((unsigned)groups, A.seqs), 64 * kWaves, 0, s>>>(W);
  }
  HCK_CHECK_LAUNCH();
  if (way.split > 1) {
    k_weigh_join<<<dim3((unsigned)(A.cols * (kPageTokens / 128) + 1) / 2, A.heads, A.seqs), 256, 0, s>>>(W);
    HCK_CHECK_LAUNCH();
  }
  return HCK_OK;
}

}  // namespace
}  // namespace hck

extern "C" size_t hck_kv4_weigh_workspace_bytes(int64_t tokens, int seqs, int kv_heads, int group, int most,
                                                int table_columns) {
  if (tokens <= 0 || seqs < 1 || seqs > 65535 || kv_heads < 1 || kv_heads > 65535 || group < 1 || most < 0 ||
      table_columns < 1 || table_columns >= 1 << 23 || (int64_t)most * group > hck::kMostRows || (int64_t)seqs * kv_heads > INT32_MAX)
    return 0;
  return hck::WeighWay(seqs, kv_heads, group, (int)std::min<int64_t>(most, tokens), table_columns).bytes(seqs, kv_heads, table_columns);
}

extern "C" int hck_kv4_weigh(const void* pool, int64_t pages, int kv_heads, int head_dim, int type, const void* queries,
                             int64_t tokens, int group, int64_t q_token_stride, int64_t q_head_stride, const int32_t* table,
                             int64_t table_stride, int table_columns, const int32_t* lengths, const int32_t* starts, int seqs,
                             int most, int causal, double scale, const float* lse, const float* prior, int64_t prior_seq_stride,
                             int64_t prior_head_stride, int prior_places, float* weights, void* workspace, size_t workspace_bytes, void* stream) {
  if (hck::kv4_bytes(head_dim) == 0 || (type != HCK_BF16 && type != HCK_F16)) return HCK_ERR_UNSUPPORTED;
  if (!pool || pages < 1 || kv_heads < 1 || kv_heads > 65535 || tokens < 0 || tokens > INT32_MAX || group < 1 || seqs < 0 ||
      seqs > 65535 || most < 0 || table_columns < 0 || table_columns >= 1 << 23 || prior_places < 0 ||
      !((float)scale > 0.f && scale <= 0x1p126) || (int64_t)most * group > hck::kMostRows || (int64_t)kv_heads * group > INT32_MAX ||
      (int64_t)seqs * kv_heads > INT32_MAX)
    return HCK_ERR_ARG;
  if (!starts && tokens != seqs) return HCK_ERR_ARG;
  if (seqs == 0 || table_columns == 0) return HCK_OK;
  if (!table || !lengths || !weights || (tokens && (!queries || !lse)) || (prior_places && !prior)) return HCK_ERR_ARG;
  hck::WeighArgs W = {};
  hck::AttendArgs& A = W.a;
  A.pool = (const uint8_t*)pool, A.q = queries, A.table = table, A.lengths = lengths, A.starts = starts;
  A.q_ts = q_token_stride, A.q_hs = q_head_stride, A.tokens = tokens, A.pages = pages, A.table_stride = table_stride;
  A.cols = table_columns, A.heads = kv_heads, A.group = group, A.causal = causal != 0, A.seqs = seqs;
  A.tiles = (int)std::min<int64_t>(most, tokens), A.size = group;
  W.row_lse = lse, W.prior = prior, W.weights = weights, W.prior_seq = prior_seq_stride, W.prior_head = prior_head_stride;
  W.prior_places = prior ? prior_places : 0;
  const double scale2 = scale * 1.4426950408889634;
  W.scale2 = (float)scale2, W.rest = (float)((scale2 - W.scale2) / scale);
  const hck::WeighWay way(seqs, kv_heads, group, (int)std::min<int64_t>(most, tokens), table_columns);
  const size_t need = tokens ? way.bytes(seqs, kv_heads, table_columns) : 0;
  if (need && (!workspace || workspace_bytes < need)) return HCK_ERR_WORKSPACE;
  W.parts = (float*)workspace, W.split = way.split, W.units = way.units;
  hipStream_t s = (hipStream_t)stream;
  if (head_dim == 128) return type == HCK_BF16 ? hck::launch<__bf16, 128>(W, way, s) : hck::launch<_Float16, 128>(W, way, s);
  return type == HCK_BF16 ? hck::launch<__bf16, 64>(W, way, s) : hck::launch<_Float16, 64>(W, way, s);
}
