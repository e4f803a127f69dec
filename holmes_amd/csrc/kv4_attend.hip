// Attention over 4-bit pages.
//
// For a query row (a query token and one of the `group` query heads that share a key head) and the
// tokens t that it sees:  s_t = scale * q.k_t,  m = max s_t,  l = sum exp(s_t - m),
// out = sum exp(s_t - m) v_t / l,  lse = m + log l, in one pass over the cache with the running m and
// l of every row.  Both products run on the matrix cores, transposed: S^T = K Q^T leaves a lane with
// one row's scores of 4 tokens of every 16-token tile, and O^T = V^T P^T takes exactly those as its
// right operand (the order of the tokens inside a product is free), so the probabilities never leave
// the lane.
//
// Roundings: codes times scales are exact in bf16 (two significant bits), and so is a bf16 query; an
// fp16 query goes in as two bf16 parts (16 bits).  Scores, maxima, sums and outputs are held in 32
// bits.  The probabilities go in as two bf16 parts as well, which leaves 2^-17 of each, far below the
// rounding of the output; the sum l takes the unrounded ones.
#include "kv4.hpp"

#include "../../include/holmes_ckks.h"
#include "internal.hpp"

namespace hck {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kUnit = 64;   // tokens that a wave takes at a time: half a page
constexpr int kWaves = 4;
// Exponentials are taken times 2^24, so that those from 2^-126 to 2^-150 of a row's largest, which the
// exponential instruction gives as 0, still count where every larger one meets a value of 0.  Sums then
// stay finite for values up to 2^103 over the number of tokens.
constexpr float kLift = 24.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttendArgs {
  const uint8_t* pool;
  const void* q;
  const int* table;
  const int* lengths;
  const int* starts;   // null: sequence b has the one query b
  void* out;
  float *lse, *low, *high;  // [token][query head]; low, high nullable
  float* part;         // with splits > 1: [row][split] of (m, l, low, 0), then [row][split][D] of sums
  long long q_ts, q_hs, tokens, pages;
  long long table_stride;
  int cols, heads, group, splits, causal;
  float scale;
};

// 16 bytes from an address that is a multiple of the elements' two bytes only.
struct __attribute__((packed, aligned(2))) Loose16 {
  u32x4 v;
};

__device__ __forceinline__ float scale_of(uint32_t word, int byte) {
  return __uint_as_float(((word >> (8 * byte)) & 0xffu) << 23);
}

template <int B>
__device__ __forceinline__ uint32_t cvt(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}

__device__ __forceinline__ bf16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(bf16x8, u32x4{a, b, c, d});
}

__device__ __forceinline__ uint32_t pack(float a, float b) {
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

__device__ __forceinline__ bool has_nan(uint32_t w) {  // a byte of 255 among the four
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u;
}

// What a lane holds of 64 tokens: lane (m, g) = (lane % 16, lane / 16) has D / 4 dims from D / 4 * g of
// token m of every 16-token tile, and D / 16 dims from D / 16 * m of the 8 tokens (g, j) of each 32.
template <int D>
struct Unit {
  uint32_t k[4][D / 32], ks, v[2][D / 16], vs[2][2];
  __device__ __forceinline__ void load(const uint8_t* page, int half, int m, int g) {
    using L = Kv4<D>;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* p = page + (64 * half + 16 * i + m) * (D / 2) + g * (D / 8);
      if constexpr (D == 128) *reinterpret_cast<u32x4*>(k[i]) = *reinterpret_cast<const u32x4*>(p);
      else *reinterpret_cast<u32x2*>(k[i]) = *reinterpret_cast<const u32x2*>(p);
    }
    ks = *reinterpret_cast<const uint32_t*>(page + L::key_scale(64 * half + m, g * (D / 4) / kRun));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* p = page + L::kVCodes + (2 * half + i) * (16 * D) + (g * 16 + m) * (D / 4);
#pragma unroll
      for (int w = 0; w < D / 64; ++w)
        reinterpret_cast<u32x4*>(v[i])[w] = reinterpret_cast<const u32x4*>(p)[w];
      *reinterpret_cast<u32x2*>(vs[i]) = *reinterpret_cast<const u32x2*>(
          page + L::kVScales + (2 * half + i) * (32 * L::kRuns) + (g * L::kRuns + m * L::kDpl / kRun) * 8);
    }
  }
  // The left operand of step s of S^T = K Q^T for tile i: dims D / 4 g + 8 s .. + 7 of the lane's token.
  __device__ __forceinline__ bf16x8 key(int i, int s, float scale) const {
    const uint32_t w = k[i][s];
    return operand(cvt<0>(w, scale), cvt<1>(w, scale), cvt<2>(w, scale), cvt<3>(w, scale));
  }
  // The left operands of O^T = V^T P^T over block i: dims 2 b and 2 b + 1 of the lane's D / 16, 8 tokens.
  template <int B>
  __device__ __forceinline__ void value(int i, const float* scale, bf16x8& even, bf16x8& odd) const {
    uint32_t x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (D == 128) x[j] = cvt<B>(v[i][j], scale[j]);
      else x[j] = (j & 1) ? cvt<(B & 1) + 2>(v[i][j / 2], scale[j]) : cvt<(B & 1)>(v[i][j / 2], scale[j]);
    }
    uint32_t e[4], o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      e[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
      o[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
    }
    even = operand(e[0], e[1], e[2], e[3]);
    odd = operand(o[0], o[1], o[2], o[3]);
  }
};

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A reduction over the four lanes that share a row.
template <typename F>
__device__ __forceinline__ float over_g(float x, F f) {
  x = f(x, __shfl_xor(x, 16));
  return f(x, __shfl_xor(x, 32));
}

__device__ __forceinline__ float fmax2(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float fmin2(float a, float b) { return fminf(a, b); }

// Sums are taken against the whole number at or above a row's running maximum, so that going over to
// another reference is an exact power of two.  The factor of sums against the maximum a, now against b:
// 1 where nothing changed, also while nothing was seen (both -inf).
__device__ __forceinline__ float rebase(float a, float b) {
  return a == b ? 1.f : __builtin_ldexpf(1.f, (int)(__builtin_ceilf(a) - __builtin_ceilf(b)));
}
__device__ __forceinline__ float reference(float m) { return fabsf(m) == INFINITY ? 0.f : __builtin_ceilf(m); }
// log2 of a row's sum, against its reference.
__device__ __forceinline__ float log2_sum(float m, float l) {
  return fabsf(m) == INFINITY ? m + l : __builtin_ceilf(m) + (__builtin_amdgcn_logf(l) - kLift);
}

// One workgroup: 16 rows of one key head, a share of their tokens; its waves take units in turn.
template <typename T, int D, bool RANGE>
__global__ __launch_bounds__(64 * kWaves) void k_attend(AttendArgs A) {
  using L = Kv4<D>;
  constexpr int kSteps = D / 32, kDpl = L::kDpl;
  constexpr bool kHalf = __is_same(T, _Float16);
  __shared__ float s_m[kWaves][16], s_l[kWaves][16], s_low[kWaves][16];
  __shared__ float s_o[kWaves][16][D + 4];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % A.splits, tile = blockIdx.x / A.splits, h = blockIdx.y, b = blockIdx.z;
  long long q0 = b, q1 = b + 1;
  if (A.starts) q0 = A.starts[b], q1 = A.starts[b + 1];
  q0 = max(q0, 0ll);
  q1 = min(q1, A.tokens);
  const int nq = (int)max(q1 - q0, 0ll);
  const int rows = nq * A.group;
  if (tile * 16 >= rows) return;
  const int length = (int)min((long long)max(A.lengths[b], 0), (long long)A.cols * kPageTokens);
  const int row = tile * 16 + m;
  const bool live = row < rows;
  const int qi = live ? row / A.group : 0, qo = live ? row % A.group : 0;
  const int seen = !live ? 0 : A.causal ? max(0, min(length, length - nq + qi + 1)) : length;
  const int last = min(tile * 16 + 15, rows - 1) / A.group;
  const int most = A.causal ? max(0, min(length, length - nq + last + 1)) : length;
  const int units = (most + kUnit - 1) / kUnit;
  const int u0 = (int)((long long)units * split / A.splits), u1 = (int)((long long)units * (split + 1) / A.splits);

  // the lane's part of its row's query: dims D / 4 g + 8 s .. + 7 of step s
  bf16x8 qh[kSteps], ql[kSteps];
  const T* qp = (const T*)A.q + (q0 + qi) * A.q_ts + (long long)(h * A.group + qo) * A.q_hs + g * (D / 4);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    u32x4 raw = {0, 0, 0, 0};
    if (live) raw = reinterpret_cast<const Loose16*>(qp + 8 * s)->v;
    if constexpr (kHalf) {
      typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
      const f16x8 x = __builtin_bit_cast(f16x8, raw);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        qh[s][k] = (__bf16)(float)x[k];
        ql[s][k] = (__bf16)((float)x[k] - (float)qh[s][k]);
      }
    } else {
      qh[s] = __builtin_bit_cast(bf16x8, raw);
    }
  }

  f32x4 acc[kDpl];
#pragma unroll
  for (int i = 0; i < kDpl; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f, low = INFINITY;
  const float scale2 = A.scale * kLog2e;

  for (int u = u0 + wave; u < u1; u += kWaves) {
    const int pg = A.table[b * A.table_stride + (u >> 1)];
    if (pg < 0 || pg >= A.pages) continue;  // no such page: its tokens are not there
    Unit<D> x;
    x.load(A.pool + ((long long)pg * A.heads + h) * L::kBytes, u & 1, m, g);

    float t[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 c = {0.f, 0.f, 0.f, 0.f};
      const uint32_t byte = (x.ks >> (8 * i)) & 0xffu;
      const float sc = __uint_as_float(byte << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const bf16x8 kk = x.key(i, s, byte == kNanByte ? __uint_as_float(0x7fc00000u) : sc);
        c = mfma(kk, qh[s], c);
        if constexpr (kHalf) c = mfma(kk, ql[s], c);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) t[i][k] = c[k] * scale2;
    }
    const int base = u * kUnit + 4 * g;
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool see = base + 16 * i + k < seen;
        if constexpr (RANGE) low = see ? fminf(low, t[i][k]) : low;
        t[i][k] = see ? t[i][k] : -INFINITY;
        mx = fmaxf(mx, t[i][k]);
      }
    mx = fmaxf(top, over_g(mx, fmax2));
    const float f = rebase(top, mx);
    top = mx;
    const float ref = reference(mx) - kLift;
    sum *= f;
#pragma unroll
    for (int i = 0; i < kDpl; ++i) acc[i] *= f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        t[i][k] = __builtin_amdgcn_exp2f(t[i][k] - ref);
        sum += t[i][k];
      }

#pragma unroll
    for (int i = 0; i < 2; ++i) {
      bf16x8 ph, pl;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float p = t[2 * i + (k >> 2)][k & 3];
        ph[k] = (__bf16)p;
        pl[k] = (__bf16)(p - (float)ph[k]);
      }
      uint32_t vs[2] = {x.vs[i][0], x.vs[i][1]};
      float sc[8];
      // A run of NaN must reach the rows that see its token, and no other: 0 * NaN is NaN.  It is taken
      // as zeros here, and counted for the rows that see it by a product of truth values.
      const bool odd = __any(has_nan(vs[0]) || has_nan(vs[1]));
      if (odd) {
        bf16x8 bad, see;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool is = ((vs[k >> 2] >> (8 * (k & 3))) & 0xffu) == kNanByte;
          bad[k] = (__bf16)(is ? 1.f : 0.f);
          see[k] = (__bf16)(base + 32 * i + 16 * (k >> 2) + (k & 3) < seen ? 1.f : 0.f);
          if (is) vs[k >> 2] &= ~(0xffu << (8 * (k & 3)));
        }
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const f32x4 n = mfma(bad, see, zero);
#pragma unroll
        for (int d = 0; d < kDpl; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n[k] > 0.f) acc[d][k] = __uint_as_float(0x7fc00000u);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sc[k] = scale_of(vs[k >> 2], k & 3);
      bf16x8 e, o;
      auto step = [&](auto B) {
        constexpr int kB = decltype(B)::value;
        x.template value<kB>(i, sc, e, o);
        acc[2 * kB] = mfma(e, ph, acc[2 * kB]);
        acc[2 * kB] = mfma(e, pl, acc[2 * kB]);
        acc[2 * kB + 1] = mfma(o, ph, acc[2 * kB + 1]);
        acc[2 * kB + 1] = mfma(o, pl, acc[2 * kB + 1]);
      };
      step(std::integral_constant<int, 0>());
      step(std::integral_constant<int, 1>());
      if constexpr (kDpl == 8) {
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
      }
    }
  }

  // join the waves: lane (m, g) holds dims D / 4 g + kDpl i + d of row m in acc[d][i]
  sum = over_g(sum, [](float a, float c) { return a + c; });
  if constexpr (RANGE) low = over_g(low, fmin2);
  if (g == 0) s_m[wave][m] = top, s_l[wave][m] = sum, s_low[wave][m] = low;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int d = 0; d < kDpl; ++d) s_o[wave][m][g * (D / 4) + kDpl * i + d] = acc[d][i];
  __syncthreads();
  constexpr int kCols = D / 16;  // dims of a thread: 16 threads to a row
  const int r = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * kCols;
  if (tile * 16 + r >= rows) return;
  float mm = -INFINITY, ll = 0.f, lo = INFINITY, o[kCols];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, s_m[w][r]);
#pragma unroll
  for (int c = 0; c < kCols; ++c) o[c] = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float f = rebase(s_m[w][r], mm);
    ll += f * s_l[w][r];
    lo = fminf(lo, s_low[w][r]);
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c] += f * s_o[w][r][c0 + c];
  }
  const int qr = (tile * 16 + r) / A.group, qc = (tile * 16 + r) % A.group;
  const long long at = (q0 + qr) * (long long)(A.heads * A.group) + h * A.group + qc;
  if (A.splits > 1) {
    float* stat = A.part + (at * A.splits + split) * 4;
    float* sums = A.part + A.tokens * A.heads * A.group * (long long)A.splits * 4 + (at * A.splits + split) * D + c0;
    if (c0 == 0) stat[0] = mm, stat[1] = ll, stat[2] = lo;
#pragma unroll
    for (int c = 0; c < kCols; ++c) sums[c] = o[c];
    return;
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  T* to = (T*)A.out + at * D + c0;
#pragma unroll
  for (int c = 0; c < kCols; ++c) to[c] = (T)(o[c] * inv);
  if (c0 == 0) {
    const bool bad = ll != ll;
    A.lse[at] = log2_sum(mm, ll) * kLn2;
    if constexpr (RANGE) A.low[at] = bad ? ll : lo * kLn2, A.high[at] = bad ? ll : mm * kLn2;
  }
}

// Joins the splits of a row: one wave a row.
template <typename T, int D, bool RANGE>
__global__ __launch_bounds__(256) void k_join(AttendArgs A) {
  const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), all = A.tokens * A.heads * A.group;
  const int lane = threadIdx.x & 63;
  if (at >= all) return;
  const float* stat = A.part + at * A.splits * 4;
  const float* sums = A.part + all * A.splits * 4 + at * A.splits * D;
  float mm = -INFINITY, ll = 0.f, lo = INFINITY, o[D / 64];
  for (int s = 0; s < A.splits; ++s) mm = fmaxf(mm, stat[4 * s]);
#pragma unroll
  for (int c = 0; c < D / 64; ++c) o[c] = 0.f;
  for (int s = 0; s < A.splits; ++s) {
    const float f = rebase(stat[4 * s], mm);
    ll += f * stat[4 * s + 1];
    lo = fminf(lo, stat[4 * s + 2]);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) o[c] += f * sums[s * D + c * 64 + lane];
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  T* to = (T*)A.out + at * D;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) to[c * 64 + lane] = (T)(o[c] * inv);
  if (lane == 0) {
    const bool bad = ll != ll;
    A.lse[at] = log2_sum(mm, ll) * kLn2;
    if constexpr (RANGE) A.low[at] = bad ? ll : lo * kLn2, A.high[at] = bad ? ll : mm * kLn2;
  }
}

// Splits of a row's tokens: enough workgroups for four on each of the 256 compute units, and no
// share under two units a wave of the longest table.
int splits_of(int64_t seqs, int heads, int64_t tiles, int cols) {
  const int64_t groups = std::max<int64_t>(1, seqs * heads * tiles);
  const int64_t want = (1024 + groups - 1) / groups, most = std::max(1, cols * (kPageTokens / kUnit) / (2 * kWaves));
  return (int)std::min<int64_t>(std::min<int64_t>(want, most), 128);
}

template <typename T, int D, bool RANGE>
int launch(const AttendArgs& A, int64_t tiles, int seqs, hipStream_t s) {
  k_attend<T, D, RANGE><<<dim3((unsigned)(tiles * A.splits), A.heads, seqs), 64 * kWaves, 0, s>>>(A);
  HCK_CHECK_LAUNCH();
  if (A.splits > 1) {
    const long long rows = A.tokens * A.heads * A.group;
    k_join<T, D, RANGE><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, s>>>(A);
    HCK_CHECK_LAUNCH();
  }
  return HCK_OK;
}

bool shape_ok(int64_t tokens, int seqs, int kv_heads, int group, int most, int cols) {
  return tokens >= 0 && seqs >= 0 && seqs <= 65535 && kv_heads >= 1 && kv_heads <= 65535 && group >= 1 &&
         group <= 1024 && most >= 0 && cols >= 0 && cols <= (1 << 24) && (int64_t)most * group <= (1 << 30) &&
         tokens * kv_heads * group <= ((int64_t)1 << 32);
}

}  // namespace
}  // namespace hck

extern "C" size_t hck_kv4_attend_workspace_bytes(int64_t tokens, int seqs, int kv_heads, int group, int head_dim,
                                                 int most, int table_columns) {
  if (!hck::shape_ok(tokens, seqs, kv_heads, group, most, table_columns)) return 0;
  const int64_t tiles = ((int64_t)most * group + 15) / 16;
  const int splits = hck::splits_of(seqs, kv_heads, tiles, table_columns);
  return splits == 1 ? 0 : (size_t)(tokens * kv_heads * group) * splits * (4 + head_dim) * sizeof(float);
}

extern "C" int hck_kv4_attend(const void* pool, int64_t pages, int kv_heads, int head_dim, int type,
                              const void* queries, int64_t tokens, int group, int64_t q_token_stride,
                              int64_t q_head_stride, const int32_t* table, int64_t table_stride, int table_columns,
                              const int32_t* lengths, const int32_t* starts, int seqs, int most, int causal,
                              float scale, void* out, float* lse, float* low, float* high, void* workspace,
                              size_t workspace_bytes, void* stream) {
  if (hck::kv4_bytes(head_dim) == 0 || (type != HCK_BF16 && type != HCK_F16)) return HCK_ERR_UNSUPPORTED;
  if (!pool || pages < 1 || !hck::shape_ok(tokens, seqs, kv_heads, group, most, table_columns)) return HCK_ERR_ARG;
  if (!(scale > 0.f) || scale > 3.0e38f || (low == nullptr) != (high == nullptr)) return HCK_ERR_ARG;
  if (tokens == 0 || seqs == 0 || most == 0) return HCK_OK;
  if (!queries || !lengths || (!table && table_columns > 0) || !out || !lse) return HCK_ERR_ARG;
  if (!starts && tokens < seqs) return HCK_ERR_ARG;
  const int64_t tiles = ((int64_t)most * group + 15) / 16;
  hck::AttendArgs A{};
  A.pool = (const uint8_t*)pool;
  A.q = queries;
  A.table = table;
  A.lengths = lengths;
  A.starts = starts;
  A.out = out;
  A.lse = lse;
  A.low = low;
  A.high = high;
  A.part = (float*)workspace;
  A.q_ts = q_token_stride;
  A.q_hs = q_head_stride;
  A.tokens = tokens;
  A.pages = pages;
  A.table_stride = table_stride;
  A.cols = table_columns;
  A.heads = kv_heads;
  A.group = group;
  A.splits = hck::splits_of(seqs, kv_heads, tiles, table_columns);
  A.causal = causal;
  A.scale = scale;
  if (tiles * A.splits > 0x7fffffff) return HCK_ERR_ARG;
  const size_t need = hck_kv4_attend_workspace_bytes(tokens, seqs, kv_heads, group, head_dim, most, table_columns);
  if (need > workspace_bytes || (need && !workspace)) return HCK_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  const bool range = low != nullptr;
  if (head_dim == 128) {
    if (type == HCK_BF16) return range ? hck::launch<__bf16, 128, true>(A, tiles, seqs, s) : hck::launch<__bf16, 128, false>(A, tiles, seqs, s);
    return range ? hck::launch<_Float16, 128, true>(A, tiles, seqs, s) : hck::launch<_Float16, 128, false>(A, tiles, seqs, s);
  }
  if (type == HCK_BF16) return range ? hck::launch<__bf16, 64, true>(A, tiles, seqs, s) : hck::launch<__bf16, 64, false>(A, tiles, seqs, s);
  return range ? hck::launch<_Float16, 64, true>(A, tiles, seqs, s) : hck::launch<_Float16, 64, false>(A, tiles, seqs, s);
}
