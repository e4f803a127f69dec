// Eviction from 4-bit pages: of every key head the heaviest tokens of a sequence, and its last ones, go to other pages.
//
// Which tokens stay is a matter of whole numbers: weights become 32-bit keys in the weights' order (NaN above all, -0 as 0),
// and the k-th largest key T is found digit by digit, from counts of the values that the digits take among the keys that
// agree with those found so far.  What is above T stays, and of the tokens at T the first ones, so that the number is met.
// Places then come from counts of what stays before: the order of the tokens is kept, and nothing depends on timing.
//
// The pages' layout (kv4.hpp) interleaves tokens in the order of a matrix product's lanes, so a kept token is moved in pieces:
// keys 16 bytes (D = 64: 8) and values 4 (2) at a time, scales by the byte.  The work follows the target page, whose 16-byte pieces are
// written whole.
#include "../../include/holmes_ckks.h"
#include "internal.hpp"
#include "kv4.hpp"

namespace hck {
namespace {

struct EvictArgs {
  uint8_t* pool;
  const int *table, *lengths, *into;
  const float* weights;
  int *kept, *new_lengths;
  float* new_weights;
  int64_t pages, table_stride, into_stride, w_seq, w_head;
  int cols, heads, width, into_cols, keep, recent;
};

constexpr int kSelect = 1024;  // threads that choose
constexpr int kSelectWaves = kSelect / 64;
constexpr int kDigit = 11;     // bits of a digit: three of them, the last of 10
constexpr int kBins = 1 << kDigit;

// The key of a weight: ordered like the weights, NaN above all.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t b = __float_as_uint(w + 0.f);  // -0 as 0
  if (w != w) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ int lanes_below(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// One row: a sequence and a key head.
__global__ __launch_bounds__(kSelect) void k_select(EvictArgs A) {
  __shared__ int s_bins[kBins];
  __shared__ int s_above[kSelectWaves], s_at[kSelectWaves], s_last[kSelectWaves];
  __shared__ int s_found[2];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = (int)min((int64_t)max(A.lengths[b], 0), (int64_t)A.cols * kPageTokens);
  const int last = max(n - A.recent, 0);  // from here on all stay
  const int* table = A.table + b * A.table_stride;
  const float* weights = A.weights + b * A.w_seq + h * A.w_head;
  int* kept = A.kept + ((int64_t)b * A.heads + h) * A.keep;
  float* out = A.new_weights + ((int64_t)b * A.heads + h) * A.keep;
  auto there = [&](int j) {  // whether place j's page is in the pool
    const int pg = table[j / kPageTokens];
    return pg >= 0 && pg < A.pages;
  };
  auto weight = [&](int j) { return j < A.width ? weights[j] : 0.f; };

  // how many there are to choose from, and how many of the last
  if (threadIdx.x < 2) s_found[threadIdx.x] = 0;
  __syncthreads();
  int mine = 0, lasts = 0;
  for (int j = threadIdx.x; j < n; j += kSelect)
    if (there(j)) (j < last ? mine : lasts) += 1;
  atomicAdd(&s_found[0], mine), atomicAdd(&s_found[1], lasts);
  __syncthreads();
  const int choice = s_found[0], must = s_found[1];
  const int want = min(choice, A.keep - must);  // of those to choose from (recent is at most keep)
  __syncthreads();

  // T, and how many tokens at T stay
  uint32_t prefix = 0;
  int left = want;
  if (want > 0 && want < choice) {
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
      for (int i = threadIdx.x; i < kBins; i += kSelect) s_bins[i] = 0;
      __syncthreads();
      const int bins = 1 << bits;
      for (int j = threadIdx.x; j < last; j += kSelect) {
        if (!there(j)) continue;
        const uint32_t key = key_of(weight(j));
        if (digit && (key >> (shift + bits)) != prefix) continue;
        atomicAdd(&s_bins[(key >> shift) & (bins - 1)], 1);
      }
      __syncthreads();
      // the largest bin with `left` tokens or more in it and above it: one wave, 32 bins a lane
      if (wave == 0) {
        int sum = 0;
        const int per = bins / 64, top = bins - 1 - lane * per;
        for (int i = 0; i < per; ++i) sum += s_bins[top - i];
        int upto = sum;
        for (int d = 1; d < 64; d *= 2) {
          const int o = __shfl_up(upto, d);
          if (lane >= d) upto += o;
        }
        int before = upto - sum;
        if (before < left && upto >= left) {  // one lane
          int i = 0;
          for (; before + s_bins[top - i] < left; ++i) before += s_bins[top - i];
          s_found[0] = top - i, s_found[1] = left - before;
        }
      }
      __syncthreads();
      prefix = prefix << bits | (uint32_t)s_found[0];
      left = s_found[1];
      __syncthreads();
    }
  }
  const bool all = want == choice, none = want <= 0;
  // Tokens above T, at T and among the last, by waves: each has a run of the places.
  const int run = ((n + kSelectWaves - 1) / kSelectWaves + 63) / 64 * 64;
  const int from = min(wave * run, n), to = from + min(run, n - from);
  int above = 0, at = 0, tail = 0;
  for (int j0 = from; j0 < to; j0 += 64) {
    const int j = j0 + lane;
    if (j >= to || !there(j)) continue;
    if (j >= last) ++tail;
    else if (all) ++above;
    else if (!none) {
      const uint32_t key = key_of(weight(j));
      above += key > prefix, at += key == prefix;
    }
  }
  for (int d = 32; d; d /= 2) above += __shfl_xor(above, d), at += __shfl_xor(at, d), tail += __shfl_xor(tail, d);
  if (lane == 0) s_above[wave] = above, s_at[wave] = at, s_last[wave] = tail;
  __syncthreads();
  int place = 0, ties = 0;
  for (int w = 0; w < wave; ++w) {
    const int t = min(s_at[w], left - ties);
    place += s_above[w] + s_last[w] + (all || none ? 0 : t), ties += all || none ? 0 : t;
  }
  for (int j0 = from; j0 < to; j0 += 64) {
    const int j = j0 + lane;
    bool stay = false, tie = false;
    float w = 0.f;
    if (j < to && there(j)) {
      w = weight(j);
      if (j >= last || all) stay = true;
      else if (!none) {
        const uint32_t key = key_of(w);
        stay = key > prefix, tie = key == prefix;
      }
    }
    const unsigned long long tied = __ballot(tie);
    if (tie && ties + lanes_below(tied) < left) stay = true;
    ties = min(left, ties + (int)__popcll(tied));
    const unsigned long long staying = __ballot(stay);
    if (stay) {
      const int p = place + lanes_below(staying);
      kept[p] = j, out[p] = w;
    }
    place += (int)__popcll(staying);
  }
  const int total = max(want, 0) + must;
  for (int p = total + threadIdx.x; p < A.keep; p += kSelect) kept[p] = -1, out[p] = 0.f;
  if (h == 0 && threadIdx.x == 0) A.new_lengths[b] = total;
}

// One head's part of a target page.  A place that takes no token has itself for its source: its bytes stay.
template <int D>
__global__ __launch_bounds__(256) void k_move(EvictArgs A) {
  using L = Kv4<D>;
  __shared__ const uint8_t* s_from[kPageTokens];  // one head's part of the source page
  __shared__ int s_place[kPageTokens];
  const int p = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int pg = A.into[b * A.into_stride + p];
  if (pg < 0 || pg >= A.pages) return;
  const int64_t each = (int64_t)A.heads * L::kBytes;
  uint8_t* to = A.pool + pg * each + h * L::kBytes;
  if (threadIdx.x < kPageTokens) {
    const int t = threadIdx.x, i = p * kPageTokens + t;
    const int j = i < A.keep ? A.kept[((int64_t)b * A.heads + h) * A.keep + i] : -1;
    s_from[t] = j < 0 ? to : A.pool + A.table[b * A.table_stride + j / kPageTokens] * each + h * L::kBytes;
    s_place[t] = j < 0 ? t : j % kPageTokens;
  }
  __syncthreads();
  constexpr int kKey = D / 8;         // bytes of a token's keys that lie together
  constexpr int kValue = L::kDpl / 2; // and of its values
  typedef uint32_t piece __attribute__((ext_vector_type(kKey / 4)));
  for (int w = threadIdx.x; w < kPageTokens * 4; w += 256) {  // keys: [tile][g][token]
    const int t = (w >> 6) * 16 + (w & 15), g = (w >> 4) & 3;
    *reinterpret_cast<piece*>(to + L::key_code(t, g * (D / 4))) =
        *reinterpret_cast<const piece*>(s_from[t] + L::key_code(s_place[t], g * (D / 4)));
  }
  for (int w = threadIdx.x; w < kPageTokens * 16 * kValue / 16; w += 256) {  // values: 16 / kValue tokens of a lane (g, c)
    const int c = w & 15, g = (w >> 4) & 3, half = w >> 6;                   // half: a block of 32 tokens, or half of one
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (kValue == 4) {
        const int t = half * 16 + 4 * g + k;
        x[k] = *reinterpret_cast<const uint32_t*>(s_from[t] + L::value_code(s_place[t], c));
      } else {
        x[k] = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = 2 * k + e, t = half * 32 + (j >> 2) * 16 + 4 * g + (j & 3);
          x[k] |= (uint32_t)*reinterpret_cast<const uint16_t*>(s_from[t] + L::value_code(s_place[t], c)) << (16 * e);
        }
      }
    }
    const int first = kValue == 4 ? half * 16 + 4 * g : half * 32 + 4 * g;
    *reinterpret_cast<uint4*>(to + L::value_code(first, c)) = uint4{x[0], x[1], x[2], x[3]};
  }
  for (int w = threadIdx.x; w < kPageTokens / 4 * L::kRuns; w += 256) {  // scales, four tokens at a time
    const int run = w % L::kRuns, q = w / L::kRuns;
    uint32_t ks = 0, vs = 0;
    const int k0 = (q >> 4) * 64 + (q & 15), v0 = (q >> 3) * 32 + ((q >> 2) & 1) * 16 + (q & 3) * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = k0 + 16 * k, v = v0 + k;
      ks |= (uint32_t)s_from[t][L::key_scale(s_place[t], run)] << (8 * k);
      vs |= (uint32_t)s_from[v][L::value_scale(s_place[v], run)] << (8 * k);
    }
    *reinterpret_cast<uint32_t*>(to + L::key_scale(k0, run)) = ks;
    *reinterpret_cast<uint32_t*>(to + L::value_scale(v0, run)) = vs;
  }
}

}  // namespace
}  // namespace hck

extern "C" int hck_kv4_evict(void* pool, int64_t pages, int kv_heads, int head_dim, const int32_t* table,
                             int64_t table_stride, int table_columns, const int32_t* lengths, int seqs,
                             const float* weights, int64_t weight_seq_stride, int64_t weight_head_stride, int weight_places,
                             const int32_t* into, int64_t into_stride, int into_columns, int keep, int recent,
                             int32_t* kept, int32_t* new_lengths, float* new_weights, void* stream) {
  if (hck::kv4_bytes(head_dim) == 0) return HCK_ERR_UNSUPPORTED;
  if (!pool || pages < 1 || kv_heads < 1 || kv_heads > 65535 || seqs < 0 || seqs > 65535 || table_columns < 0 ||
      table_columns >= 1 << 23 || weight_places < 0 || keep < 0 || recent < 0 || recent > keep || into_columns < 0 ||
      into_columns >= 1 << 23)  // (places of a sequence are counted in 30 bits)
    return HCK_ERR_ARG;
  const int need = (int)(((int64_t)keep + hck::kPageTokens - 1) / hck::kPageTokens);
  if (need > into_columns) return HCK_ERR_ARG;
  if (seqs == 0) return HCK_OK;
  if (!lengths || !new_lengths || (table_columns && !table) || (weight_places && !weights) ||
      (keep && (!into || !kept || !new_weights)))
    return HCK_ERR_ARG;
  hck::EvictArgs A = {};
  A.pool = (uint8_t*)pool, A.table = table, A.lengths = lengths, A.into = into, A.weights = weights;
  A.kept = kept, A.new_lengths = new_lengths, A.new_weights = new_weights;
  A.pages = pages, A.table_stride = table_stride, A.into_stride = into_stride, A.w_seq = weight_seq_stride,
  A.w_head = weight_head_stride, A.cols = table_columns, A.heads = kv_heads, A.width = weight_places,
  A.into_cols = into_columns, A.keep = keep, A.recent = recent;
  hipStream_t s = (hipStream_t)stream;
  hck::k_select<<<dim3(kv_heads, seqs), hck::kSelect, 0, s>>>(A);
  HCK_CHECK_LAUNCH();
  if (need) {
    const dim3 grid((unsigned)need, kv_heads, seqs);
    if (head_dim == 128) hck::k_move<128><<<grid, 256, 0, s>>>(A);
    else hck::k_move<64><<<grid, 256, 0, s>>>(A);
    HCK_CHECK_LAUNCH();
  }
  return HCK_OK;
}
