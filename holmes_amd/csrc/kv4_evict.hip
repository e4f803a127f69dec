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
#include "kv4_attend.hpp"

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

// Sums over the threads up to each, and over all; `part` has a place for every wave.
__device__ __forceinline__ int upto_thread(int x, int* part, int& all) {
  const int upto = upto_lane(x), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();  // what was read of `part` before
  if (lane == 63) part[wave] = upto;
  __syncthreads();
  const int sums = upto_lane(lane < kSelectWaves ? part[lane] : 0);
  all = __builtin_amdgcn_readlane(sums, kSelectWaves - 1);
  return upto + (wave ? __builtin_amdgcn_readlane(sums, __builtin_amdgcn_readfirstlane(wave) - 1) : 0);
}

// One row: a sequence and a key head.  Thread t has the keys of places t, 1024 + t, .. in registers, R of them, read at once
// and looked at four times; a row of more goes through them in pieces, read anew each time.  A key of 0 is no choice.
//
// Counts of the first digit, which is mostly the exponents', would meet in few places, so every eighth lane has counts of
// its own.
template <int R>
__global__ __launch_bounds__(kSelect) void k_select(EvictArgs A) {
  constexpr int kCopies = R >= 4 ? 8 : 1, kPiece = R * kSelect;
  __shared__ int s_bins[kBins * kCopies];
  __shared__ int s_stay[R * kSelectWaves], s_tie[R * kSelectWaves], s_part[kSelectWaves], s_found[2];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = (int)min((int64_t)max(A.lengths[b], 0), (int64_t)A.cols * kPageTokens);
  const int last = max(n - A.recent, 0);  // from here on all stay
  const int* table = A.table + b * A.table_stride;
  const float* weights = A.weights + b * A.w_seq + h * A.w_head;
  int* kept = A.kept + ((int64_t)b * A.heads + h) * A.keep;
  float* out = A.new_weights + ((int64_t)b * A.heads + h) * A.keep;

  // Places whose page is not in the pool: as a rule there are none, and no place asks again.
  int gone = 0;
  for (int i = threadIdx.x; i * kPageTokens < n; i += kSelect) {
    const int pg = table[i];
    gone |= pg < 0 || pg >= A.pages;
  }
  const bool whole = !__syncthreads_or(gone);
  auto there = [&](int j) {
    if (whole) return true;
    const int pg = table[j / kPageTokens];
    return pg >= 0 && pg < A.pages;
  };

  uint32_t key[R];
  const int pieces = (n + kPiece - 1) / kPiece;
  auto load = [&](int piece) {
    float w[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = piece * kPiece + r * kSelect + threadIdx.x;
      w[r] = j < last && j < A.width ? weights[j] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = piece * kPiece + r * kSelect + threadIdx.x;
      key[r] = j < last && there(j) ? key_of(w[r]) : 0;
    }
  };
  if (pieces) load(0);

  // how many there are to choose from, and how many of the last
  int choice = last, must = n - last;
  if (!whole) {
    int mine = 0, lasts = 0, all;
    for (int j = threadIdx.x; j < n; j += kSelect)
      if (there(j)) (j < last ? mine : lasts) += 1;
    upto_thread(mine, s_part, all);
    choice = all;
    upto_thread(lasts, s_part, all);
    must = all;
  }
  const int want = min(choice, A.keep - must);  // of those to choose from (recent is at most keep)

  // T, and how many tokens at T stay
  uint32_t prefix = 0;
  int left = want;
  const bool all = want == choice, none = want <= 0;
  if (!all && !none) {
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11, bins = 1 << bits;
      for (int i = threadIdx.x; i < kBins * kCopies; i += kSelect) s_bins[i] = 0;
      __syncthreads();
      for (int piece = 0; piece < pieces; ++piece) {
        if (pieces > 1) load(piece);
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (key[r] && (digit == 0 || (key[r] >> (shift + bits)) == prefix))
            atomicAdd(&s_bins[((key[r] >> shift) & (bins - 1)) * kCopies + lane % kCopies], 1);
      }
      __syncthreads();
      // the largest bin with `left` tokens or more in it and above it: two bins a thread, from the top
      const int top = bins - 1 - 2 * (int)threadIdx.x;
      int count[2] = {0, 0}, total;
      if (top > 0) {
#pragma unroll
        for (int c = 0; c < kCopies; ++c) count[0] += s_bins[top * kCopies + c], count[1] += s_bins[(top - 1) * kCopies + c];
      }
      const int upto = upto_thread(count[0] + count[1], s_part, total), before = upto - count[0] - count[1];
      if (before < left && upto >= left) {  // one thread
        const bool second = before + count[0] < left;
        s_found[0] = second ? top - 1 : top, s_found[1] = left - before - (second ? count[0] : 0);
      }
      __syncthreads();
      prefix = prefix << bits | (uint32_t)s_found[0];
      left = s_found[1];
    }
  }

  // What stays, 64 places at a time: how many for certain and how many at T; where each 64 begin; and then each place.
  int place = 0, ties = 0;
  for (int piece = 0; piece < pieces; ++piece) {
    if (pieces > 1) load(piece);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = piece * kPiece + r * kSelect + threadIdx.x;
      const bool sure = j >= last ? j < n && there(j) : key[r] && (all || (!none && key[r] > prefix));
      const bool tie = key[r] && !all && !none && key[r] == prefix;
      const unsigned long long sures = __ballot(sure), tied = __ballot(tie);
      if (lane == 0) s_stay[r * kSelectWaves + wave] = (int)__popcll(sures), s_tie[r * kSelectWaves + wave] = (int)__popcll(tied);
    }
    __syncthreads();
    constexpr int kMine = (R * kSelectWaves + kSelect - 1) / kSelect;
    int sum = 0, at[kMine], stay[kMine], got;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int e = threadIdx.x * kMine + i;
      at[i] = e < R * kSelectWaves ? s_tie[e] : 0, stay[i] = e < R * kSelectWaves ? s_stay[e] : 0, sum += at[i];
    }
    int rank = ties + upto_thread(sum, s_part, got) - sum;  // ties before the thread's first 64
    ties += got;
    sum = 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int e = threadIdx.x * kMine + i;
      if (e < R * kSelectWaves) s_tie[e] = rank;
      const int taken = max(0, min(at[i], left - rank));
      rank += at[i], stay[i] += taken, sum += stay[i];
    }
    int begin = place + upto_thread(sum, s_part, got) - sum;
    place += got;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int e = threadIdx.x * kMine + i;
      if (e < R * kSelectWaves) s_stay[e] = begin;
      begin += stay[i];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = piece * kPiece + r * kSelect + threadIdx.x;
      bool stays = j >= last ? j < n && there(j) : key[r] && (all || (!none && key[r] > prefix));
      const bool tie = key[r] && !all && !none && key[r] == prefix;
      const unsigned long long tied = __ballot(tie);
      if (tie && s_tie[r * kSelectWaves + wave] + lanes_below(tied) < left) stays = true;
      const unsigned long long staying = __ballot(stays);
      if (stays) {
        const int p = s_stay[r * kSelectWaves + wave] + lanes_below(staying);
        kept[p] = j, out[p] = j < A.width ? weights[j] : 0.f;
      }
    }
  }
  for (int p = place + threadIdx.x; p < A.keep; p += kSelect) kept[p] = -1, out[p] = 0.f;
  if (h == 0 && threadIdx.x == 0) A.new_lengths[b] = place;
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
  // the least keys a thread for which a row goes through the registers once, as far as a table tells
  const int64_t room = (int64_t)table_columns * hck::kPageTokens;
  auto* select = room <= 1 * hck::kSelect   ? hck::k_select<1>
                 : room <= 4 * hck::kSelect ? hck::k_select<4>
                 : room <= 16 * hck::kSelect ? hck::k_select<16>
                                             : hck::k_select<64>;
  select<<<dim3(kv_heads, seqs), hck::kSelect, 0, s>>>(A);
  HCK_CHECK_LAUNCH();
  if (need) {
    const dim3 grid((unsigned)need, kv_heads, seqs);
    if (head_dim == 128) hck::k_move<128><<<grid, 256, 0, s>>>(A);
    else hck::k_move<64><<<grid, 256, 0, s>>>(A);
    HCK_CHECK_LAUNCH();
  }
  return HCK_OK;
}
