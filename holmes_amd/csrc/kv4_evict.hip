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
//
// 32 sequences of 63 to 8191 tokens, 8 heads of 128, 1024 kept: choosing 14 us (dependent steps: lengths, weights, two or
// three digits, places), moving 18 (70 MB, 3.9 TB/s, of pieces of 4 bytes).
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
  int cols, heads, seqs, width, keep, recent;
  int *counts, segs;  // of long rows: Counts of each row, and its segments
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

// A row: a sequence and a key head.
struct Row {
  int n, last, seq, line;  // last: from here on all stay
  const int* table;
  const float* weights;
  int* kept;
  float* out;
  __device__ __forceinline__ Row(const EvictArgs& A, int b, int h) {
    n = (int)min((int64_t)max(A.lengths[b], 0), (int64_t)A.cols * kPageTokens);
    last = max(n - A.recent, 0), seq = b, line = b * A.heads + h;
    table = A.table + b * A.table_stride;
    weights = A.weights + b * A.w_seq + h * A.w_head;
    kept = A.kept + (int64_t)line * A.keep, out = A.new_weights + (int64_t)line * A.keep;
  }
  __device__ __forceinline__ bool in_pool(const EvictArgs& A, int page) const {
    const int pg = table[page];
    return pg >= 0 && pg < A.pages;
  }
};

// Thread t has the keys of places first + t, first + 1024 + t, .. in registers, R of them, read at once.  A key of 0 is no
// choice.
template <int R>
struct Keys {
  uint32_t key[R];
  int first, rounds;  // rounds: of R, those that have places
  bool whole;  // no place's page is outside the pool, as a rule: then no place asks again
  __device__ __forceinline__ bool there(const EvictArgs& A, const Row& row, int j) const {
    return whole || row.in_pool(A, j / kPageTokens);
  }
  __device__ __forceinline__ int place(int r) const { return first + r * kSelect + (int)threadIdx.x; }
  __device__ __forceinline__ void load(const EvictArgs& A, const Row& row, int from) {
    first = from, rounds = min(R, (max(row.n - first, 0) + kSelect - 1) / kSelect);
    float w[R];
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = place(r) < row.last && place(r) < A.width ? row.weights[place(r)] : 0.f;
    const int page = first / kPageTokens + threadIdx.x;
    const bool gone = threadIdx.x < R * kSelect / kPageTokens && page * kPageTokens < row.n && !row.in_pool(A, page);
    whole = !__syncthreads_or(gone);
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = place(r) < row.last && there(A, row, place(r)) ? key_of(w[r]) : 0;
  }
  // the tokens to choose from, and those of the last
  __device__ __forceinline__ void number(const EvictArgs& A, const Row& row, int* part, int& choice, int& must) const {
    const int to = min(first + R * kSelect, row.n);
    choice = max(0, min(to, row.last) - first), must = max(0, to - max(first, row.last));
    if (whole) return;
    int mine = 0, lasts = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) mine += key[r] != 0, lasts += place(r) >= row.last && place(r) < row.n && there(A, row, place(r));
    upto_thread(mine, part, choice);
    upto_thread(lasts, part, must);
  }
};

__device__ __forceinline__ int shift_of(int digit) { return digit == 0 ? 21 : digit == 1 ? 10 : 0; }
__device__ __forceinline__ int bits_of(int digit) { return digit == 2 ? 10 : 11; }

// Counts of a digit among the keys that agree with the digits before it.  The first digit is mostly the exponents', of which
// there are few, so every eighth lane counts by itself.
template <int R, int kCopies>
__device__ __forceinline__ void count_digit(const Keys<R>& K, int digit, uint32_t prefix, int* bins) {
  const int shift = shift_of(digit), bits = bits_of(digit);
  for (int i = threadIdx.x; i < kBins * kCopies; i += kSelect) bins[i] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (r < K.rounds && K.key[r] && (digit == 0 || (K.key[r] >> (shift + bits)) == prefix))
      atomicAdd(&bins[((K.key[r] >> shift) & ((1 << bits) - 1)) * kCopies + threadIdx.x % kCopies], 1);
  __syncthreads();
}

// The bins that a thread looks at, from the top: top_bin and the one below it (none: -1).
__device__ __forceinline__ int top_bin(int digit) { return (1 << bits_of(digit)) - 1 - 2 * (int)threadIdx.x; }

// The largest digit with `left` keys or more at it and above it, from a thread's two counts; `left` becomes how many of those
// at it; returns how many there are.  found: three places, not written again before a barrier.
__device__ __forceinline__ int find_digit(int digit, int high, int low, int* part, int* found, uint32_t& prefix, int& left) {
  int total;
  const int upto = upto_thread(high + low, part, total), before = upto - high - low;
  if (before < left && upto >= left) {  // one thread
    const bool second = before + high < left;
    found[0] = top_bin(digit) - second, found[1] = left - before - (second ? high : 0), found[2] = second ? low : high;
  }
  __syncthreads();
  prefix = prefix << bits_of(digit) | (uint32_t)found[0];
  left = found[1];
  return found[2];
}

// What stays of the keys, above T or among the first `left` at T (of which `ties` come before these keys): 64 places at a time,
// how many for certain and how many at T; where each 64 begin; and then each place, from `place` on.
template <int R>
__device__ __forceinline__ void write_kept(const EvictArgs& A, const Row& row, const Keys<R>& K, uint32_t T, int left, int ties,
                                           int place, int* s_stay, int* s_tie, int* part) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto sure = [&](int r) {
    const int j = K.place(r);
    return j >= row.last ? j < row.n && K.there(A, row, j) : K.key[r] > T;
  };
  auto tie = [&](int r) { return K.key[r] != 0 && K.key[r] == T; };
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= K.rounds) continue;
    const unsigned long long sures = __ballot(sure(r)), tied = __ballot(tie(r));
    if (lane == 0) s_stay[r * kSelectWaves + wave] = (int)__popcll(sures), s_tie[r * kSelectWaves + wave] = (int)__popcll(tied);
  }
  __syncthreads();
  static_assert(R * kSelectWaves <= kSelect, "a thread sums up 64 places");
  const int e = threadIdx.x, entries = K.rounds * kSelectWaves, mine = e < entries ? s_tie[e] : 0;
  int stay = e < entries ? s_stay[e] : 0, all;
  const int rank = ties + upto_thread(mine, part, all) - mine;
  stay += max(0, min(mine, left - rank));
  const int begin = place + upto_thread(stay, part, all) - stay;
  if (e < entries) s_tie[e] = rank, s_stay[e] = begin;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= K.rounds) continue;
    bool stays = sure(r);
    const bool t = tie(r);
    const unsigned long long tied = __ballot(t);
    if (t && s_tie[r * kSelectWaves + wave] + lanes_below(tied) < left) stays = true;
    const unsigned long long staying = __ballot(stays);
    if (stays) {
      const int p = s_stay[r * kSelectWaves + wave] + lanes_below(staying), j = K.place(r);
      row.kept[p] = j, row.out[p] = j < A.width ? row.weights[j] : 0.f;
    }
  }
}

__device__ __forceinline__ void write_rest(const EvictArgs& A, const Row& row, int total) {
  for (int p = total + threadIdx.x; p < A.keep; p += kSelect) row.kept[p] = -1, row.out[p] = 0.f;
  if (row.line % A.heads == 0 && threadIdx.x == 0) A.new_lengths[row.seq] = total;
}

// One head's part of target page p, by a workgroup's threads.  A place that takes no token has itself for its source: its bytes
// stay.
struct Sources {
  const uint8_t* from[kPageTokens];  // one head's part of the source page
  int place[kPageTokens];
};
template <int D>
__device__ __forceinline__ void move_page(const EvictArgs& A, int b, int h, int p, Sources& S) {
  using L = Kv4<D>;
  const int threads = blockDim.x;
  const int pg = A.into[b * A.into_stride + p];
  if (pg < 0 || pg >= A.pages) return;
  const int64_t each = (int64_t)A.heads * L::kBytes;
  uint8_t* to = A.pool + pg * each + h * L::kBytes;
  if (threadIdx.x < kPageTokens) {
    const int t = threadIdx.x, i = p * kPageTokens + t;
    const int j = i < A.keep ? A.kept[((int64_t)b * A.heads + h) * A.keep + i] : -1;
    S.from[t] = j < 0 ? to : A.pool + A.table[b * A.table_stride + j / kPageTokens] * each + h * L::kBytes;
    S.place[t] = j < 0 ? t : j % kPageTokens;
  }
  __syncthreads();
  constexpr int kKey = D / 8;         // bytes of a token's keys that lie together
  constexpr int kValue = L::kDpl / 2; // and of its values
  typedef uint32_t piece __attribute__((ext_vector_type(kKey / 4)));
  for (int w = threadIdx.x; w < kPageTokens * 4; w += threads) {  // keys: [tile][g][token]
    const int t = (w >> 6) * 16 + (w & 15), g = (w >> 4) & 3;
    *reinterpret_cast<piece*>(to + L::key_code(t, g * (D / 4))) =
        *reinterpret_cast<const piece*>(S.from[t] + L::key_code(S.place[t], g * (D / 4)));
  }
  for (int w = threadIdx.x; w < kPageTokens * 16 * kValue / 16; w += threads) {  // values: 16 / kValue tokens of a lane (g, c)
    const int c = w & 15, g = (w >> 4) & 3, half = w >> 6;                   // half: a block of 32 tokens, or half of one
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (kValue == 4) {
        const int t = half * 16 + 4 * g + k;
        x[k] = *reinterpret_cast<const uint32_t*>(S.from[t] + L::value_code(S.place[t], c));
      } else {
        x[k] = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = 2 * k + e, t = half * 32 + (j >> 2) * 16 + 4 * g + (j & 3);
          x[k] |= (uint32_t)*reinterpret_cast<const uint16_t*>(S.from[t] + L::value_code(S.place[t], c)) << (16 * e);
        }
      }
    }
    const int first = kValue == 4 ? half * 16 + 4 * g : half * 32 + 4 * g;
    *reinterpret_cast<uint4*>(to + L::value_code(first, c)) = uint4{x[0], x[1], x[2], x[3]};
  }
  for (int w = threadIdx.x; w < kPageTokens / 4 * L::kRuns; w += threads) {  // scales, four tokens at a time
    const int run = w % L::kRuns, q = w / L::kRuns;
    uint32_t ks = 0, vs = 0;
    const int k0 = (q >> 4) * 64 + (q & 15), v0 = (q >> 3) * 32 + ((q >> 2) & 1) * 16 + (q & 3) * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = k0 + 16 * k, v = v0 + k;
      ks |= (uint32_t)S.from[t][L::key_scale(S.place[t], run)] << (8 * k);
      vs |= (uint32_t)S.from[v][L::value_scale(S.place[v], run)] << (8 * k);
    }
    *reinterpret_cast<uint32_t*>(to + L::key_scale(k0, run)) = ks;
    *reinterpret_cast<uint32_t*>(to + L::value_scale(v0, run)) = vs;
  }
}

template <int D>
__global__ __launch_bounds__(256) void k_move(EvictArgs A) {
  __shared__ Sources s_sources;
  move_page<D>(A, blockIdx.z, blockIdx.y, blockIdx.x, s_sources);
}

// A row of up to R * 1024 places by one workgroup, which with D moves the kept tokens as well: where they are one page or two, a
// second launch costs more than it brings (384 tokens, 256 kept and read back: 15.0 us with it, 12.9 without).
template <int R, int D>
__global__ __launch_bounds__(kSelect) void k_select(EvictArgs A) {
  constexpr int kCopies = R >= 4 ? 8 : 1;
  __shared__ int s_bins[kBins * kCopies], s_stay[R * kSelectWaves], s_tie[R * kSelectWaves], s_part[kSelectWaves], s_found[3];
  const Row row(A, blockIdx.y, blockIdx.x);
  Keys<R> K;
  K.load(A, row, 0);
  int choice, must;
  K.number(A, row, s_part, choice, must);
  const int want = min(choice, A.keep - must);  // of those to choose from (recent is at most keep)
  uint32_t T = want < choice ? 0xffffffffu : 0;  // none, or all
  int left = 0;
  if (want > 0 && want < choice) {
    T = 0, left = want;
    for (int digit = 0; digit < 3; ++digit) {
      const int top = top_bin(digit);
      int high = 0, low = 0;
      if (digit == 0) {
        count_digit<R, kCopies>(K, digit, T, s_bins);
        if (top > 0) {
#pragma unroll
          for (int c = 0; c < kCopies; ++c) high += s_bins[top * kCopies + c], low += s_bins[(top - 1) * kCopies + c];
        }
      } else {
        count_digit<R, 1>(K, digit, T, s_bins);
        if (top > 0) high = s_bins[top], low = s_bins[top - 1];
      }
      if (find_digit(digit, high, low, s_part, s_found, T, left) == left) {  // all that agree so far stay
        T = (T << shift_of(digit)) - 1, left = 0;
        break;
      }
    }
  }
  write_kept<R>(A, row, K, T, left, 0, 0, s_stay, s_tie, s_part);
  write_rest(A, row, want + must);
  if constexpr (D != 0) {
    __shared__ Sources s_sources;
    for (int p = 0; p * kPageTokens < A.keep; ++p) {
      __syncthreads();  // what was kept has been written, and the sources of the page before read
      move_page<D>(A, blockIdx.y, blockIdx.x, p, s_sources);
    }
  }
}

constexpr int kMovedPages = 2;
constexpr int kWhole = 16;  // places in thousands that one workgroup takes
template <int D>
void launch_select(const EvictArgs& A, int64_t room, hipStream_t s) {
  auto* select = room <= 1 * kSelect ? k_select<1, D> : room <= 4 * kSelect ? k_select<4, D> : k_select<kWhole, D>;
  select<<<dim3(A.heads, A.seqs), kSelect, 0, s>>>(A);
}

// Longer rows, by a workgroup for every segment of 8192 places and a launch for every digit: each looks at its keys again, adds
// up the segments' counts of the digit before, and counts the next among its own.  The last launch writes what stays, from where
// the segments before end.  8 heads of 131072 places, 8192 kept: 42 us with the move (16384 places a segment 47, 4096 43; by one
// workgroup a row 306); of 20000 31, where one of 8000 takes 12.
constexpr int kSegment = 8, kSegmentPlaces = kSegment * kSelect;
struct Counts {  // of one row
  int *bins, *choice, *must, *above, *state;  // [digit][segment][bin], [segment], [segment], [digit < 2][segment], [digit < 2][2]
  static __host__ __device__ int64_t ints(int segs) { return (int64_t)segs * (3 * kBins + 4) + 4; }
  __device__ __forceinline__ Counts(const EvictArgs& A, int line) {
    bins = A.counts + line * ints(A.segs), choice = bins + (int64_t)A.segs * 3 * kBins, must = choice + A.segs;
    above = must + A.segs, state = above + 2 * A.segs;
  }
};

template <int PHASE>
__global__ __launch_bounds__(kSelect) void k_select_long(EvictArgs A) {
  constexpr int R = kSegment, kCopies = PHASE == 0 ? 8 : 1;
  __shared__ int s_bins[PHASE < 3 ? kBins * kCopies : 1], s_stay[R * kSelectWaves], s_tie[R * kSelectWaves];
  __shared__ int s_part[kSelectWaves], s_found[3];
  const int seg = blockIdx.x;
  const Row row(A, blockIdx.z, blockIdx.y);
  const Counts C(A, row.line);
  const int segs = (row.n + kSegmentPlaces - 1) / kSegmentPlaces;
  if (seg >= max(segs, 1)) return;
  Keys<R> K;
  K.load(A, row, seg * kSegmentPlaces);
  if constexpr (PHASE == 0) {
    int choice, must;
    K.number(A, row, s_part, choice, must);
    if (threadIdx.x == 0) C.choice[seg] = choice, C.must[seg] = must;
  }
  // the numbers of the whole row, and of the segments before
  int choice = 0, must = 0, choice_before = 0, must_before = 0;
  uint32_t T = 0;
  int left = 0;
  if constexpr (PHASE > 0) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < segs; s0 += 64) {
      const int s = s0 + lane, c = s < segs ? C.choice[s] : 0, m = s < segs ? C.must[s] : 0;
      choice += over_wave(c), must += over_wave(m);
      choice_before += over_wave(s < seg ? c : 0), must_before += over_wave(s < seg ? m : 0);
    }
  }
  const int want = min(choice, A.keep - must);
  const bool some = PHASE == 0 || (want > 0 && want < choice);
  int before = 0, ties_before = 0;  // of the last digit
  if (PHASE > 0 && some) {
    // the digit before this one, from all segments' counts
    constexpr int digit = PHASE - 1;
    if (digit == 0) left = want;
    else T = (uint32_t)C.state[2 * (digit - 1)], left = C.state[2 * (digit - 1) + 1];
    const int top = top_bin(digit);
    int high = 0, low = 0, own_high = 0, own_low = 0;  // own: of this segment; in the last launch, of those before
    if (top > 0) {
#pragma unroll 8
      for (int s = 0; s < segs; ++s) {
        const int2 two = *reinterpret_cast<const int2*>(C.bins + ((int64_t)digit * A.segs + s) * kBins + top - 1);
        high += two.y, low += two.x;
        if (PHASE == 3 ? s < seg : s == seg) own_high += two.y, own_low += two.x;
      }
    }
    find_digit(digit, high, low, s_part, s_found, T, left);
    const int at = (int)(T & ((1u << bits_of(digit)) - 1));
    int all;
    upto_thread((top > at ? own_high : 0) + (top - 1 > at ? own_low : 0), s_part, all);
    if constexpr (PHASE < 3) {
      if (threadIdx.x == 0) C.above[digit * A.segs + seg] = all;
      if (threadIdx.x == 0 && seg == 0) C.state[2 * digit] = (int)T, C.state[2 * digit + 1] = left;
    } else {
      before = all;
      upto_thread(top == at ? own_high : top - 1 == at ? own_low : 0, s_part, all);
      ties_before = all;
      for (int s0 = 0; s0 < seg; s0 += 64) {
        const int s = s0 + (threadIdx.x & 63);
        before += over_wave(s < seg ? C.above[s] + C.above[A.segs + s] : 0);
      }
    }
  }
  if constexpr (PHASE < 3) {
    if (!some) return;
    count_digit<R, kCopies>(K, PHASE, T, s_bins);
    int* bins = C.bins + ((int64_t)PHASE * A.segs + seg) * kBins;
    for (int i = threadIdx.x; i < kBins; i += kSelect) {
      int sum = 0;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) sum += s_bins[i * kCopies + c];
      bins[i] = sum;
    }
  } else {
    if (!some) T = want < choice ? 0xffffffffu : 0, left = 0, before = want < choice ? 0 : choice_before;
    write_kept<R>(A, row, K, T, left, ties_before, before + min(left, ties_before) + must_before, s_stay, s_tie, s_part);
    if (seg == 0) write_rest(A, row, want + must);
  }
}

// Segments of a row with room for so many pages; 0: one workgroup takes it.
int segments(int cols) {
  const int64_t room = (int64_t)cols * kPageTokens;
  return room <= kWhole * kSelect ? 0 : (int)((room + kSegmentPlaces - 1) / kSegmentPlaces);
}

}  // namespace
}  // namespace hck

extern "C" size_t hck_kv4_evict_workspace_bytes(int seqs, int kv_heads, int table_columns) {
  if (seqs < 1 || seqs > 65535 || kv_heads < 1 || kv_heads > 65535 || table_columns < 0 || table_columns >= 1 << 23 ||
      (int64_t)seqs * kv_heads > INT32_MAX)
    return 0;
  const int segs = hck::segments(table_columns);
  return segs ? (size_t)seqs * kv_heads * hck::Counts::ints(segs) * sizeof(int) : 0;
}

extern "C" int hck_kv4_evict(void* pool, int64_t pages, int kv_heads, int head_dim, const int32_t* table,
                             int64_t table_stride, int table_columns, const int32_t* lengths, int seqs,
                             const float* weights, int64_t weight_seq_stride, int64_t weight_head_stride, int weight_places,
                             const int32_t* into, int64_t into_stride, int into_columns, int keep, int recent,
                             int32_t* kept, int32_t* new_lengths, float* new_weights, void* workspace, size_t workspace_bytes,
                             void* stream) {
  if (hck::kv4_bytes(head_dim) == 0) return HCK_ERR_UNSUPPORTED;
  if (!pool || pages < 1 || kv_heads < 1 || kv_heads > 65535 || seqs < 0 || seqs > 65535 || table_columns < 0 ||
      table_columns >= 1 << 23 || weight_places < 0 || keep < 0 || recent < 0 || recent > keep || into_columns < 0 ||
      into_columns >= 1 << 23 || (int64_t)seqs * kv_heads > INT32_MAX)  // (places of a sequence are counted in 30 bits, rows in 31)
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
  A.w_head = weight_head_stride, A.cols = table_columns, A.heads = kv_heads, A.seqs = seqs, A.width = weight_places,
  A.keep = keep, A.recent = recent;
  A.segs = hck::segments(table_columns), A.counts = (int*)workspace;
  const size_t bytes = hck_kv4_evict_workspace_bytes(seqs, kv_heads, table_columns);
  if (bytes && (!workspace || workspace_bytes < bytes)) return HCK_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  // the least keys a thread for which a row goes through the registers once, as far as a table tells
  const int64_t room = (int64_t)table_columns * hck::kPageTokens;
  const bool moved = A.segs == 0 && need <= hck::kMovedPages;
  if (A.segs == 0) {
    if (!moved || need == 0) hck::launch_select<0>(A, room, s);
    else if (head_dim == 128) hck::launch_select<128>(A, room, s);
    else hck::launch_select<64>(A, room, s);
  } else {
    const dim3 grid(A.segs, kv_heads, seqs);
    hck::k_select_long<0><<<grid, hck::kSelect, 0, s>>>(A);
    hck::k_select_long<1><<<grid, hck::kSelect, 0, s>>>(A);
    hck::k_select_long<2><<<grid, hck::kSelect, 0, s>>>(A);
    hck::k_select_long<3><<<grid, hck::kSelect, 0, s>>>(A);
  }
  HCK_CHECK_LAUNCH();
  if (need && !moved) {
    const dim3 grid((unsigned)need, kv_heads, seqs);
    if (head_dim == 128) hck::k_move<128><<<grid, 256, 0, s>>>(A);
    else hck::k_move<64><<<grid, 256, 0, s>>>(A);
    HCK_CHECK_LAUNCH();
  }
  return HCK_OK;
}
