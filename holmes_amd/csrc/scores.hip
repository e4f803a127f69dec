// Log probabilities of given tokens under rows of logits, with the entropy and the top alternatives.
//
// For a row x over the vocabulary, in units of log 2 (t_i = (x_i - r) log2 e with a running reference r,
// the largest value met):  l = sum 2^(t_i),  s = sum 2^(t_i) t_i, then
//   log p(i) = x_i - r - ln 2 log2 l,   H = ln 2 (log2 l - s / l).
// Every lane keeps its own (r, l, s) over the values that it meets and they are joined at the end, so
// a row is read once.
//
// The top values: every lane keeps the maximum of what it met.  The k-th largest T of a workgroup's 256
// maxima is no more than the k-th largest value, and only lanes whose maximum reaches T can hold a value
// that does: hardly more than k of them.  A lane also keeps which block of its values had the maximum and
// the largest of the others' maxima, so that as a rule one block of it is read again (all of them cost
// 16 % more traffic at 131072 values and k = 5).  What reaches T goes into a list and is put in order by
// counting.  Where most lanes' maxima are one value (a mask that leaves little), the list takes what is
// above it and the first places that hold it.  If the list runs over, every wave keeps its k best
// in order, entry i in lane i, and goes through its values once more; they come in rising order of their
// index, so most blocks are dismissed by one comparison.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/holmes_ckks.h"
#include "internal.hpp"

namespace hck {
namespace {

constexpr int kWaves = 4, kVecs = 4;  // waves of a workgroup, 16-byte pieces of a lane in flight (twice that for long rows)
constexpr int64_t kLastCache = 256 << 20;
constexpr int kMaxTop = 32, kMaxSplits = 64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct ScoreArgs {
  const void* x;
  const long long* tokens;  // null: no given tokens
  float *given, *entropy, *top_logs;
  long long* top_ids;
  float* part;  // with splits > 1: [row][split] of (r, l, s, 0), then [row][split][top] of keys and indexes, 64 bits each
  long long row_stride;
  int rows, vocab, top, splits;
};

// Unsigned numbers in the order of the values: NaN above all, -0 as 0, nothing maps to 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k == 0xffffffffu ? 0x7fc00000u : (k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ float finite_or_zero(float m) { return fabsf(m) == INFINITY ? 0.f : m; }

// (reference, sum, weighted sum) of a part of a row; r = -inf: no finite value met, sums against 0.  The reference is a
// value of the row and is taken off before log2 e is multiplied in: scaled first, a row of the type's lowest value
// would overflow, and one product's rounding would be of the values' size and not of their differences'.
struct Sums {
  float r = -INFINITY, l = 0.f, s = 0.f;
  __device__ __forceinline__ void rebase(float to) {
    if (to == r) return;
    // no exponent below -2000, so that l d is a number
    const float d = fmaxf((finite_or_zero(r) - finite_or_zero(to)) * kLog2e, -2000.f);
    const float f = r == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(d);  // nothing but zeros to scale
    s = f * (s + (l == 0.f ? 0.f : l * d));
    l *= f;
    r = to;
  }
  __device__ __forceinline__ void add(Sums o) {
    const float to = fmaxf(r, o.r);
    rebase(to);
    o.rebase(to);
    l += o.l;
    s += o.s;
  }
};

// A wave's k best: lane i holds the i-th.
struct Best {
  uint32_t key = 0, index = 0xffffffffu;
  uint32_t last_key = 0, last_index = 0xffffffffu;  // the k-th, in every lane
  __device__ __forceinline__ static bool before(uint32_t ak, uint32_t ai, uint32_t bk, uint32_t bi) {
    return ak > bk || (ak == bk && ai < bi);
  }
  // Offers a value of every lane (key 0: none).
  __device__ __forceinline__ void offer(uint32_t k, uint32_t i, int top) {
    const int lane = threadIdx.x & 63;
    unsigned long long left = __ballot(k != 0 && before(k, i, last_key, last_index));
    while (left) {
      const int from = __ffsll((unsigned long long)left) - 1;
      const uint32_t nk = __builtin_amdgcn_readlane(k, from), ni = __builtin_amdgcn_readlane(i, from);
      const int at = __popcll(__ballot(before(key, index, nk, ni)));
      const uint32_t uk = __shfl_up(key, 1), ui = __shfl_up(index, 1);
      if (lane > at) key = uk, index = ui;
      if (lane == at) key = nk, index = ni;
      if (lane >= top) key = 0, index = 0xffffffffu;
      last_key = __builtin_amdgcn_readlane(key, top - 1);
      last_index = __builtin_amdgcn_readlane(index, top - 1);
      left &= left - 1;
      left &= __ballot(before(k, i, last_key, last_index));
    }
  }
};

template <typename T>
__device__ __forceinline__ float element(u32x4 v, int e) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(v[e]);
  } else if constexpr (__is_same(T, __bf16)) {
    return __uint_as_float((e & 1) ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
  } else {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(v[e / 2] >> (16 * (e & 1))));
  }
}

// The given token of a row and its logit, asked for before the row's work so that both are there at its end.
template <typename T>
struct Given {
  long long token = -1;
  float logit = 0.f;
  __device__ __forceinline__ Given() {}
  __device__ __forceinline__ Given(const ScoreArgs& A, long long row) {
    if (!A.tokens) return;
    token = A.tokens[row];
    if (token >= 0 && token < A.vocab) logit = (float)((const T*)A.x)[row * A.row_stride + token];
  }
};

template <typename T>
__device__ __forceinline__ void finish(const ScoreArgs& A, long long row, const Given<T>& given, const Sums& a,
                                       unsigned long long best) {
  const int lane = threadIdx.x & 63;
  const float ref = finite_or_zero(a.r);
  const float log = a.l == 0.f ? 0.f : __builtin_amdgcn_logf(a.l);  // a row without a finite value
  // No probability is above 1 and no entropy below 0, though their last bits might say so (NaN stays).
  auto most0 = [](float x) { return x > 0.f ? 0.f : x; };
  if (lane == 0) {
    A.entropy[row] = -most0(((a.l == 0.f ? 0.f : a.s / a.l) - log) * kLn2);
    if (A.tokens) {
      float lp = 0.f;
      if (given.token >= A.vocab) lp = __uint_as_float(0x7fc00000u);
      else if (given.token >= 0) lp = most0(__builtin_fmaf(-log, kLn2, given.logit - ref));
      A.given[row] = lp;
    }
  }
  if (lane < A.top) {
    A.top_ids[row * A.top + lane] = 0xffffffffu - (uint32_t)best;
    A.top_logs[row * A.top + lane] = most0(__builtin_fmaf(-log, kLn2, value_of((uint32_t)(best >> 32)) - ref));
  }
}

// f over the wave's lanes, in every lane: within 16 lanes by turning, then over the 16s.
template <typename F>
__device__ __forceinline__ uint32_t over_lanes(uint32_t x, F f) {
  x = f(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x121, 0xf, 0xf, true));
  x = f(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x122, 0xf, 0xf, true));
  x = f(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xf, 0xf, true));
  x = f(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xf, 0xf, true));
  const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = f(p[0], p[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return f(q[0], q[1]);
}
__device__ __forceinline__ Sums over_lanes(Sums a) {
  auto larger = [](uint32_t x, uint32_t y) { return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y))); };
  auto plus = [](uint32_t x, uint32_t y) { return __float_as_uint(__uint_as_float(x) + __uint_as_float(y)); };
  a.rebase(__uint_as_float(over_lanes(__float_as_uint(a.r), larger)));
  a.l = __uint_as_float(over_lanes(__float_as_uint(a.l), plus));
  a.s = __uint_as_float(over_lanes(__float_as_uint(a.s), plus));
  return a;
}

// The larger of two in one instruction, b of a NaN and b (fmaxf of bits just shifted into place takes another
// to make a number of them first).
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }

// A lane's largest value, the block that it is in and the largest value of the other blocks.
struct Most {
  float top = -INFINITY, second = -INFINITY;
  int block = -1;
  __device__ __forceinline__ void note(float m, int b) {
    second = fmaxf(second, fminf(top, m));
    block = m > top ? b : block;
    top = fmaxf(top, m);
  }
};

// `N` values of the lane, all of block b, into its sums and maximum.
template <int N, typename V>
__device__ __forceinline__ void take(Sums& a, Most& most, int b, V value) {
  float m = -INFINITY;
#pragma unroll
  for (int n = 0; n < N; ++n) m = larger(m, value(n));
  most.note(m, b);
  a.rebase(fmaxf(a.r, m));
  const float ref = finite_or_zero(a.r);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const float t = (value(n) - ref) * kLog2e;
    const float e = __builtin_amdgcn_exp2f(t);
    a.l += e;
    a.s = __builtin_fmaf(e, fmaxf(t, -1000.f), a.s);  // 2^-inf counts nothing, and 0 * -inf would
  }
}

constexpr int kThreads = 64 * kWaves, kList = 256;

// The candidates of a workgroup for the top values.
struct Candidates {
  uint32_t most[kThreads];             // every thread's largest key
  unsigned long long list[kList], best[kMaxTop];
  int count, hot[64], block[64];       // threads that reach a key, and the block to look through, -2: all
  __device__ __forceinline__ static unsigned long long order(uint32_t key, uint32_t index) {
    return (unsigned long long)key << 32 | (0xffffffffu - index);  // larger: before
  }
  __device__ __forceinline__ static uint32_t key(unsigned long long o) { return (uint32_t)(o >> 32); }
  __device__ __forceinline__ static uint32_t index(unsigned long long o) { return 0xffffffffu - (uint32_t)o; }

  // A key that `top` threads' largest reach, as large as a few more allow, and how many do.  Where many threads' largest
  // are alike there (a mask that leaves little), the key after it, with `tied`: fewer than `top` threads reach that, and
  // of the values just below it the first in the row's order are wanted.
  __device__ __forceinline__ uint32_t reach(uint32_t mine, uint32_t second, int where, int top, int& threads, bool& tied) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    most[threadIdx.x] = mine;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    uint32_t k[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) k[w] = most[64 * w + lane];
    // the bits that all keys share come first
    uint32_t most_of = k[0], least_of = k[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) most_of = max(most_of, k[w]), least_of = min(least_of, k[w]);
    most_of = over_lanes(most_of, [](uint32_t x, uint32_t y) { return max(x, y); });
    least_of = over_lanes(least_of, [](uint32_t x, uint32_t y) { return min(x, y); });
    most_of = __builtin_amdgcn_readfirstlane(most_of), least_of = __builtin_amdgcn_readfirstlane(least_of);
    const uint32_t differ = most_of ^ least_of;
    uint32_t bit = differ ? 0x80000000u >> __builtin_clz(differ) : 0;
    uint32_t t = bit ? most_of & ~(2 * bit - 1) : most_of;
    threads = kThreads;
    for (; bit != 0 && threads > top + 3; bit >>= 1) {
      int n = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) n += __popcll(__ballot(k[w] >= (t | bit)));
      if (n >= top) t |= bit, threads = n;
    }
    tied = threads > 64 && t != 0xffffffffu;
    if (tied) {
      ++t, threads = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) threads += __popcll(__ballot(k[w] >= t));
    }
    int before = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (w < wave) before += __popcll(__ballot(k[w] >= t));
    const unsigned long long here = __ballot(mine >= t);
    const int at = before + __builtin_amdgcn_mbcnt_hi((uint32_t)(here >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)here, 0));
    if (mine >= t && at < 64) hot[at] = threadIdx.x, block[at] = second >= t ? -2 : where;
    __syncthreads();
    return t;
  }
  __device__ __forceinline__ void offer(uint32_t k, uint32_t i, uint32_t least) {
    if (k < least) return;
    const int at = atomicAdd(&count, 1);
    if (at < kList) list[at] = order(k, i);
  }
  // The list's first `top` in order; false: it does not hold them.
  __device__ __forceinline__ bool sort(int top) {
    __syncthreads();
    const int n = count;
    if (n < top || n > kList) return false;
    if ((int)threadIdx.x < n) {
      const unsigned long long mine = list[threadIdx.x];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += list[i] > mine;
      if (rank < top) best[rank] = mine;
    }
    __syncthreads();
    return true;
  }
};
static_assert(kList <= kThreads, "a thread an entry");

template <typename T>
__device__ __forceinline__ u32x4 nothing() {
  if constexpr (sizeof(T) == 4) return u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
  else if constexpr (__is_same(T, __bf16)) return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
  else return u32x4{0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u};
}

// kVecs: 16-byte pieces of a lane in flight.  ONCE: the logits are more than the last cache holds, and loaded past it.
template <typename T, int kVecs, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_scores(ScoreArgs A) {
  constexpr int kPer = 16 / sizeof(T);  // values of a 16-byte piece
  __shared__ float s_sums[kWaves][3];
  __shared__ Candidates C;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long row = blockIdx.y + (long long)blockIdx.z * 32768;
  if (row >= A.rows) return;
  const T* x = (const T*)A.x + row * A.row_stride;
  const Given<T> given = A.splits == 1 ? Given<T>(A, row) : Given<T>();
  // values before the first 16-byte border, whole pieces, and the rest
  const int head = min(A.vocab, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
  const int pieces = (A.vocab - head) / kPer, tail = head + pieces * kPer;
  const int left = A.vocab - tail;  // (tail + lane may pass 31 bits)
  const u32x4* body = reinterpret_cast<const u32x4*>(x + head);
  const int blocks = (pieces + 64 * kVecs - 1) / (64 * kVecs);
  const int first = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + wave), stride = A.splits * kWaves;
  const bool heads = first == 0 && head > 0, tails = first == stride - 1 && left > 0;
  Sums a;
  Most most;
  if (heads) take<1>(a, most, -1, [&](int) { return lane < head ? (float)x[lane] : -INFINITY; });
  for (int bl = first; bl < blocks; bl += stride) {
    u32x4 v[kVecs];
    const int p0 = bl * 64 * kVecs + lane;
    if (bl * 64 * kVecs + 64 * kVecs <= pieces) {
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        if constexpr (ONCE) v[j] = __builtin_nontemporal_load(body + p0 + 64 * j);
        else v[j] = body[p0 + 64 * j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        const int p = p0 + 64 * j;
        v[j] = nothing<T>();
        if (p < pieces) v[j] = body[p];
      }
    }
    take<kVecs * kPer>(a, most, bl, [&](int n) { return element<T>(v[n / kPer], n % kPer); });
  }
  if (tails) take<1>(a, most, -1, [&](int) { return lane < left ? (float)x[tail + lane] : -INFINITY; });

  bool listed = true;
  // A thread a value and all of them listed: where fewer threads than `top` have a piece, which leaves no key to reach
  // (8 bf16 rows of 126, top 17: 5.9 us, 20.5 us by the walk below), and where ranking a half of the list costs less
  // than looking for one (1132 fp32 rows of 126, top 17: 7.1 us against 8.6; of 256, top 20: 13.6 us against 8.8).
  if (A.top > 0 && A.vocab <= kList && (A.vocab <= kList / 2 || pieces < A.top)) {
    if (threadIdx.x == 0) C.count = A.vocab;
    if ((int)threadIdx.x < A.vocab) C.list[threadIdx.x] = C.order(key_of((float)x[threadIdx.x]), threadIdx.x);
    listed = C.sort(A.top);
  } else if (A.top > 0) {
    int threads;
    bool tied;
    const bool nan = a.l != a.l;
    const uint32_t least = C.reach(nan ? 0xffffffffu : key_of(most.top), nan ? 0xffffffffu : key_of(most.second), most.block,
                                   A.top, threads, tied);
    listed = threads <= 64;
    if (listed) {
      const int per = (blocks - (int)blockIdx.x * kWaves + stride - 1) / stride * kVecs;  // pieces of a thread, at most
      for (int i = threadIdx.x; i < threads * per; i += kThreads) {
        const int t = C.hot[i / per], n = i % per, only = C.block[i / per];
        const int bl = (int)blockIdx.x * kWaves + (t >> 6) + n / kVecs * stride, p = bl * 64 * kVecs + (t & 63) + 64 * (n % kVecs);
        if ((only != -2 && only != bl) || p >= pieces) continue;
        const u32x4 x4 = body[p];
#pragma unroll
        for (int e = 0; e < kPer; ++e) C.offer(key_of(element<T>(x4, e)), (uint32_t)(head + p * kPer + e), least);
      }
      if (heads && lane < head) C.offer(key_of((float)x[lane]), (uint32_t)lane, least - tied);
      if (tied && wave == 0) {  // the workgroup's first 64 values behind the head
        const int i = head + first * 64 * kVecs * kPer + lane;
        if (i < tail) {
          const uint32_t k = key_of((float)x[i]);
          if (k == least - 1) C.offer(k, (uint32_t)i, k);
        }
      }
      if (tails && lane < left) C.offer(key_of((float)x[tail + lane]), (uint32_t)(tail + lane), least);
      listed = C.sort(A.top);
    }
  }
  if (!listed) {  // the same for all threads
    __syncthreads();
    Best best;
    auto offer = [&](bool there, float value, int index) { best.offer(there ? key_of(value) : 0, (uint32_t)index, A.top); };
    if (heads) offer(lane < head, lane < head ? (float)x[lane] : 0.f, lane);
    for (int bl = first; bl < blocks; bl += stride)
      for (int j = 0; j < kVecs; ++j) {
        const int p = bl * 64 * kVecs + lane + 64 * j;
        const u32x4 v = p < pieces ? body[p] : nothing<T>();
#pragma unroll
        for (int e = 0; e < kPer; ++e) offer(p < pieces, element<T>(v, e), head + p * kPer + e);
      }
    if (tails) offer(lane < left, lane < left ? (float)x[tail + lane] : 0.f, tail + lane);
    static_assert(kWaves * kMaxTop <= kList, "the waves' lists");
    if (lane < A.top) C.list[wave * kMaxTop + lane] = Candidates::order(best.key, best.index);
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < kWaves; ++w) {
        const unsigned long long o = lane < A.top ? C.list[w * kMaxTop + lane] : 0;
        best.offer(Candidates::key(o), Candidates::index(o), A.top);
      }
      if (lane < A.top) C.best[lane] = Candidates::order(best.key, best.index);
    }
  }
  a = over_lanes(a);
  if (lane == 0) s_sums[wave][0] = a.r, s_sums[wave][1] = a.l, s_sums[wave][2] = a.s;
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < kWaves; ++w) {
    Sums o;
    o.r = s_sums[w][0], o.l = s_sums[w][1], o.s = s_sums[w][2];
    a.add(o);
  }
  if (A.splits == 1) return finish<T>(A, row, given, a, lane < A.top ? C.best[lane] : 0);
  const long long part = row * A.splits + blockIdx.x;
  float* sums = A.part + part * 4;
  unsigned long long* tops = (unsigned long long*)(A.part + (long long)A.rows * A.splits * 4) + part * A.top;
  if (lane == 0) sums[0] = a.r, sums[1] = a.l, sums[2] = a.s;
  if (lane < A.top) tops[lane] = C.best[lane];
}

// Joins the parts of a row, one workgroup a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_join(ScoreArgs A) {
  __shared__ Candidates C;
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const unsigned long long* tops = (const unsigned long long*)(A.part + (long long)A.rows * A.splits * 4) + row * A.splits * A.top;
  const Given<T> given(A, row);
  Sums a;
  if (lane < A.splits) {
    const float* p = A.part + (row * A.splits + lane) * 4;
    a.r = p[0], a.l = p[1], a.s = p[2];
  }
  if (A.top > 0) {
    constexpr int kMost = kMaxSplits * kMaxTop / kThreads;
    const int all = A.splits * A.top;
    unsigned long long o[kMost], most = 0;
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
      const int e = threadIdx.x + kThreads * j;
      o[j] = e < all ? tops[e] : 0;
      most = o[j] > most ? o[j] : most;
    }
    int threads;
    bool tied;
    const uint32_t least = max(1u, C.reach(Candidates::key(most), 0, -1, A.top, threads, tied));
    uint32_t tie = 0, from = 0xffffffffu;  // the key below `least`, and its first places (larger: earlier)
    if (tied && least > 1) {
      tie = least - 1;
      uint32_t place = 0;
#pragma unroll
      for (int j = 0; j < kMost; ++j) place = Candidates::key(o[j]) == tie ? max(place, (uint32_t)o[j]) : place;
      from = max(1u, C.reach(place, 0, -1, A.top, threads, tied));
    }
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
      const uint32_t k = Candidates::key(o[j]);
      C.offer(k, Candidates::index(o[j]), tie && k == tie && (uint32_t)o[j] >= from ? tie : least);
    }
    if (!C.sort(A.top)) {
      Best best;
      if (threadIdx.x < 64) {
        for (int e = lane; e - lane < all; e += 64) {
          const unsigned long long n = e < all ? tops[e] : 0;
          best.offer(Candidates::key(n), Candidates::index(n), A.top);
        }
        if (lane < A.top) C.best[lane] = Candidates::order(best.key, best.index);
      }
    }
  }
  if (threadIdx.x >= 64) return;
  finish<T>(A, row, given, over_lanes(a), lane < A.top ? C.best[lane] : 0);
}

// Parts of a row: workgroups for all 256 compute units four times, none with less than one block a wave.
int splits_of(int64_t rows, int vocab, int size) {
  const int64_t want = (1024 + rows - 1) / std::max<int64_t>(rows, 1);
  const int64_t block = (int64_t)64 * kVecs * 16 / size, most = std::max<int64_t>(1, vocab / (block * kWaves));
  return (int)std::min<int64_t>(std::min<int64_t>(want, most), kMaxSplits);
}

int size_of(int type) { return type == HCK_F32 ? 4 : type == HCK_BF16 || type == HCK_F16 ? 2 : 0; }

template <typename T>
int launch(const ScoreArgs& A, hipStream_t s) {
  const int gy = std::min(A.rows, 32768), gz = (A.rows + 32767) / 32768;
  // long rows in many workgroups: 4096 bf16 rows of 131072 take 192 us with 4 pieces through the caches, 173 us with 8
  // past them; 61 rows of 50021, in short parts, 14.0 and 14.7 us
  const dim3 grid(A.splits, gy, gz);
  if ((int64_t)A.rows * A.vocab * (int64_t)sizeof(T) > kLastCache && A.splits == 1) k_scores<T, 2 * kVecs, true><<<grid, kThreads, 0, s>>>(A);
  else k_scores<T, kVecs, false><<<grid, kThreads, 0, s>>>(A);
  HCK_CHECK_LAUNCH();
  if (A.splits > 1) {
    k_join<T><<<A.rows, kThreads, 0, s>>>(A);
    HCK_CHECK_LAUNCH();
  }
  return HCK_OK;
}

}  // namespace
}  // namespace hck

extern "C" size_t hck_token_scores_workspace_bytes(int64_t rows, int vocab, int type, int top) {
  if (rows < 1 || rows > (1 << 30) || vocab < 1 || top < 0 || top > hck::kMaxTop || !hck::size_of(type)) return 0;
  const int splits = hck::splits_of(rows, vocab, hck::size_of(type));
  return splits == 1 ? 0 : (size_t)rows * splits * (4 + 2 * top) * sizeof(float);
}

extern "C" int hck_token_scores(const void* logits, int type, int64_t rows, int vocab, int64_t row_stride,
                                const int64_t* tokens, int top, float* given, float* entropy, int64_t* top_ids,
                                float* top_logs, void* workspace, size_t workspace_bytes, void* stream) {
  if (!hck::size_of(type)) return HCK_ERR_UNSUPPORTED;
  if (rows < 0 || rows > (1 << 30) || vocab < 1 || top < 0 || top > hck::kMaxTop || top > vocab) return HCK_ERR_ARG;
  if (rows == 0) return HCK_OK;
  if (!logits || !entropy || (tokens && !given) || (top && (!top_ids || !top_logs))) return HCK_ERR_ARG;
  if ((uintptr_t)logits % hck::size_of(type) || (uintptr_t)workspace % 16) return HCK_ERR_ARG;
  const size_t need = hck_token_scores_workspace_bytes(rows, vocab, type, top);
  if (need > workspace_bytes || (need && !workspace)) return HCK_ERR_WORKSPACE;
  hck::ScoreArgs A{};
  A.x = logits;
  A.tokens = (const long long*)tokens;
  A.given = given;
  A.entropy = entropy;
  A.top_logs = top_logs;
  A.top_ids = (long long*)top_ids;
  A.part = (float*)workspace;
  A.row_stride = row_stride;
  A.rows = (int)rows;
  A.vocab = vocab;
  A.top = top;
  A.splits = hck::splits_of(rows, vocab, hck::size_of(type));
  hipStream_t s = (hipStream_t)stream;
  if (type == HCK_BF16) return hck::launch<__bf16>(A, s);
  if (type == HCK_F16) return hck::launch<_Float16>(A, s);
  return hck::launch<float>(A, s);
}
