// What the two kernels of attention over 4-bit pages share (kv4_attend.hip: few rows, kv4_prompt.hip: many):
// their arguments, the sharing out of the work, and the arithmetic of a softmax in one pass.
#pragma once
#include "kv4.hpp"

#include <algorithm>

#include "../../include/holmes_ckks.h"
#include "internal.hpp"

namespace hck {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kUnit = 64;   // tokens that a wave takes at a time: half a page
constexpr int kWaves = 4;
constexpr int kComputeUnits = 256;
constexpr int kFew = 16;    // rows of k_attend's workgroup
// Exponentials are taken times 2^24, so that those from 2^-126 to 2^-150 of a row's largest, which the
// exponential instruction gives as 0, still count where every larger one meets a value of 0.
constexpr float kLift = 24.f;
// Sums of such exponentials and values below 6 2^72 stay finite over 2^29 tokens of a wave.  Where a token that is seen
// has a larger unit (a scale byte of kLargeByte or more; values reach 6 2^125), the sums of its run of 32 dims go over to
// values times 2^-56, and its scale bytes are that much less from there on (1 at the least: values below 2^-69 no longer
// count beside those of 2^73).
constexpr int kLargeByte = 200, kDown = 56;
constexpr float kDownBy = 0x1p-56f, kUpBy = 0x1p56f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttendArgs {
  const uint8_t* pool;
  const void* q;
  const int* table;
  const int* lengths;
  const int* starts;   // null: sequence b has the one query b
  void* out;
  float *lse, *low, *high;  // [token][query head]; low, high nullable
  // with `join`: [slot][row] of (m, l, low, runs that are summed times 2^-56, a bit each), [slot][row][D] of sums, and
  // [tile][head] of (first slot, slots)
  float *stat, *sums;
  int* plan;
  long long q_ts, q_hs, tokens, pages;
  long long table_stride;
  int cols, heads, group, causal;
  int seqs, tiles;     // tiles of rows that the longest sequence can have
  int size, rows;      // rows of a tile, and of a slot
  int slots, least;    // workgroups to share the work out to, units that are not worth sharing
  int join, once;      // once: no key or value is read twice, and there is room for more than the L2s hold (Way::once)
  float scale;
};

// The rows of one sequence: query tokens [q0, q0 + nq), each with `group` heads, row = query * group + head.
struct Rows {
  int q0, nq, rows, length;
  Rows() = default;
  __device__ __forceinline__ Rows(const AttendArgs& A, int b) {
    long long first = b, last = b + 1;
    if (A.starts) first = A.starts[b], last = A.starts[b + 1];
    first = max(first, 0ll);
    q0 = (int)first;
    nq = (int)max(min(last, A.tokens) - first, 0ll);
    length = (int)min((long long)max(A.lengths[b], 0), (long long)A.cols * kPageTokens);
    count(A);
  }
  __device__ __forceinline__ void count(const AttendArgs& A) {
    rows = (int)min((long long)nq * A.group, (long long)A.tiles * A.size);
  }
  // those that one lane has, for all
  __device__ __forceinline__ void of_lane(const AttendArgs& A, int lane) {
    q0 = __builtin_amdgcn_readlane(q0, lane);
    nq = __builtin_amdgcn_readlane(nq, lane);
    length = __builtin_amdgcn_readlane(length, lane);
    count(A);
  }
  // tokens that row r sees
  __device__ __forceinline__ int seen(const AttendArgs& A, int r) const {
    return A.causal ? max(0, min(length, length - nq + r / A.group + 1)) : length;
  }
};

// A workgroup's work: a tile of rows, a key head, and a part of the units of 64 tokens that they see.
struct Item {
  int b, tile, h, u0, u1, slot, slots;
  Rows rows;
  // into scalar registers
  __device__ __forceinline__ void uniform() {
    b = __builtin_amdgcn_readfirstlane(b), tile = __builtin_amdgcn_readfirstlane(tile), h = __builtin_amdgcn_readfirstlane(h);
    u0 = __builtin_amdgcn_readfirstlane(u0), u1 = __builtin_amdgcn_readfirstlane(u1);
    slot = __builtin_amdgcn_readfirstlane(slot), slots = __builtin_amdgcn_readfirstlane(slots);
  }
};

// The units that a tile's rows see, -1: no rows.
__device__ __forceinline__ int units_of(const AttendArgs& A, const Rows& R, int pair) {
  const int first = (pair % A.tiles) * A.size;
  if (first >= R.rows) return -1;
  return (R.seen(A, min(first + A.size, R.rows) - 1) + kUnit - 1) / kUnit;
}

// Sums of the lanes up to each: by 1, 2, 4 and 8 within 16, then the 16s' last lanes onwards.
__device__ __forceinline__ int upto_lane(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}
__device__ __forceinline__ int over_wave(int x) { return __builtin_amdgcn_readlane(upto_lane(x), 63); }

// Where the join finds the slots of a tile and head, from the workgroup that has their first.
__device__ __forceinline__ void publish(const AttendArgs& A, const Item& it) {
  if (!A.join || it.u0 != 0 || threadIdx.x != 0) return;
  int* to = A.plan + 2 * ((long long)(it.b * A.tiles + it.tile) * A.heads + it.h);
  to[0] = it.slot, to[1] = it.slots;
}

constexpr int kPairs = 8;  // tiles of rows that a lane looks through to share the work out

__device__ __forceinline__ int ceil_div(int n, int d) { return (int)(((uint32_t)n + (uint32_t)d - 1) / (uint32_t)d); }

// Which part of the work is workgroup w's.  Lengths are on the device, so every wave works it out: with
// all tiles' units in its lanes, a share is the smallest (to a sixteenth) for which the parts, whole shares
// of a tile and its rest, are no more than the workgroups that run at once.  Later tiles, which see more,
// come first.  (A key head's workgroups lie `heads` apart: with 8 heads each XCD has one, and its cache that
// head's keys and values.  The heads of a page side by side on one XCD, for the address translation, won 2 % of
// 48 long histories and lost 20 % of 32 uneven ones.)
__device__ __forceinline__ bool locate(const AttendArgs& A, int w, Item& it) {
  const int pairs = A.seqs * A.tiles, lane = threadIdx.x & 63;
  if (!A.join) {
    const int r = w / A.heads;
    it.h = w % A.heads;
    it.slot = w, it.slots = 1;
    const int p = pairs - 1 - r;
    it.b = p / A.tiles, it.tile = p % A.tiles;
    it.u0 = 0, it.u1 = 0x7fffffff;
    it.rows = Rows(A, it.b);
    it.rows.of_lane(A, 0);
    return true;
  }
  const int per = (pairs + 63) / 64;
  int n[kPairs];
  Rows R[kPairs] = {};
  int whole = 0, rest = 0;  // the units' sum, by 2^15: a wave's lengths may pass 31 bits
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    n[j] = -1;
    if (j < per) {
      const int p = pairs - 1 - (lane * per + j);
      if (p >= 0) {
        R[j] = Rows(A, p / A.tiles);
        n[j] = units_of(A, R[j], p);
      }
      whole += max(n[j], 0) >> 15, rest += max(n[j], 0) & 0x7fff;
    }
  }
  const long long total = (((long long)over_wave(whole) << 15) + over_wave(rest)) * A.heads;
  const int base = (int)min(1ll << 26, max((long long)A.least, (total + A.slots - 1) / A.slots));
  const int fit = A.slots / A.heads;
  int share = base, mine = 0;
  for (int f = 16;; ++f) {
    share = (int)(((long long)base * f + 15) / 16);
    mine = 0;
#pragma unroll
    for (int j = 0; j < kPairs; ++j)
      if (j < per) mine += n[j] < 0 ? 0 : max(1, ceil_div(n[j], share));
    if (f == 32 || over_wave(mine) <= fit) break;
  }
  const int upto = upto_lane(mine), all = __builtin_amdgcn_readlane(upto, 63) * A.heads;
  if (w >= all) return false;
  const int r = w / A.heads;
  it.h = w % A.heads;
  it.slot = w;
  const int owner = __popcll(__ballot(upto <= r));  // the lane that holds part r
  int pair = 0, u0 = 0, count = 1, at = upto - mine;
  it.rows = R[0];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    if (j >= per) break;
    const int c = n[j] < 0 ? 0 : max(1, ceil_div(n[j], share));
    if (r >= at && r < at + c) pair = pairs - 1 - (lane * per + j), u0 = (r - at) * share, count = c, it.rows = R[j];
    at += c;
  }
  pair = __builtin_amdgcn_readlane(pair, owner);
  it.u0 = __builtin_amdgcn_readlane(u0, owner);
  it.slots = __builtin_amdgcn_readlane(count, owner);
  it.u1 = it.u0 + share;
  it.b = pair / A.tiles, it.tile = pair % A.tiles;
  it.rows.of_lane(A, owner);
  return true;
}

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

__device__ __forceinline__ bool has_large(uint32_t w) {  // a byte of kLargeByte or more, 255 among them
  return ((w & 0x7f7f7f7fu) + (256 - kLargeByte) * 0x01010101u) & w & 0x80808080u;
}
// Scale bytes of a run whose sums are held times 2^-56 (0, which stands for a run of NaN here, stays).
__device__ __forceinline__ uint32_t down(uint32_t w) {
  uint32_t to = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = (w >> (8 * j)) & 0xffu;
    to |= (b > kDown ? b - kDown : min(b, 1u)) << (8 * j);
  }
  return to;
}
// What sums of a run are multiplied by before they join others of which `any` has the runs held times 2^-56.
__device__ __forceinline__ float to_common(uint32_t mine, uint32_t any, int run) {
  return ((any & ~mine) >> run) & 1 ? kDownBy : 1.f;
}
__device__ __forceinline__ float back(uint32_t large, int run) { return (large >> run) & 1 ? kUpBy : 1.f; }

// Eight values of a query as one bf16 operand, or, of fp16, as the sum of two.
template <typename T>
__device__ __forceinline__ void query_parts(u32x4 raw, bf16x8& head, bf16x8& rest) {
  if constexpr (__is_same(T, _Float16)) {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    const f16x8 x = __builtin_bit_cast(f16x8, raw);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      head[k] = (__bf16)(float)x[k];
      rest[k] = (__bf16)((float)x[k] - (float)head[k]);
    }
  } else {
    head = __builtin_bit_cast(bf16x8, raw);
  }
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Reductions over the two and the four lanes that share a row: each swap leaves one operand's halves (of 32
// lanes, of 16) side by side with the other's.
template <typename F>
__device__ __forceinline__ float over_half(float x, F f) {
  const uint32_t a = __float_as_uint(x);
  const auto p = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return f(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
template <typename F>
__device__ __forceinline__ float over_g(float x, F f) {
  const uint32_t a = __float_as_uint(x);
  const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  return over_half(f(__uint_as_float(p[0]), __uint_as_float(p[1])), f);
}

__device__ __forceinline__ float fmax2(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float fmin2(float a, float b) { return fminf(a, b); }
// The larger and the smaller of two in one instruction (fmaxf of a matrix product's result takes another to make
// a number of it first).  Of a NaN and b: b, and -inf, which a row with a NaN never shows.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }
__device__ __forceinline__ float smaller(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, -INFINITY); }

// Sums are taken against the multiple of 8 at or above a row's running maximum: going over to another
// reference is an exact power of two, and seldom needed.  The factor of sums against the maximum a, now
// against b: 1 where nothing changed, also while nothing was seen (both -inf).
__device__ __forceinline__ float above(float m) { return 8.f * __builtin_ceilf(0.125f * m); }
__device__ __forceinline__ float rebase(float a, float b) {
  return a == b ? 1.f : __builtin_ldexpf(1.f, (int)(above(a) - above(b)));
}
__device__ __forceinline__ float reference(float m) { return fabsf(m) == INFINITY ? 0.f : above(m); }
// What a row's scores are multiplied by and what then comes off: scale log2 e and the reference of its maximum m, whose
// largest score is `raw`.  Beyond 2^27 a rounding of m is of the exponents' size, and what it took from the largest of
// scores of 1e10 would be an exponent of 2 in infinite sums.  There the factor is the next power of 2, with which
// both products are exact; that distances are up to twice theirs is less than the scores' own roundings.
constexpr float kFar = 1 << 27;
__device__ __forceinline__ void refer(float m, float raw, float scale2, float& ref, float& factor) {
  const bool far = fabsf(m) > kFar && fabsf(m) != INFINITY;
  const float power = __uint_as_float((__float_as_uint(scale2) + 0x7fffffu) & 0xff800000u);
  factor = far ? power : scale2;
  ref = (far ? raw * power : reference(m)) - kLift;
}
// log2 of a row's sum, against its reference.
__device__ __forceinline__ float log2_sum(float m, float l) {
  return fabsf(m) == INFINITY ? m + l : above(m) + (__builtin_amdgcn_logf(l) - kLift);
}

// What two numbers' nearest bf16 leave: a0 - h0 and a1 - h1, each in one instruction (times 1 and 0: exact).
// The factors (-1, 0) and (0, -1) come out of registers: as constants the compiler makes them one inline -1.0.
__device__ __forceinline__ uint32_t rests_of(float a0, float a1, uint32_t h) {
  uint32_t low, high;
  asm("s_mov_b32 %0, 0x0000bf80" : "=s"(low));
  asm("s_mov_b32 %0, 0xbf800000" : "=s"(high));
  const bf16x2 x = __builtin_bit_cast(bf16x2, h);
  return pack(__builtin_amdgcn_fdot2_f32_bf16(x, __builtin_bit_cast(bf16x2, low), a0, false),
              __builtin_amdgcn_fdot2_f32_bf16(x, __builtin_bit_cast(bf16x2, high), a1, false));
}

// A row's results from its sums: maximum m in units of log 2, sum l, `N` values from dim d0, times `up`.
template <typename T, int N, bool RANGE>
__device__ __forceinline__ void store_row(const AttendArgs& A, long long at, int dim, int d0, float m, float l, float low,
                                          const float* o, float up) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  typedef T vec __attribute__((ext_vector_type(N)));
  vec x;
#pragma unroll
  for (int c = 0; c < N; ++c) x[c] = (T)(o[c] * inv * up);
  *reinterpret_cast<vec*>((T*)A.out + at * dim + d0) = x;
  if (d0 == 0) {
    const bool bad = l != l;
    A.lse[at] = log2_sum(m, l) * kLn2;
    if constexpr (RANGE) A.low[at] = bad ? l : low * kLn2, A.high[at] = bad ? l : m * kLn2;
  }
}

// Waves of the kernels on a SIMD that the work is shared out for, from the registers of their dims and query parts (fp16
// queries at 128 dims: some 165 registers, which a third wave would fit as well; two were measured).
constexpr int waves_of_few(int dim, bool half) { return dim == 64 ? 4 : half ? 2 : 3; }
constexpr int waves_of_many(int dim) { return dim == 64 ? 3 : 2; }

// How a call is run, from what the host knows of it.
struct Way {
  bool few, join;
  int size, rows, least;
  int64_t tiles, slots, pairs, items, most_slots;  // most_slots: of one tile and head
  Way(int64_t seqs, int heads, int group, int dim, bool half, int most, int cols) {
    const int64_t all = (int64_t)most * group, units = std::max<int64_t>(1, (int64_t)cols * (kPageTokens / kUnit));
    // Few rows, or so little work that tiles of 16 rows on many compute units come sooner than tiles of 128 on few
    // (128 tokens, 32 heads of 128: 6.1 us against 9.3; 4 of 500: 38 us against 27).
    few = all <= 32 || seqs * heads * ((all + 15) / 16) * units <= 24576;
    // 256 rows make a unit's operands half as often, but one workgroup fills a compute unit: where there is one for
    // each and a quarter more (376 of them: 271 us against 292 with 128 rows; 256: 98 us against 90).
    size = few ? kFew : dim == 128 && seqs * heads * ((all + 255) / 256) >= kComputeUnits * 5 / 4 ? 256 : 128;
    tiles = (all + size - 1) / size;
    rows = (int)std::min<int64_t>(all, size);
    slots = kComputeUnits * (few ? waves_of_few(dim, half) : waves_of_many(dim) * 128 / size);
    pairs = seqs * tiles;
    // A join costs some 4 us, as much as four units a wave (8 heads, 1000 tokens: 9.0 us whole, 12.0 us in parts);
    // parts may be half of that where they leave compute units idle (4096 tokens: 12.0 us against 13.6).
    least = few && pairs * heads >= kComputeUnits ? 4 * kWaves : 8;
    // One sequence of two tiles or more for every workgroup that runs at once: half of its tiles' units on average, so
    // that no tile has more than an even share.
    const bool even = seqs == 1 && pairs * heads >= 2 * slots;
    join = pairs <= 64 * kPairs && units > (few ? 4 * kWaves : 8) && !even;
    most_slots = std::min((units + least - 1) / least, slots / heads + 1);
    items = !join ? pairs * heads : std::min(pairs * ((units + least - 1) / least), pairs + (slots + heads - 1) / heads) * heads;
  }
  // Whether loads go past the caches: one tile of rows for each sequence, so that nothing is read twice, and room for more
  // than the L2s hold.  Lengths are not known here; no more is held than the tables have room for, nor than the pool.
  // Single tokens, 8 key heads of 128, through the caches and past them, with what was read before in the last cache or
  // not: 4 sequences, 4 MB, 9.9 and 10.5 us (there or not); one of 36 MB 16.8 and 16.9 there, 18.0 and 16.7 not there; 32,
  // 63 MB, 20.4 and 20.5, 22.1 and 21.1; one of 143 MB 33.7 and 33.6, 38.9 and 34.9; 32, 209 MB, 41.6 and 43.5, 50.5 and
  // 50.2; 48, 418 MB, 89.0 and 79.8.
  bool once(int64_t seqs, int64_t cols, int64_t pages, int heads, int dim) const {
    return tiles == 1 && std::min(seqs * cols, pages) > kL2s / ((int64_t)heads * kv4_bytes(dim));
  }
  size_t bytes(int heads, int dim) const {
    return join ? (size_t)items * rows * (4 + dim) * sizeof(float) + (size_t)pairs * heads * 2 * sizeof(int) : 0;
  }
};

int launch_prompt(const AttendArgs& A, const Way& W, int head_dim, int type, hipStream_t s);

}  // namespace hck
