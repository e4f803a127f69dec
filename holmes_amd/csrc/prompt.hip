// Attention over whole prompts whose keys and values are as the projections left them, packed one behind the other.
//
//   s = scale q.k over the tokens of the query's sequence up to its own (or all of them), m = max s, l = sum exp(s - m),
//   out = sum exp(s - m) v / l, lse = m + log l
//
// One pass over the keys with a running m and l.  A workgroup of four waves has 128 rows (row = query * group + head, so the
// heads that share a key head are side by side, whatever their number), 32 to a wave, and takes 64 tokens at a time.  Both
// products are transposed, S^T = K Q^T and O^T = V^T P^T: the scores that a lane holds after the first are exactly the ones
// that the second wants of it, and a lane's scores are all of one row.
//
// Keys and values go from memory straight into LDS (two units, so that the next one is in flight), 16 bytes a lane, with the
// 16-byte pieces of a token put where the reads meet no bank twice: keys, read as they lie, at piece ^ token; values, read
// four tokens by 16 dims at a time through the transposing LDS read, at piece ^ 4 (token % 4).  What lies behind a
// sequence's end is out of the loads' bounds and becomes zeros.
//
// Probabilities are rounded to the values' type for the second product, for every caller: one part of 16 bits, which halves that
// product's matrix instructions against two.  Half a step each, so that an output's error is that of a
// sum of rounded terms, of the size of its own rounding where there are many (against 64 bits, relative to the outputs: 8192 tokens in
// bf16 1.70e-3, where probabilities of 32 bits leave 1.66e-3).  Rows of few tokens, where it would be half as
// much again, see them in units that others of their tile see in part: there the rounding's rest goes in as well, by a second
// product.  l, and with it lse, is the sum of the unrounded ones.
//
// What bounds it: per 64 tokens and 32 rows 32 matrix instructions (1024 of the SIMD's cycles at D = 128) and some 150 vector ones, 32 of
// them exponentials (730), of two waves that share a SIMD.  8192 tokens, 32 query heads over 8 key heads of 128, bf16: 555 GFLOP in
// 524 to 571 us on different cards, 0.97 to 1.06 PFLOP/s at the 1.95 GHz that the clock falls to; a bf16 8192^3 product runs at 1.23.  References of the
// exponentials are multiples of 8 in units of log 2, so that going over to another is an exact power of two and seldom done.
#include "prompt_way.hpp"

namespace hck {
namespace {

struct PromptArgs {
  const void *q, *k, *v;
  const int* starts;  // null: one sequence of all tokens
  void* out;
  float *lse, *low, *high;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, tokens;
  int seqs, heads, group, causal, most, tiles;  // tiles that the longest sequence can have
  // where tiles' units are shared out: units of a part, parts that a tile can have, and [slot][wave][piece][lane] of four floats,
  // of which the first piece is (m, l, least score, -) of the lane's row and the others are its sums
  int part, parts, items;
  f32x4* slots;
  float scale2;                                 // scale log2 e
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Eight;
template <>
struct Eight<__bf16> {
  typedef bf16x8 type;
};
template <>
struct Eight<_Float16> {
  typedef f16x8 type;
};

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ uint32_t pack_as(float a, float b) {
  typedef T two __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, two{(T)a, (T)b});
}

// The sign bits of those of two values that are an infinity or a NaN: an exponent of ones carries into the sign's bit.
template <typename T>
__device__ __forceinline__ uint32_t odd_values(uint32_t x) {
  constexpr uint32_t kExponent = __is_same(T, _Float16) ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t kOne = __is_same(T, _Float16) ? 0x04000400u : 0x00800080u;
  return ((x & kExponent) + kOne) & 0x80008000u;
}

// A sequence's tokens, and a tile of its rows.
struct Tile {
  int64_t first;
  int n, rows, tile;
};

__device__ __forceinline__ void sequence(const PromptArgs& A, int b, int64_t& first, int& n) {
  first = 0;
  int64_t last = A.tokens;
  if (A.starts) {
    first = max((int64_t)A.starts[b], (int64_t)0);
    last = min((int64_t)A.starts[b + 1], A.tokens);
  }
  n = (int)max(last - first, (int64_t)0);
}
__device__ __forceinline__ int rows_of(const PromptArgs& A, int n) { return min(n, A.most) * A.group; }

// Tile r of all sequences' tiles.  Of up to 64 sequences (a lane has one) the tiles with the highest numbers, which see most, come
// first: those of number t and above are sum max(0, tiles - t), and t is found by halving.  Of more, a sequence's last come first.
__device__ __forceinline__ bool locate_tile(const PromptArgs& A, int r, Tile& t) {
  int b = 0;
  const int lane = threadIdx.x & 63;
  auto count = [&](int b) {
    int64_t first;
    int n = 0;
    if (b < A.seqs) sequence(A, b, first, n);
    return (rows_of(A, n) + kTileRows - 1) / kTileRows;
  };
  int last = -1;
  if (A.seqs > 64) {
    for (b = 0;; b += 64) {
      if (b >= A.seqs) return false;
      const int mine = count(b + lane), upto = upto_lane(mine), all = __builtin_amdgcn_readlane(upto, 63);
      if (r < all) {
        const int owner = __popcll(__ballot(upto <= r));
        b += owner;
        r -= __builtin_amdgcn_readlane(upto - mine, owner);
        break;
      }
      r -= all;
    }
  } else if (A.seqs > 1) {
    const int mine = count(lane);
    if (r >= over_wave(mine)) return false;
    int at = 0, none = A.tiles;  // more than r tiles of number `at` and above; no more than r of `none`
    while (none - at > 1) {
      const int middle = (at + none) / 2;
      if (over_wave(max(0, mine - middle)) > r) at = middle;
      else none = middle;
    }
    r -= over_wave(max(0, mine - at - 1));
    const unsigned long long has = __ballot(mine > at);
    const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
    b = __builtin_ctzll(__ballot(mine > at && before == r));
    last = at;
  }
  sequence(A, b, t.first, t.n);
  t.rows = rows_of(A, t.n);
  const int tiles = (t.rows + kTileRows - 1) / kTileRows;
  if (last < 0 && r >= tiles) return false;
  t.tile = last < 0 ? tiles - 1 - r : last;
  return true;
}

template <int D>
struct Staged {
  static constexpr int kPieces = D / 8;  // of 16 bytes a token
  static constexpr int kEach = kUnit * kPieces / (64 * kPromptWaves);  // pieces of a thread
  static constexpr int kStep = 64 * kPromptWaves / kPieces;            // tokens between a thread's pieces
  static constexpr int kBytes = kUnit * D * 2;
  __device__ static int key_at(int token, int piece) {
    return token * kPieces + (piece ^ (D == 128 ? token & 15 : (token >> 1) & 7));
  }
  __device__ static int value_at(int token, int piece) {
    return token * kPieces + (piece ^ (D == 128 ? (token & 3) << 2 : ((token >> 1) & 1) << 2));
  }
};

typedef uint32_t rsrc_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
// 16 bytes for each lane from base + off into LDS, lane after lane from `to` on; zeros for what is out of the bounds.
// Written out, because the compiler waits for such loads before any transposing read; whoever issues them waits with
// all_loaded().  (m0 holds the address, a wait state ahead of its use; the bounds' registers may have been written by a vector
// instruction, five ahead.)
__device__ __forceinline__ void load_lds(uint32_t to, uint32_t off, rsrc_t from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(off), "s"(from) : "memory", "m0");
}
__device__ __forceinline__ void all_loaded() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ rsrc_t bounds(const char* base, int bytes) {
  const uint64_t at = (uint64_t)base;
  return rsrc_t{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu)),
                (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}

// A row's results from its sums: maximum m in units of log 2, sum l, dims 32 d + 8 i + 4 half .. from sums(d, i).
template <typename T, int D, bool RANGE, typename F>
__device__ __forceinline__ void write_row(const PromptArgs& A, int64_t at, int half, float m, float l, float low, float lift, F sums) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = (T*)A.out + at * D + 4 * half;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 x = sums(d, i) * inv;
      *reinterpret_cast<u32x2*>(out + 32 * d + 8 * i) = u32x2{pack_as<T>(x[0], x[1]), pack_as<T>(x[2], x[3])};
    }
  if (half) return;
  A.lse[at] = fabsf(m) == INFINITY ? m + l : (above(m) + (__builtin_amdgcn_logf(l) - lift)) * kLn2;
  if constexpr (RANGE) A.low[at] = l != l ? l : low * kLn2, A.high[at] = l != l ? l : m * kLn2;
}

// Exponentials are taken times 2^lift.  fp16: the largest is between 2^7 and 2^15, so that those down to 2^-21 of it at the least, and
// 2^-29 at the most, keep all bits, and those below 2^-32 may become 0.  bf16:
// such that their sum over n tokens is at most 1, and no sum of values overflows (by eights: references, which are multiples of
// 8, stay exact to 2^27).
template <typename T>
__device__ __forceinline__ float lift_of(int n) {
  return __is_same(T, _Float16) ? 15.f : -(float)((39 - __builtin_clz(n)) / 8 * 8);
}

__device__ __forceinline__ f32x4* slot_of(const PromptArgs& A, int item, int part, int h, int wave, int dim) {
  return A.slots + (((int64_t)item * A.parts + part) * A.heads + h) * (kPromptWaves * 64 * kPieces(dim)) + wave * 64 * kPieces(dim) +
         (threadIdx.x & 63);
}

// SPLIT: a workgroup takes a part of a tile's units; parts of a tile that has several are joined by k_whole_join.
template <typename T, int D, bool RANGE, bool SPLIT>
__global__ __launch_bounds__(64 * kPromptWaves, 2) void k_whole(PromptArgs A) {
  using S = Staged<D>;
  using vec = typename Eight<T>::type;
  constexpr int kSteps = D / 16, kTiles = D / 32;
  __shared__ u32x4 s_x[2][2][kUnit * S::kPieces];  // [turn][keys, values]

  Tile t;
  const int h = blockIdx.x % A.heads;
  // (neighbours are on different XCDs: parts next to each other would leave the first ones, of which there are most, to some)
  const int part = SPLIT ? blockIdx.x / A.heads / A.items : 0, item = blockIdx.x / A.heads % (SPLIT ? A.items : 0x7fffffff);
  if (!locate_tile(A, item, t)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int n = __builtin_amdgcn_readfirstlane(t.n), rows = __builtin_amdgcn_readfirstlane(t.rows);
  const int tile = __builtin_amdgcn_readfirstlane(t.tile);
  const int64_t first = t.first;
  auto sees = [&](int row) { return A.causal ? row / A.group + 1 : n; };
  const int most = sees(min(tile * kTileRows + kTileRows, rows) - 1);
  const int all = (most + kUnit - 1) / kUnit, begin = SPLIT ? part * A.part : 0;
  const int units = SPLIT ? part_end(all, A.part, A.parts, part) : all;
  if (SPLIT && part && begin >= all) return;
  const int mine = tile * kTileRows + wave * kRowsOfWave;
  const int last = mine < rows ? sees(min(mine + kRowsOfWave, rows) - 1) : 0;
  const int row = mine + (lane & 31);
  const bool live = row < rows;
  const int qi = live ? row / A.group : 0, qo = live ? row % A.group : 0;
  const int seen = live ? sees(row) : 0;

  // what a thread brings of each unit: pieces of tokens kStep apart
  const int token0 = threadIdx.x / S::kPieces, piece0 = threadIdx.x % S::kPieces;
  const uint32_t k_off = (uint32_t)(token0 * A.k_ts * 2) + (S::key_at(token0, piece0) - token0 * S::kPieces) * 16;
  const uint32_t v_off = (uint32_t)(token0 * A.v_ts * 2) + (S::value_at(token0, piece0) - token0 * S::kPieces) * 16;
  const uint32_t k_step = (uint32_t)(S::kStep * A.k_ts * 2), v_step = (uint32_t)(S::kStep * A.v_ts * 2);
  const char* kp = (const char*)A.k + (first * A.k_ts + h * A.k_hs) * 2;
  const char* vp = (const char*)A.v + (first * A.v_ts + h * A.v_hs) * 2;
  const uint32_t lds = lds_address(s_x) + wave * 1024;
  auto bring = [&](int u) {
    const int left = min(n - u * kUnit, kUnit);
    const uint32_t to = lds + (u & 1) * (2 * S::kBytes);
    const rsrc_t kr = bounds(kp + (int64_t)u * kUnit * A.k_ts * 2, (int)((left - 1) * A.k_ts * 2 + D * 2));
    const rsrc_t vr = bounds(vp + (int64_t)u * kUnit * A.v_ts * 2, (int)((left - 1) * A.v_ts * 2 + D * 2));
#pragma unroll
    for (int j = 0; j < S::kEach; ++j) {
      load_lds(to + j * (1024 * kPromptWaves), k_off + j * k_step, kr);
      load_lds(to + j * (1024 * kPromptWaves) + S::kBytes, v_off + j * v_step, vr);
    }
  };
  if (begin < units) bring(begin);

  vec q[kSteps];
  const T* qp = (const T*)A.q + (first + qi) * A.q_ts + (int64_t)(h * A.group + qo) * A.q_hs + half * 8;
  u32x4 raw[kSteps];  // (a lane without a row has the sequence's first, whose results it does not write)
#pragma unroll
  for (int s = 0; s < kSteps; ++s) raw[s] = *reinterpret_cast<const u32x4*>(qp + s * 16);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    // (used here, or every unit's first product would wait for these loads, and with them for the next unit's)
    asm volatile("" : "+v"(raw[s]));
    q[s] = __builtin_bit_cast(vec, raw[s]);
  }

  // Where the lane reads: keys of token lane % 32 (and 32 on); values of the tokens 4 half + lane % 16 / 4 (and 8 on), of
  // which lane i of 16 gets dim i.
  const int vt = 4 * half + ((lane & 15) >> 2), vc = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  const float lift = lift_of<T>(n);

  f32x16 acc[kTiles];
#pragma unroll
  for (int d = 0; d < kTiles; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  float top = -INFINITY, sum = 0.f, low = INFINITY;
  float ref = -lift, factor = A.scale2;

  // The unit's tokens from `skip` on: all 64 (skip 0), or, PARTLY, 32 of which some of the wave's rows do not see some.
  auto unit = [&](int u, int skip, auto PARTLY) {
    constexpr bool kPartly = decltype(PARTLY)::value;
    constexpr int kX = kPartly ? 1 : 2;  // 32 tokens each
    const u32x4 *ks = s_x[u & 1][0] + skip * S::kPieces, *vs = s_x[u & 1][1] + skip * S::kPieces;
    const int here = u * kUnit + skip;
    f32x16 c[kX];
#pragma unroll
    for (int x = 0; x < kX; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) c[x][i] = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int x = 0; x < kX; ++x) {
        const vec k = __builtin_bit_cast(vec, ks[S::key_at(32 * x + (lane & 31), 2 * s + half)]);
        c[x] = mfma32(k, q[s], c[x]);
      }
    if constexpr (!kPartly && D == 128) {
      // Six reads ahead of the products, which alone the compiler would not have (8192 tokens: 576 -> 566 us; at 64 dims,
      // with half the products for as many exponentials, it costs 4 %).
      __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
      for (int s = 0; s < 2 * kSteps - 6; ++s) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
    }
    if constexpr (kPartly) {
      const int base = here + 4 * half;  // of the lane's tokens base + 8 (i / 4) + i % 4
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool see = base + 8 * (i >> 2) + (i & 3) < seen;
        if constexpr (RANGE) low = see ? fminf(low, c[0][i]) : low;
        c[0][i] = see ? c[0][i] : -INFINITY;
      }
    } else if constexpr (RANGE) {
#pragma unroll
      for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int i = 0; i < 16; i += 2)
          low = __builtin_elementwise_minimum(__builtin_elementwise_minimum(low, c[x][i]), c[x][i + 1]);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < kX; ++x)
#pragma unroll
      for (int i = 0; i < 16; i += 2) mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx, c[x][i]), c[x][i + 1]);
    const float raw = over_half(mx, fmax2);
    mx = fmaxf(top, raw * A.scale2);
    const float f = rebase(top, mx);
    top = mx;
    if (__any(f != 1.f)) {
      if (f != 1.f) {
        refer(mx, raw, A.scale2, ref, factor);
        ref += kLift - lift;
      }
      sum *= f;
#pragma unroll
      for (int d = 0; d < kTiles; ++d) acc[d] *= f;
    }

    // the left operand of 16 tokens and 32 dims
    auto values = [&](int j, int d) {
      s16x4 x[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const u32x4* at = vs + S::value_at(16 * j + 8 * p + vt, 4 * d + vc);
        x[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)((const char*)at + (lane & 1) * 8));
      }
      const u32x2 a = __builtin_bit_cast(u32x2, x[0]), b = __builtin_bit_cast(u32x2, x[1]);
      return u32x4{a[0], a[1], b[0], b[1]};
    };
    // (a wave in its softmax and second product goes before one in its first, which only waits for the matrix unit: 582 -> 576 us)
    if constexpr (D == 128) __builtin_amdgcn_s_setprio(1);
    float part[2] = {0.f, 0.f};
    auto probabilities = [&](int j, u32x4& rest) {  // PARTLY: and what their rounding left over
      float e[8];
      u32x4 p;
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(c[j >> 1][8 * (j & 1) + i], factor, -ref));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = pack_as<T>(e[2 * i], e[2 * i + 1]);
        part[i & 1] += e[2 * i] + e[2 * i + 1];
        if constexpr (kPartly) {
          typedef T two __attribute__((ext_vector_type(2)));
          const uint32_t w = p[i];  // (a cast of the vector's element itself would be one of its first)
          const two near = __builtin_bit_cast(two, w);
          rest[i] = pack_as<T>(e[2 * i] - (float)near[0], e[2 * i + 1] - (float)near[1]);
        }
      }
      return p;
    };
    if constexpr (kPartly) {
      // Tokens that a row does not see have a probability of 0, and 0 times an infinity or a NaN is NaN.  Where there
      // is one it goes into the product as 0, and is then added to the rows that see it.
      uint32_t odd = 0;
#pragma unroll 4
      for (int i = 0; i < 32 * S::kPieces / 64; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= odd_values<T>(vs[i * 64 + lane][e]);
      if (__any(odd != 0)) {
#pragma unroll
        for (int j = 0; j < 2 * kX; ++j) {
          u32x4 rest;
          const u32x4 p = probabilities(j, rest);
#pragma unroll
          for (int d = 0; d < kTiles; ++d) {
            u32x4 v = values(j, d);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] &= ~((odd_values<T>(v[e]) >> 15) * 0xffffu);
            acc[d] = mfma32(__builtin_bit_cast(vec, v), __builtin_bit_cast(vec, p), acc[d]);
            acc[d] = mfma32(__builtin_bit_cast(vec, v), __builtin_bit_cast(vec, rest), acc[d]);
          }
        }
        sum += part[0] + part[1];
        if constexpr (D == 128) __builtin_amdgcn_s_setprio(0);
#pragma unroll 1
        for (int t = 0; t < 32; ++t)
#pragma unroll
          for (int d = 0; d < kTiles; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // dims 32 d + 8 i + 4 half ..
              typedef T four __attribute__((ext_vector_type(4)));
              const u32x2 w = *reinterpret_cast<const u32x2*>((const char*)(vs + S::value_at(t, 4 * d + i)) + half * 8);
              const four v = __builtin_bit_cast(four, w);
              const uint32_t o[2] = {odd_values<T>(w[0]), odd_values<T>(w[1])};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[d][4 * i + e] += here + t < seen && (o[e >> 1] >> (e & 1 ? 31 : 15) & 1) ? (float)v[e] : 0.f;
            }
        return;
      }
    }
#pragma unroll
    for (int j = 0; j < 2 * kX; ++j) {
      u32x4 rest;
      const u32x4 p = probabilities(j, rest);
#pragma unroll
      for (int d = 0; d < kTiles; ++d) {
        const vec v = __builtin_bit_cast(vec, values(j, d));
        acc[d] = mfma32(v, __builtin_bit_cast(vec, p), acc[d]);
        if constexpr (kPartly) acc[d] = mfma32(v, __builtin_bit_cast(vec, rest), acc[d]);
      }
    }
    sum += part[0] + part[1];
    if constexpr (D == 128) __builtin_amdgcn_s_setprio(0);
  };

  auto next = [&](int u) {
    all_loaded();  // this wave's, and after the barrier all waves'; which are also done with the unit before
    __syncthreads();
    if (u + 1 < units) bring(u + 1);
  };
  const int full = sees(tile * kTileRows) / kUnit;  // units that all of the tile's rows see
  int u = begin;
  for (; u < min(full, units); ++u) {
    next(u);
    unit(u, 0, std::false_type());
  }
  for (; u < units; ++u) {
    next(u);
#pragma unroll 1
    for (int skip = 0; skip < kUnit; skip += 32)
      if (u * kUnit + skip < last) unit(u, skip, std::true_type());
  }

  sum = over_half(sum, [](float a, float c) { return a + c; });
  if constexpr (RANGE) low = over_half(low, fmin2) * A.scale2;
  auto sums = [&](int d, int i) { return f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]}; };
  if (SPLIT && all > A.part) {
    f32x4* to = slot_of(A, item, part, h, wave, D);
    to[0] = f32x4{top, sum, low, 0.f};
#pragma unroll
    for (int d = 0; d < kTiles; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) to[64 * (1 + 4 * d + i)] = sums(d, i);
    return;
  }
  if (!live) return;
  write_row<T, D, RANGE>(A, (first + qi) * (int64_t)(A.heads * A.group) + h * A.group + qo, half, top, sum, low, lift, sums);
}

// The parts of a tile's rows, lane by lane as they were left.
template <typename T, int D, bool RANGE>
__global__ __launch_bounds__(64 * kPromptWaves) void k_whole_join(PromptArgs A) {
  constexpr int kTiles = D / 32;
  Tile t;
  const int h = blockIdx.x % A.heads, item = blockIdx.x / A.heads;
  if (!locate_tile(A, item, t)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int end = min(t.tile * kTileRows + kTileRows, t.rows) - 1;
  const int all = ((A.causal ? end / A.group + 1 : t.n) + kUnit - 1) / kUnit, parts = parts_of(all, A.part, A.parts);
  const int row = t.tile * kTileRows + wave * kRowsOfWave + (lane & 31);
  if (parts <= 1 || row >= t.rows) return;
  const int64_t apart = (int64_t)A.heads * (kPromptWaves * 64 * kPieces(D));
  const f32x4* from = slot_of(A, item, 0, h, wave, D);
  float top = -INFINITY, sum = 0.f, low = INFINITY;
#pragma unroll 4
  for (int p = 0; p < parts; ++p) top = fmaxf(top, from[p * apart][0]);
  f32x4 acc[kTiles * 4];
#pragma unroll
  for (int i = 0; i < kTiles * 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int p = 0; p < parts; ++p) {
    const f32x4 s = from[p * apart];
    const float f = rebase(s[0], top);
    sum += s[1] * f, low = fminf(low, s[2]);
#pragma unroll
    for (int i = 0; i < kTiles * 4; ++i) acc[i] += from[p * apart + 64 * (1 + i)] * f;
  }
  write_row<T, D, RANGE>(A, (t.first + row / A.group) * (int64_t)(A.heads * A.group) + h * A.group + row % A.group, half, top, sum, low,
                         lift_of<T>(t.n), [&](int d, int i) { return acc[4 * d + i]; });
}

template <typename T, int D>
int launch(const PromptArgs& A, const WholeWay& way, hipStream_t s) {
  const unsigned tiles = (unsigned)(way.items * A.heads);
  constexpr int kThreads = 64 * kPromptWaves;
  if (way.parts == 1) {
    if (A.low) k_whole<T, D, true, false><<<tiles, kThreads, 0, s>>>(A);
    else k_whole<T, D, false, false><<<tiles, kThreads, 0, s>>>(A);
    HCK_CHECK_LAUNCH();
    return HCK_OK;
  }
  if (A.low) k_whole<T, D, true, true><<<tiles * way.parts, kThreads, 0, s>>>(A);
  else k_whole<T, D, false, true><<<tiles * way.parts, kThreads, 0, s>>>(A);
  HCK_CHECK_LAUNCH();
  if (A.low) k_whole_join<T, D, true><<<tiles, kThreads, 0, s>>>(A);
  else k_whole_join<T, D, false><<<tiles, kThreads, 0, s>>>(A);
  HCK_CHECK_LAUNCH();
  return HCK_OK;
}

// Whether the products that WholeWay makes stay within 63 bits.  (2^40 rows are 2^47 bytes of outputs and more.)
bool countable(int64_t tokens, int64_t seqs, int64_t heads, int64_t group) {
  return seqs * heads <= INT32_MAX && heads * group <= INT32_MAX && tokens * (heads * group) <= 1ll << 40;
}

}  // namespace
}  // namespace hck

extern "C" size_t hck_prompt_attend_workspace_bytes(int64_t tokens, int seqs, int kv_heads, int group, int head_dim, int most,
                                                    int causal) {
  if (tokens < 1 || tokens > INT32_MAX || seqs < 1 || kv_heads < 1 || group < 1 || most < 1 ||
      (head_dim != 64 && head_dim != 128) || std::min<int64_t>(most, tokens) * group > INT32_MAX - 256 ||
      !hck::countable(tokens, seqs, kv_heads, group))
    return 0;
  return hck::WholeWay(tokens, seqs, kv_heads, group, (int)std::min<int64_t>(most, tokens), causal != 0).bytes(kv_heads, head_dim);
}

extern "C" int hck_prompt_attend(const void* queries, const void* keys, const void* values, int type, int64_t tokens,
                                 int kv_heads, int group, int head_dim, int64_t q_token_stride, int64_t q_head_stride,
                                 int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                 const int32_t* starts, int seqs, int most, int causal, double scale, void* out, float* lse,
                                 float* low, float* high, void* workspace, size_t workspace_bytes, void* stream) {
  if ((head_dim != 64 && head_dim != 128) || (type != HCK_BF16 && type != HCK_F16)) return HCK_ERR_UNSUPPORTED;
  if (tokens < 0 || tokens > INT32_MAX || kv_heads < 1 || group < 1 || (int64_t)kv_heads * group > INT32_MAX || seqs < 0 ||
      most < 0 || !((float)scale > 0.f && scale <= 0x1p126) || (low == nullptr) != (high == nullptr) ||
      !hck::countable(tokens, seqs, kv_heads, group))
    return HCK_ERR_ARG;
  if (!starts && seqs != 1) return HCK_ERR_ARG;
  most = (int)std::min<int64_t>(most, tokens);
  if (seqs == 0 || most == 0) return HCK_OK;
  if (!queries || !keys || !values || !out || !lse || (int64_t)most * group > INT32_MAX - 256) return HCK_ERR_ARG;
  if (((uintptr_t)queries | (uintptr_t)keys | (uintptr_t)values | (uintptr_t)out) % 16) return HCK_ERR_ARG;
  for (int64_t stride : {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride})
    if (stride % 8) return HCK_ERR_ARG;
  // a unit's loads count its bytes in 31 bits, and tell a sequence's end by them
  for (int64_t stride : {k_token_stride, v_token_stride})
    if (tokens > 1 && (stride < head_dim || stride > 1 << 23)) return HCK_ERR_ARG;
  hck::PromptArgs A = {};
  A.q = queries, A.k = keys, A.v = values, A.starts = starts, A.out = out, A.lse = lse, A.low = low, A.high = high;
  A.q_ts = q_token_stride, A.q_hs = q_head_stride, A.tokens = tokens;
  A.k_ts = tokens > 1 ? k_token_stride : head_dim, A.k_hs = k_head_stride;
  A.v_ts = tokens > 1 ? v_token_stride : head_dim, A.v_hs = v_head_stride;
  A.seqs = seqs, A.heads = kv_heads, A.group = group, A.causal = causal != 0, A.most = most;
  const hck::WholeWay way(tokens, seqs, kv_heads, group, most, causal != 0);
  if (!hck::fits_grid(way.items * way.parts * kv_heads, 64 * hck::kPromptWaves)) return HCK_ERR_ARG;
  const size_t need = way.bytes(kv_heads, head_dim);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return HCK_ERR_WORKSPACE;
  A.tiles = way.tiles, A.part = way.part, A.parts = way.parts, A.items = (int)way.items, A.slots = (hck::f32x4*)workspace;
  A.scale2 = (float)(scale * 1.4426950408889634);
  hipStream_t s = (hipStream_t)stream;
  if (head_dim == 128) return type == HCK_BF16 ? hck::launch<__bf16, 128>(A, way, s) : hck::launch<_Float16, 128>(A, way, s);
  return type == HCK_BF16 ? hck::launch<__bf16, 64>(A, way, s) : hck::launch<_Float16, 64>(A, way, s);
}
