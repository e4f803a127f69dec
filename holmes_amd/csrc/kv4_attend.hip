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
// bits.  The probabilities go in as two bf16 parts as well, the nearest and the rest's, which leaves 2^-17 of each, far below the
// rounding of the output; the sum l takes the unrounded ones.
//
// What bounds it (8 key heads of 128, 4 query heads each): over 48 sequences of 12000 to 24576 tokens the bytes,
// 917 MB in 163 us or 5.6 TB/s (the same loads without arithmetic: 5.9); over 131072 tokens 34 us with the join for
// 142 MB, of which 5 go by before the first product; over 257 tokens the chain of loads (length, page number, codes),
// 5 to 7 us.
#include "kv4_attend.hpp"

namespace hck {
namespace {

// A load that passes the caches by where nothing is read twice.
template <bool ONCE, typename V>
__device__ __forceinline__ V fetch(const uint8_t* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  else return *reinterpret_cast<const V*>(p);
}

// What a lane holds of 64 tokens: lane (m, g) = (lane % 16, lane / 16) has D / 4 dims from D / 4 * g of
// token m of every 16-token tile, and D / 16 dims from D / 16 * m of the 8 tokens (g, j) of each 32.
template <int D>
struct Unit {
  uint32_t k[4][D / 32], ks, v[2][D / 16], vs[2][2];
  template <bool ONCE>
  __device__ __forceinline__ void load_keys(const uint8_t* page, int half, int m, int g) {
    using L = Kv4<D>;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* p = page + (4 * half + i) * (8 * D) + (g * 16 + m) * (D / 8);
      if constexpr (D == 128) *reinterpret_cast<u32x4*>(k[i]) = fetch<ONCE, u32x4>(p);
      else *reinterpret_cast<u32x2*>(k[i]) = fetch<ONCE, u32x2>(p);
    }
    ks = *reinterpret_cast<const uint32_t*>(page + L::key_scale(64 * half + m, g * (D / 4) / kRun));
  }
  template <bool ONCE>
  __device__ __forceinline__ void load_values(const uint8_t* page, int half, int m, int g) {
    using L = Kv4<D>;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* p = page + L::kVCodes + (2 * half + i) * (16 * D) + (g * 16 + m) * 16;
#pragma unroll
      for (int w = 0; w < D / 64; ++w)
        reinterpret_cast<u32x4*>(v[i])[w] = fetch<ONCE, u32x4>(p + 1024 * w);
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

// A lane's neighbours 4 and 8 on, of the 16 that share g.
template <int N>
__device__ __forceinline__ float turn(float x) {
  return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x120 + N, 0xf, 0xf, true));
}
template <int R, typename F>
__device__ __forceinline__ float over_row(float x, F f) {
  if constexpr (R <= 8) x = f(x, turn<8>(x));
  if constexpr (R <= 4) x = f(x, turn<4>(x));
  return over_g(x, f);
}

// R rows of one key head, a part of their tokens; the waves take units in turn.
//
// With R < 16 the product's 16 columns hold the rows 16 / R times.  Each copy keeps the scores of its own
// share of the 64 tokens, so that no exponential is taken for an empty column, and goes into the second
// product with zeros for the other copies' tokens; the copies' sums are added at the end.
//
// ONCE: with loads past the caches (Way::once).
//
// Keys of the next unit are loaded as soon as the first product is done with this one's, its values after the
// second, so that loads are in flight throughout without registers of their own.
template <typename T, int D, bool RANGE, int R, bool ONCE>
__global__ __launch_bounds__(64 * kWaves, waves_of_few(D, __is_same(T, _Float16))) void k_attend(AttendArgs A) {
  using L = Kv4<D>;
  constexpr int kTiles = R / 4;  // 16-token tiles of a lane's scores
  constexpr int kSteps = D / 32, kDpl = L::kDpl;
  constexpr bool kHalf = __is_same(T, _Float16);
  __shared__ float s_m[kWaves][kFew], s_l[kWaves][kFew], s_low[kWaves][kFew];
  __shared__ uint32_t s_large[kWaves];
  extern __shared__ float s_o[];  // [wave][A.rows][D + 4]

  Item it;
  if (!locate(A, blockIdx.x, it)) return;
  it.uniform();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  const int copy = m / R, tile = it.tile, h = it.h, b = it.b;
  // the first page's number, asked for at once (a column of the table, whatever the length)
  const int* table = A.table + b * A.table_stride;
  int u = it.u0 + wave;
  const int begin = (u >> 1) < A.cols ? table[u >> 1] : 0;
  const Rows S = it.rows;
  const long long q0 = S.q0;
  const int rows = S.rows;
  if (tile * kFew >= rows) return;
  const int row = tile * kFew + m % R;
  const bool live = row < rows;
  const int qi = live ? row / A.group : 0, qo = live ? row % A.group : 0;
  const int seen = live ? S.seen(A, row) : 0;
  const int all = S.seen(A, tile * kFew), most = S.seen(A, min(tile * kFew + R, rows) - 1);
  const int u1 = min((most + kUnit - 1) / kUnit, it.u1);

  // the lane's part of its row's query: dims D / 4 g + 8 s .. + 7 of step s
  bf16x8 qh[kSteps], ql[kSteps];
  const T* qp = (const T*)A.q + (q0 + qi) * A.q_ts + (long long)(h * A.group + qo) * A.q_hs + g * (D / 4);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    u32x4 raw = {0, 0, 0, 0};
    if (live) raw = reinterpret_cast<const Loose16*>(qp + 8 * s)->v;
    query_parts<T>(raw, qh[s], ql[s]);
  }

  f32x4 acc[kDpl];
#pragma unroll
  for (int i = 0; i < kDpl; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f, low = INFINITY;
  const float scale2 = A.scale * kLog2e;
  float ref = -kLift, factor = scale2;
  uint32_t large = 0;  // runs whose sums are held times 2^-56

  // a page number that is not in the pool is read as page 0, and its tokens are left out
  auto page_of = [&](int pg) { return A.pool + ((long long)(pg < 0 || pg >= A.pages ? 0 : pg) * A.heads + h) * L::kBytes; };
  int pg = __builtin_amdgcn_readfirstlane(begin), next = 0;
  Unit<D> x;
  auto load_keys = [&](const uint8_t* page, int half) { x.template load_keys<ONCE>(page, half, m, g); };
  auto load_values = [&](const uint8_t* page, int half) { x.template load_values<ONCE>(page, half, m, g); };
  if (u < u1) {
    load_keys(page_of(pg), u & 1);
    load_values(page_of(pg), u & 1);
    if (u + kWaves < u1) next = table[(u + kWaves) >> 1];
  }
  for (; u < u1; u += kWaves) {
    const bool there = pg >= 0 && pg < A.pages, more = u + kWaves < u1;
    pg = __builtin_amdgcn_readfirstlane(next);
    if (u + 2 * kWaves < u1) next = table[(u + 2 * kWaves) >> 1];
    const uint8_t* page = page_of(pg);
    if (!there) {
      if (more) load_keys(page, u & 1), load_values(page, u & 1);
      continue;
    }

    float t[kTiles][4];
    f32x4 c[4];
    float sc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t byte = (x.ks >> (8 * i)) & 0xffu;
      sc[i] = byte == kNanByte ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
      c[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 kk = x.key(i, s, sc[i]);
        c[i] = mfma(kk, qh[s], c[i]);
        if constexpr (kHalf) c[i] = mfma(kk, ql[s], c[i]);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) t[i % kTiles][k] = i < kTiles || copy == i / kTiles ? c[i][k] : t[i % kTiles][k];
    if (more) load_keys(page, u & 1);
    const int base = u * kUnit + 4 * g, own = base + 16 * kTiles * copy;
    if (__builtin_amdgcn_readfirstlane(u * kUnit) + kUnit > all) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool see = own + 16 * i + k < seen;
          if constexpr (RANGE) low = see ? fminf(low, t[i][k]) : low;
          t[i][k] = see ? t[i][k] : -INFINITY;
        }
    } else if constexpr (RANGE) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) low = smaller(low, t[i][k]);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) mx = larger(mx, t[i][k]);
    const float raw = over_row<R>(mx, fmax2);
    mx = fmaxf(top, raw * scale2);
    const float f = rebase(top, mx);
    top = mx;
    if (__any(f != 1.f)) {
      if (f != 1.f) refer(mx, raw, scale2, ref, factor);
      sum *= f;
#pragma unroll
      for (int i = 0; i < kDpl; ++i) acc[i] *= f;
    }
    u32x2 hi[kTiles], lo[kTiles];  // the probabilities in two bf16 parts
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        t[i][k] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[i][k], factor, -ref));
        sum += t[i][k];
      }
      hi[i] = u32x2{pack(t[i][0], t[i][1]), pack(t[i][2], t[i][3])};
      lo[i] = u32x2{rests_of(t[i][0], t[i][1], hi[i][0]), rests_of(t[i][2], t[i][3], hi[i][1])};
    }

    if (__builtin_expect(large || __any(has_large(x.vs[0][0]) || has_large(x.vs[0][1]) || has_large(x.vs[1][0]) || has_large(x.vs[1][1])), false)) {
      bool beyond = false;
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        // A run of NaN must reach the rows that see its token, and no other: 0 * NaN is NaN.  It is taken as zeros
        // in the product, and counted for the rows that see it by a product of truth values.
        uint32_t vs[2] = {i ? x.vs[1][0] : x.vs[0][0], i ? x.vs[1][1] : x.vs[0][1]};
        bf16x8 bad, see;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t byte = (vs[k >> 2] >> (8 * (k & 3))) & 0xffu;
          const int token = base + 32 * i + 16 * (k >> 2) + (k & 3);
          const bool is = byte == kNanByte;
          bad[k] = (__bf16)(is ? 1.f : 0.f);
          see[k] = (__bf16)(token < seen ? 1.f : 0.f);
          if (is) vs[k >> 2] &= ~(0xffu << (8 * (k & 3)));
          else beyond = beyond || (byte >= kLargeByte && token < most);
        }
        x.vs[0][0] = i ? x.vs[0][0] : vs[0], x.vs[0][1] = i ? x.vs[0][1] : vs[1];
        x.vs[1][0] = i ? vs[0] : x.vs[1][0], x.vs[1][1] = i ? vs[1] : x.vs[1][1];
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const f32x4 n = mfma(bad, see, zero);
#pragma unroll
        for (int d = 0; d < kDpl; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n[k] > 0.f) acc[d][k] = __uint_as_float(0x7fc00000u);
      }
      const unsigned long long all4 = __ballot(beyond);
      uint32_t lanes = (uint32_t)all4 | (uint32_t)(all4 >> 32), runs = 0;
      lanes |= lanes >> 16;  // of every g
#pragma unroll
      for (int r = 0; r < L::kRuns; ++r)  // a run's lanes: kRun / kDpl neighbours
        runs |= (lanes >> (r * (kRun / kDpl))) & ((1u << (kRun / kDpl)) - 1) ? 1u << r : 0u;
      int here = lane;  // (worked out here and not kept from before the loop)
      asm volatile("" : "+v"(here));
      if (const uint32_t fresh = runs & ~large) {
        large |= fresh;
        const float by = (fresh >> ((here >> 4) * (D / 4) / kRun)) & 1 ? kDownBy : 1.f;
#pragma unroll
        for (int d = 0; d < kDpl; ++d) acc[d] *= by;
      }
      if ((large >> ((here & 15) * kDpl / kRun)) & 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) x.vs[i][0] = down(x.vs[i][0]), x.vs[i][1] = down(x.vs[i][1]);
      }
    }

#pragma unroll
    for (int i = 0; i < 2; ++i) {
      auto part = [&](const u32x2* p) {
        u32x2 w[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const bool mine = copy == (2 * i + n) / kTiles;
          w[n] = kTiles == 4 ? p[(2 * i + n) % kTiles] : u32x2{mine ? p[n % kTiles][0] : 0u, mine ? p[n % kTiles][1] : 0u};
        }
        return operand(w[0][0], w[0][1], w[1][0], w[1][1]);
      };
      const bf16x8 ph = part(hi), pl = part(lo);
      float sc[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) sc[k] = scale_of(x.vs[i][k >> 2], k & 3);
      bf16x8 e, o;
      auto step = [&](auto B) {
        constexpr int kB = decltype(B)::value;
        x.template value<kB>(i, sc, e, o);
        acc[2 * kB] = mfma(e, ph, acc[2 * kB]);
        acc[2 * kB + 1] = mfma(o, ph, acc[2 * kB + 1]);
        acc[2 * kB] = mfma(e, pl, acc[2 * kB]);
        acc[2 * kB + 1] = mfma(o, pl, acc[2 * kB + 1]);
      };
      step(std::integral_constant<int, 0>());
      step(std::integral_constant<int, 1>());
      if constexpr (kDpl == 8) {
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
      }
    }
    if (more) load_values(page, u & 1);
  }

  publish(A, it);
  // join the waves: lane (m, g) holds dims D / 4 g + kDpl i + d of row m in acc[d][i]
  sum = over_row<R>(sum, [](float a, float c) { return a + c; });
  if constexpr (RANGE) low = over_row<R>(low, fmin2) * scale2;
#pragma unroll
  for (int d = 0; d < kDpl; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (R <= 8) acc[d][i] += turn<8>(acc[d][i]);
      if constexpr (R <= 4) acc[d][i] += turn<4>(acc[d][i]);
    }
  if (lane < R) s_m[wave][m] = top, s_l[wave][m] = sum, s_low[wave][m] = low;
  if (lane == 0) s_large[wave] = large;
  if (m < R && m < A.rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < kDpl; ++d) s_o[(wave * A.rows + m) * (D + 4) + g * (D / 4) + kDpl * i + d] = acc[d][i];
  }
  __syncthreads();
  constexpr int kCols = D / 16;  // dims of a thread: 16 threads to a row
  const int r = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * kCols;
  if (r >= A.rows || tile * kFew + r >= rows) return;
  float mm = -INFINITY, ll = 0.f, lo = INFINITY, o[kCols];
  uint32_t any = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, s_m[w][r]), any |= s_large[w];
#pragma unroll
  for (int c = 0; c < kCols; ++c) o[c] = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    float f = rebase(s_m[w][r], mm);
    ll += f * s_l[w][r];
    lo = fminf(lo, s_low[w][r]);
    f *= to_common(s_large[w], any, c0 / kRun);
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c] += f * s_o[(w * A.rows + r) * (D + 4) + c0 + c];
  }
  if (it.slots > 1) {
    const long long at = (long long)it.slot * A.rows + r;
    if (c0 == 0) *reinterpret_cast<f32x4*>(A.stat + at * 4) = f32x4{mm, ll, lo, __uint_as_float(any)};
#pragma unroll
    for (int c = 0; c < kCols; c += 4)
      *reinterpret_cast<f32x4*>(A.sums + at * D + c0 + c) = f32x4{o[c], o[c + 1], o[c + 2], o[c + 3]};
    return;
  }
  const int qr = (tile * kFew + r) / A.group, qc = (tile * kFew + r) % A.group;
  store_row<T, kCols, RANGE>(A, (q0 + qr) * (long long)(A.heads * A.group) + h * A.group + qc, D, c0, mm, ll, lo, o,
                             back(any, c0 / kRun));
}

// Joins the slots of a row of few, where it has more than one: one workgroup a row, its W waves taking 8 slots
// at a time.  What bounds it is the trips to memory one after another: where the slots are, and then everything
// in them at once.  (Slots of a tile and head lie `heads` apart.)
template <typename T, int D, bool RANGE, int W>
__global__ __launch_bounds__(64 * W) void k_join_few(AttendArgs A) {
  constexpr int kCols = D / 64, kBatch = 8;
  __shared__ float s_m[W], s_l[W], s_low[W], s_o[W][D];
  __shared__ uint32_t s_large[W];
  const int pair = blockIdx.x / A.heads, h = blockIdx.x % A.heads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = A.plan[2 * blockIdx.x], slots = A.plan[2 * blockIdx.x + 1];  // nothing there, if no rows
  const Rows R(A, pair / A.tiles);
  const int row = (pair % A.tiles) * kFew + blockIdx.y;
  if (row >= R.rows || slots < 2) return;
  const long long step = (long long)A.heads * A.rows, at = (long long)slot * A.rows + blockIdx.y;
  const float* stat = A.stat + at * 4;
  const float* sums = A.sums + at * D + lane * kCols;
  float top = -INFINITY, ll = 0.f, lo = INFINITY, o[kCols] = {};
  uint32_t large = 0;
  const int run = lane * kCols / kRun;
  for (int s0 = wave; s0 < slots; s0 += kBatch * W) {
    f32x4 st[kBatch];
    float x[kBatch][kCols];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const long long s = min(s0 + i * W, slots - 1);
      st[i] = *reinterpret_cast<const f32x4*>(stat + s * step * 4);
#pragma unroll
      for (int c = 0; c < kCols; ++c) x[i][c] = sums[s * step * D + c];
    }
    float m = top;
    uint32_t any = large;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) m = fmaxf(m, st[i][0]), any |= __float_as_uint(st[i][3]);
    float f = rebase(top, m);
    top = m;
    ll *= f;
    f *= to_common(large, any, run);
    large = any;
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c] *= f;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (s0 + i * W >= slots) break;
      float e = rebase(st[i][0], m);
      ll += e * st[i][1];
      lo = fminf(lo, st[i][2]);
      e *= to_common(__float_as_uint(st[i][3]), large, run);
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[c] += e * x[i][c];
    }
  }
  if (lane == 0) s_m[wave] = top, s_l[wave] = ll, s_low[wave] = lo, s_large[wave] = large;
#pragma unroll
  for (int c = 0; c < kCols; ++c) s_o[wave][lane * kCols + c] = o[c];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < W; ++w) top = fmaxf(top, s_m[w]), large |= s_large[w];
  ll = 0.f;
#pragma unroll
  for (int c = 0; c < kCols; ++c) o[c] = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    float f = rebase(s_m[w], top);
    ll += f * s_l[w];
    lo = fminf(lo, s_low[w]);
    f *= to_common(s_large[w], large, run);
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c] += f * s_o[w][lane * kCols + c];
  }
  store_row<T, kCols, RANGE>(A, (R.q0 + row / A.group) * (long long)(A.heads * A.group) + h * A.group + row % A.group, D,
                             lane * kCols, top, ll, lo, o, back(large, run));
}

// The same of many rows, which have few slots each: D / 4 threads a row, a workgroup a 4th to a 16th of a tile
// (fewer where there are many tiles, of which most may have nothing to join).
template <typename T, int D, bool RANGE>
__global__ __launch_bounds__(64 * kWaves) void k_join_many(AttendArgs A) {
  constexpr int kThreads = D / 4, kRows = 64 * kWaves / kThreads;
  const int pair = blockIdx.x / A.heads, h = blockIdx.x % A.heads;
  const int slot = A.plan[2 * blockIdx.x], slots = A.plan[2 * blockIdx.x + 1];  // nothing there, if no rows
  const Rows R(A, pair / A.tiles);
  const int first = (pair % A.tiles) * A.size, c0 = threadIdx.x % kThreads * 4;
  if (first >= R.rows || slots < 2) return;
  const int part = A.size / gridDim.y, end = min(min(A.rows, R.rows - first), (int)(blockIdx.y + 1) * part);
  const long long step = (long long)A.heads * A.rows;
  for (int r = blockIdx.y * part + threadIdx.x / kThreads; r < end; r += kRows) {
    const long long at = (long long)slot * A.rows + r;
    const float* stat = A.stat + at * 4;
    const float* sums = A.sums + at * D + c0;
    float top = -INFINITY, ll = 0.f, lo = INFINITY;
    uint32_t large = 0;
#pragma unroll 4
    for (int s = 0; s < slots; ++s) top = fmaxf(top, stat[s * step * 4]), large |= __float_as_uint(stat[s * step * 4 + 3]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < slots; ++s) {
      const f32x4 st = *reinterpret_cast<const f32x4*>(stat + s * step * 4);
      const f32x4 x = *reinterpret_cast<const f32x4*>(sums + s * step * D);
      const float f = rebase(st[0], top);
      ll += f * st[1];
      lo = fminf(lo, st[2]);
      o += f * to_common(__float_as_uint(st[3]), large, c0 / kRun) * x;
    }
    const float v[4] = {o[0], o[1], o[2], o[3]};
    const int qr = (first + r) / A.group, qc = (first + r) % A.group;
    store_row<T, 4, RANGE>(A, (R.q0 + qr) * (long long)(A.heads * A.group) + h * A.group + qc, D, c0, top, ll, lo, v,
                            back(large, c0 / kRun));
  }
}

template <typename T, int D, bool RANGE>
int launch(const AttendArgs& A, const Way& W, hipStream_t s) {
  const dim3 grid((unsigned)W.items);
  const size_t lds = kWaves * W.rows * (D + 4) * sizeof(float);
  if (!W.few) {
    if (const int err = launch_prompt(A, W, D, __is_same(T, _Float16) ? HCK_F16 : HCK_BF16, s)) return err;
  } else {
    auto run = [&](auto rows, auto once) {
      k_attend<T, D, RANGE, decltype(rows)::value, decltype(once)::value><<<grid, 64 * kWaves, lds, s>>>(A);
    };
    typedef std::integral_constant<int, 4> Four;
    typedef std::integral_constant<int, 8> Eight;
    typedef std::integral_constant<int, 16> Sixteen;
    if (W.rows <= 4) A.once ? run(Four(), std::true_type()) : run(Four(), std::false_type());
    else if (W.rows <= 8) A.once ? run(Eight(), std::true_type()) : run(Eight(), std::false_type());
    else A.once ? run(Sixteen(), std::true_type()) : run(Sixteen(), std::false_type());
  }
  HCK_CHECK_LAUNCH();
  if (W.join) {
    const unsigned pairs = (unsigned)(W.pairs * A.heads);
    if (!W.few) k_join_many<T, D, RANGE><<<dim3(pairs, pairs <= 128 ? 16 : pairs <= 256 ? 8 : 4), 64 * kWaves, 0, s>>>(A);
    else if (W.most_slots > 32) k_join_few<T, D, RANGE, 16><<<dim3(pairs, W.rows), 64 * 16, 0, s>>>(A);
    else k_join_few<T, D, RANGE, 4><<<dim3(pairs, W.rows), 64 * 4, 0, s>>>(A);
    HCK_CHECK_LAUNCH();
  }
  return HCK_OK;
}

// (Columns below 2^24: a token's number, and the first one behind its unit, are within 31 bits.)
bool shape_ok(int64_t tokens, int seqs, int kv_heads, int group, int most, int cols) {
  return tokens >= 0 && seqs >= 0 && seqs <= 65535 && kv_heads >= 1 && kv_heads <= 65535 && group >= 1 &&
         group <= 1024 && most >= 0 && cols >= 0 && cols < (1 << 24) && (int64_t)most * group <= (1 << 30) &&
         tokens * kv_heads * group <= ((int64_t)1 << 32);
}

}  // namespace
}  // namespace hck

extern "C" size_t hck_kv4_attend_workspace_bytes(int64_t tokens, int seqs, int kv_heads, int group, int head_dim,
                                                 int most, int table_columns) {
  if (!hck::shape_ok(tokens, seqs, kv_heads, group, most, table_columns)) return 0;
  // the type is not known here: the most that either needs
  size_t most_bytes = 0;
  for (bool half : {false, true})
    most_bytes = std::max(most_bytes, hck::Way(seqs, kv_heads, group, head_dim, half, most, table_columns).bytes(kv_heads, head_dim));
  return most_bytes;
}

extern "C" int hck_kv4_attend(const void* pool, int64_t pages, int kv_heads, int head_dim, int type,
                              const void* queries, int64_t tokens, int group, int64_t q_token_stride,
                              int64_t q_head_stride, const int32_t* table, int64_t table_stride, int table_columns,
                              const int32_t* lengths, const int32_t* starts, int seqs, int most, int causal,
                              float scale, void* out, float* lse, float* low, float* high, void* workspace,
                              size_t workspace_bytes, void* stream) {
  if (hck::kv4_bytes(head_dim) == 0 || (type != HCK_BF16 && type != HCK_F16)) return HCK_ERR_UNSUPPORTED;
  if (!pool || pages < 1 || !hck::shape_ok(tokens, seqs, kv_heads, group, most, table_columns)) return HCK_ERR_ARG;
  // (times log2 e it is at most 2^127, and so is the power of 2 that stands for it beyond kFar)
  if (!(scale > 0.f) || scale > 0x1p126f || (low == nullptr) != (high == nullptr)) return HCK_ERR_ARG;
  if (tokens == 0 || seqs == 0 || most == 0) return HCK_OK;
  if (!queries || !lengths || (!table && table_columns > 0) || !out || !lse) return HCK_ERR_ARG;
  if (!starts && tokens < seqs) return HCK_ERR_ARG;
  if (((uintptr_t)pool | (uintptr_t)out | (uintptr_t)workspace) % 16) return HCK_ERR_ARG;
  const hck::Way W(seqs, kv_heads, group, head_dim, type == HCK_F16, most, table_columns);
  const size_t need = W.bytes(kv_heads, head_dim);
  if (W.items > 0x7fffffff || W.pairs > 0x7fffffff) return HCK_ERR_ARG;
  if (need > workspace_bytes || (need && !workspace)) return HCK_ERR_WORKSPACE;
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
  if (W.join) {
    A.stat = (float*)workspace;
    A.sums = A.stat + W.items * W.rows * 4;
    A.plan = (int*)(A.sums + W.items * W.rows * head_dim);
  }
  A.q_ts = q_token_stride;
  A.q_hs = q_head_stride;
  A.tokens = tokens;
  A.pages = pages;
  A.table_stride = table_stride;
  A.cols = table_columns;
  A.heads = kv_heads;
  A.group = group;
  A.causal = causal;
  A.seqs = seqs;
  A.tiles = (int)W.tiles;
  A.size = W.size;
  A.rows = W.rows;
  A.slots = (int)W.slots;
  A.least = W.least;
  A.join = W.join;
  A.once = W.once(seqs, table_columns, pages, kv_heads, head_dim);
  A.scale = scale;
  hipStream_t s = (hipStream_t)stream;
  const bool range = low != nullptr;
  if (head_dim == 128) {
    if (type == HCK_BF16) return range ? hck::launch<__bf16, 128, true>(A, W, s) : hck::launch<__bf16, 128, false>(A, W, s);
    return range ? hck::launch<_Float16, 128, true>(A, W, s) : hck::launch<_Float16, 128, false>(A, W, s);
  }
  if (type == HCK_BF16) return range ? hck::launch<__bf16, 64, true>(A, W, s) : hck::launch<__bf16, 64, false>(A, W, s);
  return range ? hck::launch<_Float16, 64, true>(A, W, s) : hck::launch<_Float16, 64, false>(A, W, s);
}
