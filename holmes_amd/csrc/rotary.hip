// Rotary positions: pairs of a head's dims turned by an angle that grows with the token's position.
//
//   y0 = a (x0 cos t - x1 sin t),  y1 = a (x1 cos t + x0 sin t),  t = position * frequency of the pair
//
// The pairs are (i, i + rotated / 2), or, interleaved, (2 i, 2 i + 1); dims behind `rotated` are copied.
//
// A frequency is held as turns per token in units of 2^-64, so position * frequency modulo 2^64 is the angle's part of a
// turn with nothing lost but the frequency's rounding to whole units (position * 2^-65 turns): no reduction of a large angle,
// and no cosine of one.  What is left, within an eighth of a turn of a multiple of a quarter, goes through double into float, and
// sine and cosine are their Taylor polynomials there (terms up to x^9 and x^10: off by less than 2^-26), in 32 bits, as are their
// products with the amount: half a step of float each, which only fp32 outputs can show.
//
// Bound by the bytes.  A workgroup takes all heads of a few tokens, so that each angle is made once, into LDS, for queries
// and keys together.  32768 tokens, 32 query heads and 8 key heads of 128 in bf16, 671 MB: 108 us, 6.2 TB/s (a large copy
// through the caches reaches 5.1); one token 2.7 us, of a call's 5.
#include "../../include/holmes_ckks.h"
#include "internal.hpp"
#include "kv4.hpp"

#include <algorithm>

namespace hck {
namespace {

constexpr int kThreads = 256;
constexpr int kAngles = 1024;  // angles that a workgroup's LDS has room for

struct RotaryArgs {
  const void* positions;
  const uint64_t* turns;
  const void* x[2];  // queries and keys: [token][head][head_dim]
  void* y[2];        // dense
  int64_t ts[2], hs[2];
  int heads[2];
  int64_t tokens;
  int wide, inverse, per;  // wide: positions of 8 bytes; per: tokens of a workgroup
  int pairs, dim, units, turned;  // units of a head, of which the first `turned` hold pairs
  uint32_t by_units, by_heads;    // 2^32 / d, rounded up
  float amount;
};

// n / d for n * d < 2^32, from m = ceil(2^32 / d).
__device__ __forceinline__ uint32_t over(uint32_t n, uint32_t m, uint32_t d) { return d == 1 ? n : __umulhi(n, m); }

__device__ __forceinline__ float2 turned_by(uint64_t t) {
  const uint32_t quarter = (uint32_t)((t + (1ull << 61)) >> 62);
  const int64_t rest = (int64_t)(t - ((uint64_t)quarter << 62));
  const float x = (float)((double)rest * 3.4061215800304093e-19);  // 2 pi 2^-64
  const float z = x * x;
  const float s = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
  const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
  const float a = (quarter & 1) ? s : c, b = (quarter & 1) ? c : s;  // cosine and sine but for their signs
  return float2{((quarter + 1) & 2) ? -a : a, (quarter & 2) ? -b : b};
}

// V neighbouring values; with V * sizeof(T) = 16 in one access, else one by one.
template <typename T, int V>
struct Some {
  T v[V];
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  template <bool PAST>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V * sizeof(T) == 16) {
      const u32x4* at = reinterpret_cast<const u32x4*>(p);
      const u32x4 w = PAST ? __builtin_nontemporal_load(at) : *at;
      __builtin_memcpy(v, &w, 16);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = p[i];
    }
  }
  template <bool PAST>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V * sizeof(T) == 16) {
      u32x4 w;
      __builtin_memcpy(&w, v, 16);
      if constexpr (PAST) __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
      else *reinterpret_cast<u32x4*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = v[i];
    }
  }
};

// PAST: more is written than the L2 caches hold; loads and stores go past them (32768 tokens: 108 us; the stores alone 110, through
// the caches 114).
template <typename T, int V, bool INTERLEAVED, bool PAST>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryArgs A) {
  __shared__ float2 s_turn[kAngles];
  const int64_t first = (int64_t)blockIdx.x * A.per;
  const int tokens = (int)min((int64_t)A.per, A.tokens - first);
  for (int w = threadIdx.x; w < tokens * A.pairs; w += kThreads) {
    const int i = w / A.pairs, pair = w % A.pairs;
    const int64_t at = first + i;
    const int64_t position = A.wide ? static_cast<const int64_t*>(A.positions)[at] : static_cast<const int32_t*>(A.positions)[at];
    uint64_t t = (uint64_t)position * A.turns[pair];
    if (A.inverse) t = 0 - t;
    const float2 cs = turned_by(t);
    s_turn[w] = float2{cs.x * A.amount, cs.y * A.amount};
  }
  __syncthreads();
  const int heads = A.heads[0] + A.heads[1];
  for (uint32_t w = threadIdx.x; w < (uint32_t)(tokens * heads * A.units); w += kThreads) {
    const uint32_t row = over(w, A.by_units, A.units), u = w - row * A.units;
    const uint32_t i = over(row, A.by_heads, heads);
    int h = (int)(row - i * heads);
    const int side = h >= A.heads[0];
    h -= side ? A.heads[0] : 0;
    const int64_t token = first + i;
    const T* x = (const T*)A.x[side] + token * A.ts[side] + h * A.hs[side];
    T* y = (T*)A.y[side] + (token * A.heads[side] + h) * A.dim;
    Some<T, V> a, b;
    if ((int)u >= A.turned) {  // behind the pairs
      const int d = 2 * A.pairs + ((int)u - A.turned) * V;
      a.template load<PAST>(x + d);
      a.template store<PAST>(y + d);
      continue;
    }
    const float2* turn = s_turn + i * A.pairs;
    if constexpr (INTERLEAVED) {
      const int d = (int)u * V;
      a.template load<PAST>(x + d);
#pragma unroll
      for (int k = 0; k < V; k += 2) {
        const float2 cs = turn[(d + k) / 2];
        const float p = (float)a.v[k], q = (float)a.v[k + 1];
        a.v[k] = (T)(p * cs.x - q * cs.y);
        a.v[k + 1] = (T)(q * cs.x + p * cs.y);
      }
      a.template store<PAST>(y + d);
    } else {
      const int d = (int)u * V;
      a.template load<PAST>(x + d);
      b.template load<PAST>(x + A.pairs + d);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 cs = turn[d + k];
        const float p = (float)a.v[k], q = (float)b.v[k];
        a.v[k] = (T)(p * cs.x - q * cs.y);
        b.v[k] = (T)(q * cs.x + p * cs.y);
      }
      a.template store<PAST>(y + d);
      b.template store<PAST>(y + A.pairs + d);
    }
  }
}

uint32_t inverse_of(int d) { return (uint32_t)(((1ull << 32) + d - 1) / d); }

template <typename T>
int launch(RotaryArgs A, int rotated, bool interleaved, hipStream_t s) {
  constexpr int kWide = 16 / sizeof(T);
  // 16 bytes at a time where every access is so aligned, else single values
  bool wide = A.dim % kWide == 0 && (interleaved ? rotated : A.pairs) % kWide == 0;
  for (int i = 0; i < 2; ++i) {
    if (!A.heads[i]) continue;
    wide = wide && ((uintptr_t)A.x[i] | (uintptr_t)A.y[i]) % 16 == 0;
    wide = wide && (A.tokens == 1 || A.ts[i] % kWide == 0) && (A.heads[i] == 1 || A.hs[i] % kWide == 0);
  }
  const int v = wide ? kWide : interleaved ? 2 : 1;
  A.turned = (interleaved ? rotated : A.pairs) / v;
  A.units = A.turned + (A.dim - rotated) / v;
  const int heads = A.heads[0] + A.heads[1];
  A.by_units = inverse_of(A.units), A.by_heads = inverse_of(heads);
  // Tokens of a workgroup: about 8 KB of values, what the angles have room for, and no more than leave 1024 workgroups.  (Tokens of
  // 128 bytes to 40 KB, 2500 to 32768 of them, both kinds of pairs, all of a head and half, any alignment, 1 to 32 tokens
  // a workgroup: this is off the best by 2 % on average and 13 at the most; by 16 KB 3 and 14, by 6 KB 3 and 19.  32768
  // tokens of 1280 bytes: one 27.4 us, two 22.1, six 17.4, twelve 17.9; of 10 KB: one 106, two 114.)
  const int64_t size = (int64_t)heads * A.dim * sizeof(T), many = ((8 << 10) + size / 2) / size;
  A.per = (int)std::max<int64_t>(1, std::min({many, (int64_t)kAngles / A.pairs, A.tokens / 1024}));
  const int64_t groups = (A.tokens + A.per - 1) / A.per;
  if (!fits_grid(groups, kThreads)) return HCK_ERR_ARG;
  const dim3 grid((unsigned)groups);
  const bool past = wide && A.tokens * heads * A.dim * (int64_t)sizeof(T) > kL2s;
  if (interleaved) {
    if (past) k_rotary<T, kWide, true, true><<<grid, kThreads, 0, s>>>(A);
    else if (wide) k_rotary<T, kWide, true, false><<<grid, kThreads, 0, s>>>(A);
    else k_rotary<T, 2, true, false><<<grid, kThreads, 0, s>>>(A);
  } else {
    if (past) k_rotary<T, kWide, false, true><<<grid, kThreads, 0, s>>>(A);
    else if (wide) k_rotary<T, kWide, false, false><<<grid, kThreads, 0, s>>>(A);
    else k_rotary<T, 1, false, false><<<grid, kThreads, 0, s>>>(A);
  }
  HCK_CHECK_LAUNCH();
  return HCK_OK;
}

}  // namespace
}  // namespace hck

extern "C" int hck_rotary(const void* positions, int position_bytes, int64_t tokens, const uint64_t* turns, int rotated,
                          int interleaved, int inverse, float amount, int type, int head_dim, const void* queries,
                          int64_t q_token_stride, int64_t q_head_stride, int heads, void* out_queries, const void* keys,
                          int64_t k_token_stride, int64_t k_head_stride, int kv_heads, void* out_keys, void* stream) {
  if (type < HCK_BF16 || type > HCK_F32 || head_dim < 2 || head_dim > HCK_ROTARY_MAX || head_dim % 2) return HCK_ERR_UNSUPPORTED;
  if (rotated < 2 || rotated > head_dim || rotated % 2 || tokens < 0 || heads < 0 || kv_heads < 0) return HCK_ERR_ARG;
  // (so many that a workgroup's divisions stay within 2^32)
  if ((int64_t)heads + kv_heads > 65535 || ((int64_t)heads + kv_heads) * head_dim > HCK_ROTARY_TOKEN) return HCK_ERR_ARG;
  if (tokens == 0 || heads + kv_heads == 0) return HCK_OK;
  if ((position_bytes != 4 && position_bytes != 8) || !positions || !turns) return HCK_ERR_ARG;
  if ((heads && (!queries || !out_queries)) || (kv_heads && (!keys || !out_keys))) return HCK_ERR_ARG;
  hck::RotaryArgs A = {};
  A.positions = positions, A.turns = turns, A.tokens = tokens;
  A.x[0] = queries, A.y[0] = out_queries, A.ts[0] = q_token_stride, A.hs[0] = q_head_stride, A.heads[0] = heads;
  A.x[1] = keys, A.y[1] = out_keys, A.ts[1] = k_token_stride, A.hs[1] = k_head_stride, A.heads[1] = kv_heads;
  A.wide = position_bytes == 8, A.inverse = inverse != 0, A.pairs = rotated / 2, A.dim = head_dim, A.amount = amount;
  hipStream_t s = (hipStream_t)stream;
  if (type == HCK_BF16) return hck::launch<__bf16>(A, rotated, interleaved != 0, s);
  if (type == HCK_F16) return hck::launch<_Float16>(A, rotated, interleaved != 0, s);
  return hck::launch<float>(A, rotated, interleaved != 0, s);
}
