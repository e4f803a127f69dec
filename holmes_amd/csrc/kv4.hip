// Writing keys and values into 4-bit pages, and reading them back.
#include "kv4.hpp"

#include "../../include/holmes_ckks.h"
#include "internal.hpp"

namespace hck {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct alignas(sizeof(T)) Eight {
  T v[8];
};

// Eight neighbouring values of one token, key or value, per thread: four threads share a run of 32.
// Both directions only move bytes, so the layout of the work follows the larger side: neighbouring
// threads take neighbouring eights of the unquantised tensor (16 bytes a thread in 16-bit types), and
// a workgroup holds 32 tokens of one head, whose value codes fill whole lines of the page.  32768 tokens of 8 heads
// of 128 in bf16, 152 MB each way: 44 us written and 31 us read while each pushes the other's data out of the last
// cache, 31 and 27 us where it does not.
constexpr int kTokensPerGroup = 32;

template <typename T, int D>
__global__ __launch_bounds__(256) void k_append(uint8_t* __restrict__ pool, long long pages, int heads,
                                                const T* __restrict__ keys, const T* __restrict__ values,
                                                long long k_ts, long long k_hs, long long v_ts, long long v_hs,
                                                const long long* __restrict__ slots, long long tokens) {
  using L = Kv4<D>;
  constexpr int kPer = D / 8;  // threads of a token's keys (or values)
  const int h = blockIdx.y;
  const long long first = (long long)blockIdx.x * kTokensPerGroup;
  for (int w = threadIdx.x; w < kTokensPerGroup * 2 * kPer; w += 256) {
    const int e = w % kPer, side = (w / kPer) & 1, i = w / (2 * kPer);
    const long long tok = first + i;
    const bool live = tok < tokens;
    const long long slot = live ? slots[tok] : -1;
    const bool ok = slot >= 0 && slot < pages * kPageTokens;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (ok) {
      const T* p = side ? values + tok * v_ts + h * v_hs : keys + tok * k_ts + h * k_hs;
      const Eight<T> in = *reinterpret_cast<const Eight<T>*>(p + 8 * e);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = (float)in.v[k];
    }
    // the run's largest magnitude by its bits, which order like the magnitudes and put an infinity
    // or a NaN above every number
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    const bool nan = top >= 0x7f800000u;
    // half of the last kept mantissa bit carries 1.75 * 2^e up to 2^(e + 1): the largest value then
    // becomes 4 units, never 7 or more, so no value is off by more than half a step
    const int b = min(max((int)((top + (1u << 21)) >> 23) - 2, 2), 252);
    const float unit = __uint_as_float((uint32_t)b << 23);
    uint32_t codes = 0;
    if (!nan) {
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], unit, 0);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], unit, 1);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], unit, 2);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], unit, 3);
    }
    if (!ok) continue;
    const int t = (int)(slot & (kPageTokens - 1));
    uint8_t* page = pool + ((slot >> 7) * heads + h) * (long long)L::kBytes;
    if (side == 0) {
      *reinterpret_cast<uint32_t*>(page + L::key_code(t, 8 * e)) = codes;
    } else if constexpr (L::kDpl == 8) {
      *reinterpret_cast<uint32_t*>(page + L::value_code(t, e)) = codes;
    } else {
      *reinterpret_cast<uint16_t*>(page + L::value_code(t, 2 * e)) = (uint16_t)codes;
      *reinterpret_cast<uint16_t*>(page + L::value_code(t, 2 * e + 1)) = (uint16_t)(codes >> 16);
    }
    if ((e & 3) == 0) page[side ? L::value_scale(t, e / 4) : L::key_scale(t, e / 4)] = (uint8_t)(nan ? kNanByte : b);
  }
}

template <typename T>
__device__ __forceinline__ T narrow(float x) {
  if constexpr (sizeof(T) == 4) {
    return x;
  } else if constexpr (__is_same(T, _Float16)) {
    return (T)(x != x ? x : fminf(fmaxf(x, -65504.f), 65504.f));  // the type's largest instead of an infinity
  } else {
    return (T)x;  // exact: two significant bits, and 6 * 2^125 is below bf16's largest
  }
}

// PAST: more is written than the L2 caches hold, and stored past them (32768 tokens, 8 heads of 128, written and
// read back: 80 us a round with stores that push the keys and values out of the last cache, 71 us so).
template <typename T, int D, bool PAST>
__global__ __launch_bounds__(256) void k_read(const uint8_t* __restrict__ pool, long long pages, int heads,
                                              const long long* __restrict__ slots, long long tokens,
                                              T* __restrict__ keys, T* __restrict__ values) {
  using L = Kv4<D>;
  constexpr int kPer = D / 8;
  const int h = blockIdx.y;
  const long long first = (long long)blockIdx.x * kTokensPerGroup;
  for (int w = threadIdx.x; w < kTokensPerGroup * 2 * kPer; w += 256) {
    const int e = w % kPer, side = (w / kPer) & 1, i = w / (2 * kPer);
    const long long tok = first + i;
    if (tok >= tokens) continue;
    const long long slot = slots[tok];
    Eight<T> out;
    if (slot >= 0 && slot < pages * kPageTokens) {
      const int t = (int)(slot & (kPageTokens - 1));
      const uint8_t* page = pool + ((slot >> 7) * heads + h) * (long long)L::kBytes;
      uint32_t codes;
      if (side == 0) {
        codes = *reinterpret_cast<const uint32_t*>(page + L::key_code(t, 8 * e));
      } else if constexpr (L::kDpl == 8) {
        codes = *reinterpret_cast<const uint32_t*>(page + L::value_code(t, e));
      } else {
        codes = *reinterpret_cast<const uint16_t*>(page + L::value_code(t, 2 * e)) |
                (uint32_t)*reinterpret_cast<const uint16_t*>(page + L::value_code(t, 2 * e + 1)) << 16;
      }
      const int b = page[side ? L::value_scale(t, e / 4) : L::key_scale(t, e / 4)];
      const float unit = __uint_as_float(b == kNanByte ? 0x7fc00000u : (uint32_t)b << 23);
      bf16x2 p[4];
      p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 0);
      p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 1);
      p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 2);
      p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 3);
#pragma unroll
      for (int k = 0; k < 8; ++k) out.v[k] = narrow<T>((float)p[k / 2][k & 1] * unit);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) out.v[k] = (T)0.f;
    }
    T* to = (side ? values : keys) + (tok * heads + h) * D + 8 * e;
    if constexpr (PAST) {
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      u32x4 w[sizeof(out) / 16];
      __builtin_memcpy(w, &out, sizeof(out));
#pragma unroll
      for (int i = 0; i < (int)sizeof(out) / 16; ++i) __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4*>(to) + i);
    } else {
      *reinterpret_cast<Eight<T>*>(to) = out;
    }
  }
}

template <typename F>
int by_type(int type, int head_dim, F&& f) {
  if (head_dim == 128) {
    if (type == HCK_BF16) return f((__bf16*)nullptr, std::integral_constant<int, 128>());
    if (type == HCK_F16) return f((_Float16*)nullptr, std::integral_constant<int, 128>());
    if (type == HCK_F32) return f((float*)nullptr, std::integral_constant<int, 128>());
  } else if (head_dim == 64) {
    if (type == HCK_BF16) return f((__bf16*)nullptr, std::integral_constant<int, 64>());
    if (type == HCK_F16) return f((_Float16*)nullptr, std::integral_constant<int, 64>());
    if (type == HCK_F32) return f((float*)nullptr, std::integral_constant<int, 64>());
  }
  return HCK_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace hck

extern "C" size_t hck_kv4_page_bytes(int head_dim) { return (size_t)hck::kv4_bytes(head_dim); }

extern "C" int hck_kv4_append(void* pool, int64_t pages, int kv_heads, int head_dim, int type, const void* keys,
                              int64_t key_token_stride, int64_t key_head_stride, const void* values,
                              int64_t value_token_stride, int64_t value_head_stride, const int64_t* slots,
                              int64_t tokens, void* stream) {
  if (hck::kv4_bytes(head_dim) == 0 || type < HCK_BF16 || type > HCK_F32) return HCK_ERR_UNSUPPORTED;
  if (!pool || pages < 1 || kv_heads < 1 || kv_heads > 65535 || tokens < 0) return HCK_ERR_ARG;
  if (tokens == 0) return HCK_OK;
  const int64_t groups = (tokens + hck::kTokensPerGroup - 1) / hck::kTokensPerGroup;
  if (!keys || !values || !slots || groups > 0x7fffffff) return HCK_ERR_ARG;
  return hck::by_type(type, head_dim, [&](auto* t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    hck::k_append<T, decltype(d)::value><<<dim3((unsigned)groups, kv_heads), 256, 0, (hipStream_t)stream>>>(
        (uint8_t*)pool, pages, kv_heads, (const T*)keys, (const T*)values, key_token_stride, key_head_stride,
        value_token_stride, value_head_stride, (const long long*)slots, tokens);
    HCK_CHECK_LAUNCH();
    return HCK_OK;
  });
}

extern "C" int hck_kv4_read(const void* pool, int64_t pages, int kv_heads, int head_dim, int type,
                            const int64_t* slots, int64_t tokens, void* keys, void* values, void* stream) {
  if (hck::kv4_bytes(head_dim) == 0 || type < HCK_BF16 || type > HCK_F32) return HCK_ERR_UNSUPPORTED;
  if (!pool || pages < 1 || kv_heads < 1 || kv_heads > 65535 || tokens < 0) return HCK_ERR_ARG;
  if (tokens == 0) return HCK_OK;
  const int64_t groups = (tokens + hck::kTokensPerGroup - 1) / hck::kTokensPerGroup;
  if (!keys || !values || !slots || groups > 0x7fffffff) return HCK_ERR_ARG;
  if (((uintptr_t)keys | (uintptr_t)values) % 16) return HCK_ERR_ARG;
  return hck::by_type(type, head_dim, [&](auto* t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    const bool past = 2 * sizeof(T) * tokens * kv_heads * head_dim > (size_t)hck::kL2s;
    auto* kernel = past ? hck::k_read<T, decltype(d)::value, true> : hck::k_read<T, decltype(d)::value, false>;
    kernel<<<dim3((unsigned)groups, kv_heads), 256, 0, (hipStream_t)stream>>>(
        (const uint8_t*)pool, pages, kv_heads, (const long long*)slots, tokens, (T*)keys, (T*)values);
    HCK_CHECK_LAUNCH();
    return HCK_OK;
  });
}
