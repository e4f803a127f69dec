// Attention of many rows over 4-bit pages: the mathematics of kv4_attend.hip, with 128 or 256 rows to a workgroup.
//
// Here a tile is 32 by 32: a lane has one row's scores of half of 64 tokens, and a matrix instruction keeps the
// vector unit from issuing for 8 cycles of its 32, where two of 16 by 16 do for 20 (measured), which counts where
// both are busy.  Making operands of the codes takes some 190 vector instructions per 64 tokens, as many as the
// softmax of 32 rows; so it is done once for a workgroup: each of its 4 or 8 waves makes its share of them, in the
// lanes' order, in LDS (keys and values 32 KB per 64 tokens, twice, so that one barrier is enough; with 8 waves two
// units to a barrier), and takes all of them for its own 32 rows.  The next codes are in flight meanwhile.  Which runs are
// summed times 2^-56 (kLargeByte) is the workgroup's, known after the barrier; where a step brings a new one, its
// operands are made again.
//
// What bounds it: per 64 tokens and 32 rows 48 matrix and some 350 vector instructions (D = 128), which two waves of
// a SIMD issue through one port.  4096 tokens, 32 query heads over 8 key heads of 128: 139 GFLOP in 195 to 205 us on
// different cards, at 198 us 702 TFLOP/s, and 1.05 PFLOP/s of the products that are done (three for two, by the
// probabilities' two parts); a bf16 8192^3 product runs at 1.20 PFLOP/s.
#include "kv4_attend.hpp"

namespace hck {
namespace {

// One thread's share of 64 tokens, with W waves: of one token's keys 32 dims (D = 64: 16), and of 4 tokens' values
// 8 (4) dims; with 8 waves half of these, which half by the wave.
template <int D, int W>
struct Share {
  static constexpr int kWords = D / 8 / W;
  uint32_t k[kWords], v[D / 32], ks, vs;
  struct Offsets {  // of a thread's bytes in the first half of a page
    uint32_t k, v, ks, vs;
    __device__ __forceinline__ Offsets(int wave, int lane) {
      using L = Kv4<D>;
      const int m = lane & 15, g = lane >> 4, quarter = wave & 3, block = quarter >> 1, piece = quarter & 1;
      k = quarter * (8 * D) + lane * (D / 8) + (wave >> 2) * (4 * kWords);
      ks = L::kKScales + g * (D / 4) / kRun * 64 + m * 4 + quarter;
      v = L::kVCodes + block * (16 * D) + (D == 128 ? piece * 1024 + lane * 16 : lane * 16 + piece * 8);
      vs = L::kVScales + block * (32 * L::kRuns) + (g * L::kRuns + m * L::kDpl / kRun) * 8 + 4 * piece;
    }
  };
  __device__ __forceinline__ void load(const uint8_t* page, int half, const Offsets& at) {
    typedef uint32_t kwords __attribute__((ext_vector_type(kWords)));
    typedef uint32_t vwords __attribute__((ext_vector_type(D / 32)));
    const uint8_t* codes = page + half * (32 * D);
    const uint8_t* scales = page + half * (64 * Kv4<D>::kRuns);
    *reinterpret_cast<kwords*>(k) = *reinterpret_cast<const kwords*>(codes + at.k);
    ks = scales[at.ks];
    *reinterpret_cast<vwords*>(v) = *reinterpret_cast<const vwords*>(codes + at.v);
    vs = *reinterpret_cast<const uint32_t*>(scales + at.vs);
  }
};

// The left operands of 64 tokens.  Keys: lane (token % 32, h) of step s has dims 8 of the D / 4 that follow
// (2 (s / (D / 32)) + h) D / 4.  Values: lane (i, h) of tile d has dim i / 2 kDpl + 2 d + i % 2 of the tokens
// 16 j + 4 h + 0..3 and 8 on, whose scores a lane with that h holds.
template <int D>
struct Operands {
  u32x4 k[2][D / 16][64];       // [32-token tile][step][lane]
  u32x2 v[4][D / 32][64][2];    // [16 tokens][32-dim tile][lane][4 tokens]
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Writes the thread's share, values of the runs `large` times 2^-56; whether it holds a run of NaN among the values, which
// are taken as zeros.
template <int D, int W>
__device__ __forceinline__ bool store(Operands<D>& o, const Share<D, W>& x, int wave, int lane, uint32_t large) {
  constexpr int kWords = Share<D, W>::kWords;
  const int m = lane & 15, g = lane >> 4, quarter = wave & 3, part = (wave >> 2) * kWords;
  const float sc = x.ks == kNanByte ? __uint_as_float(0x7fc00000u) : __uint_as_float(x.ks << 23);
#pragma unroll
  for (int s = 0; s < kWords; ++s)
    o.k[quarter >> 1][(g >> 1) * (D / 32) + part + s][(g & 1) * 32 + (quarter & 1) * 16 + m] =
        u32x4{cvt<0>(x.k[s], sc), cvt<1>(x.k[s], sc), cvt<2>(x.k[s], sc), cvt<3>(x.k[s], sc)};
  uint32_t vs = x.vs;
  const bool odd = has_nan(vs);
  if (odd) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (((vs >> (8 * j)) & 0xffu) == kNanByte) vs &= ~(0xffu << (8 * j));
  }
  if ((large >> (m * Kv4<D>::kDpl / kRun)) & 1) vs = down(vs);
  float f[4];
  uint32_t v[D / 32];
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = scale_of(vs, j);
#pragma unroll
  for (int j = 0; j < D / 32; ++j) v[j] = W == 4 ? x.v[j] : x.v[j] >> (8 * part);
  auto pair = [&](auto B) {  // dims 2 b, 2 b + 1 of the thread's
    constexpr int b = decltype(B)::value;
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (D == 128) y[j] = cvt<b>(v[j], f[j]);
      else y[j] = (j & 1) ? cvt<(b & 1) + 2>(v[j / 2], f[j]) : cvt<(b & 1)>(v[j / 2], f[j]);
    }
    u32x2(*to)[2] = &o.v[quarter][part + b][(g & 1) * 32 + 2 * m];
    to[0][g >> 1] = u32x2{__builtin_amdgcn_perm(y[1], y[0], 0x05040100u), __builtin_amdgcn_perm(y[3], y[2], 0x05040100u)};
    to[1][g >> 1] = u32x2{__builtin_amdgcn_perm(y[1], y[0], 0x07060302u), __builtin_amdgcn_perm(y[3], y[2], 0x07060302u)};
  };
  pair(std::integral_constant<int, 0>());
  if constexpr (kWords >= 2) pair(std::integral_constant<int, 1>());
  if constexpr (kWords >= 4) {
    pair(std::integral_constant<int, 2>());
    pair(std::integral_constant<int, 3>());
  }
  return odd;
}

// The bit of the thread's run, if one of its tokens before `most` has a unit of kLargeByte or more.
template <int D, int W>
__device__ __forceinline__ uint32_t large_run(const Share<D, W>& x, int wave, int lane, int unit, int most) {
  const int first = unit * kUnit + ((wave & 3) >> 1) * 32 + (wave & 1) * 16 + (lane >> 4) * 4;
  bool is = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t byte = (x.vs >> (8 * j)) & 0xffu;
    is = is || (byte >= kLargeByte && byte != kNanByte && first + j < most);
  }
  return is ? 1u << ((lane & 15) * Kv4<D>::kDpl / kRun) : 0;
}

template <typename T, int D, bool RANGE, int W>
__global__ __launch_bounds__(64 * W, waves_of_many(D)) void k_prompt(AttendArgs A) {
  using L = Kv4<D>;
  constexpr int kSteps = D / 16, kTiles = D / 32, kDpl = L::kDpl;
  constexpr bool kHalf = __is_same(T, _Float16);
  constexpr int kStep = W / 4;  // units between two barriers: a page where the LDS is one workgroup's
  __shared__ Operands<D> s_x[2][kStep];
  __shared__ int s_odd[2][kStep];  // 1 + the unit whose values hold a run of NaN
  __shared__ uint32_t s_large[2];  // runs with units of kLargeByte or more, a bit each

  Item it;
  if (!locate(A, blockIdx.x, it)) return;
  it.uniform();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const Rows S = it.rows;
  const int rows = S.rows, first = it.tile * (32 * W);
  if (first >= rows) return;
  const int most = S.seen(A, min(first + 32 * W, rows) - 1);
  const int u0 = it.u0, u1 = min((most + kUnit - 1) / kUnit, it.u1);
  const int mine = first + 32 * wave;  // the wave's rows
  const int least = mine < rows ? S.seen(A, mine) : 0, last = mine < rows ? S.seen(A, min(mine + 32, rows) - 1) : 0;
  const int row = mine + (lane & 31);
  const bool live = row < rows;
  const int qi = live ? row / A.group : 0, qo = live ? row % A.group : 0;
  const int seen = live ? S.seen(A, row) : 0;

  bf16x8 qh[kSteps], ql[kSteps];
  const T* qp = (const T*)A.q + (long long)(S.q0 + qi) * A.q_ts + (long long)(it.h * A.group + qo) * A.q_hs + h * (D / 4);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    u32x4 raw = {0, 0, 0, 0};
    if (live) raw = reinterpret_cast<const Loose16*>(qp + s / (D / 32) * (D / 2) + s % (D / 32) * 8)->v;
    query_parts<T>(raw, qh[s], ql[s]);
  }

  f32x16 acc[kTiles];
#pragma unroll
  for (int d = 0; d < kTiles; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  float top = -INFINITY, sum = 0.f, low = INFINITY;
  const float scale2 = A.scale * kLog2e;
  float ref = -kLift, factor = scale2;
  uint32_t large = 0;  // runs whose sums are held times 2^-56, the workgroup's

  const int* table = A.table + it.b * A.table_stride;
  const uint8_t* pool = A.pool + it.h * L::kBytes;
  const long long each = (long long)A.heads * L::kBytes;
  auto page_of = [&](int pg) { return pool + (pg < 0 || pg >= A.pages ? 0 : pg) * each; };
  const typename Share<D, W>::Offsets offsets(wave, lane);
  Share<D, W> x[kStep];
  auto load = [&](Share<D, W>* x, const uint8_t* page, int first) {
#pragma unroll
    for (int n = 0; n < kStep; ++n) x[n].load(page, kStep == 2 ? n : first & 1, offsets);
  };
  int pg = 0, next = 0, step = u0 / kStep * kStep;
  if (threadIdx.x < 2 * kStep) s_odd[threadIdx.x / kStep][threadIdx.x % kStep] = 0;
  if (threadIdx.x < 2) s_large[threadIdx.x] = 0;
  if (step < u1) {
    pg = __builtin_amdgcn_readfirstlane(table[step >> 1]);
    load(x, page_of(pg), step);
    if (step + kStep < u1) next = table[(step + kStep) >> 1];
  }
  __syncthreads();
  for (int turn = 0; step < u1; step += kStep, turn ^= 1) {
    Operands<D>(&os)[kStep] = s_x[turn];
    const bool there = pg >= 0 && pg < A.pages;
#pragma unroll
    for (int n = 0; n < kStep; ++n) {
      if (store(os[n], x[n], wave, lane, large)) s_odd[turn][n] = step + n + 1;
      if (there && has_large(x[n].vs)) atomicOr(&s_large[turn], large_run(x[n], wave, lane, step + n, most));
    }
    const uint8_t* page = page_of(pg);
    pg = __builtin_amdgcn_readfirstlane(next);
    if (step + kStep < u1) load(x, page_of(pg), step + kStep);
    if (step + 2 * kStep < u1) next = table[(step + 2 * kStep) >> 1];
    __syncthreads();
    if (!there) continue;
    if (const uint32_t fresh = __builtin_amdgcn_readfirstlane(s_large[turn]) & ~large) {
      // the first such units of their runs: the same for all waves, which make this step's operands again
      large |= fresh;
      Share<D, W> again[kStep];
      load(again, page, step);
#pragma unroll
      for (int n = 0; n < kStep; ++n) store(os[n], again[n], wave, lane, large);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if ((fresh >> ((i >> 2) * (D / 4) / kRun)) & 1) {  // registers 4 q .. 4 q + 3 have dims D / 4 q ..
#pragma unroll
          for (int d = 0; d < kTiles; ++d) acc[d][i] *= kDownBy;
        }
    }
#pragma unroll 1
    for (int n = 0; n < kStep; ++n) {
      const int u = step + n;
      const int here = __builtin_amdgcn_readfirstlane(u * kUnit);
      if (here >= last || u < u0 || u >= u1) continue;
      const Operands<D>& o = os[n];
      const int odd = s_odd[turn][n];

      f32x16 t[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) t[0][i] = t[1][i] = 0.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const bf16x8 kk = __builtin_bit_cast(bf16x8, o.k[n][s][lane]);
          t[n] = mfma32(kk, qh[s], t[n]);
          if constexpr (kHalf) t[n] = mfma32(kk, ql[s], t[n]);
        }
      const int base = here + 4 * h;  // of the lane's tokens base + 32 n + 8 (i / 4) + i % 4
      if (here + kUnit > least) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const bool see = base + 32 * n + 8 * (i >> 2) + (i & 3) < seen;
            if constexpr (RANGE) low = see ? fminf(low, t[n][i]) : low;
            t[n][i] = see ? t[n][i] : -INFINITY;
          }
      } else if constexpr (RANGE) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) low = smaller(low, t[n][i]);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = larger(mx, t[n][i]);
      const float raw = over_half(mx, fmax2);
      mx = fmaxf(top, raw * scale2);
      const float f = rebase(top, mx);
      top = mx;
      if (__any(f != 1.f)) {
        if (f != 1.f) refer(mx, raw, scale2, ref, factor);
        sum *= f;
#pragma unroll
        for (int d = 0; d < kTiles; ++d) acc[d] *= f;
      }

      if (odd == u + 1) {
        // A run of NaN must reach the rows that see its token, and no other: 0 * NaN is NaN.  Its values are
        // zeros here, and it is counted for the rows that see it by a product of truth values.
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          bf16x8 bad, see;
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint32_t vs = *reinterpret_cast<const uint32_t*>(
                page + L::kVScales + (2 * (u & 1) + (j >> 1)) * (32 * L::kRuns) +
                ((2 * p + h) * L::kRuns + (lane & 31) / 2 * kDpl / kRun) * 8 + 4 * (j & 1));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              bad[4 * p + k] = (__bf16)(((vs >> (8 * k)) & 0xffu) == kNanByte ? 1.f : 0.f);
              see[4 * p + k] = (__bf16)(base + 16 * j + 8 * p + k < seen ? 1.f : 0.f);
            }
          }
          f32x16 n;
#pragma unroll
          for (int i = 0; i < 16; ++i) n[i] = 0.f;
          n = mfma32(bad, see, n);
#pragma unroll
          for (int d = 0; d < kTiles; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (n[i] > 0.f) acc[d][i] = __uint_as_float(0x7fc00000u);
        }
      }

      // (a wave in its softmax and second product goes before one in its first, which only waits for the matrix unit)
      __builtin_amdgcn_s_setprio(1);
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float p[8];
        uint32_t hi[4], lo[4];  // the probabilities in two bf16 parts
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[j >> 1][8 * (j & 1) + e], factor, -ref));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          hi[e] = pack(p[2 * e], p[2 * e + 1]);
          lo[e] = rests_of(p[2 * e], p[2 * e + 1], hi[e]);
          part[e & 1] += p[2 * e] + p[2 * e + 1];
        }
        const bf16x8 ph = operand(hi[0], hi[1], hi[2], hi[3]), pl = operand(lo[0], lo[1], lo[2], lo[3]);
        bf16x8 vv[kTiles];
#pragma unroll
        for (int d = 0; d < kTiles; ++d) vv[d] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(o.v[j][d][lane]));
#pragma unroll
        for (int d = 0; d < kTiles; ++d) acc[d] = mfma32(vv[d], ph, acc[d]);
#pragma unroll
        for (int d = 0; d < kTiles; ++d) acc[d] = mfma32(vv[d], pl, acc[d]);
      }
      sum += part[0] + part[1];
      __builtin_amdgcn_s_setprio(0);
    }
  }

  publish(A, it);
  sum = over_half(sum, [](float a, float c) { return a + c; });
  if constexpr (RANGE) low = over_half(low, fmin2) * scale2;
  if (row >= rows || row - first >= A.rows) return;
  const int qr = row / A.group, qc = row % A.group;
  const long long out = (S.q0 + qr) * (long long)(A.heads * A.group) + it.h * A.group + qc;
  const long long at = (long long)it.slot * A.rows + (row - first);
  if (it.slots > 1 && h == 0) *reinterpret_cast<f32x4*>(A.stat + at * 4) = f32x4{top, sum, low, __uint_as_float(large)};
  // registers 4 q + 2 p + b of tile d: dim (2 h + 4 q + p) kDpl + 2 d + b of the lane's row
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d0 = (2 * h + 4 * (i >> 1) + (i & 1)) * kDpl;
    float v[kDpl];
#pragma unroll
    for (int d = 0; d < kDpl; ++d) v[d] = acc[d >> 1][2 * i + (d & 1)];
    if (it.slots > 1) {
#pragma unroll
      for (int d = 0; d < kDpl; d += 4) *reinterpret_cast<f32x4*>(A.sums + at * D + d0 + d) = f32x4{v[d], v[d + 1], v[d + 2], v[d + 3]};
    } else {
      store_row<T, kDpl, RANGE>(A, out, D, d0, top, sum, low, v, back(large, d0 / kRun));
    }
  }
}

template <typename T, int D, int W>
int launch(const AttendArgs& A, const Way& way, hipStream_t s) {
  if (A.low) k_prompt<T, D, true, W><<<dim3((unsigned)way.items), 64 * W, 0, s>>>(A);
  else k_prompt<T, D, false, W><<<dim3((unsigned)way.items), 64 * W, 0, s>>>(A);
  HCK_CHECK_LAUNCH();
  return HCK_OK;
}

}  // namespace

int launch_prompt(const AttendArgs& A, const Way& W, int head_dim, int type, hipStream_t s) {
  const bool half = type == HCK_F16;
  if (head_dim == 64) return half ? launch<_Float16, 64, 4>(A, W, s) : launch<__bf16, 64, 4>(A, W, s);
  if (W.size == 256) return half ? launch<_Float16, 128, 8>(A, W, s) : launch<__bf16, 128, 8>(A, W, s);
  return half ? launch<_Float16, 128, 4>(A, W, s) : launch<__bf16, 128, 4>(A, W, s);
}

}  // namespace hck
