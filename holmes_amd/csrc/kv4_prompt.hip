// Attention of many rows over 4-bit pages: the mathematics of kv4_attend.hip, with 128 rows to a workgroup.
//
// Per 64 tokens and 16 rows the products take 48 matrix instructions of 16 cycles (D = 128: 16 for the scores,
// 32 for the two parts of the probabilities) and the softmax some 150 vector instructions of 4; making operands
// of the codes would take 190 more.  So it is done once for 128 rows: the four waves each make a quarter of 64
// tokens' operands, in the lanes' order, in LDS (keys and values 32 KB, twice, so that one barrier a unit is
// enough), and each takes all of them for its own 32 rows.  Codes of the next unit are in flight meanwhile.
#include "kv4_attend.hpp"

namespace hck {
namespace {

// One thread's quarter-wave share of 64 tokens: 32 dims (D = 64: 16) of one token's keys, and 8 (4) dims of 4
// tokens' values.
template <int D>
struct Share {
  uint32_t k[D / 32], v[D / 32], ks, vs;
  __device__ __forceinline__ void load(const uint8_t* page, int half, int wave, int lane) {
    using L = Kv4<D>;
    typedef uint32_t words __attribute__((ext_vector_type(D / 32)));
    const int m = lane & 15, g = lane >> 4, block = 2 * half + (wave >> 1), piece = wave & 1;
    *reinterpret_cast<words*>(k) = *reinterpret_cast<const words*>(page + (4 * half + wave) * (8 * D) + lane * (D / 8));
    ks = page[L::kKScales + half * (64 * L::kRuns) + g * (D / 4) / kRun * 64 + m * 4 + wave];
    *reinterpret_cast<words*>(v) = *reinterpret_cast<const words*>(
        page + L::kVCodes + block * (16 * D) + (D == 128 ? piece * 1024 + lane * 16 : lane * 16 + piece * 8));
    vs = *reinterpret_cast<const uint32_t*>(page + L::kVScales + block * (32 * L::kRuns) +
                                            (g * L::kRuns + m * L::kDpl / kRun) * 8 + 4 * piece);
  }
};

template <int D>
struct Operands {
  u32x4 k[4][D / 32][64];            // [16-token tile][step][lane]
  u32x2 v[2][Kv4<D>::kDpl][64][2];   // [32-token block][dim of the lane][lane][4 tokens]
};

// Writes the thread's share; whether it holds a run of NaN among the values, which are taken as zeros.
template <int D>
__device__ __forceinline__ bool store(Operands<D>& o, const Share<D>& x, int wave, int lane) {
  const float sc = x.ks == kNanByte ? __uint_as_float(0x7fc00000u) : __uint_as_float(x.ks << 23);
#pragma unroll
  for (int s = 0; s < D / 32; ++s)
    o.k[wave][s][lane] = u32x4{cvt<0>(x.k[s], sc), cvt<1>(x.k[s], sc), cvt<2>(x.k[s], sc), cvt<3>(x.k[s], sc)};
  uint32_t vs = x.vs;
  const bool odd = has_nan(vs);
  if (odd) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (((vs >> (8 * j)) & 0xffu) == kNanByte) vs &= ~(0xffu << (8 * j));
  }
  float f[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = scale_of(vs, j);
  auto pair = [&](auto B) {
    constexpr int b = decltype(B)::value;
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (D == 128) y[j] = cvt<b>(x.v[j], f[j]);
      else y[j] = (j & 1) ? cvt<(b & 1) + 2>(x.v[j / 2], f[j]) : cvt<(b & 1)>(x.v[j / 2], f[j]);
    }
    o.v[wave >> 1][2 * b][lane][wave & 1] =
        u32x2{__builtin_amdgcn_perm(y[1], y[0], 0x05040100u), __builtin_amdgcn_perm(y[3], y[2], 0x05040100u)};
    o.v[wave >> 1][2 * b + 1][lane][wave & 1] =
        u32x2{__builtin_amdgcn_perm(y[1], y[0], 0x07060302u), __builtin_amdgcn_perm(y[3], y[2], 0x07060302u)};
  };
  pair(std::integral_constant<int, 0>());
  pair(std::integral_constant<int, 1>());
  if constexpr (D == 128) {
    pair(std::integral_constant<int, 2>());
    pair(std::integral_constant<int, 3>());
  }
  return odd;
}

template <typename T, int D, bool RANGE>
__global__ __launch_bounds__(64 * kWaves, waves_of_many(D)) void k_prompt(AttendArgs A) {
  using L = Kv4<D>;
  constexpr int kSteps = D / 32, kDpl = L::kDpl, kTiles = kMany / (16 * kWaves);  // 16-row tiles of a wave
  constexpr bool kHalf = __is_same(T, _Float16);
  __shared__ Operands<D> s_x[2];
  __shared__ int s_odd[2];  // 1 + the unit whose values hold a run of NaN

  Item it;
  if (!locate(A, kMany, blockIdx.x, it)) return;
  it.uniform();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  const int h = it.h;
  const Rows S = Rows(A, it.b).uniform();
  const int rows = S.rows, first = it.tile * kMany;
  if (first >= rows) return;
  const int most = S.seen(A, min(first + kMany, rows) - 1);
  const int u0 = it.u0, u1 = min((most + kUnit - 1) / kUnit, it.u1);
  const int mine = first + 16 * kTiles * wave;  // the wave's rows
  const int least = mine < rows ? S.seen(A, mine) : 0, last = mine < rows ? S.seen(A, min(mine + 16 * kTiles, rows) - 1) : 0;

  // the lane's part of its rows' queries: dims D / 4 g + 8 s .. + 7 of step s
  bf16x8 qh[kTiles][kSteps], ql[kTiles][kSteps];
  int seen[kTiles];
#pragma unroll
  for (int r = 0; r < kTiles; ++r) {
    const int row = mine + 16 * r + m;
    const bool live = row < rows;
    const int qi = live ? row / A.group : 0, qo = live ? row % A.group : 0;
    seen[r] = live ? S.seen(A, row) : 0;
    const T* qp = (const T*)A.q + (S.q0 + qi) * A.q_ts + (long long)(h * A.group + qo) * A.q_hs + g * (D / 4);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      u32x4 raw = {0, 0, 0, 0};
      if (live) raw = reinterpret_cast<const Loose16*>(qp + 8 * s)->v;
      query_parts<T>(raw, qh[r][s], ql[r][s]);
    }
  }

  f32x4 acc[kTiles][kDpl];
  float top[kTiles], sum[kTiles], low[kTiles];
#pragma unroll
  for (int r = 0; r < kTiles; ++r) {
    top[r] = -INFINITY, sum[r] = 0.f, low[r] = INFINITY;
#pragma unroll
    for (int d = 0; d < kDpl; ++d) acc[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float scale2 = A.scale * kLog2e;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  const int* table = A.table + it.b * A.table_stride;
  auto page_of = [&](int pg) { return A.pool + ((long long)(pg < 0 || pg >= A.pages ? 0 : pg) * A.heads + h) * L::kBytes; };
  Share<D> x;
  int pg = 0, next = 0;
  if (threadIdx.x < 2) s_odd[threadIdx.x] = 0;
  if (u0 < u1) {
    pg = __builtin_amdgcn_readfirstlane(table[u0 >> 1]);
    x.load(page_of(pg), u0 & 1, wave, lane);
    if (u0 + 1 < u1) next = table[(u0 + 1) >> 1];
  }
  __syncthreads();
  for (int u = u0; u < u1; ++u) {
    Operands<D>& o = s_x[u & 1];
    if (store(o, x, wave, lane)) s_odd[u & 1] = u + 1;
    const bool there = pg >= 0 && pg < A.pages;
    const uint8_t* page = page_of(pg);
    pg = __builtin_amdgcn_readfirstlane(next);
    if (u + 1 < u1) x.load(page_of(pg), (u + 1) & 1, wave, lane);
    if (u + 2 < u1) next = table[(u + 2) >> 1];
    __syncthreads();
    const int here = __builtin_amdgcn_readfirstlane(u * kUnit);
    if (!there || here >= last) continue;
    const bool full = here + kUnit <= least;  // every row sees every token

    f32x4 t[kTiles][4];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 kk = __builtin_bit_cast(bf16x8, o.k[i][s][lane]);
#pragma unroll
        for (int r = 0; r < kTiles; ++r) {
          t[r][i] = mfma(kk, qh[r][s], s == 0 ? zero : t[r][i]);
          if constexpr (kHalf) t[r][i] = mfma(kk, ql[r][s], t[r][i]);
        }
      }
    const int base = u * kUnit + 4 * g;
    u32x2 hi[kTiles][4], lo[kTiles][4];  // the probabilities in two bf16 parts
#pragma unroll
    for (int r = 0; r < kTiles; ++r) {
      if (!full) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bool see = base + 16 * i + k < seen[r];
            if constexpr (RANGE) low[r] = see ? fminf(low[r], t[r][i][k]) : low[r];
            t[r][i][k] = see ? t[r][i][k] : -INFINITY;
          }
      } else if constexpr (RANGE) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) low[r] = smaller(low[r], t[r][i][k]);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) mx = larger(mx, t[r][i][k]);
      mx = fmaxf(top[r], over_g(mx, fmax2) * scale2);
      const float f = rebase(top[r], mx);
      top[r] = mx;
      const float ref = reference(mx) - kLift;
      if (__any(f != 1.f)) {
        sum[r] *= f;
#pragma unroll
        for (int d = 0; d < kDpl; ++d) acc[r][d] *= f;
      }
      float part[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) t[r][i][k] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[r][i][k], scale2, -ref));
        part[i] = (t[r][i][0] + t[r][i][1]) + (t[r][i][2] + t[r][i][3]);
        hi[r][i] = u32x2{heads_of(t[r][i][0], t[r][i][1]), heads_of(t[r][i][2], t[r][i][3])};
        lo[r][i] = u32x2{rests_of(t[r][i][0], t[r][i][1], hi[r][i][0]), rests_of(t[r][i][2], t[r][i][3], hi[r][i][1])};
      }
      sum[r] += (part[0] + part[1]) + (part[2] + part[3]);
    }

    if (s_odd[u & 1] == u + 1) {
      // A run of NaN must reach the rows that see its token, and no other: 0 * NaN is NaN.  Its values are
      // zeros here, and it is counted for the rows that see it by a product of truth values.
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const u32x2 vs = *reinterpret_cast<const u32x2*>(page + L::kVScales + (2 * (u & 1) + i) * (32 * L::kRuns) +
                                                         (g * L::kRuns + m * L::kDpl / kRun) * 8);
        bf16x8 bad;
#pragma unroll
        for (int k = 0; k < 8; ++k) bad[k] = (__bf16)(((vs[k >> 2] >> (8 * (k & 3))) & 0xffu) == kNanByte ? 1.f : 0.f);
#pragma unroll
        for (int r = 0; r < kTiles; ++r) {
          bf16x8 see;
#pragma unroll
          for (int k = 0; k < 8; ++k) see[k] = (__bf16)(base + 32 * i + 16 * (k >> 2) + (k & 3) < seen[r] ? 1.f : 0.f);
          const f32x4 n = mfma(bad, see, zero);
#pragma unroll
          for (int d = 0; d < kDpl; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (n[k] > 0.f) acc[r][d][k] = __uint_as_float(0x7fc00000u);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 0; d < kDpl; ++d) {
        const bf16x8 vv = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(o.v[i][d][lane]));
#pragma unroll
        for (int r = 0; r < kTiles; ++r) {
          acc[r][d] = mfma(vv, operand(hi[r][2 * i][0], hi[r][2 * i][1], hi[r][2 * i + 1][0], hi[r][2 * i + 1][1]), acc[r][d]);
          acc[r][d] = mfma(vv, operand(lo[r][2 * i][0], lo[r][2 * i][1], lo[r][2 * i + 1][0], lo[r][2 * i + 1][1]), acc[r][d]);
        }
      }
  }

  publish(A, it);
  // lane (m, g) holds dims D / 4 g + kDpl i + d of row m in acc[d][i]
#pragma unroll
  for (int r = 0; r < kTiles; ++r) {
    sum[r] = over_g(sum[r], [](float a, float c) { return a + c; });
    if constexpr (RANGE) low[r] = over_g(low[r], fmin2) * scale2;
    const int row = mine + 16 * r + m;
    if (row >= rows || row - first >= A.rows) continue;
    if (it.slots > 1) {
      const long long at = (long long)it.slot * A.rows + (row - first);
      if (g == 0) *reinterpret_cast<f32x4*>(A.stat + at * 4) = f32x4{top[r], sum[r], low[r], 0.f};
      float* to = A.sums + at * D + g * (D / 4);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < kDpl; d += 4)
          *reinterpret_cast<f32x4*>(to + kDpl * i + d) = f32x4{acc[r][d][i], acc[r][d + 1][i], acc[r][d + 2][i], acc[r][d + 3][i]};
    } else {
      float v[D / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < kDpl; ++d) v[kDpl * i + d] = acc[r][d][i];
      const int qr = row / A.group, qc = row % A.group;
      store_row<T, D / 4, RANGE>(A, (S.q0 + qr) * (long long)(A.heads * A.group) + h * A.group + qc, D, g * (D / 4), top[r],
                                 sum[r], low[r], v);
    }
  }
}

template <typename T, int D>
int launch(const AttendArgs& A, const Way& W, hipStream_t s) {
  if (A.low) k_prompt<T, D, true><<<dim3((unsigned)W.items), 64 * kWaves, 0, s>>>(A);
  else k_prompt<T, D, false><<<dim3((unsigned)W.items), 64 * kWaves, 0, s>>>(A);
  HCK_CHECK_LAUNCH();
  return HCK_OK;
}

}  // namespace

int launch_prompt(const AttendArgs& A, const Way& W, int head_dim, int type, hipStream_t s) {
  if (head_dim == 128) return type == HCK_F16 ? launch<_Float16, 128>(A, W, s) : launch<__bf16, 128>(A, W, s);
  return type == HCK_F16 ? launch<_Float16, 64>(A, W, s) : launch<__bf16, 64>(A, W, s);
}

}  // namespace hck
