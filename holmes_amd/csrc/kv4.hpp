// The 4-bit page format of the cleartext cache (kv4.hip, kv4_attend.hip).
//
// A page holds 128 tokens; the pool is [page][kv head][kBytes].  Values are e2m1 codes (0, .5, 1,
// 1.5, 2, 3, 4, 6 and their negatives) times 2^(b - 127), one byte b for each run of 32 values along
// the head dimension.  One head's part of a page is
//   key codes    [16-token tile][g < 4][token % 16][D / 8 bytes]: lane (token % 16, g) of a matrix product's
//                left operand holds dims g D/4 .. (g + 1) D/4 - 1, so a wave loads a tile as it lies
//   value codes  [32-token block][piece][g < 4][c < 16][16 bytes]: the product over tokens wants a lane to
//                hold one dim of 8 tokens, so lane (c, g) finds dims c D/16 .. (c + 1) D/16 - 1 of its tokens
//                j < 8 there, D/32 bytes each, 4 to a piece at D = 128 and all 8 at D = 64; tokens 4 g + j
//                (j < 4) and 16 + 4 g + j - 4 are the ones whose scores that lane holds after the first product
//   key scales   [64 tokens][run][token % 16][token / 16 % 4]: the bytes of a lane's token in four tiles
//   value scales [32-token block][g][run][j]: the bytes of a lane's 8 tokens
// A token owns every byte that it writes, so appends never read.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hck {

constexpr int kPageTokens = 128;
constexpr int kRun = 32;          // values that share a scale byte
constexpr int kNanByte = 255;     // the scale byte of a run that held an infinity or a NaN

template <int D>
struct Kv4 {
  static constexpr int kRuns = D / kRun;
  static constexpr int kDpl = D / 16;                       // dims of a lane in the product over tokens
  static constexpr int kCodes = kPageTokens * D / 2;        // bytes of the key or value codes
  static constexpr int kScales = kPageTokens * kRuns;
  static constexpr int kVCodes = kCodes, kKScales = 2 * kCodes, kVScales = kKScales + kScales;
  static constexpr int kBytes = 2 * (kCodes + kScales);
  __device__ static int key_code(int t, int d) {
    return (t >> 4) * (8 * D) + (d / (D / 4) * 16 + (t & 15)) * (D / 8) + d % (D / 4) / 2;
  }
  __device__ static int key_scale(int t, int run) {
    return kKScales + (t >> 6) * (64 * kRuns) + run * 64 + (t & 15) * 4 + ((t >> 4) & 3);
  }
  __device__ static int value_j(int t) { return ((t >> 4) & 1) * 4 + (t & 3); }
  __device__ static int value_g(int t) { return (t >> 2) & 3; }
  __device__ static int value_code(int t, int c) {
    const int at = value_j(t) * (kDpl / 2);
    return kVCodes + (t >> 5) * (16 * D) + (at >> 4) * 1024 + (value_g(t) * 16 + c) * 16 + (at & 15);
  }
  __device__ static int value_scale(int t, int run) {
    return kVScales + (t >> 5) * (32 * kRuns) + (value_g(t) * kRuns + run) * 8 + value_j(t);
  }
};

constexpr int64_t kL2s = 32 << 20;  // bytes of the XCDs' L2 caches together

// Whether so many workgroups can be launched along x: their threads are counted in 32 bits.
inline bool fits_grid(int64_t groups, int threads) { return groups <= 0xffffffffll / threads; }

// Bytes of one head's part of a page (host side; 0: no such head dimension).
inline int kv4_bytes(int head_dim) {
  return head_dim == 128 ? Kv4<128>::kBytes : head_dim == 64 ? Kv4<64>::kBytes : 0;
}

}  // namespace hck
