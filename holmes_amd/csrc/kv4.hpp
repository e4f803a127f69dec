// The 4-bit page format of the cleartext cache (kv4.hip, kv4_attend.hip).
//
// A page holds 128 tokens; the pool is [page][kv head][kBytes].  Values are e2m1 codes (0, .5, 1,
// 1.5, 2, 3, 4, 6 and their negatives) times 2^(b - 127), one byte b for each run of 32 values along
// the head dimension.  One head's part of a page is
//   key codes    [token][D / 2 bytes], as the matrix product's left operand takes a token's dims
//   value codes  [32-token block][g < 4][c < 16][j < 8][D / 16 codes]: the product over tokens wants a
//                lane to hold one dim of 8 tokens, so lane (c, g) finds its 8 tokens' dims
//                c D/16 .. (c + 1) D/16 - 1 in one piece of memory; tokens 4 g + j (j < 4) and
//                16 + 4 g + j - 4 are the ones whose scores that lane holds after the first product
//   key scales   [run][token % 16][token / 16]: the bytes of a lane's token in all eight 16-token tiles
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
  __device__ static int key_code(int t, int d) { return t * (D / 2) + d / 2; }
  __device__ static int key_scale(int t, int run) { return kKScales + run * kPageTokens + (t & 15) * 8 + (t >> 4); }
  __device__ static int value_j(int t) { return ((t >> 4) & 1) * 4 + (t & 3); }
  __device__ static int value_g(int t) { return (t >> 2) & 3; }
  __device__ static int value_code(int t, int c) {
    return kVCodes + (t >> 5) * (16 * D) + ((value_g(t) * 16 + c) * 8 + value_j(t)) * (kDpl / 2);
  }
  __device__ static int value_scale(int t, int run) {
    return kVScales + (t >> 5) * (32 * kRuns) + (value_g(t) * kRuns + run) * 8 + value_j(t);
  }
};

// Bytes of one head's part of a page (host side; 0: no such head dimension).
inline int kv4_bytes(int head_dim) {
  return head_dim == 128 ? Kv4<128>::kBytes : head_dim == 64 ? Kv4<64>::kBytes : 0;
}

}  // namespace hck
