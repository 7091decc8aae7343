// Storage of the paged 4-bit KV cache, shared by the kernels that write and read it.
//
// A page holds P tokens of every KV head; the block of one (page, head) is
//
//   K codes  P x D/2 bytes    token t at t * D/2: dword (q, i) = q * D/32 + i of it holds the
//                             values d = 32 i + 8 q + e: byte e & 3, low nibbles for e < 4
//   V codes  P x D/2 bytes    unit u = t/4 of four tokens: bytes [m 0..15][g][t/2 & 1][j/2][t & 1]
//                             hold the values d = 64 g + 4 m + j, low nibbles for even j
//   K scales P x [g] (s, lo)  fp16 pairs
//   V scales P/4 x [g] x (s of the unit's four tokens, lo of the four), fp16
//
// with G = D/64 groups of 64 values a token, each value = code * s + lo.  The order is the one in
// which the matrix instructions take their operands, so that attention loads 8 to 32 consecutive
// bytes a lane straight into registers: a dword masked to its low (or shifted, its high) nibbles is
// two pairs of codes that lie next to each other in an operand.  v_mfma_f32_16x16x32 wants 8 values
// along its sum in each lane.  For scores the sum runs over d: lane (token, q) takes d = 32 i + 8 q +
// (0..7) for step i, one dword.  For the output it runs over tokens: lane (m, q) takes the tokens
// 4 q + (0..3) of two 16-token tiles, which is also where the scores' result leaves the weights, so
// these never cross lanes; a unit of four tokens is one load.  Every token still owns whole bytes,
// so appending one never rewrites another's bits.
#pragma once

#include "qs_common.h"

namespace qs {

constexpr int kKv4Group = 64;
// Values are held to this much before they are coded, so that a group's largest value, its
// scale's rounding included, stays below fp16's 65504.
constexpr float kKv4Max = 60000.f;

struct Kv4Layout {
  int P, D, G;
  __host__ __device__ Kv4Layout(int P_, int D_) : P(P_), D(D_), G(D_ / kKv4Group) {}
  __host__ __device__ int v_codes() const { return P * D / 2; }
  __host__ __device__ int k_scales() const { return P * D; }
  __host__ __device__ int v_scales() const { return P * D + P * G * 4; }
  __host__ __device__ int bytes() const { return P * D + P * G * 8; }
  // byte offsets inside a block
  __host__ __device__ int k_dword(int t, int d) const {  // the dword that holds value d
    return t * (D / 2) + (((d & 31) >> 3) * (D / 32) + (d >> 5)) * 4;
  }
  __host__ __device__ static int k_shift(int d) { return 8 * (d & 3) + (d & 4); }
  // the byte that holds values d and d + 1 (d even); those of d + 2 lie two bytes on
  __host__ __device__ int v_byte(int t, int d) const {
    return v_codes() + ((((t >> 2) * 16 + ((d & 63) >> 2)) * G + (d >> 6)) * 2 + (t >> 1 & 1)) * 4 + (d & 2) + (t & 1);
  }
  __host__ __device__ int k_scale(int t, int g) const { return k_scales() + (t * G + g) * 4; }
  __host__ __device__ int v_scale(int t, int g) const {  // s; lo lies 8 bytes on
    return v_scales() + ((t >> 2) * G + g) * 16 + (t & 3) * 2;
  }
};

inline bool kv4_shape_ok(int64_t head_dim, int64_t page_size) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
         (page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128 || page_size == 256);
}

}  // namespace qs
