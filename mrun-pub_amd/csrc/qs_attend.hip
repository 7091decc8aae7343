// Attention over the paged 4-bit KV cache (gfx950).
//
//   k_kv4_attend : a wave takes 16 or 32 query rows of one KV head -- (new token, query head) pairs,
//                  the heads that share the KV head next to each other -- and walks the request's
//                  tokens 32 at a time; the waves of a block and the blocks of a split take every
//                  NW-th step of their range and join their results.
//   k_kv4_join   : joins the splits of a long context.
//
// o = sum_t p_t v_t / sum_t p_t with p_t = 2^(x_t - m), x the scores in units of log2 and m their
// running maximum, one pass over the cache.
#include "qs_kv4.h"
#include "qs_values.h"

namespace qs {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct AttendArgs {
  const void* q;
  const uint8_t* cache;
  const int* tables;
  const int* starts;
  const int* context;
  void* out;
  float* part_o;
  float2* part_ml;
  int64_t ldq_t, ldq_h, ld_table, T;
  int pages, P, shift, width, Hkv, grp, B, window, splits;
  float scale_log2;
};

// ---- operand arithmetic ----------------------------------------------------------------
// Eight values along the sum for the matrix instruction, of which 16-bit activations multiply
// fp16: cache values are code * s + lo in fp16 (one rounding, 2^-12), queries are exact, since a
// row of bf16 is first divided by a power of two that takes its largest value below 1 (8 bits fit
// fp16's 11 down to 2^-17 of that), weights are 0..1.  fp32 activations multiply fp32.

template <class T>
struct Ops {
  typedef f16x8 Frag;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pair(uint32_t w, int j) {  // codes j and j + 4 of w, as 1024 + c
    return (w >> (4 * j) & 0x000f000fu) | 0x64006400u;
  }
  static __device__ __forceinline__ f16x2 value(uint32_t p, f16x2 s, f16x2 lo) {
    const f16x2 off = {(_Float16)1024.f, (_Float16)1024.f};
    return __builtin_elementwise_fma(__builtin_bit_cast(f16x2, p) - off, s, lo);
  }
  // One dword of a token's key, and its (s, lo).
  static __device__ __forceinline__ Frag key(uint32_t w, uint32_t sl) {
    const f16x2 h = __builtin_bit_cast(f16x2, sl);
    const f16x2 s = {h[0], h[0]}, lo = {h[1], h[1]};
    Frag f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f16x2 v = value(pair(w, j), s, lo);
      f[2 * j] = v[0];
      f[2 * j + 1] = v[1];
    }
    return f;
  }
  // Values j (of four) of eight tokens: u holds the 16-bit words of token pairs, s and lo theirs.
  static __device__ __forceinline__ Frag val(const uint32_t (&u)[4], const uint32_t (&s)[4], const uint32_t (&lo)[4], int j) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 v = value(pair(u[i], j), __builtin_bit_cast(f16x2, s[i]), __builtin_bit_cast(f16x2, lo[i]));
      f[2 * i] = v[0];
      f[2 * i + 1] = v[1];
    }
    return f;
  }
  static __device__ __forceinline__ Frag weights(const float (&p)[8]) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<_Float16>(p[i]);
    return f;
  }
};

template <>
struct Ops<float> {
  struct Frag {
    float v[8];
  };
  static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag key(uint32_t w, uint32_t sl) {
    const float s = f16_bits_to_f32((uint16_t)sl), lo = f16_bits_to_f32((uint16_t)(sl >> 16));
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = __builtin_fmaf((float)(w >> Kv4Layout::k_shift(e) & 15u), s, lo);
    return f;
  }
  static __device__ __forceinline__ Frag val(const uint32_t (&u)[4], const uint32_t (&s)[4], const uint32_t (&lo)[4], int j) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int up = 16 * (i & 1);
      f.v[i] = __builtin_fmaf((float)(u[i / 2] >> (up + 4 * j) & 15u), f16_bits_to_f32((uint16_t)(s[i / 2] >> up)),
                              f16_bits_to_f32((uint16_t)(lo[i / 2] >> up)));
    }
    return f;
  }
  static __device__ __forceinline__ Frag weights(const float (&p)[8]) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = p[i];
    return f;
  }
};

// Maximum / sum over the four lanes of a query row (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float max_of(float a, float b) { return a > b ? a : b; }
__device__ __forceinline__ float quad_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = max_of(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_of(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- which rows a block has ---------------------------------------------------------------
// Request b's tiles of R rows start at floor(starts[b] grp / R) + b, which leaves each request room
// for its last, partial one and can be searched without sums over requests.  Tokens past the last
// request are those of one more, with nothing to see.
struct Tile {
  int64_t q0;       // first token of the request
  int b, n, row0;   // request, its new tokens, first row of the tile
  bool any;
};
__device__ __forceinline__ int64_t start_of(const AttendArgs& a, int b) {
  const int64_t s = b == 0 ? 0 : a.starts[b];
  return s < 0 ? 0 : s < a.T ? s : a.T;
}
__device__ __forceinline__ Tile find_tile(const AttendArgs& a, int64_t tile, int R) {
  const int lane = threadIdx.x & 63;
  int at = -1;
  for (int b0 = 0; b0 <= a.B; b0 += 64) {
    const int b = b0 + lane;
    const bool before = b <= a.B && (int64_t)((uint64_t)(start_of(a, b) * a.grp) / (unsigned)R) + b <= tile;
    const int n = __popcll(__ballot(before));
    at += n;
    if (n < 64) break;
  }
  Tile t;
  t.b = at;
  t.q0 = start_of(a, at);
  const int64_t q1 = at < a.B ? start_of(a, at + 1) : a.T;
  t.n = q1 > t.q0 ? (int)(q1 - t.q0) : 0;
  const int64_t row0 = (tile - ((int64_t)((uint64_t)(t.q0 * a.grp) / (unsigned)R) + at)) * R;
  t.any = row0 >= 0 && row0 < (int64_t)t.n * a.grp;
  t.row0 = (int)row0;
  return t;
}

template <class T, int D, int RT, int NW>
__global__ __launch_bounds__(64 * NW) void k_kv4_attend(AttendArgs a) {
  using O = Ops<T>;
  typedef typename O::Frag Frag;
  constexpr int G = D / kKv4Group, KS = D / 32, R = 16 * RT, W = 2 * G;
  constexpr bool kHalf = sizeof(T) == 2;
  __shared__ float s_o[NW][16][D + 4];
  __shared__ float2 s_ml[NW][16];
  const int lane = threadIdx.x & 63, n = lane & 15, qq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.y;
  const Tile tile = find_tile(a, blockIdx.x, R);
  if (!tile.any) return;
  const int rows = tile.n * a.grp;
  int ctx = tile.b < a.B ? a.context[tile.b] : 0;
  ctx = ctx < 0 ? 0 : ctx < (1 << 30) ? ctx : 1 << 30;
  const int past = ctx - tile.n;  // position of the first new token
  const int r_last = tile.row0 + R - 1 < rows ? tile.row0 + R - 1 : rows - 1;
  const int pos_min = past + tile.row0 / a.grp, pos_max = past + r_last / a.grp;
  // tokens [lo, hi) are seen by some row of the tile
  int hi = pos_max + 1;
  const int64_t reach = (int64_t)a.width << a.shift;
  if (hi > reach) hi = (int)reach;
  int lo = a.window > 0 && pos_min - a.window + 1 > 0 ? pos_min - a.window + 1 : 0;
  if (tile.b >= a.B || hi < lo) hi = lo;

  // queries: the lane's row, values d = 32 i + 8 qq + (0..7)
  Frag qf[RT][KS];
  float rs[RT];
  int pos[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = tile.row0 + rt * 16 + n;
    const bool in = row < rows;
    const int i = (in ? row : rows - 1) / a.grp;
    const int head = hk * a.grp + (in ? row : rows - 1) - i * a.grp;
    pos[rt] = past + i;
    const T* q = static_cast<const T*>(a.q) + (tile.q0 + i) * a.ldq_t + head * a.ldq_h + 8 * qq;
    float v[KS][8];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      load_values<T, 8>(q + 32 * k, v[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max_of(top, __builtin_fabsf(v[k][e]));
    }
    rs[rt] = a.scale_log2;
    if constexpr (kHalf) {
      int e2 = 0;
      if constexpr (__is_same(T, __bf16)) {
        top = quad_max(top);
        e2 = top < __builtin_inff() ? __builtin_amdgcn_frexp_expf(top) : 0;
        rs[rt] = __builtin_amdgcn_ldexpf(a.scale_log2, e2);
      }
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[rt][k][e] = static_cast<_Float16>(__builtin_amdgcn_ldexpf(v[k][e], -e2));
    } else {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[rt][k].v[e] = v[k][e];
    }
  }

  // this block's steps of 32 tokens, of which the wave takes every NW-th
  const int first = lo >> 5, steps = ((hi + 31) >> 5) - first;
  const int s0 = first + (int)((int64_t)steps * blockIdx.z / a.splits);
  const int s1 = first + (int)((int64_t)steps * (blockIdx.z + 1) / a.splits);

  const Kv4Layout L(a.P, D);
  const int64_t block_bytes = L.bytes();
  const int* table = a.tables + (int64_t)(tile.b < a.B ? tile.b : 0) * a.ld_table;

  f32x4 o[RT][G][4];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -__builtin_inff();
    l[rt] = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[rt][g][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  struct Raw {
    uint32_t k[2][KS], ks[2][G], v[2][W], vs[2][G][4];
    bool bad[2];
  };
  int ids = 0;
  // the pages of the wave's next 32 steps: lane l holds that of step l / 2, tokens 16 (l & 1)
  auto load_ids = [&](int it) {
    const int64_t t = (int64_t)(s0 + wave + NW * (it + (lane >> 1))) * 32 + 16 * (lane & 1);
    ids = t < hi ? table[t >> a.shift] : -1;
  };
  auto load = [&](int it, Raw& r) {
    if ((it & 31) == 0) load_ids(it);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = (s0 + wave + NW * it) * 32 + 16 * h;
      const int id = __builtin_amdgcn_readlane(ids, 2 * (it & 31) + h);
      r.bad[h] = id < 0 || id >= a.pages;
      const uint8_t* block = a.cache + ((int64_t)(r.bad[h] ? 0 : id) * a.Hkv + hk) * block_bytes;
      const int tl = t & (a.P - 1);
      const uint8_t* kp = block + (tl + n) * (D / 2) + qq * (KS * 4);
      const uint8_t* sp = block + L.k_scales() + (tl + n) * (G * 4);
      const uint8_t* vp = block + L.v_codes() + (tl / 4 + qq) * (32 * W * 4 / 2) + n * (W * 4);
      const uint8_t* wp = block + L.v_scales() + (tl / 4 + qq) * (G * 16);
      __builtin_memcpy(r.k[h], __builtin_assume_aligned(kp, KS * 4 < 16 ? KS * 4 : 16), KS * 4);
      __builtin_memcpy(r.ks[h], __builtin_assume_aligned(sp, G * 4), G * 4);
      __builtin_memcpy(r.v[h], __builtin_assume_aligned(vp, W * 4 < 16 ? W * 4 : 16), W * 4);
      __builtin_memcpy(r.vs[h], __builtin_assume_aligned(wp, 16), G * 16);
    }
  };

  Raw cur, next;
  const int its = s1 - s0 > wave ? (s1 - s0 - wave + NW - 1) / NW : 0;
  if (its > 0) load(0, cur);
  for (int it = 0; it < its; ++it) {
    if (it + 1 < its) load(it + 1, next);
    const int t0 = (s0 + wave + NW * it) * 32;
    const bool edge = t0 + 31 > pos_min || t0 + 32 > hi || t0 < lo || (a.window > 0 && t0 <= pos_max - a.window) ||
                      cur.bad[0] || cur.bad[1];
    if (edge) {  // tokens that no row sees take no part whatever their page holds
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int t = t0 + 16 * h + 4 * qq + 2 * c;
          const uint32_t keep = (!cur.bad[h] && t >= lo && t < hi ? 0xffffu : 0u) |
                                (!cur.bad[h] && t + 1 >= lo && t + 1 < hi ? 0xffff0000u : 0u);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            cur.vs[h][g][c] &= keep;
            cur.vs[h][g][2 + c] &= keep;
          }
        }
    }
    f32x4 sc[RT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sc[rt][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const Frag kf = O::key(cur.k[h][k], cur.ks[h][k / 2]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sc[rt][h] = O::mma(kf, qf[rt][k], sc[rt][h]);
      }
    }
    Frag pf[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = sc[rt][e >> 2][e & 3] * rs[rt];
      if (edge) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = t0 + 16 * (e >> 2) + 4 * qq + (e & 3);
          const bool see = t <= pos[rt] && t < hi && (a.window <= 0 || t > pos[rt] - a.window) && !cur.bad[e >> 2];
          x[e] = see ? x[e] : -__builtin_inff();
        }
      }
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = max_of(top, x[e]);
      top = max_of(m[rt], quad_max(top));
      const float base = top == -__builtin_inff() ? 0.f : top;
      if (__any(top > m[rt])) {
        const float f = __builtin_amdgcn_exp2f(m[rt] - base);
        l[rt] *= f;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[rt][g][j] *= f;
        m[rt] = top;
      }
      float p[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(x[e] - base);
        sum += p[e];
      }
      l[rt] += sum;
      pf[rt] = O::weights(p);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      uint32_t u[4], s[4], z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // token pairs (0, 1), (2, 3) of both tiles' units
        const int h = i >> 1, c = i & 1;
        if constexpr (G == 1) {
          u[i] = cur.v[h][c];
        } else {
          const uint32_t w0 = cur.v[h][(2 * c) * (G / 2) + g / 2], w1 = cur.v[h][(2 * c + 1) * (G / 2) + g / 2];
          u[i] = __builtin_amdgcn_perm(w1, w0, g & 1 ? 0x07060302u : 0x05040100u);
        }
        s[i] = cur.vs[h][g][c];
        z[i] = cur.vs[h][g][2 + c];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Frag vf = O::val(u, s, z, j);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][g][j] = O::mma(vf, pf[rt], o[rt][g][j]);
      }
    }
    cur = next;
  }

  // join the waves, 16 rows at a time
  constexpr int TPR = 64 * NW / 16, C = D / TPR;  // threads a row, values a thread
  const int row_of = threadIdx.x / TPR, d0 = (threadIdx.x % TPR) * C;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float sum = quad_sum(l[rt]);
    if (rt) __syncthreads();
    if (qq == 0) s_ml[wave][n] = {m[rt], sum};
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 w = {o[rt][g][0][r], o[rt][g][1][r], o[rt][g][2][r], o[rt][g][3][r]};
        *reinterpret_cast<f32x4*>(&s_o[wave][n][64 * g + 16 * qq + 4 * r]) = w;
      }
    __syncthreads();
    float top = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < NW; ++w) top = max_of(top, s_ml[w][row_of].x);
    const float base = top == -__builtin_inff() ? 0.f : top;
    float all = 0.f, v[C] = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 ml = s_ml[w][row_of];
      const float f = __builtin_amdgcn_exp2f(ml.x - base);
      all = __builtin_fmaf(ml.y, f, all);
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = __builtin_fmaf(s_o[w][row_of][d0 + c], f, v[c]);
    }
    const int row = tile.row0 + rt * 16 + row_of;
    if (row < rows) {
      const int i = row / a.grp;
      const int64_t at = (tile.q0 + i) * ((int64_t)a.Hkv * a.grp) + hk * a.grp + row - i * a.grp;
      if (a.splits == 1) {
        const float inv = all == 0.f ? 0.f : 1.f / all;
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] *= inv;
        store_values<T, C>(static_cast<T*>(a.out) + at * D + d0, v);
      } else {
        const int64_t pa = (int64_t)blockIdx.z * a.T * a.Hkv * a.grp + at;
        store_values<float, C>(a.part_o + pa * D + d0, v);
        if (d0 == 0) a.part_ml[pa] = {top, all};
      }
    }
  }
}

// A wave a row: the splits' maxima and sums first, then their results with weights.
template <class T, int D>
__global__ __launch_bounds__(256) void k_kv4_join(const float* part_o, const float2* part_ml, int64_t rows, int splits,
                                                  T* out) {
  constexpr int C = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  float2 ml = {-__builtin_inff(), 0.f};
  if (lane < splits) ml = part_ml[lane * rows + row];  // at most 64 splits
  const float top = wave_max(ml.x);
  const float base = top == -__builtin_inff() ? 0.f : top;
  const float f = __builtin_amdgcn_exp2f(ml.x - base);
  const float all = wave_sum_dpp(ml.y * f);
  float v[C] = {};
  for (int s = 0; s < splits; ++s) {
    const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), s));
    float x[C];
    load_values<float, C>(part_o + (s * rows + row) * D + lane * C, x);
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = __builtin_fmaf(x[c], w, v[c]);
  }
  const float inv = all == 0.f ? 0.f : 1.f / all;
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] *= inv;
  if constexpr (C * sizeof(T) >= 4) {
    store_values<T, C>(out + row * D + lane * C, v);
  } else {
    out[row * D + lane] = from_f32<T>(v[0]);
  }
}

// ---- launch -------------------------------------------------------------------------------

struct Plan {
  int rt, splits;
  int64_t tiles;
};

Plan plan_of(int64_t T, int64_t B, int Hkv, int grp, int D, int64_t max_query, int64_t max_context, int64_t window) {
  Plan p;
  const int64_t rows = (max_query > 0 && max_query < T ? max_query : T) * grp;
  p.rt = rows > 16 && D < 256 ? 2 : 1;
  const int R = 16 * p.rt;
  p.tiles = T * grp / R + B + 1;
  // blocks with work: a request's rows fill its tiles but for the last
  const int64_t real = (cdiv(rows, R) * B < p.tiles ? cdiv(rows, R) * B : p.tiles) * Hkv;
  int64_t span = max_context;
  if (window > 0 && span > window + max_query) span = window + max_query;
  const int64_t most = span / 256;  // two steps a wave at least
  int64_t s = real > 0 ? cdiv(1024, real) : 1;
  if (s > most) s = most;
  p.splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
  return p;
}

template <class T, int D>
int launch_attend(const AttendArgs& a, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)p.tiles, (unsigned)a.Hkv, (unsigned)p.splits);
  if (p.rt == 1)
    hipLaunchKernelGGL((k_kv4_attend<T, D, 1, 4>), grid, dim3(256), 0, s, a);
  else if constexpr (D < 256)
    hipLaunchKernelGGL((k_kv4_attend<T, D, 2, 4>), grid, dim3(256), 0, s, a);
  if (p.splits > 1) {
    const int64_t rows = a.T * a.Hkv * a.grp;
    hipLaunchKernelGGL((k_kv4_join<T, D>), dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, s, a.part_o, a.part_ml, rows,
                       p.splits, static_cast<T*>(a.out));
  }
  return hip_check(hipGetLastError(), "k_kv4_attend launch");
}

template <class T>
int launch_attend_d(const AttendArgs& a, const Plan& p, int D, hipStream_t s) {
  if (D == 64) return launch_attend<T, 64>(a, p, s);
  if (D == 128) return launch_attend<T, 128>(a, p, s);
  return launch_attend<T, 256>(a, p, s);
}

int check_sizes(int64_t T, int64_t B, int Hkv, int Hq, int D, int64_t page_size) {
  if (!kv4_shape_ok(D, page_size))
    return fail(QS_ERR_UNSUPPORTED, "kv4_attend: head size %d, page size %lld", D, (long long)page_size);
  if (T < 0 || B < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv) return fail(QS_ERR_INVALID, "kv4_attend: bad shape");
  if (B > (1 << 20) || Hkv > 65535 || T * Hq >= (int64_t(1) << 31))
    return fail(QS_ERR_LIMIT, "kv4_attend: over 2^20 requests, 65535 heads or 2^31 query rows");
  return QS_OK;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" size_t qs_kv4_attend_workspace_bytes(int64_t T, int64_t B, int Hkv, int Hq, int D, int64_t page_size,
                                                int64_t max_query, int64_t max_context, int64_t window) {
  if (check_sizes(T, B, Hkv, Hq, D, page_size) != QS_OK) return 0;
  const Plan p = plan_of(T, B, Hkv, Hq / Hkv, D, max_query, max_context, window);
  return p.splits > 1 ? (size_t)p.splits * T * Hq * (D + 2) * sizeof(float) : 0;
}

extern "C" int qs_kv4_attend(const void* q, int dtype, int64_t ldq_t, int64_t ldq_h, const uint8_t* cache,
                             int64_t pages, int64_t page_size, int Hkv, int Hq, int D, const int32_t* tables,
                             int64_t ld_table, int64_t width, const int32_t* starts, const int32_t* context, int64_t B,
                             int64_t T, int64_t max_query, int64_t max_context, float scale, int64_t window, void* out,
                             void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_sizes(T, B, Hkv, Hq, D, page_size);
  if (bad != QS_OK) return bad;
  if (pages <= 0 || pages >= (int64_t(1) << 31) || width < 0 || width >= (int64_t(1) << 31) || (B > 1 && ld_table < width))
    return fail(QS_ERR_INVALID, "kv4_attend: bad page table");
  if (!(scale > 0.f) || scale > 3e38f) return fail(QS_ERR_INVALID, "kv4_attend: the scale is positive and finite");
  if (window < 0 || max_query < 0 || max_context < 0) return fail(QS_ERR_INVALID, "kv4_attend: negative bound");
  if (T == 0) return QS_OK;
  if (!q || !cache || !out || (B > 0 && (!starts || !context)) || (B > 0 && width > 0 && !tables))
    return fail(QS_ERR_INVALID, "kv4_attend: null pointer");
  const int per16 = dtype == QS_F32 ? 4 : 8;
  if (ldq_t % per16 || ldq_h % per16 || !aligned(q, 16) || !aligned(out, 16) || !aligned(cache, 16))
    return fail(QS_ERR_INVALID, "kv4_attend: 16-byte alignment");
  const int grp = Hq / Hkv;
  const Plan p = plan_of(T, B, Hkv, grp, D, max_query, max_context, window);
  const int64_t part = (int64_t)p.splits * T * Hq;
  if (p.splits > 1 && (!workspace || workspace_bytes < (size_t)part * (D + 2) * sizeof(float) || !aligned(workspace, 16)))
    return fail(QS_ERR_INVALID, "kv4_attend: workspace of qs_kv4_attend_workspace_bytes() bytes, 16-byte aligned");
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  AttendArgs a{q, cache, tables, starts, context, out, static_cast<float*>(workspace),
               reinterpret_cast<float2*>(static_cast<float*>(workspace) + part * D), ldq_t, ldq_h, ld_table, T,
               (int)pages, (int)page_size, shift, (int)width, Hkv, grp, (int)B,
               (int)(window < (1 << 30) ? window : 1 << 30), p.splits, scale * 1.44269504088896340736f};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == QS_F32) return launch_attend_d<float>(a, p, D, s);
  if (dtype == QS_BF16) return launch_attend_d<__bf16>(a, p, D, s);
  if (dtype == QS_F16) return launch_attend_d<_Float16>(a, p, D, s);
  return fail(QS_ERR_INVALID, "kv4_attend: dtype must be F32, BF16 or F16");
}
