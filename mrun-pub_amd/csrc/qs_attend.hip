// Attention over the paged 4-bit KV cache (gfx950).
//
//   k_attend_few  : up to 32 query rows of one KV head -- (new token, query head) pairs, the heads
//                   that share the KV head next to each other -- a block.  Each wave takes all rows
//                   over every NW-th step of 32 tokens, codes straight from memory into the matrix
//                   instructions' operands; the waves' results join in LDS.
//   k_attend_rows : 128 rows a block, 32 a wave; the block unpacks 64 tokens at a time into LDS,
//                   where every wave reads them.
//
// o = sum_t p_t v_t / sum_t p_t with p_t = 2^(x_t - m), x the scores in units of log2 and m their
// running maximum, one pass over the cache.  Blocks share the requests' tokens out among themselves
// (pick_part); where several take parts of one tile's tokens, the last of them to finish joins them.
//
// Measured on an MI355X whose copy reaches 4.84 TB/s and whose 8192^3 bf16 product 1217 TFLOP/s, heads
// of 128, a call from Python:
//   1 token over 513, 12 + 2 heads           7.4 us  latency: plan, pages, first codes, 3 steps, join
//   29 requests up to 8100, 32 + 8 heads    30.8 us  3.6 TB/s; the vector unit unpacks 58% of it
//   2 contexts of 131000, fp16              65.4 us  4.6 TB/s
//   11 requests of 5 tokens up to 6001      18.6 us  latency
//   4095 tokens, 32 + 8 heads                171 us  803 TFLOP/s: vector operations 49% and products 38%
//                                                    of the cycles, hardly at once
//   chunks of 701, window 1024, fp32 of 64  36.3 us  152 TFLOP/s, the fp32 product's own rate
#include <atomic>
#include <type_traits>

#include "qs_kv4.h"
#include "qs_span.h"
#include "qs_values.h"

namespace qs {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct AttendArgs {
  const void* q;
  const uint8_t* cache;
  const int* tables;
  const int* starts;
  const int* context;
  void* out;
  // places: `blocks` of them, for the parts of tiles that are cut into several
  float* part_o;    // [place][rows of a tile * D]
  float2* part_ml;  // [place][rows of a tile]
  int* done;        // [place]: parts finished of the tile whose first part's it is; 0 between calls
  int64_t ldq_t, ldq_h, ld_table;
  int pages, P, shift, Hkv, grp, T, B, window;
  int reach;                // tokens that a table row has room for, 2^30 at most
  int blocks, least, whole;  // parts: blocks to fill (0: no parts), steps of a part at least, steps that stay whole
  int rows_from, rows_upto;  // requests of other row counts are the other kernel's
  float scale_log2;
};

// ---- operand arithmetic ----------------------------------------------------------------
// A byte 0..15 read as an e4m3 number is byte * 2^-9 (subnormals below 8, one binade above), so one
// conversion with scale 2^9 gives two codes as 16-bit floats.
//
// bf16 activations multiply fp16: cache values are code * s + lo in fp16 (one rounding, 2^-11),
// queries are exact, since a row of bf16 is first divided by a power of two that takes its largest
// value below 1 (8 bits fit fp16's 11 down to 2^-17 of that; smaller values keep steps of 2^-24 of the
// row's largest), weights are fp16.
//
// fp16 and fp32 activations, whose own rounding is no coarser than that, multiply the codes, which
// both 16-bit types hold exactly: q.k = s (q.code) + lo sum(q) a group, and for the output the
// weights are p s, with p lo summed beside.  fp16 queries are operands as they are, fp32 ones sums of
// three bf16 numbers (8 bits each, all of fp32's 24); p s is a sum of two or three bf16 numbers.
// Three instructions of the 16-bit rate replace the fp32 instruction's sixteenfold time.  Codes are
// 0..15 and lo is near -7.5 s, so the two sums of an output are large and cancel: fp32 adds p lo to the
// products' sum at every step, where both are still small, which leaves the result as exact as values
// multiplied in fp32 (a prompt of 300, heads of 128: 3.4e-7 off 64 bits, 8.5e-7 with two sums to the end).
constexpr uint32_t kNibbles = 0x0f0f0f0fu;

template <class T>
constexpr int kKind = __is_same(T, __bf16) ? 0 : sizeof(T) == 2 ? 1 : 2;
template <class T>
constexpr bool kCodes = kKind<T> != 0;
template <class T>
constexpr bool kFold = kKind<T> == 2;  // p lo joins the products' sum at every step
template <class T>
constexpr int kQueryParts = kKind<T> == 2 ? 3 : 1;
template <class T>
constexpr int kWeightParts = kKind<T> + 1;

template <bool HI>
__device__ __forceinline__ f16x2 f16_codes(uint32_t w) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 512.f, HI);
}
template <bool HI>
__device__ __forceinline__ bf16x2 bf16_codes(uint32_t w) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 512.f, HI);
}

__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The eight codes of a key's dword.
__device__ __forceinline__ void codes_of(uint32_t w, f16x8& f) {
  const uint32_t a = w & kNibbles, b = w >> 4 & kNibbles;
  const f16x2 v0 = f16_codes<false>(a), v1 = f16_codes<true>(a), v2 = f16_codes<false>(b), v3 = f16_codes<true>(b);
  f = f16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}
__device__ __forceinline__ void codes_of(uint32_t w, bf16x8& f) {
  const uint32_t a = w & kNibbles, b = w >> 4 & kNibbles;
  const bf16x2 v0 = bf16_codes<false>(a), v1 = bf16_codes<true>(a), v2 = bf16_codes<false>(b), v3 = bf16_codes<true>(b);
  f = bf16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

template <class T>
struct Ops {
  typedef std::conditional_t<kKind<T> == 2, bf16x8, f16x8> KFrag;  // of keys and queries
  typedef std::conditional_t<kCodes<T>, bf16x8, f16x8> VFrag;      // of values and weights
  // One dword of a token's key, and its (s, lo).
  static __device__ __forceinline__ KFrag key(uint32_t w, uint32_t sl) {
    KFrag f;
    codes_of(w, f);
    if constexpr (!kCodes<T>) {
      const f16x2 h = __builtin_bit_cast(f16x2, sl);
      const f16x2 s = {h[0], h[0]}, lo = {h[1], h[1]};
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const f16x2 v = __builtin_elementwise_fma(f16x2{f[i], f[i + 1]}, s, lo);
        f[i] = v[0];
        f[i + 1] = v[1];
      }
    }
    return f;
  }
  // Values 4 m + J of eight tokens: u holds the bytes of token pairs, s and lo the pairs' own.
  template <int J>
  static __device__ __forceinline__ VFrag val(const uint32_t (&u)[4], const uint32_t (&s)[4], const uint32_t (&lo)[4]) {
    VFrag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = (J & 1 ? u[i] >> 4 : u[i]) & kNibbles;
      if constexpr (kCodes<T>) {
        const bf16x2 v = bf16_codes<(J >> 1) != 0>(w);
        f[2 * i] = v[0];
        f[2 * i + 1] = v[1];
      } else {
        const f16x2 v = __builtin_elementwise_fma(f16_codes<(J >> 1) != 0>(w), __builtin_bit_cast(f16x2, s[i]),
                                                  __builtin_bit_cast(f16x2, lo[i]));
        f[2 * i] = v[0];
        f[2 * i + 1] = v[1];
      }
    }
    return f;
  }
};

// Eight fp32 values as operands: rounded to fp16, or as two or three bf16 parts.
__device__ __forceinline__ void parts_of(const float (&v)[8], f16x8 (&p)[1]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) p[0][i] = static_cast<_Float16>(v[i]);
}
template <int N>
__device__ __forceinline__ void parts_of(const float (&v)[8], bf16x8 (&p)[N]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float r = v[i];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      p[k][i] = static_cast<__bf16>(r);
      r -= static_cast<float>(p[k][i]);
    }
  }
}

// Adds eight weights to l: the rounded ones in pairs where they are fp16, which is what the values are
// multiplied by.
__device__ __forceinline__ float add_weights(const float (&)[8], const f16x8 (&p)[1], float l) {
  const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
  for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2(f16x2{p[0][i], p[0][i + 1]}, one, l, false);
  return l;
}

__device__ __forceinline__ float max_of(float a, float b) { return a > b ? a : b; }
// The larger, NaN if either is: one operation for two more values, and none to quiet its inputs.
__device__ __forceinline__ float top_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// Maximum / sum over lanes l and l ^ 32, and over the four of l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_of(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float quad_max(float v) {
  v = pair_max(v);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_of(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
  v = pair_sum(v);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 2^(score - maximum), the score still to be multiplied by rs.  Codes: multiplied first, so that the score
// that is the maximum has weight 1 exactly; what code s and lo cancel of each other then loses nothing
// in a row that sees one token, and in others 2^-24 of the group's range, not of the value.
template <class T>
__device__ __forceinline__ float weight_of(float x, float rs, float base) {
  if constexpr (kCodes<T>) return __builtin_amdgcn_exp2f(x * rs - base);
  return __builtin_amdgcn_exp2f(__builtin_fmaf(x, rs, -base));
}

// A maximum is moved only by scores that pass it by 2^8: weights up to 256 lose nothing in fp16 or
// fp32, and most steps then leave the sums alone.
constexpr float kSlack = 8.f;

// ---- which rows and tokens a block has -----------------------------------------------------
struct Work {
  int64_t q0;         // first token of the request
  int b, n, ctx, row0;  // request, its new tokens and context, first row of the tile
  int part, parts;    // which part of the tile's tokens, of how many
  int64_t first;      // place of the tile's part 0 (of one KV head's, as are blocks)
  int hk;
  bool any;
};

__device__ __forceinline__ int64_t start_of(const AttendArgs& a, int b) {
  const int64_t s = b == 0 ? 0 : a.starts[b];
  return s < 0 ? 0 : s < a.T ? s : a.T;
}
// New tokens of request b; tokens past the last request are those of one more, with nothing to see.
__device__ __forceinline__ int new_of(const AttendArgs& a, int b, int64_t q0) {
  const int64_t q1 = b < a.B ? start_of(a, b + 1) : a.T;
  return q1 > q0 ? (int)(q1 - q0) : 0;
}
__device__ __forceinline__ int context_of(const AttendArgs& a, int b) {
  const int c = b < a.B ? a.context[b] : 0;
  return c < 0 ? 0 : c < (1 << 30) ? c : 1 << 30;
}
__device__ __forceinline__ bool mine(const AttendArgs& a, int rows) { return rows >= a.rows_from && rows <= a.rows_upto; }

// Without parts: request b's tiles of R rows start at floor(starts[b] grp / R) + b, which leaves each
// request room for its last, partial one and can be searched without sums over requests.
template <int R>
__device__ __forceinline__ Work pick_tile(const AttendArgs& a, int64_t y) {
  const int lane = threadIdx.x & 63;
  Work t;
  int64_t tile;
  if (a.B < 64) {  // a lane a request (and one for the tokens after them): one round trip
    const int start = lane <= a.B ? (int)start_of(a, lane) : 0, ctx = lane <= a.B ? context_of(a, lane) : 0;
    const bool before = lane <= a.B && (int64_t)((uint64_t)((int64_t)start * a.grp) / R) + lane <= y;
    t.b = __popcll(__ballot(before)) - 1;
    t.q0 = __builtin_amdgcn_readlane(start, t.b);
    const int q1 = t.b < a.B ? __builtin_amdgcn_readlane(start, t.b + 1) : a.T;
    t.n = q1 > t.q0 ? q1 - (int)t.q0 : 0;
    t.ctx = __builtin_amdgcn_readlane(ctx, t.b);
  } else {
    int at = -1;
    for (int b0 = 0; b0 <= a.B; b0 += 64) {
      const int b = b0 + lane;
      const bool before = b <= a.B && (int64_t)((uint64_t)(start_of(a, b) * a.grp) / R) + b <= y;
      const int n = __popcll(__ballot(before));
      at += n;
      if (n < 64) break;
    }
    t.b = at;
    t.q0 = start_of(a, at);
    t.n = new_of(a, at, t.q0);
    t.ctx = context_of(a, at);
  }
  tile = y - ((int64_t)((uint64_t)(t.q0 * a.grp) / R) + t.b);
  const int64_t tiles = ((int64_t)t.n * a.grp + R - 1) / R;
  t.any = tile >= 0 && tile < tiles && mine(a, t.n * a.grp);
  t.row0 = (int)((tiles - 1 - tile) * R);  // the last rows see most: they start first
  t.part = 0;
  t.parts = 1;
  t.first = 0;
  return t;
}

// Inclusive sum over the wave, register lane moves only.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_from(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_from<0x111, 0xf>(v);  // row_shr:1
  v += dpp_from<0x112, 0xf>(v);
  v += dpp_from<0x114, 0xf>(v);
  v += dpp_from<0x118, 0xf>(v);
  v += dpp_from<0x142, 0xa>(v);  // row_bcast:15
  v += dpp_from<0x143, 0xc>(v);  // row_bcast:31
  return v;
}

// With parts: a tile whose tokens take W steps is cut into ceil(W / size) parts, size so that all
// requests' tiles and parts come to at most a.blocks blocks, which run at once, if the tiles alone
// do not pass that.  The parts of tiles that are cut come to no more in any case, so they have places
// of their own and tiles that are not cut need none: 34 MB hold the parts of prompts of heads of 128,
// where a place a block took 103 MB for a prompt of 4095 and more for longer ones.
// Every block does the sums over the requests itself: up to 63 requests each of its waves, a lane a
// request; more with all its threads, and LDS between the waves.
template <int R, int STEP, int THREADS>
__device__ __forceinline__ Work pick_part(const AttendArgs& a, int y, float* s_sum, Work* s_work) {
  constexpr int NW = THREADS / 64;
  const bool alone = a.B < 64;  // the wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int me = alone ? lane : threadIdx.x, each = alone ? 1 : a.B / THREADS + 1;  // of B + 1 requests
  const int b0 = me * each < a.B + 1 ? me * each : a.B + 1, b1 = b0 + each < a.B + 1 ? b0 + each : a.B + 1;
  int64_t q0 = 0;
  int n = 0, ctx = 0, tiles = 0, steps = 0;
  bool falls = false;
  auto look = [&](int b) {
    q0 = start_of(a, b);
    const int64_t q1 = b < a.B ? start_of(a, b + 1) : a.T;
    falls |= q1 < q0;
    n = q1 > q0 ? (int)(q1 - q0) : 0;
    const int rows = n * a.grp;
    tiles = mine(a, rows) ? (rows + R - 1) / R : 0;
    ctx = context_of(a, b);
    int span = ctx < a.reach ? ctx : a.reach;
    if (a.window > 0 && span > a.window + R) span = a.window + R;  // of one tile
    steps = (span + STEP - 1) / STEP;
  };
  auto total_of = [&](float v) {
    v = wave_sum_dpp(v);
    if (alone) return v;
    __syncthreads();
    if (lane == 0) s_sum[wave] = v;
    __syncthreads();
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) all += s_sum[w];
    return all;
  };
  auto parts_for = [&](float per_step) {
    if (steps <= a.whole) return 1;
    return (int)__builtin_ceilf((float)steps * per_step);
  };
  float sum = 0.f;
  for (int b = b0; b < b1; ++b) {
    look(b);
    sum += (float)tiles * (float)steps;
  }
  const float most = (float)a.blocks / (float)a.Hkv;
  const float total = total_of(falls ? __builtin_inff() : sum);
  if (total == __builtin_inff()) {  // starts that decrease: requests would share rows, and no bound here would hold
    Work t;
    t.any = false;
    return t;
  }
  float size = total * 1.00001f / most + 1.f;  // sums of rounded products: never too small
  if (size < (float)a.least) size = (float)a.least;
  int count, before, place;
#pragma unroll 1
  for (int round = 0;; ++round) {
    int cut = 0;  // blocks of tiles with several parts, of this thread's
    count = 0;
    for (int b = b0; b < b1; ++b) {
      if (each > 1) look(b);
      const int parts = parts_for(1.f / size);
      count += tiles * parts;
      cut += parts > 1 ? tiles * parts : 0;
    }
    if (round < 3) {
      const float all = total_of((float)count);
      if (all > most) {
        // what rounding up adds to total / size parts changes little with the size
        const float room = most - (all - total / size);
        size = room > 0.5f * total / size ? total * 1.001f / room : 2.f * size;
        continue;
      }
      round = 3;
    }
    // Blocks and places before this thread's, in one sum: both are below 2^15, at most 4096 tiles
    // (plan_grid) and a block more for each of 1024 parts, while starts do not decrease.
    const int both = count | cut << 16;
    int sum = wave_scan(both), all = __builtin_amdgcn_readlane(sum, 63);
    sum -= both;
    if (!alone) {
      __syncthreads();
      if (lane == 0) s_sum[wave] = __int_as_float(all);
      if (threadIdx.x == 0) s_work->any = false;
      __syncthreads();
      all = 0;
#pragma unroll 1
      for (int w = 0; w < NW; ++w) {
        const int other = __float_as_int(s_sum[w]);
        if (w < wave) sum += other;
        all += other;
      }
    }
    before = sum & 0xffff;
    place = sum >> 16;
    if ((float)(all >> 16) <= most) break;
    size *= 1.25f;  // no tile is cut at the latest where this passes its steps
  }
  const float per_step = 1.f / size;
  Work t;
  const bool found = y >= before && y < before + count;
  if (alone) {
    const uint64_t who = __ballot(found);
    if (!who) {
      t.any = false;
      return t;
    }
    const int from = __builtin_ctzll(who);
    t.b = from;
    t.q0 = (int64_t)__builtin_amdgcn_readlane((int)q0, from);  // below 2^31
    t.n = __builtin_amdgcn_readlane(n, from);
    t.ctx = __builtin_amdgcn_readlane(ctx, from);
    before = __builtin_amdgcn_readlane(before, from);
    place = __builtin_amdgcn_readlane(place, from);
    tiles = __builtin_amdgcn_readlane(tiles, from);
    t.parts = __builtin_amdgcn_readlane(parts_for(per_step), from);
    const int tile = (y - before) / t.parts;
    t.row0 = (tiles - 1 - tile) * R;
    t.part = y - before - tile * t.parts;
    t.first = place + tile * t.parts;
    t.any = true;
  } else {
    if (found) {
      for (int b = b0; b < b1; ++b) {
        if (each > 1) look(b);
        const int parts = parts_for(per_step);
        if (y < before + tiles * parts) {
          const int tile = (y - before) / parts;
          t.q0 = q0;
          t.b = b;
          t.n = n;
          t.ctx = ctx;
          t.row0 = (tiles - 1 - tile) * R;
          t.part = y - before - tile * parts;
          t.parts = parts;
          t.first = place + tile * parts;
          t.any = true;
          *s_work = t;
          break;
        }
        before += tiles * parts;
        if (parts > 1) place += tiles * parts;
      }
    }
    __syncthreads();
    t = *s_work;
  }
  return t;
}

template <int R, int STEP, int THREADS>
__device__ __forceinline__ Work pick_work(const AttendArgs& a, float* s_sum, Work* s_work) {
  const unsigned x = blockIdx.x, y = x / (unsigned)a.Hkv;  // heads side by side: each to its own XCD's cache
  Work t = a.blocks > 0 ? pick_part<R, STEP, THREADS>(a, (int)y, s_sum, s_work) : pick_tile<R>(a, y);
  t.hk = (int)(x - y * (unsigned)a.Hkv);
  t.q0 = __builtin_amdgcn_readfirstlane((int)t.q0);  // both below 2^31
  t.first = __builtin_amdgcn_readfirstlane((int)t.first);
  t.b = __builtin_amdgcn_readfirstlane(t.b);
  t.n = __builtin_amdgcn_readfirstlane(t.n);
  t.ctx = __builtin_amdgcn_readfirstlane(t.ctx);
  t.row0 = __builtin_amdgcn_readfirstlane(t.row0);
  t.part = __builtin_amdgcn_readfirstlane(t.part);
  t.parts = __builtin_amdgcn_readfirstlane(t.parts);
  return t;
}

// The lane's query row: KS pieces of 8 values, STRIDE apart, as operands.
template <class T, int KS, int STRIDE>
struct QueryRow {
  float v[KS][8];
  __device__ __forceinline__ void load(const T* q) {
#pragma unroll
    for (int k = 0; k < KS; ++k) load_values<T, 8>(q + STRIDE * k, v[k]);
  }
  // Returns what the row's scores have to be multiplied by; sums: this lane's part of its groups' sums.
  template <int G, class Frag>
  __device__ __forceinline__ float operands(float scale_log2, Frag (&qf)[KS][kQueryParts<T>], float (&sums)[G]) {
    int e2 = 0;
    if constexpr (__is_same(T, __bf16)) {
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(v[k][e]));
      top = STRIDE == 32 ? quad_max(top) : pair_max(top);
      e2 = top < __builtin_inff() ? __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] = __builtin_amdgcn_ldexpf(v[k][e], -e2);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) sums[g] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      parts_of(v[k], qf[k]);
      if constexpr (kCodes<T>)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[k * STRIDE / kKv4Group] += v[k][e];
    }
    // neither 0 nor infinite, either of which would make NaN of a score: hidden ones are -inf, others may be 0
    return __builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(scale_log2, e2), 0x1p-126f, 0x1.fffffep127f);
  }
};

// N dwords (1, 2 or a multiple of 4) of a block.
template <int N>
__device__ __forceinline__ void fetch(uint32_t* to, __amdgpu_buffer_rsrc_t r, int lane_at, int at) {
  if constexpr (N == 1) to[0] = __builtin_amdgcn_raw_buffer_load_b32(r, lane_at, at, 0);
  if constexpr (N == 2) {
    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, lane_at, at, 0);
    to[0] = v[0];
    to[1] = v[1];
  }
#pragma unroll
  for (int i = 0; i + 3 < N; i += 4) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, lane_at + 4 * i, at, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) to[i + e] = v[e];
  }
}

// Parts go past this chip part's own cache to where every block sees them (the sc1 bit of a store or
// load), so that no cache has to be written back or dropped for them.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t shared_at(void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, bytes, 0x00020000);
}
constexpr int kDevice = 16;
__device__ __forceinline__ void put4(__amdgpu_buffer_rsrc_t r, int at, f32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, at, 0, kDevice);
}
__device__ __forceinline__ f32x4 get4(__amdgpu_buffer_rsrc_t r, int at) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, kDevice));
}
__device__ __forceinline__ void put2(__amdgpu_buffer_rsrc_t r, int at, float2 v) {
  __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(v.x), __float_as_uint(v.y)}, r, at, 0, kDevice);
}
__device__ __forceinline__ float2 get2(__amdgpu_buffer_rsrc_t r, int at) {
  const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, kDevice);
  return {__uint_as_float(v[0]), __uint_as_float(v[1])};
}

// This block's part is stored: true in the block that is the last of its tile's.
__device__ __forceinline__ bool last_part(const AttendArgs& a, const Work& w, int* s_last) {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the thread's stores are where all see them
  __syncthreads();
  if (threadIdx.x == 0) {
    int* count = a.done + w.first * a.Hkv + w.hk;
    const int before = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before == w.parts - 1) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *s_last = before == w.parts - 1;
  }
  __syncthreads();
  return *s_last;
}

// ---- few rows --------------------------------------------------------------------------------
// Bound by the codes' bytes and by their unpacking: 176 operations of about 250 for 32 tokens of a head
// of 128, whatever the number of rows.
// Forms of the kernel.  kAhead: registers hold the next step's codes too, which hides a load's time
// where few waves run.  kLean: room for up to twice the waves where their number does that, in blocks
// of half the size, which share out ragged requests more evenly.  kDeep: the same in blocks of eight
// waves, which leave half the parts to join where long contexts of few requests are cut into dozens.
// Single tokens of ragged requests, 32 + 8 heads of 128, us of kAhead / kLean / kDeep:
//   few steps    bf16 1 of 32768 17.4 / 20.9 / 19.7, 16 up to 2048 13.1 / 15.7 / 16.6; fp16 1 of 32768 18.7 / 21.3
//   few tiles    bf16 2 up to 131072 50.8 / 54.5 / 50.6, 8 up to 16384 24.4 / 25.7 / 24.3; fp16 47.1 / 51.1, 28.4 / 28.4
//   neither      bf16 16 up to 8192 28.1 / 27.5 / 26.5, 64 up to 2000 36.0 / 27.5 / 25.8; fp16 46.9 / 28.7, 39.5 / 30.6
//   short tiles  bf16 40 up to 250 10.5 / 7.8, 64 up to 64 12.1 / 7.4, 60 of 5 tokens up to 34 18.1 / 10.4
enum { kAhead, kLean, kDeep };
constexpr bool few_wide(int kind, int D, int rt) { return D * rt >= (kind == 2 ? 256 : 512); }
constexpr int few_waves(int kind, int D, int rt, int form) {  // a SIMD, as the registers allow
  if (few_wide(kind, D, rt)) return 1;
  return form == kAhead ? 2 : D * rt <= 64 || (kind == 0 && D * rt <= 128) ? 4 : kind == 1 && D * rt <= 128 ? 3 : 2;
}
constexpr int few_block(int form) { return form == kLean ? 4 : 8; }  // waves of a block
constexpr int few_fill(int kind, int D, int rt, int form) {          // blocks that run at once
  return 1024 * few_waves(kind, D, rt, form) / few_block(form);
}
constexpr int few_form(int kind, int D, int rt, bool few_steps, bool few_tiles, bool short_tiles) {
  if (short_tiles || few_wide(kind, D, rt) || D == 256 || (kind == 1 && D * rt == 256)) return kLean;
  const int waves = few_waves(kind, D, rt, kLean);
  if (few_steps || waves == 2) return kAhead;
  return !few_tiles ? kLean : waves == 4 ? kDeep : kAhead;
}
constexpr bool few_used(int kind, int D, int rt, int form) {
  return form == kLean || form == few_form(kind, D, rt, true, true, false) || form == few_form(kind, D, rt, false, true, false);
}
// Whether registers hold two tiles of 16 rows.
constexpr bool few_pairs(int kind, int D) { return kind == 0 || D < 256; }
// Steps of a part at least, and steps that stay whole.  32 + 8 heads, us with parts and without: a token
// over 4000 12.1 and 24.6, over 2000 12.1 and 15.2, over 1000 11.3 and 10.3 (parts of 8 from 16 on: 11.7,
// 10.9 and 10.7, but 10.6 where 8.0 over 600, and 13.1 where 11.8 for 16 over 1000); 200 rows of tokens
// over 4000 39 and 98, over 1000 19.4 and 29.8 (parts of 2 from 4 on: 39.9 and 21.8, of 8 from 16 on: 39.1 and 30.8).
constexpr int kFewLeast = 16, kFewWhole = 32;
constexpr int kRowsLeast = 4, kRowsWhole = 8, kRowsFill = 512;

template <class T, int D, int RT, int FORM>
__global__ __launch_bounds__(64 * few_block(FORM), (few_waves(kKind<T>, D, RT, FORM))) void k_attend_few(
    const int* starts, const int* context, int tokens, int requests, int Hkv, int grp, int reach, int window, int blocks, AttendArgs a) {
  a.starts = starts, a.context = context, a.T = tokens, a.B = requests, a.Hkv = Hkv, a.grp = grp, a.reach = reach;
  a.window = window, a.blocks = blocks;
  constexpr int NW = few_block(FORM);
  constexpr bool AHEAD = FORM == kAhead;
  using O = Ops<T>;
  typedef typename O::KFrag KFrag;
  typedef typename O::VFrag VFrag;
  constexpr int G = D / kKv4Group, KS = D / 32, R = 16 * RT, W = 2 * G, NQ = kQueryParts<T>, NP = kWeightParts<T>;
  constexpr int KW = kCodes<T> ? 4 * G : G;  // dwords of key scales: the scores' four tokens, or the operand's own
  __shared__ float s_o[NW][16][D + 4];
  __shared__ float2 s_ml[NW][16];
  __shared__ float s_sum[NW];
  __shared__ Work s_work;
  __shared__ int s_last;
  const int lane = threadIdx.x & 63, n = lane & 15, qq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Work tile = pick_work<R, 32, 64 * NW>(a, s_sum, &s_work);
  if (!tile.any) return;
  const int hk = tile.hk, rows = tile.n * a.grp;
  const int past = tile.ctx - tile.n;  // position of the first new token
  const int r_last = tile.row0 + R - 1 < rows ? tile.row0 + R - 1 : rows - 1;
  const int pos_min = past + tile.row0 / a.grp, pos_max = past + r_last / a.grp;
  const Span span = span_of(pos_min, pos_max, a.window, a.reach, tile.b < a.B);
  const int lo = span.lo, hi = span.hi;

  // this block's steps of 32 tokens, of which the wave takes every NW-th
  const int first = lo >> 5, steps = ((hi + 31) >> 5) - first;
  const int s0 = first + (int)((int64_t)steps * tile.part / tile.parts);
  const int s1 = first + (int)((int64_t)steps * (tile.part + 1) / tile.parts);
  const int its = s1 - s0 > wave ? (s1 - s0 - wave + NW - 1) / NW : 0;
  const int* table = a.tables + (int64_t)(tile.b < a.B ? tile.b : 0) * a.ld_table;
  const Kv4Layout L(a.P, D);
  const int block_bytes = L.bytes();

  // lane l holds the page of the wave's step l / 2, tokens 16 (l & 1), of a run of 32 steps
  int ids = -1;
  uint64_t gone = 0;  // those that are no page
  auto load_ids = [&](int it0) {
    const int64_t t = (int64_t)(s0 + wave + NW * (it0 + (lane >> 1))) * 32 + 16 * (lane & 1);
    ids = it0 + (lane >> 1) < its && t < hi ? table[t >> a.shift] : -1;
  };
  load_ids(0);

  struct RawK {
    uint32_t k[2][KS], s[2][KW];
  };
  struct RawV {
    uint32_t v[2][W], s[2][G][4];
  };
  // Codes come through a descriptor of their (page, head) block, so that offsets are one lane
  // constant and one scalar; no page is a block of no bytes, which reads as zeros.
  const int k_lane = n * (D / 2) + qq * (KS * 4), ks_lane = (kCodes<T> ? 4 * qq : n) * (G * 4);
  const int v_lane = qq * (128 * G) + n * (W * 4), vs_lane = qq * (G * 16);
  auto block_of = [&](int at, int h) {
    const int id = __builtin_amdgcn_readlane(ids, (2 * at + h) & 63);
    const bool in = at < 32 && id >= 0 && id < a.pages;
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(a.cache) + ((int64_t)(in ? id : 0) * a.Hkv + hk) * block_bytes, 0, in ? block_bytes : 0, 0x00020000);
  };
  auto load_k = [&](int at, int step, RawK& r) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto block = block_of(at, h);
      const int tl = (step * 32 + 16 * h) & (a.P - 1);
      fetch<KS>(r.k[h], block, k_lane, tl * (D / 2));
      fetch<KW>(r.s[h], block, ks_lane, L.k_scales() + tl * (G * 4));
    }
  };
  auto load_v = [&](int at, int step, RawV& r) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto block = block_of(at, h);
      const int tl = (step * 32 + 16 * h) & (a.P - 1);
      fetch<W>(r.v[h], block, v_lane, L.v_codes() + tl * (32 * G));
      fetch<4 * G>(&r.s[h][0][0], block, vs_lane, L.v_scales() + tl * (G * 4));
    }
  };

  // queries: the lane's row, values d = 32 i + 8 qq + (0..7), under way while the pages arrive
  KFrag qf[RT][KS][NQ];
  float rs[RT], qs[RT][G];
  int pos[RT];
  QueryRow<T, KS, 32> raw_q[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int row = tile.row0 + rt * 16 + n;
    if (row >= rows) row = rows - 1;
    const int i = (int)((unsigned)row / (unsigned)a.grp), head = hk * a.grp + row - i * a.grp;
    pos[rt] = past + i;
    raw_q[rt].load(static_cast<const T*>(a.q) + (tile.q0 + i) * a.ldq_t + head * a.ldq_h + 8 * qq);
  }
  RawK rk[AHEAD ? 2 : 1];
  RawV rv[AHEAD ? 2 : 1];
  if (its > 0) {
    load_k(0, s0 + wave, rk[0]);
    load_v(0, s0 + wave, rv[0]);
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    rs[rt] = raw_q[rt].template operands<G>(a.scale_log2, qf[rt], qs[rt]);
    if constexpr (kCodes<T>)
#pragma unroll
      for (int g = 0; g < G; ++g) qs[rt][g] = quad_sum(qs[rt][g]);
  }

  f32x4 o[RT][G][4];
  float m[RT], l[RT], ol[RT][G];  // ol: the codes' sum of p lo, if it has one of its own
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -__builtin_inff();
    l[rt] = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      ol[rt][g] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[rt][g][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  auto step_of = [&](int step, int at, bool more, RawK& rk, RawV& rv, RawK& next_k, RawV& next_v) {
    const int ahead = more ? at + 1 : 32;  // past the run's end: no bytes
    if constexpr (AHEAD) {
      load_k(ahead, step + NW, next_k);
      load_v(ahead, step + NW, next_v);
      __builtin_amdgcn_sched_barrier(0);
    }
    const int t0 = step * 32;
    const int bad = (int)(gone >> (2 * at)) & 3;
    const bool edge = t0 + 31 > pos_min || t0 + 32 > hi || t0 < lo || (a.window > 0 && t0 <= pos_max - a.window) || bad;
    if (edge) {  // tokens that no row sees take no part whatever their page holds
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int t = t0 + 16 * h + 4 * qq + 2 * c;
          const bool ok = !(bad >> h & 1);
          const uint32_t keep = (ok && t >= lo && t < hi ? 0xffffu : 0u) | (ok && t + 1 >= lo && t + 1 < hi ? 0xffff0000u : 0u);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            rv.s[h][g][c] &= keep;
            rv.s[h][g][2 + c] &= keep;
          }
        }
    }
    float x[RT][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (kCodes<T>) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) x[rt][4 * h + e] = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          f32x4 sc[RT];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 2 * g; k < 2 * g + 2; ++k) {
            const KFrag kf = O::key(rk.k[h][k], 0);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int p = NQ - 1; p >= 0; --p) sc[rt] = mma(kf, qf[rt][k][p], sc[rt]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t sl = rk.s[h][r * G + g];
            const float s = f16_bits_to_f32((uint16_t)sl), z = f16_bits_to_f32((uint16_t)(sl >> 16));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              x[rt][4 * h + r] = __builtin_fmaf(s, sc[rt][r], __builtin_fmaf(z, qs[rt][g], x[rt][4 * h + r]));
          }
        }
      } else {
        f32x4 sc[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sc[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const KFrag kf = O::key(rk.k[h][k], rk.s[h][k / 2]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt] = mma(kf, qf[rt][k][0], sc[rt]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[rt][4 * h + r] = sc[rt][r];
      }
    }
    float p[RT][8];
    VFrag pf[RT][NP];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (edge) {
        const int last = pos[rt] < hi - 1 ? pos[rt] : hi - 1, upto = last - t0 - 4 * qq;
        const int from = a.window > 0 ? pos[rt] - a.window + 1 - t0 - 4 * qq : -(1 << 30);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = 16 * (e >> 2) + (e & 3);
          x[rt][e] = ((at > upto) | (at < from)) ? -__builtin_inff() : x[rt][e];
        }
        if (bad)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[rt][e] = bad >> (e >> 2) & 1 ? -__builtin_inff() : x[rt][e];
      }
      float top = x[rt][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = top_of(top, x[rt][e]);
      top = quad_max(top) * rs[rt];
      if (__any(top > m[rt] + kSlack)) {
        const float to = max_of(m[rt], top);
        const float f = to == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m[rt] - to);
        l[rt] *= f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if constexpr (kCodes<T> && !kFold<T>) ol[rt][g] *= f;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[rt][g][j] *= f;
        }
        m[rt] = to;
      }
      const float base = m[rt] == -__builtin_inff() ? 0.f : m[rt];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[rt][e] = weight_of<T>(x[rt][e], rs[rt], base);
        if constexpr (kCodes<T>) l[rt] += p[rt][e];
      }
      if constexpr (!kCodes<T>) {
        parts_of(p[rt], pf[rt]);
        l[rt] = add_weights(p[rt], pf[rt], l[rt]);
      }
    }
    if constexpr (!AHEAD) {  // registers of keys and scores are free: the next step's are under way from here
      __builtin_amdgcn_sched_barrier(0);
      load_k(ahead, step + NW, next_k);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      uint32_t u[4], s[4], z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // token pairs (0, 1), (2, 3) of both tiles' units
        u[i] = rv.v[i >> 1][2 * g + (i & 1)];
        s[i] = rv.s[i >> 1][g][i & 1];
        z[i] = rv.s[i >> 1][g][2 + (i & 1)];
      }
      if constexpr (kCodes<T>) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float w[8], low = kFold<T> ? 0.f : ol[rt][g];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int up = 16 * (e & 1);
            w[e] = p[rt][e] * f16_bits_to_f32((uint16_t)(s[e >> 1] >> up));
            low = __builtin_fmaf(p[rt][e], f16_bits_to_f32((uint16_t)(z[e >> 1] >> up)), low);
          }
          parts_of(w, pf[rt]);
          if constexpr (kFold<T>) {
            low = quad_sum(low);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[rt][g][j] += low;
          } else {
            ol[rt][g] = low;
          }
        }
      }
      auto product = [&](const VFrag& vf, int j) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int q = NP - 1; q >= 0; --q) o[rt][g][j] = mma(vf, pf[rt][q], o[rt][g][j]);
      };
      product(O::template val<0>(u, s, z), 0);
      product(O::template val<1>(u, s, z), 1);
      product(O::template val<2>(u, s, z), 2);
      product(O::template val<3>(u, s, z), 3);
    }
    if constexpr (!AHEAD) {
      __builtin_amdgcn_sched_barrier(0);
      load_v(ahead, step + NW, next_v);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  for (int it0 = 0; it0 < its; it0 += 32) {
    const int run = its - it0 < 32 ? its - it0 : 32;
    const int base = s0 + wave + NW * it0;
    if (it0 > 0) {
      load_ids(it0);
      load_k(0, base, rk[0]);
      load_v(0, base, rv[0]);
    }
    gone = __ballot(ids < 0 || ids >= a.pages);
    if constexpr (AHEAD) {
      for (int i = 0;; i += 2) {
        step_of(base + NW * i, i, i + 1 < run, rk[0], rv[0], rk[1], rv[1]);
        if (i + 1 >= run) break;
        step_of(base + NW * (i + 1), i + 1, i + 2 < run, rk[1], rv[1], rk[0], rv[0]);
        if (i + 2 >= run) break;
      }
    } else {
      for (int i = 0; i < run; ++i) step_of(base + NW * i, i, i + 1 < run, rk[0], rv[0], rk[0], rv[0]);
    }
  }

  // join the waves, 16 rows at a time
  constexpr int TPR = 64 * NW / 16, C = D / TPR;  // threads a row, values a thread
  const int live = rows - tile.row0 < R ? rows - tile.row0 : R;  // rows that exist
  auto part_row = [&](int part) { return (tile.first * a.Hkv + hk + (int64_t)part * a.Hkv) * R; };  // the part's row 0
  auto out_at = [&](int r) {
    const int row = tile.row0 + r, i = (int)((unsigned)row / (unsigned)a.grp);
    return static_cast<T*>(a.out) + ((tile.q0 + i) * ((int64_t)a.Hkv * a.grp) + hk * a.grp + row - i * a.grp) * D;
  };
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (rt * 16 >= live) break;
    const float sum = quad_sum(l[rt]);
    if (rt) __syncthreads();
    if (qq == 0) s_ml[wave][n] = {m[rt], sum};
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float add = kCodes<T> && !kFold<T> ? quad_sum(ol[rt][g]) : 0.f;
      if (rt * 16 + n >= live) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f32x4 w = {o[rt][g][0][r], o[rt][g][1][r], o[rt][g][2][r], o[rt][g][3][r]};
        if constexpr (kCodes<T> && !kFold<T>) w += add;
        *reinterpret_cast<f32x4*>(&s_o[wave][n][64 * g + 16 * qq + 4 * r]) = w;
      }
    }
    __syncthreads();
    const int r16 = threadIdx.x / TPR, d0 = (threadIdx.x % TPR) * C, r = rt * 16 + r16;
    if (r >= live) continue;
    float top = -__builtin_inff(), all = 0.f, v[C] = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) top = max_of(top, s_ml[w][r16].x);
    const float base = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 ml = s_ml[w][r16];
      const float f = __builtin_amdgcn_exp2f(ml.x - base);
      all = __builtin_fmaf(ml.y, f, all);
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = __builtin_fmaf(s_o[w][r16][d0 + c], f, v[c]);
    }
    if (tile.parts == 1) {
      const float inv = all == 0.f ? 0.f : 1.f / all;
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] *= inv;
      store_values<T, C>(out_at(r) + d0, v);
    } else {
      const int64_t at = part_row(tile.part);
      const auto po = shared_at(a.part_o + at * D, 4 * R * D);
#pragma unroll
      for (int c = 0; c + 3 < C; c += 4) put4(po, (r * D + d0 + c) * 4, f32x4{v[c], v[c + 1], v[c + 2], v[c + 3]});
      if constexpr (C == 2) put2(po, (r * D + d0) * 4, {v[0], v[1]});
      if (d0 == 0) put2(shared_at(a.part_ml + at, 8 * R), r * 8, {top, all});
    }
  }
  if (tile.parts == 1 || !last_part(a, tile, &s_last)) return;

  // In a tile's last block, join the parts: a wave takes sets of RI rows, four values a lane, and all
  // parts of a set if there are sets for every wave, else every `share`-th of them.
  constexpr int RI = 256 / D, LR = 64 / RI, BATCH = 64 / NW;  // rows of a set, lanes a row, parts read at once
  const int sets = (live + RI - 1) / RI, share = sets >= NW ? 1 : NW / sets, sub = wave % share;
  f32x4* joined = reinterpret_cast<f32x4*>(&s_o[0][0][0]);  // [share][sets][64]
  float2* joined_ml = reinterpret_cast<float2*>(joined + NW * 64);
  const int dl = (lane % LR) * 4;
  auto give = [&](int r, f32x4 v, float all) {
    if (r >= live) return;
    const float inv = all == 0.f ? 0.f : 1.f / all;
    const float w[4] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
    store_values<T, 4>(out_at(r) + dl, w);
  };
  for (int set = wave / share; set < sets; set += NW / share) {
    const int r = set * RI + lane / LR;
    float2 ml = {-__builtin_inff(), 0.f};
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int c0 = sub; c0 < tile.parts; c0 += BATCH * share) {
      float2 pm[BATCH];
      f32x4 po[BATCH];
#pragma unroll
      for (int c = 0; c < BATCH; ++c) {
        const int part = c0 + c * share;
        const bool in = part < tile.parts;  // no bytes otherwise
        const int64_t at = part_row(in ? part : 0);
        pm[c] = get2(shared_at(a.part_ml + at, in ? 8 * live : 0), r * 8);
        po[c] = get4(shared_at(a.part_o + at * D, in ? 4 * D * live : 0), (r * D + dl) * 4);
      }
      float to = ml.x;
#pragma unroll
      for (int c = 0; c < BATCH; ++c) {
        if (c0 + c * share >= tile.parts) pm[c].x = -__builtin_inff();
        to = max_of(to, pm[c].x);
      }
      const float base = to == -__builtin_inff() ? 0.f : to, f = __builtin_amdgcn_exp2f(ml.x - base);
      ml = {to, ml.y * f};
      acc *= f;
#pragma unroll
      for (int c = 0; c < BATCH; ++c) {
        const float g = __builtin_amdgcn_exp2f(pm[c].x - base);
        ml.y = __builtin_fmaf(pm[c].y, g, ml.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(po[c][e], g, acc[e]);
      }
    }
    if (share == 1) {
      give(r, acc, ml.y);
    } else {
      joined[(sub * sets + set) * 64 + lane] = acc;
      joined_ml[(sub * sets + set) * 64 + lane] = ml;
    }
  }
  if (share == 1) return;
  __syncthreads();
  if (wave < sets) {  // fewer than the waves
    float2 ml = {-__builtin_inff(), 0.f};
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int u = 0; u < share; ++u) ml.x = max_of(ml.x, joined_ml[(u * sets + wave) * 64 + lane].x);
    const float base = ml.x == -__builtin_inff() ? 0.f : ml.x;
    for (int u = 0; u < share; ++u) {
      const float2 pm = joined_ml[(u * sets + wave) * 64 + lane];
      const float g = __builtin_amdgcn_exp2f(pm.x - base);
      ml.y = __builtin_fmaf(pm.y, g, ml.y);
      acc += joined[(u * sets + wave) * 64 + lane] * g;
    }
    give(wave * RI + lane / LR, acc, ml.y);
  }
}

// ---- many rows -------------------------------------------------------------------------------
// Unpacking once a block of 128 rows costs a wave a quarter of what it costs alone; 32 rows a wave and
// two waves a SIMD, since a wave alone issues a vector operation only every 7 cycles (64 rows a wave,
// one a SIMD: 197 us on the prompt of 4095 where this takes 171).
// 64 tokens (32 of heads of 256) unpacked in LDS, each eight values along a product's sum in 16
// bytes, in the order in which v_mfma_f32_32x32x16 takes them:
//   keys   [token / 32][d / 16][d / 8 & 1][token & 31]
//   values [d' / 32][token / 16][h][d' & 31]: d' = 64 g + 16 j + m of value 64 g + 4 m + j, and the
//          tokens 16 s + 4 h + (0..3), 16 s + 8 + 4 h + (0..3), which is where the scores' result
//          leaves the weights: these never cross lanes.
template <class T, int D>
struct RowsTile {
  static constexpr int TT = D == 256 ? 32 : 64, U = TT / 32, G = D / kKv4Group;
  static constexpr int kChunks = TT * D / 8;  // of 16 bytes, for keys and for values
  typename Ops<T>::KFrag k[kChunks];
  typename Ops<T>::VFrag v[kChunks];
  float ks[kCodes<T> ? G : 1][kCodes<T> ? TT : 1], kl[kCodes<T> ? G : 1][kCodes<T> ? TT : 1];
  float vs[kCodes<T> ? G : 1][kCodes<T> ? TT : 1], vl[kCodes<T> ? G : 1][kCodes<T> ? TT : 1];
};

template <class T, int D>
__global__ __launch_bounds__(256, D == 256 || (kKind<T> == 2 && D == 128) ? 1 : 2) void k_attend_rows(
    const int* starts, const int* context, int tokens, int requests, int Hkv, int grp, int reach, int window, int blocks, AttendArgs a) {
  a.starts = starts, a.context = context, a.T = tokens, a.B = requests, a.Hkv = Hkv, a.grp = grp, a.reach = reach;
  a.window = window, a.blocks = blocks;
  using O = Ops<T>;
  typedef typename O::KFrag KFrag;
  typedef typename O::VFrag VFrag;
  typedef RowsTile<T, D> Tile;
  constexpr int G = D / kKv4Group, KS = D / 16, DT = D / 32, NQ = kQueryParts<T>, NP = kWeightParts<T>, TT = Tile::TT, U = Tile::U, R = 128;
  constexpr int UB = kCodes<T> ? 1 : U;       // halves of 32 tokens that share a softmax step (registers)
  constexpr int C = Tile::kChunks / 256;      // chunks of keys (and of values) a thread unpacks
  constexpr int KG = D == 64 ? 1 : 2;         // groups that a thread's dwords of keys belong to
  extern __shared__ __attribute__((aligned(16))) char s_mem[];
  Tile* s_tile = reinterpret_cast<Tile*>(s_mem);  // two
  __shared__ float s_sum[4];
  __shared__ Work s_work;
  __shared__ int s_last;
  const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Work tile = pick_work<R, TT, 256>(a, s_sum, &s_work);
  if (!tile.any) return;
  const int hk = tile.hk, rows = tile.n * a.grp;
  const int past = tile.ctx - tile.n;
  const int r_last = tile.row0 + R - 1 < rows ? tile.row0 + R - 1 : rows - 1;
  const Span span = span_of(past + tile.row0 / a.grp, past + r_last / a.grp, a.window, a.reach, tile.b < a.B);
  const int lo = span.lo, hi = span.hi;

  // the wave's 32 rows, and the positions between which they stand
  const int wrow = tile.row0 + 32 * wave;
  const bool busy = wrow < rows;
  const int wlast = wrow + 31 < rows ? wrow + 31 : rows - 1;
  const int pos_min = past + (busy ? wrow : wlast) / a.grp, pos_max = past + wlast / a.grp;
  const int row = wrow + n < rows ? wrow + n : rows - 1;
  const int qi = row / a.grp, head = hk * a.grp + row - qi * a.grp;
  const int pos = past + qi;
  KFrag qf[KS][NQ];
  float qs[G];
  QueryRow<T, KS, 16> raw_q;
  raw_q.load(static_cast<const T*>(a.q) + (tile.q0 + qi) * a.ldq_t + head * a.ldq_h + 8 * h);
  const float rs = raw_q.template operands<G>(a.scale_log2, qf, qs);
  if constexpr (kCodes<T>)
#pragma unroll
    for (int g = 0; g < G; ++g) qs[g] = pair_sum(qs[g]);

  const int first = lo / TT, steps = (hi + TT - 1) / TT - first;
  const int s0 = first + (int)((int64_t)steps * tile.part / tile.parts);
  const int s1 = first + (int)((int64_t)steps * (tile.part + 1) / tile.parts);
  const Kv4Layout L(a.P, D);
  const int block_bytes = L.bytes();
  const int* table = a.tables + (int64_t)(tile.b < a.B ? tile.b : 0) * a.ld_table;

  // ---- unpacking: a wave takes 16 tokens of a step (which one page holds)
  // keys: token kt, dwords qq D/32 + k0 .. + C - 1
  // values: units u0 and u0 + 2 of four tokens, words n16 of group vg; of heads of 64 half the nibbles
  const int n16 = lane & 15, qq = lane >> 4;
  const int sub = D == 256 ? wave & 1 : wave, kt = 16 * sub + n16, k0 = D == 256 ? 4 * (wave >> 1) : 0;
  const int u0 = qq & 1, vg = D == 64 ? 0 : (D == 256 ? 2 * (wave >> 1) : 0) + (qq >> 1);
  const int k_lane = n16 * (D / 2) + (qq * (D / 32) + k0) * 4, ks_lane = (n16 * G + k0 / 2) * 4;
  const int v_lane = (u0 * 16 + n16) * (8 * G) + vg * 8, vs_lane = (u0 * G + vg) * 16;
  struct Raw {
    uint32_t k[C], ks[KG], v[4], vs[2][4];
  };
  // lane l holds the page of tokens 16 l .. of a run of 1024 tokens
  constexpr int RUN = 1024 / TT, E = TT / 16;
  int ids = 0;
  uint64_t gone = 0;
  auto load = [&](int at, int step, Raw& r) {
    const int id = __builtin_amdgcn_readlane(ids, E * at + sub);
    const bool in = id >= 0 && id < a.pages;  // else a block of no bytes, which reads as zeros
    const auto block = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(a.cache) + ((int64_t)(in ? id : 0) * a.Hkv + hk) * block_bytes, 0, in ? block_bytes : 0, 0x00020000);
    const int tl = (step * TT + 16 * sub) & (a.P - 1);
    fetch<C>(r.k, block, k_lane, tl * (D / 2));
    fetch<KG>(r.ks, block, ks_lane, L.k_scales() + tl * (G * 4));
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      fetch<2>(r.v + 2 * x, block, v_lane, L.v_codes() + tl * (32 * G) + x * (256 * G));
      fetch<4>(r.vs[x], block, vs_lane, L.v_scales() + tl * (G * 4) + x * (32 * G));
    }
  };
  auto unpack = [&](int at, int step, Raw& r, Tile& t) {
    // tokens that no row sees take no part whatever their page holds
    const int t0 = step * TT;
    const int bad = (int)(gone >> (E * at)) & ((1 << E) - 1);
    if (t0 < lo || t0 + TT > hi || bad) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int tok = t0 + 16 * sub + 4 * (u0 + 2 * x) + 2 * c;
          const bool ok = !(bad >> sub & 1);
          const uint32_t keep = (ok && tok >= lo && tok < hi ? 0xffffu : 0u) | (ok && tok + 1 >= lo && tok + 1 < hi ? 0xffff0000u : 0u);
          r.vs[x][c] &= keep;
          r.vs[x][2 + c] &= keep;
        }
    }
    KFrag* kd = t.k + ((kt >> 5) * KS) * 64 + (kt & 31) + (qq & 1) * 32;
#pragma unroll
    for (int c = 0; c < C; ++c) kd[(2 * (k0 + c) + (qq >> 1)) * 64] = O::key(r.k[c], r.ks[c / 2]);
    const uint32_t s[4] = {r.vs[0][0], r.vs[0][1], r.vs[1][0], r.vs[1][1]};
    const uint32_t z[4] = {r.vs[0][2], r.vs[0][3], r.vs[1][2], r.vs[1][3]};
    VFrag* vd = t.v + (2 * vg * (TT / 16) + sub) * 64 + u0 * 32 + n16;
    if constexpr (D == 64) {  // nibbles 2 (qq >> 1) and the next, moved to the place of 0 and 1
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = r.v[i] >> (16 * (qq >> 1));
      vd += (qq >> 1) * (TT / 16) * 64;
      vd[0] = O::template val<0>(u, s, z);
      vd[16] = O::template val<1>(u, s, z);
    } else {
      vd[0] = O::template val<0>(r.v, s, z);
      vd[16] = O::template val<1>(r.v, s, z);
      vd[(TT / 16) * 64] = O::template val<2>(r.v, s, z);
      vd[(TT / 16) * 64 + 16] = O::template val<3>(r.v, s, z);
    }
    if constexpr (kCodes<T>) {
      if (qq == 0) {
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          t.ks[k0 / 2 + g][kt] = f16_bits_to_f32((uint16_t)r.ks[g]);
          t.kl[k0 / 2 + g][kt] = f16_bits_to_f32((uint16_t)(r.ks[g] >> 16));
        }
      }
      if (n16 == 0) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            t.vs[vg][16 * sub + 4 * (u0 + 2 * x) + e] = f16_bits_to_f32((uint16_t)(r.vs[x][e >> 1] >> (16 * (e & 1))));
            t.vl[vg][16 * sub + 4 * (u0 + 2 * x) + e] = f16_bits_to_f32((uint16_t)(r.vs[x][2 + (e >> 1)] >> (16 * (e & 1))));
          }
      }
    }
  };

  f32x16 o[DT];
  float m = -__builtin_inff(), l = 0.f, ol[G];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
#pragma unroll
  for (int g = 0; g < G; ++g) ol[g] = 0.f;

  auto compute = [&](int at, int step, const Tile& t) {
    const int t0 = step * TT;
    const int bad = (int)(gone >> (E * at)) & ((1 << E) - 1);
    if (!busy || t0 > pos_max || (a.window > 0 && t0 + TT <= pos_min - a.window + 1)) return;  // nothing of it is seen
    const bool edge = t0 + TT - 1 > pos_min || t0 + TT > hi || (a.window > 0 && t0 <= pos_max - a.window) || bad;
#pragma unroll
    for (int h0 = 0; h0 < U; h0 += UB) {
      f32x16 x[UB];
      if constexpr (kCodes<T>) {
        x[0] = f32x16{};
#pragma unroll
        for (int g = 0; g < G; ++g) {
          KFrag kf[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) kf[k] = t.k[(h0 * KS + 4 * g + k) * 64 + lane];
          __builtin_amdgcn_sched_barrier(0);
          f32x16 sc = {};
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int p = NQ - 1; p >= 0; --p) sc = mma(kf[k], qf[4 * g + k][p], sc);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 s4 = *reinterpret_cast<const f32x4*>(&t.ks[g][32 * h0 + 8 * q + 4 * h]);
            const f32x4 l4 = *reinterpret_cast<const f32x4*>(&t.kl[g][32 * h0 + 8 * q + 4 * h]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[0][4 * q + e] = __builtin_fmaf(s4[e], sc[4 * q + e], __builtin_fmaf(l4[e], qs[g], x[0][4 * q + e]));
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        // every operand is on its way before the first product waits for one
        KFrag kf[UB][KS];
#pragma unroll
        for (int u = 0; u < UB; ++u)
#pragma unroll
          for (int k = 0; k < KS; ++k) kf[u][k] = t.k[((h0 + u) * KS + k) * 64 + lane];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < UB; ++u) {
          x[u] = f32x16{};
#pragma unroll
          for (int k = 0; k < KS; ++k) x[u] = mma(kf[u][k], qf[k][0], x[u]);
        }
      }
      constexpr int VB = kCodes<T> ? 1 : 2;  // sets of operands that registers have room for
      VFrag vf[VB][DT];
      auto load_values_of = [&](int i, VFrag (&f)[DT]) {  // tokens 16 i .. of the half (or halves)
#pragma unroll
        for (int d = 0; d < DT; ++d) f[d] = t.v[(d * (TT / 16) + 2 * h0 + i) * 64 + lane];
      };
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (!kCodes<T>) load_values_of(0, vf[0]);
      __builtin_amdgcn_sched_barrier(0);
      if (edge) {  // the row sees tokens from + 4 h + t0 .. upto + 4 h + t0
        const int last = pos < hi - 1 ? pos : hi - 1, upto = last - t0 - 4 * h - 32 * h0;
        const int from = a.window > 0 ? pos - a.window + 1 - t0 - 4 * h - 32 * h0 : -(1 << 30);
#pragma unroll
        for (int u = 0; u < UB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int at = 32 * u + 8 * (i >> 2) + (i & 3);
            const bool hide = (at > upto) | (at < from) | ((bad >> (2 * (h0 + u) + (i >> 3)) & 1) != 0);
            x[u][i] = hide ? -__builtin_inff() : x[u][i];
          }
      }
      float top = x[0][0];
#pragma unroll
      for (int u = 0; u < UB; ++u)
#pragma unroll
        for (int i = u ? 0 : 1; i < 16; ++i) top = top_of(top, x[u][i]);
      top = pair_max(top) * rs;
      if (__any(top > m + kSlack)) {
        const float to = max_of(m, top);
        const float f = to == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - to);
        l *= f;
#pragma unroll
        for (int g = 0; g < G; ++g)
          if constexpr (!kFold<T>) ol[g] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
        m = to;
      }
      const float base = m == -__builtin_inff() ? 0.f : m;
      if constexpr (kFold<T>)
#pragma unroll
        for (int g = 0; g < G; ++g) ol[g] = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * UB; ++i) {
        if (VB == 2 && i + 1 < 2 * UB) load_values_of(i + 1, vf[(i + 1) % VB]);
        if (kCodes<T>) load_values_of(i, vf[0]);
        const int u = i >> 1, s = i & 1;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = weight_of<T>(x[u][8 * s + e], rs, base);
          if constexpr (kCodes<T>) l += p[e];
        }
        VFrag pf[NP];
        if constexpr (!kCodes<T>) {
          parts_of(p, pf);
          l = add_weights(p, pf, l);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if constexpr (kCodes<T>) {
            float w[8];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const f32x4 s4 = *reinterpret_cast<const f32x4*>(&t.vs[g][32 * (h0 + u) + 16 * s + 8 * q + 4 * h]);
              const f32x4 l4 = *reinterpret_cast<const f32x4*>(&t.vl[g][32 * (h0 + u) + 16 * s + 8 * q + 4 * h]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                w[4 * q + e] = p[4 * q + e] * s4[e];
                ol[g] = __builtin_fmaf(p[4 * q + e], l4[e], ol[g]);
              }
            }
            parts_of(w, pf);
          }
#pragma unroll
          for (int d = 2 * g; d < 2 * g + 2; ++d)
#pragma unroll
            for (int q = NP - 1; q >= 0; --q) o[d] = mma(vf[i % VB][d], pf[q], o[d]);
        }
      }
      if constexpr (kFold<T>)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float low = pair_sum(ol[g]);
#pragma unroll
          for (int d = 2 * g; d < 2 * g + 2; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] += low;
        }
    }
  };

  for (int r0 = s0; r0 < s1; r0 += RUN) {
    const int run = s1 - r0 < RUN ? s1 - r0 : RUN;
    {
      const int64_t t = (int64_t)r0 * TT + 16 * lane;
      const bool used = lane < run * E && t < hi;
      ids = used ? table[t >> a.shift] : -1;
      const bool bad = ids < 0 || ids >= a.pages;
      gone = __ballot(bad);
    }
    Raw raw;
    load(0, r0, raw);
    unpack(0, r0, raw, s_tile[0]);
    load(run > 1 ? 1 : 0, run > 1 ? r0 + 1 : r0, raw);
    __syncthreads();
    for (int i = 0; i < run; ++i) {
      // the next step's tile is written while this one is read, and the loads of the one after are under way
      if (i + 1 < run) unpack(i + 1, r0 + i + 1, raw, s_tile[(i + 1) & 1]);
      const int ahead = i + 2 < run ? i + 2 : run - 1;
      load(ahead, r0 + ahead, raw);
      compute(i, r0 + i, s_tile[i & 1]);
      __syncthreads();
    }
  }

  // a wave has its rows to itself: parts are stored as the registers lie
  l = pair_sum(l);
  if constexpr (kCodes<T> && !kFold<T>)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float add = pair_sum(ol[g]);
#pragma unroll
      for (int d = 2 * g; d < 2 * g + 2; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] += add;
    }
  if (tile.parts > 1) {
    const int64_t at0 = tile.first * a.Hkv + hk;
    auto part_at = [&](int part) { return (at0 + (int64_t)part * a.Hkv) * 4 + wave; };  // of waves
    if (busy) {
      const int64_t at = part_at(tile.part);
      const auto po = shared_at(a.part_o + at * (32 * D), 128 * D);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          put4(po, ((d * 4 + i) * 64 + lane) * 16, f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]});
      if (h == 0) put2(shared_at(a.part_ml + at * 32, 256), n * 8, {m, l});
    }
    if (!last_part(a, tile, &s_last)) return;
    if (!busy) return;
    m = -__builtin_inff();
    for (int c = 0; c < tile.parts; ++c) m = max_of(m, get2(shared_at(a.part_ml + part_at(c) * 32, 256), n * 8).x);
    const float base = m == -__builtin_inff() ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
#pragma unroll 1
    for (int c = 0; c < tile.parts; ++c) {
      const int64_t at = part_at(c);
      const float2 ml = get2(shared_at(a.part_ml + at * 32, 256), n * 8);
      const auto po = shared_at(a.part_o + at * (32 * D), 128 * D);
      f32x4 v[DT * 4];
#pragma unroll
      for (int i = 0; i < DT * 4; ++i) v[i] = get4(po, (i * 64 + lane) * 16);
      const float f = __builtin_amdgcn_exp2f(ml.x - base);
      l = __builtin_fmaf(ml.y, f, l);
#pragma unroll
      for (int i = 0; i < DT * 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i / 4][4 * (i % 4) + e] = __builtin_fmaf(v[i][e], f, o[i / 4][4 * (i % 4) + e]);
    }
  }
  int mine = wrow + n;
  asm volatile("" : "+v"(mine));  // its place is computed again, not held through the loop
  if (!busy || mine >= rows) return;
  const int token = (int)((unsigned)mine / (unsigned)a.grp);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(a.out) + ((tile.q0 + token) * ((int64_t)a.Hkv * a.grp) + hk * a.grp + mine - token * a.grp) * D;
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int q = 0; q < 2; ++q) {  // words m = 8 q + 4 h + (0..3): 16 values side by side
      float v[16];
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * w + j] = o[2 * g + (j >> 1)][8 * (j & 1) + 4 * q + w] * inv;
      store_values<T, 16>(out + 64 * g + 4 * (8 * q + 4 * h), v);
    }
}

// ---- launch -------------------------------------------------------------------------------
constexpr int kFewRows = 32;
constexpr int kSyncWords = 8192;  // of the workspace's start, one a place: at most 1024 blocks run at once

struct Plan {
  int rt;           // 16-row tiles of k_attend_few, 0: not used
  bool rows;        // k_attend_rows runs
  int form;         // of k_attend_few
  int64_t grid_few, grid_rows;
  int fill_few, fill_rows;  // blocks that parts fill, 0: no parts
};

// Blocks of one kernel, R rows a tile: a block a tile and head, and with parts `fill` more, if by the
// caller's bounds some tile has more steps than stay whole.  Tiles in thousands fill the chip without
// parts, and the sums over many requests would cost every block more.  upto: rows of the requests that
// are this kernel's, whose tiles then are bounded by the requests (without parts a tile's block is
// found by the tokens before it, so those of every request count).
void plan_grid(int64_t T, int64_t B, int Hkv, int grp, int R, int64_t rows, int64_t upto, int64_t steps, int whole, int least,
               int most, int64_t& grid, int& fill) {
  const int64_t all = T * grp / R + B + 1, own = (B + 1) * cdiv(upto, R);
  const int64_t tiles = (own < all ? own : all) * Hkv;
  const int64_t likely = cdiv(rows, R) * B * Hkv * cdiv(steps, least);
  fill = steps > whole && tiles <= 4 * most && B < 1024 ? (int)(likely < most ? likely : most) : 0;
  if (fill < Hkv) fill = 0;  // not a part a head
  grid = fill ? tiles + fill + Hkv : all * Hkv;
}

Plan plan_of(int kind, int D, int64_t T, int64_t B, int Hkv, int grp, int64_t max_query, int64_t max_context, int64_t window) {
  Plan p{};
  const int64_t rows = (max_query < T ? max_query : T) * grp;  // of a request
  int64_t span = max_context;
  if (window > 0 && span > window + 128) span = window + 128;
  p.rt = rows > 16 && few_pairs(kind, D) ? 2 : 1;
  p.rows = rows > kFewRows && !(kind == 2 && D == 256);  // three parts of 32 such queries pass the registers
  // few steps: 256 blocks of 8 waves, four each; few tiles: each cut into eight parts or more; short
  // ones: more than run at once in blocks of eight waves, of which each would have a step at most
  const int64_t steps = cdiv(span, 32), tiles = (T * grp / (16 * p.rt) + B + 1) * Hkv;
  p.form = few_form(kind, D, p.rt, B * Hkv * steps <= 8192, B * Hkv <= 64, tiles > 256 && steps <= 8);
  const int most = few_fill(kind, D, p.rt, p.form);
  // The tiles of a few requests' few rows find room beside the others, unless their contexts are long:
  // a block of 128 rows reads a context no faster for 4 of them.  32 + 8 heads, one launch and two: 15
  // tokens over 2000 beside a prompt of 500 31 and 42 us, over 4000 45 and 48, over 8000 75 and 62, over
  // 16000 140 and 83; 31 over 2000 (256 heads) 58 and 49; 3 over 131072 beside 4000 1682 and 277; and where
  // no request has few rows, 4 chunks of 512 over 4000 153 and 160, over 16000 574 and 574.
  if (p.rows && B * Hkv <= 128 && (B == 1 || span <= 4096)) p.rt = 0;
  if (p.rt)
    plan_grid(T, B, Hkv, grp, 16 * p.rt, rows < kFewRows ? rows : kFewRows, p.rows ? kFewRows : INT32_MAX, cdiv(span, 32) + 1,
              kFewWhole, kFewLeast, most, p.grid_few, p.fill_few);
  if (p.rows)
    plan_grid(T, B, Hkv, grp, 128, rows, INT32_MAX, cdiv(span, D == 256 ? 32 : 64) + 1, kRowsWhole, kRowsLeast, kRowsFill, p.grid_rows,
              p.fill_rows);
  return p;
}

size_t space_of(const Plan& p, int D) {  // the kernels' parts, which run one after the other
  const size_t few = p.rt ? (size_t)p.fill_few * 16 * p.rt : 0;
  const size_t rows = p.rows ? (size_t)p.fill_rows * 128 : 0;
  const size_t most = few > rows ? few : rows;
  return most ? (kSyncWords + most * (D + 2)) * sizeof(float) : 0;
}

template <class T, int D>
int launch_attend(AttendArgs a, const Plan& p, hipStream_t s) {
  constexpr bool wide = kKind<T> == 2 && D == 256;
  if constexpr (!wide)
    if (p.rows) {
      a.part_ml = reinterpret_cast<float2*>(a.part_o + (int64_t)p.fill_rows * 128 * D);
      a.rows_from = p.rt ? kFewRows + 1 : 0;
      a.rows_upto = 0x7fffffff;
      a.blocks = p.fill_rows;
      a.least = kRowsLeast;
      a.whole = kRowsWhole;
      const size_t lds = 2 * sizeof(RowsTile<T, D>);
      static std::atomic<uint64_t> allowed{0};  // a bit a device
      int device = 0;
      int status = hip_check(hipGetDevice(&device), "k_attend_rows device");
      if (status != QS_OK) return status;
      if (!(allowed.load(std::memory_order_relaxed) >> (device & 63) & 1)) {
        status = hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_attend_rows<T, D>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds),
                           "k_attend_rows shared memory");
        if (status != QS_OK) return status;
        allowed.fetch_or(uint64_t(1) << (device & 63), std::memory_order_relaxed);
      }
      hipLaunchKernelGGL((k_attend_rows<T, D>), dim3((unsigned)p.grid_rows), dim3(256), lds, s, a.starts, a.context, a.T,
                       a.B, a.Hkv, a.grp, a.reach, a.window, a.blocks, a);
    }
  if (p.rt) {
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (int64_t)p.fill_few * 16 * p.rt * D);
    a.rows_from = 0;
    a.rows_upto = p.rows ? kFewRows : 0x7fffffff;
    a.blocks = p.fill_few;
    a.least = kFewLeast;
    a.whole = kFewWhole;
    auto go = [&](auto rt, auto form) {
      constexpr int RT = decltype(rt)::value, FORM = decltype(form)::value;
      if constexpr (few_used(kKind<T>, D, RT, FORM))
        hipLaunchKernelGGL((k_attend_few<T, D, RT, FORM>), dim3((unsigned)p.grid_few), dim3(64 * few_block(FORM)), 0, s, a.starts,
                           a.context, a.T, a.B, a.Hkv, a.grp, a.reach, a.window, a.blocks, a);
    };
    auto go_rows = [&](auto rt) {
      if (p.form == kAhead)
        go(rt, std::integral_constant<int, kAhead>{});
      else if (p.form == kLean)
        go(rt, std::integral_constant<int, kLean>{});
      else
        go(rt, std::integral_constant<int, kDeep>{});
    };
    if constexpr (few_pairs(kKind<T>, D)) {
      if (p.rt == 1)
        go_rows(std::integral_constant<int, 1>{});
      else
        go_rows(std::integral_constant<int, 2>{});
    } else {
      go_rows(std::integral_constant<int, 1>{});
    }
  }
  return hip_check(hipGetLastError(), "k_attend launch");
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
  if (B > (1 << 20) || Hkv > 65535 || T * Hq >= (int64_t(1) << 31) || (T * Hq / 16 + (B + 2) * Hkv) >= (int64_t(1) << 31))
    return fail(QS_ERR_LIMIT, "kv4_attend: over 2^20 requests, 65535 heads or 2^31 query rows or blocks");
  return QS_OK;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" size_t qs_kv4_attend_workspace_bytes(int64_t T, int64_t B, int Hkv, int Hq, int D, int64_t page_size,
                                                int64_t max_query, int64_t max_context, int64_t window) {
  if (check_sizes(T, B, Hkv, Hq, D, page_size) != QS_OK) return 0;
  size_t most = 0;
  for (int kind = 0; kind < 3; ++kind) {
    const size_t bytes = space_of(plan_of(kind, D, T, B, Hkv, Hq / Hkv, max_query, max_context, window), D);
    most = bytes > most ? bytes : most;
  }
  return most;
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
  const Plan p = plan_of(dtype == QS_F32 ? 2 : dtype == QS_F16 ? 1 : 0, D, T, B, Hkv, grp, max_query, max_context, window);
  if ((p.rt && p.grid_few > most_blocks(64 * few_block(p.form))) || (p.rows && p.grid_rows > most_blocks(256)))
    return fail(QS_ERR_LIMIT, "kv4_attend: %lld query rows need more threads than the 2^32 of a grid", (long long)(T * Hq));
  const size_t need = space_of(p, D);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(QS_ERR_INVALID, "kv4_attend: workspace of qs_kv4_attend_workspace_bytes() bytes, 16-byte aligned");
  AttendArgs a{};
  a.q = q;
  a.cache = cache;
  a.tables = tables;
  a.starts = starts;
  a.context = context;
  a.out = out;
  a.done = static_cast<int*>(workspace);
  a.part_o = static_cast<float*>(workspace) + kSyncWords;
  a.ldq_t = ldq_t;
  a.ldq_h = ldq_h;
  a.ld_table = ld_table;
  a.T = (int)T;
  a.pages = (int)pages;
  a.P = (int)page_size;
  while ((int64_t(1) << a.shift) < page_size) ++a.shift;
  a.reach = (int)(width << a.shift < (1 << 30) ? width << a.shift : 1 << 30);
  a.Hkv = Hkv;
  a.grp = grp;
  a.B = (int)B;
  a.window = (int)(window < (1 << 30) ? window : 1 << 30);
  a.scale_log2 = scale * 1.44269504088896340736f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == QS_F32) return launch_attend_d<float>(a, p, D, s);
  if (dtype == QS_BF16) return launch_attend_d<__bf16>(a, p, D, s);
  if (dtype == QS_F16) return launch_attend_d<_Float16>(a, p, D, s);
  return fail(QS_ERR_INVALID, "kv4_attend: dtype must be F32, BF16 or F16");
}
