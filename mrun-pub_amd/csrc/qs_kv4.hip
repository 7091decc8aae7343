// The paged 4-bit KV cache: new tokens in, values out (gfx950).
//
//   k_kv4_append : a block per token turns its queries and keys by the token's position (angles
//                  once, through LDS), rounds them to the activation type, and codes keys and
//                  values: 16 lanes a group of 64 values, 4 values a lane, minimum and maximum
//                  by register lane moves.
//   k_kv4_read   : what the cache holds for given slots, 8 values a thread.
//
// A group's lo = fp16(min), s = fp16((max - min) / 15) and code = clamp(rint((x - lo) / s), 0, 15);
// its value is code * s + lo, exact in fp32 but for that sum's rounding.  NaN is coded as 0 and
// values are held to +-60000, so the cache itself never holds what is not finite.
//
// A block a token and the first loads under way during the angles: 4099 tokens of 32 + 16 heads of 128
// take 24.4 us (88 MB: 3.6 TB/s, the vector unit busy for 83%) and 7.4 us to read back; 13 tokens of
// 12 + 4 heads 4.5 and 2.3 us, latency.  Queries go 16 bytes an item, keys and values four a lane:
// eight (half the reductions) took 25.8 us, for their registers.
#include "qs_kv4.h"
#include "qs_rotary.h"
#include "qs_values.h"

namespace qs {
namespace {

struct AppendArgs {
  const void* k;
  const void* v;
  const void* q;
  void* q_out;
  const int64_t* slots;
  const int* pos;
  const double* freq;
  uint8_t* cache;
  int64_t ldk_t, ldk_h, ldv_t, ldv_h, ldq_t, ldq_h;
  int64_t slots_all;  // pages * P
  int P, D, Hkv, Hq, rot, interleaved, wide;  // wide: 16 bytes of queries an item
  double mag;
};

// Maximum over the 16 lanes of a row, in every lane of it.
__device__ __forceinline__ float row_max(float v) {
  v = dpp_max<0xB1, 0xf>(v);   // quad_perm [1,0,3,2]
  v = dpp_max<0x4E, 0xf>(v);   // quad_perm [2,3,0,1]
  v = dpp_max<0x141, 0xf>(v);  // row_half_mirror
  return dpp_max<0x140, 0xf>(v);  // row_mirror
}

// Codes of the lane's four values of the row's group: code e at bits 4 e.
__device__ __forceinline__ uint32_t code4(const float (&x)[4], _Float16& s16, _Float16& lo16) {
  float v[4], hi = -kKv4Max, ng = -kKv4Max;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -kKv4Max), kKv4Max) : 0.f;
    hi = fmaxf(hi, v[e]);
    ng = fmaxf(ng, -v[e]);
  }
  hi = row_max(hi);
  const float low = -row_max(ng);
  lo16 = static_cast<_Float16>(low);
  s16 = static_cast<_Float16>((hi - low) / 15.f);
  const float lo = static_cast<float>(lo16), s = static_cast<float>(s16);
  const float r = s > 0.f ? 1.f / s : 0.f;
  uint32_t c = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // the corrected quotient is the correctly rounded (x - lo) / s: r is a correctly rounded
    // reciprocal and nothing leaves the normal range (s >= 2^-24)
    const float q = rintf(quot_markstein(v[e] - lo, s, r));
    c |= (uint32_t)(int)fminf(fmaxf(q, 0.f), 15.f) << (4 * e);
  }
  return s > 0.f ? c : 0u;
}

// Four values of a head from d on, and with the halves' layout their partners.
template <class T>
struct Quad {
  float v[4], o[4];
  __device__ __forceinline__ void load(const T* x, int d, int rot, int interleaved) {
    load_values<T, 4>(x + d, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = 0.f;
    if (d < rot && !interleaved) load_values<T, 4>(x + (d < rot / 2 ? d + rot / 2 : d - rot / 2), o);
  }
  __device__ __forceinline__ void turn(int d, int rot, int interleaved, const float2* cs) {
    if (d >= rot) return;
    // partners and factors by selection: the interleaved layout's partner is the value next to it
    const bool low = d < rot / 2;
    const float2* w = cs + (interleaved ? d / 2 : low ? d : d - rot / 2);
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = w[interleaved ? e / 2 : e];
      const float other = interleaved ? v[e ^ 1] : o[e];
      const bool first = interleaved ? !(e & 1) : low;
      r[e] = first ? v[e] * f.x - other * f.y : v[e] * f.x + other * f.y;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = r[e];
  }
};

template <class T>
__global__ __launch_bounds__(256) void k_kv4_append(AppendArgs a) {
  using Item = TurnItem<T>;
  __shared__ float2 cs[128];
  const int64_t t = blockIdx.x;
  const Kv4Layout L(a.P, a.D);
  const int64_t slot = a.slots[t];
  const T* q = static_cast<const T*>(a.q) + t * a.ldq_t;
  T* qo = static_cast<T*>(a.q_out) + t * a.Hq * a.D;
  // queries: items of 16 bytes, or of four values
  const int turned = a.wide ? Item::turned(a.rot, a.interleaved) : 0;
  const int per_head = a.wide ? turned + (a.D - a.rot) / Item::V : a.D / 4;
  const int items = a.Hq * per_head;
  // keys, then values: 16 lanes a (head, group); a whole row of lanes is in or out
  const int groups = a.Hkv * L.G, m = threadIdx.x & 15;
  auto group_of = [&](int i, int& h, int& d) {
    const int hg = i < groups ? i : i - groups;
    h = hg / L.G;
    d = (hg - h * L.G) * kKv4Group + 4 * m;
  };
  auto load_quad = [&](int i, int h, int d, Quad<T>& x) {
    if (i < groups)
      x.load(static_cast<const T*>(a.k) + t * a.ldk_t + h * a.ldk_h, d, a.rot, a.interleaved);
    else
      load_values<T, 4>(static_cast<const T*>(a.v) + t * a.ldv_t + h * a.ldv_h + d, x.v);
  };
  // the first of each is under way while the angles are computed
  Item item;
  Quad<T> quad;
  int h, d, qh = 0;
  const bool wide = a.wide;
  if (wide && threadIdx.x < items) {
    qh = threadIdx.x / per_head;
    item.load(q + qh * a.ldq_h, threadIdx.x - qh * per_head, turned, a.rot, a.interleaved);
  }
  const bool in = slot >= 0 && slot < a.slots_all;
  int i = threadIdx.x >> 4;
  group_of(i, h, d);
  if (in && i < 2 * groups) load_quad(i, h, d, quad);
  if (a.rot) {
    for (int j = threadIdx.x; j < a.rot / 2; j += 256) cs[j] = rotary_cos_sin(a.pos[t], a.freq[j], a.mag);
    __syncthreads();
  }
  if (wide) {
    for (int j = threadIdx.x; j < items; j += 256) {
      if (j >= 256) {
        qh = j / per_head;
        item.load(q + qh * a.ldq_h, j - qh * per_head, turned, a.rot, a.interleaved);
      }
      item.store(qo + qh * a.D, j - qh * per_head, turned, a.rot, a.interleaved, cs);
    }
  } else {
    for (int j = threadIdx.x; j < items; j += 256) {
      const int qd = (j % per_head) * 4;
      Quad<T> x;
      qh = j / per_head;
      x.load(q + qh * a.ldq_h, qd, a.rot, a.interleaved);
      x.turn(qd, a.rot, a.interleaved, cs);
      store_values<T, 4>(qo + qh * a.D + qd, x.v);
    }
  }
  if (!in) return;
  const int64_t page = slot / a.P;
  const int row = (int)(slot - page * a.P);
  for (; i < 2 * groups; i += 16) {
    if (i >= 16) {
      group_of(i, h, d);
      load_quad(i, h, d, quad);
    }
    const bool key = i < groups;
    if (key) {
      quad.turn(d, a.rot, a.interleaved, cs);
#pragma unroll
      for (int e = 0; e < 4; ++e) quad.v[e] = to_f32(from_f32<T>(quad.v[e]));
    }
    _Float16 s, lo;
    const uint32_t c = code4(quad.v, s, lo);
    const int g = d / kKv4Group;
    uint8_t* block = a.cache + (page * a.Hkv + h) * (int64_t)L.bytes();
    if (key) {
      // a nibble in each byte: the even lane's low ones, the odd lane's high ones
      uint32_t w = (c & 0xf) | (c >> 4 & 0xf) << 8 | (c >> 8 & 0xf) << 16 | (c >> 12 & 0xf) << 24;
      if (m & 1) w <<= 4;
      w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xf, 0xf, true);  // the neighbour's half
      if (!(m & 1)) *reinterpret_cast<uint32_t*>(block + L.k_dword(row, d)) = w;
      if (m == 0) {
        const uint32_t pair = (uint32_t)__builtin_bit_cast(uint16_t, s) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
        *reinterpret_cast<uint32_t*>(block + L.k_scale(row, g)) = pair;
      }
    } else {
      uint8_t* to = block + L.v_byte(row, d);
      to[0] = (uint8_t)c;
      to[2] = (uint8_t)(c >> 8);
      if (m == 0) {
        uint8_t* at = block + L.v_scale(row, g);
        *reinterpret_cast<uint16_t*>(at) = __builtin_bit_cast(uint16_t, s);
        *reinterpret_cast<uint16_t*>(at + 8) = __builtin_bit_cast(uint16_t, lo);
      }
    }
  }
}

template <class T>
int launch_append(const AppendArgs& a, int64_t tokens, hipStream_t s) {
  const int64_t each = most_blocks(256);
  for (int64_t t0 = 0; t0 < tokens; t0 += each) {
    AppendArgs part = a;
    part.k = static_cast<const T*>(a.k) + t0 * a.ldk_t;
    part.v = static_cast<const T*>(a.v) + t0 * a.ldv_t;
    if (a.Hq) {
      part.q = static_cast<const T*>(a.q) + t0 * a.ldq_t;
      part.q_out = static_cast<T*>(a.q_out) + t0 * a.Hq * a.D;
    }
    part.slots = a.slots + t0;
    if (a.rot) part.pos = a.pos + t0;
    hipLaunchKernelGGL(k_kv4_append<T>, dim3((unsigned)(tokens - t0 < each ? tokens - t0 : each)), dim3(256), 0, s, part);
    const int status = hip_check(hipGetLastError(), "k_kv4_append launch");
    if (status != QS_OK) return status;
  }
  return QS_OK;
}

template <class T>
__global__ __launch_bounds__(256) void k_kv4_read(const uint8_t* cache, const int64_t* slots, int64_t slots_all, int P,
                                                  int D, int Hkv, int64_t n, T* k_out, T* v_out) {
  const Kv4Layout L(P, D);
  const int per_head = D / 8, per_token = Hkv * per_head;
  const int64_t items = n * per_token;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / per_token;
    const int rest = (int)(i - t * per_token);
    const int h = rest / per_head, d = (rest - h * per_head) * 8, g = d / kKv4Group;
    const int64_t slot = slots[t];
    float k[8] = {}, v[8] = {};
    if (slot >= 0 && slot < slots_all) {
      const int64_t page = slot / P;
      const int row = (int)(slot - page * P);
      const uint8_t* block = cache + (page * Hkv + h) * (int64_t)L.bytes();
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(block + L.k_dword(row, d));
      const uint32_t ks = *reinterpret_cast<const uint32_t*>(block + L.k_scale(row, g));
      const uint8_t* v0 = block + L.v_byte(row, d);
      const uint8_t* v1 = block + L.v_byte(row, d + 4);
      const uint32_t vw = v0[0] | v0[2] << 8 | v1[0] << 16 | (uint32_t)v1[2] << 24;
      const float vs = f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(block + L.v_scale(row, g)));
      const float vl = f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(block + L.v_scale(row, g) + 8));
      const float sc = f16_bits_to_f32((uint16_t)ks), lo = f16_bits_to_f32((uint16_t)(ks >> 16));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        k[e] = (float)(kw >> Kv4Layout::k_shift(e) & 15) * sc + lo;
        v[e] = (float)(vw >> (4 * e) & 15) * vs + vl;
      }
    }
    const int64_t at = (t * Hkv + h) * D + d;
    if (k_out) store_values<T, 8>(k_out + at, k);
    if (v_out) store_values<T, 8>(v_out + at, v);
  }
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" size_t qs_kv4_block_bytes(int64_t head_dim, int64_t page_size) {
  return kv4_shape_ok(head_dim, page_size) ? (size_t)Kv4Layout((int)page_size, (int)head_dim).bytes() : 0;
}

extern "C" int qs_kv4_append(const void* k, int64_t ldk_t, int64_t ldk_h, const void* v, int64_t ldv_t, int64_t ldv_h,
                             int dtype, const int64_t* slots, uint8_t* cache, int64_t pages, int64_t page_size,
                             int Hkv, int D, int64_t T, const void* q, int64_t ldq_t, int64_t ldq_h, int Hq, void* q_out,
                             const int32_t* positions, const double* freq, int rot, int interleaved, double magnitude,
                             void* stream) {
  if (!kv4_shape_ok(D, page_size)) return fail(QS_ERR_UNSUPPORTED, "kv4_append: head size %d, page size %lld", D,
                                               (long long)page_size);
  if (T < 0 || pages <= 0 || Hkv <= 0 || Hkv > 4096 || Hq < 0 || Hq > 65536)
    return fail(QS_ERR_INVALID, "kv4_append: bad shape");
  if (T >= (int64_t(1) << 31) || pages >= (int64_t(1) << 31)) return fail(QS_ERR_LIMIT, "kv4_append: 2^31 tokens or pages or more");
  if (rot < 0 || rot > D || rot % 8) return fail(QS_ERR_INVALID, "kv4_append: rotated size %d of a head of %d", rot, D);
  if (T == 0) return QS_OK;
  if (!k || !v || !slots || !cache || (Hq > 0 && (!q || !q_out)) || (rot > 0 && (!positions || !freq)))
    return fail(QS_ERR_INVALID, "kv4_append: null pointer");
  const int size = dtype == QS_F32 ? 4 : 2;
  const int64_t ld = ldk_t | ldk_h | ldv_t | ldv_h | (Hq ? ldq_t | ldq_h : 0);
  if (ld % 4 || !aligned(k, 4 * size) || !aligned(v, 4 * size) || (Hq && (!aligned(q, 4 * size) || !aligned(q_out, 4 * size))) ||
      !aligned(cache, 16))
    return fail(QS_ERR_INVALID, "kv4_append: heads are aligned to four values");
  AppendArgs a{k, v, q, q_out, slots, positions, freq, cache, ldk_t, ldk_h, ldv_t, ldv_h, ldq_t, ldq_h,
               pages * page_size, (int)page_size, D, Hkv, Hq, rot, interleaved, 0, magnitude};
  const int per16 = 16 / size;
  a.wide = Hq > 0 && aligned(q, 16) && aligned(q_out, 16) && ldq_t % per16 == 0 && ldq_h % per16 == 0 &&
           (size == 4 ? TurnItem<float>::fits(D, rot, interleaved) : TurnItem<__bf16>::fits(D, rot, interleaved));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == QS_F32) return launch_append<float>(a, T, s);
  if (dtype == QS_BF16) return launch_append<__bf16>(a, T, s);
  if (dtype == QS_F16) return launch_append<_Float16>(a, T, s);
  return fail(QS_ERR_INVALID, "kv4_append: dtype must be F32, BF16 or F16");
}

extern "C" int qs_kv4_read(const uint8_t* cache, int64_t pages, int64_t page_size, int Hkv, int D, const int64_t* slots,
                           int64_t n, void* k_out, void* v_out, int out_dtype, void* stream) {
  if (!kv4_shape_ok(D, page_size)) return fail(QS_ERR_UNSUPPORTED, "kv4_read: head size %d, page size %lld", D,
                                               (long long)page_size);
  if (n < 0 || pages <= 0 || Hkv <= 0 || Hkv > 4096) return fail(QS_ERR_INVALID, "kv4_read: bad shape");
  if (pages >= (int64_t(1) << 31)) return fail(QS_ERR_LIMIT, "kv4_read: 2^31 pages or more");
  if (n == 0) return QS_OK;
  if (!cache || !slots || (!k_out && !v_out)) return fail(QS_ERR_INVALID, "kv4_read: null pointer");
  if (!aligned(cache, 16) || !aligned(k_out, 16) || !aligned(v_out, 16))
    return fail(QS_ERR_INVALID, "kv4_read: 16-byte alignment");
  const int64_t want = cdiv(n * Hkv * (D / 8), 256);
  const dim3 grid((unsigned)(want < 65536 ? want : 65536)), block(256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t all = pages * page_size;
  if (out_dtype == QS_F32)
    hipLaunchKernelGGL(k_kv4_read<float>, grid, block, 0, s, cache, slots, all, (int)page_size, D, Hkv, n,
                       static_cast<float*>(k_out), static_cast<float*>(v_out));
  else if (out_dtype == QS_BF16)
    hipLaunchKernelGGL(k_kv4_read<__bf16>, grid, block, 0, s, cache, slots, all, (int)page_size, D, Hkv, n,
                       static_cast<__bf16*>(k_out), static_cast<__bf16*>(v_out));
  else if (out_dtype == QS_F16)
    hipLaunchKernelGGL(k_kv4_read<_Float16>, grid, block, 0, s, cache, slots, all, (int)page_size, D, Hkv, n,
                       static_cast<_Float16*>(k_out), static_cast<_Float16*>(v_out));
  else
    return fail(QS_ERR_INVALID, "kv4_read: dtype must be F32, BF16 or F16");
  return hip_check(hipGetLastError(), "k_kv4_read launch");
}
