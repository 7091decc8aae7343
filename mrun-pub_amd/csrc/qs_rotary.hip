// Rotary positions of activations on gfx950.
//
//   k_rotary_v : 16 bytes of both halves of a pair (half layout) or of 2 to 4 whole pairs
//                (interleaved) a work item; aligned rows whose sizes divide.
//   k_rotary_1 : one pair or one untouched value an item, any sizes and strides.
//
// y1 = x1 c - x2 s, y2 = x2 c + x1 s, products and sums each rounded in fp32 and the result once to
// x's type; the inverse (which is also the gradient) turns by -s.  Bound by memory: every value is
// read once and written once, and a block's threads share their tokens' angles through LDS.  8191
// tokens of 40 heads of 128 (168 MB) take 35.6 us, 4.7 TB/s of a copy's 5.1; one token 2.4.
#include "qs_rotary.h"
#include "qs_values.h"

namespace qs {
namespace {

struct RotaryArgs {
  const void* x;
  void* y;
  const int* pos;
  const double* freq;
  int64_t ldx_t, ldx_h, ldy_t, ldy_h, T;
  int H, D, rot, interleaved, inverse, tokens;
  double mag;
};

// Cos and sin of the block's tokens, [tokens][rot/2].
__device__ __forceinline__ void block_angles(const RotaryArgs& a, int64_t t0, float2* cs) {
  const int half = a.rot / 2;
  for (int i = threadIdx.x; i < a.tokens * half; i += blockDim.x) {
    const int t = i / half;
    if (t0 + t >= a.T) break;
    float2 v = rotary_cos_sin(a.pos[t0 + t], a.freq[i - t * half], a.mag);
    if (a.inverse) v.y = -v.y;
    cs[i] = v;
  }
  __syncthreads();
}

template <class T>
__global__ __launch_bounds__(256) void k_rotary_v(RotaryArgs a) {
  using Item = TurnItem<T>;
  extern __shared__ float2 cs[];
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int turned = Item::turned(a.rot, a.interleaved);  // items of a head that turn
  const int per_head = turned + (a.D - a.rot) / Item::V;
  const int per_token = per_head * a.H;
  const int64_t left = a.T - t0;
  const int items = per_token * (int)(left < a.tokens ? left : a.tokens);
  auto at = [&](int i, int& t, int& c, int& h) {
    t = i / per_token;
    const int rest = i - t * per_token;
    h = rest / per_head;
    c = rest - h * per_head;
  };
  Item item;  // the first is under way while the angles are computed
  int t, c, h;
  if (threadIdx.x < items) {
    at(threadIdx.x, t, c, h);
    item.load(static_cast<const T*>(a.x) + (t0 + t) * a.ldx_t + h * a.ldx_h, c, turned, a.rot, a.interleaved);
  }
  block_angles(a, t0, cs);
  for (int i = threadIdx.x; i < items; i += 256) {
    if (i >= 256) {
      at(i, t, c, h);
      item.load(static_cast<const T*>(a.x) + (t0 + t) * a.ldx_t + h * a.ldx_h, c, turned, a.rot, a.interleaved);
    }
    item.store(static_cast<T*>(a.y) + (t0 + t) * a.ldy_t + h * a.ldy_h, c, turned, a.rot, a.interleaved, cs + t * (a.rot / 2));
  }
}

template <class T>
__global__ __launch_bounds__(256) void k_rotary_1(RotaryArgs a) {
  extern __shared__ float2 cs[];
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int half = a.rot / 2;
  const int per_head = half + a.D - a.rot;
  const int per_token = per_head * a.H;
  block_angles(a, t0, cs);
  const int64_t left = a.T - t0;
  const int items = per_token * (int)(left < a.tokens ? left : a.tokens);
  for (int i = threadIdx.x; i < items; i += 256) {
    const int t = i / per_token, rest = i - t * per_token;
    const int h = rest / per_head, c = rest - h * per_head;
    const T* x = static_cast<const T*>(a.x) + (t0 + t) * a.ldx_t + h * a.ldx_h;
    T* y = static_cast<T*>(a.y) + (t0 + t) * a.ldy_t + h * a.ldy_h;
    if (c >= half) {
      y[a.rot + c - half] = x[a.rot + c - half];
      continue;
    }
    const int d1 = a.interleaved ? 2 * c : c, d2 = a.interleaved ? 2 * c + 1 : c + half;
    const float2 w = cs[t * half + c];
    const float x1 = to_f32(x[d1]), x2 = to_f32(x[d2]);
    y[d1] = from_f32<T>(x1 * w.x - x2 * w.y);
    y[d2] = from_f32<T>(x2 * w.x + x1 * w.y);
  }
}

template <class T>
int launch_rotary(RotaryArgs a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = TurnItem<T>::fits(a.D, a.rot, a.interleaved) && aligned(a.x, 16) && aligned(a.y, 16) &&
                    a.ldx_t % V == 0 && a.ldx_h % V == 0 && a.ldy_t % V == 0 && a.ldy_h % V == 0;
  const int64_t per_token = (int64_t)a.H * (wide ? (a.interleaved ? a.D / V : a.D / V - a.rot / 2 / V)
                                                 : a.D - a.rot / 2);
  // tokens of few items share a block, up to 16, whose angles are at most 16 x 1024 x 8 bytes
  a.tokens = (int)(per_token >= 256 ? 1 : 256 / per_token < 16 ? 256 / per_token : 16);
  if (a.tokens * a.rot > 8192) a.tokens = a.rot > 8192 ? 1 : 8192 / a.rot;
  const size_t lds = (size_t)a.tokens * (a.rot / 2) * sizeof(float2);
  const int64_t each = most_blocks(256) * a.tokens, all = a.T;  // tokens of a launch
  for (int64_t t0 = 0; t0 < all; t0 += each) {
    RotaryArgs part = a;
    part.x = static_cast<const T*>(a.x) + t0 * a.ldx_t;
    part.y = static_cast<T*>(a.y) + t0 * a.ldy_t;
    part.pos = a.pos + t0;
    part.T = all - t0 < each ? all - t0 : each;
    const dim3 grid((unsigned)cdiv(part.T, a.tokens));
    if (wide)
      hipLaunchKernelGGL(k_rotary_v<T>, grid, dim3(256), lds, s, part);
    else
      hipLaunchKernelGGL(k_rotary_1<T>, grid, dim3(256), lds, s, part);
    const int status = hip_check(hipGetLastError(), "k_rotary launch");
    if (status != QS_OK) return status;
  }
  return QS_OK;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" int qs_rotary(const void* x, int dtype, int64_t ldx_t, int64_t ldx_h, const int32_t* positions,
                         const double* freq, int rot, int interleaved, int inverse, double magnitude, void* y,
                         int64_t ldy_t, int64_t ldy_h, int64_t T, int H, int D, void* stream) {
  if (T < 0 || H <= 0 || D <= 0) return fail(QS_ERR_INVALID, "rotary: bad shape");
  if (rot <= 0 || rot % 2 || rot > D) return fail(QS_ERR_INVALID, "rotary: rotated size %d of a head of %d", rot, D);
  if (D > 4096) return fail(QS_ERR_LIMIT, "rotary: head size above 4096");
  if ((int64_t)H * D > (int64_t(1) << 24)) return fail(QS_ERR_LIMIT, "rotary: a token's row above 2^24 values");
  if (T >= (int64_t(1) << 31)) return fail(QS_ERR_LIMIT, "rotary: 2^31 tokens or more");
  if (T == 0) return QS_OK;
  if (!x || !y || !positions || !freq) return fail(QS_ERR_INVALID, "rotary: null pointer");
  RotaryArgs a{x, y, positions, freq, ldx_t, ldx_h, ldy_t, ldy_h, T, H, D, rot, interleaved, inverse, 1, magnitude};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == QS_F32) return launch_rotary<float>(a, s);
  if (dtype == QS_BF16) return launch_rotary<__bf16>(a, s);
  if (dtype == QS_F16) return launch_rotary<_Float16>(a, s);
  return fail(QS_ERR_INVALID, "rotary: dtype must be F32, BF16 or F16");
}
