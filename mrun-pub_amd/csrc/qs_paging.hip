// Paging metadata of a step, built on the GPU from request lengths (gfx950).
//
// A request with p tokens in the cache and n new ones owns ceil(p / P) pages and needs
// ceil((p + n) / P) - ceil(p / P) more.  Requests take theirs in order from a ring of free pages, so
// a page's rank in the ring is an exclusive sum over the requests, and everything else follows from
// the ranks.
//
//   k_plan_step     : one launch.  Every block redoes the sums over all requests (8 bytes each, in
//                     LDS for kPlanThreads at a time) and then fills its own tokens, so no
//                     block waits for another.  The ring's new state goes to a place of its own:
//                     the step can be planned again, and captured into a graph.
//   k_release_pages : finished requests' pages back to the ring's end, in request order.
//
// Bound by latency: 7 requests take 3.9 us, 511 requests with 48,000 tokens 5.5 (two chunks of 256
// requests and four tokens a thread took 8.7).
#include "qs_common.h"

namespace qs {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanTokens = 512;  // of a block

struct PlanArgs {
  const int* ring;
  int64_t ring_size;
  const int64_t* state;
  int64_t* state_out;
  int* tables;
  int64_t ld;
  int width;
  const int* past;
  const int* fresh;
  int B, P, shift;
  int64_t T;
  int64_t* slots;
  int* positions;
  int* requests;
  int* starts;
  int* context;
};

// Inclusive sum over the wave.
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t o = __shfl_up(v, off, 64);
    if (lane >= off) v += o;
  }
  return v;
}

// Exclusive sum of v over the block, and the total.
struct Scan {
  int64_t before, total;
};
__device__ __forceinline__ Scan block_scan(int64_t v, int64_t* part) {
  const int wave = threadIdx.x >> 6;
  const int64_t inclusive = wave_scan(v);
  if ((threadIdx.x & 63) == 63) part[wave] = inclusive;
  __syncthreads();
  Scan r{inclusive - v, 0};
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) r.before += part[w];
    r.total += part[w];
  }
  __syncthreads();
  return r;
}

// Ring entry `at` places after place `from` (both below the ring's size).
__device__ __forceinline__ int64_t ring_at(int64_t from, int64_t at, int64_t size) {
  const int64_t i = from + at;
  return i < size ? i : i - size;
}

__global__ __launch_bounds__(kPlanThreads) void k_plan_step(PlanArgs p) {
  __shared__ int64_t part[kPlanThreads / 64];
  __shared__ int64_t s_start[kPlanThreads + 1], s_rank[kPlanThreads];
  __shared__ int s_past[kPlanThreads];
  const int64_t head = p.state[0], tail = p.state[1];
  const int64_t avail = tail > head ? (tail - head < p.ring_size ? tail - head : p.ring_size) : 0;
  const int64_t from = (int64_t)((uint64_t)head % (uint64_t)p.ring_size);
  const int64_t t0 = (int64_t)blockIdx.x * kPlanTokens;
  const int64_t t1 = t0 + kPlanTokens < p.T ? t0 + kPlanTokens : p.T;
  int64_t tokens = 0, pages = 0;  // of the requests before this chunk
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    int64_t past = 0, n = 0;
    if (b < p.B) {
      past = p.past[b] > 0 ? p.past[b] : 0;
      n = p.fresh[b] > 0 ? p.fresh[b] : 0;
    }
    const Scan st = block_scan(n, part);
    const int64_t start = tokens + st.before;
    // rows past T and columns past the table take no page
    n = start >= p.T ? 0 : n < p.T - start ? n : p.T - start;
    const int64_t owned = (past + p.P - 1) >> p.shift;
    const int64_t whole = (past + n + p.P - 1) >> p.shift;
    const int64_t last = whole < p.width ? whole : p.width;
    const Scan sp = block_scan(last > owned ? last - owned : 0, part);
    s_start[threadIdx.x] = start;
    s_rank[threadIdx.x] = pages + sp.before - owned;  // of the page at table column 0
    s_past[threadIdx.x] = (int)past;
    if (threadIdx.x == 0) s_start[kPlanThreads] = tokens + st.total;
    if (blockIdx.x == 0 && b < p.B) {
      p.starts[b] = (int)(start < p.T ? start : p.T);
      p.context[b] = (int)(past + n);
    }
    __syncthreads();
    // this block's tokens that fall to this chunk of requests
    const int count = p.B - b0 < kPlanThreads ? p.B - b0 : kPlanThreads;
    const int64_t lo = t0 > tokens ? t0 : tokens;
    const int64_t end = s_start[kPlanThreads];
    const int64_t hi = t1 < end ? t1 : end;
    for (int64_t t = lo + threadIdx.x; t < hi; t += kPlanThreads) {
      int at = 0;  // the last request that starts at or before t
#pragma unroll
      for (int step = kPlanThreads / 2; step >= 1; step >>= 1)
        if (at + step < count && s_start[at + step] <= t) at += step;
      const int64_t pos = s_past[at] + (t - s_start[at]);
      const int64_t col = pos >> p.shift;
      const int64_t own = ((int64_t)s_past[at] + p.P - 1) >> p.shift;
      int64_t page = -1;
      if (col < p.width) {
        int* entry = p.tables + (b0 + at) * p.ld + col;
        if (col < own) {
          page = *entry;
        } else {
          const int64_t rank = s_rank[at] + col;
          if (rank < avail) page = p.ring[ring_at(from, rank, p.ring_size)];
          if ((pos & (p.P - 1)) == 0) *entry = (int)page;
        }
      }
      p.slots[t] = page >= 0 ? (page << p.shift) + (pos & (p.P - 1)) : -1;
      p.positions[t] = (int)pos;
      p.requests[t] = b0 + at;
    }
    tokens += st.total;
    pages += sp.total;
    __syncthreads();
  }
  for (int64_t t = (t0 > tokens ? t0 : tokens) + threadIdx.x; t < t1; t += kPlanThreads) {  // padding
    p.slots[t] = -1;
    p.positions[t] = 0;
    p.requests[t] = -1;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.starts[p.B] = (int)(tokens < p.T ? tokens : p.T);
    const int64_t taken = pages < avail ? pages : avail;
    p.state_out[0] = head + taken;
    p.state_out[1] = tail;
    p.state_out[2] = pages - taken;
  }
}

struct ReleaseArgs {
  int* ring;
  int64_t ring_size;
  const int64_t* state;
  int64_t* state_out;
  const int* tables;
  int64_t ld;
  int width;
  const int* lens;
  const uint8_t* done;
  int B, P, shift;
};

// One block: the finished requests in turn, 512 table columns at a time.  Only pages come back: a
// table entry of -1 (no page was left for it) takes no place in the ring.
__global__ __launch_bounds__(kPlanThreads) void k_release_pages(ReleaseArgs p) {
  __shared__ int64_t part[kPlanThreads / 64];
  __shared__ int64_t s_columns[kPlanThreads];
  int64_t tail = p.state[1];
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int own = b0 + threadIdx.x;
    int64_t columns = 0;
    if (own < p.B && p.done[own] && p.lens[own] > 0) {
      columns = ((int64_t)p.lens[own] + p.P - 1) >> p.shift;
      if (columns > p.width) columns = p.width;
    }
    s_columns[threadIdx.x] = columns;
    __syncthreads();
    for (int i = 0; i < kPlanThreads; ++i) {
      for (int64_t c0 = 0; c0 < s_columns[i]; c0 += kPlanThreads) {
        const int64_t c = c0 + threadIdx.x;
        const int page = c < s_columns[i] ? p.tables[(int64_t)(b0 + i) * p.ld + c] : -1;
        const Scan s = block_scan(page >= 0, part);
        if (page >= 0) p.ring[(uint64_t)(tail + s.before) % (uint64_t)p.ring_size] = page;
        tail += s.total;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    p.state_out[0] = p.state[0];
    p.state_out[1] = tail;
    p.state_out[2] = 0;
  }
}

int log2_page(int64_t P) {
  for (int s = 0; s <= 20; ++s)
    if (P == (int64_t(1) << s)) return s;
  return -1;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" int qs_plan_step(const int32_t* ring, int64_t ring_size, const int64_t* state, int64_t* state_out,
                            int32_t* tables, int64_t ld_table, int64_t width, const int32_t* past,
                            const int32_t* fresh, int64_t B, int64_t page_size, int64_t T, int64_t* slots,
                            int32_t* positions, int32_t* requests, int32_t* starts, int32_t* context, void* stream) {
  if (B < 0 || T < 0 || width < 0 || ring_size <= 0 || (B > 1 && ld_table < width))
    return fail(QS_ERR_INVALID, "plan_step: bad shape");
  const int shift = log2_page(page_size);
  if (shift < 0) return fail(QS_ERR_INVALID, "plan_step: page size %lld is not a power of two up to 2^20",
                             (long long)page_size);
  if (B > (1 << 20) || T >= (int64_t(1) << 31) || width >= (int64_t(1) << 31) || ring_size >= (int64_t(1) << 31))
    return fail(QS_ERR_LIMIT, "plan_step: over 2^20 requests, or 2^31 tokens, columns or pages or more");
  if (!ring || !state || !state_out || !starts || (B > 0 && (!past || !fresh || !context)) ||
      (B > 0 && width > 0 && !tables) || (T > 0 && (!slots || !positions || !requests)))
    return fail(QS_ERR_INVALID, "plan_step: null pointer");
  if (state == state_out) return fail(QS_ERR_INVALID, "plan_step: the ring's new state needs a place of its own");
  PlanArgs p{ring, ring_size, state, state_out, tables, ld_table, (int)width, past, fresh, (int)B, (int)page_size,
             shift, T, slots, positions, requests, starts, context};
  const int64_t blocks = T > 0 ? cdiv(T, kPlanTokens) : 1;
  hipLaunchKernelGGL(k_plan_step, dim3((unsigned)blocks), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), p);
  return hip_check(hipGetLastError(), "k_plan_step launch");
}

extern "C" int qs_release_pages(int32_t* ring, int64_t ring_size, const int64_t* state, int64_t* state_out,
                                const int32_t* tables, int64_t ld_table, int64_t width, const int32_t* lens,
                                const uint8_t* done, int64_t B, int64_t page_size, void* stream) {
  if (B < 0 || width < 0 || ring_size <= 0 || (B > 1 && ld_table < width))
    return fail(QS_ERR_INVALID, "release_pages: bad shape");
  const int shift = log2_page(page_size);
  if (shift < 0) return fail(QS_ERR_INVALID, "release_pages: page size %lld is not a power of two up to 2^20",
                             (long long)page_size);
  if (B > (1 << 20) || width >= (int64_t(1) << 31) || ring_size >= (int64_t(1) << 31))
    return fail(QS_ERR_LIMIT, "release_pages: over 2^20 requests, or 2^31 columns or pages or more");
  if (!ring || !state || !state_out || (B > 0 && (!lens || !done)) || (B > 0 && width > 0 && !tables))
    return fail(QS_ERR_INVALID, "release_pages: null pointer");
  if (state == state_out) return fail(QS_ERR_INVALID, "release_pages: the ring's new state needs a place of its own");
  ReleaseArgs p{ring, ring_size, state, state_out, tables, ld_table, (int)width, lens, done, (int)B, (int)page_size,
                shift};
  hipLaunchKernelGGL(k_release_pages, dim3(1), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), p);
  return hip_check(hipGetLastError(), "k_release_pages launch");
}
