// mtp_kvevict.cuh -- cuts every sequence of a paged cache to `budget` tokens,
// key head by key head: the first `sinks`, the last `recent` and, of the
// others, those with the greatest accumulated attention weight (ties: the
// lower index; a NaN weight counts as the lowest).  The kept tokens keep their
// order and move down to positions 0 .. budget-1; their weights move along and
// the weights behind them become 0.  A sequence of at most `budget` tokens
// stays as it is.
//
// evict_select_kernel (one block per (sequence, head)): the m-th greatest
// weight by a radix search over the order-preserving bits of the weights (11 +
// 11 + 10 bits, three reads of the row from L2 and a histogram in shared
// memory), then one more read that numbers the kept tokens with block scans
// and writes their source and destination rows of the pool.
// evict_move_kernel: moves the rows.  A row moves down or stays (the i-th
// kept token has index >= i), so a block that holds a slice of every row of its
// unit walks through them in order: all its threads read the rows of a step
// before any of them writes one, and rows read later lie above everything that
// has been written.  Slices of a row (and K and V) do not meet, so they are
// blocks of their own.  Bytes-bound: budget rows of K and V read and written.
// Measured (B200): 16 sequences of 2000 .. 8192 tokens cut to 4096, Hkv 8, D 128,
// bf16: 18 us of selection and 58 us of moves on a fresh cache.  A cache that was
// cut before moves fewer rows (those already in place stay): 30 us.
#pragma once

#include "mtp_common.cuh"

namespace mtp {
namespace evict {

constexpr int kThreads = 1024;     // select
constexpr int kPerThread = 8;      // consecutive tokens per thread and step
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 4;

struct Args {
  void* pages[2];
  const int32_t* page_table;
  int64_t table_stride, num_pages, page_size;
  const int32_t* seq_lens;
  float* weights;  // [B, H, weight_ld]
  int64_t weight_ld;
  int32_t* kept;      // [B, H, budget]
  int32_t* new_lens;  // [B]
  int2* rows;         // [B, H, budget] source and destination rows of the pool (-1: not moved)
  int B, H, D, budget, sinks, recent;
};

__device__ __forceinline__ int length(const Args& a, int b, bool report) {
  const int len = a.seq_lens[b];
  const int cap = (int)min(min(a.table_stride, a.weight_ld), (int64_t)INT32_MAX);
  const int r = max(0, min(len, cap));
  if (report && r != len) record_error(MTP_ERR_DEVICE);
  return r;
}

// order-preserving bits of a weight; -0 and 0 are equal
__device__ __forceinline__ uint32_t order_bits(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// exclusive prefix of v over the block and its total
__device__ __forceinline__ int block_scan(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // s_warp may still be read from the call before
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int w = lane < kThreads / 32 ? s_warp[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, warp) - __shfl_sync(0xffffffffu, x, 31);
  return before + x - v;
}

__global__ void __launch_bounds__(kThreads) evict_select_kernel(Args a) {
  __shared__ int s_hist[kBins];
  __shared__ int s_warp[kThreads / 32];
  __shared__ int s_digit, s_left;
  const int h = blockIdx.x % a.H, b = blockIdx.x / a.H, tid = threadIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the moving kernel waits for this one's end
  const int len = length(a, b, h == 0 && tid == 0);
  const int n = min(len, a.budget);
  if (h == 0 && tid == 0) a.new_lens[b] = n;
  const int64_t unit = (int64_t)b * a.H + h;
  int32_t* kept = a.kept + unit * a.budget;
  int2* rows = a.rows + unit * a.budget;
  float* w = a.weights + unit * a.weight_ld;
  if (len <= a.budget) {
    for (int i = tid; i < a.budget; i += kThreads) {
      kept[i] = i < len ? i : -1;
      rows[i] = make_int2(-1, -1);
    }
    return;
  }
  const int lo = a.sinks, hi = len - a.recent;  // the tokens that compete
  int left = a.budget - a.sinks - a.recent;     // and how many of them stay
  // threshold: keys above it stay, of the keys equal to it the first `left`
  uint32_t threshold = 0xffffffffu;
  if (left > 0) {
    uint32_t prefix = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      const int bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kBins; i += kThreads) s_hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int j = lo + tid; j < hi; j += kThreads) {
        const uint32_t k = order_bits(w[j]);
        if (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits)))
          atomicAdd(&s_hist[(k >> shift) & ((1u << bits) - 1u)], 1);
      }
      __syncthreads();
      // bins from the greatest down, two per thread
      const int b0 = kBins - 1 - 2 * tid, b1 = b0 - 1;
      const int c0 = s_hist[b0], c1 = s_hist[b1];
      int total;
      const int before = block_scan(c0 + c1, s_warp, &total);
      if (before < left && before + c0 + c1 >= left) {
        const bool first = before + c0 >= left;
        s_digit = first ? b0 : b1;
        s_left = left - before - (first ? 0 : c0);
      }
      __syncthreads();
      prefix |= (uint32_t)s_digit << shift;
      left = s_left;
      __syncthreads();
    }
    threshold = prefix;
  }
  // number the kept tokens: forced or above the threshold, and the first `left` equal ones
  int above = 0, equal = 0;  // before this step
  for (int base = 0; base < len; base += kThreads * kPerThread) {
    const int j0 = base + tid * kPerThread;
    uint32_t up = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int j = j0 + i;
      if (j < len) {
        if (j < lo || j >= hi) {
          up |= 1u << i;
        } else if (a.budget > a.sinks + a.recent) {
          const uint32_t k = order_bits(w[j]);
          if (k > threshold) up |= 1u << i;
          if (k == threshold) eq |= 1u << i;
        }
      }
    }
    // both counts in one scan: at most 8192 of each per step
    int total;
    const int before = block_scan(__popc(up) | (__popc(eq) << 16), s_warp, &total);
    int u = above + (before & 0xffff), e = equal + (before >> 16);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const bool is_up = (up >> i) & 1u, is_eq = (eq >> i) & 1u;
      if (is_up || (is_eq && e < left)) kept[u + min(e, left)] = j0 + i;
      u += is_up;
      e += is_eq;
    }
    above += total & 0xffff;
    equal += total >> 16;
  }
  __syncthreads();
  // rows of the pool, and the weights (read a step, then write it: sources lie at or above it)
  const int32_t* table = a.page_table + b * a.table_stride;
  for (int base = 0; base < a.budget; base += kThreads) {
    const int i = base + tid;
    float x = 0.f;
    if (i < a.budget) {
      const int j = kept[i];
      x = w[j];
      const int64_t from = resolve_page(table[j], a.num_pages), to = resolve_page(table[i], a.num_pages);
      int2 r = make_int2(-1, -1);
      if (from < 0 || to < 0) {
        record_error(MTP_ERR_DEVICE);
      } else if (j != i) {
        r.x = (int)(((from * a.B + b) * a.H + h) * a.page_size + j % a.page_size);
        r.y = (int)(((to * a.B + b) * a.H + h) * a.page_size + i % a.page_size);
      }
      rows[i] = r;
    }
    __syncthreads();
    if (i < a.budget) w[i] = x;
  }
  __syncthreads();
  for (int j = a.budget + tid; j < len; j += kThreads) w[j] = 0.f;
}

// V: the word that rows are moved in; a block holds `lanes` of the `words` words
// of every row of its unit (lanes a power of two that divides words).
template <typename V>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(Args a, int words, int lanes) {
  const int slices = words / lanes;
  const int unit = blockIdx.x / (2 * slices), part = blockIdx.x % (2 * slices);
  const int b = unit / a.H;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (length(a, b, false) <= a.budget) return;
  V* pool = static_cast<V*>(a.pages[part / slices]) + (part % slices) * lanes + threadIdx.x % lanes;
  const int2* rows = a.rows + (int64_t)unit * a.budget;
  const int per_pass = kMoveThreads / lanes, first = threadIdx.x / lanes;
  const int step = per_pass * kMoveUnroll;
  auto load_rows = [&](int base, int2 (&r)[kMoveUnroll]) {
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = base + u * per_pass + first;
      r[u] = i < a.budget ? rows[i] : make_int2(-1, -1);
    }
  };
  int2 r0[kMoveUnroll], r1[kMoveUnroll];
  V v0[kMoveUnroll], v1[kMoveUnroll];
  load_rows(0, r0);
  load_rows(step, r1);
#pragma unroll
  for (int u = 0; u < kMoveUnroll; ++u)
    if (r0[u].x >= 0) v0[u] = pool[(int64_t)r0[u].x * words];
  for (int base = 0; base < a.budget; base += step) {
    // the next step's rows lie above everything written so far and in this step
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u)
      if (r1[u].x >= 0) v1[u] = pool[(int64_t)r1[u].x * words];
    int2 r2[kMoveUnroll];
    load_rows(base + 2 * step, r2);
    __syncthreads();  // every thread has read this step's rows (and the next one's)
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u)
      if (r0[u].x >= 0) pool[(int64_t)r0[u].y * words] = v0[u];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      r0[u] = r1[u];
      r1[u] = r2[u];
      v0[u] = v1[u];
    }
  }
}

}  // namespace evict
}  // namespace mtp
