// mtp_qknorm_rope.cuh -- RMSNorm of every query and key head, the position
// rotation and (paged form) the write of keys and values into the page pool,
// in one pass over the projection's output.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                       per head, fp32
//   (a, b) -> (a cos - b sin, b cos + a sin)                 first R values
//
// The pair (a, b) is (y[i], y[i + R/2]) or, interleaved, (y[2i], y[2i + 1]),
// with cos/sin row `position` of the caller's tables.  Everything is fp32
// with one rounding to the output dtype at the end (composing a norm and a
// rotation operator rounds twice).
//
// Bytes-bound: every value is read once and written once.  A head is spread
// over LPH = 8, 16 or 32 lanes with 8 values (16 bytes of a 16-bit type) each,
// so that a load or store instruction moves whole heads, the sum of squares is
// a shuffle over LPH lanes and the partner of a split pair sits in lane
// +- R/16.  A group of LPH lanes stays with one token and walks over its
// heads: its cos/sin values are loaded once into registers and serve all of
// them, and four heads' loads are in flight before the first is used.
#pragma once

#include "mtp_common.cuh"
#include "mtp_rowattn.cuh"

namespace mtp {
namespace rope {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;

struct Args {
  const void* x[3];       // q, k, v: last dimension contiguous
  int64_t sb[3], ss[3], sh[3];  // element strides of (b, s, h)
  const int32_t* positions;  // [B, S]; null: start[b] + s
  const float* cos;          // [max_pos, half]
  const float* sin;
  int64_t max_pos;
  int half;  // R / 2
  const void* w[2];  // q, k norm weights [D], nullable
  int w_dtype[2];
  float eps;
  int normalise, interleaved;
  void* q_out;  // [B, S, Hq, D]
  void* k_out;  // [B, Hkv, S, D]; null in the paged form
  void* pages[2];  // k, v pools [P, B, Hkv, page_size, D]
  const int32_t* page_table;
  int64_t table_stride, num_pages, page_size;
  const int32_t* start;  // [B], paged form
  const int32_t* count;  // [B] or null
  int B, S, Hq, Hkv, D, dtype;
  int tokens;  // per block (power of two)
};

// Where token s of sequence b goes and how it is turned.
struct Token {
  bool live;      // rotate and write; a token that is not live gets a zero query
  int64_t pos;    // row of cos/sin
  int64_t page;   // paged form: -1 = nothing is written to the pool
  int64_t slot;
};

__device__ __forceinline__ Token locate(const Args& a, int b, int s, bool report) {
  Token t;
  t.page = -1;
  t.slot = 0;
  const int n = a.count ? min(a.count[b], a.S) : a.S;
  t.live = s < n;
  const int64_t logical = a.start ? (int64_t)a.start[b] + s : 0;
  t.pos = a.positions ? (int64_t)a.positions[(int64_t)b * a.S + s] : logical;
  if (!t.live) return t;
  bool bad = false;
  if (a.page_table) {
    if (logical >= 0 && logical < a.table_stride) {
      t.page = resolve_page(a.page_table[b * a.table_stride + logical], a.num_pages);
      t.slot = logical % a.page_size;
    }
    bad = t.page < 0;
  }
  if (t.pos < 0 || t.pos >= a.max_pos) {
    bad = true;
    t.live = false;
    t.page = -1;
  }
  if (bad && report) record_error(MTP_ERR_DEVICE);
  return t;
}

// Whether a later token of this call lands in the same (page, slot): the later
// one stays, as in paged_kv_write.  Tokens share a slot only if they are a
// multiple of page_size apart.  m = 1, 2, ... counts those multiples.
__device__ __forceinline__ bool overtaken(const Args& a, int b, int s, int64_t page, int64_t m0, int64_t step) {
  const int n = a.count ? min(a.count[b], a.S) : a.S;
  const int32_t* row = a.page_table + b * a.table_stride;
  const int64_t start = a.start[b];
  bool later = false;
  for (int64_t t = s + m0 * a.page_size; t < n && start + t < a.table_stride; t += step * a.page_size) {
    // a later token whose position is outside the tables writes nothing
    const int64_t pos = a.positions ? (int64_t)a.positions[(int64_t)b * a.S + t] : start + t;
    later |= pos >= 0 && pos < a.max_pos && resolve_page(row[start + t], a.num_pages) == page;
  }
  return later;
}

// Destination of head h (0 .. Hq-1 queries, then keys, then values) of a token; null: not written.
__device__ __forceinline__ int64_t out_offset(const Args& a, int kind, int h, int b, int s, const Token& t) {
  if (kind == 0) return (((int64_t)b * a.S + s) * a.Hq + h) * a.D;
  if (a.k_out) return (((int64_t)b * a.Hkv + h) * a.S + s) * a.D;
  return ((((int64_t)t.page * a.B + b) * a.Hkv + h) * a.page_size + t.slot) * a.D;
}

template <typename T>
struct Vec8;  // 8 values as 16-byte words
template <>
struct Vec8<float> {
  uint4 u[2];
};
template <>
struct Vec8<__nv_bfloat16> {
  uint4 u[1];
};
template <>
struct Vec8<__half> {
  uint4 u[1];
};

template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> v;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(v) / 16); ++i) v.u[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return v;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Vec8<T>& v) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(v) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = v.u[i];
}

// LPH lanes per head (D <= 8 LPH); every base and stride a multiple of 16 bytes,
// half a multiple of 8 (of 4 when interleaved).
template <typename T, int LPH, bool INTER>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(Args a) {
  constexpr int kGroups = kThreads / LPH;
  __shared__ int s_over[kGroups];
  const int grp = threadIdx.x / LPH, c = threadIdx.x % LPH;
  const int tok = grp % a.tokens;
  const int per_seq = (a.S + a.tokens - 1) / a.tokens;
  const int b = blockIdx.x / per_seq;
  const int s = (blockIdx.x % per_seq) * a.tokens + tok;
  const bool in = s < a.S;
  Token t{};
  t.page = -1;
  if (in) t = locate(a, b, s, grp < a.tokens && c == 0 && blockIdx.y == 0);
  const bool paged = a.page_table != nullptr;
  if (paged && a.S > a.page_size) {  // block-uniform
    if (threadIdx.x < a.tokens) s_over[threadIdx.x] = 0;
    __syncthreads();
    const int ct = threadIdx.x % a.tokens;  // neighbouring threads look at neighbouring columns
    const int cs = (blockIdx.x % per_seq) * a.tokens + ct;
    if (cs < a.S) {
      const Token mine = locate(a, b, cs, false);
      if (mine.page >= 0 &&
          overtaken(a, b, cs, mine.page, 1 + threadIdx.x / a.tokens, kThreads / a.tokens))
        s_over[ct] = 1;
    }
    __syncthreads();
    if (s_over[tok]) t.page = -1;
  }

  const int d0 = c * 8;
  const bool active = d0 < a.D;
  const int R = 2 * a.half;
  const bool turn = active && d0 < R;
  // cos/sin of this lane's values; a value outside the rotation keeps itself
  float cs[INTER ? 4 : 8], sn[INTER ? 4 : 8];
  constexpr int kN = INTER ? 4 : 8;
  {
    const int i0 = INTER ? d0 / 2 : (d0 < a.half ? d0 : d0 - a.half);
    const bool need = in && t.live && turn;
    const float* cp = a.cos + (need ? t.pos : 0) * a.half + (need ? i0 : 0);
    const float* sp = a.sin + (need ? t.pos : 0) * a.half + (need ? i0 : 0);
#pragma unroll
    for (int i = 0; i < kN; i += 4) {
      const float4 u = need ? __ldg(reinterpret_cast<const float4*>(cp + i)) : make_float4(1.f, 1.f, 1.f, 1.f);
      const float4 w = need ? __ldg(reinterpret_cast<const float4*>(sp + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
      cs[i] = u.x, cs[i + 1] = u.y, cs[i + 2] = u.z, cs[i + 3] = u.w;
      sn[i] = w.x, sn[i + 1] = w.y, sn[i + 2] = w.z, sn[i + 3] = w.w;
    }
  }
  // lane of the partner values of a split pair; the sign of its term
  const int partner = turn ? (d0 < a.half ? c + a.half / 8 : c - a.half / 8) : c;
  const float sign = d0 < a.half ? -1.f : 1.f;
  float wq[8], wk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    wq[i] = a.w[0] && active ? load_f32(a.w[0], a.w_dtype[0], d0 + i) : 1.f;
    wk[i] = a.w[1] && active ? load_f32(a.w[1], a.w_dtype[1], d0 + i) : 1.f;
  }
  const float inv_d = 1.0f / (float)a.D;

  const int heads = a.Hq + a.Hkv + (paged ? a.Hkv : 0);
  const int step = (kGroups / a.tokens) * gridDim.y;
  // the loop bound is the same for every group of a warp, so its shuffles stay converged
  for (int base = (kGroups / a.tokens) * blockIdx.y; base < heads; base += step * kUnroll) {
    Vec8<T> x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int hh = base + u * step + grp / a.tokens;
      const int kind = hh < a.Hq ? 0 : (hh < a.Hq + a.Hkv ? 1 : 2);
      const int h = kind == 0 ? hh : (kind == 1 ? hh - a.Hq : hh - a.Hq - a.Hkv);
      const bool go = in && active && t.live && hh < heads && (kind == 0 || !paged || t.page >= 0);
#pragma unroll
      for (int i = 0; i < (int)(sizeof(Vec8<T>) / 16); ++i) x[u].u[i] = make_uint4(0, 0, 0, 0);
      if (go)
        x[u] = load8(static_cast<const T*>(a.x[kind]) + b * a.sb[kind] + s * a.ss[kind] + h * a.sh[kind] + d0);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (base + u * step >= heads) break;  // block-uniform
      const int hh = base + u * step + grp / a.tokens;
      const int kind = hh < a.Hq ? 0 : (hh < a.Hq + a.Hkv ? 1 : 2);
      const int h = kind == 0 ? hh : (kind == 1 ? hh - a.Hq : hh - a.Hq - a.Hkv);
      const T* xe = reinterpret_cast<const T*>(&x[u]);
      float y[8];
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = rowattn::to_f32(xe[i]);
        sq = fmaf(y[i], y[i], sq);
      }
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o, LPH);
      const float rstd = a.normalise ? 1.0f / sqrtf(sq * inv_d + a.eps) : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * rstd * (kind == 0 ? wq[i] : wk[i]);
      Vec8<T> o;
      T* oe = reinterpret_cast<T*>(&o);
      if constexpr (INTER) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = y[2 * i], r = y[2 * i + 1];
          oe[2 * i] = rowattn::from_f32<T>(turn ? p * cs[i] - r * sn[i] : p);
          oe[2 * i + 1] = rowattn::from_f32<T>(turn ? r * cs[i] + p * sn[i] : r);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float other = __shfl_sync(0xffffffffu, y[i], partner, LPH);
          oe[i] = rowattn::from_f32<T>(turn ? y[i] * cs[i] + sign * (other * sn[i]) : y[i]);
        }
      }
      if (!in || !active || hh >= heads) continue;
      if (kind == 2) o = x[u];
      if (!t.live) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(Vec8<T>) / 16); ++i) o.u[i] = make_uint4(0, 0, 0, 0);
      }
      if (kind != 0 && paged && t.page < 0) continue;
      void* dst = kind == 0 ? a.q_out : (a.k_out ? a.k_out : a.pages[kind - 1]);
      store8(static_cast<T*>(dst) + out_offset(a, kind, h, b, s, t) + d0, o);
    }
  }
}

// Every other shape (head sizes, strides or rotations that do not come in 16
// bytes): one warp per (token, head), value by value.
__global__ void __launch_bounds__(kThreads) qk_norm_rope_any_kernel(Args a) {
  const bool paged = a.page_table != nullptr;
  const int heads = a.Hq + a.Hkv + (paged ? a.Hkv : 0);
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= (int64_t)a.B * a.S * heads) return;
  const int hh = (int)(row % heads);
  const int s = (int)(row / heads % a.S);
  const int b = (int)(row / ((int64_t)heads * a.S));
  Token t = locate(a, b, s, hh == 0 && lane == 0);
  const int kind = hh < a.Hq ? 0 : (hh < a.Hq + a.Hkv ? 1 : 2);
  const int h = kind == 0 ? hh : (kind == 1 ? hh - a.Hq : hh - a.Hq - a.Hkv);
  if (paged && kind != 0) {
    if (t.page < 0) return;
    if (__any_sync(0xffffffffu, overtaken(a, b, s, t.page, 1 + lane, 32))) return;
  }
  void* dst = kind == 0 ? a.q_out : (a.k_out ? a.k_out : a.pages[kind - 1]);
  const int64_t off = out_offset(a, kind, h, b, s, t);
  if (!t.live) {
    for (int d = lane; d < a.D; d += 32) store_f32(dst, a.dtype, off + d, 0.f);
    return;
  }
  const int64_t src = b * a.sb[kind] + s * a.ss[kind] + h * a.sh[kind];
  if (kind == 2) {
    for (int d = lane; d < a.D; d += 32) store_f32(dst, a.dtype, off + d, load_f32(a.x[2], a.dtype, src + d));
    return;
  }
  float sq = 0.f;
  for (int d = lane; d < a.D; d += 32) {
    const float v = load_f32(a.x[kind], a.dtype, src + d);
    sq = fmaf(v, v, sq);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
  const float rstd = a.normalise ? 1.0f / sqrtf(sq / (float)a.D + a.eps) : 1.0f;
  auto value = [&](int d) {
    const float w = a.w[kind] ? load_f32(a.w[kind], a.w_dtype[kind], d) : 1.f;
    return load_f32(a.x[kind], a.dtype, src + d) * rstd * w;
  };
  const float* cp = a.cos + t.pos * a.half;
  const float* sp = a.sin + t.pos * a.half;
  for (int d = lane; d < a.D; d += 32) {
    float y = value(d);
    if (d < 2 * a.half) {
      const int i = a.interleaved ? d / 2 : (d < a.half ? d : d - a.half);
      const bool first = a.interleaved ? (d & 1) == 0 : d < a.half;
      const float other = value(a.interleaved ? (d ^ 1) : (first ? d + a.half : d - a.half));
      y = first ? y * cp[i] - other * sp[i] : y * cp[i] + other * sp[i];
    }
    store_f32(dst, a.dtype, off + d, y);
  }
}

}  // namespace rope
}  // namespace mtp
