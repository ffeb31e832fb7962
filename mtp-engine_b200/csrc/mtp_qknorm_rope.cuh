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
// over LPH = 4, 8 or 16 lanes with two 16-byte pieces each; the sum of squares
// is a shuffle over them.  A group of LPH lanes stays with one token and walks
// over its heads, so cos, sin and the weights are loaded once into registers
// and serve all of them.  Measured (B200): four prompts of 2500 .. 4093 tokens, 32
// query and 8 key heads of 128, bf16, into the pool (352 MB): 76 us, 4.6 TB/s =
// 0.71 of the measured copy rate; the 1024 tokens of 16 draft trees 13 us cold.
#pragma once

#include "mtp_common.cuh"
#include "mtp_rowattn.cuh"

namespace mtp {
namespace rope {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // heads whose loads are in flight (2: 84 us on four ragged prompts, 4: 76 us)

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
  int w_vec[2];  // weights of the data's type on 16 bytes
  float eps;
  int normalise, interleaved;
  void* q_out;  // [B, S, Hq, D]
  void* k_out;  // [B, Hkv, S, D]; null in the paged form
  void* pages[2];  // k, v pools [P, B, Hkv, page_size, D]
  const int32_t* page_table;
  int64_t table_stride, num_pages;
  int page_size;
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
  int slot;
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
      t.slot = (int)((uint32_t)logical % (uint32_t)a.page_size);
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
// multiple of page_size apart; this thread looks at the multiples m0, m0 +
// step, ..., four at a time.  S^2 / (2 page_size) reads of the table per
// sequence: little up to some 10^4 tokens a call, the larger part beyond (one
// key head of 128, pages of 8: 4096 tokens 22 us, 32768 182 us, 131072 2.3 ms;
// pages of 64: 18, 66 and 440 us).
__device__ __forceinline__ bool overtaken(const Args& a, int b, int s, int64_t page, int m0, int step) {
  const int n = a.count ? min(a.count[b], a.S) : a.S;
  const int start = a.start[b];
  const int last = (int)min((int64_t)n, a.table_stride - start);  // tokens that have a column
  const int32_t* row = a.page_table + b * a.table_stride + start;
  const int32_t* pos = a.positions ? a.positions + (int64_t)b * a.S : nullptr;
  bool later = false;
  for (int64_t t = s + (int64_t)m0 * a.page_size; t < last; t += 4ll * step * a.page_size) {
    int32_t id[4];
    int64_t p[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t x = t + (int64_t)u * step * a.page_size;
      id[u] = x < last ? row[x] : INT32_MIN;
      p[u] = x < last ? (pos ? (int64_t)pos[x] : start + x) : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)  // a later token whose position is outside the tables writes nothing
      later |= p[u] >= 0 && p[u] < a.max_pos && resolve_page(id[u], a.num_pages) == page;
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
struct Vec8 {  // 8 values as 16-byte words
  uint4 u[sizeof(T) / 2];
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

template <typename T>
__device__ __forceinline__ void unpack(const Vec8<T>& v, float (&f)[8]) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = rowattn::to_f32(e[i]);
}
__device__ __forceinline__ void pack(const float (&f)[8], Vec8<float>& v) {
  v.u[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  v.u[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
}
__device__ __forceinline__ void pack(const float (&f)[8], Vec8<__nv_bfloat16>& v) {
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void pack(const float (&f)[8], Vec8<__half>& v) {
  __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
}

// two fp32 operations in one instruction
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0,
                                     float c1) {
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mul2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

// 1 / sqrt(x): the approximation and one Newton step, r (3 - x r^2) / 2
__device__ __forceinline__ float inv_sqrt(float x) {
  const float r = rsqrtf(x);
  const float e = fmaf(-x * r, r, 1.0f);
  return x > 0.f && x < INFINITY ? fmaf(0.5f * r, e, r) : r;
}

// LPH lanes per head (D <= 16 LPH); every base and stride a multiple of 16 bytes,
// half a multiple of 8 (of 4 when interleaved).
//
// A lane holds two pieces of 8 values: X and, half a rotation further, Y, so
// that both values of a split pair are its own (the pieces behind the rotation,
// and all pieces when interleaved, are neighbours).  With the weight w and the
// pair's other value x', a value becomes
//   y = rstd * (x * A + x' * B),   A = w cos,  B = -+ w' sin
// so A and B (16 + 16 registers, once per token and norm) leave three fp32
// operations per value in the loop over the heads.  A value outside the
// rotation has A = w and no second term.
template <typename T, int LPH, bool INTER>
__global__ void __launch_bounds__(kThreads, 2) qk_norm_rope_kernel(Args a) {
  constexpr int kGroups = kThreads / LPH;
  __shared__ int s_over[kGroups];
  const int grp = threadIdx.x / LPH, c = threadIdx.x % LPH;
  const int tok = grp % a.tokens;
  const int64_t id = (int64_t)blockIdx.x * a.tokens + tok;  // tokens of all sequences in one line
  const bool in = id < (int64_t)a.B * a.S;
  const int b = in ? (int)(id / a.S) : 0, s = in ? (int)(id - (int64_t)b * a.S) : 0;
  Token t{};
  t.page = -1;
  if (in) t = locate(a, b, s, grp < a.tokens && c == 0 && blockIdx.y == 0);
  const bool paged = a.page_table != nullptr;
  const bool shared_slots = paged && a.S > a.page_size;  // two tokens of the call may share a slot
  if (shared_slots) {
    if (threadIdx.x < a.tokens) s_over[threadIdx.x] = 0;
    __syncthreads();
    if (t.page >= 0 && overtaken(a, b, s, t.page, 1 + grp / a.tokens * LPH + c, kThreads / a.tokens))
      s_over[tok] = 1;
  }

  const int turned = a.half / 8;  // split pairs: lanes that hold some
  const bool split_pair = !INTER && c < turned;
  int d[2];  // first value of X and Y
  d[0] = split_pair ? 8 * c : (INTER ? 16 * c : 2 * a.half + 16 * (c - turned));
  d[1] = split_pair ? d[0] + a.half : d[0] + 8;
  const bool active[2] = {d[0] < a.D, d[1] < a.D};
  bool turn[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) turn[p] = INTER ? d[p] < 2 * a.half : split_pair;
  float cs[8], sn[8];  // split: of the 8 pairs; interleaved: 4 pairs of X, 4 of Y
  {
    const bool go = in && t.live;
    const int64_t row = go ? t.pos * a.half : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool need = go && turn[INTER ? i : 0];
      const int64_t at = need ? row + (INTER ? d[i] / 2 : d[0] + 4 * i) : 0;
      const float4 u = need ? __ldg(reinterpret_cast<const float4*>(a.cos + at)) : make_float4(1.f, 1.f, 1.f, 1.f);
      const float4 w = need ? __ldg(reinterpret_cast<const float4*>(a.sin + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
      cs[4 * i] = u.x, cs[4 * i + 1] = u.y, cs[4 * i + 2] = u.z, cs[4 * i + 3] = u.w;
      sn[4 * i] = w.x, sn[4 * i + 1] = w.y, sn[4 * i + 2] = w.z, sn[4 * i + 3] = w.w;
    }
  }
  const float inv_d = 1.0f / (float)a.D;

  const int slots = kGroups / a.tokens;  // heads of a token that the block has under way
  const int step = slots * gridDim.y, slot = grp / a.tokens + slots * blockIdx.y;
  // heads of a kind that follow `before` others, dealt out round robin over all of them
  auto first_of = [&](int before) {
    const int r = (slot - before) % step;
    return r < 0 ? r + step : r;
  };

#pragma unroll 1
  for (int kind = 0; kind < 2; ++kind) {
    const int H = kind == 0 ? a.Hq : a.Hkv;
    if (kind == 1 && shared_slots) {
      __syncthreads();
      if (s_over[tok]) t.page = -1;
    }
    float A[2][8], Bm[2][8];
    {
      float w[2][8];
      const void* wp = a.w[kind];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        if (wp == nullptr || !active[p]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[p][i] = 1.f;
        } else if (a.w_vec[kind]) {
          unpack(load8(static_cast<const T*>(wp) + d[p]), w[p]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[p][i] = load_f32(wp, a.w_dtype[kind], d[p] + i);
        }
      }
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float wo = INTER ? w[p][i ^ 1] : w[p ^ 1][i];
          const float co = INTER ? cs[4 * p + i / 2] : cs[i], si = INTER ? sn[4 * p + i / 2] : sn[i];
          const bool first = INTER ? (i & 1) == 0 : p == 0;
          A[p][i] = turn[p] ? w[p][i] * co : w[p][i];
          Bm[p][i] = turn[p] ? (first ? -wo * si : wo * si) : 0.f;
        }
    }
    const int h0 = first_of(kind == 0 ? 0 : a.Hq);
    const T* src = static_cast<const T*>(a.x[kind]) + b * a.sb[kind] + s * a.ss[kind] + h0 * a.sh[kind];
    const int64_t src_step = step * a.sh[kind];
    void* out = kind == 0 ? a.q_out : (paged ? a.pages[0] : a.k_out);
    T* dst = static_cast<T*>(out) + out_offset(a, kind, h0, b, s, t);
    const int64_t dst_step = kind == 0 ? (int64_t)step * a.D : (int64_t)step * a.D * (paged ? a.page_size : a.S);
    const bool reads = in && t.live, writes = in && (kind == 0 || !paged || t.page >= 0);
    const int left = h0 < H ? (H - h0 + step - 1) / step : 0;  // heads of this group
    const int iters = (H + step - 1) / step;                   // the same for every lane: the shuffles stay converged
#pragma unroll 1
    for (int i = 0; i < iters; i += kUnroll) {
      Vec8<T> x[kUnroll][2];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
          for (int k = 0; k < (int)(sizeof(Vec8<T>) / 16); ++k) x[u][p].u[k] = make_uint4(0, 0, 0, 0);
          if (reads && active[p] && i + u < left) x[u][p] = load8(src + d[p]);
        }
        src += src_step;
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (i + u >= iters) break;
        float y[2][8];
        unpack(x[u][0], y[0]);
        unpack(x[u][1], y[1]);
        float sq0 = 0.f, sq1 = 0.f;
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int k = 0; k < 8; k += 2) fma2(sq0, sq1, y[p][k], y[p][k + 1], y[p][k], y[p][k + 1], sq0, sq1);
        float sq = sq0 + sq1;
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o, LPH);
        const float rstd = a.normalise ? inv_sqrt(fmaf(sq, inv_d, a.eps)) : 1.0f;
        float z[2][8];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            // outside the rotation the other value is not looked at
            const float o0 = INTER ? y[p][k + 1] : y[p ^ 1][k], o1 = INTER ? y[p][k] : y[p ^ 1][k + 1];
            mul2(z[p][k], z[p][k + 1], turn[p] ? o0 : 0.f, turn[p] ? o1 : 0.f, Bm[p][k], Bm[p][k + 1]);
            fma2(z[p][k], z[p][k + 1], y[p][k], y[p][k + 1], A[p][k], A[p][k + 1], z[p][k], z[p][k + 1]);
            mul2(z[p][k], z[p][k + 1], z[p][k], z[p][k + 1], rstd, rstd);
          }
        if (writes && i + u < left) {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            Vec8<T> o;
            pack(z[p], o);
            if (!t.live) {
#pragma unroll
              for (int k = 0; k < (int)(sizeof(Vec8<T>) / 16); ++k) o.u[k] = make_uint4(0, 0, 0, 0);
            }
            if (active[p]) store8(dst + d[p], o);
          }
        }
        dst += dst_step;
      }
    }
  }
  if (!paged || !in || t.page < 0) return;
  // values: copied
  const int h0 = first_of(a.Hq + a.Hkv);
  const T* src = static_cast<const T*>(a.x[2]) + b * a.sb[2] + s * a.ss[2];
  T* dst = static_cast<T*>(a.pages[1]) + out_offset(a, 2, 0, b, s, t);
#pragma unroll 2
  for (int h = h0; h < a.Hkv; h += step)
#pragma unroll
    for (int p = 0; p < 2; ++p)
      if (active[p]) store8(dst + (int64_t)h * a.page_size * a.D + d[p], load8(src + h * a.sh[2] + d[p]));
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
  const float rstd = a.normalise ? inv_sqrt(sq / (float)a.D + a.eps) : 1.0f;
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
