// mtp_splitattn.cuh -- attention of few query rows over a long paged cache:
// one new token per sequence (decode), or a handful of new tokens, with
// grouped-query heads, ragged lengths, a sliding window and first tokens
// ("sinks") that stay visible.
//
// Row s of sequence b (s < n_b new tokens, len_b tokens in all) sits at
// position p = len_b - n_b + s and sees key j iff j <= p and (j > p - window or
// j < sinks).  out = sum_j exp(q k_j scale - m) v_j / sum_j exp(q k_j scale - m).
//
// HBM-bound: every visible K and V row is read once per key head and serves
// the G = Hq/Hkv query heads that share it.  The 16 rows of an m16n8k16 tile
// hold them (G S <= 16 as a rule; more rows are further tiles), which takes the
// dot products off the CUDA cores: at G = 8 those would need 1.4x their
// peak to keep up with HBM.  The tensor work is ~2 % of what the memory
// allows, so the warp-level instructions serve as well as tcgen05 tiles of 128
// rows would (7/8 of them empty) and need no hand-over between warps.
//
// Work is cut into blocks of 16 keys over all (sequence, row tile, key head)
// units in one line, and every warp takes an equal, contiguous piece of it,
// whatever the lengths: a warp runs its blocks through its own ring of
// asynchronous 16-byte copies (kStages x 16 keys of K and V in flight), keeps
// the running maximum, sum and output in registers and meets no barrier.  A
// unit that one warp covered is written out at once; pieces of a unit that
// several warps share go to the workspace as (output, maximum, sum) and
// split_merge_kernel joins them in a fixed order.
//
// Keys that no row of the unit sees are not read: the visible keys are
// numbered 0 .. nvis-1 (first the sinks below the window, then the window), so
// blocks hold visible keys only; places past the last one are zero-filled.
//
// Measured (B200): 16 sequences of 1 .. 32768 tokens, Hq 32, Hkv 8, D 128, bf16
// (1.08 GB) 205 us, 5.2 TB/s = 0.80 of the measured copy rate; one sequence of
// 4096 tokens 16 us with both launches; 8 sequences of 9001 .. 16000 tokens, Hq
// 40, f16, with key weights 106 us, of which the scores' second pass takes 13.
//
// Many row tiles (prompts whose head size the 128-row tiles do not take) are
// served, not fast: K and V are read once per 16 rows, and every warp, and every
// block of the join, goes through all (sequence, row tile) pairs to find its
// place.  2048 new tokens, Hq 32, Hkv 8: 2.75 ms at D 256, 1.62 ms at D 56,
// where the 128-row tiles take 0.055 ms at D 128.
#pragma once

#include <type_traits>

#include "mtp_common.cuh"
#include "mtp_rowattn.cuh"

namespace mtp {
namespace split {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 16;   // keys per block
constexpr int kRows = 16;   // query rows per tile
constexpr int kStages = 3;  // blocks in flight per warp
constexpr int kMergeWarps = 8;

struct Args {
  const void* q;  // [B, S, Hq, D]
  void* out;
  const void* k_pages;  // [P, B, Hkv, page_size, D]
  const void* v_pages;
  const int32_t* page_table;  // [B, table_stride]
  int64_t table_stride, num_pages, page_size;
  const int32_t* seq_lens;  // [B]
  const int32_t* q_lens;    // [B]; null: S each (decode: the one token of every non-empty sequence)
  int B, S, Hq, Hkv, G, D, dtype;
  int window;  // 2^30: everything
  int sinks;
  float scale_log2;  // softmax scale * log2(e)
  int row_tiles;    // ceil(S * G / kRows)
  int max_warps;    // warps of the launch
  int min_blocks;   // least blocks a warp takes
  float* part_o;    // [2 * max_warps][kRows][D]
  float* part_ml;   // [2 * max_warps][kRows][2]
  // key weights (S == 1): raw scores and each row's (maximum, 1 / sum), in log2 units
  float* scores;    // [B, Hq, score_ld]
  int64_t score_ld;
  float* row_ml;    // [B, Hq, 2]
  float* key_weights;  // [B, Hkv, weight_ld]
  int64_t weight_ld;
};

struct Seq {
  int len, n;
};

// Lengths as the caller's device arrays give them, forced into range (an entry
// outside it is recorded once, by the caller that passes report).
__device__ __forceinline__ Seq lengths(const int32_t* seq_lens, const int32_t* q_lens, int64_t table_stride, int S,
                                       int b, bool report = false) {
  const int len = __ldg(seq_lens + b);
  const int cap = (int)min(table_stride, (int64_t)INT32_MAX);
  Seq s;
  s.len = max(0, min(len, cap));
  const int n = q_lens ? __ldg(q_lens + b) : min(S, s.len);
  s.n = max(0, min(n, min(S, s.len)));
  if (report && (s.len != len || s.n != n)) record_error(MTP_ERR_DEVICE);
  return s;
}

__device__ __forceinline__ Seq sequence(const Args& a, int b, bool report = false) {
  return lengths(a.seq_lens, a.q_lens, a.table_stride, a.S, b, report);
}

// Visible keys of rows s0 .. s1 of a sequence: numbers [0, sinks) are the keys
// below the window, the others lo, lo + 1, ...
struct Span {
  int lo, sinks, nvis;
  __device__ __forceinline__ int key(int v) const { return v < sinks ? v : v - sinks + lo; }
};

__device__ __forceinline__ Span span_of(const Seq& q, int s0, int s1, int window, int sinks) {
  Span r;
  const int first = q.len - q.n + s0, last = q.len - q.n + s1;
  r.lo = max(0, first - window + 1);
  r.sinks = min(sinks, r.lo);
  r.nvis = r.sinks + last + 1 - r.lo;
  return r;
}

// (sequence, row tile) pair `pr`: its valid rows and visible keys
struct Tile {
  int b, row0, rows;  // rows row0 .. row0 + rows - 1 of the sequence's n * G
  Seq q;
  Span sp;
};

__device__ __forceinline__ Tile tile_of(const Args& a, int pr, bool report = false) {
  Tile t;
  t.b = pr / a.row_tiles;
  t.row0 = (pr % a.row_tiles) * kRows;
  t.q = sequence(a, t.b, report && t.row0 == 0);
  t.rows = max(0, min(kRows, t.q.n * a.G - t.row0));
  t.sp.lo = t.sp.sinks = t.sp.nvis = 0;
  if (t.rows > 0) t.sp = span_of(t.q, t.row0 / a.G, (t.row0 + t.rows - 1) / a.G, a.window, a.sinks);
  return t;
}

__device__ __forceinline__ int blocks_of(const Tile& t) { return (t.sp.nvis + kKeys - 1) / kKeys; }

// One line of blocks: pair by pair, key head by key head.  find_block() is called
// by a whole warp: total blocks, and where the asked block lies (pair, blocks of the
// line before the pair).
struct Line {
  int64_t total;
  int pair;
  int64_t before;
};

template <typename Pick>  // total blocks -> the block to find
__device__ __forceinline__ Line find_block(const Args& a, Pick pick) {
  const int lane = threadIdx.x & 31;
  const int pairs = a.B * a.row_tiles;
  Line r;
  r.total = 0;
  for (int p0 = 0; p0 < pairs; p0 += 32) {
    int64_t n = p0 + lane < pairs ? (int64_t)blocks_of(tile_of(a, p0 + lane)) * a.Hkv : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    r.total += n;
  }
  const int64_t at = pick(r.total);
  r.pair = pairs;
  r.before = 0;
  int64_t sum = 0;
  for (int p0 = 0; p0 < pairs; p0 += 32) {
    int64_t n = p0 + lane < pairs ? (int64_t)blocks_of(tile_of(a, p0 + lane)) * a.Hkv : 0;
    const int64_t own = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, sum + n > at);
    if (hit) {
      const int l = __ffs(hit) - 1;
      r.pair = p0 + l;
      r.before = sum + __shfl_sync(0xffffffffu, n - own, l);
      break;
    }
    sum += __shfl_sync(0xffffffffu, n, 31);
  }
  return r;
}

__host__ __device__ __forceinline__ int64_t warps_used(int64_t total, int max_warps, int min_blocks) {
  const int64_t w = total / min_blocks;
  return w < 1 ? 1 : (w > max_warps ? max_warps : w);
}
__host__ __device__ __forceinline__ int64_t piece_start(int64_t total, int64_t warps, int64_t w) {
  return w * total / warps;
}
// the warp whose piece holds block `at`: the largest w with piece_start(w) <= at
__host__ __device__ __forceinline__ int64_t piece_owner(int64_t total, int64_t warps, int64_t at) {
  return ((at + 1) * warps + total - 1) / total - 1;
}

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <>
struct Mma<__half> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr int stage_bytes(int dp) { return 2 * kKeys * dp * 2; }  // K and V rows of one block
constexpr int smem_bytes(int dp) { return kWarps * kStages * stage_bytes(dp); }

// Walks the blocks of the line: (pair, key head, block).
struct Cursor {
  Tile t;
  int pair, hk, blk, nblk;
  __device__ __forceinline__ void set(const Args& a, int pair_, int64_t rest) {
    pair = pair_;
    t = tile_of(a, pair);
    nblk = blocks_of(t);
    hk = (int)(rest / nblk);
    blk = (int)(rest % nblk);
  }
  // to the next block; the caller knows that there is one
  __device__ __forceinline__ void next(const Args& a) {
    if (++blk < nblk) return;
    blk = 0;
    if (++hk < a.Hkv) return;
    hk = 0;
    do {
      t = tile_of(a, ++pair);
      nblk = blocks_of(t);
    } while (nblk == 0);
  }
};

// Pool row (page, b, head, slot) of the cursor's key `lane` (lanes 0 .. 15); -1:
// past the visible keys, or a page id outside the pool (recorded).
__device__ __forceinline__ int pool_row(const Args& a, const Cursor& c, int lane) {
  const int v = c.blk * kKeys + lane;
  if (lane >= kKeys || v >= c.t.sp.nvis) return -1;
  const int j = c.t.sp.key(v);
  const int64_t pg = resolve_page(__ldg(a.page_table + c.t.b * a.table_stride + j), a.num_pages);
  if (pg < 0) {
    record_error(MTP_ERR_DEVICE);
    return -1;
  }
  return (int)(((pg * a.B + c.t.b) * a.Hkv + c.hk) * a.page_size + j % a.page_size);
}

// DP: the head size the tiles are built for (D <= DP; dimensions past D are
// zero).  MANY: rows at several positions (S > 1), each with its own last key.
template <typename T, int DP, bool MANY>
__global__ void __launch_bounds__(kThreads) split_attention_kernel(Args a) {
  constexpr int kChunks = DP / 8;          // 16-byte pieces of a row
  constexpr int kRowsPerCopy = 32 / kChunks;
  constexpr int kPitch = DP * 2;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kWarps + warp;
  uint8_t* ring = smem + warp * (kStages * stage_bytes(DP));
  // the joining kernel may be set up on SMs that run out of blocks; it waits for this one's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t ring_addr = smem_u32(ring);

  const Line line = find_block(a, [&](int64_t total) {
    const int64_t n = warps_used(total, a.max_warps, a.min_blocks);
    return w < n ? piece_start(total, n, w) : total;
  });
  const int64_t used = warps_used(line.total, a.max_warps, a.min_blocks);
  if (w == 0)  // once per launch: lengths outside their range
    for (int b = lane; b < a.B; b += 32) sequence(a, b, true);
  if (line.total == 0 || w >= used) return;
  const int64_t begin = piece_start(line.total, used, w), end = piece_start(line.total, used, w + 1);
  if (begin >= end) return;
  const int count = (int)(end - begin);

  const int D = a.D;
  if (D < DP) {  // dimensions past D: zero once, never copied over
    for (int i = lane; i < kStages * stage_bytes(DP) / 16; i += 32)
      reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }

  Cursor ahead, cur;
  ahead.set(a, line.pair, begin - line.before);
  cur = ahead;
  const uint8_t* kp = static_cast<const uint8_t*>(a.k_pages);
  const uint8_t* vp = static_cast<const uint8_t*>(a.v_pages);
  const int piece = lane % kChunks, sub = lane / kChunks;
  const bool piece_ok = piece * 8 < D;
  auto issue = [&](int stage, int row_of_lane) {
    const uint32_t base = ring_addr + stage * stage_bytes(DP);
#pragma unroll
    for (int i = 0; i < kKeys / kRowsPerCopy; ++i) {
      const int r = i * kRowsPerCopy + sub;
      const int row = __shfl_sync(0xffffffffu, row_of_lane, r);
      const int64_t off = row >= 0 ? (int64_t)row * D * 2 + piece * 16 : 0;
      const uint32_t dst = base + r * kPitch + (((piece & ~7) | ((piece ^ r) & 7)) << 4);
      if (piece_ok) {
        copy16(dst, kp + off, row >= 0 ? 16u : 0u);
        copy16(dst + kKeys * kPitch, vp + off, row >= 0 ? 16u : 0u);
      }
    }
  };

  // the first kStages blocks' page ids are read together, then all their copies start
  int rows[kStages];
  int issued = 0;
#pragma unroll
  for (int s = 0; s < kStages; ++s) {
    rows[s] = -1;
    if (s < count) {
      rows[s] = pool_row(a, ahead, lane);
      if (s + 1 < count) ahead.next(a);
    }
  }
#pragma unroll
  for (int s = 0; s < kStages; ++s) {
    if (s < count) issue(s, rows[s]);
    copy_commit();
  }
  issued = min(count, kStages);
  int next_rows = issued < count ? pool_row(a, ahead, lane) : -1;

  uint32_t qf[DP / 16][4];
  float o[DP / 8][4];
  float m[2], l[2];
  int row_pos[2];
  const int r0 = lane >> 2, cq = lane & 3;

  auto load_q = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = cur.t.row0 + r0 + 8 * i;
      const bool ok = r0 + 8 * i < cur.t.rows;
      const int s = r / a.G, g = r % a.G;
      row_pos[i] = cur.t.q.len - cur.t.q.n + s;
      const T* src = static_cast<const T*>(a.q) +
                     ((((int64_t)cur.t.b * a.S + s) * a.Hq) + (int64_t)cur.hk * a.G + g) * D + cq * 2;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d = k * 16 + h * 8;
          qf[k][i + 2 * h] = ok && d + cq * 2 < D ? __ldg(reinterpret_cast<const uint32_t*>(src + d)) : 0u;
        }
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  };
  load_q();
  int seg_first = cur.blk;  // first block of this warp's piece of the unit
  bool seg_starts = true;   // the piece begins where the warp begins

  for (int it = 0; it < count; ++it) {
    copy_wait<kStages - 1>();
    __syncwarp();
    const int stage = it % kStages;
    const uint32_t ka = ring_addr + stage * stage_bytes(DP);
    const uint32_t va = ka + kKeys * kPitch;
    // S = Q K^T: keys 0-7 in c[0], 8-15 in c[1]; even and odd steps of the
    // head dimension in chains of their own
    float c[2][2][4];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[e][n][i] = 0.f;
    {
      const int key = ((lane >> 4) << 3) + (lane & 7);
      const uint32_t row = ka + key * kPitch;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const int pc = k * 2 + ((lane >> 3) & 1);
        uint32_t b[4];
        ldsm4(row + (((pc & ~7) | ((pc ^ key) & 7)) << 4), b);
        Mma<T>::mma(c[k & 1][0], qf[k], b[0], b[1]);
        Mma<T>::mma(c[k & 1][1], qf[k], b[2], b[3]);
      }
    }
    const int left = cur.t.sp.nvis - cur.blk * kKeys;  // visible keys from this block on
    float s[2][4];  // [row][key 2cq, 2cq+1, 8+2cq, 8+2cq+1]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = e >> 1, kk = n * 8 + cq * 2 + (e & 1);
        float x = (c[0][n][2 * i + (e & 1)] + c[1][n][2 * i + (e & 1)]) * a.scale_log2;
        bool seen = kk < left;
        if (MANY && seen) {
          const int j = cur.t.sp.key(cur.blk * kKeys + kk);
          seen = j <= row_pos[i] && (j > row_pos[i] - a.window || j < a.sinks);
        }
        s[i][e] = seen ? x : -INFINITY;
      }
    if (!MANY && a.scores) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (r0 + 8 * i < cur.t.rows) {
          float* dst = a.scores + ((int64_t)cur.t.b * a.Hq + cur.hk * a.G + cur.t.row0 + r0 + 8 * i) * a.score_ld +
                       cur.blk * kKeys + cq * 2;
          *reinterpret_cast<float2*>(dst) = make_float2(s[i][0], s[i][1]);
          *reinterpret_cast<float2*>(dst + 8) = make_float2(s[i][2], s[i][3]);
        }
    }
    float alpha[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float mx = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[i], mx);
      const float use = mn == -INFINITY ? 0.f : mn;
      alpha[i] = exp2_fast(m[i] - use);  // m = -inf: 0
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = exp2_fast(s[i][e] - use);
        sum += s[i][e];
      }
      l[i] = l[i] * alpha[i] + sum;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        o[n][0] *= alpha[0];
        o[n][1] *= alpha[0];
        o[n][2] *= alpha[1];
        o[n][3] *= alpha[1];
      }
    }
    // O += P V, P rounded to the 16-bit type of V, which is what the tensor
    // cores take beside 16-bit values (the sum l keeps the unrounded weights).
    // Half a step of every weight: an error of at most half a step of
    // sum p |v| / l, on top of the output's own half step of |sum p v| / l.
    // The first is as large as the second or larger where values cancel; over
    // random values the two together are 1.1-1.2 times the second alone
    // (decode; 1.2-1.4 times for prompts).
    const uint32_t p[4] = {Mma<T>::pack(s[0][0], s[0][1]), Mma<T>::pack(s[1][0], s[1][1]),
                           Mma<T>::pack(s[0][2], s[0][3]), Mma<T>::pack(s[1][2], s[1][3])};
    {
      const int key = (((lane >> 3) & 1) << 3) + (lane & 7);
      const uint32_t row = va + key * kPitch;
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        const int pc = n * 2 + (lane >> 4);
        uint32_t b[4];
        ldsm4_t(row + (((pc & ~7) | ((pc ^ key) & 7)) << 4), b);
        Mma<T>::mma(o[2 * n], p, b[0], b[1]);
        Mma<T>::mma(o[2 * n + 1], p, b[2], b[3]);
      }
    }
    __syncwarp();  // every lane is done with the stage before it is filled again
    if (issued < count) {
      issue(stage, next_rows);
      ++issued;
      if (issued < count) {
        ahead.next(a);
        next_rows = pool_row(a, ahead, lane);
      }
    }
    copy_commit();

    const bool last_of_unit = cur.blk + 1 == cur.nblk, last = it + 1 == count;
    if (last_of_unit || last) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      }
      const bool whole = seg_first == 0 && last_of_unit;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = r0 + 8 * i;
        if (r >= cur.t.rows) continue;
        if (whole) {
          const int rr = cur.t.row0 + r, sq = rr / a.G, g = rr % a.G;
          const int64_t head = ((int64_t)cur.t.b * a.S + sq) * a.Hq + (int64_t)cur.hk * a.G + g;
          const float inv = l[i] > 0.f ? 1.0f / l[i] : 0.f;
          T* dst = static_cast<T*>(a.out) + head * D + cq * 2;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n)
            if (n * 8 < D)
              *reinterpret_cast<uint32_t*>(dst + n * 8) = Mma<T>::pack(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
          if (!MANY && a.scores && cq == 0) {
            a.row_ml[head * 2] = m[i];
            a.row_ml[head * 2 + 1] = inv;
          }
        } else {
          const int64_t slot = (2 * w + (seg_starts ? 0 : 1)) * kRows + r;
          float* dst = a.part_o + slot * D + cq * 2;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n)
            if (n * 8 < D) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
          if (cq == 0) {
            a.part_ml[slot * 2] = m[i];
            a.part_ml[slot * 2 + 1] = l[i];
          }
        }
      }
      if (!last) {
        cur.next(a);
        load_q();
        seg_first = 0;
        seg_starts = false;
      }
    } else {
      ++cur.blk;
    }
  }
  copy_wait<0>();
}

// Joins the pieces of the units that several warps shared (out = sum_i w_i O_i /
// sum_i w_i l_i with w_i = 2^(m_i - max m), i in the order of the keys) and
// writes zeros to rows that see nothing: sequences of length 0 and rows past
// q_lens.  One block per (pair, key head, row of the tile); its warps take every
// kMergeWarps-th piece and are summed in warp order.
template <typename T>
__global__ void __launch_bounds__(kMergeWarps * 32) split_merge_kernel(Args a) {
  __shared__ float s_m[kMergeWarps], s_l[kMergeWarps];
  __shared__ float s_o[kMergeWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_unit = min(kRows, a.S * a.G);  // rows of a tile that exist
  const int r = blockIdx.x % per_unit;
  const int hk = (blockIdx.x / per_unit) % a.Hkv;
  const int pair = blockIdx.x / per_unit / a.Hkv;
  const int b = pair / a.row_tiles, row = (pair % a.row_tiles) * kRows + r;
  if (row >= a.S * a.G) return;
  const Tile t = tile_of(a, pair);
  const int D = a.D;
  const int64_t head = ((int64_t)b * a.S + row / a.G) * a.Hq + (int64_t)hk * a.G + row % a.G;
  T* dst = static_cast<T*>(a.out) + head * D;
  // all that needs no piece is worked out while the pieces are still being made
  const int nblk = blocks_of(t);
  int64_t before = 0, total = 0;  // blocks of the line before this pair, and in all
  for (int p = lane; p < a.B * a.row_tiles; p += 32) {
    const int64_t n = (int64_t)blocks_of(tile_of(a, p)) * a.Hkv;
    total += n;
    before += p < pair ? n : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  const int64_t first = before + (int64_t)hk * nblk;
  const int64_t used = warps_used(total, a.max_warps, a.min_blocks);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (r >= t.rows) {
    for (int d = threadIdx.x; d < D; d += blockDim.x) dst[d] = rowattn::from_f32<T>(0.f);
    if (a.scores && threadIdx.x == 0) a.row_ml[head * 2] = a.row_ml[head * 2 + 1] = 0.f;
    return;
  }
  const int64_t w0 = piece_owner(total, used, first), w1 = piece_owner(total, used, first + nblk - 1);
  if (w0 == w1) return;  // one warp had it all and wrote it
  auto slot_of = [&](int64_t w) {
    return (2 * w + (piece_start(total, used, w) < first ? 1 : 0)) * kRows + r;
  };
  // this warp's pieces: maximum first, then the sums
  float mx = -INFINITY;
  for (int64_t w = w0 + warp + (int64_t)lane * kMergeWarps; w <= w1; w += 32 * kMergeWarps)
    mx = fmaxf(mx, a.part_ml[slot_of(w) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float acc[2][4] = {};
  float l = 0.f;
#pragma unroll 4
  for (int64_t w = w0 + warp; w <= w1; w += kMergeWarps) {
    const int64_t slot = slot_of(w);
    const float m = a.part_ml[slot * 2];
    const float f = m == -INFINITY ? 0.f : exp2_fast(m - mx);
    l += f * a.part_ml[slot * 2 + 1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int d = (h * 32 + lane) * 4;
      if (d < D) {
        const float4 v = *reinterpret_cast<const float4*>(a.part_o + slot * D + d);
        acc[h][0] += f * v.x;
        acc[h][1] += f * v.y;
        acc[h][2] += f * v.z;
        acc[h][3] += f * v.w;
      }
    }
  }
  if (lane == 0) {
    s_m[warp] = mx;
    s_l[warp] = l;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((h * 32 + lane) * 4 < D) s_o[warp][(h * 32 + lane) * 4 + i] = acc[h][i];
  __syncthreads();
  // A maximum of -inf comes with nothing (a warp that had no piece: sums of 0)
  // or with NaN scores (a maximum passes them over, the sums hold them): the
  // sums are multiplied by 0, not left out, so that a NaN query stays NaN.
  float M = -INFINITY, L = 0.f, f[kMergeWarps];
#pragma unroll
  for (int i = 0; i < kMergeWarps; ++i) M = fmaxf(M, s_m[i]);
#pragma unroll
  for (int i = 0; i < kMergeWarps; ++i) {
    f[i] = s_m[i] == -INFINITY ? 0.f : exp2_fast(s_m[i] - M);
    L += s_l[i] * f[i];
  }
  const float inv = L > 0.f ? 1.0f / L : 0.f;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kMergeWarps; ++i) v += s_o[i][d] * f[i];
    dst[d] = rowattn::from_f32<T>(v * inv);
  }
  if (a.scores && threadIdx.x == 0) {
    a.row_ml[head * 2] = M;
    a.row_ml[head * 2 + 1] = inv;
  }
}

// key_weights[b, hk, j] += sum over the group's heads of 2^(score - max) / sum,
// heads in order.  One thread per visible key.
__global__ void __launch_bounds__(256) split_key_weights_kernel(Args a) {
  const int hk = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv;
  const Seq q = sequence(a, b);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (q.n < 1) return;
  const Span sp = span_of(q, 0, 0, a.window, a.sinks);
  for (int v = blockIdx.y * 256 + threadIdx.x; v < sp.nvis; v += gridDim.y * 256) {
    float sum = 0.f;
    for (int g = 0; g < a.G; ++g) {
      const int64_t head = (int64_t)b * a.Hq + hk * a.G + g;
      sum += exp2_fast(a.scores[head * a.score_ld + v] - a.row_ml[head * 2]) * a.row_ml[head * 2 + 1];
    }
    float* dst = a.key_weights + ((int64_t)b * a.Hkv + hk) * a.weight_ld + sp.key(v);
    *dst += sum;
  }
}

// Every other type and head size up to 256 (fp32, sizes or addresses that do
// not come in 16 bytes): one block per query row, its warps take every 8th
// visible key, fp32 throughout.
constexpr int kAnyWarps = 8;
constexpr int kAnyPerLane = 8;

__global__ void __launch_bounds__(kAnyWarps * 32) split_any_kernel(Args a) {
  __shared__ float s_m[kAnyWarps], s_l[kAnyWarps];
  __shared__ float s_o[kAnyWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = (int)(blockIdx.x % a.Hq);
  const int s = (int)(blockIdx.x / a.Hq % a.S);
  const int b = (int)(blockIdx.x / a.Hq / a.S);
  const int64_t head = ((int64_t)b * a.S + s) * a.Hq + h;
  const Seq q = sequence(a, b, h == 0 && s == 0 && threadIdx.x == 0);
  const int D = a.D;
  if (s >= q.n) {
    for (int d = threadIdx.x; d < D; d += blockDim.x) store_f32(a.out, a.dtype, head * D + d, 0.f);
    return;
  }
  const Span sp = span_of(q, s, s, a.window, a.sinks);
  const int hk = h / a.G;
  float qv[kAnyPerLane], acc[kAnyPerLane];
#pragma unroll
  for (int i = 0; i < kAnyPerLane; ++i) {
    const int d = lane + 32 * i;
    qv[i] = d < D ? load_f32(a.q, a.dtype, head * D + d) : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int v = warp; v < sp.nvis; v += kAnyWarps) {
    const int j = sp.key(v);
    const int64_t pg = resolve_page(a.page_table[b * a.table_stride + j], a.num_pages);
    float x = 0.f;
    int64_t off = 0;
    if (pg < 0) {
      if (lane == 0) record_error(MTP_ERR_DEVICE);
    } else {
      off = (((pg * a.B + b) * a.Hkv + hk) * a.page_size + j % a.page_size) * D;
#pragma unroll
      for (int i = 0; i < kAnyPerLane; ++i) {
        const int d = lane + 32 * i;
        if (d < D) x = fmaf(qv[i], load_f32(a.k_pages, a.dtype, off + d), x);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    x *= a.scale_log2;
    if (a.scores && lane == 0) a.scores[head * a.score_ld + v] = x;
    const float mn = fmaxf(m, x);
    const float use = mn == -INFINITY ? 0.f : mn;
    const float corr = exp2f(m - use), p = exp2f(x - use);
    l = l * corr + p;
#pragma unroll
    for (int i = 0; i < kAnyPerLane; ++i) {
      const int d = lane + 32 * i;
      if (d < D) acc[i] = acc[i] * corr + (pg < 0 ? 0.f : p * load_f32(a.v_pages, a.dtype, off + d));
    }
    m = mn;
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < kAnyPerLane; ++i)
    if (lane + 32 * i < D) s_o[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  float M = -INFINITY, L = 0.f, f[kAnyWarps];
#pragma unroll
  for (int i = 0; i < kAnyWarps; ++i) M = fmaxf(M, s_m[i]);
#pragma unroll
  for (int i = 0; i < kAnyWarps; ++i) {
    f[i] = s_m[i] == -INFINITY ? 0.f : exp2f(s_m[i] - M);
    L += s_l[i] * f[i];
  }
  const float inv = L > 0.f ? 1.0f / L : 0.f;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kAnyWarps; ++i) v += s_o[i][d] * f[i];
    store_f32(a.out, a.dtype, head * D + d, v * inv);
  }
  if (a.scores && threadIdx.x == 0) {
    a.row_ml[head * 2] = M;
    a.row_ml[head * 2 + 1] = inv;
  }
}

}  // namespace split
}  // namespace mtp
